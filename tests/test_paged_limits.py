"""Sizes and strides that the paged cache's C entry points refuse before a launch: numbers past
32 bits that would be cut to legal ones, and layers that would overlap or lie before the pool."""
import pytest

from test_paged_host import P, append, attend, lib, read  # noqa: F401

BIG = 1 << 32


@pytest.mark.parametrize("call", [append, attend, read])
@pytest.mark.parametrize("page", [BIG + 32, BIG * 16 + 16, -BIG + 64])
def test_page_tokens_past_32_bits(lib, call, page):  # noqa: F811
    assert call(lib, page=page, total=0) == 1 and b"page_tokens" in lib.kvq_last_error()


@pytest.mark.parametrize("page", [BIG + 32, -BIG + 32, 24, 0])
def test_page_tokens_of_the_page_operations(lib, page):  # noqa: F811
    assert lib.kvq_paged_free(P, 3, 2, P, P, 4, page, None, 0, P, None) == 1
    assert lib.kvq_paged_fork(P, 3, 2, P, P, 4, page, None, None, 0, P, None) == 1
    ws = lib.kvq_paged_extend_workspace(4)
    assert lib.kvq_paged_extend(P, 2, 4096, 1024, P, 3, 2, P, P, 4, page, None, 0, None, 0, P, P, ws,
                                None) == 1


@pytest.mark.parametrize("page_bytes", [1 << 33, 1 << 61, 1 << 62])
def test_page_bytes_whose_pool_passes_64_bits(lib, page_bytes):  # noqa: F811
    ws = lib.kvq_paged_extend_workspace(4)
    assert lib.kvq_paged_extend(P, 2, 0, page_bytes, P, 3, 2, P, P, 4, 32, None, 0, None, 0, P, P, ws,
                                None) == 1
    assert lib.kvq_paged_copy(P, 4, 0, P, 4, 0, 1, page_bytes, None, None, 0, None, 0, None) == 1


@pytest.mark.parametrize("strides", [(4096, 4080), (4080, 4096), (-4096, 4096), (4096, 0)])
def test_layers_of_a_copy_do_not_overlap(lib, strides):  # noqa: F811
    copy = lambda layers, a, b: lib.kvq_paged_copy(  # noqa: E731
        P, 4, a, P, 4, b, layers, 1024, None, None, 0, None, 0, None)
    assert copy(2, *strides) == 1 and copy(1, *strides) == 0 and copy(2, 4096, 8192) == 0
