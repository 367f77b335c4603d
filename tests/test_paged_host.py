"""Paged 8-bit cache without a GPU: the oracle's codes and records, and every argument
that the library refuses before a launch."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import paged_oracle as PO


@pytest.fixture(scope="module")
def lib():
    from kvquant.kernels.cuda_ops import load_library
    return load_library()


def test_oracle_e4m3_codes_equal_the_framework_cast():
    rng = np.random.default_rng(0)
    y = (rng.standard_normal(100000) * np.exp(rng.uniform(-8, 6, 100000))).astype(np.float32)
    mid = PO.e4m3_values()[:126].astype(np.float32)
    y = np.concatenate([y, mid, (mid + PO.e4m3_values()[1:127].astype(np.float32)) / 2])
    y = np.clip(y, -448, 448)
    want = torch.from_numpy(y).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    np.testing.assert_array_equal(PO.encode(y, "e4m3"), want)


@pytest.mark.parametrize("D", [64, 128])
def test_record_maps_cover_every_byte_once(D):
    key, val = PO.record_maps(D)
    assert sorted(key.ravel()) == list(range(16 * D))
    assert sorted(val.ravel()) == list(range(16 * D, 32 * D))


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_oracle_append_error(kind):
    """A block written at once is within half a code of its tokens."""
    rng = np.random.default_rng(1)
    pool = np.zeros((2, 1, 1, 32 * 64 + 16), np.uint8)
    k, v = (rng.standard_normal((16, 1, 64)).astype(np.float32) for _ in range(2))
    PO.append(pool, np.array([[1, 0]]), 0, 16, k, v, kind)
    gk, gv, _ = PO.token_values(pool, np.array([[1, 0]]), 0, 16, 0, 64, kind)
    for x, y in ((k, gk), (v, gv)):
        s = np.abs(x).max() / float(PO.QMAX[kind])
        # int8: half a step; e4m3: 2**-4 of the value or half the least step
        tol = s / 2 if kind == "int8" else np.maximum(np.abs(x[:, 0]) * 2.0 ** -4, s * 2.0 ** -10)
        assert (np.abs(x[:, 0] - y) <= tol * 1.001).all()


P = ctypes.c_void_p(256)  # stands for an aligned pointer; nothing is read from it


def append(lib, **kw):
    a = dict(k=P, kt=256, kh=128, v=P, vt=256, vh=128, dtype=0, pool=P, kind=0, pages=4, heads=2,
             dim=128, page=32, table=P, slots=3, cols=2, lengths=P, sl=None, ip=None, B=3, total=3)
    a.update(kw)
    return lib.kvq_paged_append(*a.values(), None)


def attend(lib, **kw):
    a = dict(q=P, qt=1024, qh=128, dtype=0, group=4, pool=P, kind=0, pages=4, heads=2, dim=128,
             page=32, table=P, slots=3, cols=2, lengths=P, sl=None, ip=None, B=3, total=3,
             max_new=1, scale=0.1, window=0, out=P, ml=None, ws=P, wsb=1 << 40)
    a.update(kw)
    return lib.kvq_paged_attention(*a.values(), None)


def read(lib, **kw):
    a = dict(pool=P, kind=0, pages=4, heads=2, dim=128, page=32, table=P, slots=3, cols=2,
             lengths=P, sl=None, starts=None, ip=None, B=3, total=3, k=P, v=P, dtype=0)
    a.update(kw)
    return lib.kvq_paged_read(*a.values(), None)


BAD_CACHE = [(dict(dim=96), 3, b"head_dim"), (dict(kind=2), 3, b"kind"),
             (dict(page=24), 1, b"page_tokens"), (dict(page=2048), 1, b"page_tokens"),
             (dict(page=0), 1, b"page_tokens"), (dict(pages=0), 1, b"impossible"),
             (dict(heads=-1), 1, b"impossible"), (dict(cols=0), 1, b"impossible"),
             (dict(B=0), 1, b"sequences"), (dict(B=4), 1, b"sequences"),
             (dict(B=5000, sl=P), 1, b"sequences"), (dict(total=4), 1, b"divide"),
             (dict(total=-1), 1, b"divide"), (dict(pool=None), 1, b"aligned"),
             (dict(pool=ctypes.c_void_p(8)), 1, b"aligned"), (dict(table=None), 1, b"aligned"),
             (dict(lengths=None), 1, b"aligned")]


@pytest.mark.parametrize("call", [append, attend, read])
@pytest.mark.parametrize("kw,rc,what", BAD_CACHE)
def test_cache_arguments_are_checked(lib, call, kw, rc, what):
    assert call(lib, **kw) == rc and what in lib.kvq_last_error()


@pytest.mark.parametrize("call,kw,rc,what", [
    (append, dict(dtype=2), 3, b"dtype"), (append, dict(k=None), 1, b"aligned"),
    (append, dict(v=ctypes.c_void_p(8)), 1, b"aligned"), (append, dict(kt=132), 1, b"strides"),
    (attend, dict(dtype=2), 3, b"dtype"), (attend, dict(group=65), 3, b"query heads"),
    (attend, dict(group=0), 3, b"query heads"), (attend, dict(max_new=0), 1, b"max_new"),
    (attend, dict(max_new=0, ip=P), 1, b"max_new"), (attend, dict(window=-1), 1, b"window"), (attend, dict(q=None), 1, b"aligned"),
    (attend, dict(out=ctypes.c_void_p(8)), 1, b"aligned"), (attend, dict(wsb=64), 1, b"workspace"),
    (attend, dict(ws=None), 1, b"workspace"), (attend, dict(ml=ctypes.c_void_p(4)), 1, b"aligned"),
    (read, dict(dtype=3), 3, b"dtype"), (read, dict(k=None), 1, b"aligned"),
])
def test_call_arguments_are_checked(lib, call, kw, rc, what):
    assert call(lib, **kw) == rc and what in lib.kvq_last_error()


def test_empty_calls_launch_nothing(lib):
    assert append(lib, total=0) == 0 and attend(lib, total=0) == 0 and read(lib, total=0) == 0


def test_page_operations_check_their_arguments(lib):
    meta = (P, 3, 2, P, P, 4, 32)
    assert lib.kvq_paged_free(*meta, P, 5000, P, None) == 1
    assert lib.kvq_paged_free(None, 3, 2, P, P, 4, 32, P, 1, P, None) == 1
    assert lib.kvq_paged_free(*meta, P, 1, None, None) == 1
    assert lib.kvq_paged_free(*meta, None, 0, P, None) == 0
    assert lib.kvq_paged_fork(*meta, P, None, 1, P, None) == 1
    assert lib.kvq_paged_fork(P, 3, 2, P, P, 4, 20, P, P, 1, P, None) == 1
    ws = lib.kvq_paged_extend_workspace(4)
    ext = lambda pool=P, layers=2, stride=4096, page=1024, n=1, new=1, w=P, wb=ws: (  # noqa: E731
        lib.kvq_paged_extend(pool, layers, stride, page, *meta, P, n, None, new, P, w, wb, None))
    for kw in (dict(pool=None), dict(layers=0), dict(stride=1024), dict(page=1000), dict(n=5000),
               dict(new=-1), dict(w=None), dict(wb=ws - 1)):
        assert ext(**kw) == 1, kw
    assert ext(n=0) == 0
    com = lambda stride=4096, live=P, w=P, wb=ws: lib.kvq_paged_compact(  # noqa: E731
        P, 2, stride, 1024, P, 3, 2, P, 4, live, w, wb, None)
    for kw in (dict(stride=16), dict(live=None), dict(w=None), dict(wb=8)):
        assert com(**kw) == 1, kw
    assert lib.kvq_paged_copy(P, 4, 0, P, 4, 0, 1, 1024, P, P, -1, P, 1 << 20, None) == 1
    assert lib.kvq_paged_copy(P, 4, 0, P, 4, 0, 1, 1024, P, P, 2, P, 8, None) == 1
    assert lib.kvq_paged_copy(P, 4, 0, P, 4, 0, 1, 1024, None, None, 0, None, 0, None) == 0


def test_python_wrappers_refuse_cpu_tensors_and_wrong_shapes():
    from kvquant.kernels import paged_append, paged_attention, paged_free, paged_read
    pool = torch.zeros((2, 1, 2, 32 * 64 + 16), dtype=torch.uint8)
    table, lengths = torch.zeros((1, 2), dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    x = torch.zeros((1, 1, 64), dtype=torch.float16)
    for call in (lambda: paged_append(x, x, pool, table, lengths, "int8"),
                 lambda: paged_attention(x, pool, table, lengths, "int8"),
                 lambda: paged_read(pool, table, lengths, "int8", None, None, 1),
                 lambda: paged_free(table, lengths, lengths, lengths, 32, lengths)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
