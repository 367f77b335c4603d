"""The paged 8-bit cache at the ends of what its calls accept."""
import numpy as np
import pytest
import torch

from paged_cases import Cache, check, expected
from test_gpu_paged_attention import run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 5, 2 ** 30])
@pytest.mark.parametrize("max_new", [None, 64])  # the kernel of few rows, that of many
def test_windows_that_hide_nothing(cuda, window, max_new):
    """Windows up to the largest 32-bit number, with more rows than tokens: rows before the
    first token see nothing, the others everything before them."""
    c = Cache([3, 40, 0, 131], kind="e4m3", seed=21)
    new, G = [6, 2, 4, 1], 3
    q = c.queries(new, G)
    out, ml = run(cuda, c, q, new, G, window=window, max_new=max_new)
    e_out, e_ml, b_out, b_ml = expected(c, q, new, G)
    assert (out[:3] == 0).all() and np.isneginf(ml[:3, :, 0]).all()
    check(out, e_out, b_out, "out")
    check(ml, e_ml, b_ml, "ml")


@pytest.mark.parametrize("n", [255, 256, 257, 1000])
def test_copy_of_many_pages(cuda, n):
    """Lists longer than one scan of the planning block, with pairs out of range among them."""
    from kvquant.kernels import paged_copy
    from kvquant.kernels.cuda_ops import get_cuda_ops
    rng = np.random.default_rng(n)
    a, b = (rng.integers(0, 256, (2, n + 3, 1, 1, 32 * 64 + 16), dtype=np.uint8) for _ in range(2))
    src, dst = (rng.integers(0, n + 3, n), rng.permutation(n + 3)[:n])
    bad = rng.random(n) < 0.1
    src[bad & (rng.random(n) < 0.5)] = -1
    dst[bad & (src >= 0)] = n + 3
    t = lambda x: torch.from_numpy(np.ascontiguousarray(x)).to(cuda)  # noqa: E731
    ga, gb = t(a), t(b)
    paged_copy(ga, gb, t(src.astype(np.int32)), t(dst.astype(np.int32)))
    with pytest.raises(RuntimeError, match="out of range"):
        get_cuda_ops().check_status(cuda)
    b[:, dst[~bad]] = a[:, src[~bad]]
    np.testing.assert_array_equal(gb.cpu().numpy(), b)
    np.testing.assert_array_equal(ga.cpu().numpy(), a)


def test_extend_by_more_pages_than_32_bits_count(cuda):
    """17 slots of 134217727 pages each: their sum is past 2**31. The call is refused and the
    table (9 GB) stays as it is."""
    from kvquant.kernels import paged_extend
    from kvquant.kernels.paged import NO_PAGES, pool_shape
    ints = dict(dtype=torch.int32, device=cuda)
    n, cols = 17, (2 ** 31 - 1) // 16
    pool = torch.zeros(pool_shape(8, 1, 64, 16), dtype=torch.uint8, device=cuda)
    table = torch.full((n, cols), -1, **ints)
    lengths, refs, status = torch.zeros(n, **ints), torch.zeros(8, **ints), torch.zeros(1, **ints)
    slots = torch.arange(n, **ints)
    paged_extend(pool, table, lengths, refs, slots, torch.full((n,), 16 * cols, **ints), status)
    assert int(status.item()) == NO_PAGES
    assert int(table.max().item()) == -1 and int(table.min().item()) == -1
    assert not lengths.any() and not refs.any()
    paged_extend(pool, table, lengths, refs, slots[:8], 16, status)
    assert torch.equal(table[:8, 0], slots[:8]) and refs.eq(1).all() and lengths[:8].eq(16).all()


def test_more_rows_than_any_sequence_may_have(cuda):
    """80000 rows of 40 prompts, without max_new: no sequence is near the limit of 65536."""
    from kvquant.kernels import paged_attention
    from kvquant.kernels.cuda_ops import get_cuda_ops
    c = Cache([2000], H=1, D=64, page=64, seed=22)
    pool, table, lengths = c.gpu(cuda)
    table, lengths = table.repeat(40, 1), lengths.repeat(40)  # the same pages for all
    q = torch.from_numpy(c.queries([2000], 1)).to(cuda).half().repeat(40, 1, 1)
    ip = torch.arange(0, 80001, 2000, dtype=torch.int32, device=cuda)
    got = paged_attention(q, pool, table, lengths, "int8", indptr=ip)
    get_cuda_ops().check_status(cuda)
    want = paged_attention(q, pool, table, lengths, "int8", indptr=ip, max_new=2000)
    assert torch.equal(got, want)
    out, _, bound, _ = expected(c, q[:2000].float().cpu().numpy(), [2000], 1)
    for i in (0, 17, 39):
        check(got[2000 * i:2000 * (i + 1)].float().cpu().numpy(), out, bound, f"prompt {i}")
