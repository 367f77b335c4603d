"""The paged attention where its loops take their later turns: hundreds to thousands of
sequences, large groups, heads and pages; and the rows that go wrong first (rows that see
nothing, hidden and extreme scores, scales of either sign) in the kernel of many rows too.

Bounds as in test_gpu_paged_attention. A large max_new sends a call to the kernel of many rows.
"""
import numpy as np
import pytest
import torch

from oracle import paged_oracle as PO
from paged_cases import DT, Cache, check, expected, make_tokens, rounded
from test_gpu_paged_attention import compare, run

pytestmark = pytest.mark.gpu

# 24 to 48 rows in all: without max_new the kernel of few rows
KERNELS = pytest.mark.parametrize("max_new", [None, 300])


# ---------------------------------------------------------------- many sequences
@pytest.mark.parametrize("B", [129, 385, 513, 1025, 4096])
@pytest.mark.parametrize("max_new", [2, 64])
def test_many_sequences(cuda, B, max_new):
    """Past every block-wide scan's width and the sequences kept in shared memory; some
    sequences without tokens, some without rows."""
    rng = np.random.default_rng(B)
    lens = [int(x) for x in rng.integers(0, 50, B)]
    new = [int(x) for x in rng.integers(0, 3, B)]
    lens[3], new[3], lens[B - 1], new[B - 1] = 0, 1, 400, 2
    c = Cache(lens, H=1, D=64, page=16, kind="e4m3", seed=B)
    compare(cuda, c, new, 2, max_new=max_new)


@pytest.mark.parametrize("B", [513, 2000])
def test_many_prompts(cuda, B):
    """Whole prompts of 1 to 40 tokens (up to 320 rows a sequence), in the order of other slots."""
    rng = np.random.default_rng(B)
    c = Cache([int(x) for x in rng.integers(1, 41, B + 5)], H=1, D=64, page=32, dtype="bf16", seed=B)
    slots = [int(s) for s in rng.permutation(B + 5)[:B]]
    compare(cuda, c, [c.lens[s] for s in slots], 8, slots=slots, max_new=40)


def test_thousands_of_sequences_with_one_token_each(cuda):
    """A uniform batch (no indptr) that holds the same pages: every sequence gives one answer."""
    from kvquant.kernels import paged_attention
    B, G = 4096, 4
    c = Cache([301], H=2, D=128, page=64, dtype="bf16", seed=1)
    pool, table, lengths = c.gpu(cuda)
    q = c.queries([1], G)
    qt = torch.from_numpy(q).to(cuda).to(DT["bf16"]).expand(B, 2 * G, 128)
    got = paged_attention(qt, pool, table.repeat(B, 1), lengths.repeat(B), "int8")
    out, _, bound, _ = expected(c, q, [1], G)
    far = (got.double() - torch.from_numpy(out).to(cuda)).abs() - torch.from_numpy(bound).to(cuda)
    assert float(far.max()) <= 0


# ---------------------------------------------------------------- large groups, heads, pages
@pytest.mark.parametrize("G,new", [(64, [1, 2]), (48, [1, 1]), (33, [3, 1]), (24, [2, 1]), (24, [1, 1])])
def test_large_groups(cuda, G, new):
    compare(cuda, Cache([40, 333], H=1, seed=G), new, G)


@pytest.mark.parametrize("H,page,D", [(32, 1024, 64), (40, 512, 128)])
@KERNELS
def test_heads_and_large_pages(cuda, H, page, D, max_new):
    c = Cache([1030, 70], H=H, D=D, page=page, kind="e4m3", spare=1, seed=H)
    compare(cuda, c, [1, 1], 1, max_new=max_new)


# ---------------------------------------------------------------- edges, in both kernels
@KERNELS
def test_rows_that_see_nothing(cuda, max_new):
    """More rows than tokens, no tokens at all; with a window too."""
    c = Cache([0, 3, 20, 260], seed=4)
    new = [2, 5, 1, 3]
    for window in (0, 2, 100):
        q = c.queries(new, 2)
        out, ml = run(cuda, c, q, new, 2, window, max_new=max_new)
        e_out, e_ml, b_out, b_ml = expected(c, q, new, 2, window)
        assert (out[:4] == 0).all() and np.isneginf(ml[:4, :, 0]).all()
        assert np.isposinf(ml[:4, :, 1]).all()
        check(out, e_out, b_out, "out")
        check(ml, e_ml, b_ml, "ml")


@KERNELS
@pytest.mark.parametrize("scale", [0.5, -0.1, 0.0])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_scales(cuda, max_new, scale, dtype):
    compare(cuda, Cache([300, 17, 140], dtype=dtype, seed=8), [1, 2, 9], 2, scale=scale, max_new=max_new)


def test_chunks_with_a_negative_scale(cuda):
    compare(cuda, Cache([700, 420], H=1, kind="e4m3", seed=9), [150, 290], 4, scale=-0.07)


@KERNELS
@pytest.mark.parametrize("grow", [False, True])
def test_value_blocks_far_apart(cuda, max_new, grow):
    """Value blocks 2**-14 to 2**12 apart, in turn or growing, and blocks of zeros: the
    reference of the weights moves on again and again."""
    c = Cache([352, 96], H=1, seed=12, fill=False)
    for i, n in enumerate(c.lens):
        k, v = make_tokens(c.rng, n, 1, 128)
        for blk in range(n // 16):
            v[16 * blk:16 * blk + 16] *= 2.0 ** (-14 + (26 * blk * 16 / n if grow else 13 * (blk % 3)))
        v[32:48] = 0
        k[16:32] = 0
        PO.append(c.pool, c.table, i, n, rounded(k, "fp16"), rounded(v, "fp16"), "int8")
    compare(cuda, c, [4, 8], 4, max_new=max_new)


@KERNELS
def test_scores_that_grow(cuda, max_new):
    """Keys that grow along the context: the maximum moves in every block, by less and by
    more than the lag that the kernel of many rows allows it."""
    c = Cache([520], H=1, seed=13, fill=False)
    k, v = make_tokens(c.rng, 520, 1, 128)
    k *= np.linspace(0.01, 3, 520, dtype=np.float32)[:, None, None]
    PO.append(c.pool, c.table, 0, 520, rounded(k, "fp16"), rounded(v, "fp16"), "int8")
    compare(cuda, c, [12], 4, scale=0.3, max_new=max_new)


@KERNELS
@pytest.mark.parametrize("size", [2.0 ** -30, 2.0 ** 30, 60000.0])
def test_extreme_queries(cuda, max_new, size):
    dtype = "fp16" if size == 60000.0 else "bf16"
    c = Cache([170], dtype=dtype, seed=13)
    q = c.queries([20], 2)
    q = q / np.abs(q).max() * np.float32(size)
    q[0, 0] = 0
    q = rounded(q, dtype)
    out, ml = run(cuda, c, q, [20], 2, scale=1.0 / size, max_new=max_new)
    e = expected(c, q, [20], 2, scale=1.0 / size)
    check(out, e[0], e[2], "out")
    check(ml, e[1], e[3], "ml")


@KERNELS
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_non_finite_queries_stay_in_their_rows(cuda, max_new, bad, dtype):
    """One element of a row, and a whole row: the other rows do not change."""
    c = Cache([170, 33], dtype=dtype, seed=14)
    new, G = [10, 2], 4
    q = c.queries(new, G)
    q[1, 3], q[7, 2, 5] = bad, bad
    out, ml = run(cuda, c, q, new, G, max_new=max_new)
    assert np.isnan(out[1, 3]).all()
    q[1, 3] = q[7, 2] = 0
    e_out, e_ml, b_out, b_ml = expected(c, q, new, G)
    for x, e in ((out, e_out), (ml, e_ml)):
        x[1, 3] = e[1, 3] = x[7, 2] = e[7, 2] = 0
    check(out, e_out, b_out, "out")
    check(ml, e_ml, b_ml, "ml")


@KERNELS
def test_bad_indices(cuda, max_new):
    """A bad page, length, slot or row range: reported, and the other sequence's rows hold."""
    from kvquant.kernels import paged_attention
    from kvquant.kernels.cuda_ops import get_cuda_ops
    ops = get_cuda_ops()
    c = Cache([40, 64], seed=18)
    pool, table, lengths = c.gpu(cuda)
    q = torch.from_numpy(c.queries([1, 1], 2)).to(cuda).half()
    good = paged_attention(q, pool, table, lengths, "int8", max_new=max_new)
    for what in ("page", "length", "slot", "rows"):
        t, n, slots, ip = table.clone(), lengths.clone(), None, None
        if what == "page":
            t[0, 1] = pool.shape[0]
        elif what == "length":
            n[0] = t.shape[1] * c.page + 1
        elif what == "slot":
            slots = torch.tensor([2, 1], dtype=torch.int32, device=cuda)
        else:
            ip = torch.tensor([5, 1, 2], dtype=torch.int32, device=cuda)
        got = paged_attention(q, pool, t, n, "int8", slots=slots, indptr=ip, max_new=max_new or 2)
        with pytest.raises(RuntimeError, match="out of range"):
            ops.check_status(cuda)
        assert torch.equal(got[1], good[1]), what


@KERNELS
def test_repeats_agree_bit_for_bit(cuda, max_new):
    """Units cut by the shares' ends are joined in a fixed order."""
    from kvquant.kernels import paged_attention
    c = Cache([500, 900, 33], H=4, seed=16)
    pool, table, lengths = c.gpu(cuda)
    q = torch.from_numpy(c.queries([3, 3, 3], 4)).to(cuda).half()
    first = paged_attention(q, pool, table, lengths, "int8", max_new=max_new)
    for _ in range(20):
        assert torch.equal(paged_attention(q, pool, table, lengths, "int8", max_new=max_new), first)
