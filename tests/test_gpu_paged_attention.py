"""Attention over the paged 8-bit cache against float64, element by element.

The bounds come from the number of roundings (oracle.paged_oracle.attention). The
pools hold NaN bytes wherever no token is stored, and pages lie in shuffled order.
"""
import numpy as np
import pytest
import torch

from paged_cases import DT, Cache, check, expected

pytestmark = pytest.mark.gpu


def indptr_of(new):
    return np.concatenate([[0], np.cumsum(new)]).astype(np.int32)


def run(cuda, c, q, new, G, window=0, scale=None, slots=None, uniform=False, max_new=None):
    from kvquant.kernels import paged_attention
    from kvquant.kernels.cuda_ops import get_cuda_ops
    pool, table, lengths = c.gpu(cuda)
    qt = torch.from_numpy(q).to(cuda).to(DT[c.dtype])
    ml = torch.full((q.shape[0], c.H * G, 2), 7.0, device=cuda)
    ip = None if uniform else torch.from_numpy(indptr_of(new)).to(cuda)
    st = None if slots is None else torch.tensor(slots, dtype=torch.int32, device=cuda)
    out = paged_attention(qt, pool, table, lengths, c.kind, slots=st, indptr=ip, window=window,
                          scale=scale, ml_out=ml, max_new=max_new)
    get_cuda_ops().check_status(cuda)
    return out.float().cpu().numpy(), ml.cpu().numpy()


def compare(cuda, c, new, G, window=0, scale=None, slots=None, **kw):
    q = c.queries(new, G)
    out, ml = run(cuda, c, q, new, G, window, scale, slots, **kw)
    e_out, e_ml, b_out, b_ml = expected(c, q, new, G, window, scale, slots)
    check(out, e_out, b_out, "out")
    check(ml, e_ml, b_ml, "ml")


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
def test_single_token(cuda, kind, dtype, D):
    """Lengths around the block, tile and page ends, one query token each."""
    lens = [1, 2, 15, 16, 17, 31, 32, 33, 129, 700]
    compare(cuda, Cache(lens, H=3, D=D, page=32, kind=kind, dtype=dtype, seed=D), [1] * len(lens), 4,
            uniform=True)


@pytest.mark.parametrize("G", [1, 2, 3, 7, 8, 12])
def test_groups(cuda, G):
    compare(cuda, Cache([40, 333], H=2, seed=G), [1, 1], G, uniform=True)


@pytest.mark.parametrize("page", [16, 48, 64, 128])
def test_pages(cuda, page):
    compare(cuda, Cache([5, 130, 391], page=page, kind="e4m3", seed=page), [1, 1, 1], 2)


@pytest.mark.parametrize("window", [1, 2, 16, 17, 100, 5000])
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_window(cuda, window, kind):
    compare(cuda, Cache([3, 130, 391], kind=kind, dtype="bf16", seed=window), [1, 5, 40], 3,
            window=window)


@pytest.mark.parametrize("new", [[5, 0, 3, 1], [16, 1, 0, 2], [33, 20, 7, 64]])
@pytest.mark.parametrize("D", [64, 128])
def test_ragged_new_tokens(cuda, new, D):
    compare(cuda, Cache([200, 64, 33, 64], D=D, seed=sum(new)), new, 4)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("D,G", [(64, 4), (128, 2), (128, 5)])
def test_prompt_chunks(cuda, kind, D, G):
    """Chunks of hundreds of rows: a whole prompt, and one behind a cached prefix."""
    compare(cuda, Cache([290, 401, 150], H=2, D=D, page=64, kind=kind, dtype="bf16", seed=G),
            [290, 131, 150], G)


def test_chunk_window(cuda):
    compare(cuda, Cache([500, 260], H=1, page=16, seed=3), [200, 260], 4, window=77)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_long_context(cuda, dtype):
    compare(cuda, Cache([20011, 300], H=1, page=128, kind="e4m3", dtype=dtype, seed=9), [1, 2], 2)


def test_empty_rows(cuda):
    """A sequence without tokens, and more query rows than tokens: rows that see nothing."""
    c = Cache([0, 3, 20], seed=4)
    new = [2, 5, 1]
    q = c.queries(new, 2)
    out, ml = run(cuda, c, q, new, 2)
    e_out, e_ml, b_out, b_ml = expected(c, q, new, 2)
    assert (out[:4] == 0).all() and np.isneginf(ml[:4, :, 0]).all() and np.isposinf(ml[:4, :, 1]).all()
    check(out, e_out, b_out, "out")
    check(ml, e_ml, b_ml, "ml")


def test_slots_and_order(cuda):
    """Sequences in another order than their slots, some slots left out."""
    c = Cache([50, 7, 300, 0, 129], seed=6)
    compare(cuda, c, [1, 3, 2], 4, slots=[4, 0, 2])


def test_scale_and_sign(cuda):
    c = Cache([100, 17], seed=8)
    compare(cuda, c, [1, 2], 2, scale=0.5)
    compare(cuda, c, [1, 2], 2, scale=-0.1)


def test_block_scales_far_apart(cuda):
    """Value blocks from 2**-14 to 2**12 of each other, and a block of zeros: the weights
    are relative to the largest contribution."""
    from oracle import paged_oracle as PO
    from paged_cases import make_tokens, rounded
    c = Cache([96, 64], H=1, seed=12, fill=False)
    for i, n in enumerate(c.lens):
        k, v = make_tokens(c.rng, n, 1, 128)
        for blk in range(n // 16):
            v[16 * blk:16 * blk + 16] *= 2.0 ** (-14 + 13 * (blk % 3))
        if i:
            v[32:48] = 0
            k[16:32] = 0
        PO.append(c.pool, c.table, i, n, rounded(k, "fp16"), rounded(v, "fp16"), "int8")
    compare(cuda, c, [1, 4], 4)


@pytest.mark.parametrize("size", [2.0 ** -30, 2.0 ** 30, 60000.0])
def test_queries_of_extreme_size(cuda, size):
    dtype = "fp16" if size == 60000.0 else "bf16"
    c = Cache([70], dtype=dtype, seed=13)
    q = c.queries([2], 2)
    q = q / np.abs(q).max() * np.float32(size)
    q[0, 0] = 0
    q = torch.from_numpy(q).to(DT[dtype]).float().numpy()
    scale = 1.0 / size
    out, ml = run(cuda, c, q, [2], 2, scale=scale)
    e = expected(c, q, [2], 2, scale=scale)
    check(out, e[0], e[2], "out")
    check(ml, e[1], e[3], "ml")


def test_nan_query_stays_in_its_row(cuda):
    c = Cache([70, 33], seed=14)
    q = c.queries([1, 2], 4)
    q[1, 3] = np.nan
    out, ml = run(cuda, c, q, [1, 2], 4)
    assert np.isnan(out[1, 3]).all()
    q[1, 3] = 0
    e_out, _, b_out, _ = expected(c, q, [1, 2], 4)
    out[1, 3], e_out[1, 3] = 0, 0
    check(out, e_out, b_out, "out")


def test_strided_queries_and_other_stream(cuda):
    from kvquant.kernels import paged_attention
    c = Cache([90, 41], seed=15)
    q = c.queries([3, 1], 4)
    pool, table, lengths = c.gpu(cuda)
    wide = torch.zeros((4, 3, 8, 128), dtype=torch.float16, device=cuda)  # q of a fused q, k, v
    wide[:, 1] = torch.from_numpy(q).to(cuda).half()
    ip = torch.tensor([0, 3, 4], dtype=torch.int32, device=cuda)
    want = paged_attention(wide[:, 1].contiguous(), pool, table, lengths, "int8", indptr=ip)
    stream = torch.cuda.Stream(cuda)
    stream.wait_stream(torch.cuda.current_stream(cuda))
    with torch.cuda.stream(stream):
        got = paged_attention(wide[:, 1], pool, table, lengths, "int8", indptr=ip)
    stream.synchronize()
    assert torch.equal(got, want)


def test_repeatable_and_captured_in_a_graph(cuda):
    """Two calls agree bit for bit; a captured call follows lengths that change later."""
    from kvquant.kernels import DecodeWorkspace, paged_attention
    c = Cache([500, 900, 33], H=4, seed=16)
    q = torch.from_numpy(c.queries([1, 1, 1], 4)).to(cuda).half()
    pool, table, lengths = c.gpu(cuda)
    ws = DecodeWorkspace()
    a = paged_attention(q, pool, table, lengths, "int8", workspace=ws)
    b = paged_attention(q, pool, table, lengths, "int8", workspace=ws)
    assert torch.equal(a, b)
    out = torch.empty_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged_attention(q, pool, table, lengths, "int8", out=out, workspace=ws)
    graph.replay()
    assert torch.equal(out, a)
    lengths.copy_(torch.tensor([17, 640, 1], dtype=torch.int32))
    graph.replay()
    want = paged_attention(q, pool, table, lengths, "int8")
    assert torch.equal(out, want) and not torch.equal(out, a)


def test_merge_with_another_part_of_the_context(cuda):
    """Two caches holding halves of a context join through merge_shards."""
    from kvquant.kernels import merge_shards, paged_attention
    whole = Cache([480], H=2, seed=17)
    pool, table, lengths = whole.gpu(cuda)
    q = torch.from_numpy(whole.queries([1], 4)).to(cuda).half()
    ml0, ml1, ml = (torch.empty((1, 8, 2), device=cuda) for _ in range(3))
    want = paged_attention(q, pool, table, lengths, "int8", ml_out=ml)
    half = torch.tensor([224], dtype=torch.int32, device=cuda)
    rest = torch.tensor([256], dtype=torch.int32, device=cuda)
    a = paged_attention(q, pool, table, half, "int8", ml_out=ml0)
    b = paged_attention(q, pool, table[:, 7:].contiguous(), rest, "int8", ml_out=ml1)
    got = merge_shards(torch.stack([a, b]), torch.stack([ml0, ml1]))
    # each part is rounded to fp16 (2**-11 of it), then the result
    scale = (a.float().abs() + b.float().abs())
    assert ((got.float() - want.float()).abs() <= 2.0 ** -9 * scale + 2.0 ** -20).all()


def test_bad_indices_are_reported_and_skipped(cuda):
    from kvquant.kernels import paged_attention
    from kvquant.kernels.cuda_ops import get_cuda_ops
    ops = get_cuda_ops()
    c = Cache([40, 64], seed=18)
    pool, table, lengths = c.gpu(cuda)
    q = torch.from_numpy(c.queries([1, 1], 2)).to(cuda).half()
    good = paged_attention(q, pool, table, lengths, "int8")
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
        got = paged_attention(q, pool, t, n, "int8", slots=slots, indptr=ip, max_new=2)
        with pytest.raises(RuntimeError, match="out of range"):
            ops.check_status(cuda)
        assert torch.equal(got[1], good[1]), what


@pytest.mark.parametrize("kind,D,G,lens,new,window", [
    ("int8", 128, 4, [2600] * 6, [70] * 6, 0),        # many token tiles and units per SM
    ("e4m3", 64, 4, [1800, 2900, 5, 700] * 4, [5] * 16, 1000),
    ("int8", 64, 8, [900] * 8, [17, 40, 33, 64, 3, 0, 100, 900], 0),
])
def test_many_tiles_per_sm(cuda, kind, D, G, lens, new, window):
    """More work than one token tile per SM: rings and slots are used many times over."""
    c = Cache(lens, H=3, D=D, page=32, kind=kind, dtype="bf16", seed=D + G)
    compare(cuda, c, new, G, window=window)
