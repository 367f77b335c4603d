"""Attention over the paged 8-bit cache where one block's value scale dwarfs the others':
every output element against a bound on its own terms.

An output is a sum of p_j v_j over the tokens. Besides the roundings that scale with its
own terms sum_j p_j |v_j| (weights 2**-11, scores, fp32 sums) it may carry only the step of
fp16 subnormals, 2**-36 of the largest contribution p_j vs_j of any block, per code unit:
weights are held relative to that contribution and lifted by at least 2**11 into fp16's range,
whose least step is 2**-24 (half of it rounds).
"""
import numpy as np
import pytest
import torch

from oracle import paged_oracle as PO
from paged_cases import DT, U_OUT, Cache, make_tokens, rounded
from test_gpu_paged_attention import run

pytestmark = pytest.mark.gpu


def bound_of(c, q, b, new, r, h, G, scale):
    """float64 outputs [new, G, D] of sequence b, head h, and the bound described above."""
    n = c.lens[b]
    k, v, vs = PO.token_values(c.pool, c.table, b, n, h, c.D, c.kind)
    out, bound = np.zeros((new, G, c.D)), np.zeros((new, G, c.D))
    for i in range(new):
        for g in range(G):
            x = q[r + i, h * G + g].astype(np.float64)
            see = n - new + i + 1
            s = k[:see] @ x * scale
            p = np.exp(s - s.max())
            p /= p.sum()
            size = (np.abs(k[:see]) @ np.abs(x) * scale).max()
            eps = (c.D + 8) * 2.0 ** -24 * size + 2.0 ** -21
            own = p @ np.abs(v[:see])
            step = 2.0 ** -36 * (p * vs[:see]).max() * (np.abs(v[:see]) / vs[:see, None]).sum(0)
            out[i, g] = p @ v[:see]
            bound[i, g] = (own * (2.0 ** -11 + 2 * eps + 2.0 ** -19) + step
                           + np.abs(out[i, g]) * U_OUT[c.dtype] + 2.0 ** -24)
    return out, bound


def cache_with_a_large_value(lens, e, kind, dtype):
    """Tokens of deviation 1 but for one value of 2**e in channel 0."""
    c = Cache(lens, H=1, kind=kind, dtype=dtype, seed=e, fill=False)
    for b, n in enumerate(lens):
        k, _ = make_tokens(c.rng, n, 1, c.D)
        v = c.rng.standard_normal((n, 1, c.D)).astype(np.float32)
        v[n // 2, 0, 0] = 2.0 ** e
        PO.append(c.pool, c.table, b, n, rounded(k, dtype), rounded(v, dtype), kind)
    return c


LARGE = [("fp16", 15), ("bf16", 18), ("bf16", 22), ("bf16", 26)]


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype,e", LARGE)
def test_many_rows(cuda, kind, dtype, e):
    c = cache_with_a_large_value([32, 200], e, kind, dtype)
    new, G = [1, 5], 4
    q = rounded(c.queries(new, G) * np.float32(0.3), dtype)
    out, _ = run(cuda, c, q, new, G, max_new=64)
    r = 0
    for b, m in enumerate(new):
        want, bound = bound_of(c, q, b, m, r, 0, G, c.D ** -0.5)
        far = np.abs(out[r:r + m] - want) / bound
        assert far.max() <= 1, f"sequence {b}: {far.max():.3g} of the bound"
        r += m


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype,e", LARGE)
@pytest.mark.parametrize("n", [32, 48])
def test_few_rows(cuda, kind, dtype, e, n):
    """1500 sequences that hold the same pages: more blocks than warps, so that a warp has
    several blocks of one sequence."""
    from kvquant.kernels import paged_attention
    copies, G = 1500, 4
    c = cache_with_a_large_value([n], e, kind, dtype)
    q = rounded(c.queries([1], G) * np.float32(0.3), dtype)
    pool, table, lengths = c.gpu(cuda)
    qt = torch.from_numpy(q).to(cuda).to(DT[dtype]).expand(copies, G, c.D)
    out = paged_attention(qt, pool, table.repeat(copies, 1), lengths.repeat(copies), kind)
    want, bound = bound_of(c, q, 0, 1, 0, 0, G, c.D ** -0.5)
    far = np.abs(out.float().cpu().numpy() - want) / bound
    assert far.max() <= 1, f"{far.max():.3g} of the bound"
