"""The paged cache as a decoder uses it: PagedKVCache through prompts, forks, steps, frees
and compactions, against the oracle's cache; and the example."""
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

from oracle import paged_oracle as PO
from paged_cases import DT, U_OUT, check, make_tokens, rounded

pytestmark = pytest.mark.gpu


class Model:
    """One layer's cache in the oracle: pool, pages and lengths, driven like PagedKVCache."""

    def __init__(self, c, kind, layer):
        self.kind, self.layer, self.dim = kind, layer, c.head_dim
        self.pages = PO.Pages(c.table.cpu().numpy(), c.lengths.cpu().numpy(), c.refs.cpu().numpy(),
                              c.page_tokens, c.pool.cpu().numpy())

    def append(self, slots, tokens):
        for s, (k, v) in zip(slots, tokens):
            PO.append(self.pages.pool[self.layer], self.pages.table, s, int(self.pages.lengths[s]),
                      k, v, self.kind)

    def attend(self, q, slots, rows, G, dtype):
        out, bound, r = [], [], 0
        for s, n in zip(slots, rows):
            heads, bounds = [], []
            for h in range(self.pages.pool.shape[2]):
                L = int(self.pages.lengths[s])
                k, v, vs = PO.token_values(self.pages.pool[self.layer], self.pages.table, s, L, h,
                                           self.dim, self.kind)
                o, _, b, _ = PO.attention(q[r:r + n, h * G:(h + 1) * G].astype(np.float64), k, v, vs,
                                          L - n, 0, self.dim ** -0.5, U_OUT[dtype])
                heads.append(o)
                bounds.append(b)
            out.append(np.concatenate(heads, 1))
            bound.append(np.concatenate(bounds, 1))
            r += n
        return np.concatenate(out), np.concatenate(bound)


@pytest.mark.parametrize("kind,dtype", [("int8", "fp16"), ("e4m3", "bf16")])
def test_decoder_life(cuda, kind, dtype):
    from kvquant.paged_cache import PagedKVCache
    H, G, D, layer = 2, 4, 64, 1
    c = PagedKVCache(2, 48, H, max_slots=8, max_tokens=400, head_dim=D, page_tokens=32, kind=kind,
                     device=cuda)
    m = Model(c, kind, layer)
    rng = np.random.default_rng(3)
    t = lambda x: torch.from_numpy(np.ascontiguousarray(x)).to(cuda)  # noqa: E731

    def step(slots, rows):
        c.extend(slots, t(np.int32(rows)))
        m.pages.extend(slots, rows)
        tokens = [tuple(rounded(x, dtype) for x in make_tokens(rng, n, H, D)) for n in rows]
        m.append(slots, tokens)
        ip = t(np.concatenate([[0], np.cumsum(rows)]).astype(np.int32))
        k, v = (t(np.concatenate(x)).to(DT[dtype]) for x in zip(*tokens))
        c.append(layer, k, v, slots, ip)
        q = rounded(rng.standard_normal((sum(rows), H * G, D)), dtype)
        got = c.attend(layer, t(q).to(DT[dtype]), slots, ip, max_new=max(rows))
        want, bound = m.attend(q, slots, rows, G, dtype)
        check(got.float().cpu().numpy(), want, bound, f"step {slots}")

    step([0, 1, 2], [77, 5, 160])
    c.fork([0, 0, 2], [3, 4, 5])
    m.pages.fork([0, 0, 2], [3, 4, 5])
    step([3, 4, 5, 0], [1, 1, 1, 1])
    step([5, 1, 4], [3, 30, 1])
    c.free([0, 2])
    m.pages.free([0, 2])
    assert int(c.compact().item()) == m.pages.compact()
    step([4, 3, 1, 5], [1, 2, 1, 20])
    step([6, 3], [64, 1])
    np.testing.assert_array_equal(c.table.cpu().numpy(), m.pages.table)
    np.testing.assert_array_equal(c.refs.cpu().numpy(), m.pages.refs)
    np.testing.assert_array_equal(c.pool[layer].cpu().numpy(), m.pages.pool[layer])
    c.check()


def test_refusals_are_reported(cuda):
    from kvquant.paged_cache import PagedKVCache
    c = PagedKVCache(1, 4, 1, max_slots=3, max_tokens=128, head_dim=64, page_tokens=32, device=cuda)
    c.extend([0, 1], torch.tensor([60, 40], dtype=torch.int32, device=cuda))
    c.check()
    c.extend([2], 1)
    with pytest.raises(RuntimeError, match="no free pages"):
        c.check()
    c.fork([0], [1])
    with pytest.raises(RuntimeError, match="bad slot"):
        c.check()
    c.check()
    for kw in (dict(kind="fp4"), dict(head_dim=96), dict(page_tokens=24), dict(n_pages=0),
               dict(device="cpu")):
        args = dict(n_layers=1, n_pages=4, heads=1, max_slots=1, max_tokens=32)
        with pytest.raises(RuntimeError, match="PagedKVCache"):
            PagedKVCache(**{**args, **kw})
    q = torch.zeros((1, 1, 64), dtype=torch.float32, device=cuda)
    with pytest.raises(RuntimeError, match="fp16 or bf16"):
        c.attend(0, q, [0], max_new=1)
    with pytest.raises(RuntimeError, match="must be"):
        c.append(0, q.half()[:, :, :32], q.half(), [0])
    with pytest.raises(RuntimeError, match="int32"):
        c.attend(0, q.half(), torch.zeros(1, dtype=torch.int64, device=cuda), max_new=1)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_example(cuda, kind):
    """8-bit keys and values: a step's outputs stay within 2 % (int8: 1 / 254 of a block's
    largest value per code) or 6 % (e4m3: 2**-4) of the fp32 cache's."""
    sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))
    import paged_sampling
    assert paged_sampling.main(["--kind", kind, "--steps", "12"]) < (0.02 if kind == "int8" else 0.06)
