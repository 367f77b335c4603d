"""Builds paged 8-bit caches for the tests: pages in shuffled order, filled by the
oracle's append, with bytes of another kind of garbage wherever nothing is stored."""
from __future__ import annotations

import numpy as np
import torch

from oracle import paged_oracle as PO

DT = {"fp16": torch.float16, "bf16": torch.bfloat16}
U_OUT = {"fp16": 2.0 ** -11, "bf16": 2.0 ** -8}


def rounded(x: np.ndarray, dtype: str) -> np.ndarray:
    """fp32 values that the 16-bit type holds."""
    return torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(DT[dtype]).float().numpy()


def make_tokens(rng, n, H, D):
    """Keys with channels of unlike size, values with tokens of unlike size, fp32 [n, H, D]."""
    k = rng.standard_normal((n, H, D)).astype(np.float32)
    k *= np.exp(rng.uniform(-1.5, 1, (H, D))).astype(np.float32)
    v = rng.standard_normal((n, H, D)).astype(np.float32)
    v *= np.exp(rng.standard_normal((n, H, 1))).astype(np.float32)
    return k, v


class Cache:
    """lens: tokens of each slot; order: slots of the call's sequences (default all)."""

    def __init__(self, lens, H=2, D=128, page=32, kind="int8", dtype="fp16", seed=0, spare=2,
                 fill=True, extra_cols=1, garbage=0xFF):
        rng = np.random.default_rng(seed)
        self.lens, self.H, self.D, self.page, self.kind, self.dtype = lens, H, D, page, kind, dtype
        need = [-(-n // page) for n in lens]
        n_pages = sum(need) + spare
        perm = rng.permutation(n_pages)
        cols = max(need + [0]) + extra_cols
        self.table = np.full((len(lens), cols), -1, np.int32)
        self.refs = np.zeros(n_pages, np.int32)
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = perm[at:at + n]
            self.refs[perm[at:at + n]] = 1
            at += n
        # 0xFF is a NaN in e4m3, and a NaN as a scale
        self.pool = np.full((n_pages, H, page // 16, 32 * D + 16), garbage, np.uint8)
        self.lengths = np.array(lens, np.int32)
        self.rng = rng
        if fill:
            for i, n in enumerate(lens):
                k, v = make_tokens(rng, n, H, D)
                PO.append(self.pool, self.table, i, n, rounded(k, dtype), rounded(v, dtype), kind)
                if n % 16:  # the places after the last token hold garbage too
                    blk = n // 16
                    for at in PO.record_maps(D):
                        for h in range(H):
                            self.pool[self.table[i, blk * 16 // page], h,
                                      blk % (page // 16)][at[n % 16:]] = garbage

    def queries(self, new, G):
        q = self.rng.standard_normal((sum(new), self.H * G, self.D)).astype(np.float32)
        return rounded(q, self.dtype)

    def gpu(self, dev):
        t = lambda x: torch.from_numpy(np.ascontiguousarray(x)).to(dev)  # noqa: E731
        return t(self.pool), t(self.table), t(self.lengths)


def expected(c: Cache, q, new, G, window=0, scale=None, slots=None):
    """Oracle outputs of a call and the bounds: out, ml, b_out, b_ml over the rows."""
    scale = c.D ** -0.5 if scale is None else scale
    N = q.shape[0]
    out, ml = np.zeros((N, c.H * G, c.D)), np.zeros((N, c.H * G, 2))
    b_out, b_ml = np.zeros_like(out), np.zeros_like(ml)
    r = 0
    for b, m in enumerate(new):
        s = b if slots is None else slots[b]
        n = c.lens[s]
        for h in range(c.H if m else 0):
            k, v, vs = PO.token_values(c.pool, c.table, s, n, h, c.D, c.kind)
            hs = slice(h * G, (h + 1) * G)
            for x, y in zip((out, ml, b_out, b_ml),
                            PO.attention(q[r:r + m, hs].astype(np.float64), k, v, vs, n - m, window,
                                         scale, U_OUT[c.dtype])):
                x[r:r + m, hs] = y
        r += m
    return out, ml, b_out, b_ml


def check(got, ref, bound, what):
    got = np.asarray(got, np.float64)
    fin = np.isfinite(ref)
    assert np.array_equal(got[~fin], ref[~fin]), what
    far = np.abs(got[fin] - ref[fin])
    assert (far <= bound[fin]).all(), \
        f"{what}: {np.nanmax(far / np.maximum(bound[fin], 1e-300)):.3g} of the bound"
