"""Plain numpy model of the paged 8-bit KV cache (the oracle of its kernels).

Records and append follow the definition step by step in the arithmetic that fixes
the codes (fp32: maximum, one product, one division, round to nearest even);
attention and its error bound are in float64; the page operations are plain
sequential Python.
"""
from __future__ import annotations

import math

import numpy as np

F32, F64 = np.float32, np.float64
BLOCK = 16
QMAX = {"int8": F32(127), "e4m3": F32(448)}
FLOOR = F32(2.0 ** -32)


# ---------------------------------------------------------------- codes
def e4m3_values() -> np.ndarray:
    """Value of each of the 256 codes (127 and 255 are NaN)."""
    out = np.empty(256, F64)
    for b in range(256):
        e, f = (b >> 3) & 15, b & 7
        x = f * 2.0 ** -9 if e == 0 else (1 + f / 8) * 2.0 ** (e - 7)
        if b & 127 == 127:
            x = math.nan
        out[b] = -x if b & 128 else x
    return out


_E4M3 = e4m3_values()


def encode(y: np.ndarray, kind: str) -> np.ndarray:
    """Code bytes of fp32 values already divided by their scale; NaN gives 0."""
    y = np.where(np.isnan(y), F32(0), y).astype(F32)
    y = np.clip(y, -QMAX[kind], QMAX[kind])
    if kind == "int8":
        return (np.rint(y).astype(np.int64) + 128).astype(np.uint8)
    a = np.abs(y).astype(F64)
    pos = _E4M3[:127]
    hi = np.clip(np.searchsorted(pos, a), 1, 126)
    lo = hi - 1
    d_lo, d_hi = a - pos[lo], pos[hi] - a
    code = np.where((d_hi < d_lo) | ((d_hi == d_lo) & (hi % 2 == 0)), hi, lo)
    return (code | np.where(np.signbit(y), 128, 0)).astype(np.uint8)


def decode(b: np.ndarray, kind: str) -> np.ndarray:
    return b.astype(F64) - 128 if kind == "int8" else _E4M3[b]


# ---------------------------------------------------------------- records
def record_maps(D: int):
    """Byte of (token, channel) in a record: key codes and value codes, int [16, D]."""
    t, d = np.arange(BLOCK)[:, None], np.arange(D)[None, :]
    key = d // 32 * 512 + t % 8 * 64 + d // 4 % 4 * 16 + d // 16 % 2 * 8 + t // 8 * 4 + d % 4
    val = (d // 32 * 512 + d % 8 * 64 + t // 2 % 4 * 16 + d // 16 % 2 * 8 + d // 8 % 2 * 4
           + t // 8 * 2 + t % 2)
    return key, 16 * D + val


def read_record(rec: np.ndarray, D: int, kind: str):
    """(key codes, value codes) float64 [16, D] and (key, value) scales of one record."""
    key, val = record_maps(D)
    sc = rec[32 * D:32 * D + 8].copy().view(F32)
    return decode(rec[key], kind), decode(rec[val], kind), F32(sc[0]), F32(sc[1])


def token_values(pool, table, slot, n, h, D, kind):
    """(k, v) float64 [n, D] of the first n tokens of a slot, and the value scale per token."""
    nb = pool.shape[2]
    k, v, vs = np.zeros((n, D)), np.zeros((n, D)), np.ones(n)
    for blk in range(-(-n // BLOCK)):
        kc, vc, ks, s = read_record(pool[table[slot, blk // nb], h, blk % nb], D, kind)
        m = min(BLOCK, n - blk * BLOCK)
        k[blk * BLOCK:blk * BLOCK + m] = kc[:m] * F64(ks)
        v[blk * BLOCK:blk * BLOCK + m] = vc[:m] * F64(s)
        vs[blk * BLOCK:blk * BLOCK + m] = s
    return k, v, vs


# ---------------------------------------------------------------- append
def append(pool, table, slot, length, x_k, x_v, kind):
    """Writes the last len(x_k) of the slot's `length` tokens, in place. x: fp32 [m, H, D]."""
    m, H, D = x_k.shape
    nb, start = pool.shape[2], length - m
    if m == 0:
        return
    maps = record_maps(D)
    zero = 128 if kind == "int8" else 0
    for blk in range(start // BLOCK, (length - 1) // BLOCK + 1):
        t0 = blk * BLOCK
        first, last = max(0, start - t0), min(BLOCK, length - t0)
        for h in range(H):
            rec = pool[table[slot, blk // nb], h, blk % nb]
            for which, x in enumerate((x_k, x_v)):
                new = x[t0 + first - start:t0 + last - start, h].astype(F32)
                at = rec[32 * D + 4 * which:32 * D + 4 * which + 4]
                old = at.copy().view(F32)[0] if first else F32(0)
                fine = np.abs(new[np.isfinite(new)])
                amax = fine.max() if fine.size else F32(0)
                s = max(old, amax * (F32(1) / QMAX[kind]), FLOOR)
                inv = F32(1) / s
                out = np.full((BLOCK, D), zero, np.uint8)
                if first:
                    codes = rec[maps[which]][:first]
                    if s > old:
                        codes = encode(decode(codes, kind).astype(F32) * (old * inv), kind)
                    out[:first] = codes
                with np.errstate(invalid="ignore", over="ignore"):
                    out[first:last] = encode(new * inv, kind)
                rec[maps[which]] = out
                at[:] = np.array([s], F32).view(np.uint8)
            rec[32 * D + 8:] = 0


# ---------------------------------------------------------------- attention
def attention(q, k, v, vs, first_pos, window, scale, u_out):
    """One sequence and KV head: q fp64 [rows, G, D] at positions first_pos + row.

    Returns out [rows, G, D], ml [rows, G, 2] in float64 and bounds on the kernels'
    deviations from them. The kernels round the weights p * vs to fp16 (2**-11 of
    each, or 2**-25 of the largest), the output (u_out), and have fp32 scores (D + 8
    roundings of the sum of |q k|) and exponentials (2**-21)."""
    rows, G, D = q.shape
    T = k.shape[0]
    pos = first_pos + np.arange(rows)
    j = np.arange(T)
    seen = j[None] <= pos[:, None]
    if window:
        seen &= j[None] > pos[:, None] - window
    out, ml = np.zeros((rows, G, D)), np.zeros((rows, G, 2))
    b_out, b_ml = np.zeros((rows, G, D)), np.zeros((rows, G, 2))
    for g in range(G):
        x = q[:, g] @ k.T * scale
        size = np.abs(q[:, g]) @ np.abs(k).T * abs(scale)
        for r in range(rows):
            ok = seen[r]
            if not ok.any():
                ml[r, g] = -math.inf, math.inf
                continue
            xs = x[r, ok]
            M = xs.max()
            e = np.exp(xs - M)
            L = e.sum()
            p = e / L
            vv = np.abs(v[ok])
            out[r, g] = p @ v[ok]
            ml[r, g] = M, 1 / L
            eps = (D + 8) * 2.0 ** -24 * size[r, ok].max() + 2.0 ** -21
            weight = p @ vv
            top = (p * vs[ok]).max()
            tiny = 2.0 ** -24 * top * (vv / vs[ok][:, None]).sum(0)
            b_out[r, g] = (weight * (2.0 ** -11 + 2 * eps + 2.0 ** -19) + tiny
                           + np.abs(out[r, g]) * u_out + 2.0 ** -24)
            b_ml[r, g, 0] = eps + 2.0 ** -22 * abs(M)
            b_ml[r, g, 1] = (2 * eps + (T / 8 + 64) * 2.0 ** -24 + 2.0 ** -19) / L
    return out, ml, b_out, b_ml


# ---------------------------------------------------------------- page operations
class Pages:
    """table, lengths, refs and (optionally) one page's worth of content, sequentially."""

    def __init__(self, table, lengths, refs, page_tokens, pool=None):
        self.table, self.lengths, self.refs = table.copy(), lengths.copy(), refs.copy()
        self.P, self.pool, self.status = page_tokens, None if pool is None else pool.copy(), 0

    def free(self, slots):
        for i, s in enumerate(slots):
            if not 0 <= s < len(self.lengths) or s in slots[:i]:
                self.status |= 2
                continue
            for p in self.table[s]:
                if p >= 0:
                    self.refs[p] -= 1
            self.table[s] = -1
            self.lengths[s] = 0

    def fork(self, src, dst):
        for i, (a, b) in enumerate(zip(src, dst)):
            n = len(self.lengths)
            if (not 0 <= a < n or not 0 <= b < n or b in dst[:i] or b in src
                    or self.lengths[b] != 0):
                self.status |= 2
                continue
            self.table[b] = self.table[a]
            self.lengths[b] = self.lengths[a]
            for p in self.table[a]:
                if p >= 0:
                    self.refs[p] += 1

    def extend(self, slots, n_new):
        P, cols = self.P, self.table.shape[1]
        for i, (s, m) in enumerate(zip(slots, n_new)):
            if (not 0 <= s < len(self.lengths) or s in slots[:i] or m < 0
                    or -(-(self.lengths[s] + m) // P) > cols):
                self.status |= 2
                return
        free = [p for p in range(len(self.refs)) if self.refs[p] == 0]
        refs, table = self.refs.copy(), self.table.copy()
        moves = []
        for s, m in zip(slots, n_new):
            n = int(self.lengths[s])
            col = -(-n // P)
            if m > 0 and n % P and refs[table[s, n // P]] > 1:
                if not free:
                    self.status |= 1
                    return
                p = free.pop(0)
                moves.append((table[s, n // P], p))
                refs[table[s, n // P]] -= 1
                table[s, n // P], refs[p] = p, 1
            for c in range(col, -(-(n + m) // P)):
                if not free:
                    self.status |= 1
                    return
                p = free.pop(0)
                table[s, c], refs[p] = p, 1
        self.refs, self.table = refs, table
        for s, m in zip(slots, n_new):
            self.lengths[s] += m
        if self.pool is not None:
            for a, b in moves:
                self.pool[:, b] = self.pool[:, a]

    def compact(self):
        live = [p for p in range(len(self.refs)) if self.refs[p] > 0]
        n = len(live)
        holes = [p for p in range(n) if self.refs[p] == 0]
        to = dict(zip([p for p in live if p >= n], holes))
        for a, b in to.items():
            self.refs[b], self.refs[a] = self.refs[a], 0
            if self.pool is not None:
                self.pool[:, b] = self.pool[:, a]
        self.table = np.vectorize(lambda p: to.get(p, p), otypes=[self.table.dtype])(self.table)
        return n
