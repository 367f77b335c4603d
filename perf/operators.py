"""What is measured of the paged 8-bit KV cache: append, attention and page operations.

The cache holds keys and values in 8 bits. A block is 16 tokens of one KV head; it is one record
of 32 * D + 16 bytes: the key codes, the value codes, then two fp32 scales (keys, values) and 8
zero bytes. A page is page_tokens / 16 blocks of every head, a pool is uint8
[layers, pages, heads, blocks, record]; table int32 [slots, columns] names each slot's pages (-1:
none), lengths int32 [slots] its tokens, refs int32 [pages] how many slots hold a page.

Byte order inside a record (D channels, token t, channel d; the order in which the attention's
matrix instructions take them):
  keys    [d / 32][t % 8][(d / 4) % 4][(d / 16) % 2][t / 8][d % 4]
  values  [d / 32][d % 8][(t / 2) % 4][(d / 16) % 2][(d / 8) % 2][t / 8][t % 2]
"int8" codes are stored as code + 128 with code in -127..127, "e4m3" codes are the 8-bit float.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

BLOCK = 16
FLOOR = 2.0 ** -32  # the least scale of a block
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
QMAX = {"int8": 127.0, "e4m3": 448.0}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one short conversation's next token: nothing but latency
        _attend("attend-short", 1, 8, 4, 128, 64, "e4m3", "bf16", 129, 129, 1),
        # one decode step of a 32-head layer over 4096 tokens, the framework's smallest configuration
        _attend("attend-4k", 1, 32, 1, 128, 64, "int8", "fp16", 4096, 4096, 1),
        # a serving batch of 16 at grouped heads, contexts from nothing up to 8192, a sequence that is empty
        _attend("attend-batch", 16, 8, 4, 128, 64, "e4m3", "bf16", 0, 8192, 1),
        # one long context, every head its own keys: pure bandwidth
        _attend("attend-long", 1, 32, 1, 128, 128, "int8", "fp16", 262144, 262144, 1),
        # checking five drafted tokens per sequence, small heads, small pages, a sliding window
        _attend("attend-verify", 23, 8, 4, 64, 16, "int8", "bf16", 5, 6000, 5, window=2500),
        # a prompt's next chunk over what is there already: matrix products bound it
        _attend("attend-chunk", 2, 8, 4, 128, 64, "int8", "bf16", 8200, 10007, 2048),
        # one new token for each of 64 sequences, blocks half full
        _append("append-step", 64, 8, 128, 64, "int8", "fp16", 1, 4000, 1, 1),
        # a ragged batch of whole prompts
        _append("append-prompt", 17, 8, 128, 64, "e4m3", "bf16", 0, 0, 1, 4099),
        # a parallel-sampling step of two prompts: drop the old children, fork new ones, extend each by a token
        _fork("fork-small", 2, 4, 8, 64, 2, 40, 700),
        # the same for 16 beams of 15 children each over long shared prefixes, eight layers to copy open pages in
        _fork("fork-beams", 16, 15, 8, 64, 8, 1000, 30000),
        # a small pool closed up after requests left
        _compact("compact-small", 61, 8, 64, 2, 12, 0.6),
        # a gigabyte of pages, a good half of them live and scattered
        _compact("compact-large", 4001, 8, 64, 2, 200, 0.6),
    ]


def _attend(name, batch, heads, group, dim, page, kind, dtype, lo, hi, new, window=0, mix=1):
    return {"name": name, "op": "attend", "batch": batch, "heads": heads, "group": group,
            "dim": dim, "page": page, "kind": kind, "dtype": dtype, "lo": lo, "hi": hi, "new": new,
            "window": window, "mix": mix}


def _append(name, batch, heads, dim, page, kind, dtype, lo, hi, new_lo, new_hi, mix=1):
    return {"name": name, "op": "append", "batch": batch, "heads": heads, "dim": dim, "page": page,
            "kind": kind, "dtype": dtype, "lo": lo, "hi": hi, "new_lo": new_lo, "new_hi": new_hi,
            "mix": mix}


def _fork(name, parents, children, heads, page, layers, lo, hi, mix=1):
    return {"name": name, "op": "fork", "parents": parents, "children": children, "heads": heads,
            "dim": 128, "page": page, "layers": layers, "lo": lo, "hi": hi, "mix": mix}


def _compact(name, pages, heads, page, layers, slots, live, mix=1):
    return {"name": name, "op": "compact", "pages": pages, "heads": heads, "dim": 128, "page": page,
            "layers": layers, "slots": slots, "live": live, "mix": mix}


def _log(rng, lo, hi):
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(lo, min(hi, n))


def draw(rng):
    op = rng.choice(["attend"] * 6 + ["append"] * 2 + ["fork"] * 2 + ["compact"] * 2)
    mix = rng.randrange(1, 1 << 30)
    page, kind, dtype = rng.choice([16, 32, 64, 128]), rng.choice(["int8", "e4m3"]), rng.choice(["fp16", "bf16"])
    dim, heads = rng.choice([64, 128, 128]), rng.choice([1, 2, 4, 5, 8, 8, 32])
    if op == "attend":
        while True:
            batch, group = _log(rng, 1, 64), rng.choice([1, 2, 4, 7, 8])
            hi = _log(rng, 1, 262144)
            new = 1 if rng.random() < 0.6 else _log(rng, 1, min(2048, hi))
            if (batch * hi * heads * dim <= 3 * 2 ** 28 and batch * new * heads * group * hi <= 2 ** 29
                    and heads * group <= 64 and batch * new * heads * group * dim <= 2 ** 25):
                break
        lo = hi if rng.random() < 0.3 else rng.randint(0, hi)
        window = 0 if rng.random() < 0.7 else _log(rng, 1, hi)
        c = _attend("", batch, heads, group, dim, page, kind, dtype, max(lo, new if rng.random() < 0.7 else 0),
                    hi, new, window, mix)
    elif op == "append":
        while True:
            batch, hi = _log(rng, 1, 128), _log(rng, 1, 4099)
            new_hi = 1 if rng.random() < 0.4 else _log(rng, 1, 4099)
            if batch * new_hi * heads * dim <= 2 ** 26:
                break
        c = _append("", batch, heads, dim, page, kind, dtype, 0, hi, 1 if rng.random() < 0.8 else 0, new_hi, mix)
    elif op == "fork":
        while True:
            parents, children, layers = _log(rng, 1, 16), _log(rng, 1, 15), _log(rng, 1, 8)
            hi = _log(rng, 1, 30000)
            if layers * heads * page * (parents * children + 2) <= 8 * 8 * 64 * 256:
                break
        c = _fork("", parents, children, heads, page, layers, rng.randint(0, hi), hi, mix)
    else:
        while True:
            pages, layers = _log(rng, 3, 30000), _log(rng, 1, 8)
            if pages * layers * heads * page <= 4001 * 2 * 8 * 64:
                break
        c = _compact("", pages, heads, page, layers, _log(rng, 1, 200), rng.choice([0.0, 0.1, 0.3, 0.6, 0.9, 1.0]), mix)
    del c["name"]
    return c


# ------------------------------------------------------------------ what a case's lengths are
def _lengths(case):
    """(tokens in each sequence, its new tokens among them)"""
    r = random.Random(case["mix"] * 7919 + 17)
    if case["op"] == "attend":
        lens = [r.randint(case["lo"], case["hi"]) for _ in range(case["batch"])]
        lens[-1] = case["hi"]
        if case["lo"] == 0 and case["batch"] > 1:
            lens[0] = 0
        return lens, [min(n, case["new"]) for n in lens]
    if case["op"] == "append":
        old = [r.randint(case["lo"], case["hi"]) for _ in range(case["batch"])]
        new = [r.randint(case["new_lo"], case["new_hi"]) for _ in range(case["batch"])]
        new[-1] = case["new_hi"]
        return [a + b for a, b in zip(old, new)], new
    return [r.randint(case["lo"], case["hi"]) for _ in range(case["parents"])], None


def _fork_size(case):
    """(pages used by the parents, pages taken by the children, copied pages) of a fork case"""
    lens, _ = _lengths(case)
    used = sum(-(-n // case["page"]) for n in lens)
    return used, len(lens) * case["children"], sum(case["children"] for n in lens if n % case["page"])


def _live(case):
    """Which pages of a compact case are live, as a list of truth values."""
    r = random.Random(case["mix"] * 104729 + 5)
    return [r.random() < case["live"] for _ in range(case["pages"])]


def _record(case):
    return 32 * case["dim"] + 16


def work(case):
    record = _record(case)
    if case["op"] == "attend":
        lens, new = _lengths(case)
        hq, pairs, blocks = case["heads"] * case["group"], 0, 0
        for n, m in zip(lens, new):
            w = case["window"] or n
            # query i sits at n - m + i and sees min(its position + 1, window) tokens
            pairs += sum(min(n - m + i + 1, w) for i in range(m)) if m else 0
            if m:
                blocks += (n - max(0, n - m + 1 - w) + BLOCK - 1) // BLOCK
        rows = sum(new) * hq
        return {"bytes": blocks * case["heads"] * record + rows * (4 * case["dim"] + 8),
                "flops": 4 * case["dim"] * hq * pairs}
    if case["op"] == "append":
        lens, new = _lengths(case)
        written = old = back = 0
        for n, m in zip(lens, new):
            if m:
                first = (n - m) // BLOCK
                written += (n - 1) // BLOCK + 1 - first
                old += 1 if (n - m) % BLOCK else 0
                back += n - first * BLOCK
        row = case["heads"] * case["dim"]
        # the new tokens in, the open blocks in, the blocks out; then the touched tokens read back
        return {"bytes": case["heads"] * record * (2 * written + old) + 4 * row * (sum(new) + back),
                "flops": 4 * row * sum(new)}
    if case["op"] == "fork":
        used, taken, copied = _fork_size(case)
        page = case["heads"] * (case["page"] // BLOCK) * record
        entries = used * (case["children"] + 1)
        return {"bytes": 2 * copied * page * case["layers"] + 12 * entries, "flops": entries}
    live = _live(case)
    n = sum(live)
    moved = sum(live[n:])
    page = case["heads"] * (case["page"] // BLOCK) * record
    return {"bytes": 2 * moved * page * case["layers"] + 20 * case["pages"], "flops": case["pages"]}


# ------------------------------------------------------------------ inputs
def _keys_values(n, heads, dim, gen, chan):
    """n x 16 tokens of keys and values in 32 bits: keys with channels of unlike size, a few of them
    large, as rotated keys have; values with tokens of unlike size."""
    k = torch.randn((n, BLOCK, heads, dim), generator=gen, device="cuda") * chan
    v = torch.randn((n, BLOCK, heads, dim), generator=gen, device="cuda")
    v *= torch.exp(0.5 * torch.randn((n, BLOCK, heads, 1), generator=gen, device="cuda"))
    return k, v


def _channels(heads, dim, gen):
    c = torch.exp(torch.rand((heads, dim), generator=gen, device="cuda") * 2.3 - 1.5)
    big = torch.rand((heads, dim), generator=gen, device="cuda") < 0.03
    return torch.where(big, c * 4, c)


def _filled(shape, kind, gen, dim):
    """A pool whose every block holds quantised keys and values."""
    pages, heads, blocks, record = shape
    pool = torch.empty(shape, dtype=torch.uint8, device="cuda")
    chan = _channels(heads, dim, gen)
    step = max(1, 2 ** 27 // (heads * blocks * BLOCK * dim))
    for a in range(0, pages, step):
        n = min(step, pages - a)
        k, v = _keys_values(n * blocks, heads, dim, gen, chan)
        rec = _pack(*(_codes(x, x.abs().amax((1, 3)), kind) for x in (k, v)), kind)
        pool[a:a + n] = rec.view(n, blocks, heads, record).transpose(1, 2)
    return pool


def _paged(lens, page, perm):
    """table for sequences of these lengths, over the pages of a permutation"""
    cols = max(1, max(-(-n // page) for n in lens))
    table, at = np.full((len(lens), cols), -1, np.int32), 0
    for i, n in enumerate(lens):
        p = -(-n // page)
        table[i, :p] = perm[at:at + p]
        at += p
    return table


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed * 1000003 + case["mix"])
    rng = np.random.RandomState((seed * 31 + case["mix"]) % (1 << 31))
    blocks, record = case["page"] // BLOCK, _record(case)
    s = dict(case)
    if case["op"] in ("attend", "append"):
        lens, new = _lengths(case)
        pages = sum(-(-n // case["page"]) for n in lens) + 3  # a few that nobody holds
        perm = rng.permutation(pages)
        s["pool"] = _filled((pages, case["heads"], blocks, record), case["kind"], gen, case["dim"])
        s["table"] = torch.from_numpy(_paged(lens, case["page"], perm)).cuda()
        s["lengths"], s["indptr"] = _ints(lens), _ints([0] + list(np.cumsum(new)))
        s["total"], s["most"] = sum(new), max(new)
        dtype = TYPES[case["dtype"]]
        if case["op"] == "attend":
            hq = case["heads"] * case["group"]
            s["q"] = torch.randn((s["total"], hq, case["dim"]), generator=gen, device="cuda").to(dtype)
            s["out"] = torch.empty_like(s["q"])
            s["ml"] = torch.empty((s["total"], hq, 2), dtype=torch.float32, device="cuda")
        else:
            chan = _channels(case["heads"], case["dim"], gen)
            k, v = _keys_values(-(-max(1, s["total"]) // BLOCK), case["heads"], case["dim"], gen, chan)
            s["k"], s["v"] = (x.reshape(-1, case["heads"], case["dim"])[:s["total"]].to(dtype) for x in (k, v))
            # what is read back: each sequence from the first block that the new tokens touch
            first = [(n - m) // BLOCK * BLOCK for n, m in zip(lens, new)]
            back = [n - f if m else 0 for n, m, f in zip(lens, new, first)]
            s["starts"], s["back"] = _ints(first), _ints([0] + list(np.cumsum(back)))
            s["back_total"] = sum(back)
        return s
    if case["op"] == "fork":
        lens, _ = _lengths(case)
        used, taken, _ = _fork_size(case)
        pages = used + taken + 5
        n, c = len(lens), case["children"]
        perm = rng.permutation(pages)
        cols = max(1, max(-(-x // case["page"]) for x in lens)) + 1
        table = np.full((n * (c + 1), cols), -1, np.int32)
        held = _paged(lens, case["page"], perm)
        table[:n, :held.shape[1]] = held
        refs = np.zeros(pages, np.int32)
        refs[held[held >= 0]] = 1
        s["table"], s["refs"] = torch.from_numpy(table).cuda(), torch.from_numpy(refs).cuda()
        s["lengths"] = _ints(lens + [0] * (n * c))
        s["src"] = _ints([i for i in range(n) for _ in range(c)])
        s["dst"] = _ints([n + i for i in range(n * c)])
    else:
        pages, slots = case["pages"], case["slots"]
        live = np.flatnonzero(np.array(_live(case)))
        live = rng.permutation(live).astype(np.int32)
        # the live pages go to the slots in turn; one in eight is shared with the next slot
        mine = [list(live[i::slots]) for i in range(slots)]
        for i in range(slots - 1):
            mine[i + 1] = mine[i][:len(mine[i]) // 8] + mine[i + 1]
        cols = max(1, max(len(m) for m in mine)) + 2
        table, refs = np.full((slots, cols), -1, np.int32), np.zeros(pages, np.int32)
        for i, m in enumerate(mine):
            table[i, :len(m)] = m
            refs[m] += 1
        # table and counts in one buffer, and its copy: the state before the pool is closed up
        s["saved"] = torch.from_numpy(np.concatenate([table.ravel(), refs])).cuda()
        s["meta"] = s["saved"].clone()
        s["table"], s["refs"] = s["meta"][:table.size].view(slots, cols), s["meta"][table.size:]
    s["pool"] = torch.randint(0, 256, (case["layers"], pages, case["heads"], blocks, record), generator=gen,
                              dtype=torch.uint8, device="cuda")
    s["status"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    return s


# ------------------------------------------------------------------ plain forms
def _codes(x, amax, kind, old=None):
    """Codes of x [n, 16, heads, dim] in 32 bits and the scale [n, heads], which is at least `old`."""
    scale = torch.clamp(amax * (1.0 / QMAX[kind]), min=FLOOR)
    if old is not None:
        scale = torch.maximum(scale, old)
    inv = (torch.ones_like(scale) / scale)[:, None, :, None]
    return _round(x * inv, kind), scale


def _round(y, kind):
    y = torch.where(torch.isnan(y), torch.zeros_like(y), y).clamp(-QMAX[kind], QMAX[kind])
    return torch.round(y) if kind == "int8" else y.to(torch.float8_e4m3fn).float()


def _pack(keys, values, kind):
    """Records [n, heads, 32 * dim + 16] of (codes [n, 16, heads, dim], scale [n, heads]) pairs."""
    (kc, ks), (vc, vs) = keys, values
    n, _, heads, dim = kc.shape
    kb, vb = (((x + 128).to(torch.uint8) if kind == "int8" else x.to(torch.float8_e4m3fn).view(torch.uint8))
              for x in (kc, vc))
    kb = kb.view(n, 2, 8, heads, dim // 32, 2, 4, 4).permute(0, 3, 4, 2, 6, 5, 1, 7)
    vb = vb.view(n, 2, 4, 2, heads, dim // 32, 2, 2, 8).permute(0, 4, 5, 8, 2, 6, 7, 1, 3)
    scales = torch.stack([ks, vs, torch.zeros_like(ks), torch.zeros_like(ks)], -1).view(torch.uint8)
    return torch.cat([kb.reshape(n, heads, -1), vb.reshape(n, heads, -1), scales], -1)


def _unpack(rec, dim, kind):
    """(key codes, value codes) [n, 16, heads, dim] and (key, value) scales [n, heads] of records."""
    n, heads = rec.shape[:2]
    k = rec[..., :16 * dim].reshape(n, heads, dim // 32, 8, 4, 2, 2, 4).permute(0, 6, 3, 1, 2, 5, 4, 7)
    v = rec[..., 16 * dim:32 * dim].reshape(n, heads, dim // 32, 8, 4, 2, 2, 2, 2).permute(0, 7, 4, 8, 1, 2, 5, 6, 3)
    k, v = k.reshape(n, BLOCK, heads, dim), v.reshape(n, BLOCK, heads, dim)
    scales = rec[..., 32 * dim:].contiguous().view(torch.float32)
    k, v = ((x.float() - 128 if kind == "int8" else x.view(torch.float8_e4m3fn).float()) for x in (k, v))
    return k, v, scales[..., 0], scales[..., 1]


def _of_sequence(indptr, total):
    """For each of `total` rows its sequence and its place in it."""
    rows = torch.arange(total, device="cuda")
    seq = torch.searchsorted(indptr[1:].long(), rows, right=True)
    return seq, rows - indptr.long()[seq]


def _plain_attend(s):
    dim, heads, group, page = s["dim"], s["heads"], s["group"], s["page"]
    batch, cols = s["table"].shape
    total = s["total"]
    lens, new = s["lengths"].long(), (s["indptr"][1:] - s["indptr"][:-1]).long()
    rec = s["pool"][s["table"].clamp(min=0).long()]  # [batch, cols, heads, blocks, record]
    rec = rec.transpose(2, 3).reshape(-1, heads, rec.shape[-1])
    k, v, ks, vs = _unpack(rec, dim, s["kind"])
    del rec
    tokens = cols * page
    k = k.mul_(ks[:, None, :, None]).view(batch, tokens, heads, dim)
    v = v.mul_(vs[:, None, :, None]).view(batch, tokens, heads, dim)
    seq, place = _of_sequence(s["indptr"], total)
    most = s["most"]
    q = torch.zeros((batch, most, heads * group, dim), device="cuda")
    q[seq, place] = s["q"].float()
    q = q.view(batch, most, heads, group, dim).permute(0, 2, 3, 1, 4).reshape(batch, heads, group * most, dim)
    x = torch.matmul(q, k.permute(0, 2, 3, 1)).mul_(1.0 / math.sqrt(dim)).view(batch, heads, group, most, tokens)
    at = (lens - new)[:, None] + torch.arange(most, device="cuda")  # each query's own position
    j = torch.arange(tokens, device="cuda")
    seen = (j <= at[:, :, None]) & (j < lens[:, None, None])
    if s["window"]:
        seen &= j > at[:, :, None] - s["window"]
    x.masked_fill_(~seen[:, None, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    p = x.sub_(torch.where(m == -math.inf, torch.zeros_like(m), m)).exp_()
    z = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(batch, heads, group * most, tokens), v.transpose(1, 2)).view(batch, heads, group, most, dim)
    o = torch.where(z > 0, o / z, torch.zeros_like(o))
    o = o.permute(0, 3, 1, 2, 4).reshape(batch, most, heads * group, dim)[seq, place]
    ml = torch.cat([m, torch.ones_like(z) / z], -1).permute(0, 3, 1, 2, 4).reshape(batch, most, heads * group, 2)
    return {"out": o.to(TYPES[s["dtype"]]), "ml": ml[seq, place]}


def _plain_append(s):
    dim, heads, kind, page = s["dim"], s["heads"], s["kind"], s["page"]
    pool, table, lens = s["pool"], s["table"].long(), s["lengths"].long()
    new = (s["indptr"][1:] - s["indptr"][:-1]).long()
    start = lens - new
    count = torch.where(new > 0, (lens - 1) // BLOCK + 1 - start // BLOCK, torch.zeros_like(new))
    seq = torch.repeat_interleave(torch.arange(len(new), device="cuda"), count)
    block = torch.arange(len(seq), device="cuda") - (count.cumsum(0) - count)[seq] + start[seq] // BLOCK
    where = table[seq, block * BLOCK // page], block % (page // BLOCK)
    rec = pool[where[0], :, where[1]]  # [n, heads, record]
    pos = block[:, None] * BLOCK + torch.arange(BLOCK, device="cuda")
    is_old = (pos < start[seq, None])[:, :, None, None]
    is_new = ((pos >= start[seq, None]) & (pos < lens[seq, None]))[:, :, None, None]
    rows = (pos - start[seq, None] + s["indptr"].long()[seq, None]).clamp(0, max(0, s["total"] - 1))
    kc, vc, ks, vs = _unpack(rec, dim, kind)
    half = []
    for x, code, scale in ((s["k"], kc, ks), (s["v"], vc, vs)):
        x = torch.where(is_new, x[rows].float(), 0.0)
        fine = torch.where(torch.isfinite(x), x.abs(), 0.0)
        before = torch.where((pos[:, 0] < start[seq])[:, None], scale, 0.0)
        codes, scale = _codes(x, fine.amax((1, 3)), kind, before)
        again = _round(code * (before * (torch.ones_like(scale) / scale))[:, None, :, None], kind)
        again = torch.where((scale > before)[:, None, :, None], again, code)
        half.append((torch.where(is_old, again, codes), scale))
    pool[where[0], :, where[1]] = _pack(*half, kind)
    seq, place = _of_sequence(s["back"], s["back_total"])
    t = s["starts"].long()[seq] + place
    rec = pool[table[seq, t // page], :, t % page // BLOCK]
    k, v, ks, vs = _unpack(rec, dim, kind)
    i = torch.arange(len(t), device="cuda")
    dtype = TYPES[s["dtype"]]
    return {"k": (k[i, t % BLOCK] * ks[..., None]).to(dtype), "v": (v[i, t % BLOCK] * vs[..., None]).to(dtype)}


def _plain_free(s, slots):
    table, refs = s["table"], s["refs"]
    pages = table[slots]
    refs.index_add_(0, pages.clamp(min=0).reshape(-1).long(), -(pages >= 0).int().reshape(-1))
    table[slots] = -1
    s["lengths"][slots] = 0


def _plain_fork(s):
    page, table, lengths, refs, pool = s["page"], s["table"], s["lengths"], s["refs"], s["pool"]
    src, dst = s["src"].long(), s["dst"].long()
    _plain_free(s, dst)
    pages = table[src]
    table[dst] = pages
    lengths[dst] = lengths[src]
    refs.index_add_(0, pages.clamp(min=0).reshape(-1).long(), (pages >= 0).int().reshape(-1))
    # extend each child by one token: a page of its own where the open one is shared
    lens = lengths[dst].long()
    last = table[dst, (lens - 1).clamp(min=0) // page].long()
    shared = (last[:, None] == last[None, :]).tril(-1).sum(1)
    is_open = lens % page != 0
    copy = is_open & (refs[last.clamp(min=0)] - shared > 1)
    count = (copy | ~is_open).long()
    at = count.cumsum(0) - count
    free = torch.nonzero(refs == 0)[:, 0]
    take = count > 0
    given = free[at[take]]
    table[dst[take], lens[take] // page] = given.int()
    pool[:, free[at[copy]]] = pool[:, last[copy]]
    refs[given] = 1
    refs.index_add_(0, last[copy], torch.full_like(last[copy], -1, dtype=torch.int32))
    lengths[dst] += 1
    return {"table": table, "lengths": lengths, "refs": refs, "pool": pool.view(-1).view(torch.int64)}


def _plain_compact(s):
    s["meta"].copy_(s["saved"])
    table, refs, pool = s["table"], s["refs"], s["pool"]
    ids = torch.arange(len(refs), device="cuda")
    live = refs > 0
    n = live.sum()
    to, src = ids[~live & (ids < n)], ids[live & (ids >= n)]
    pool[:, to] = pool[:, src]
    new = ids.clone()
    new[src] = to
    table.copy_(torch.where(table >= 0, new[table.clamp(min=0).long()].int(), table))
    refs[to] = refs[src]
    refs[src] = 0
    return {"table": table, "refs": refs, "live": n.int().view(1), "pool": pool.view(-1).view(torch.int64)}


# ------------------------------------------------------------------ one pass
def run(s):
    if not own:
        return {"attend": _plain_attend, "append": _plain_append, "fork": _plain_fork,
                "compact": _plain_compact}[s["op"]](s)
    K = _kernels()
    if "workspace" not in s:
        s["workspace"] = K.DecodeWorkspace()
    if s["op"] == "attend":
        K.paged_attention(s["q"], s["pool"], s["table"], s["lengths"], s["kind"], indptr=s["indptr"],
                          max_new=s["most"], window=s["window"], out=s["out"], ml_out=s["ml"],
                          workspace=s["workspace"])
        return {"out": s["out"], "ml": s["ml"]}
    if s["op"] == "append":
        K.paged_append(s["k"], s["v"], s["pool"], s["table"], s["lengths"], s["kind"], indptr=s["indptr"],
                       max_new=s["most"])
        k, v = K.paged_read(s["pool"], s["table"], s["lengths"], s["kind"], s["starts"], s["back"],
                            s["back_total"], dtype=TYPES[s["dtype"]])
        return {"k": k, "v": v}
    # pages are moved as they are, so their bytes are what a pass returns
    if s["op"] == "fork":
        meta = (s["table"], s["lengths"], s["refs"])
        K.paged_free(*meta, s["dst"], s["page"], s["status"])
        K.paged_fork(*meta, s["src"], s["dst"], s["page"], s["status"])
        K.paged_extend(s["pool"], *meta, s["dst"], 1, s["status"], workspace=s["workspace"])
        return {"table": s["table"], "lengths": s["lengths"], "refs": s["refs"], "pool": s["pool"].view(-1).view(torch.int64)}
    s["meta"].copy_(s["saved"])
    live = K.paged_compact(s["pool"], s["table"], s["refs"], workspace=s["workspace"])
    return {"table": s["table"], "refs": s["refs"], "live": live, "pool": s["pool"].view(-1).view(torch.int64)}


def _kernels():
    here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "kvquant-paper-repro_b200")
    if here not in sys.path:
        sys.path.insert(0, here)
    import kvquant.kernels as K
    return K


# ------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    if case["op"] not in ("attend", "append"):
        return None  # whole numbers and moved bytes
    s = prepare(case, seed)
    lens, new = _lengths(case)
    dim, heads, page, kind = case["dim"], case["heads"], case["page"], case["kind"]
    t, d = torch.arange(BLOCK, device="cuda")[:, None], torch.arange(dim, device="cuda")[None, :]
    at_k = d // 32 * 512 + t % 8 * 64 + d // 4 % 4 * 16 + d // 16 % 2 * 8 + t // 8 * 4 + d % 4
    at_v = 16 * dim + d // 32 * 512 + d % 8 * 64 + t // 2 % 4 * 16 + d // 16 % 2 * 8 + d // 8 % 2 * 4 + t // 8 * 2 + t % 2

    def value(byte):
        if kind == "int8":
            return byte.double() - 128
        b = byte.long()
        e, f = b >> 3 & 15, (b & 7).double()
        mag = torch.where(e == 0, f * 2.0 ** -9, torch.ldexp(1 + f / 8, e - 7))
        return torch.where(b >= 128, -mag, mag)

    def stored(i, h, n):
        """keys, values of the first n tokens of sequence i, head h, and the codes and scales"""
        held = s["table"][i, :-(-n // page)].long()
        rec = s["pool"][held, h].reshape(-1, s["pool"].shape[-1])[:-(-n // BLOCK)]
        sc = rec[:, 32 * dim:32 * dim + 8].contiguous().view(torch.float32).double()
        kc, vc = value(rec[:, at_k]), value(rec[:, at_v])
        return kc, vc, sc

    if case["op"] == "attend":
        group = case["group"]
        out = torch.zeros((s["total"], heads * group, dim), dtype=torch.float64, device="cuda")
        ml = torch.zeros((s["total"], heads * group, 2), dtype=torch.float64, device="cuda")
        row = 0
        for i, (n, m) in enumerate(zip(lens, new)):
            for h in range(heads if m else 0):
                kc, vc, sc = stored(i, h, n)
                k = (kc * sc[:, 0, None, None]).reshape(-1, dim)[:n]
                v = (vc * sc[:, 1, None, None]).reshape(-1, dim)[:n]
                pos = torch.arange(n - m, n, device="cuda")
                j = torch.arange(n, device="cuda")
                hide = j[None, :] > pos[:, None]
                if case["window"]:
                    hide |= j[None, :] <= pos[:, None] - case["window"]
                for g in range(group):
                    x = s["q"][row:row + m, h * group + g].double() @ k.T / math.sqrt(dim)
                    x.masked_fill_(hide, -math.inf)
                    top = x.max(1).values
                    p = torch.exp(x - top[:, None])
                    z = p.sum(1)
                    out[row:row + m, h * group + g] = p @ v / z[:, None]
                    ml[row:row + m, h * group + g] = torch.stack([top, 1 / z], 1)
            row += m
        return {"out": out, "ml": ml}

    def near(y):
        if kind == "int8":
            return torch.round(y).clamp(-127, 127)
        y = y.clamp(-448, 448)
        unit = torch.ldexp(torch.ones_like(y), torch.frexp(y).exponent.clamp(min=-5) - 4)
        return torch.round(y / unit) * unit

    got = {"k": [], "v": []}
    row = 0
    for i, (n, m) in enumerate(zip(lens, new)):
        if not m:
            continue
        a = n - m
        first = a // BLOCK * BLOCK
        pad = -(-n // BLOCK) * BLOCK - n
        kc, vc, sc = zip(*(stored(i, h, n) for h in range(heads)))
        for name, codes, which in (("k", kc, 0), ("v", vc, 1)):
            code = torch.stack(codes, 1)[first // BLOCK:]  # [blocks, heads, 16, dim]
            old = torch.stack(sc, 1)[first // BLOCK:, :, which]
            x = torch.zeros((n - first + pad, heads, dim), dtype=torch.float64, device="cuda")
            x[a - first:n - first] = s[name][row:row + m].double()
            x = x.view(-1, BLOCK, heads, dim).transpose(1, 2)
            scale = x.abs().amax((2, 3)).div(QMAX[kind]).clamp(min=FLOOR)
            if a > first:
                scale[0] = torch.maximum(scale[0], old[0])
            y = near(x / scale[..., None, None]) * scale[..., None, None]
            if a > first:
                f = (old[0] / scale[0])[:, None, None]
                y[0, :, :a - first] = (torch.where(f < 1, near(code[0] * f), code[0]) * scale[0][:, None, None])[:, :a - first]
            got[name].append(y.transpose(1, 2).reshape(-1, heads, dim)[:n - first])
        row += m
    return {name: torch.cat(x) if x else torch.zeros((0, heads, dim), dtype=torch.float64) for name, x in got.items()}
