#!/usr/bin/env python
"""Parallel sampling over a paged 8-bit KV cache: prompts of unlike length, several samples
of each that share the prompt's pages, finished samples dropped, the pool closed up.

The "model" is a stack of attention layers with random weights (no MLP, no vocabulary):
enough to run the cache as a decoder would, step by step, and to compare the outputs with
the same stack over an unquantised fp32 cache.

  python examples/paged_sampling.py [--layers 2] [--samples 4] [--steps 40] [--kind int8|e4m3]
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "kvquant-paper-repro_b200"))

from kvquant.kernels.cuda_ops import get_cuda_ops  # noqa: E402
from kvquant.paged_cache import PagedKVCache  # noqa: E402


class Stack:
    """Attention layers x += Wo attention(q, k, v): projections only, fp16."""

    def __init__(self, layers, width, hq, hkv, dim, dev, seed=0):
        g = torch.Generator(device=dev).manual_seed(seed)
        w = lambda a, b: torch.randn(layers, a, b, generator=g, device=dev).mul_(a ** -0.5).half()  # noqa: E731
        self.q, self.k, self.v, self.o = w(width, hq * dim), w(width, hkv * dim), \
            w(width, hkv * dim), w(hq * dim, width)
        self.layers, self.hq, self.hkv, self.dim = layers, hq, hkv, dim

    def run(self, x, attention):
        """x [N, width] fp16; attention(layer, q, k, v) -> [N, hq, dim]."""
        for i in range(self.layers):
            h = torch.nn.functional.rms_norm(x, x.shape[-1:])
            q, k, v = ((h @ w[i]).view(len(x), -1, self.dim) for w in (self.q, self.k, self.v))
            x = x + attention(i, q, k, v).reshape(len(x), -1) @ self.o[i]
        return x


class Dense:
    """The same attention over plain fp32 lists of every sequence's keys and values."""

    def __init__(self, layers):
        self.kv = [{} for _ in range(layers)]

    def fork(self, src, dst):
        for kv in self.kv:
            for a, b in zip(src, dst):
                kv[b] = tuple(x.clone() for x in kv[a])

    def attend(self, layer, q, k, v, slots, rows):
        out, r = [], 0
        for s, n in zip(slots, rows):
            old = self.kv[layer].get(s)
            new = k[r:r + n].float(), v[r:r + n].float()
            kk, vv = new if old is None else (torch.cat([a, b]) for a, b in zip(old, new))
            self.kv[layer][s] = kk, vv
            G = q.shape[1] // kk.shape[1]
            x = torch.einsum("nhd,thd->hnt", q[r:r + n].float(), kk.repeat_interleave(G, 1))
            x = x * q.shape[-1] ** -0.5
            t = torch.arange(len(kk), device=q.device)
            x = x.masked_fill(t[None, None] > (len(kk) - n + torch.arange(n, device=q.device))[None, :, None],
                              float("-inf"))
            out.append(torch.einsum("hnt,thd->nhd", x.softmax(-1), vv.repeat_interleave(G, 1)))
            r += n
        return torch.cat(out).half()


def main(argv=None):
    ap = argparse.ArgumentParser()
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--samples", type=int, default=4)
    ap.add_argument("--steps", type=int, default=40)
    ap.add_argument("--kind", choices=["int8", "e4m3"], default="int8")
    args = ap.parse_args(argv)
    dev = torch.device("cuda", torch.cuda.current_device())
    width, hq, hkv, dim = 512, 8, 2, 64
    prompts = [700, 33, 256]
    n_p, n_s = len(prompts), len(prompts) * args.samples
    net = Stack(args.layers, width, hq, hkv, dim, dev)
    cache = PagedKVCache(args.layers, n_pages=256, heads=hkv, max_slots=n_p + n_s, max_tokens=2048,
                         head_dim=dim, kind=args.kind, device=dev)
    dense = Dense(args.layers)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    worst = 0.0

    def step(x, slots, rows):
        """One pass of the stack over new tokens of the slots, on both caches."""
        nonlocal worst
        s, n = ints(slots), ints(rows)
        indptr = torch.nn.functional.pad(n.cumsum(0, dtype=torch.int32), (1, 0))
        cache.extend(s, n)

        def paged(i, q, k, v):
            cache.append(i, k, v, s, indptr)
            return cache.attend(i, q, s, indptr, max_new=max(rows))
        got = net.run(x, paged)
        want = net.run(x, lambda i, q, k, v: dense.attend(i, q, k, v, slots, rows))
        worst = max(worst, float((got.float() - want.float()).norm() / want.float().norm()))
        return got

    torch.manual_seed(1)
    x = step(torch.randn(sum(prompts), width, device=dev).half(), list(range(n_p)), prompts)
    src = [p for p in range(n_p) for _ in range(args.samples)]
    live = [n_p + i for i in range(n_s)]
    cache.fork(src, live)
    dense.fork(src, live)
    cache.free(list(range(n_p)))  # the prompts' own slots; the samples hold their pages
    n_live = cache.compact()
    x = x[(ints(prompts).cumsum(0) - 1).long()].repeat_interleave(args.samples, 0)
    for i in range(args.steps):
        x = step(x + 0.3 * torch.randn_like(x), live, [1] * len(live))
        if i == args.steps // 2:  # every third sample is done: drop it, close the pool up
            done, keep = live[::3], [j for j in range(len(live)) if j % 3]
            cache.free(done)
            n_live = cache.compact()
            live, x = [live[j] for j in keep], x[keep]
    cache.check()
    get_cuda_ops().check_status(dev)
    used = int((cache.refs > 0).sum())
    assert int(n_live) <= used <= cache.refs.numel()
    print(f"{args.kind}: {n_s} samples of {n_p} prompts, {args.steps} steps, {used} live pages; largest "
          f"rel-L2 distance of a step's outputs from the fp32 cache {worst:.2e}")
    return worst


if __name__ == "__main__":
    main()
