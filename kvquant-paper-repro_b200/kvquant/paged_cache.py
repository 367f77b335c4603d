"""Paged 8-bit KV cache of a whole model (no counterpart in the reference, whose
QuantizedKVCache holds one slot per layer, kvquant/kv_cache.py:12-32).

A slot is one sequence. Its pages are shared by all layers: page p of layer l is
pool[l, p]. Table, lengths and reference counts live on the device and only kernels
change them, so a decode loop neither synchronises nor copies them to the host, and
its calls can be captured in a CUDA graph. (Slots as int32 tensors: a Python list is
copied to the device by every call that gets it, which waits for the copy.)

    cache = PagedKVCache(n_layers=32, n_pages=4096, heads=8, max_slots=64, max_tokens=8192)
    cache.extend(slots, n_new)                      # room for the new tokens; lengths grow
    for layer in range(32):
        cache.append(layer, k, v, slots, indptr)    # the new tokens' rotated keys, values
        o = cache.attend(layer, q, slots, indptr, max_new=most)  # causal over everything cached
    cache.fork(src, dst)                            # dst share src's pages (copy-on-write)
    cache.free(slots); cache.compact()
    cache.check()                                   # RuntimeError if something was refused

append writes only tokens that the slot's last extend granted. When an extend is refused
(no free pages, a bad slot), the appends of its slots write nothing until an extend of theirs
is granted, and their attend sees the tokens stored before.
"""
from __future__ import annotations

import torch

from .kernels import (DecodeWorkspace, paged_append, paged_attention, paged_compact,
                      paged_extend, paged_fork, paged_free, paged_read)
from .kernels.cuda_ops import get_cuda_ops
from .kernels.paged import BAD_SLOT, KINDS, NO_PAGES, pool_shape


class PagedKVCache:
    def __init__(self, n_layers: int, n_pages: int, heads: int, max_slots: int, max_tokens: int,
                 head_dim: int = 128, page_tokens: int = 64, kind: str = "int8", device="cuda"):
        if kind not in KINDS:
            raise RuntimeError(f"PagedKVCache: kind must be one of {sorted(KINDS)}, got {kind!r}")
        if head_dim not in (64, 128):
            raise RuntimeError(f"PagedKVCache: head_dim must be 64 or 128, got {head_dim}")
        if page_tokens < 16 or page_tokens > 1024 or page_tokens % 16:
            raise RuntimeError("PagedKVCache: page_tokens must be a multiple of 16 in 16..1024, "
                               f"got {page_tokens}")
        if min(n_layers, n_pages, heads, max_slots, max_tokens) < 1:
            raise RuntimeError("PagedKVCache: sizes must be positive")
        dev = torch.device(device)
        if dev.type != "cuda":
            raise RuntimeError("PagedKVCache: kvquant_b200 runs on CUDA devices only")
        self.kind, self.page_tokens, self.heads, self.head_dim = kind, page_tokens, heads, head_dim
        self.pool = torch.zeros((n_layers, *pool_shape(n_pages, heads, head_dim, page_tokens)),
                                dtype=torch.uint8, device=dev)
        ints = dict(dtype=torch.int32, device=dev)
        self.table = torch.full((max_slots, -(-max_tokens // page_tokens)), -1, **ints)
        self.lengths = torch.zeros(max_slots, **ints)
        self.refs = torch.zeros(n_pages, **ints)
        self.status = torch.zeros(1, **ints)
        # the first token that a slot's last extend granted; none yet
        self.granted = torch.full((max_slots,), 2 ** 31 - 1, **ints)
        # One stream at a time. As large as any call needs (20 or 40 MB at head_dim 64 or 128):
        # a buffer that grew would leave captured calls with an address that is given back.
        lib = get_cuda_ops().lib
        self.workspace = DecodeWorkspace()
        self.workspace.get(max(lib.kvq_paged_extend_workspace(n_pages),
                               *(lib.kvq_paged_attention_workspace(head_dim, n, 1)
                                 for n in (1, 48, 65536))), self.pool.device)

    def _slots(self, slots):
        if slots is None or isinstance(slots, torch.Tensor):
            return slots
        return torch.tensor(slots, dtype=torch.int32, device=self.table.device)

    # -- pages --------------------------------------------------------------------
    def extend(self, slots, n_new) -> None:
        """Room for n_new (int, or int32 tensor) more tokens in each of the slots."""
        paged_extend(self.pool, self.table, self.lengths, self.refs, self._slots(slots), n_new,
                     self.status, workspace=self.workspace, granted=self.granted)

    def fork(self, src, dst) -> None:
        """dst[i] (empty) becomes a copy of src[i] that shares its pages."""
        paged_fork(self.table, self.lengths, self.refs, self._slots(src), self._slots(dst),
                   self.page_tokens, self.status)

    def free(self, slots) -> None:
        """Empties the slots; pages that nobody else holds are free again."""
        paged_free(self.table, self.lengths, self.refs, self._slots(slots), self.page_tokens,
                   self.status)

    def compact(self) -> torch.Tensor:
        """Moves the live pages to the lowest ids; their number (int32 [1], on the device)."""
        return paged_compact(self.pool, self.table, self.refs, workspace=self.workspace)

    def check(self) -> None:
        """Raises RuntimeError when a page operation since the last check was refused (one
        host synchronisation)."""
        s = int(self.status.item())
        if s:
            self.status.zero_()
            why = [t for bit, t in ((NO_PAGES, "no free pages"), (BAD_SLOT, "a bad slot")) if s & bit]
            raise RuntimeError(f"PagedKVCache: {' and '.join(why)}; nothing was changed for it "
                               "and its tokens were not written")

    # -- tokens -------------------------------------------------------------------
    def append(self, layer: int, k, v, slots=None, indptr=None) -> None:
        """Writes the new tokens' keys and values [N, heads, D]: the last ones of the slots, as
        far as their last extend granted them."""
        paged_append(k, v, self.pool[layer], self.table, self.lengths, self.kind,
                     slots=self._slots(slots), indptr=indptr, granted=self.granted)

    def attend(self, layer: int, q, slots=None, indptr=None, max_new=None, **kw):
        """Causal attention of the new tokens' queries [N, Hq, D]. With indptr give max_new, the
        most rows of any slot (see paged_attention)."""
        return paged_attention(q, self.pool[layer], self.table, self.lengths, self.kind,
                               slots=self._slots(slots), indptr=indptr, max_new=max_new,
                               workspace=self.workspace, **kw)

    def read(self, layer: int, starts, indptr, total: int, slots=None, dtype=torch.float16):
        """Stored values of the slots' tokens [starts, starts + rows) (see paged_read)."""
        return paged_read(self.pool[layer], self.table, self.lengths, self.kind, starts, indptr,
                          total, slots=self._slots(slots), dtype=dtype)

    def memory_bytes(self) -> int:
        return sum(t.numel() * t.element_size()
                   for t in (self.pool, self.table, self.lengths, self.refs))
