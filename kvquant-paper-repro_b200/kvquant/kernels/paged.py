"""Paged 8-bit KV cache: append, read, attention and page operations.

No counterpart in the reference, whose cache is one contiguous slot per layer
(kvquant/kv_cache.py:4-44). Keys (as the attention uses them, i.e. rotated) and
values are held in 8 bits with one scale per 16 tokens and KV head, in pages
that sequences may share.

A layer's pool is uint8 [n_pages, heads, page_tokens / 16, 32 * D + 16] (see
pool_shape): one record per 16 tokens and head. `kind` names the codes: "int8"
(largest code 127) or "e4m3" (8-bit float, largest 448). table int32 [slots,
columns] holds each slot's pages in token order (-1: none), lengths int32 [slots]
its tokens, refs int32 [n_pages] how many slots hold a page; all three live on the
device and nothing here copies them to the host. kvquant.paged_cache.PagedKVCache
keeps them together for all layers of a model.

A call's rows (k, v, q) are the new tokens of its sequences, one after another:
indptr int32 [B + 1] gives each sequence's rows, or every sequence has the same
number. slots int32 [B] names their slots (default: 0, 1, ...). lengths already
counts the new tokens (paged_extend), which are the last ones of their slots.
A slot appears at most once in a call.

All tensors are CUDA tensors; work is launched on the current stream. Page ids,
slots and row ranges that are out of range are skipped and reported by
get_cuda_ops().check_status(); output rows of a skipped sequence, and rows that indptr gives
to none, are not written.
"""
from __future__ import annotations

import torch

from .cuda_ops import _check, _ptr, get_cuda_ops
from .decode import DecodeWorkspace

BLOCK_TOKENS = 16
MAX_NEW = 65536  # most rows of one sequence in a call of paged_attention
KINDS = {"int8": 0, "e4m3": 1}
_DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}


# Calls take microseconds on the GPU, so the checks below use the cheapest form of each
# question (device numbers, identity of dtypes) and the device is switched only when it
# has to be.
_current_device = torch.cuda.current_device
_raw_stream = torch._C._cuda_getCurrentRawStream


def _launch(fn, lib, dev: int, *args) -> None:
    """fn(*args, current stream of device dev) with dev current."""
    if dev == _current_device():
        rc = fn(*args, _raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _raw_stream(dev))
    if rc:
        _check(rc, lib)


def record_bytes(head_dim: int) -> int:
    return 32 * head_dim + 16


def pool_shape(n_pages: int, heads: int, head_dim: int, page_tokens: int) -> tuple:
    """Shape of one layer's pool (uint8)."""
    return n_pages, heads, page_tokens // BLOCK_TOKENS, record_bytes(head_dim)


def _int32(what: str, name: str, t, dev: int, n: int | None = None):
    """Pointer of a contiguous int32 tensor on device dev (with n elements), or None."""
    if t is None:
        return None
    if (t.dtype is not torch.int32 or t.get_device() != dev or not t.is_contiguous()
            or (n is not None and t.numel() != n)):
        size = "" if n is None else f" with {n} elements"
        raise RuntimeError(f"{what}: {name} must be contiguous int32{size} on cuda:{dev}")
    return t.data_ptr()


def _cache_args(what: str, pool, kind, table, lengths, slots, indptr):
    """The arguments that describe a layer's cache and a call's sequences, the latter's
    number, KV heads, channels and the device."""
    dev = pool.get_device()
    if dev < 0:
        raise RuntimeError(f"{what}: kvquant_b200 runs on CUDA tensors only")
    if pool.dtype is not torch.uint8 or pool.dim() != 4 or not pool.is_contiguous():
        raise RuntimeError(f"{what}: pool must be contiguous uint8 [pages, heads, blocks, record]")
    code = KINDS.get(kind)
    if code is None:
        raise RuntimeError(f"{what}: kind must be one of {sorted(KINDS)}, got {kind!r}")
    n_pages, heads, blocks, rec = pool.shape
    if rec % 32 != 16:
        raise RuntimeError(f"{what}: the pool's records have {rec} bytes, not 32 * D + 16")
    if table.dim() != 2:
        raise RuntimeError(f"{what}: table must be [slots, columns]")
    n_slots, n_cols = table.shape
    B = (indptr.numel() - 1 if indptr is not None else n_slots if slots is None
         else slots.numel())
    dim = rec // 32
    return (pool.data_ptr(), code, n_pages, heads, dim, blocks * BLOCK_TOKENS,
            _int32(what, "table", table, dev), n_slots, n_cols,
            _int32(what, "lengths", lengths, dev, n_slots),
            _int32(what, "slots", slots, dev, B)), \
        _int32(what, "indptr", indptr, dev), B, heads, dim, dev


def _rows(what: str, name: str, t, heads, dim, dev: int):
    """t [N, heads, dim] with 16-byte rows, and its strides; copied when they do not allow
    that."""
    if t.dim() != 3 or t.get_device() != dev or t.shape[1:] != (heads, dim):
        raise RuntimeError(f"{what}: {name} must be [rows, {heads}, {dim}] on cuda:{dev}, "
                           f"got {tuple(t.shape)} on {t.device}")
    row, head, one = t.stride()
    if one != 1 or row % 8 or head % 8 or t.data_ptr() % 16:
        t = t.contiguous()
        if t.data_ptr() % 16:
            t = t.clone()
        row, head, _ = t.stride()
    return t, row, head


def paged_append(k: torch.Tensor, v: torch.Tensor, pool: torch.Tensor, table: torch.Tensor,
                 lengths: torch.Tensor, kind: str, slots: torch.Tensor | None = None,
                 indptr: torch.Tensor | None = None, max_new: int | None = None,
                 granted: torch.Tensor | None = None) -> None:
    """Writes the new tokens' keys and values [N, heads, D] (fp16 or bf16) into their blocks.

    A block that the call starts gets the scale max|x| / largest code (at least
    2**-32) over its new tokens; a block that is open already keeps the larger of
    its own scale and that, its older codes rounded anew when the scale grew. Codes
    are rounded to nearest even; infinities are stored as the largest code, NaN as 0,
    and neither counts towards the scale. max_new is accepted for symmetry with
    paged_attention and not needed.

    granted (int32 [slots], kept by paged_extend): sequences whose rows reach before the
    first token that their slot's last extend granted are skipped and flagged, so that an
    append after a refused extend leaves what is stored alone. Without it the caller has
    to know that the extend was not refused: the rows would overwrite the slots' last
    tokens, in shared pages too.
    """
    what = "paged_append"
    cache, ip, B, heads, dim, dev = _cache_args(what, pool, kind, table, lengths, slots, indptr)
    k, k_row, k_head = _rows(what, "k", k, heads, dim, dev)
    v, v_row, v_head = _rows(what, "v", v, heads, dim, dev)
    code = _DTYPES.get(k.dtype, 2)
    if k.shape != v.shape or k.dtype is not v.dtype or code == 2:
        raise RuntimeError("paged_append: k and v must have one shape and be fp16 or bf16")
    lib = get_cuda_ops().lib
    _launch(lib.kvq_paged_append_granted, lib, dev, k.data_ptr(), k_row, k_head, v.data_ptr(), v_row,
            v_head, code, *cache, ip, B, k.shape[0],
            _int32(what, "granted", granted, dev, cache[7]))


def paged_read(pool: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, kind: str,
               starts: torch.Tensor | None, indptr: torch.Tensor | None, total: int,
               slots: torch.Tensor | None = None, dtype: torch.dtype = torch.float16):
    """The values (code * scale) of the tokens [starts[b], starts[b] + rows of b) of each
    sequence: (k, v), both [total, heads, D] in fp16, bf16 or fp32. starts None: from 0."""
    what = "paged_read"
    cache, ip, B, heads, dim, dev = _cache_args(what, pool, kind, table, lengths, slots, indptr)
    code = _DTYPES.get(dtype)
    if code is None:
        raise RuntimeError(f"paged_read: dtype must be fp16, bf16 or fp32, got {dtype}")
    k, v = torch.empty((2, int(total), heads, dim), dtype=dtype, device=pool.device).unbind(0)
    lib = get_cuda_ops().lib
    _launch(lib.kvq_paged_read, lib, dev, *cache, _int32(what, "starts", starts, dev, B), ip, B,
            int(total), k.data_ptr(), v.data_ptr(), code)
    return k, v


def paged_attention(q: torch.Tensor, pool: torch.Tensor, table: torch.Tensor,
                    lengths: torch.Tensor, kind: str, slots: torch.Tensor | None = None,
                    indptr: torch.Tensor | None = None, max_new: int | None = None,
                    scale: float | None = None, window: int = 0,
                    out: torch.Tensor | None = None, ml_out: torch.Tensor | None = None,
                    workspace: DecodeWorkspace | None = None) -> torch.Tensor:
    """Causal attention of the new tokens' queries over their sequences' cached tokens.

    q [N, Hq, D] (fp16 or bf16): a sequence's rows are its last tokens, a row sees the
    tokens up to its own position (with window > 0 the last `window` of those). Query
    head hq reads KV head hq // (Hq / heads). Returns [N, Hq, D] in q's type; rows that
    see nothing are 0. ml_out (fp32 [N, Hq, 2], optional) receives each row's softmax
    statistics (M, 1/L) of softmax(scores * scale), (-inf, inf) for such rows: with
    the fp16 outputs merge_shards joins them with other parts of the same context.
    max_new: the most rows of any sequence, at most 65536 (a sequence with more is skipped and
    flagged). Give it with indptr: it also picks the kernel, and the default there, N or
    65536 if N is more, takes a batch of single tokens for one prompt chunk and pads every
    sequence to 256 rows. scale defaults to 1 / sqrt(D).
    """
    what = "paged_attention"
    cache, ip, B, heads, dim, dev = _cache_args(what, pool, kind, table, lengths, slots, indptr)
    if q.dim() != 3 or q.shape[1] == 0 or q.shape[1] % heads:
        raise RuntimeError(f"paged_attention: q {tuple(q.shape)} does not match {heads} KV heads")
    N, Hq, _ = q.shape
    q, row, head = _rows(what, "q", q, Hq, dim, dev)
    code = _DTYPES.get(q.dtype, 2)
    if code == 2:
        raise RuntimeError("paged_attention: q must be fp16 or bf16")
    if out is None:
        out = torch.empty((N, Hq, dim), dtype=q.dtype, device=q.device)
    elif (out.shape != q.shape or out.dtype is not q.dtype or out.get_device() != dev
          or not out.is_contiguous()):
        raise RuntimeError("paged_attention: out must be contiguous, of q's shape and type")
    if ml_out is not None and (ml_out.dtype is not torch.float32 or not ml_out.is_contiguous()
                               or ml_out.numel() != N * Hq * 2 or ml_out.get_device() != dev):
        raise RuntimeError("paged_attention: ml_out must be contiguous fp32 [N, Hq, 2]")
    if max_new is None:
        max_new = min(N, MAX_NEW) if indptr is not None else N // max(1, B)
    lib = get_cuda_ops().lib
    need = lib.kvq_paged_attention_workspace(dim, max_new, Hq // heads)
    ws = (workspace or DecodeWorkspace()).get(need, pool.device)
    _launch(lib.kvq_paged_attention, lib, dev, q.data_ptr(), row, head, code, Hq // heads, *cache,
            ip, B, N, max_new, dim ** -0.5 if scale is None else scale, window, out.data_ptr(),
            _ptr(ml_out), ws.data_ptr(), ws.numel())
    return out


# ---------------------------------------------------------------------------
# Page operations
# ---------------------------------------------------------------------------
NO_PAGES, BAD_SLOT = 1, 2  # bits of `status`


def _meta_args(what: str, table, lengths, refs, page_tokens):
    dev = table.get_device()
    if dev < 0 or table.dim() != 2:
        raise RuntimeError(f"{what}: table must be a CUDA tensor [slots, columns]")
    n_slots, n_cols = table.shape
    return (_int32(what, "table", table, dev), n_slots, n_cols,
            _int32(what, "lengths", lengths, dev, n_slots), _int32(what, "refs", refs, dev),
            refs.numel(), page_tokens), dev


def _pool_args(what: str, pool):
    """(pointer, layers, bytes between layers, bytes of a page), pages and page tokens of a
    pool [pages, ...] or [layers, pages, ...]."""
    if not pool.is_cuda or pool.dtype is not torch.uint8 or pool.dim() not in (4, 5):
        raise RuntimeError(f"{what}: pool must be a CUDA uint8 tensor [pages, heads, blocks, "
                           "record] or [layers, pages, heads, blocks, record]")
    if not pool.is_contiguous():
        raise RuntimeError(f"{what}: pool must be contiguous")
    *layers, pages, heads, blocks, rec = pool.shape
    page = heads * blocks * rec
    return (pool.data_ptr(), layers[0] if layers else 1, pages * page, page), pages, \
        blocks * BLOCK_TOKENS


def paged_free(table, lengths, refs, slots, page_tokens: int, status) -> None:
    """Gives up the pages of the slots (int32): counts down, rows -1, lengths 0. status
    (int32 [1]) gets BAD_SLOT for a slot out of range or named twice, which is skipped."""
    what = "paged_free"
    meta, dev = _meta_args(what, table, lengths, refs, page_tokens)
    lib = get_cuda_ops().lib
    _launch(lib.kvq_paged_free, lib, dev, *meta, _int32(what, "slots", slots, dev), slots.numel(),
            _int32(what, "status", status, dev, 1))


def paged_fork(table, lengths, refs, src, dst, page_tokens: int, status) -> None:
    """dst[i] becomes a copy of src[i] that shares all its pages (an open last page too:
    paged_extend gives a writer its own copy). A pair whose dst holds tokens, is a src,
    is named twice or is out of range is skipped and sets BAD_SLOT in status."""
    what = "paged_fork"
    meta, dev = _meta_args(what, table, lengths, refs, page_tokens)
    n = src.numel()
    lib = get_cuda_ops().lib
    _launch(lib.kvq_paged_fork, lib, dev, *meta, _int32(what, "src", src, dev),
            _int32(what, "dst", dst, dev, n), n, _int32(what, "status", status, dev, 1))


def paged_extend(pool, table, lengths, refs, slots, n_new, status,
                 workspace: DecodeWorkspace | None = None,
                 granted: torch.Tensor | None = None) -> None:
    """Room for n_new (int, or int32 per slot) more tokens in every slot; lengths grow.

    Free pages are taken in ascending order, slot after slot. A slot whose last page is
    open and shared gets its own copy of it, in every layer of pool ([layers, ...] or one
    layer's), unless all other holders stand before it in `slots`. When pages run out
    (NO_PAGES in status), or a slot is out of range, named twice or too long for its row
    (BAD_SLOT), nothing changes. granted (int32 [slots of the table], for paged_append)
    gets each slot's first new token, or 2**31 - 1 when the call is refused.
    """
    what = "paged_extend"
    where, pages, page_tokens = _pool_args(what, pool)
    meta, dev = _meta_args(what, table, lengths, refs, page_tokens)
    if meta[5] != pages or pool.get_device() != dev:
        raise RuntimeError(f"{what}: refs must have one entry per page of the pool")
    n = slots.numel()
    each = isinstance(n_new, torch.Tensor)
    lib = get_cuda_ops().lib
    ws = (workspace or DecodeWorkspace()).get(lib.kvq_paged_extend_workspace(pages), pool.device)
    _launch(lib.kvq_paged_extend_granting, lib, dev, *where, *meta,
            _int32(what, "slots", slots, dev), n,
            _int32(what, "n_new", n_new, dev, n) if each else None, 0 if each else n_new,
            _int32(what, "status", status, dev, 1), ws.data_ptr(), ws.numel(),
            _int32(what, "granted", granted, dev, meta[1]))


def paged_compact(pool, table, refs, workspace: DecodeWorkspace | None = None,
                  n_live: torch.Tensor | None = None) -> torch.Tensor:
    """Moves the live pages to the lowest ids: those at or past their number, in
    ascending order, into the free ones below it, in every layer; table and refs follow.
    Returns the number of live pages (int32 [1] on the device)."""
    what = "paged_compact"
    where, pages, _ = _pool_args(what, pool)
    dev = table.get_device()
    if refs.numel() != pages or pool.get_device() != dev or table.dim() != 2:
        raise RuntimeError(f"{what}: refs must have one entry per page of the pool")
    if n_live is None:
        n_live = torch.empty(1, dtype=torch.int32, device=pool.device)
    lib = get_cuda_ops().lib
    ws = (workspace or DecodeWorkspace()).get(lib.kvq_paged_extend_workspace(pages), pool.device)
    _launch(lib.kvq_paged_compact, lib, dev, *where, _int32(what, "table", table, dev),
            *table.shape, _int32(what, "refs", refs, dev), pages,
            _int32(what, "n_live", n_live, dev, 1), ws.data_ptr(), ws.numel())
    return n_live


def paged_copy(src_pool, dst_pool, src, dst, workspace: DecodeWorkspace | None = None) -> None:
    """Copies pages src[i] of src_pool to pages dst[i] of dst_pool (which may be the same
    pool), every layer. dst pages are distinct, and in one pool none of them is in src."""
    what = "paged_copy"
    (sp, layers, s_stride, page), s_pages, _ = _pool_args(what, src_pool)
    (dp, d_layers, d_stride, d_page), d_pages, _ = _pool_args(what, dst_pool)
    dev = src_pool.get_device()
    if layers != d_layers or page != d_page or dst_pool.get_device() != dev:
        raise RuntimeError(f"{what}: the pools differ in layers, page size or device")
    n = src.numel()
    lib = get_cuda_ops().lib
    ws = (workspace or DecodeWorkspace()).get(lib.kvq_paged_copy_workspace(n), src_pool.device)
    _launch(lib.kvq_paged_copy, lib, dev, sp, s_pages, s_stride, dp, d_pages, d_stride, layers,
            page, _int32(what, "src", src, dev), _int32(what, "dst", dst, dev, n), n,
            ws.data_ptr(), ws.numel())
