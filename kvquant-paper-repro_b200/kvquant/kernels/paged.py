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
get_cuda_ops().check_status().
"""
from __future__ import annotations

import math

import torch

from .cuda_ops import _check, _ptr, get_cuda_ops
from .decode import DecodeWorkspace

BLOCK_TOKENS = 16
KINDS = {"int8": 0, "e4m3": 1}
_DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}


def _launch(fn, lib, dev, *args) -> None:
    """fn(*args, current stream of dev) with dev current. These calls take microseconds on
    the GPU, so the device is switched only when it has to be."""
    i = dev.index
    if i == torch.cuda.current_device():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(i))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(i))
    if rc:
        _check(rc, lib)


def record_bytes(head_dim: int) -> int:
    return 32 * head_dim + 16


def pool_shape(n_pages: int, heads: int, head_dim: int, page_tokens: int) -> tuple:
    """Shape of one layer's pool (uint8)."""
    return n_pages, heads, page_tokens // BLOCK_TOKENS, record_bytes(head_dim)


def _kind(what: str, kind: str) -> int:
    if kind not in KINDS:
        raise RuntimeError(f"{what}: kind must be one of {sorted(KINDS)}, got {kind!r}")
    return KINDS[kind]


def _int32(what: str, name: str, t, device, shape=None):
    if t is None:
        return None
    if (t.dtype != torch.int32 or t.device != device or not t.is_contiguous()
            or (shape is not None and tuple(t.shape) != shape)):
        want = "" if shape is None else f" {shape}"
        raise RuntimeError(f"{what}: {name} must be contiguous int32{want} on {device}")
    return t.data_ptr()


def _cache_args(what: str, pool, kind, table, lengths, slots, indptr, total):
    """The arguments that describe a layer's cache and a call's sequences; and B."""
    if not pool.is_cuda:
        raise RuntimeError(f"{what}: kvquant_b200 runs on CUDA tensors only")
    if pool.dtype != torch.uint8 or pool.dim() != 4 or not pool.is_contiguous():
        raise RuntimeError(f"{what}: pool must be contiguous uint8 [pages, heads, blocks, record]")
    n_pages, heads, blocks, rec = pool.shape
    dev = pool.device
    if table.dim() != 2:
        raise RuntimeError(f"{what}: table must be [slots, columns]")
    n_slots, n_cols = table.shape
    if indptr is not None:
        if indptr.dim() != 1:
            raise RuntimeError(f"{what}: indptr must be [sequences + 1]")
        B = indptr.numel() - 1
    else:
        B = n_slots if slots is None else slots.numel()
    head = (pool.data_ptr(), _kind(what, kind), n_pages, heads, (rec - 16) // 32,
            blocks * BLOCK_TOKENS, _int32(what, "table", table, dev), n_slots, n_cols,
            _int32(what, "lengths", lengths, dev, (n_slots,)),
            _int32(what, "slots", slots, dev, (B,)))
    if rec % 32 != 16:
        raise RuntimeError(f"{what}: the pool's records have {rec} bytes, not 32 * D + 16")
    return head, _int32(what, "indptr", indptr, dev), B


def _rows(what: str, name: str, t, heads, dim, device):
    """t [N, heads, dim] with 16-byte rows; copied when its strides do not allow that."""
    if t.dim() != 3 or t.shape[1] != heads or t.shape[2] != dim or t.device != device:
        raise RuntimeError(f"{what}: {name} must be [rows, {heads}, {dim}] on {device}, "
                           f"got {tuple(t.shape)} on {t.device}")
    if t.stride(2) != 1 or t.stride(0) % 8 or t.stride(1) % 8 or t.data_ptr() % 16:
        t = t.contiguous()
        if t.data_ptr() % 16:
            t = t.clone()
    return t


def paged_append(k: torch.Tensor, v: torch.Tensor, pool: torch.Tensor, table: torch.Tensor,
                 lengths: torch.Tensor, kind: str, slots: torch.Tensor | None = None,
                 indptr: torch.Tensor | None = None, max_new: int | None = None) -> None:
    """Writes the new tokens' keys and values [N, heads, D] (fp16 or bf16) into their blocks.

    A block that the call starts gets the scale max|x| / largest code (at least
    2**-32) over its new tokens; a block that is open already keeps the larger of
    its own scale and that, its older codes rounded anew when the scale grew. Codes
    are rounded to nearest even; infinities are stored as the largest code, NaN as 0,
    and neither counts towards the scale. max_new is accepted for symmetry with
    paged_attention and not needed.
    """
    head, ip, B = _cache_args("paged_append", pool, kind, table, lengths, slots, indptr, None)
    heads, dim, dev = head[3], head[4], pool.device
    k = _rows("paged_append", "k", k, heads, dim, dev)
    v = _rows("paged_append", "v", v, heads, dim, dev)
    if k.shape != v.shape or k.dtype != v.dtype or _DTYPES.get(k.dtype, 2) == 2:
        raise RuntimeError("paged_append: k and v must have one shape and be fp16 or bf16")
    lib = get_cuda_ops().lib
    _launch(lib.kvq_paged_append, lib, dev, k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(),
                                    v.stride(0), v.stride(1), _DTYPES[k.dtype], *head, ip, B,
                                    k.shape[0])


def paged_read(pool: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, kind: str,
               starts: torch.Tensor | None, indptr: torch.Tensor | None, total: int,
               slots: torch.Tensor | None = None, dtype: torch.dtype = torch.float16):
    """The values (code * scale) of the tokens [starts[b], starts[b] + rows of b) of each
    sequence: (k, v), both [total, heads, D] in fp16, bf16 or fp32. starts None: from 0."""
    head, ip, B = _cache_args("paged_read", pool, kind, table, lengths, slots, indptr, total)
    if dtype not in _DTYPES:
        raise RuntimeError(f"paged_read: dtype must be fp16, bf16 or fp32, got {dtype}")
    dev = pool.device
    k = torch.empty((int(total), head[3], head[4]), dtype=dtype, device=dev)
    v = torch.empty_like(k)
    lib = get_cuda_ops().lib
    _launch(lib.kvq_paged_read, lib, dev, *head, _int32("paged_read", "starts", starts, dev, (B,)),
                                  ip, B, int(total), k.data_ptr(), v.data_ptr(), _DTYPES[dtype])
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
    max_new: the most rows of any sequence (default: N when indptr is given; a smaller
    bound gives a better split); scale defaults to 1 / sqrt(D).
    """
    head, ip, B = _cache_args("paged_attention", pool, kind, table, lengths, slots, indptr, None)
    heads, dim, dev = head[3], head[4], pool.device
    if q.dim() != 3 or q.shape[1] == 0 or q.shape[1] % heads:
        raise RuntimeError(f"paged_attention: q {tuple(q.shape)} does not match {heads} KV heads")
    N, Hq, _ = q.shape
    q = _rows("paged_attention", "q", q, Hq, dim, dev)
    if _DTYPES.get(q.dtype, 2) == 2:
        raise RuntimeError("paged_attention: q must be fp16 or bf16")
    if out is None:
        out = torch.empty((N, Hq, dim), dtype=q.dtype, device=dev)
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != dev \
            or not out.is_contiguous():
        raise RuntimeError("paged_attention: out must be contiguous, of q's shape and type")
    if ml_out is not None and (ml_out.dtype != torch.float32 or not ml_out.is_contiguous()
                               or ml_out.numel() != N * Hq * 2 or ml_out.device != dev):
        raise RuntimeError("paged_attention: ml_out must be contiguous fp32 [N, Hq, 2]")
    if max_new is None:
        max_new = N if indptr is not None else N // max(1, B)
    lib = get_cuda_ops().lib
    need = lib.kvq_paged_attention_workspace(dim, int(max_new), Hq // heads)
    ws = (workspace or DecodeWorkspace()).get(need, dev)
    _launch(lib.kvq_paged_attention, lib, dev, 
            q.data_ptr(), q.stride(0), q.stride(1), _DTYPES[q.dtype], Hq // heads, *head, ip, B, N,
            int(max_new), 1.0 / math.sqrt(dim) if scale is None else float(scale), int(window),
            out.data_ptr(), _ptr(ml_out), ws.data_ptr(), ws.numel())
    return out


# ---------------------------------------------------------------------------
# Page operations
# ---------------------------------------------------------------------------
NO_PAGES, BAD_SLOT = 1, 2  # bits of `status`


def _meta_args(what: str, table, lengths, refs, page_tokens):
    if not table.is_cuda or table.dim() != 2:
        raise RuntimeError(f"{what}: table must be a CUDA tensor [slots, columns]")
    dev = table.device
    return (_int32(what, "table", table, dev), table.shape[0], table.shape[1],
            _int32(what, "lengths", lengths, dev, (table.shape[0],)),
            _int32(what, "refs", refs, dev), refs.numel(), int(page_tokens))


def _pool_args(what: str, pool):
    """(pointer, layers, bytes between layers, bytes of a page) of a pool [pages, ...] or
    [layers, pages, ...]."""
    if not pool.is_cuda or pool.dtype != torch.uint8 or pool.dim() not in (4, 5):
        raise RuntimeError(f"{what}: pool must be a CUDA uint8 tensor [pages, heads, blocks, "
                           "record] or [layers, pages, heads, blocks, record]")
    if not pool.is_contiguous():
        raise RuntimeError(f"{what}: pool must be contiguous")
    page = pool.shape[-3] * pool.shape[-2] * pool.shape[-1]
    layers = pool.shape[0] if pool.dim() == 5 else 1
    return pool.data_ptr(), layers, pool.shape[-4] * page, page


def paged_free(table, lengths, refs, slots, page_tokens: int, status) -> None:
    """Gives up the pages of the slots (int32): counts down, rows -1, lengths 0. status
    (int32 [1]) gets BAD_SLOT for a slot out of range or named twice, which is skipped."""
    meta = _meta_args("paged_free", table, lengths, refs, page_tokens)
    dev = table.device
    lib = get_cuda_ops().lib
    _launch(lib.kvq_paged_free, lib, dev, *meta, _int32("paged_free", "slots", slots, dev), slots.numel(),
                                  _int32("paged_free", "status", status, dev, (1,)))


def paged_fork(table, lengths, refs, src, dst, page_tokens: int, status) -> None:
    """dst[i] becomes a copy of src[i] that shares all its pages (an open last page too:
    paged_extend gives a writer its own copy). A pair whose dst holds tokens, is a src,
    is named twice or is out of range is skipped and sets BAD_SLOT in status."""
    meta = _meta_args("paged_fork", table, lengths, refs, page_tokens)
    dev = table.device
    lib = get_cuda_ops().lib
    _launch(lib.kvq_paged_fork, lib, dev, *meta, _int32("paged_fork", "src", src, dev),
                                  _int32("paged_fork", "dst", dst, dev, tuple(src.shape)),
                                  src.numel(), _int32("paged_fork", "status", status, dev, (1,)))


def paged_extend(pool, table, lengths, refs, slots, n_new, status,
                 workspace: DecodeWorkspace | None = None) -> None:
    """Room for n_new (int, or int32 per slot) more tokens in every slot; lengths grow.

    Free pages are taken in ascending order, slot after slot. A slot whose last page is
    open and shared gets its own copy of it, in every layer of pool ([layers, ...] or one
    layer's), unless all other holders stand before it in `slots`. When pages run out
    (NO_PAGES in status), or a slot is out of range, named twice or too long for its row
    (BAD_SLOT), nothing changes.
    """
    what = "paged_extend"
    ptr, layers, stride, page = _pool_args(what, pool)
    meta = _meta_args(what, table, lengths, refs, pool.shape[-2] * BLOCK_TOKENS)
    dev = table.device
    if refs.numel() != pool.shape[-4] or pool.device != dev:
        raise RuntimeError(f"{what}: refs must have one entry per page of the pool")
    each = isinstance(n_new, torch.Tensor)
    lib = get_cuda_ops().lib
    ws = (workspace or DecodeWorkspace()).get(lib.kvq_paged_extend_workspace(refs.numel()), dev)
    _launch(lib.kvq_paged_extend, lib, dev, 
            ptr, layers, stride, page, *meta, _int32(what, "slots", slots, dev), slots.numel(),
            _int32(what, "n_new", n_new, dev, tuple(slots.shape)) if each else None,
            0 if each else int(n_new), _int32(what, "status", status, dev, (1,)), ws.data_ptr(),
            ws.numel())


def paged_compact(pool, table, refs, workspace: DecodeWorkspace | None = None,
                  n_live: torch.Tensor | None = None) -> torch.Tensor:
    """Moves the live pages to the lowest ids: those at or past their number, in
    ascending order, into the free ones below it, in every layer; table and refs follow.
    Returns the number of live pages (int32 [1] on the device)."""
    what = "paged_compact"
    ptr, layers, stride, page = _pool_args(what, pool)
    dev = table.device
    if refs.numel() != pool.shape[-4] or pool.device != dev or table.dim() != 2:
        raise RuntimeError(f"{what}: refs must have one entry per page of the pool")
    if n_live is None:
        n_live = torch.empty(1, dtype=torch.int32, device=dev)
    lib = get_cuda_ops().lib
    ws = (workspace or DecodeWorkspace()).get(lib.kvq_paged_extend_workspace(refs.numel()), dev)
    _launch(lib.kvq_paged_compact, lib, dev, 
            ptr, layers, stride, page, _int32(what, "table", table, dev), table.shape[0],
            table.shape[1], _int32(what, "refs", refs, dev), refs.numel(),
            _int32(what, "n_live", n_live, dev, (1,)), ws.data_ptr(), ws.numel())
    return n_live


def paged_copy(src_pool, dst_pool, src, dst, workspace: DecodeWorkspace | None = None) -> None:
    """Copies pages src[i] of src_pool to pages dst[i] of dst_pool (which may be the same
    pool), every layer. dst pages are distinct, and in one pool none of them is in src."""
    what = "paged_copy"
    sp, layers, s_stride, page = _pool_args(what, src_pool)
    dp, d_layers, d_stride, d_page = _pool_args(what, dst_pool)
    dev = src_pool.device
    if layers != d_layers or page != d_page or dst_pool.device != dev:
        raise RuntimeError(f"{what}: the pools differ in layers, page size or device")
    n = src.numel()
    lib = get_cuda_ops().lib
    ws = (workspace or DecodeWorkspace()).get(lib.kvq_paged_copy_workspace(n), dev)
    _launch(lib.kvq_paged_copy, lib, dev, 
            sp, src_pool.shape[-4], s_stride, dp, dst_pool.shape[-4], d_stride, layers, page,
            _int32(what, "src", src, dev), _int32(what, "dst", dst, dev, tuple(src.shape)), n,
            ws.data_ptr(), ws.numel())
