"""Attention for programs that serve a language model, on MI355X: prompts of different lengths without padding, and a cache of
keys and values in pages with the attention of new tokens over it.

* ``flash_attention_varlen``  the dense forward over packed sequences,
* ``paged_attention``         the newest token (or tokens) of every sequence against its cached keys and values,
* ``append_to_cache``         rows of new tokens into the pages,
* ``copy_pages``              pages to other pages (sequences that split, pages moved together).

Lengths, tables, slots and page lists stay on the device: no call waits for the GPU, and a captured graph follows their present
values.  Entries that lead nowhere (a negative slot, a page that the cache does not have) move and read nothing.  The cache
belongs to the caller; these functions allocate outputs and scratch memory only.  Forward only: tensors that require grad raise,
and so do those with a tangent.
"""
from __future__ import annotations

import math

import torch
from torch.autograd import forward_ad

from . import _lib
from .sage_attention._common import DTYPE_CODE, current_stream_ptr, device_guard, require_gpu, split_workspace

__all__ = ["flash_attention_varlen", "paged_attention", "append_to_cache", "copy_pages"]


def _host():
    return _lib._host_module or _lib.host()


def _no_grad(what, *tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise NotImplementedError(f"{what}: forward only (no backward pass is built); call it under torch.no_grad() or on "
                                  "tensors that do not require grad")
    if getattr(forward_ad, "_current_level", 0) >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{what}: tangents of forward-mode differentiation are not carried on")


def _written(*tensors):
    """Autograd's notice of tensors that a kernel has changed in place: a graph that kept one for its backward pass then raises
    instead of using the new contents."""
    torch.autograd.graph.increment_version(tensors)


def _same_device(device, **tensors):
    for name, t in tensors.items():
        require_gpu(t, name)
        if t.device != device:
            raise ValueError(f"{name} is on {t.device}, the other tensors on {device}")


def _int32(t, name, dim):
    if t.dtype != torch.int32:
        raise TypeError(f"{name} must be an int32 tensor")
    if t.dim() != dim:
        raise ValueError(f"{name} must have {dim} dimension(s)")


def _index_list(t, name):
    if t.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{name} must be an int32 or int64 tensor")
    if t.dim() != 1:
        raise ValueError(f"{name} must have one dimension")
    return t.contiguous()


def _strides(t):
    """The strides of a tensor, 0 for a dimension of one entry: what torch keeps there is arbitrary."""
    shape, strides = t.shape, t.stride()
    return [s if n > 1 else 0 for n, s in zip(shape, strides)] if 1 in shape else strides


def _aligned(t):
    """Rows on 16-byte boundaries that run along the last axis (which the kernels read 16 bytes at a time)."""
    e = t.element_size()
    if t.data_ptr() % 16 != 0:
        return False
    if t.is_contiguous() and t.shape[-1] * e % 16 == 0:  # (the common case, decided without walking the strides)
        return True
    s = _strides(t)
    return (s[-1] == 1 or t.shape[-1] == 1) and (t.numel() == 0 or all(x * e % 16 == 0 for x in s[:-1]))


def _rows16(t):
    return t if _aligned(t) else t.clone(memory_format=torch.contiguous_format)


def _no_overlap(t, name):
    if not t.is_contiguous() and any(n > 1 and s == 0 for n, s in zip(t.shape, t.stride())):
        raise ValueError(f"{name}: entries share memory (an expanded tensor) and cannot be written one by one")


def _check_out(out, like):
    if out.shape != like.shape or out.dtype != like.dtype or out.device != like.device:
        raise ValueError("out must have the shape, dtype and device of q")
    if not _aligned(out):
        raise ValueError("out: rows must be 16-byte aligned, with a unit innermost stride")
    _no_overlap(out, "out")


def _check_heads(hq, hkv, hv):
    if hkv != hv:
        raise ValueError("num of heads in k and v should be equal")
    if hkv == 0 or hq == 0 or hq % hkv != 0:
        raise ValueError("number of heads in q must be a positive multiple of that in k & v")


def _check_float16s(q, k, v):
    if q.dtype not in (torch.float16, torch.bfloat16) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError("q, k, v must share one of torch.float16 / torch.bfloat16")


def _token_desc(t):  # [tokens, heads, head_dim]
    s = _strides(t)
    return _lib.SageTensor(t.data_ptr(), 0, s[1], s[0])


def _cache_desc(t, hnd):
    s = _strides(t)
    return _lib.SageTensor(t.data_ptr(), s[0], s[1] if hnd else s[2], s[2] if hnd else s[1])


def _row_desc(t):  # [sequences, heads, head_dim] or [sequences, new tokens, heads, head_dim]
    s = _strides(t)
    return _lib.SageTensor(t.data_ptr(), s[0], s[-2], s[1] if len(s) == 4 else 0)


def _layout(tensor_layout):
    if tensor_layout not in ("HND", "NHD"):
        raise ValueError(f"Unknown tensor layout: {tensor_layout}")
    return tensor_layout == "HND"


def _check_caches(k_cache, v_cache, hnd):
    """(pages, heads_kv, page_size, head_dim)"""
    if k_cache.dim() != 4 or v_cache.dim() != 4:
        raise ValueError("k_cache and v_cache must be (pages, heads, page_size, head_dim) tensors, or (pages, page_size, heads, head_dim) "
                         "with tensor_layout='NHD'")
    if k_cache.shape != v_cache.shape:
        raise ValueError("k_cache and v_cache must have the same shape")
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
        if not _aligned(t):
            raise ValueError(f"{name}: rows must be 16-byte aligned, with a unit innermost stride (a cache is not copied)")
    p, a, b, d = k_cache.shape
    return (p, a, b, d) if hnd else (p, b, a, d)


def flash_attention_varlen(q, k, v, cu_seqlens_q, cu_seqlens_k=None, causal=False, sm_scale=None, return_log_normalizer=False,
                           *, out=None):
    """The dense forward of ``flash_attention`` over packed sequences of different lengths.

    ``q`` ``[total_q, H, D]``, ``k`` and ``v`` ``[total_k, Hk, D]`` (fp16 / bf16, any strides with a unit innermost one): the tokens of
    all sequences, one after the other.  ``cu_seqlens_q`` / ``cu_seqlens_k`` (int32, on the GPU, one entry more than there are
    sequences; ``cu_seqlens_k`` defaults to ``cu_seqlens_q``): where each sequence begins, and where the last one ends.  Every
    sequence attends to itself only; ``causal`` is bottom-right aligned per sequence (query i sees the keys j <= i + Lk - Lq), so a
    sequence with more keys than queries is a chunk of a longer prompt.  Queries that see no key get a zero row.  Lengths of
    0 are fine.

    Returns ``o`` ``[total_q, H, D]``, or ``(o, log_normalizer)`` with the natural log-sum-exp ``[H, total_q]`` in fp32 (-inf where no
    key is seen).  ``out``: where to write instead of a new tensor.  Rows behind the last sequence are not written: those of
    ``out`` stay as they were, those of a new tensor and of the log normalizer are undefined.  The softmax's weights are rounded to
    16 bits before they multiply V, as in ``flash_attention``; maxima and sums are fp32.
    """
    if cu_seqlens_k is None:
        cu_seqlens_k = cu_seqlens_q
    call = (q, k, v, cu_seqlens_q, cu_seqlens_k, causal, sm_scale, return_log_normalizer)
    if out is None:
        res = _host().varlen(*call)  # a call shape seen before: (o, log normalizer), or a status
        if res is not None:
            if type(res) is int:
                _lib.check(res, "sage_flash_varlen_fwd")
            return res if return_log_normalizer else res[0]
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
        raise ValueError("q, k, v must be (tokens, heads, head_dim) tensors")
    T, H, D = q.shape
    Tk, Hk, Dk = k.shape
    if Dk != D or v.shape[2] != D:
        raise ValueError("feature size of q, k, v should be equal")
    _check_heads(H, Hk, v.shape[1])
    if v.shape[0] != Tk:
        raise ValueError("k and v must have the same number of tokens")
    if D not in (16, 32, 64, 128):
        raise NotImplementedError(f"flash_attention_varlen: head_dim {D} is not built (16, 32, 64 or 128)")
    _check_float16s(q, k, v)
    _int32(cu_seqlens_q, "cu_seqlens_q", 1)
    _int32(cu_seqlens_k, "cu_seqlens_k", 1)
    if cu_seqlens_q.numel() != cu_seqlens_k.numel() or cu_seqlens_q.numel() == 0:
        raise ValueError("cu_seqlens_q and cu_seqlens_k must have one entry more than there are sequences")
    _no_grad("flash_attention_varlen", q, k, v, out)
    _same_device(q.device, q=q, k=k, v=v, cu_seqlens_q=cu_seqlens_q, cu_seqlens_k=cu_seqlens_k)
    if out is not None:
        _check_out(out, q)
    sm_scale = 1.0 / math.sqrt(D) if sm_scale is None else float(sm_scale)

    with device_guard(q.device):
        cu_seqlens_q, cu_seqlens_k = cu_seqlens_q.contiguous(), cu_seqlens_k.contiguous()
        o = out
        if D < 64:  # zero channels change neither Q K^T nor the first D columns of P V
            q, k, v = (torch.nn.functional.pad(t, (0, 64 - D)) for t in (q, k, v))
            o = torch.empty_like(q) if out is None else torch.nn.functional.pad(out, (0, 64 - D))
        q, k, v = _rows16(q), _rows16(k), _rows16(v)
        if o is None:
            o = torch.empty((T, H, D), dtype=q.dtype, device=q.device)
        L = torch.empty((H, T), dtype=torch.float32, device=q.device) if return_log_normalizer else None
        p = _lib.VarlenParams()
        p.q, p.k, p.v, p.out = (_token_desc(t) for t in (q, k, v, o))
        p.log_normalizer = L.data_ptr() if L is not None else None
        p.cu_seqlens_q, p.cu_seqlens_k = cu_seqlens_q.data_ptr(), cu_seqlens_k.data_ptr()
        p.seqs, p.total_q, p.total_k = cu_seqlens_q.numel() - 1, T, Tk
        p.heads_q, p.heads_kv, p.head_dim = H, Hk, max(D, 64)
        p.dtype, p.causal, p.sm_scale = DTYPE_CODE[q.dtype], 1 if causal else 0, sm_scale
        lib = _lib.load()
        ws_bytes = lib.sage_flash_varlen_workspace_bytes(p)
        if ws_bytes < 0:
            _lib.check(-1, "sage_flash_varlen_workspace_bytes")
        if out is None and all(x is y for x, y in zip((q, k, v, cu_seqlens_q, cu_seqlens_k), call)):  # (nothing was copied)
            _host().put_varlen(*call, bytes(p), ws_bytes)
        ws = split_workspace(q.device, ws_bytes) if ws_bytes else None
        _lib.check(lib.sage_flash_varlen_fwd(p, ws.data_ptr() if ws is not None else None, ws_bytes, current_stream_ptr(q.device)),
                   "sage_flash_varlen_fwd")
        if D < 64:
            o = o[..., :D].contiguous() if out is None else out.copy_(o[..., :D])
        elif out is not None:
            _written(out)
    return (o, L) if return_log_normalizer else o


def paged_attention(q, k_cache, v_cache, block_table, seq_lens, sm_scale=None, tensor_layout="HND", return_log_normalizer=False,
                    *, out=None):
    """Attention of the newest token of every sequence over a cache of keys and values in pages.

    ``q`` ``[S, H, D]``, or ``[S, M, H, D]`` for the M newest tokens of every sequence (fp16 / bf16).  ``k_cache``, ``v_cache``
    ``[pages, Hk, page_size, D]`` ("HND") or ``[pages, page_size, Hk, D]`` ("NHD"), any strides with a unit innermost one and 16-byte
    aligned rows, any page size; head_dim 64 or 128.  ``block_table`` ``[S, width]`` int32: the pages of every sequence in order.
    ``seq_lens`` ``[S]`` int32: tokens of every sequence in the cache, the new ones among them (write those with
    ``append_to_cache`` first).  Of M new tokens, token m sees the keys up to ``seq_lens - M + m``.  A sequence of length 0 (a slot
    that is not in use) gets zero rows; table entries that are no page of the cache hide their tokens; lengths beyond the table are
    cut to it, to 0 where it has no entries or the cache no pages.

    Returns ``o`` in the shape of ``q``, or ``(o, log_normalizer)`` with the natural log-sum-exp ``[S, H]`` (``[S, H, M]``) in fp32.
    ``out``: where to write instead of a new tensor.  Roundings as in ``flash_attention_varlen``.
    """
    call = (q, k_cache, v_cache, block_table, seq_lens, sm_scale, tensor_layout, return_log_normalizer)
    if out is None:
        res = _host().paged(*call)  # a call shape seen before: (o, log normalizer), or a status
        if res is not None:
            if type(res) is int:
                _lib.check(res, "sage_paged_attn")
            return res if return_log_normalizer else res[0]
    hnd = _layout(tensor_layout)
    if q.dim() not in (3, 4):
        raise ValueError("q must be (sequences, heads, head_dim) or (sequences, new tokens, heads, head_dim)")
    S, H, D = q.shape[0], q.shape[-2], q.shape[-1]
    M = q.shape[1] if q.dim() == 4 else 1
    pages, Hk, page_size, Dk = _check_caches(k_cache, v_cache, hnd)
    if Dk != D:
        raise ValueError("feature size of q and the caches should be equal")
    _check_heads(H, Hk, Hk)
    if D not in (64, 128):
        raise NotImplementedError(f"paged_attention: head_dim {D} is not built (64 or 128)")
    _check_float16s(q, k_cache, v_cache)
    _int32(block_table, "block_table", 2)
    _int32(seq_lens, "seq_lens", 1)
    if block_table.shape[0] != S or seq_lens.shape[0] != S:
        raise ValueError("block_table and seq_lens must have a row for every sequence of q")
    _no_grad("paged_attention", q, k_cache, v_cache, out)
    _same_device(q.device, q=q, k_cache=k_cache, v_cache=v_cache, block_table=block_table, seq_lens=seq_lens)
    if out is not None:
        _check_out(out, q)
    sm_scale = 1.0 / math.sqrt(D) if sm_scale is None else float(sm_scale)

    with device_guard(q.device):
        q = _rows16(q)
        o = torch.empty(q.shape, dtype=q.dtype, device=q.device) if out is None else out
        if block_table.stride(1) != 1 or block_table.stride(0) < 0:
            block_table = block_table.contiguous()
        seq_lens = seq_lens.contiguous()
        L = None
        if return_log_normalizer:
            L = torch.empty((S, H) if q.dim() == 3 else (S, H, M), dtype=torch.float32, device=q.device)
        if page_size > 0 and (pages == 0 or block_table.shape[1] == 0):  # (no place for a key)
            o.fill_(0)
            return (o, L.fill_(-math.inf)) if return_log_normalizer else o
        p = _lib.PagedParams()
        p.q, p.out = _row_desc(q), _row_desc(o)
        p.k_cache, p.v_cache = _cache_desc(k_cache, hnd), _cache_desc(v_cache, hnd)
        p.log_normalizer = L.data_ptr() if L is not None else None
        p.block_table, p.seq_lens = block_table.data_ptr(), seq_lens.data_ptr()
        p.table_stride, p.table_width = block_table.stride(0), block_table.shape[1]
        p.seqs, p.new_tokens, p.heads_q, p.heads_kv, p.head_dim = S, M, H, Hk, D
        p.pages, p.page_size, p.dtype, p.sm_scale = pages, page_size, DTYPE_CODE[q.dtype], sm_scale
        lib = _lib.load()
        ws_bytes = lib.sage_paged_attn_workspace_bytes(p)
        if ws_bytes < 0:
            _lib.check(-1, "sage_paged_attn_workspace_bytes")
        if out is None and q is call[0] and block_table is call[3] and seq_lens is call[4]:  # (nothing was copied)
            _host().put_paged(*call, bytes(p), ws_bytes)
        ws = split_workspace(q.device, ws_bytes) if ws_bytes else None
        _lib.check(lib.sage_paged_attn(p, ws.data_ptr() if ws is not None else None, ws_bytes, current_stream_ptr(q.device)),
                   "sage_paged_attn")
        if out is not None:
            _written(out)
    return (o, L) if return_log_normalizer else o


def append_to_cache(k, v, k_cache, v_cache, slots, tensor_layout="HND"):
    """Writes the keys and values of new tokens into the pages of a cache, in place.

    ``k``, ``v`` ``[tokens, Hk, D]`` (any strides), caches as for ``paged_attention`` (fp16, bf16 or fp32, one dtype; rows of a multiple of 16
    bytes).  ``slots`` ``[tokens]`` (int32 or int64, on the GPU): token t goes to place ``slots[t] % page_size`` of page
    ``slots[t] // page_size``.  Tokens whose slot the cache does not have are left out: -1 for the rows a batch is padded with.
    The other slots of a call have to differ.
    """
    call = (k, v, k_cache, v_cache, slots, tensor_layout)
    status = _host().append(*call)  # a call shape seen before
    if status is not None:
        return _lib.check(status, "sage_cache_append")
    hnd = _layout(tensor_layout)
    if k.dim() != 3 or k.shape != v.shape:
        raise ValueError("k and v must be (tokens, heads, head_dim) tensors of the same shape")
    pages, Hk, page_size, D = _check_caches(k_cache, v_cache, hnd)
    if k.shape[1:] != (Hk, D):
        raise ValueError("heads and head_dim of k, v and the caches should be equal")
    if k.dtype not in DTYPE_CODE or any(t.dtype != k.dtype for t in (v, k_cache, v_cache)):
        raise TypeError("k, v and the caches must share one of torch.float16 / torch.bfloat16 / torch.float32")
    _no_overlap(k_cache, "k_cache")
    _no_overlap(v_cache, "v_cache")
    slots = _index_list(slots, "slots")
    if slots.shape[0] != k.shape[0]:
        raise ValueError("slots must have an entry for every token")
    _no_grad("append_to_cache", k, v, k_cache, v_cache)
    _same_device(k.device, k=k, v=v, k_cache=k_cache, v_cache=v_cache, slots=slots)
    with device_guard(k.device):
        k, v = _rows16(k), _rows16(v)
        p = _lib.AppendParams()
        p.k, p.v = _token_desc(k), _token_desc(v)
        p.k_cache, p.v_cache = _cache_desc(k_cache, hnd), _cache_desc(v_cache, hnd)
        p.slots, p.slots_int64 = slots.data_ptr(), 1 if slots.dtype == torch.int64 else 0
        p.tokens, p.heads_kv, p.head_dim, p.pages, p.page_size = k.shape[0], Hk, D, pages, page_size
        p.dtype = DTYPE_CODE[k.dtype]
        if k is call[0] and v is call[1] and slots is call[4]:  # (nothing was copied)
            _host().put_append(*call, bytes(p))
        _lib.check(_lib.load().sage_cache_append(p, current_stream_ptr(k.device)), "sage_cache_append")
        _written(k_cache, v_cache)


def _page_bytes(t):
    """Bytes of a page (all dimensions but the first) that lies in one piece, whatever the order of its dimensions."""
    size = 1
    for n, s in sorted(zip(t.shape[1:], t.stride()[1:]), key=lambda x: x[1]):
        if n == 1:
            continue
        if s != size:
            return None
        size *= n
    return size * t.element_size()


def copy_pages(k_cache, v_cache, src, dst):
    """Copies pages of a cache, keys and values, in place: page ``src[i]`` to page ``dst[i]``.

    ``k_cache``, ``v_cache`` ``[pages, ...]`` (four dimensions), or ``[layers, pages, ...]`` (five): the pages of all layers in one launch.
    Each page lies in one piece of a multiple of 16 bytes.  ``src``, ``dst`` ``[count]`` (int32 or int64, on the GPU); pairs with a page that the
    cache does not have are left out.  Pages that are written must differ from each other and from every page that is read: that is
    so where sequences split (the last page of each goes to a new one) and where pages in use move to unused ones.
    """
    call = (k_cache, v_cache, src, dst)
    status = _host().copy(*call)  # a call shape seen before
    if status is not None:
        return _lib.check(status, "sage_cache_copy_pages")
    if k_cache.dim() not in (4, 5) or k_cache.shape != v_cache.shape or k_cache.dtype != v_cache.dtype:
        raise ValueError("k_cache and v_cache must be (pages, ...) or (layers, pages, ...) tensors of the same shape and dtype")
    src, dst = _index_list(src, "src"), _index_list(dst, "dst")
    if src.shape != dst.shape:
        raise ValueError("src and dst must have the same number of pages")
    _no_grad("copy_pages", k_cache, v_cache)
    _same_device(k_cache.device, k_cache=k_cache, v_cache=v_cache, src=src, dst=dst)
    layered = k_cache.dim() == 5
    p = _lib.CopyParams()
    p.layers, p.pages, p.count = k_cache.shape[0] if layered else 1, k_cache.shape[1 if layered else 0], src.shape[0]
    if k_cache.numel() == 0 or p.count == 0:
        return
    e = k_cache.element_size()
    for t in (k_cache, v_cache):
        nbytes = _page_bytes(t[0] if layered else t)
        if nbytes is None:
            raise ValueError("a page of k_cache or v_cache does not lie in one piece of memory")
        p.page_bytes = nbytes
    for name, t in (("k", k_cache), ("v", v_cache)):
        if p.pages > 1 and t.stride(1 if layered else 0) * e < p.page_bytes:
            raise ValueError(f"{name}_cache: pages overlap")
        _no_overlap(t, f"{name}_cache")
        setattr(p, f"{name}_cache", t.data_ptr())
        strides = _strides(t)
        setattr(p, f"{name}_stride_layer", strides[0] * e if layered else 0)
        setattr(p, f"{name}_stride_page", strides[1 if layered else 0] * e)
    p.src, p.src_int64 = src.data_ptr(), 1 if src.dtype == torch.int64 else 0
    p.dst, p.dst_int64 = dst.data_ptr(), 1 if dst.dtype == torch.int64 else 0
    if src is call[2] and dst is call[3]:  # (nothing was copied)
        _host().put_copy(*call, bytes(p))
    with device_guard(k_cache.device):
        _lib.check(_lib.load().sage_cache_copy_pages(p, current_stream_ptr(k_cache.device)), "sage_cache_copy_pages")
        _written(k_cache, v_cache)
