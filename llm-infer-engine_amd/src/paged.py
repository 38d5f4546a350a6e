"""Paged KV cache, the append to it and the attention over it.

The dense ``KVCache`` (src/kv_cache.py) reserves max_batch_size x max_seq_len
slots and appends every row at one position.  ``PagedKVCache`` holds pages of
``page_size`` tokens that any sequence may use; a page table [batch, slots]
(int32, on the device) names each row's pages, and every row has its own length:

  rope_and_paged_update   RoPE of q and k at each row's own positions, and the
                          append of k and v (mi_rope_paged_append, one launch)
  paged_flash_attention   causal attention of a row's newest tokens, one or many,
                          over all its keys (mi_paged_attn)

Pages hold the activations' dtype or, with ``kv_dtype=torch.float8_e4m3fn``, 8-bit
floats with a power-of-two scale for each page, KV head and K / V.  V pages are
transposed ([head_dim, page_size]): the attention's matrix instructions take V in
that order straight from memory.

Everything that varies while serving (lengths, counts, the table) is read on the
device, so a captured step stays valid for other values of them.  A table entry
that is no page of the cache takes no write and gives no key.  The paged cache has
no counterpart in the reference, whose cache is dense (src/kv_cache.py:4-57).
"""
from __future__ import annotations

import math

import torch

from . import _lib
from .config import ModelArgs

PAGE_SIZES = (16, 32, 64, 128, 256)


class PagedKVCache:
    """k [n_layers, num_pages, n_kv_heads, page_size, head_dim], v [n_layers,
    num_pages, n_kv_heads, head_dim, page_size] and, for 8-bit pages, scales
    [n_layers, num_pages, n_kv_heads, 2] (fp32; of K and V)."""

    def __init__(self, args: ModelArgs, num_pages: int, page_size: int = 64,
                 dtype: torch.dtype | None = None, *, kv_dtype: torch.dtype | None = None):
        dtype = dtype if dtype is not None else torch.get_default_dtype()
        kv_dtype = kv_dtype if kv_dtype is not None else dtype
        d = args.dim // args.n_heads
        shape = (args.n_layers, num_pages, args.n_kv_heads)
        _check_pages(dtype, kv_dtype, num_pages, page_size, d)
        k = torch.zeros((*shape, page_size, d), device=args.device, dtype=kv_dtype)
        v = torch.zeros((*shape, d, page_size), device=args.device, dtype=kv_dtype)
        scales = None
        if kv_dtype != dtype:
            scales = torch.zeros((*shape, 2), device=args.device, dtype=torch.float32)
        self._set(k, v, scales, dtype)

    @classmethod
    def from_pages(cls, k: torch.Tensor, v: torch.Tensor, scales: torch.Tensor | None = None, *,
                   dtype: torch.dtype | None = None) -> "PagedKVCache":
        """A cache over existing pages (not copied): k [n_layers, num_pages, n_kv_heads,
        page_size, head_dim] or one layer's [num_pages, ..], v the same transposed, scales
        for 8-bit pages (powers of two, as the append leaves them); ``dtype`` is the
        activations' (default: k's)."""
        dtype = dtype if dtype is not None else k.dtype
        if k.dim() == 4:
            k, v = k[None], v[None] if v.dim() == 4 else v
            scales = scales[None] if scales is not None and scales.dim() == 3 else scales
        if k.dim() != 5 or v.shape != (*k.shape[:3], k.shape[4], k.shape[3]):
            raise ValueError(f"PagedKVCache: k pages {tuple(k.shape)} and transposed v pages "
                             f"{tuple(v.shape)} do not match")
        if v.dtype != k.dtype or v.device != k.device:
            raise TypeError("PagedKVCache: k and v must share a dtype and a device")
        _check_pages(dtype, k.dtype, k.shape[1], k.shape[3], k.shape[4])
        if (scales is None) != (k.dtype == dtype):
            raise ValueError("PagedKVCache: 8-bit pages, and only they, have scales")
        if scales is not None and (scales.shape != (*k.shape[:3], 2)
                                   or scales.dtype != torch.float32
                                   or scales.device != k.device):
            raise ValueError(f"PagedKVCache: scales must be fp32 {(*k.shape[:3], 2)} on {k.device}")
        for t in (k, v, scales):
            if t is not None and not t.is_contiguous():
                raise ValueError("PagedKVCache: pages and scales must be contiguous")
        self = cls.__new__(cls)
        self._set(k, v, scales, dtype)
        return self

    def _set(self, k, v, scales, dtype):
        self.k, self.v, self.scales, self.dtype = k, v, scales, dtype
        self.n_layers, self.num_pages, self.n_kv_heads, self.page_size, self.head_dim = k.shape
        self.kv_dtype = k.dtype
        self.store = _lib.MI_STORE_SAME if scales is None else _lib.MI_STORE_E4M3
        self._code = _lib.dtype_code(dtype)
        self._layer_bytes = k.stride(0) * k.element_size()

    def reset(self):
        """Empty pages (zeros).  Not needed before a page is used again: its first
        append starts it anew."""
        self.k.zero_()
        self.v.zero_()
        if self.scales is not None:
            self.scales.zero_()

    def _layer(self, layer_idx: int, what: str):
        """Addresses of a layer's k, v and scales."""
        n = self.n_layers
        if not -n <= layer_idx < n:
            raise ValueError(f"{what}: layer_idx {layer_idx} out of range for a cache of {n} layers")
        i, s = layer_idx % n, self.scales
        at = i * self._layer_bytes
        return (self.k.data_ptr() + at, self.v.data_ptr() + at,
                None if s is None else s.data_ptr() + 8 * i * self.num_pages * self.n_kv_heads)


def _check_pages(dtype, kv_dtype, num_pages, page_size, head_dim):
    if dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise TypeError(f"PagedKVCache: unsupported dtype {dtype}; expected bfloat16, float16 or "
                        "float32")
    if kv_dtype not in (dtype, torch.float8_e4m3fn):
        raise TypeError(f"PagedKVCache: pages hold {dtype} or float8_e4m3fn, not {kv_dtype}")
    if page_size not in PAGE_SIZES:
        raise ValueError(f"PagedKVCache: page_size must be one of {PAGE_SIZES}, got {page_size}")
    if num_pages < 1:
        raise ValueError(f"PagedKVCache: num_pages must be positive, got {num_pages}")
    if head_dim % 2 != 0 or not 2 <= head_dim <= 256:
        raise ValueError(f"PagedKVCache: head_dim must be even and at most 256, got {head_dim}")


_I32, _I64, _F32 = torch.int32, torch.int64, torch.float32


def _per_row(t, batch: int, index: int, name: str, what: str):
    """A device int64 [batch] tensor of row lengths or positions (None stays None)."""
    if t is None:
        return None
    if t.shape != (batch,):
        raise ValueError(f"{what}: {name} must have shape ({batch},), got {tuple(t.shape)}")
    if t.dtype is _I64 and t.get_device() == index and t.stride() == (1,):
        return t
    if t.is_floating_point() or t.dtype == torch.bool:
        raise TypeError(f"{what}: {name} must hold integers, got {t.dtype}")
    device = torch.device("cpu") if index < 0 else torch.device("cuda", index)
    return t.to(device=device, dtype=torch.int64).contiguous()


def _table(page_table, batch: int, index: int, what: str):
    shape = page_table.shape
    if len(shape) != 2 or shape[0] != batch or shape[1] < 1:
        raise ValueError(f"{what}: page_table must have shape ({batch}, slots), got {tuple(shape)}")
    if page_table.dtype is not _I32:
        raise TypeError(f"{what}: page_table must have dtype torch.int32, got {page_table.dtype}")
    if page_table.get_device() != index:
        raise ValueError(f"{what}: page_table must be on device {index}, got {page_table.device}")
    stride = page_table.stride()
    if stride[1] != 1:
        page_table = page_table.contiguous()
        stride = page_table.stride()
    return page_table, shape[1], stride[0]


def _device_of(what: str, *tensors) -> int:
    """The index of the one CUDA device that all of them are on."""
    index = tensors[0].get_device()
    for t in tensors:
        if t.get_device() != index or index < 0:
            break
    else:
        return index
    if not all(x.is_cuda for x in tensors):
        raise ValueError(f"{what} requires CUDA tensors")
    raise ValueError(f"{what}: all tensors must be on one device, got "
                     f"{', '.join(sorted({str(x.device) for x in tensors}))}")


def _check_heads(H, dtype, cache, what):
    if H % cache.n_kv_heads != 0:
        raise ValueError(f"query heads ({H}) must be divisible by KV heads ({cache.n_kv_heads})")
    if dtype is not cache.dtype:
        raise TypeError(f"{what}: q dtype {dtype} must match the cache's activations {cache.dtype}")


def rope_and_paged_update(xk, xv, rope_cos, rope_sin, cache: PagedKVCache, layer_idx: int,
                          page_table, start_pos, *, query_lens=None, xq=None):
    """RoPE of xk (and xq) and the append of xk, xv to the rows' pages.

    xk, xv: [B, n_kv_heads, S, head_dim]; xq [B, n_heads, S, head_dim] or None.
    Token s of row b is at position start_pos[b] + s (start_pos: device int64 [B],
    or an int for all rows) and takes that row of the full tables rope_cos /
    rope_sin [positions, head_dim // 2] (in xk's dtype or fp32; the nearest row
    outside them).  With ``query_lens`` (device int64 [B]) only a row's first
    query_lens[b] tokens are appended.  Positions behind the table's slots, before 0 or
    in slots without a page are not written.  Rows may share pages that they only read;
    a page that two rows append to holds undefined entries.

    Returns the rotated xq (with xq's strides), or None.
    """
    what = "rope_and_paged_update"
    shape, dtype = xk.shape, xk.dtype
    if len(shape) != 4 or xv.shape != shape:
        raise ValueError(f"xk and xv shapes must match, got {tuple(shape)} and {tuple(xv.shape)}")
    B, Hkv, S, D = shape
    if Hkv != cache.n_kv_heads or D != cache.head_dim:
        raise ValueError(f"xk/xv shape {tuple(shape)} does not fit a cache of {cache.n_kv_heads} "
                         f"heads of {cache.head_dim}")
    if dtype is not cache.dtype or xv.dtype is not dtype:
        raise TypeError(f"xk/xv dtype {dtype} must match the cache's activations {cache.dtype}")
    H = Hkv
    if xq is not None:
        q_shape = xq.shape
        if len(q_shape) != 4 or q_shape[0] != B or q_shape[2] != S or q_shape[3] != D:
            raise ValueError(f"xq shape {tuple(q_shape)} does not match xk {tuple(shape)}")
        H = q_shape[1]
        _check_heads(H, xq.dtype, cache, what)
    t_shape, t_dtype = rope_cos.shape, rope_cos.dtype
    if len(t_shape) != 2 or rope_sin.shape != t_shape or 2 * t_shape[1] < D:
        raise ValueError(f"{what}: cos/sin must be 2-D [positions, head_dim // 2 = {D // 2}], got "
                         f"{tuple(t_shape)} and {tuple(rope_sin.shape)}")
    if rope_sin.dtype is not t_dtype or (t_dtype is not dtype and t_dtype is not _F32):
        raise TypeError(f"{what}: cos/sin must have dtype {dtype} or float32, got {t_dtype} and "
                        f"{rope_sin.dtype}")
    kp, vp, sp = cache._layer(layer_idx, what)
    index = _device_of(what, xk, xv, rope_cos, rope_sin, cache.k, xk if xq is None else xq)
    page_table, slots, pt_stride = _table(page_table, B, index, what)
    first, start = 0, None
    if isinstance(start_pos, torch.Tensor):
        start = _per_row(start_pos, B, index, "start_pos", what)
    else:
        first = int(start_pos)
    lens = _per_row(query_lens, B, index, "query_lens", what)
    ks, vs, cs, ss = xk.stride(), xv.stride(), rope_cos.stride(), rope_sin.stride()
    if ks[3] != 1:
        xk = xk.contiguous()
        ks = xk.stride()
    if vs[3] != 1:
        xv = xv.contiguous()
        vs = xv.stride()
    if cs[1] != 1 or ss[1] != 1:
        rope_cos, rope_sin = rope_cos.contiguous(), rope_sin.contiguous()
        cs, ss = rope_cos.stride(), rope_sin.stride()
    out = dst = q_ptr = o_ptr = None
    qs = os_ = (0, 0, 0, 1)
    if xq is not None:
        out = dst = torch.empty_like(xq)
        qs, os_ = xq.stride(), out.stride()
        if qs[3] != 1:
            xq = xq.contiguous()
            qs = xq.stride()
        if os_[3] != 1:
            dst = torch.empty(q_shape, dtype=dtype, device=out.device)
            os_ = dst.stride()
        q_ptr, o_ptr = xq.data_ptr(), dst.data_ptr()
    if B == 0 or S == 0:
        return out
    with _lib.on_device(index):
        st = _lib.load().mi_rope_paged_append(
            q_ptr, xk.data_ptr(), xv.data_ptr(), rope_cos.data_ptr(), rope_sin.data_ptr(), o_ptr,
            kp, vp, sp, page_table.data_ptr(), first, None if start is None else start.data_ptr(),
            None if lens is None else lens.data_ptr(),
            t_shape[0], B, H, Hkv, S, D, cache.num_pages, cache.page_size, slots,
            qs[0], qs[1], qs[2], ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], os_[0], os_[1], os_[2],
            pt_stride, cs[0], ss[0], cache._code, _lib.dtype_code(t_dtype), cache.store,
            torch._C._cuda_getCurrentRawStream(index))
    if st:
        _lib.check(st, what)
    if dst is not out:
        out.copy_(dst)
    return out


def paged_flash_attention(q, cache: PagedKVCache, layer_idx: int, page_table, seq_lens, *,
                          query_lens=None, num_splits: int | None = None,
                          return_lse: bool = False, sm_scale: float | None = None):
    """Causal attention of each row's newest tokens over the row's pages.

    q: [B, n_heads, S, head_dim]; seq_lens (device int64 [B]) counts the row's keys,
    those of its query tokens (already appended) among them.  The first
    query_lens[b] of the S tokens (default: all) are row b's newest: token s sees
    keys j < seq_lens[b] - query_lens[b] + s + 1.  Tokens behind query_lens[b], and a
    token that sees no key, give 0.  out has q's strides; with ``return_lse`` also
    the fp32 log-sum-exp [B, n_heads, S] of the scaled scores (-inf for those).
    ``num_splits``: into how many parts a KV head's keys, those of all rows together, are
    divided (default: chosen from the CU count; 1: no row is divided).
    """
    what = "paged_flash_attention"
    shape = q.shape
    if len(shape) != 4:
        raise ValueError("q must be a rank-4 tensor")
    B, H, S, D = shape
    if D != cache.head_dim:
        raise ValueError(f"q head_dim {D} does not fit a cache of head_dim {cache.head_dim}")
    _check_heads(H, q.dtype, cache, what)
    kp, vp, sp = cache._layer(layer_idx, what)
    index = _device_of(what, q, cache.k)
    page_table, slots, pt_stride = _table(page_table, B, index, what)
    if seq_lens is None:
        raise ValueError(f"{what}: seq_lens must be given")
    seq_lens = _per_row(seq_lens, B, index, "seq_lens", what)
    lens = _per_row(query_lens, B, index, "query_lens", what)
    if num_splits is not None and not 1 <= int(num_splits) <= _lib.MI_PAGED_ATTN_MAX_SPLITS:
        raise ValueError(f"num_splits must be 1..{_lib.MI_PAGED_ATTN_MAX_SPLITS}, got {num_splits}")
    scale = 1.0 / math.sqrt(D) if sm_scale is None else float(sm_scale)
    if not 0.0 < scale < math.inf:
        raise ValueError(f"{what}: sm_scale must be positive and finite, got {sm_scale}")
    out = dst = torch.empty_like(q)
    lse = q.new_empty((B, H, S), dtype=_F32) if return_lse else None
    if B == 0 or S == 0:
        return (out, lse) if return_lse else out
    qs, os_ = q.stride(), out.stride()
    if qs[3] != 1:
        q = q.contiguous()
        qs = q.stride()
    if os_[3] != 1:
        dst = torch.empty(shape, dtype=q.dtype, device=q.device)
        os_ = dst.stride()
    lib, code, Hkv = _lib.load(), cache._code, cache.n_kv_heads
    with _lib.on_device(index):
        if num_splits is None:
            num_splits = lib.mi_paged_attn_splits(B, H, Hkv, S, D, cache.page_size, slots, code,
                                                  cache.store)
        num_splits = int(num_splits)
        part, n = None, 0
        if num_splits > 1:
            n = lib.mi_paged_attn_workspace(B, H, Hkv, S, D, num_splits, code)
            part = q.new_empty((n,), dtype=_F32)
        st = lib.mi_paged_attn(
            q.data_ptr(), kp, vp, sp, page_table.data_ptr(), seq_lens.data_ptr(),
            None if lens is None else lens.data_ptr(), None if part is None else part.data_ptr(),
            n, dst.data_ptr(), None if lse is None else lse.data_ptr(), B, H, Hkv, S, D,
            cache.num_pages, cache.page_size, slots, num_splits, qs[0], qs[1], qs[2],
            os_[0], os_[1], os_[2], pt_stride, scale, code, cache.store,
            torch._C._cuda_getCurrentRawStream(index))
    if st:
        _lib.check(st, what)
    if dst is not out:
        out.copy_(dst)
    return (out, lse) if return_lse else out
