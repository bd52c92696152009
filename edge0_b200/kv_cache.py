"""The paged cache of keys and values of one attention layer and the calls on it: rows are quantised as they are written
(b200moe_kv_write), can be read back (b200moe_kv_read) and are attended over (b200moe_attention).

With Context.rope in front and MoeLayer.forward behind, these are the device side of a decoder layer's attention half (reference:
edge0-infer/src/models/edge0_35b/forward.cpp:174-214).  Tensors are torch CUDA tensors used as device memory; all arithmetic happens in
libedge0_b200.so.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

import torch

from .capi import KV_BF16, KV_Q4, KV_Q8, Attn, KvCacheDesc
from .moe import Context, _ptr, _x_type, int32_on, rows_view

KIND_BY_NAME = {"bf16": KV_BF16, "q8": KV_Q8, "q4": KV_Q4}


class KvCache:
    """n_pages pages of page_size positions.  kind: "bf16", "q8" (8 bits, a scale a row) or "q4" (4 bits, a scale to 32 values).  Which page
    belongs to which sequence is the caller's affair: calls name slots (page * page_size + place) and tables of pages."""

    def __init__(self, ctx: Context, *, kind: str, n_pages: int, page_size: int, n_head_kv: int, head_dim: int):
        if kind not in KIND_BY_NAME:
            raise ValueError(f"kind must be one of {', '.join(KIND_BY_NAME)}")
        self.ctx, self.kind = ctx, kind
        self.n_pages, self.page_size, self.n_head_kv, self.head_dim = n_pages, page_size, n_head_kv, head_dim
        self.desc = KvCacheDesc(type=KIND_BY_NAME[kind], n_head_kv=n_head_kv, head_dim=head_dim, page_size=page_size, n_pages=n_pages)
        values, scales = C.c_int64(), C.c_int64()
        rc = ctx.lib.b200moe_kv_cache_bytes(C.byref(self.desc), C.byref(values), C.byref(scales))
        if rc:
            raise ValueError(f"no cache of {n_pages} pages of {page_size} x {n_head_kv} heads x {head_dim}: {ctx.lib.b200moe_status_string(rc).decode()}")
        self.device = torch.device("cuda", ctx.device)
        self.k, self.v = (torch.zeros(values.value, dtype=torch.uint8, device=self.device) for _ in range(2))
        self.k_scale, self.v_scale = (torch.zeros(scales.value, dtype=torch.uint8, device=self.device) if scales.value else None for _ in range(2))
        for name in ("k", "v", "k_scale", "v_scale"):
            t = getattr(self, name)
            setattr(self.desc, name, None if t is None else t.data_ptr())

    def nbytes(self) -> int:
        return sum(t.numel() for t in (self.k, self.v, self.k_scale, self.v_scale) if t is not None)

    def _here(self, t: torch.Tensor, what: str) -> torch.Tensor:
        if t.device != self.device:
            raise ValueError(f"{what} must be on {self.device}")
        return t

    def write(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        """k, v [T, n_head_kv, head_dim] float32 or bfloat16 go to slots int32 [T]; slots below zero are passed over, the others must differ."""
        if k.dtype != v.dtype:
            raise TypeError("k and v must have the same type")
        s = int32_on(slots, self.device, "slots", (k.shape[0],))
        c = self.ctx
        c.check(c.lib.b200moe_kv_write(c.handle, C.byref(self.desc), C.byref(rows_view(self._here(k, "k"), "k")), C.byref(rows_view(self._here(v, "v"), "v")),
                                       _x_type(k), s, c._stream()))

    def read(self, slots: torch.Tensor, dtype: torch.dtype = torch.bfloat16, out=None):
        """The (k, v) that slots int32 [T] hold, [T, n_head_kv, head_dim] each; slots below zero give zeros.  out: that pair, allocated by the caller."""
        s = int32_on(slots, self.device, "slots", (slots.numel(),))
        if out is None:
            shape = (slots.numel(), self.n_head_kv, self.head_dim)
            k, v = (torch.empty(shape, dtype=dtype, device=self.device) for _ in range(2))
        else:
            k, v = out
            if k.dtype != v.dtype or k.shape[0] != slots.numel():
                raise ValueError("out must be a pair of [T, n_head_kv, head_dim] tensors of one type")
        c = self.ctx
        c.check(c.lib.b200moe_kv_read(c.handle, C.byref(self.desc), s, C.byref(rows_view(self._here(k, "k"), "k")), C.byref(rows_view(self._here(v, "v"), "v")),
                                      _x_type(k), c._stream()))
        return k, v

    def attend(self, q: torch.Tensor, kv_len: torch.Tensor, pages: torch.Tensor, *, max_kv_len: Optional[int] = None,
               q_start: Optional[torch.Tensor] = None, max_new: int = 1, prefix_pages: Optional[torch.Tensor] = None, prefix_len: int = 0,
               scale: Optional[float] = None, out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None,
               workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Attention of the new tokens q [T, n_head, head_dim] of kv_len.numel() sequences over their cached positions behind a shared prefix.

        kv_len int32 [n_seq]: positions of each sequence, its new tokens' last; pages int32 [n_seq, m]: the pages that hold them; prefix_pages int32:
        those of the prefix_len positions in front of every sequence.  q_start int32 [n_seq + 1]: first row of each sequence in q (default: a row each),
        max_new the most rows of one.  max_kv_len (default: what the table has room for) bounds the lengths; the work is split by it, so a
        near bound is faster than a far one.  scale: default head_dim ** -0.5.  lse float32 [T, n_head] receives the logarithms of the sums.
        out, lse: rows that belong to no sequence stay as they are (a new `out` has zeros there)."""
        n_seq = kv_len.numel()
        T, n_head, d = self._here(q, "q").shape
        a = Attn(n_seq=n_seq, max_new=max_new, prefix_len=prefix_len, scale=d ** -0.5 if scale is None else scale)
        a.kv_len = int32_on(kv_len, self.device, "kv_len", (n_seq,))
        a.pages = int32_on(pages, self.device, "pages", (n_seq, pages.shape[-1]))
        a.pages_stride = pages.shape[-1]
        a.max_kv_len = a.pages_stride * self.page_size if max_kv_len is None else max_kv_len
        if q_start is not None:
            a.q_start = int32_on(q_start, self.device, "q_start", (n_seq + 1,))
        if prefix_len:
            if prefix_pages is None or prefix_pages.numel() * self.page_size < prefix_len:
                raise ValueError(f"prefix_pages must name {-(-prefix_len // self.page_size)} pages")
            a.prefix_pages = int32_on(prefix_pages, self.device, "prefix_pages", (prefix_pages.numel(),))
        if out is None:
            out = (torch.empty if q_start is None and T == n_seq else torch.zeros)(q.shape, dtype=q.dtype, device=self.device)
        elif out.dtype != q.dtype or out.shape != q.shape or out.device != self.device:
            raise ValueError("out must be like q")
        if lse is not None and (lse.dtype != torch.float32 or lse.device != self.device or tuple(lse.shape) != (T, n_head) or not lse.is_contiguous()):
            raise ValueError("lse must be a contiguous float32 [T, n_head] tensor")
        c = self.ctx
        need = C.c_size_t()
        c.check(c.lib.b200moe_attention_workspace(c.handle, C.byref(self.desc), C.byref(a), n_head, T, C.byref(need)))
        if workspace is None:
            workspace = torch.empty(need.value, dtype=torch.uint8, device=self.device) if need.value else None
        elif workspace.device != self.device or not workspace.is_contiguous():
            raise ValueError(f"workspace must be a contiguous tensor on {self.device}")
        size = 0 if workspace is None else workspace.numel() * workspace.element_size()
        c.check(c.lib.b200moe_attention(c.handle, C.byref(self.desc), C.byref(a), C.byref(rows_view(q, "q")), _x_type(q), C.byref(rows_view(out, "out")),
                                        _ptr(lse), _ptr(workspace), size, c._stream()))
        return out
