"""A cache of keys and values in pages that grows token by token, and attention over it.

``sageattn`` takes keys and values in one piece.  A program that answers token by token keeps them instead: in
pages of a few tokens that belong to a sequence through a page table, so that sequences grow without being moved.
Per layer and step:

    cache = PagedKV.allocate(num_pages, 16, num_kv_heads, 128, dtype=torch.bfloat16)
    q = paged_kv_append(cache, k, v, page_table, kv_lens, rotary=rope, q=q)     # turned on the way into the pages
    o = sageattn_paged(q, cache, page_table, kv_lens)

The tokens of a batch lie one behind the other, ``[T, heads, D]``: one per sequence, or those of sequence b in rows
``cu_q[b]`` to ``cu_q[b + 1]`` (prompts in chunks, drafted tokens, a mixture of both).  Page table and lengths stay on the
device: no call synchronises, and every call can be captured in a CUDA graph.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Union

import torch

from . import _native
from .core import _LAYOUT_CODE, _prepare_status, _raise_pending, _status_word
from .rotary import RotaryAxes, _vector_aligned

PAGE_SIZES = (16, 32, 64, 128, 256)


@dataclass
class PagedKV:
    """Pages of keys and values: ``[pages, page_size, Hkv, D]`` ("NHD") or ``[pages, Hkv, page_size, D]`` ("HND")."""
    k_pages: torch.Tensor
    v_pages: torch.Tensor
    tensor_layout: str = "NHD"

    def __post_init__(self) -> None:
        k, v = self.k_pages, self.v_pages
        assert self.tensor_layout in _LAYOUT_CODE, f"tensor_layout must be 'HND' or 'NHD', got {self.tensor_layout!r}."
        assert k.dim() == 4 and k.shape == v.shape, "k_pages and v_pages must be 4-D tensors of the same shape."
        assert k.dtype == v.dtype and k.dtype in (torch.float16, torch.bfloat16), "pages must both be fp16 or bf16."
        assert k.device == v.device, "k_pages and v_pages must be on the same device."
        assert self.head_dim in (64, 128), f"head_dim must be 64 or 128, got {self.head_dim}."
        assert self.page_size in PAGE_SIZES, f"page_size must be one of {PAGE_SIZES}, got {self.page_size}."
        assert k.size(0) > 0 and self.num_kv_heads > 0, "the cache needs a page and a head."
        for t in (k, v):
            assert t.stride(3) == 1 and t.data_ptr() % 16 == 0 and all(
                n == 1 or (s % 8 == 0 and s > 0) for n, s in zip(t.shape[:3], t.stride()[:3])), (
                "pages need a contiguous last dim, a 16-byte aligned base and strides that are multiples of 8; "
                f"got strides {t.stride()}.")
        if k.is_cuda and not torch.cuda.is_current_stream_capturing():
            _prepare_status(k.device)        # so that the first call on the device may be a captured one

    @classmethod
    def allocate(cls, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int, dtype: torch.dtype = torch.bfloat16,
                 tensor_layout: str = "NHD", device: Union[torch.device, int, str, None] = None) -> "PagedKV":
        """A cache of zeros on ``device`` (the current CUDA device)."""
        shape = ((num_pages, num_kv_heads, page_size, head_dim) if tensor_layout == "HND"
                 else (num_pages, page_size, num_kv_heads, head_dim))
        dev = "cuda" if device is None else device
        return cls(torch.zeros(shape, dtype=dtype, device=dev), torch.zeros(shape, dtype=dtype, device=dev), tensor_layout)

    @property
    def page_size(self) -> int:
        return self.k_pages.size(2 if self.tensor_layout == "HND" else 1)

    @property
    def num_kv_heads(self) -> int:
        return self.k_pages.size(1 if self.tensor_layout == "HND" else 2)

    @property
    def num_pages(self) -> int:
        return self.k_pages.size(0)

    @property
    def head_dim(self) -> int:
        return self.k_pages.size(3)


def _check_batch(cache: PagedKV, rows: torch.Tensor, page_table: torch.Tensor, kv_lens: torch.Tensor,
                 cu_q: Optional[torch.Tensor]) -> None:
    assert isinstance(cache, PagedKV), "cache must be a PagedKV."
    dev = cache.k_pages.device
    for name, t, dim in (("page_table", page_table, 2), ("kv_lens", kv_lens, 1), ("cu_q", cu_q, 1)):
        if t is None:
            continue
        assert t.dtype == torch.int32 and t.device == dev and t.dim() == dim, (
            f"{name} must be a {dim}-D int32 tensor on the device of the cache.")
        assert t.size(-1) <= 1 or t.stride(-1) == 1, f"{name}: last dim must be contiguous."
    B = kv_lens.size(0)
    assert page_table.size(0) == B, "page_table and kv_lens differ in the number of sequences."
    if cu_q is None:
        assert rows.size(0) == B, f"without cu_q there is one token per sequence: {rows.size(0)} rows for {B} sequences."
    else:
        assert cu_q.size(0) == B + 1, f"cu_q must have {B + 1} entries, got {cu_q.size(0)}."


def _check_rows(cache: PagedKV, name: str, t: torch.Tensor, heads: Optional[int] = None) -> None:
    assert t.dim() == 3 and t.size(2) == cache.head_dim and (heads is None or t.size(1) == heads), (
        f"{name} must be [T, {'heads' if heads is None else heads}, {cache.head_dim}], got {tuple(t.shape)}.")
    assert t.dtype == cache.k_pages.dtype and t.device == cache.k_pages.device, (
        f"{name} must have the dtype and device of the cache.")
    assert not (torch.is_grad_enabled() and t.requires_grad), (
        f"{name} requires a gradient: the paged cache has none (detach it, or call under torch.no_grad()).")


def paged_kv_append(cache: PagedKV, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor, kv_lens: torch.Tensor,
                    cu_q: Optional[torch.Tensor] = None, rotary: Optional[RotaryAxes] = None,
                    positions: Optional[torch.Tensor] = None, q: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Stores the keys and values of new tokens in their pages, one launch.

    k, v: ``[T, Hkv, D]`` in the dtype of the cache; any strides with a contiguous last dim (slices of a joint
    projection are read in place where 16-byte loads allow).  kv_lens: ``[B]`` int32, the length of every sequence WITH its new
    tokens; new token i of n stands at position ``kv_lens[b] - n + i``, in slot ``position % page_size`` of page
    ``page_table[b, position // page_size]``.  page_table: ``[B, pages]`` int32; entries behind the last token are not looked at.

    rotary: k is turned on its way, and q (``[T, Hq, D]``) too: the turned q is returned, a new tensor.  The position is the one in
    the sequence, on every axis, unless ``positions`` (``[T]`` or ``[T, axes]``, int32 / int64) gives others.

    Rows that belong to no sequence (T may be padded) are not stored, and zero in the returned q.  A page index
    outside the cache, a position outside the page table or more new tokens than ``kv_lens`` says are not stored either; they
    are reported like the errors of ``sageattn``, by the next call or ``check_status()``.  Two sequences that share a page
    must not append to it at once."""
    _check_batch(cache, k, page_table, kv_lens, cu_q)
    _check_rows(cache, "k", k, cache.num_kv_heads)
    _check_rows(cache, "v", v, cache.num_kv_heads)
    T = k.size(0)
    assert v.size(0) == T, "k and v differ in length."
    if q is not None:
        assert rotary is not None, "q is only turned: it needs rotary."
        _check_rows(cache, "q", q)
        assert q.size(0) == T, "q and k differ in length."
        q = _vector_aligned(q)
    assert positions is None or rotary is not None, "positions are those of rotary."
    if rotary is not None:
        assert isinstance(rotary, RotaryAxes) and rotary.head_dim == cache.head_dim, "rotary must come from rotary_axes() with the head_dim of the cache."
        assert rotary.freq.device == cache.k_pages.device, "the rotary table is on another device than the cache."
    if positions is not None:
        assert positions.device == cache.k_pages.device and positions.dtype in (torch.int32, torch.int64), (
            "positions must be int32 or int64 on the device of the cache.")
        if rotary.n_axes == 1 and positions.dim() == 1:
            positions = positions.unsqueeze(-1)
        assert tuple(positions.shape) == (T, rotary.n_axes), (
            f"positions must be [T{'' if rotary.n_axes == 1 else ', axes'}] with T = {T}, got {tuple(positions.shape)}.")
        if rotary.n_axes > 1 and positions.stride(-1) != 1:
            positions = positions.contiguous()
    dev = cache.k_pages.device
    assert dev.type == "cuda", "the cache must be on a CUDA device."
    ops = _native.load_ops()
    _raise_pending(dev)
    out = ops.paged_append(cache.k_pages, cache.v_pages, _LAYOUT_CODE[cache.tensor_layout], _vector_aligned(k), _vector_aligned(v),
                           page_table, kv_lens, cu_q, q, None if rotary is None else rotary.freq,
                           None if rotary is None else rotary.axis, 0 if rotary is None else rotary.n_axes,
                           0 if rotary is None else int(rotary.interleaved), positions, _status_word(dev))
    return out[0] if q is not None else None
