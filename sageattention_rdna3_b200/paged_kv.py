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

import os
from dataclasses import dataclass
from typing import Optional, Tuple, Union

import torch
import torch.autograd.forward_ad as fwAD

from . import _native
from .core import _LAYOUT_CODE, _prepare_status, _raise_pending, _register, _status_word, check_status
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
        assert not (k.requires_grad or v.requires_grad), "pages must not require a gradient: the paged cache has none."
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


def _check_if_asked(device: torch.device) -> None:
    if os.environ.get("SAGEATTN_B200_CHECK_STATUS", "0") == "1":
        check_status(device)


def _table_of(rotary: Optional[RotaryAxes]) -> tuple:
    """(frequencies, axes, number of axes, interleaved) as the operators take them."""
    return (None, None, 0, False) if rotary is None else (rotary.freq, rotary.axis, len(rotary.axes), rotary.interleaved)


def _check_no_derivative(name: str, t: torch.Tensor) -> None:
    assert not (torch.is_grad_enabled() and t.requires_grad), (
        f"{name} requires a gradient: the paged cache has none (detach it, or call under torch.no_grad()).")
    assert fwAD.unpack_dual(t).tangent is None, f"{name} has a tangent: the paged cache has no derivative in forward mode either."


def _check_rows(cache: PagedKV, name: str, t: torch.Tensor, heads: Optional[int] = None) -> None:
    assert t.dim() == 3 and t.size(2) == cache.head_dim and (heads is None or t.size(1) == heads), (
        f"{name} must be [T, {'heads' if heads is None else heads}, {cache.head_dim}], got {tuple(t.shape)}.")
    assert t.dtype == cache.k_pages.dtype and t.device == cache.k_pages.device, (
        f"{name} must have the dtype and device of the cache.")
    _check_no_derivative(name, t)


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

    Rows that belong to no sequence (T may be padded) are not stored, and zero in the returned q; without ``cu_q`` also those of
    length 0, slots of a batch that are not in use.  A page index
    outside the cache, a position outside the page table or more new tokens than ``kv_lens`` says are not stored either; they
    are reported like the errors of ``sageattn``, by the next call or ``check_status()``.  Two sequences that share a page
    must not append to it at once, and k, v and q must not lie in the cache."""
    assert isinstance(cache, PagedKV), "cache must be a PagedKV."
    assert rotary is None or (isinstance(rotary, RotaryAxes) and rotary.head_dim == cache.head_dim), (
        "rotary must come from rotary_axes() with the head_dim of the cache.")
    if not torch.compiler.is_compiling():
        got = _native.load_module().paged_append_plain(
            cache.k_pages, cache.v_pages, cache.tensor_layout, k, v, page_table, kv_lens, cu_q, q, *_table_of(rotary), positions)
        if got is not None:                  # None: not a plain call, or one that the checks below refuse
            return None if got is True else got
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
    _register(dev)
    out = ops.paged_append(cache.k_pages, cache.v_pages, _LAYOUT_CODE[cache.tensor_layout], _vector_aligned(k), _vector_aligned(v),
                           page_table, kv_lens, cu_q, q, *_table_of(rotary), positions, _status_word(dev))
    _check_if_asked(dev)
    return out[0] if q is not None else None


def sageattn_paged(q: torch.Tensor, cache: PagedKV, page_table: torch.Tensor, kv_lens: torch.Tensor,
                   cu_q: Optional[torch.Tensor] = None, max_q: Optional[int] = None, is_causal: bool = True,
                   sm_scale: Optional[float] = None, return_lse: bool = False, shared_pages: Optional[torch.Tensor] = None,
                   out: Optional[torch.Tensor] = None) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Attention of the newest tokens of every sequence over its keys and values in the cache.

    q: ``[T, Hq, D]`` in the dtype of the cache, the tokens that ``paged_kv_append`` stored last (Hq a multiple of the cache's
    heads, at most 128 times them).  kv_lens: ``[B]`` int32, keys of every sequence with its new tokens.  ``cu_q`` as in
    ``paged_kv_append``; ``max_q`` is an upper bound of the new tokens of one sequence and chooses the kernel, not the result: with ``cu_q``
    give it where it is known (64 single tokens took 126 us with it, 197 without).  ``is_causal`` aligns the last new token with the last key (a token sees the keys up to its own
    position); without it every token sees all keys of its sequence.  A row without keys is zero, its log-sum-exp -inf.
    Keys that a row does not see may be anything.  Values of new tokens that are not finite may reach the rows of earlier tokens of
    the same step and sequence (0 * inf), as they do in a product of matrices; no other sequence.

    shared_pages: ``[n]`` int32.  The first ``n * page_size`` keys of every sequence stand in these pages (a system
    prompt, one question with many answers); they are read once for the whole batch, and the first n columns of ``page_table``
    are not looked at.  Positions and ``kv_lens`` count them as ever, and the result is the same as without the argument, up to
    rounding.

    Returns ``[T, Hq, D]``, with ``return_lse`` also the natural log-sum-exp ``[T, Hq]`` (fp32).  Rows that belong to no sequence are
    zero (-inf); given ``out``, which receives the result, they are left as they were there.  ``out`` may be ``q``, but must not
    overlap it otherwise, nor the cache.  Keys and values behind a
    sequence's last one may be anything, NaN too.  Lengths beyond the page table are cut to it, page indices
    outside the cache are read as page 0, and both are reported like the errors of ``sageattn``, by the next call or
    ``check_status()``.  No gradient."""
    assert isinstance(cache, PagedKV), "cache must be a PagedKV."
    if out is None and not torch.compiler.is_compiling():
        got = _native.load_module().paged_attn_plain(q, cache.k_pages, cache.v_pages, cache.tensor_layout, page_table, kv_lens, cu_q,
                                                     max_q, is_causal, sm_scale, return_lse, shared_pages)
        if got is not None:                  # None: not a plain call, or one that the checks below refuse
            return got
    _check_batch(cache, q, page_table, kv_lens, cu_q)
    _check_rows(cache, "q", q)
    T, heads, B = q.size(0), q.size(1), kv_lens.size(0)
    assert heads > 0 and heads % cache.num_kv_heads == 0 and heads // cache.num_kv_heads <= 128, (
        f"num_qo_heads must be a multiple of num_kv_heads, at most 128 times it; got {heads} and {cache.num_kv_heads}.")
    assert max_q is None or max_q >= 0, f"max_q must not be negative, got {max_q}."
    dev = cache.k_pages.device
    if shared_pages is not None:
        assert shared_pages.dtype == torch.int32 and shared_pages.device == dev and shared_pages.dim() == 1, (
            "shared_pages must be a 1-D int32 tensor on the device of the cache.")
        assert shared_pages.size(0) <= 1 or shared_pages.stride(0) == 1, "shared_pages must be contiguous."
        assert shared_pages.size(0) <= page_table.size(1), "page_table has fewer columns than there are shared pages."
    if out is not None:
        assert out.shape == q.shape and out.dtype == q.dtype and out.device == q.device, (
            "out must have the shape, dtype and device of q.")
        _check_no_derivative("out", out)
        assert out.stride(2) == 1 and out.data_ptr() % 16 == 0 and all(
            n <= 1 or (s % 8 == 0 and s > 0) for n, s in zip(out.shape[:2], out.stride()[:2])), (
            f"out needs a contiguous last dim, 16-byte aligned rows and a place for every row; got strides {out.stride()}.")
    assert dev.type == "cuda", "the cache must be on a CUDA device."
    ops = _native.load_ops()
    _raise_pending(dev)
    _register(dev)
    zero_rest = out is None and cu_q is not None
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=dev) if B > 0 else torch.zeros(q.shape, dtype=q.dtype, device=dev)
    lse = None
    if return_lse:
        lse = torch.empty(T, heads, dtype=torch.float32, device=dev)
        if B == 0 or (cu_q is not None and not zero_rest):
            lse.fill_(float("-inf"))
    if any(n > 1 and s == 0 for n, s in zip(q.shape, q.stride())):      # an expanded q
        q = q.contiguous()
    ops.paged_attn(_vector_aligned(q), out, cache.k_pages, cache.v_pages, _LAYOUT_CODE[cache.tensor_layout], page_table, kv_lens,
                   cu_q, 0 if max_q is None else min(int(max_q), T), int(is_causal),
                   cache.head_dim ** -0.5 if sm_scale is None else float(sm_scale), lse, shared_pages, int(zero_rest),
                   _status_word(dev))
    _check_if_asked(dev)
    return (out, lse) if return_lse else out
