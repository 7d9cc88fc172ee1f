"""A key-value cache in pages: the append that fills them, attention of one new token over them, and the eviction that keeps
a sequence within a budget.

Pools `k_pages`, `v_pages` [pages, G, page, D] hold rows of all sequences; slot j of sequence b is row j % page of page
`table[b, j // page]`, and `lengths[b]` slots are in use.  `mass` [B, G, slots] collects the attention weight every cached key
gets, `positions` [B, G, slots] tells which token a slot holds: after an eviction slots are no longer in the order of tokens,
and differ from head to head.  Attention needs neither order nor positions.

Nothing here synchronises with the host, and nothing has a CPU path.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple

import torch
from torch import Tensor

from . import _lib
from ._lib import check, dtype_code, lib, on_device, ptr, stream_ptr
from .few_rows import _require_on
from .ops import _require_cuda


def _params(k_pages: Tensor, v_pages: Tensor, table: Tensor, lengths: Tensor, mass: Optional[Tensor], positions: Optional[Tensor],
            status: Optional[Tensor]) -> _lib.PagedCacheParams:
    """The parameter block of a cache, its tensors checked."""
    _require_cuda(k_pages)
    dev = k_pages.device
    _require_on(dev, v_pages, table, lengths, mass, positions, status)
    n, G, page, D = k_pages.shape
    B, width = table.shape
    assert v_pages.shape == k_pages.shape and v_pages.dtype == k_pages.dtype and k_pages.stride(3) == v_pages.stride(3) == 1
    assert table.dtype == torch.int32 and (width <= 1 or table.stride(1) == 1)
    assert lengths.dtype == torch.int32 and lengths.shape == (B,) and lengths.is_contiguous()
    mb = mh = pb = ph = 0
    if mass is not None:
        assert mass.dtype == torch.float32
        mb, mh = _book(mass, B, G, width * page)
    if positions is not None:
        assert positions.dtype == torch.int32
        pb, ph = _book(positions, B, G, width * page)
    if status is not None:
        assert status.dtype == torch.int32 and status.numel() == 1
    return _lib.PagedCacheParams(k_pages.data_ptr(), v_pages.data_ptr(), table.data_ptr(), lengths.data_ptr(), ptr(mass), ptr(positions),
                                 ptr(status), *k_pages.stride()[:3], *v_pages.stride()[:3], table.stride(0), n, mb, mh, pb, ph,
                                 dtype_code(k_pages), B, G, D, page, width)


def _book(t: Tensor, B: int, G: int, slots: int) -> Tuple[int, int]:
    """Strides of what is kept per sequence, head and slot."""
    assert t.dim() == 3 and t.shape[0] == B and t.shape[1] == G and t.shape[2] >= slots and (slots <= 1 or t.stride(2) == 1)
    return t.stride(0), t.stride(1)


def append(k_new: Tensor, v_new: Tensor, k_pages: Tensor, v_pages: Tensor, table: Tensor, lengths: Tensor, *,
           counts: Optional[Tensor] = None, first: Optional[Tensor] = None, positions: Optional[Tensor] = None,
           mass: Optional[Tensor] = None, status: Optional[Tensor] = None) -> None:
    """k_new, v_new [B, S, G, D] go to the slots from lengths[b] on: all S tokens, or the first counts[b] (int32) of a padded
    batch.  Their mass starts at 0; their positions are first[b] (int32; without it the slot) and up.  `lengths` stays as it is:
    the caller adds the counts once every layer has appended.  Pages written belong to one sequence each."""
    p = _params(k_pages, v_pages, table, lengths, mass, positions, status)
    _require_on(k_pages.device, k_new, v_new, counts, first)
    B, S = k_new.shape[:2]
    assert B == p.B and k_new.shape == v_new.shape == (B, S, p.G, p.D) and k_new.dtype == v_new.dtype == k_pages.dtype
    assert p.D == 1 or k_new.stride(3) == v_new.stride(3) == 1
    for t in (counts, first):
        assert t is None or (t.dtype == torch.int32 and t.shape == (B,) and t.is_contiguous())
    on_device(k_pages.device, check, lib().sk_paged_append, "sk_paged_append", C.byref(p), k_new.data_ptr(), *k_new.stride()[:3],
              v_new.data_ptr(), *v_new.stride()[:3], S, ptr(counts), ptr(first))


def attn_workspace(H: int, k_pages: Tensor, v_pages: Tensor, table: Tensor, lengths: Tensor, *, mass: Optional[Tensor] = None) -> int:
    """Scratch bytes of `attn` with H query heads on this cache."""
    return int(lib().sk_paged_attn_workspace_bytes(C.byref(_params(k_pages, v_pages, table, lengths, mass, None, None)), H))


def attn(q: Tensor, k_pages: Tensor, v_pages: Tensor, table: Tensor, lengths: Tensor, *, extra: int = 0, scale: Optional[float] = None,
         mass: Optional[Tensor] = None, out: Optional[Tensor] = None, workspace: Optional[Tensor] = None,
         status: Optional[Tensor] = None) -> Tensor:
    """q [B, H, D], one new token per sequence, attends to the first lengths[b] + extra slots of its pages -> [B, H, D]; a
    sequence without keys gets zeros.  `scale` defaults to 1 / sqrt(D).  With `mass` every attended slot collects its weight,
    summed over the query heads of its key/value head.  A workspace that is absent or too small is allocated; calls that may
    run at the same time need one each."""
    p = _params(k_pages, v_pages, table, lengths, mass, None, status)
    dev = k_pages.device
    _require_on(dev, q, out, workspace)
    B, H, D = q.shape
    assert B == p.B and D == p.D and H % p.G == 0 and q.dtype == k_pages.dtype and q.stride(2) == 1
    if out is None:
        out = torch.empty(B, H, D, dtype=q.dtype, device=dev)
    assert out.shape == q.shape and out.dtype == q.dtype and out.stride(2) == 1
    need = lib().sk_paged_attn_workspace_bytes(C.byref(p), H)
    if need and (workspace is None or workspace.numel() * workspace.element_size() < need):
        workspace = torch.empty(need, dtype=torch.uint8, device=dev)
    on_device(dev, check, lib().sk_paged_attn, "sk_paged_attn", C.byref(p), q.data_ptr(), *q.stride()[:2], out.data_ptr(), *out.stride()[:2],
              H, extra, D ** -0.5 if scale is None else float(scale), ptr(workspace),
              0 if workspace is None else workspace.numel() * workspace.element_size())
    return out


def evict(k_pages: Tensor, v_pages: Tensor, table: Tensor, lengths: Tensor, mass: Tensor, positions: Tensor, *, budget: int,
          recent: int = 0, sink: int = 0, out: Optional[Tuple[Tensor, Tensor, Tensor]] = None,
          status: Optional[Tensor] = None) -> Tuple[Tensor, Tensor, Tensor]:
    """Cuts every sequence to at most `budget` slots, each key/value head by itself: kept are the tokens at positions below
    `sink`, the newest `recent` ones, and of the others those with the largest mass (the lowest slot of equal ones).  Kept slots
    below the budget stay, the others move into the freed ones, keys and values in place.  Returns mass, positions (0 and -1
    behind the new lengths) and lengths; `out` names the tensors that get them, (mass, positions, lengths) themselves for an
    eviction in place.  Other tensors must not overlap the inputs, nor one another.  Pages of one sequence are no other's."""
    p = _params(k_pages, v_pages, table, lengths, mass, positions, status)
    dev = k_pages.device
    slots = p.width * p.page
    if out is None:
        out = (torch.empty(p.B, p.G, slots, dtype=torch.float32, device=dev),
               torch.empty(p.B, p.G, slots, dtype=torch.int32, device=dev), torch.empty_like(lengths))
    m, q, n = out
    _require_on(dev, m, q, n)
    assert m.dtype == torch.float32 and q.dtype == n.dtype == torch.int32 and n.shape == lengths.shape and n.is_contiguous()
    strides = (*_book(m, p.B, p.G, slots), *_book(q, p.B, p.G, slots))
    need = lib().sk_paged_evict_workspace_bytes(C.byref(p), budget)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    on_device(dev, check, lib().sk_paged_evict, "sk_paged_evict", C.byref(p), budget, recent, sink, m.data_ptr(), *strides[:2], q.data_ptr(),
              *strides[2:], n.data_ptr(), ptr(ws), need)
    return out
