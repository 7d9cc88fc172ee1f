"""A key-value cache in pages: the append that fills them, attention of one new token over them, and the eviction that keeps
a sequence within a budget.

Pools `k_pages`, `v_pages` [pages, G, page, D] hold rows of all sequences; slot j of sequence b is row j % page of page
`table[b, j // page]`, and `lengths[b]` slots are in use.  `mass` [B, G, slots] collects the attention weight every cached key
gets, `positions` [B, G, slots] tells which token a slot holds: after an eviction slots are no longer in the order of tokens,
and differ from head to head.  Attention needs neither order nor positions.  What a call only reads may be expanded; what it writes
must not (an error).

Nothing here synchronises with the host, and nothing has a CPU path.
"""
from __future__ import annotations

import struct
from dataclasses import dataclass
from typing import List, Optional, Tuple

import torch
import torch.nn as nn
from torch import Tensor

from . import _lib
from ._lib import _raw_stream, check, dtype_code, lib, on_device, ptr

# `sk_paged_cache` as bytes: filling in a ctypes structure field by field costs a call of a few microseconds another three
_pack = struct.Struct("7P12q6i").pack


def _elsewhere(index: int, t: Tensor) -> RuntimeError:
    """Every tensor of a call lies on the device of its pools: the kernels read and write addresses."""
    return RuntimeError(f"tensors of one call on device {index} and on {t.device}")


def _same_device(index: int, *tensors: Optional[Tensor]) -> None:
    for t in tensors:
        if t is not None and t.get_device() != index:
            raise _elsewhere(index, t)


def _run(index: int, entry, what: str, *args) -> None:
    """entry(*args, stream) on the current stream of device `index`, the current device."""
    status = entry(*args, torch.cuda.current_stream(index).cuda_stream if _raw_stream is None else _raw_stream(index))
    if status != 0:
        check(status, what)


def _cache(k_pages: Tensor, v_pages: Tensor, table: Tensor, lengths: Tensor, mass: Optional[Tensor], positions: Optional[Tensor],
           status: Optional[Tensor]) -> bytes:
    """The parameter block of a cache, its tensors checked."""
    index = k_pages.get_device()
    if index < 0:
        raise RuntimeError("socket_b200 operators need CUDA tensors (there is no CPU path)")
    if not index == v_pages.get_device() == table.get_device() == lengths.get_device():
        _same_device(index, v_pages, table, lengths)
    shape, ks, vs = k_pages.shape, k_pages.stride(), v_pages.stride()
    n, G, page, D = shape
    B, width = table.shape
    ts = table.stride()
    assert v_pages.shape == shape and v_pages.dtype == k_pages.dtype and ks[3] == vs[3] == 1
    assert table.dtype == lengths.dtype == torch.int32 and (width <= 1 or ts[1] == 1)
    assert lengths.shape == (B,) and lengths.is_contiguous()
    mb = mh = pb = ph = 0
    if mass is not None:
        if mass.get_device() != index:
            raise _elsewhere(index, mass)
        assert mass.dtype == torch.float32
        mb, mh = _book(mass, B, G, width * page)
    if positions is not None:
        if positions.get_device() != index:
            raise _elsewhere(index, positions)
        assert positions.dtype == torch.int32
        pb, ph = _book(positions, B, G, width * page)
    if status is not None:
        if status.get_device() != index:
            raise _elsewhere(index, status)
        assert status.dtype == torch.int32 and status.numel() == 1
    return _pack(k_pages.data_ptr(), v_pages.data_ptr(), table.data_ptr(), lengths.data_ptr(), ptr(mass), ptr(positions), ptr(status),
                 ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], ts[0], n, mb, mh, pb, ph, dtype_code(k_pages), B, G, D, page, width)


def _book(t: Tensor, B: int, G: int, slots: int) -> Tuple[int, int]:
    """Strides of what is kept per sequence, head and slot."""
    b, g, n = t.shape
    s = t.stride()
    assert b == B and g == G and n >= slots and (slots <= 1 or s[2] == 1)
    return s[0], s[1]


def append(k_new: Tensor, v_new: Tensor, k_pages: Tensor, v_pages: Tensor, table: Tensor, lengths: Tensor, *,
           counts: Optional[Tensor] = None, first: Optional[Tensor] = None, positions: Optional[Tensor] = None,
           mass: Optional[Tensor] = None, status: Optional[Tensor] = None) -> None:
    """k_new, v_new [B, S, G, D] go to the slots from lengths[b] on: all S tokens, or the first counts[b] (int32) of a padded
    batch.  Their mass starts at 0; their positions are first[b] (int32; without it the slot) and up.  `lengths` stays as it is:
    the caller adds the counts once every layer has appended.  Pages written belong to one sequence each; rows of k_new and
    v_new start on 16-byte boundaries."""
    c = _cache(k_pages, v_pages, table, lengths, mass, positions, status)
    _same_device(k_pages.get_device(), k_new, v_new, counts, first)
    B, S, G, D = k_new.shape
    ks, vs = k_new.stride(), v_new.stride()
    assert v_new.shape == k_new.shape and B == table.shape[0] and G == k_pages.shape[1] and D == k_pages.shape[3]
    assert k_new.dtype == v_new.dtype == k_pages.dtype and ks[3] == vs[3] == 1
    for t in (counts, first):
        assert t is None or (t.dtype == torch.int32 and t.shape == (B,) and t.is_contiguous())
    on_device(k_pages.get_device(), check, lib().sk_paged_append, "sk_paged_append", c, k_new.data_ptr(), ks[0], ks[1], ks[2],
              v_new.data_ptr(), vs[0], vs[1], vs[2], S, ptr(counts), ptr(first))


def attn_workspace(H: int, k_pages: Tensor, v_pages: Tensor, table: Tensor, lengths: Tensor, *, mass: Optional[Tensor] = None) -> int:
    """Scratch bytes of `attn` with H query heads on this cache."""
    if k_pages.get_device() not in (-1, torch.cuda.current_device()):          # sized for the SMs of the cache's device
        with torch.cuda.device(k_pages.device):
            return attn_workspace(H, k_pages, v_pages, table, lengths, mass=mass)
    return int(lib().sk_paged_attn_workspace_bytes(_cache(k_pages, v_pages, table, lengths, mass, None, None), H))


def attn(q: Tensor, k_pages: Tensor, v_pages: Tensor, table: Tensor, lengths: Tensor, *, extra: int = 0, scale: Optional[float] = None,
         mass: Optional[Tensor] = None, out: Optional[Tensor] = None, workspace: Optional[Tensor] = None,
         status: Optional[Tensor] = None) -> Tensor:
    """q [B, H, D], one new token per sequence, attends to the first lengths[b] + extra slots of its pages -> [B, H, D]; a
    sequence without keys gets zeros.  `scale` defaults to 1 / sqrt(D).  With `mass` every attended slot collects its weight,
    summed over the query heads of its key/value head.  Rows of q and out start on 16-byte boundaries, as those of the pools do.
    A workspace that is absent or too small is allocated; calls that may run at the same time need one each."""
    c = _cache(k_pages, v_pages, table, lengths, mass, None, status)
    index = k_pages.get_device()
    if index != torch.cuda.current_device():                  # the split, and its scratch, go by the device's SMs
        with torch.cuda.device(index):
            return attn(q, k_pages, v_pages, table, lengths, extra=extra, scale=scale, mass=mass, out=out, workspace=workspace, status=status)
    _same_device(index, q, out, workspace)
    shape, qs = q.shape, q.stride()
    B, H, D = shape
    assert B == table.shape[0] and D == k_pages.shape[3] and H % k_pages.shape[1] == 0 and q.dtype == k_pages.dtype and qs[2] == 1
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    os = out.stride()
    assert out.shape == shape and out.dtype == q.dtype and os[2] == 1
    entry = lib()
    need = entry.sk_paged_attn_workspace_bytes(c, H)
    assert workspace is None or workspace.is_contiguous()
    have = 0 if workspace is None else workspace.numel() * workspace.element_size()
    if have < need:
        workspace, have = torch.empty(need, dtype=torch.uint8, device=q.device), need
    _run(index, entry.sk_paged_attn, "sk_paged_attn", c, q.data_ptr(), qs[0], qs[1], out.data_ptr(), os[0], os[1], H, extra,
              D ** -0.5 if scale is None else float(scale), ptr(workspace), have)
    return out


def evict(k_pages: Tensor, v_pages: Tensor, table: Tensor, lengths: Tensor, mass: Tensor, positions: Tensor, *, budget: int,
          recent: int = 0, sink: int = 0, out: Optional[Tuple[Tensor, Tensor, Tensor]] = None,
          status: Optional[Tensor] = None) -> Tuple[Tensor, Tensor, Tensor]:
    """Cuts every sequence to at most `budget` slots, each key/value head by itself: kept are the tokens at positions below
    `sink`, the newest `recent` ones, and of the others those with the largest mass (the lowest slot of equal ones).  Kept slots
    below the budget stay, the others move into the freed ones, keys and values in place.  Returns mass, positions (0 and -1
    behind the new lengths) and lengths; `out` names the tensors that get them, (mass, positions, lengths) themselves for an
    eviction in place.  Other tensors must not overlap the inputs, nor one another.  Pages of one sequence are no other's."""
    c = _cache(k_pages, v_pages, table, lengths, mass, positions, status)
    index, dev = k_pages.get_device(), k_pages.device
    if index != torch.cuda.current_device():
        with torch.cuda.device(index):
            return evict(k_pages, v_pages, table, lengths, mass, positions, budget=budget, recent=recent, sink=sink, out=out, status=status)
    B, G, slots = table.shape[0], k_pages.shape[1], table.shape[1] * k_pages.shape[2]
    if out is None:
        out = tuple(torch.empty_like(t if t.shape[2] == slots else t[..., :slots], memory_format=torch.contiguous_format)
                    for t in (mass, positions)) + (torch.empty_like(lengths),)
    m, q, n = out
    _same_device(index, m, q, n)
    assert m.dtype == torch.float32 and q.dtype == n.dtype == torch.int32 and n.shape == lengths.shape and n.is_contiguous()
    (mb, mh), (pb, ph) = _book(m, B, G, slots), _book(q, B, G, slots)
    entry = lib()
    need = entry.sk_paged_evict_workspace_bytes(c, budget)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    _run(index, entry.sk_paged_evict, "sk_paged_evict", c, budget, recent, sink, m.data_ptr(), mb, mh, q.data_ptr(), pb, ph,
              n.data_ptr(), ptr(ws), need)
    return out


# ---------------------------------------------------------------------------------- caches of a decoder
@dataclass(frozen=True)
class Paging:
    """How a decoder keeps its caches in pages.  With a budget, sequences that have grown `every` tokens beyond it are cut back to
    it: the first `sink` tokens, the last `recent` ones and the keys that decoded tokens attended to most stay.

    A prompt's queries collect no weights.  One longer than `budget + every` is cut behind the first decoded token, by that token's
    weights alone, and a later turn's tokens start from nothing beside keys that have collected for long: what has to outlast
    that is `sink`'s and `recent`'s to keep."""
    page: int = 64
    pages: int = 0                      # of the pool; 0: as many as all sequences need at their longest
    budget: int = 0                     # 0: nothing is evicted
    recent: int = 0
    sink: int = 0
    every: int = 64

    def __post_init__(self):
        if self.page < 16 or self.page & (self.page - 1):
            raise ValueError(f"pages of {self.page} rows: a power of two, at least 16")
        if self.budget < 0 or self.recent < 0 or self.sink < 0 or self.pages < 0 or (self.budget and self.recent + self.sink > self.budget):
            raise ValueError(f"a budget of {self.budget} for {self.sink} first and {self.recent} last tokens, {self.pages} pages")
        if self.budget and self.every < 1:
            raise ValueError("evictions need at least one token between them")


class PageTable:
    """Which pages a decoder's sequences hold, the same in every layer: all sequences grow in step.  The host decides, the device
    reads `table`, `lengths` and `positions` (of the next token)."""

    def __init__(self, batch: int, max_length: int, page: int, pages: int = 0, device=None):
        self.page, self.width = page, -(-max_length // page)
        self.pages = pages or batch * self.width
        self.table = torch.full((batch, self.width), -1, dtype=torch.int32, device=device)
        self.counters = torch.zeros(2, batch, dtype=torch.int32, device=device)
        self.lengths, self.positions = self.counters[0], self.counters[1]
        self.reset()

    def reset(self) -> None:
        """No tokens, all pages free."""
        self.free = list(range(self.pages - 1, -1, -1))
        self.held: List[List[int]] = [[] for _ in range(self.table.shape[0])]
        self.length = self.position = 0
        self.counters.zero_()
        self._show()

    def _show(self) -> None:
        rows = [held + [-1] * (self.width - len(held)) for held in self.held]
        rows = torch.tensor(rows, dtype=torch.int32).view(self.table.shape)
        if self.table.is_cuda:                                # from pinned memory the host does not wait; it is not used again before it is read
            rows = rows.pin_memory()
        self.table.copy_(rows, non_blocking=True)

    def hide(self) -> None:
        """The device sees no pages until `show`: calls on the cache then write and read nothing."""
        self.table.fill_(-1)

    show = _show

    def reserve(self, length: int) -> None:
        """Pages for `length` slots of every sequence."""
        want = -(-length // self.page)
        if want > self.width:
            raise RuntimeError(f"{length} slots in a cache of {self.width * self.page}")
        if all(len(held) >= want for held in self.held):
            return
        if sum(max(0, want - len(held)) for held in self.held) > len(self.free):
            raise RuntimeError(f"out of pages: {len(self.free)} of {self.pages} free, sequences of {length} slots asked for")
        for held in self.held:
            while len(held) < want:
                held.append(self.free.pop())
        self._show()

    def cut(self, length: int) -> None:
        """Slots from `length` on are given back; the device's lengths are the caller's."""
        keep = -(-length // self.page)
        for held in self.held:
            self.free += reversed(held[keep:])
            del held[keep:]
        self.length = length
        self._show()

    def advance(self, tokens: int, on_device: bool = True) -> None:
        """`tokens` more of every sequence are cached.  Without `on_device` the device has counted them itself."""
        self.length += tokens
        self.position += tokens
        if on_device:
            self.counters.add_(tokens)


class PagedKVCache(nn.Module):
    """One layer's keys and values in pages, with what eviction goes by."""

    def __init__(self, pages: PageTable, n_heads: int, head_dim: int, dtype=torch.bfloat16, device=None, collect: bool = False):
        super().__init__()
        self.pages = pages
        shape = (pages.pages, n_heads, pages.page, head_dim)
        self.register_buffer("k_pages", torch.zeros(shape, dtype=dtype, device=device))
        self.register_buffer("v_pages", torch.zeros(shape, dtype=dtype, device=device))
        book = (pages.table.shape[0], n_heads, pages.width * pages.page)
        self.register_buffer("mass", torch.zeros(book, dtype=torch.float32, device=device) if collect else None)
        self.register_buffer("slot_positions", torch.zeros(book, dtype=torch.int32, device=device) if collect else None)
        self.register_buffer("status", torch.zeros((), dtype=torch.int32, device=device))

    def append(self, k: Tensor, v: Tensor) -> None:
        """k, v [B, S, heads, D] behind the cached tokens; `pages.advance` follows once every layer has appended."""
        append(k, v, self.k_pages, self.v_pages, self.pages.table, self.pages.lengths, first=self.pages.positions,
               positions=self.slot_positions, mass=self.mass, status=self.status)

    def attend(self, q: Tensor, out: Tensor, workspace: Optional[Tensor] = None) -> Tensor:
        """q [B, H, D] of the token just appended over everything cached."""
        return attn(q, self.k_pages, self.v_pages, self.pages.table, self.pages.lengths, extra=1, mass=self.mass, out=out,
                    workspace=workspace, status=self.status)

    def attend_workspace(self, n_head: int) -> int:
        return attn_workspace(n_head, self.k_pages, self.v_pages, self.pages.table, self.pages.lengths, mass=self.mass)

    def evict(self, budget: int, recent: int, sink: int, lengths: Tensor) -> None:
        """Down to `budget` slots; `lengths` gets the new lengths, those of the table stay for the other layers."""
        evict(self.k_pages, self.v_pages, self.pages.table, self.pages.lengths, self.mass, self.slot_positions, budget=budget, recent=recent,
              sink=sink, out=(self.mass, self.slot_positions, lengths), status=self.status)

    def rows(self, length: int) -> Tuple[Tensor, Tensor]:
        """Keys and values [B, heads, length, D] of the first slots, copied out of the pages."""
        at = self.pages.table[:, :-(-length // self.pages.page)].long()
        return tuple(pool[at].transpose(1, 2).flatten(2, 3)[:, :, :length] for pool in (self.k_pages, self.v_pages))
