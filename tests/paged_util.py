"""Paged caches and their plain forms in 64 bits, for the tests."""
import math

import torch

HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


class Cache:
    """Pools of randomly ordered pages for sequences of the given lengths; what no sequence uses is NaN and infinities."""

    def __init__(self, lengths, G, D, page, dtype, device, *, room=0, spare=3, seed=0, combined=False, width=None):
        g = torch.Generator(device=device).manual_seed(seed)
        B = len(lengths)
        self.width = max(1, -(-(max(lengths) + room) // page)) if width is None else width
        n = B * self.width + spare
        if combined:                                  # keys and values of a page side by side, heads inside rows
            pool = torch.full((n, page, 2, G, D), float("nan"), dtype=dtype, device=device)
            self.k, self.v = pool[:, :, 0].permute(0, 2, 1, 3), pool[:, :, 1].permute(0, 2, 1, 3)
        else:
            self.k = torch.full((n, G, page, D), float("nan"), dtype=dtype, device=device)
            self.v = torch.full((n, G, page, D), float("inf"), dtype=dtype, device=device)
        self.table = torch.randperm(n, generator=g, device=device)[:B * self.width].to(torch.int32).view(B, self.width)
        self.lengths = torch.tensor(lengths, dtype=torch.int32, device=device)
        self.page, self.G, self.D, self.cap = page, G, D, self.width * page
        self.rows_k = [torch.randn(G, m, D, generator=g, device=device).to(dtype) for m in lengths]
        self.rows_v = [torch.randn(G, m, D, generator=g, device=device).to(dtype) for m in lengths]
        for b, m in enumerate(lengths):
            self.set(self.k, b, 0, self.rows_k[b])
            self.set(self.v, b, 0, self.rows_v[b])
        self.gen = g

    def places(self, b, slots):
        return self.table[b].long()[slots // self.page], slots % self.page

    def set(self, pool, b, start, rows):
        """rows [G, m, D] into the slots from `start` on."""
        p, r = self.places(b, torch.arange(start, start + rows.shape[1], device=rows.device))
        pool[p, :, r] = rows.transpose(0, 1)

    def get(self, pool, b, m):
        """[G, m, D]: the first m slots."""
        p, r = self.places(b, torch.arange(m, device=pool.device))
        return pool[p, :, r].transpose(0, 1)

    @property
    def tensors(self):
        return self.k, self.v, self.table, self.lengths


def attend(q, rows_k, rows_v, scale=None):
    """q [H, D], rows [G, n, D] -> out [H, D], weights [H, n] and the bound of an fp32 computation's error relative to the sum of
    weighted |v|: a score is a sum of D rounded products (each sum off by at most D half steps of its terms' sizes), and a weight
    follows the difference of two scores; exponentials, sums and weights kept in two halves of 8 bits add 2^-14."""
    H, D = q.shape
    G, n, _ = rows_k.shape
    scale = D ** -0.5 if scale is None else scale
    if n == 0:
        return torch.zeros(H, D, dtype=torch.float64, device=q.device), torch.zeros(H, 0, dtype=torch.float64, device=q.device), 0.0
    k, v = (t.double().repeat_interleave(H // G, 0) for t in (rows_k, rows_v))
    x = torch.einsum("hd,hnd->hn", q.double(), k) * scale
    w = torch.softmax(x, -1)
    size = torch.einsum("hd,hnd->hn", q.double().abs(), k.abs()).max().item() * abs(scale)
    return torch.einsum("hn,hnd->hd", w, v), w, 2 * (D + 2) * 2.0 ** -24 * size + 2.0 ** -14


def check_attention(out, mass, mass_before, q, cache, lengths, scale=None):
    for b, n in enumerate(lengths):
        k, v = cache.get(cache.k, b, n), cache.get(cache.v, b, n)
        want, w, err = attend(q[b], k, v, scale)
        rep = q.shape[1] // cache.G
        spread = torch.einsum("hn,hnd->hd", w, v.double().abs().repeat_interleave(rep, 0)) if n else want.abs()
        tol = HALF_STEP[out.dtype] * (want.abs() + err * spread) + err * spread
        assert ((out[b].double() - want).abs() <= tol).all(), (b, n, (out[b].double() - want).abs().max().item(), tol.min().item())
        if mass is not None:
            add = w.view(cache.G, rep, n).sum(1)
            new = mass_before[b, :, :n].double() + add
            assert ((mass[b, :, :n].double() - new).abs() <= err * add + 2.0 ** -24 * new * (1 + rep)).all(), (b, n)
            assert torch.equal(mass[b, :, n:], mass_before[b, :, n:])


def keep(mass, positions, n, budget, recent, sink):
    """The slots of one head that stay, as the definition sorts them: sure ones, NaN, then by mass, then by slot."""
    newest = max(positions[:n])

    def rank(j):
        if positions[j] < sink or positions[j] > newest - recent:
            return (0, 0.0, j)
        return (1, 0.0, j) if math.isnan(mass[j]) else (2, -mass[j], j)

    return set(sorted(range(n), key=rank)[:budget])


def moves(kept, budget):
    """(from, to) of the slots that move, in order."""
    return list(zip(sorted(j for j in kept if j >= budget), sorted(set(range(budget)) - kept)))
