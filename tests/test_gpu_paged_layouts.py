"""Layouts of what a paged cache's calls write: any order of dimensions, but no element twice."""
import pytest
import torch

from tests.paged_util import Cache, check_attention
from socket_b200 import _lib, paged

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _cache():
    return Cache([150, 40, 90], 2, 64, 16, torch.bfloat16, DEV, room=2)


def _books(c):
    return torch.rand(3, 2, c.cap, device=DEV), torch.stack([torch.randperm(c.cap, device=DEV) for _ in range(6)]).view(3, 2, c.cap).to(torch.int32)


def _bits(t):
    return t.contiguous().view(torch.int16)


def _turned(t):
    """A copy with the heads outermost."""
    return t.transpose(0, 1).clone(memory_format=torch.contiguous_format).transpose(0, 1)


def test_heads_outermost():
    """Pools, books and results whose heads are the outermost dimension: the same as in the usual order."""
    plain, turned = _cache(), _cache()
    turned.k, turned.v = _turned(turned.k), _turned(turned.v)
    q, new = torch.randn(3, 4, 64, device=DEV).bfloat16(), torch.randn(3, 2, 2, 64, device=DEV).bfloat16()
    mass, positions = _books(plain)
    got = []
    for c, order in ((plain, torch.clone), (turned, _turned)):
        m, p, out = order(mass), order(positions), order(torch.empty_like(q))
        paged.append(new, new, *c.tensors, mass=m, positions=p)
        paged.attn(q, *c.tensors, extra=2, mass=m, out=out)
        cut = paged.evict(*c.tensors, m, p, budget=60, recent=8, sink=2, out=(order(m), order(p), torch.empty_like(c.lengths)))
        got.append((out, m, p, *cut))
    for a, b in zip(*got):
        assert torch.equal(a, b)
    assert torch.equal(_bits(plain.k), _bits(turned.k)) and torch.equal(_bits(plain.v), _bits(turned.v))


def test_what_is_only_read_may_be_expanded():
    c = _cache()
    mass, positions = _books(c)
    mass, positions = mass[:, :1].expand(3, 2, c.cap), positions[:, :1].expand(3, 2, c.cap)
    k, v = c.k.clone(), c.v.clone()
    got = paged.evict(k, v, c.table, c.lengths, mass, positions, budget=30)
    want = paged.evict(*c.tensors, mass.contiguous(), positions.contiguous(), budget=30)
    for a, b in zip((*got, _bits(k), _bits(v)), (*want, _bits(c.k), _bits(c.v))):
        assert torch.equal(a, b)
    q = torch.randn(3, 4, 64, device=DEV).bfloat16()
    pool = torch.randn(1, 1, 16, 64, device=DEV).bfloat16().expand(3, 2, 16, 64)
    c = Cache([16, 5, 9], 2, 64, 16, torch.bfloat16, DEV, width=1)
    c.k, c.v, c.table = pool, pool, torch.tensor([[0], [2], [1]], dtype=torch.int32, device=DEV)
    check_attention(paged.attn(q, *c.tensors), None, None, q, c, [16, 5, 9])


def test_what_is_written_must_not_be_expanded():
    c = _cache()
    mass, positions = _books(c)
    q, new = torch.randn(3, 4, 64, device=DEV).bfloat16(), torch.randn(3, 2, 2, 64, device=DEV).bfloat16()
    out = torch.empty_like(c.lengths)
    for refused in (lambda: paged.attn(q, *c.tensors, out=q[:, :1].expand(3, 4, 64)),
                    lambda: paged.attn(q, *c.tensors, out=q[:1].expand(3, 4, 64)),
                    lambda: paged.attn(q, *c.tensors, mass=mass[:1].expand(3, 2, c.cap)),
                    lambda: paged.append(new, new, *c.tensors, mass=mass[:, :1].expand(3, 2, c.cap)),
                    lambda: paged.append(new, new, *c.tensors, positions=positions[:1].expand(3, 2, c.cap)),
                    lambda: paged.append(new, new, c.k[:, :1].expand_as(c.k), c.v, c.table, c.lengths),
                    lambda: paged.evict(c.k, c.v[:1].expand_as(c.v), c.table, c.lengths, mass, positions, budget=30),
                    lambda: paged.evict(*c.tensors, mass, positions, budget=30, out=(mass[:, :1].expand(3, 2, c.cap), positions, out)),
                    lambda: paged.evict(*c.tensors, mass, positions, budget=30, out=(mass, positions[:1].expand(3, 2, c.cap), out))):
        with pytest.raises(_lib.SocketError, match="overlap"):
            refused()
