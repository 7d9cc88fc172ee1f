"""One sequence, one token, one head: the stride of a dimension of one says nothing, whatever it is."""
import pytest
import torch

from tests.paged_util import Cache, check_attention
from socket_b200 import paged

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _odd(t, *dims):
    """t with strides of 3 elements for its dimensions of one."""
    assert all(t.shape[d] == 1 for d in dims)
    return t.as_strided(t.shape, [3 if d in dims else s for d, s in enumerate(t.stride())], t.storage_offset())


@pytest.mark.parametrize("dtype", TYPES)
def test_one_sequence_of_one_head(dtype):
    plain, odd = (Cache([70], 1, 64, 16, dtype, DEV, room=1) for _ in range(2))
    odd.k, odd.v, odd.table = _odd(odd.k, 1), _odd(odd.v, 1), _odd(odd.table, 0)
    q, new = torch.randn(1, 1, 64, device=DEV).to(dtype), torch.randn(1, 1, 1, 64, device=DEV).to(dtype)
    mass, positions = torch.rand(1, 1, plain.cap, device=DEV), torch.randperm(plain.cap, device=DEV).to(torch.int32).view(1, 1, -1)
    got = []
    for c, turn in ((plain, lambda t, *d: t.clone()), (odd, lambda t, *d: _odd(t.clone(), *d))):
        m, p, out = turn(mass, 0, 1), turn(positions, 0, 1), turn(torch.empty_like(q), 0, 1)
        paged.append(turn(new, 0, 1, 2), turn(new, 0, 1, 2), *c.tensors, mass=m, positions=p)
        paged.attn(turn(q, 0, 1), *c.tensors, extra=1, mass=m, out=out)
        check_attention(out, None, None, q, c, [71])
        cut = paged.evict(*c.tensors, m, p, budget=40, recent=3, out=(turn(m, 0, 1), turn(p, 0, 1), torch.empty_like(c.lengths)))
        got.append((out, m, p, *cut, c.get(c.k, 0, 40), c.get(c.v, 0, 40)))
    for a, b in zip(*got):
        assert torch.equal(a, b)


def test_one_sequence_of_wider_rows():
    """The first of two sequences' projections, which stand side by side with a few more elements behind them."""
    c = Cache([200], 2, 64, 16, torch.bfloat16, DEV, room=1)
    wide = torch.randn(2, (4 + 2 + 2) * 64 + 5, device=DEV).bfloat16()
    q, k, v = (wide[:, a * 64:b * 64].unflatten(1, (b - a, 64))[:1] for a, b in ((0, 4), (4, 6), (6, 8)))
    assert q.stride(0) % 8
    paged.append(k.unsqueeze(1), v.unsqueeze(1), *c.tensors)
    check_attention(paged.attn(q, *c.tensors, extra=1), None, None, q, c, [201])
    assert torch.equal(c.get(c.k, 0, 201)[:, 200], k[0]) and torch.equal(c.get(c.v, 0, 201)[:, 200], v[0])
