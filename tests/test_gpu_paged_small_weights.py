"""Attention over pages where most keys' weights are small beside a few: what they add up to is not lost."""
import pytest
import torch

from tests.paged_util import HALF_STEP, Cache, attend
from socket_b200 import paged

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.bfloat16, torch.float16, torch.float32]
LOWEST_STEP = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}          # half a step of the type's subnormals


def _sink(c, b, at, gap, q, value):
    """Key `at` of sequence b scores `gap` above nought with the first query of every key/value head, its values are `value`."""
    n = int(c.lengths[b])
    k, v = c.get(c.k, b, n).clone(), c.get(c.v, b, n).clone()
    first = q[b, ::q.shape[1] // c.G].float()
    k[:, at] = (first * (gap * c.D ** 0.5 / (first * first).sum(-1, keepdim=True))).to(k.dtype)
    v[:, at] = value
    c.set(c.k, b, 0, k)
    c.set(c.v, b, 0, v)


def _case(lengths, G, rep, D, dtype, gap, at, equal, value=0.0, spread=0.3):
    c = Cache(lengths, G, D, 16, dtype, DEV, seed=D + rep)
    g = torch.Generator(device=DEV).manual_seed(7)
    one = torch.randn(len(lengths), G, 1, D, generator=g, device=DEV)
    # query heads of one key/value head that lean the same way, so that the key is far above for all of them
    q = (one + spread * torch.randn(len(lengths), G, rep, D, generator=g, device=DEV)).flatten(1, 2).to(dtype)
    for b, n in enumerate(lengths):
        k, v = c.get(c.k, b, n) * 0.1, c.get(c.v, b, n).abs() * 100 + 900        # values that do not cancel
        if equal:
            k = k[:, :1].expand_as(k)
        c.set(c.k, b, 0, k.to(dtype))
        c.set(c.v, b, 0, v.to(dtype))
        if n > at:
            _sink(c, b, at, gap, q, value)
    mass = torch.zeros(len(lengths), G, c.cap, device=DEV)
    for collected in (None, mass):
        out = paged.attn(q, *c.tensors, mass=collected)
        for b, n in enumerate(lengths):
            k, v = c.get(c.k, b, n), c.get(c.v, b, n)
            want, w, err = attend(q[b], k, v)
            weighted = torch.einsum("hn,hnd->hd", w, v.double().abs().repeat_interleave(rep, 0))
            tol = (1 + HALF_STEP[dtype]) * err * weighted + HALF_STEP[dtype] * want.abs() + LOWEST_STEP[dtype]
            off = (out[b].double() - want).abs()
            assert (off <= tol).all(), (b, n, (off / want.abs().clamp_min(1e-30)).max().item(), (tol / want.abs().clamp_min(1e-30)).max().item())
    for b, n in enumerate(lengths):
        _, w, err = attend(q[b], c.get(c.k, b, n), c.get(c.v, b, n))
        add = w.view(G, rep, n).sum(1)
        assert ((mass[b, :, :n].double() - add).abs() <= (err + 2.0 ** -24 * (1 + rep)) * add + rep * 2.0 ** -126).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("equal", [False, True])
@pytest.mark.parametrize("gap", [5.0, 10.0, 12.0, 15.0, 17.3, 18.0, 22.0, 30.0, 45.0])
def test_many_small_weights_behind_a_large_one(gap, equal, dtype):
    """A key far above all others whose value is nought: the result is what the others add up to."""
    _case([8192, 40, 16, 200], 2, 4, 64, dtype, gap, 0, equal)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("G,rep,D", [(8, 1, 128), (2, 8, 128), (1, 16, 64), (1, 12, 256), (4, 4, 96), (1, 20, 128)])
@pytest.mark.parametrize("at", [0, 77, 699])
def test_small_weights_of_other_heads(at, G, rep, D, dtype):
    _case([700, 3000], G, rep, D, dtype, 17.3, at, False)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("gap,value", [(17.5, 0.0), (18.0, 1.0), (24.0, 0.0)])
def test_small_weights_of_a_long_cache(gap, value, dtype):
    _case([131072], 1, 4, 128, dtype, gap, 0, True, value)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [1e3, 1e5, 3e6, 3e7, 6e7, 1e8, 2e8, 5e8, 2e9])
def test_huge_scores_give_weights_all_the_same(size, dtype):
    """Scores so large that fp32 has them in steps of up to 256: whatever they round to, weights are at most one and add up to one, so
    a result is finite and lies among the values."""
    lengths = [1, 16, 17, 300, 3000]
    c = Cache(lengths, 1, 64, 16, dtype, DEV, seed=2)
    g = torch.Generator(device=DEV).manual_seed(3)
    q = torch.zeros(len(lengths), 4, 64, device=DEV)
    q[..., 0], q[..., 1] = size / 6e4, 1.0                    # keys differ by what their second column adds: less than a step, or a few
    for b, n in enumerate(lengths):
        k = torch.zeros(1, n, 64, device=DEV)
        k[..., 0], k[..., 1] = 6e4, torch.randint(-60, 60, (1, n), generator=g, device=DEV).float()
        c.set(c.k, b, 0, k.to(dtype))
    mass = torch.zeros(len(lengths), 1, c.cap, device=DEV)
    out = paged.attn(q.to(dtype), *c.tensors, scale=1.0, mass=mass)
    for b, n in enumerate(lengths):
        v = c.get(c.v, b, n)[0].double()
        low, high = v.amin(0) - 2.0 ** -7 * v.abs().amax(0), v.amax(0) + 2.0 ** -7 * v.abs().amax(0)
        assert ((out[b].double() >= low) & (out[b].double() <= high)).all()
        assert (mass[b] >= 0).all() and (mass[b].sum() - 4).abs() <= 4 * (n + 64) * 2.0 ** -23
