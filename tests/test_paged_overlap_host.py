"""Tensors that a call on a paged cache writes and that share elements with themselves: refused before anything is launched."""
import ctypes as C

import pytest

from socket_b200 import _lib

A = 1 << 20                                                   # an address nothing on the host reads
B, G, H, D, PAGE, WIDTH = 2, 8, 32, 128, 64, 16
SLOTS = WIDTH * PAGE


def _cache(**over):
    p = _lib.PagedCacheParams()
    for i, name in enumerate(("k", "v", "table", "lengths", "mass", "positions", "status")):
        setattr(p, name, A * (i + 1))
    p.k_rs = p.v_rs = D
    p.k_hs = p.v_hs = PAGE * D
    p.k_ps = p.v_ps = G * PAGE * D
    p.table_ld = p.width = WIDTH
    p.n_pages, p.dtype, p.B, p.G, p.D, p.page = 100, _lib.SK_BF16, B, G, D, PAGE
    p.mass_hs = p.pos_hs = SLOTS
    p.mass_bs = p.pos_bs = G * SLOTS
    for k, v in over.items():
        setattr(p, k, v)
    return p


def _attn(c, o_bs=H * D, o_hs=D):
    return _lib.lib().sk_paged_attn(C.byref(c), A, H * D, D, 2 * A, o_bs, o_hs, H, 0, 0.1, 4 * A, 1 << 40, None)


def _append(c):
    return _lib.lib().sk_paged_append(C.byref(c), A, 4096, 1024, 128, A, 4096, 1024, 128, 4, None, None, None)


def _evict(c, mo=(G * SLOTS, SLOTS), po=(G * SLOTS, SLOTS)):
    return _lib.lib().sk_paged_evict(C.byref(c), 512, 64, 4, A, *mo, A, *po, A, A, 1 << 40, None)


OVERLAPS = [(0, SLOTS), (G * SLOTS, 0), (0, 0), (G * SLOTS, SLOTS - 1), (G * SLOTS - 1, SLOTS), (SLOTS, SLOTS), (SLOTS, 2 * SLOTS - 1)]


def _refused(status):
    assert status == -1 and b"overlap" in _lib.lib().sk_last_error(), (status, _lib.lib().sk_last_error())


@pytest.mark.parametrize("bs,hs", OVERLAPS)
def test_books_that_overlap(bs, hs):
    for call, over in ((_attn, dict(mass_bs=bs, mass_hs=hs)), (_append, dict(mass_bs=bs, mass_hs=hs)), (_append, dict(pos_bs=bs, pos_hs=hs))):
        _refused(call(_cache(**over)))
    _refused(_evict(_cache(), mo=(bs, hs)))
    _refused(_evict(_cache(), po=(bs, hs)))


@pytest.mark.parametrize("bs,hs", [(0, D), (H * D, 0), (0, 0), (H * D, D - 8), (H * D - 8, D), (D, D), (D, 2 * D - 8)])
def test_results_that_overlap(bs, hs):
    _refused(_attn(_cache(), o_bs=bs, o_hs=hs))


@pytest.mark.parametrize("call", [_append, _evict])
@pytest.mark.parametrize("name", ["k", "v"])
@pytest.mark.parametrize("ps,hs,rs", [(0, PAGE * D, D), (G * PAGE * D, 0, D), (G * PAGE * D, PAGE * D, 0), (G * PAGE * D, PAGE * D, D - 8),
                                      (G * PAGE * D - 8, PAGE * D, D), (G * PAGE * D, PAGE * D - 8, D), (G * PAGE * D, D, D), (PAGE * D, D, PAGE * D)])
def test_pools_that_overlap(call, name, ps, hs, rs):
    _refused(call(_cache(**{f"{name}_ps": ps, f"{name}_hs": hs, f"{name}_rs": rs})))
