"""The paged cache's operators against plain forms in 64 bits, at the sizes and contents where they can go wrong."""
import math

import pytest
import torch

from tests.paged_util import Cache, attend, check_attention, keep, moves
from socket_b200 import _lib, paged

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.bfloat16, torch.float16, torch.float32]
LENGTHS = [0, 1, 15, 16, 17, 127, 128, 129, 300, 2049]


def _flag():
    return torch.zeros(1, dtype=torch.int32, device=DEV)


def _run(c, H, mass=False, seed=1, q_scale=1.5, **kw):
    g = torch.Generator(device=DEV).manual_seed(seed)
    q = (torch.randn(len(c.rows_k), H, c.D, generator=g, device=DEV) * q_scale).to(c.k.dtype)
    m = torch.rand(len(c.rows_k), c.G, c.cap, generator=g, device=DEV) if mass else None
    before = None if m is None else m.clone()
    flag = _flag()
    out = paged.attn(q, *c.tensors, mass=m, status=flag, **kw)
    assert int(flag) == 0
    return q, out, m, before


# ------------------------------------------------------------------------------------------- attention
@pytest.mark.parametrize("mass", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,G,D", [(8, 8, 128), (8, 2, 64), (32, 8, 128), (8, 1, 256), (16, 1, 128), (12, 4, 96), (6, 2, 8), (20, 1, 72), (34, 1, 64)])
def test_attention(H, G, D, dtype, mass):
    c = Cache(LENGTHS, G, D, 16, dtype, DEV, seed=D + H)
    q, out, m, before = _run(c, H, mass)
    check_attention(out, m, before, q, c, LENGTHS)


@pytest.mark.parametrize("D", [4, 12, 100, 132, 252])
def test_attention_of_fp32_heads_of_odd_sizes(D):
    c = Cache(LENGTHS, 2, D, 16, torch.float32, DEV, seed=D)
    q, out, m, before = _run(c, 10, True)
    check_attention(out, m, before, q, c, LENGTHS)


@pytest.mark.parametrize("scale", [-0.7, 0.0, 3.0])
def test_attention_scales(scale):
    c = Cache(LENGTHS, 2, 64, 32, torch.float16, DEV)
    q, out, m, before = _run(c, 6, True, scale=scale)
    check_attention(out, m, before, q, c, LENGTHS, scale=scale)


def test_queries_and_new_rows_that_are_expanded():
    """One query for every sequence, one new row for every head."""
    c = Cache([70, 5, 300], 2, 64, 16, torch.bfloat16, DEV, room=3)
    q = torch.randn(1, 4, 64, device=DEV).bfloat16().expand(3, 4, 64)
    out = paged.attn(q, *c.tensors)
    check_attention(out, None, None, q, c, [70, 5, 300])
    new = torch.randn(3, 1, 1, 64, device=DEV).bfloat16().expand(3, 3, 2, 64)
    paged.append(new, new, *c.tensors)
    for b, n in enumerate((70, 5, 300)):
        assert torch.equal(c.get(c.k, b, n + 3)[:, n:], new[b].transpose(0, 1)) and torch.equal(c.get(c.v, b, n + 3)[:, n:], new[b].transpose(0, 1))


@pytest.mark.parametrize("page", [16, 32, 64, 128, 512])
@pytest.mark.parametrize("lengths", [[1], [7, 0, 0, 3], [5000], [0, 0], [3000, 1, 2999, 130, 0, 64]])
def test_attention_pages(page, lengths):
    c = Cache(lengths, 2, 128, page, torch.bfloat16, DEV)
    q, out, m, before = _run(c, 8, True)
    check_attention(out, m, before, q, c, lengths)


@pytest.mark.parametrize("mass", [False, True])
@pytest.mark.parametrize("n", [30001, 131072])
def test_attention_long(n, mass):
    c = Cache([n, 5, n // 3], 2, 128, 64, torch.bfloat16, DEV)
    q, out, m, before = _run(c, 8, mass)
    check_attention(out, m, before, q, c, [n, 5, n // 3])


def test_attention_many_short_sequences():
    lengths = [(7 * i) % 200 for i in range(700)]
    c = Cache(lengths, 2, 64, 32, torch.float16, DEV)
    q, out, m, before = _run(c, 8, True)
    check_attention(out, m, before, q, c, lengths)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_of_strided_tensors(dtype):
    """Keys and values of a page side by side and heads inside its rows; queries and results inside wider rows; a wider table."""
    lengths = [70, 0, 333]
    c = Cache(lengths, 4, 64, 32, dtype, DEV, combined=True)
    wide = torch.randn(3, 8 + 2, 64 + 16, device=DEV).to(dtype)
    q = wide[:, 1:9, 16:]
    out = torch.full((3, 8, 2, 64), 7.0, dtype=dtype, device=DEV)
    table = torch.full((3, c.width + 5), -1, dtype=torch.int32, device=DEV)
    table[:, :c.width] = c.table
    m = torch.rand(3, 4, c.cap + 9, device=DEV)
    before = m.clone()
    paged.attn(q, c.k, c.v, table[:, :c.width], c.lengths, out=out[:, :, 0], mass=m)
    check_attention(out[:, :, 0], m, before, q, c, lengths)
    assert (out[:, :, 1] == 7).all()


def test_sequences_without_pages():
    """A table without columns, a pool without pages, no sequences: nothing to attend to, nothing to move."""
    k = torch.empty(0, 2, 16, 64, dtype=torch.bfloat16, device=DEV)
    table, n = torch.empty(3, 0, dtype=torch.int32, device=DEV), torch.tensor([0, -2, 0], dtype=torch.int32, device=DEV)
    q, mass, pos = torch.randn(3, 4, 64, device=DEV).bfloat16(), torch.empty(3, 2, 0, device=DEV), torch.empty(3, 2, 0, dtype=torch.int32, device=DEV)
    flag = _flag()
    for m in (None, mass):
        assert (paged.attn(q, k, k, table, n, mass=m, status=flag) == 0).all()
    assert paged.evict(k, k, table, n, mass, pos, budget=4, status=flag)[2].tolist() == [0, 0, 0] and int(flag) == 0
    assert (paged.attn(q, k, k, table, n, extra=1, status=flag) == 0).all() and int(flag) == _lib.SK_DEV_POS_OUT_OF_RANGE
    c = Cache([5], 2, 64, 16, torch.bfloat16, DEV)
    none = (c.k, c.v, c.table[:0], c.lengths[:0])
    assert paged.attn(q[:0], *none).shape == (0, 4, 64)
    paged.append(q[:0, None, :2], q[:0, None, :2], *none)
    books = torch.empty(0, 2, c.cap, device=DEV), torch.empty(0, 2, c.cap, dtype=torch.int32, device=DEV)
    assert paged.evict(*none, *books, budget=4)[2].shape == (0,)


def test_results_in_place_of_the_queries():
    c = Cache([3000, 40, 129, 7], 2, 128, 16, torch.bfloat16, DEV)
    q, out, m, before = _run(c, 8, False)
    assert paged.attn(q, *c.tensors, out=q) is q and torch.equal(q, out)


def test_attention_extra_and_scale():
    c = Cache([40, 1, 0], 2, 64, 16, torch.float32, DEV, room=2)
    for b in range(3):
        c.set(c.k, b, int(c.lengths[b]), torch.randn(2, 2, 64, device=DEV))
        c.set(c.v, b, int(c.lengths[b]), torch.randn(2, 2, 64, device=DEV))
    q, out, m, before = _run(c, 4, True, extra=2, scale=0.3)
    check_attention(out, m, before, q, c, [42, 3, 2], scale=0.3)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_of_extreme_scores(dtype):
    """One key far above all others, all keys equal, scores that underflow: weights stay exact."""
    c = Cache([200, 200, 200], 1, 64, 16, dtype, DEV)
    big = c.get(c.k, 0, 200).clone()
    big[0, 137] *= 30
    c.set(c.k, 0, 0, big)
    c.set(c.k, 1, 0, c.get(c.k, 1, 1).expand(1, 200, 64).contiguous())
    q, out, m, before = _run(c, 4, True, q_scale=8.0)
    check_attention(out, m, before, q, c, [200, 200, 200])


def test_infinite_and_nan_inputs_stay_in_their_rows():
    c = Cache([100, 100, 100], 2, 64, 16, torch.bfloat16, DEV)
    q = torch.randn(3, 4, 64, device=DEV).bfloat16()
    clean = paged.attn(q, *c.tensors)
    q[1, 2, 5] = float("nan")
    v = c.get(c.v, 2, 100).clone()
    v[1, 50, 3] = float("inf")
    c.set(c.v, 2, 0, v)
    out = paged.attn(q, *c.tensors)
    assert torch.equal(out[0], clean[0]) and torch.equal(out[1, [0, 1, 3]], clean[1, [0, 1, 3]]) and out[1, 2].isnan().all()
    assert torch.equal(out[2, :2], clean[2, :2]) and not out[2, 2:, 3].isfinite().any()
    rest = [i for i in range(64) if i != 3]
    assert torch.equal(out[2, 2:, rest], clean[2, 2:, rest])


def test_attention_leaves_out_bad_pages_and_cuts_long_lengths():
    c = Cache([100, 64, 30], 2, 64, 16, torch.bfloat16, DEV)
    c.table[0, 2] = c.k.shape[0]                              # 16 keys without a page
    c.table[2, 0] = -1
    c.lengths[1] = c.cap + 1000
    fill = torch.randn(2, c.cap, 64, device=DEV).bfloat16()
    c.set(c.k, 1, 0, fill)
    c.set(c.v, 1, 0, fill)
    q, flag = torch.randn(3, 4, 64, device=DEV).bfloat16(), _flag()
    mass = torch.zeros(3, 2, c.cap, device=DEV)
    out = paged.attn(q, *c.tensors, mass=mass, status=flag)
    assert int(flag) == _lib.SK_DEV_INDEX_OUT_OF_RANGE | _lib.SK_DEV_POS_OUT_OF_RANGE
    left = [[j for j in range(100) if j // 16 != 2], list(range(c.cap)), list(range(16, 30))]
    for b, keys in enumerate(left):
        n = max(keys) + 1
        safe = c.table.clone()
        c.table.clamp_(0, c.k.shape[0] - 1)
        k, v = c.get(c.k, b, n)[:, keys], c.get(c.v, b, n)[:, keys]
        c.table.copy_(safe)
        want, w, _ = attend(q[b], k, v)
        assert (out[b].double() - want).abs().max() < 2.0 ** -8 * want.abs().max() + 1e-3
        assert (mass[b][:, keys].double() - w.view(2, 2, -1).sum(1)).abs().max() < 1e-4
        gone = [j for j in range(c.cap) if j not in keys]
        assert (mass[b][:, gone] == 0).all()
    assert int(_flag()) == 0 and torch.equal(paged.attn(q, *c.tensors), out)      # without a status word too


def test_attention_behind_32_bit_offsets():
    """Pools of 2^31 elements and more."""
    page, G, D = 64, 8, 128
    n = 2 ** 31 // (page * G * D) + 70
    k, v = (torch.empty(n, G, page, D, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    table = torch.arange(n - 5, n, dtype=torch.int32, device=DEV).view(1, 5)
    for pool in (k, v):
        pool[-5:].normal_()
    c = Cache([300], G, D, page, torch.bfloat16, DEV)
    c.k, c.v, c.table, c.lengths = k, v, table, torch.tensor([300], dtype=torch.int32, device=DEV)
    q, out, m, before = _run(c, 32, True)
    check_attention(out, m, before, q, c, [300])
    new = torch.randn(1, 2, G, D, device=DEV).bfloat16()
    paged.append(new, new, *c.tensors)
    assert torch.equal(k[n - 1, :, 44:46], new[0].transpose(0, 1)) and torch.equal(v[n - 1, :, 44:46], new[0].transpose(0, 1))


def test_attention_is_the_same_every_time_and_on_other_streams():
    c = Cache([5000, 17, 900], 2, 128, 16, torch.bfloat16, DEV)
    q, out, m, before = _run(c, 8, True)
    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        m2 = before.clone()
        again = paged.attn(q, *c.tensors, mass=m2)
    side.synchronize()
    assert torch.equal(again, out) and torch.equal(m2, m)


def test_attention_with_its_own_workspace():
    c = Cache([5000, 17], 2, 128, 16, torch.bfloat16, DEV)
    q, out, m, before = _run(c, 8, True)
    need = paged.attn_workspace(8, *c.tensors, mass=before)
    for ws in (torch.full((need,), 255, dtype=torch.uint8, device=DEV), torch.zeros(3, dtype=torch.uint8, device=DEV)):
        m2 = before.clone()
        assert torch.equal(paged.attn(q, *c.tensors, mass=m2, workspace=ws), out) and torch.equal(m2, m)


def test_refused_tensors():
    c = Cache([40, 9], 2, 64, 16, torch.float16, DEV)
    q = torch.randn(2, 4, 64, device=DEV).half()
    mass, pos = torch.zeros(2, 2, c.cap, device=DEV), torch.zeros(2, 2, c.cap, dtype=torch.int32, device=DEV)
    need = 65536                                              # without weights so short a batch needs none: an empty one would be contiguous
    for ws in (torch.zeros(1, dtype=torch.uint8, device=DEV).expand(need), torch.zeros(2 * need, dtype=torch.uint8, device=DEV)[::2]):
        with pytest.raises(AssertionError):                    # fewer bytes, or others, than it counts
            paged.attn(q, *c.tensors, workspace=ws)
    for refused in (lambda: paged.attn(q.float(), *c.tensors), lambda: paged.attn(q[:1], *c.tensors), lambda: paged.attn(q[:, :3], *c.tensors),
                    lambda: paged.attn(q, *c.tensors, mass=mass[..., :-1]), lambda: paged.attn(q, *c.tensors, mass=mass.double()),
                    lambda: paged.attn(q, c.k, c.v, c.table.long(), c.lengths), lambda: paged.attn(q, c.k, c.v, c.table, c.lengths[:1]),
                    lambda: paged.append(q[:, None], q[:, None], *c.tensors), lambda: paged.evict(*c.tensors, mass, pos.long(), budget=8),
                    lambda: paged.evict(*c.tensors, mass, pos, budget=8, out=(mass, pos, c.lengths.long()))):
        with pytest.raises(AssertionError):
            refused()
    for refused in (lambda: paged.evict(*c.tensors, mass, pos, budget=0), lambda: paged.attn(q, *c.tensors, extra=-1)):
        with pytest.raises(_lib.SocketError):
            refused()
    with pytest.raises(RuntimeError):
        paged.attn(q.cpu(), *c.tensors)


def test_two_captured_steps_that_replay_together():
    """Two graphs of append and attention on two streams, replayed while lengths grow: every replay is a fresh call's result."""
    caches = [Cache([600, 31], 2, 64, 16, torch.bfloat16, DEV, room=8, seed=i) for i in range(2)]
    steps = []
    for i, c in enumerate(caches):
        q, new = torch.randn(2, 4, 64, device=DEV).bfloat16(), torch.randn(2, 1, 2, 64, device=DEV).bfloat16()
        m = torch.zeros(2, 2, c.cap, device=DEV)
        paged.attn(q, *c.tensors, extra=1, mass=m)
        m.zero_()
        side = torch.cuda.Stream(DEV)
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            paged.append(new, new, *c.tensors, mass=m)
            out = paged.attn(q, *c.tensors, extra=1, mass=m)
            c.lengths.add_(1)
        steps.append((graph, side, q, new, m, out, c))
    torch.cuda.synchronize()
    want = []
    for graph, side, q, new, m, out, c in steps:              # what eager calls give, on copies
        k, v, n, mm, outs = c.k.clone(), c.v.clone(), c.lengths.clone(), torch.zeros_like(m), None
        for _ in range(5):
            paged.append(new, new, k, v, c.table, n, mass=mm)
            outs = paged.attn(q, k, v, c.table, n, extra=1, mass=mm)
            n += 1
        want.append((outs, mm, n))
    torch.cuda.synchronize()
    for _ in range(5):
        for graph, side, *_ in steps:
            with torch.cuda.stream(side):
                graph.replay()
    torch.cuda.synchronize()
    for (graph, side, q, new, m, out, c), (outs, mm, n) in zip(steps, want):
        assert torch.equal(out, outs) and torch.equal(m, mm) and torch.equal(c.lengths, n)


# ------------------------------------------------------------------------------------------- append
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("G,D,page,S", [(8, 128, 64, 1), (2, 64, 16, 37), (1, 256, 128, 200), (3, 8, 16, 5), (4, 96, 32, 65)])
def test_append(G, D, page, S, dtype):
    lengths, counts = [0, 15, 16, 100], [S, max(S - 3, 0), 1, S // 2]
    c = Cache(lengths, G, D, page, dtype, DEV, room=S)
    wide = torch.randn(4, S, 2 * G + 1, D, device=DEV).to(dtype)
    k_new, v_new = wide[:, :, :G], wide[:, :, G + 1:]
    k, v = c.k.clone(), c.v.clone()
    mass, positions = torch.rand(4, G, c.cap, device=DEV), torch.randint(0, 99, (4, G, c.cap), dtype=torch.int32, device=DEV)
    m, p = mass.clone(), positions.clone()
    first = torch.tensor([5, 1000, 7, 2 ** 30], dtype=torch.int32, device=DEV)
    flag = _flag()
    for n, f in ((None, None), (torch.tensor(counts, dtype=torch.int32, device=DEV), first)):
        paged.append(k_new, v_new, *c.tensors, counts=n, first=f, positions=positions, mass=mass, status=flag)
        for b in range(4):
            now = S if n is None else counts[b]
            pg, r = c.places(b, torch.arange(lengths[b], lengths[b] + now, device=DEV))
            k[pg, :, r], v[pg, :, r] = k_new[b, :now], v_new[b, :now]
            m[b, :, lengths[b]:lengths[b] + now] = 0
            at = lengths[b] if f is None else int(first[b])
            p[b, :, lengths[b]:lengths[b] + now] = torch.arange(at, at + now, device=DEV)
        as_bits = torch.int32 if dtype == torch.float32 else torch.int16
        assert torch.equal(c.k.view(as_bits), k.view(as_bits)) and torch.equal(c.v.view(as_bits), v.view(as_bits))
        assert torch.equal(mass, m) and torch.equal(positions, p)
    assert int(flag) == 0


def test_append_outside_the_cache():
    c = Cache([30, 32, 5, 0], 1, 64, 16, torch.bfloat16, DEV, width=2)
    c.lengths[3] = -4                                         # counts as empty
    c.table[2, 0] = c.k.shape[0]
    new = torch.randn(4, 4, 1, 64, device=DEV).bfloat16()
    k, flag = c.k.clone(), _flag()
    paged.append(new, new, *c.tensors, counts=torch.tensor([4, 1, 2, 99], dtype=torch.int32, device=DEV), status=flag)
    assert int(flag) == _lib.SK_DEV_INDEX_OUT_OF_RANGE | _lib.SK_DEV_POS_OUT_OF_RANGE
    k[int(c.table[0, 1]), 0, 14:] = new[0, :2, 0]
    k[int(c.table[3, 0]), 0, :4] = new[3, :, 0]
    assert torch.equal(c.k.view(torch.int16), k.view(torch.int16))
    paged.append(new, new, *c.tensors, counts=torch.tensor([0, -1, 0, 0], dtype=torch.int32, device=DEV))
    assert torch.equal(c.k.view(torch.int16), k.view(torch.int16))


# ------------------------------------------------------------------------------------------- eviction
def _check_evict(c, lengths, mass, positions, budget, recent, sink, got, k_before, v_before):
    m2, p2, n2 = (t.cpu() for t in got)
    mass, positions, table = mass.cpu(), positions.cpu(), c.table.cpu()
    want_k, want_v = k_before.clone(), v_before.clone()
    to, frm = [], []
    for b, n in enumerate(lengths):
        assert int(n2[b]) == min(n, budget)
        for g in range(c.G):
            m, p = mass[b, g].tolist(), positions[b, g].tolist()
            if n > budget:
                for f, t in moves(keep(m, p, n, budget, recent, sink), budget):
                    m[t], p[t] = m[f], p[f]
                    frm.append((int(table[b, f // c.page]), g, f % c.page))
                    to.append((int(table[b, t // c.page]), g, t % c.page))
            n_new = min(n, budget)
            new_m, new_p = m[:n_new] + [0.0] * (c.cap - n_new), p[:n_new] + [-1] * (c.cap - n_new)
            assert p2[b, g, :c.cap].tolist() == new_p
            torch.testing.assert_close(m2[b, g, :c.cap], torch.tensor(new_m), rtol=0, atol=0, equal_nan=True)
    if to:
        to, frm = torch.tensor(to, device=DEV).T, torch.tensor(frm, device=DEV).T
        for want, before in ((want_k, k_before), (want_v, v_before)):
            want[to[0], to[1], to[2]] = before[frm[0], frm[1], frm[2]]
    bits = torch.int32 if c.k.dtype == torch.float32 else torch.int16
    assert torch.equal(c.k.contiguous().view(bits), want_k.contiguous().view(bits))
    assert torch.equal(c.v.contiguous().view(bits), want_v.contiguous().view(bits))


def _evict_case(lengths, G, D, page, dtype, budget, recent, sink, fill, seed=0, in_place=False, combined=False, room=0):
    c = Cache(lengths, G, D, page, dtype, DEV, seed=seed, combined=combined, room=room)
    g = torch.Generator(device=DEV).manual_seed(seed + 1)
    shape = (len(lengths), G, c.cap)
    mass = {"random": lambda: torch.rand(shape, generator=g, device=DEV), "equal": lambda: torch.full(shape, 0.25, device=DEV),
            "zero": lambda: torch.zeros(shape, device=DEV) * torch.where(torch.rand(shape, generator=g, device=DEV) < 0.5, -1.0, 1.0),
            "few": lambda: torch.randint(0, 3, shape, generator=g, device=DEV).float() * 1e-30,
            "odd": lambda: torch.where(torch.rand(shape, generator=g, device=DEV) < 0.1,
                                       torch.tensor([math.nan, math.inf, -math.inf, -1.0], device=DEV)[torch.randint(0, 4, shape, generator=g, device=DEV)],
                                       torch.rand(shape, generator=g, device=DEV))}[fill]()
    positions = torch.stack([torch.randperm(c.cap, generator=g, device=DEV) for _ in range(shape[0] * G)]).view(shape).to(torch.int32)
    k, v, m, p = c.k.clone(), c.v.clone(), mass.clone(), positions.clone()
    out = (m, p, c.lengths) if in_place else None
    flag = _flag()
    got = paged.evict(c.k, c.v, c.table, c.lengths, m, p, budget=budget, recent=recent, sink=sink, out=out, status=flag)
    assert int(flag) == 0
    _check_evict(c, lengths, mass, positions, budget, recent, sink, got, k, v)
    if not in_place:
        assert torch.equal(p, positions) and torch.equal(m.nan_to_num(7.0), mass.nan_to_num(7.0)) and c.lengths.tolist() == lengths


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("fill", ["random", "equal", "zero", "few", "odd"])
@pytest.mark.parametrize("budget,recent,sink", [(1, 0, 0), (1, 1, 0), (16, 4, 2), (100, 100, 0), (100, 0, 100), (333, 50, 3), (2000, 10, 4)])
def test_evict(budget, recent, sink, fill, in_place):
    _evict_case([0, 1, 17, 100, 101, 640, 1500], 2, 64, 16, torch.bfloat16, budget, recent, sink, fill, budget, in_place)


@pytest.mark.parametrize("G,D,page,dtype,combined", [(8, 128, 64, torch.float16, False), (1, 256, 128, torch.float32, False),
                                                    (3, 8, 16, torch.bfloat16, True), (4, 96, 32, torch.float32, True)])
def test_evict_layouts(G, D, page, dtype, combined):
    _evict_case([700, 699, 350], G, D, page, dtype, 350, 40, 4, "random", D, combined=combined)


@pytest.mark.parametrize("n,budget", [(20000, 1000), (33000, 32000), (70001, 4096), (131072, 2), (140000, 139999)])
@pytest.mark.parametrize("fill", ["random", "few"])
def test_evict_long(n, budget, fill):
    _evict_case([n, n // 2], 2, 8, 64, torch.bfloat16, budget, min(100, budget // 2), 1, fill)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("lengths,budget", [([410000, 7], 100000), ([400, 70000] + [3] * 22, 350)])
@pytest.mark.parametrize("fill", ["random", "few"])
def test_evict_slots_without_room_on_chip(lengths, budget, fill, in_place):
    """More slots than sixteen blocks hold; more sequences than find a place at once, with tables as wide."""
    room = max(0, 200000 - max(lengths))
    _evict_case(lengths, 1, 8, 64, torch.bfloat16, budget, 100, 1, fill, in_place=in_place, room=room)


@pytest.mark.parametrize("n,over", [(600, 0), (600, 1), (600, -1), (20000, 0), (20000, 1), (20000, -1)])
@pytest.mark.parametrize("byte", [3, 2, 1, 0])
@pytest.mark.parametrize("base", [0x00000000, 0x3E123455])
def test_evict_cut_between_bytes(base, byte, n, over):
    """Two masses that differ in one byte, the larger ones as many as the budget, one more or one fewer."""
    c = Cache([n], 2, 8, 64, torch.bfloat16, DEV, seed=byte)
    g = torch.Generator(device=DEV).manual_seed(byte)
    large = torch.rand(1, 2, c.cap, generator=g, device=DEV).argsort(-1) < n // 3
    large[..., n:] = False
    budget = int(large[0, 0].sum()) - over
    bits = torch.where(large, base + (1 << 8 * byte), base).to(torch.int32)
    mass = bits.view(torch.float32)
    positions = torch.arange(c.cap, device=DEV, dtype=torch.int32).expand(1, 2, c.cap).contiguous()
    k, v = c.k.clone(), c.v.clone()
    got = paged.evict(c.k, c.v, c.table, c.lengths, mass.clone(), positions.clone(), budget=budget)
    _check_evict(c, [n], mass, positions, budget, 0, 0, got, k, v)


def test_evictions_captured_and_replayed():
    """A graph that collects weights and cuts in place, replayed: the same as eager calls on copies."""
    c = Cache([200, 90, 131], 2, 64, 16, torch.bfloat16, DEV, room=40)
    q, new = torch.randn(3, 4, 64, device=DEV).bfloat16(), torch.randn(3, 30, 2, 64, device=DEV).bfloat16()
    mass = torch.rand(3, 2, c.cap, device=DEV)
    pos = torch.arange(c.cap, dtype=torch.int32, device=DEV).expand(3, 2, c.cap).contiguous()

    def turn(k, v, n, m, p):
        paged.append(new, new, k, v, c.table, n, positions=p, mass=m)
        n.add_(30)
        paged.attn(q, k, v, c.table, n, mass=m)
        paged.evict(k, v, c.table, n, m, p, budget=100, recent=7, sink=2, out=(m, p, n))

    copies = [t.clone() for t in (c.k, c.v, c.lengths, mass, pos)]
    turn(*[t.clone() for t in copies])                        # kernels loaded
    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        turn(c.k, c.v, c.lengths, mass, pos)
    for _ in range(3):
        turn(*copies)
        graph.replay()
    torch.cuda.synchronize()
    assert c.lengths.tolist() == [100, 100, 100]
    for a, b in zip((c.k, c.v, c.lengths, mass, pos), copies):
        assert torch.equal(a.view(torch.int16) if a.dtype == torch.bfloat16 else a, b.view(torch.int16) if b.dtype == torch.bfloat16 else b)


def test_evict_with_bad_pages_and_lengths():
    c = Cache([64, 64, 0], 1, 64, 16, torch.bfloat16, DEV)
    c.table[0, 3] = -7
    c.lengths[1], c.lengths[2] = c.cap + 5, -3
    mass = torch.arange(c.cap, device=DEV).float().expand(3, 1, c.cap).contiguous()      # the last slots are kept
    positions = torch.arange(c.cap, device=DEV, dtype=torch.int32).expand(3, 1, c.cap).contiguous()
    k, flag = c.k.clone(), _flag()
    m, p, n = paged.evict(*c.tensors, mass, positions, budget=32, status=flag)
    assert int(flag) == _lib.SK_DEV_INDEX_OUT_OF_RANGE | _lib.SK_DEV_POS_OUT_OF_RANGE
    assert n.tolist() == [32, 32, 0] and m[0, 0, :32].tolist() == m[1, 0, :32].tolist() == list(range(32, 64)) and (m[2] == 0).all() and (p[2] == -1).all()
    for b, moved in ((0, range(32, 48)), (1, range(32, 64))):
        for i, f in enumerate(moved):
            k[int(c.table[b, i // 16]), 0, i % 16] = k[int(c.table[b, f // 16]), 0, f % 16]
    assert torch.equal(c.k.view(torch.int16), k.view(torch.int16))


# ------------------------------------------------------------------------------------------- together
def test_a_sequence_within_a_budget():
    """Append, attend and evict as a decoder does, against a plain list of keys per head."""
    G, H, D, page, budget, every, recent, sink = 2, 4, 64, 16, 40, 8, 10, 2
    c = Cache([0, 0], G, D, page, torch.float32, DEV, room=budget + every)
    mass, positions = torch.zeros(2, G, c.cap, device=DEV), torch.full((2, G, c.cap), -1, dtype=torch.int32, device=DEV)
    plain = [[[] for _ in range(G)] for _ in range(2)]        # [position, key, value, mass] per slot
    g = torch.Generator(device=DEV).manual_seed(3)
    for step in range(150):
        q, kn, vn = torch.randn(2, H, D, generator=g, device=DEV), *(torch.randn(2, 1, G, D, generator=g, device=DEV) for _ in range(2))
        first = torch.full((2,), step, dtype=torch.int32, device=DEV)
        paged.append(kn, vn, *c.tensors, first=first, positions=positions, mass=mass)
        out = paged.attn(q, *c.tensors, extra=1, mass=mass)
        c.lengths += 1
        for b in range(2):
            for h in range(G):
                rows = plain[b][h]
                rows.append([step, kn[b, 0, h], vn[b, 0, h], 0.0])
                k, v = torch.stack([r[1] for r in rows])[None], torch.stack([r[2] for r in rows])[None]
                want, w, _ = attend(q[b, 2 * h:2 * h + 2], k, v)
                assert (out[b, 2 * h:2 * h + 2].double() - want).abs().max() < 1e-4
                for r, x in zip(rows, w.sum(0).tolist()):
                    r[3] += x
                assert positions[b, h, :len(rows)].tolist() == [r[0] for r in rows]
                assert (mass[b, h, :len(rows)].cpu() - torch.tensor([r[3] for r in rows])).abs().max() < 1e-3
                for r, x in zip(rows, mass[b, h, :len(rows)].tolist()):
                    r[3] = x                                  # the kernel's own sums decide what is kept
        if len(plain[0][0]) == budget + every:
            paged.evict(*c.tensors, mass, positions, budget=budget, recent=recent, sink=sink, out=(mass, positions, c.lengths))
            for b in range(2):
                for h in range(G):
                    rows = plain[b][h]
                    stay = keep([r[3] for r in rows], [r[0] for r in rows], len(rows), budget, recent, sink)
                    for f, t in moves(stay, budget):
                        rows[t] = rows[f]
                    del rows[budget:]
                    assert {step - i for i in range(recent)} | set(range(sink)) <= {r[0] for r in rows}
    assert c.lengths.tolist() == [len(plain[0][0])] * 2
