"""Log probabilities, entropy and alternatives of logits against float64, at the sizes and contents where they can go wrong."""
import math

import pytest
import torch

from socket_b200 import _lib, few_rows

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _plain(x, tokens, top):
    x = x.double()
    lp = x - torch.logsumexp(x, -1, keepdim=True)
    entropy = -torch.where(lp == -math.inf, 0.0, lp.exp() * lp).sum(-1)
    value, index = torch.sort(lp, dim=-1, descending=True, stable=True)
    return lp.gather(1, tokens.view(-1, 1)).view(-1), entropy, value[:, :top], index[:, :top]


def _check(x, tokens, top, library="step"):
    """fp32: an exponential and a logarithm are off by a few half steps, sums of up to 2^18 positive terms by far fewer than the
    2^-19 they are allowed here; a difference of logits by half a step of their size."""
    got = few_rows.token_logprobs(x, tokens, top=top, library=library)
    lp, entropy, value, index = _plain(x, tokens, top)
    size = x.double().masked_fill(x == -math.inf, 0.0).abs().amax(-1)
    tol = 2.0 ** -19 * (2 + size)
    finite = lp > -math.inf
    assert torch.equal(got.logprobs > -math.inf, finite)
    assert ((got.logprobs.double() - lp).abs() <= tol)[finite].all()
    assert ((got.entropy.double() - entropy).abs() <= 2 * tol).all()
    assert torch.equal(got.top_tokens, index)
    both = value > -math.inf
    assert torch.equal(got.top_logprobs > -math.inf, both) and ((got.top_logprobs.double() - value).abs() <= tol[:, None])[both].all()
    return got


@pytest.mark.parametrize("library", ["step", "blocks"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (2, 7), (5, 64), (1, 1000), (9, 4097), (4, 32768), (2, 50257), (8, 128256), (300, 8191), (700, 513)])
def test_rows(rows, vocab, dtype, library):
    g = torch.Generator(device=DEV).manual_seed(vocab + rows)
    x = (torch.randn(rows, vocab, generator=g, device=DEV) * 4).to(dtype)
    tokens = torch.randint(0, vocab, (rows,), generator=g, device=DEV)
    for top in sorted({0, 1, min(5, vocab), min(20, vocab), min(64, vocab)}):
        _check(x, tokens, top, library)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [100, 5000, 70000, 150000])
def test_orders_of_logits(vocab, dtype):
    """Rising, falling, equal and nearly equal rows, peaks at the ends: whatever order a row is walked in."""
    i = torch.arange(vocab, device=DEV).float() / vocab * 20
    rows = torch.stack([i, -i, torch.zeros_like(i), (i * 7 % 1).round(), torch.where(i == 0, 50.0, -50.0), torch.where(i == i[-1], 9.0, 0.0),
                        torch.full_like(i, -3e4), torch.full_like(i, 3e4), torch.where(i > 10, 1e-3, 0.0)]).to(dtype)
    tokens = torch.randint(0, vocab, (len(rows),), device=DEV)
    for top in (1, 64):
        _check(rows, tokens, top)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [66, 9000, 128256])
def test_masked_logits(vocab, dtype):
    """-inf and the type's lowest value in masked places; fewer live logits than alternatives."""
    x = torch.randn(6, vocab, device=DEV).to(dtype)
    x[0, ::2] = -math.inf
    x[1, 1:] = -math.inf
    x[2, :vocab - 3] = -math.inf
    x[3, 1::2] = torch.finfo(dtype).min
    x[4] = torch.finfo(dtype).min
    x[5, 5] = torch.finfo(dtype).max
    tokens = torch.tensor([1, 0, vocab - 1, 1, 7, 5], device=DEV)
    got = _check(x[:4], tokens[:4], 64)
    assert got.logprobs[1] == 0 and got.entropy[1] == 0
    masked = _check(x[:3], torch.tensor([0, 1, 0], device=DEV), 1)
    assert (masked.logprobs == -math.inf).all()
    got = few_rows.token_logprobs(x[4:], tokens[4:], top=2)
    torch.testing.assert_close(got.logprobs, torch.tensor([-math.log(vocab), 0.0], device=DEV), rtol=1e-6, atol=1e-6)
    torch.testing.assert_close(got.entropy, torch.tensor([math.log(vocab), 0.0], device=DEV), rtol=1e-6, atol=1e-6)
    assert got.top_tokens[0].tolist() == [0, 1] and got.top_tokens[1, 0] == 5


@pytest.mark.parametrize("vocab", [50, 40000])
def test_rows_without_a_distribution(vocab):
    x = torch.randn(5, vocab, device=DEV)
    x[0] = -math.inf
    x[1, 3] = math.inf
    x[2, 9] = math.nan
    x[3, [4, 30]] = math.nan
    clean = few_rows.token_logprobs(x[4:], torch.tensor([2], device=DEV), top=5)
    got = few_rows.token_logprobs(x, torch.full((5,), 2, device=DEV), top=5)
    assert got.entropy[:4].isnan().all() and got.logprobs[[0, 2, 3]].isnan().all() and got.top_logprobs[0].isnan().all()
    assert got.top_tokens[0].tolist() == [0, 1, 2, 3, 4] and got.top_tokens[1, 0] == 3 and got.top_tokens[2, 0] == 9 and got.top_tokens[3, :2].tolist() == [4, 30]
    for a, b in zip(got, clean):
        assert torch.equal(a[4], b[0])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [100, 3000, 60000, 128256])
def test_a_token_that_is_nearly_certain(vocab, dtype):
    """One logit far above the sum of all others: its log probability is that sum, to a few half steps of itself (terms are exponentials
    of differences of up to 45, each off by 45 half steps and two of the exponential's; they are summed in a few hundred steps at most)."""
    g = torch.Generator(device=DEV).manual_seed(vocab)
    x = torch.randn(12, vocab, generator=g, device=DEV).to(dtype)
    at = torch.randint(0, vocab, (12,), generator=g, device=DEV)
    gap = torch.arange(12, device=DEV) * 2.0 + 6 + math.log(vocab)
    x[torch.arange(12, device=DEV), at] = gap.to(dtype)
    got = few_rows.token_logprobs(x, at, top=2)
    y = x.double()
    d = y - y.gather(1, at[:, None])
    rest = torch.where(d == 0, 0.0, d.exp()).sum(-1)
    want = -torch.log1p(rest)
    assert (want > -0.01).all() and ((got.logprobs.double() - want).abs() <= want.abs() * 600 * 2.0 ** -24).all()
    p, q = d.exp() / (1 + rest[:, None]), d + want[:, None]
    entropy = -(p * q).sum(-1)
    assert ((got.entropy.double() - entropy).abs() <= entropy * 800 * 2.0 ** -24).all()
    assert torch.equal(got.top_logprobs[:, 0], got.logprobs) and torch.equal(got.top_tokens[:, 0], at)


@pytest.mark.parametrize("vocab", [2000, 50000])
def test_rows_with_many_nan(vocab):
    """NaN everywhere, at the front, in every second place: the lowest indices come first, whatever the list is cut by."""
    x = torch.randn(3, vocab, device=DEV)
    x[0] = math.nan
    x[1, :1500] = math.nan
    x[2, ::2] = math.nan
    for top in (1, 2, 64):
        got = few_rows.token_logprobs(x, top=top)
        i = torch.arange(top, device=DEV)
        assert torch.equal(got.top_tokens, torch.stack([i, i, 2 * i])) and got.top_logprobs.isnan().all() and got.entropy.isnan().all()


def test_rows_of_other_layouts():
    big = torch.randn(40, 3001, device=DEV).bfloat16()
    tokens = torch.randint(0, 2999, (40,), device=DEV)
    for x in (big[:, 1:3000], big[::2, 2:3001], big[3:4, :2999].expand(40, 2999), torch.randn(2999, 40, device=DEV).bfloat16().t()):
        _check(x, tokens[:x.shape[0]], 5)
    none = few_rows.token_logprobs(big[:, :100], top=2)
    assert none.logprobs is None and torch.equal(none.top_tokens, few_rows.token_logprobs(big[:, :100], tokens % 100, top=2).top_tokens)
    empty = few_rows.token_logprobs(big[:0], tokens[:0], top=3)
    assert empty.logprobs.shape == (0,) and empty.top_tokens.shape == (0, 3)


def test_tokens_outside_the_vocabulary():
    x, flag = torch.randn(4, 100, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    got = few_rows.token_logprobs(x, torch.tensor([-1, 100, 5, 2 ** 40], device=DEV), status=flag)
    assert got.logprobs.isnan().tolist() == [True, True, False, True] and int(flag) == _lib.SK_DEV_INDEX_OUT_OF_RANGE
    with pytest.raises(RuntimeError):
        few_rows.token_logprobs(x, top=65)
    with pytest.raises(RuntimeError):
        few_rows.token_logprobs(x[:, :3], top=4)


def test_captured_and_on_another_stream():
    x, tokens = torch.randn(8, 40000, device=DEV).bfloat16(), torch.randint(0, 40000, (8, 1), device=DEV)
    want = few_rows.token_logprobs(x, tokens, top=9)
    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = few_rows.token_logprobs(x, tokens, top=9)
    for _ in range(3):
        with torch.cuda.stream(side):
            graph.replay()
        side.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
