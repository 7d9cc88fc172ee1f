"""A second turn behind caches that evictions have cut: its portion attends to what was kept and to itself, and decoding goes on."""
import pytest
import torch

from socket_b200 import model as transformer
from socket_b200.model import ModelArgs, Transformer
from socket_b200.paged import Paging

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
PAGING = Paging(page=16, budget=96, recent=32, sink=4, every=8)


def _model():
    return Transformer(ModelArgs.from_name("tiny")).to(device=DEV, dtype=torch.bfloat16).init_random(seed=3, std=0.05)


def _decode(model, first, position, steps):
    """Tokens at positions position .. position + steps - 1, as they were fed."""
    model.start_decode(first, position)
    fed = [first]
    for _ in range(steps):
        fed.append(model.decode_one_token().clone())
    return torch.cat(fed[:-1], 1), fed[-1]


@pytest.mark.parametrize("turn", [1, 7, 40])
def test_a_second_turn_behind_evicted_caches(turn, monkeypatch):
    B, T, new = 2, 150, 60
    model = _model().use_pages(PAGING)
    g = torch.Generator().manual_seed(1)
    prompt, more = (torch.randint(0, 512, (B, n), generator=g).to(DEV) for n in (T, turn))
    model.setup_caches(B, 400)
    model.setup_decode(B, "paged")
    first = torch.argmax(model.prefill(prompt), -1, keepdim=True)
    fed, last = _decode(model, first, T, new)
    tokens, seen = torch.cat([prompt, fed], 1), T + new
    pages = model.pages
    done = pages.length
    assert pages.position == seen and PAGING.budget <= done < PAGING.budget + PAGING.every
    before = [(c.rows(done), c.slot_positions[:, :, :done].clone(), c.mass[:, :, :done].clone()) for c in (x.attention.kv_cache for x in model.layers)]

    # the portion, with what every layer's attention is given and returns
    calls, attention = [], transformer._causal_attention
    monkeypatch.setattr(transformer, "_causal_attention", lambda q, k, v, start: calls.append((q, k, v, start, attention(q, k, v, start))) or calls[-1][-1])
    logits = model.forward_portion(more, seen, range(turn))
    monkeypatch.undo()
    assert logits.shape == (B, turn, model.config.vocab_size) and len(calls) == len(model.layers)
    assert pages.length == done + turn and pages.position == seen + turn
    assert pages.lengths.tolist() == [done + turn] * B and pages.positions.tolist() == [seen + turn] * B
    for layer, (q, k, v, start, out), ((old_k, old_v), old_positions, old_mass) in zip(model.layers, calls, before):
        c = layer.attention.kv_cache
        assert start == done and int(c.status) == 0
        assert torch.equal(k[:, :, :done], old_k) and torch.equal(v[:, :, :done], old_v) and k.shape[2] == done + turn
        for got, want in zip(c.rows(done + turn), (k, v)):
            assert torch.equal(got, want)
        assert torch.equal(c.slot_positions[:, :, :done], old_positions) and torch.equal(c.mass[:, :, :done], old_mass)
        assert (c.slot_positions[:, :, done:done + turn] == torch.arange(seen, seen + turn, device=DEV)).all()
        assert (c.mass[:, :, done:done + turn] == 0).all()
        # every kept key and the portion's own up to the query: library attention with weights of 8 bits, so two half steps of weighted |v| and one of the result
        rep = q.shape[2] // k.shape[1]
        k, v = (t.double().repeat_interleave(rep, 1) for t in (k, v))
        x = torch.einsum("bshd,bhnd->bhsn", q.double(), k) * q.shape[3] ** -0.5
        behind = torch.arange(done + turn, device=DEV) > done + torch.arange(turn, device=DEV)[:, None]
        w = torch.softmax(x.masked_fill(behind, -torch.inf), -1)
        want, spread = (torch.einsum("bhsn,bhnd->bshd", w, t) for t in (v, v.abs()))
        assert ((out.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2 * 2.0 ** -8 * spread).all()

    # the keys of the first layer depend on token and position alone: those of a model that keeps everything.  Products in other tiles may
    # round differently, before and behind the rotation: four half steps of a key's largest element
    dense = _model()
    dense.setup_caches(B, 400)
    dense.prefill(torch.cat([tokens, more], 1))
    c, every = model.layers[0].attention.kv_cache, dense.layers[0].attention.kv_cache.k_cache
    k, _ = c.rows(done + turn)
    at = c.slot_positions[:, :, :done + turn].long()
    want = every.gather(2, at.unsqueeze(-1).expand(k.shape)).double()
    assert ((k.double() - want).abs() <= 4 * 2.0 ** -8 * want.abs().amax(-1, keepdim=True)).all()

    # decoding goes on, through another eviction
    nxt = torch.argmax(logits[:, -1], -1, keepdim=True)
    _decode(model, nxt, seen + turn, 50)
    seen += turn + 50
    assert pages.position == seen and pages.length < PAGING.budget + PAGING.every
    for layer in model.layers:
        c = layer.attention.kv_cache
        kept = set(range(PAGING.sink)) | set(range(seen - PAGING.recent, seen))
        for row in c.slot_positions[:, :, :pages.length].flatten(0, 1).tolist():
            assert kept <= set(row) and len(set(row)) == len(row) and max(row) == seen - 1
        assert int(c.status) == 0 and (c.mass[:, :, pages.length:] == 0).all()


def test_a_turn_in_portions_is_the_turn_in_one():
    """Portions of a turn continue one another behind evicted caches: the same keys in the first layer, the same places in all."""
    more = torch.randint(0, 512, (2, 45), generator=torch.Generator().manual_seed(5)).to(DEV)
    held = []
    for cuts in ((45,), (16, 29), (1, 3, 41)):
        model = _model().use_pages(PAGING)
        model.setup_caches(2, 400)
        model.setup_decode(2, "paged")
        first = torch.argmax(model.prefill(more.repeat(1, 4)[:, :150]), -1, keepdim=True)
        _decode(model, first, 150, 30)
        at = 180
        for n in cuts:
            model.forward_portion(more[:, at - 180:at - 180 + n], at)
            at += n
        c = model.layers[0].attention.kv_cache
        held.append((model.pages.length, c.slot_positions[:, :, :model.pages.length].clone(), c.rows(model.pages.length)[0].double()))
    for length, positions, k in held[1:]:
        assert length == held[0][0] and torch.equal(positions, held[0][1])
        assert ((k - held[0][2]).abs() <= 4 * 2.0 ** -8 * held[0][2].abs().amax(-1, keepdim=True)).all()
