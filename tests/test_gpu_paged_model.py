"""The paged cache, evictions and log probabilities inside the decoders."""
import json

import pytest
import torch

from tests.paged_util import attend
from socket_b200 import generate as command
from socket_b200.decoder import generate
from socket_b200.model import ModelArgs, Transformer
from socket_b200.paged import Paging
from socket_b200.registry import build_model, write_safetensors
from tests.radapel_util import CONFIGS

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _model(dtype=torch.bfloat16, **over):
    cfg = ModelArgs.from_name("tiny", **over)
    return Transformer(cfg).to(device=DEV, dtype=dtype).init_random(seed=3, std=0.05)


def _prompt(B, T, seed=0):
    return torch.randint(0, 512, (B, T), generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("page", [16, 64])
def test_graph_replayed_paged_decode_equals_eager_decode(page):
    model, prompt = _model().use_pages(Paging(page=page)), _prompt(2, 700)
    a, _ = generate(model, prompt, 40, mode="paged", use_graph=True, prefill_chunk=256)
    b, _ = generate(model, prompt, 40, mode="paged", use_graph=False, prefill_chunk=256)
    assert torch.equal(a, b)
    pages = model.pages
    assert pages.length == pages.position == 700 + 39 and pages.lengths.tolist() == pages.positions.tolist() == [739] * 2
    assert all(int(x.attention.kv_cache.status) == 0 for x in model.layers)
    assert sum(map(len, pages.held)) == 2 * -(-739 // page) and len(pages.free) + sum(map(len, pages.held)) == pages.pages


def test_paged_layers_hold_what_the_dense_ones_do():
    """The same prompt and token through both kinds of cache: equal keys and values, attention by the formula."""
    prompt, T = _prompt(2, 300).to(DEV), 300
    dense, paged = _model(), _model().use_pages(Paging(page=32))
    for m, mode in ((dense, "dense"), (paged, "paged")):
        m.setup_caches(2, T + 8)
        m.setup_decode(2, mode, use_graph=False)
        m.prefill(prompt)
        m.decode_given_token(prompt[:, :1].contiguous(), T)
    for i, (x, y) in enumerate(zip(dense.layers, paged.layers)):
        c, d = x.attention.kv_cache, y.attention
        k, v = d.kv_cache.rows(T + 1)
        if i == 0:                                             # later layers' inputs differ by the attentions' rounding
            assert torch.equal(k, c.k_cache[:, :, :T + 1]) and torch.equal(v, c.v_cache[:, :, :T + 1])
        for b in range(2):
            want, _, err = attend(d.q_s[b], k[b], v[b])
            assert (d.o_s[b].double() - want).abs().max() <= 2.0 ** -8 * want.abs().max() + err * v[b].double().abs().max()


@pytest.mark.parametrize("use_graph", [False, True])
def test_sequences_stay_within_their_budget(use_graph):
    p = Paging(page=16, budget=96, recent=32, sink=4, every=8)
    model = _model().use_pages(p)
    B, T, new = 2, 150, 60
    prompt = _prompt(B, T).to(DEV)
    model.setup_caches(B, T + new)
    model.setup_decode(B, "paged", use_graph)
    tok = torch.argmax(model.prefill(prompt), -1, keepdim=True)
    model.start_decode(tok, T)
    before = {}
    for step in range(new):
        model.decode_one_token()
        seen = T + step + 1
        assert model.pages.lengths.tolist() == [model.pages.length] * B and model.pages.positions.tolist() == [seen] * B
        assert model.pages.length < p.budget + p.every and sum(map(len, model.pages.held)) == B * -(-model.pages.length // p.page)
        for i, layer in enumerate(model.layers):
            c = layer.attention.kv_cache
            held = c.slot_positions[:, :, :model.pages.length]
            kept = set(range(p.sink)) | set(range(seen - p.recent, seen))
            for row, m in zip(held.reshape(-1, held.shape[2]).tolist(), c.mass.flatten(0, 1)):
                assert kept <= set(row) and len(set(row)) == len(row) and max(row) == seen - 1
                assert (m[:model.pages.length] >= 0).all() and (m[model.pages.length:] == 0).all()
            k, v = c.rows(model.pages.length)
            if step > 0:                                       # a key that stays keeps its row
                old, ok, ov = before[i]
                for b in range(B):
                    at = {q: s for s, q in enumerate(old[b, 0].tolist())}
                    pairs = [(s, at[q]) for s, q in enumerate(held[b, 0].tolist()) if q in at]
                    assert len(pairs) >= model.pages.length - 1
                    new_at, old_at = (torch.tensor(z, device=DEV) for z in zip(*pairs))
                    assert torch.equal(k[b, 0, new_at], ok[b, 0, old_at]) and torch.equal(v[b, 0, new_at], ov[b, 0, old_at])
            before[i] = (held.clone(), k, v)
            assert int(c.status) == 0
    # a second turn behind the evicted caches, then a new conversation
    more = model.forward_portion(prompt[:, :7], T + new - 0) if T + new + 7 <= model.max_seq_length else None
    assert more is None or torch.isfinite(more).all()
    model.prefill(prompt)
    assert model.pages.length == T and model.pages.lengths.tolist() == [T] * B


def test_a_small_pool_is_enough_within_a_budget_and_too_small_one_says_so():
    prompt = _prompt(1, 100)
    model = _model().use_pages(Paging(page=16, pages=9, budget=64, recent=16, every=16))
    seq, _ = generate(model, prompt, 200, mode="paged")
    assert seq.shape == (1, 300) and model.pages.length < 80
    model = _model().use_pages(Paging(page=16, pages=7))
    with pytest.raises(RuntimeError, match="out of pages"):
        generate(model, prompt, 200, mode="paged")


def test_calls_that_pages_refuse():
    model, prompt = _model().use_pages(Paging(page=16)), _prompt(2, 50).to(DEV)
    model.setup_caches(2, 100)
    for mode in ("sparse", "dense"):
        with pytest.raises(RuntimeError, match="pages"):
            model.setup_decode(2, mode, use_graph=False)
    with pytest.raises(RuntimeError, match="sequences"):
        model.setup_decode(1, "paged")
    with pytest.raises(RuntimeError, match="sequences"):
        model.prefill(prompt[:1])
    model.setup_decode(2, "paged")
    model.prefill(prompt)
    with pytest.raises(RuntimeError, match="end at 50"):
        model.forward_portion(prompt[:, :5], 40)
    with pytest.raises(RuntimeError, match="end at 50"):
        model.start_decode(prompt[:, :1].contiguous(), 49)
    with pytest.raises(RuntimeError, match="budget"):
        model.evict(10)
    plain = _model()
    plain.setup_caches(2, 100)
    with pytest.raises(RuntimeError, match="pages"):
        plain.setup_decode(2, "paged", use_graph=False)
    # other numbers of sequences get caches of their own
    for B in (1, 3):
        seq, _ = generate(model, _prompt(B, 30), 5)
        assert seq.shape == (B, 35) and model.pages.lengths.tolist() == [34] * B
    # and back again
    generate(model, prompt.cpu(), 5, mode="sparse")
    assert model.pages is None
    generate(model, prompt.cpu(), 5, mode="paged")
    assert model.pages.length == 54


def test_decode_is_set_up_behind_a_prompt_without_touching_it():
    model, prompt = _model().use_pages(Paging(page=16, budget=64, every=100)), _prompt(2, 40).to(DEV)
    model.setup_caches(2, 100)
    model.prefill(prompt)
    rows = [x.attention.kv_cache.rows(40) for x in model.layers]
    model.setup_decode(2, "paged")
    for x, (k, v) in zip(model.layers, rows):
        c = x.attention.kv_cache
        assert all(torch.equal(a, b) for a, b in zip(c.rows(40), (k, v))) and (c.mass == 0).all() and int(c.status) == 0
    assert model.pages.lengths.tolist() == [40, 40]


# ------------------------------------------------------------------------------------------- log probabilities
@pytest.mark.parametrize("paged", [False, True])
def test_scores_of_a_prompt(paged):
    model, prompt = _model(), _prompt(3, 90).to(DEV)
    if paged:
        model.use_pages(Paging(page=16))
    model.setup_caches(3, 100)
    logits = torch.cat([model.forward_portion(prompt[:, :50], 0, range(50)), model.forward_portion(prompt[:, 50:], 50, range(40))], 1)
    got = model.score(prompt, top=3, chunk=50)
    lp = torch.log_softmax(logits[:, :-1].double(), -1)
    want = lp.gather(2, prompt[:, 1:, None])[..., 0]
    # the head's products may be taken in other tiles: logits of either call are a rounding of theirs off
    tol = 2 * 2.0 ** -8 * logits.double().abs().max() + 1e-4
    assert got.logprobs.shape == (3, 89) and (got.logprobs.double() - want).abs().max() <= tol
    assert ((got.entropy.double() + (lp.exp() * lp).sum(-1)).abs() <= 8 * tol).all()
    assert got.top_tokens.shape == (3, 89, 3) and (got.top_logprobs.double() - lp.topk(3).values).abs().max() <= tol


def test_scores_of_a_prompt_through_listed_layers():
    model = build_model(CONFIGS["wide"], None, torch.float32, DEV).init_random(5)
    prompt = torch.randint(0, CONFIGS["wide"]["vocab"], (2, 70), generator=torch.Generator().manual_seed(1)).to(DEV)
    model.setup_caches(2, 80)
    logits = model.forward_portion(prompt, 0, range(70)).double()
    lp = torch.log_softmax(logits[:, :-1], -1)
    got = model.score(prompt, top=1, chunk=33)
    # fp32 products summed in other tiles: a few thousand half steps of the logits' size
    tol = 4096 * 2.0 ** -24 * (1 + logits.abs().max())
    assert ((got.logprobs.double() - lp.gather(2, prompt[:, 1:, None])[..., 0]).abs() <= tol).all()
    assert ((got.entropy.double() + (lp.exp() * lp).sum(-1)).abs() <= 8 * tol).all()
    seq, stats = generate(model, prompt.cpu(), 5, logprobs=2)
    assert torch.equal(stats["logprobs"].top_tokens[..., 0], seq[:, 70:])


@pytest.mark.parametrize("mode", ["sparse", "dense", "paged"])
def test_log_probabilities_of_generated_tokens(mode):
    model, prompt = _model(), _prompt(2, 60)
    seq, stats = generate(model, prompt, 7, mode=mode, logprobs=4)
    p = stats["logprobs"]
    assert p.logprobs.shape == p.entropy.shape == (2, 7) and p.top_tokens.shape == (2, 7, 4)
    assert torch.equal(p.top_tokens[..., 0], seq[:, 60:]) and torch.equal(p.top_logprobs[..., 0], p.logprobs)
    assert (p.logprobs <= 0).all() and (p.entropy > 0).all() and (p.top_logprobs.diff(dim=-1) <= 0).all()
    plain, _ = generate(model, prompt, 7, mode=mode)
    assert torch.equal(plain, seq)


def test_the_command_tells_log_probabilities_and_keeps_a_budget(tmp_path, capsys):
    model = _model()
    write_safetensors(str(tmp_path / "model.safetensors"), {k: v for k, v in model.state_dict().items()})
    cfg = {k: v for k, v in vars(model.config).items()}
    (tmp_path / "config.json").write_text(json.dumps({"architecture": "Transformer", **cfg}))
    args = ["--model", str(tmp_path), "--tokens", "5,17,3,9,8,7,1,2;8,2,9,4,4,4,6,6", "--new", "40", "--mode", "paged", "--page", "16"]
    assert command.main(args) == 0
    rows = [[int(t) for t in line.split(",")] for line in capsys.readouterr().out.split()]
    assert command.main(args + ["--logprobs", "2"]) == 0
    found = [json.loads(line) for line in capsys.readouterr().out.splitlines()]
    assert [f["tokens"] for f in found] == rows and all(len(f["logprobs"]) == 40 and len(f["top_tokens"][0]) == 2 for f in found)
    assert command.main(args + ["--kv-budget", "16", "--kv-recent", "8", "--kv-every", "4"]) == 0
    assert len(capsys.readouterr().out.splitlines()) == 2
    with pytest.raises(SystemExit):
        command.main(args[:4] + ["--kv-budget", "16"])
