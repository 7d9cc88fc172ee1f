"""Performance cases of serving from a paged cache: what a decoded token does with its cache, and how likely it was.

Four operators:

* `append`    new keys and values of a padded batch go into the pages of a cache (`paged.append`).
* `attn`      one new token per sequence attends over its pages; with `mass` every cached key also collects the
              weight it got (`paged.attn`).
* `evict`     sequences over a budget lose the keys that collected the least weight (`paged.evict`).
* `logprobs`  log probabilities of given tokens, entropy and the likeliest alternatives of rows of logits
              (`few_rows.token_logprobs`).

A pool of pages is [pages, KV heads, page, head size]; slot j of a sequence is row j % page of the page that
column j / page of its row in the table names.  `own` chooses between the framework's operators and their plain forms.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

torch.backends.cuda.matmul.allow_tf32 = False          # products of fp32 stay fp32

DEV = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}


# ------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # one user's first tokens: nothing but latency
        dict(name="attn short f32", kind="attn", B=1, H=8, G=2, D=64, page=16, lo=37, hi=37, mass=False, dtype="f32"),
        # one user with a 32K context, 8B-shape heads
        dict(name="attn 32k", kind="attn", B=1, H=32, G=8, D=128, page=64, lo=32768, hi=32768, mass=False, dtype="bf16"),
        # a batch of conversations of all lengths whose caches are bounded, so weights are collected
        dict(name="attn ragged x64 mass f16", kind="attn", B=64, H=32, G=8, D=128, page=16, lo=1, hi=8003, mass=True, dtype="f16"),
        # four long contexts, the headline sizes, collecting weights
        dict(name="attn 128k x4 mass", kind="attn", B=4, H=32, G=8, D=128, page=64, lo=131072, hi=131072, mass=True, dtype="bf16"),
        # the new token of every sequence of a batch
        dict(name="append token x64", kind="append", B=64, G=8, D=128, page=16, S=1, lo=1, hi=8003, dtype="f16"),
        # a padded batch of prompts behind what earlier turns left
        dict(name="append prompts x8", kind="append", B=8, G=8, D=128, page=64, S=4096, lo=100, hi=5000, dtype="bf16"),
        # a batch at its budget, after 256 more tokens
        dict(name="evict 4352 to 4096 x32", kind="evict", B=32, G=8, D=128, page=64, lo=4352, hi=4352, budget=4096, recent=256, sink=16,
             dtype="bf16"),
        # a long prompt cut to a few thousand keys
        dict(name="evict 32k to 4096", kind="evict", B=1, G=8, D=128, page=64, lo=32768, hi=32768, budget=4096, recent=1024, sink=64,
             dtype="bf16"),
        # the tokens of a batch just decoded, small vocabulary, fp32 logits of the listed-layer decoders
        dict(name="logprobs token x4 f32", kind="logprobs", rows=4, vocab=32768, top=5, dtype="f32"),
        # the same of the Llama-shaped decoder
        dict(name="logprobs token x8", kind="logprobs", rows=8, vocab=128256, top=20, dtype="bf16"),
        # a prompt's tokens scored, a vocabulary no vector divides
        dict(name="logprobs prompt odd", kind="logprobs", rows=1001, vocab=50257, top=1, dtype="bf16"),
        # a long prompt's
        dict(name="logprobs prompt 2048", kind="logprobs", rows=2048, vocab=128256, top=8, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attn", "attn", "attn", "append", "evict", "evict", "logprobs", "logprobs"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind == "logprobs":
        vocab = _log(rng, 300, 160000)
        return dict(kind=kind, rows=_log(rng, 1, max(2, min(8192, 2 ** 28 // vocab // BYTES[dtype]))), vocab=vocab, top=rng.randrange(0, 21),
                    dtype=dtype)
    H, G = rng.choice([(32, 8), (32, 8), (16, 4), (8, 2), (8, 1), (64, 8), (8, 8), (16, 1), (12, 4)])
    D, page, B = rng.choice([64, 128, 128, 128, 96, 256]), rng.choice([16, 32, 64, 128]), _log(rng, 1, 64)
    most = 2 ** 31 // (B * G * D * 2 * BYTES[dtype])       # keys of the longest sequence: pools of 2 GB
    if kind == "attn":
        hi = _log(rng, 1, min(131072, most))
        return dict(kind=kind, B=B, H=H, G=G, D=D, page=page, lo=rng.choice([hi, hi, 1 + hi // 7, 1]), hi=hi, mass=rng.random() < 0.5, dtype=dtype)
    if kind == "append":
        hi = _log(rng, 1, min(8000, most // 2))
        return dict(kind=kind, B=B, G=G, D=D, page=page, S=_log(rng, 1, min(8192, most // 2)), lo=rng.choice([hi, 1]), hi=hi, dtype=dtype)
    hi = _log(rng, 100, min(65536, most))
    budget = max(4, int(hi * rng.choice([0.1, 0.5, 0.9, 0.97])))
    return dict(kind=kind, B=B, G=G, D=D, page=page, lo=rng.choice([hi, hi, 1 + hi // 3]), hi=hi, budget=budget, recent=budget // 8,
                sink=rng.choice([0, min(4, budget // 4)]), dtype=dtype)


def _lengths(case):
    """The cached lengths of a case's sequences, spread over the logarithm of their range; `prepare` shuffles them."""
    B, lo, hi = case["B"], case["lo"], case["hi"]
    return [hi if i == B - 1 else int(round(lo * (hi / lo) ** ((i + 0.5) / B))) for i in range(B)]


def _counts(case):
    """New tokens of each row of a padded batch: from a full row down to a fifth."""
    B, S = case["B"], case["S"]
    return [max(1, S - (S * 4 * i) // (5 * B)) for i in range(B)]


# ------------------------------------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _pool(case, width, g):
    """Two pools whose pages the sequences hold in a shuffled order, and their table."""
    pages = case["B"] * width
    shape, dt = (pages, case["G"], case["page"], case["D"]), DTYPES[case["dtype"]]
    k, v = (torch.empty(shape, dtype=dt, device=DEV).normal_(0.0, 1.0, generator=g) for _ in range(2))
    table = torch.randperm(pages, generator=g, device=DEV).to(torch.int32).view(case["B"], width)
    return k, v, table


def _shuffled(values, g):
    return torch.tensor(values, dtype=torch.int32, device=DEV)[torch.randperm(len(values), generator=g, device=DEV)]


def prepare(case, seed):
    g = _generator(seed)
    dt = DTYPES[case["dtype"]]
    state = {"case": case}
    if case["kind"] == "logprobs":
        # a peaked distribution over many near-equal logits, as a language model's head gives
        x = torch.empty(case["rows"], case["vocab"], dtype=dt, device=DEV).normal_(0.0, 2.5, generator=g)
        peak = torch.randint(0, case["vocab"], (case["rows"], 1), generator=g, device=DEV)
        x.scatter_(1, peak, torch.full_like(peak, 14, dtype=dt))
        other = torch.randint(0, case["vocab"], (case["rows"], 1), generator=g, device=DEV)
        state["logits"], state["tokens"] = x, torch.where(torch.rand(peak.shape, generator=g, device=DEV) < 0.7, peak, other).view(-1)
        return state
    lengths = _lengths(case)
    extra = case.get("S", 0)
    width = -(-(max(lengths) + extra) // case["page"])
    state["k"], state["v"], state["table"] = _pool(case, width, g)
    state["lengths"] = _shuffled(lengths, g)
    B, G, D, cap = case["B"], case["G"], case["D"], width * case["page"]
    new = lambda *s: torch.empty(*s, dtype=dt, device=DEV).normal_(0.0, 1.0, generator=g)  # noqa: E731
    if case["kind"] == "attn":
        # queries that lean towards some keys: weights of very different sizes
        state["q"] = new(B, case["H"], D) * 1.7
        state["mass"] = torch.rand(B, G, cap, generator=g, device=DEV) if case["mass"] else None
    elif case["kind"] == "append":
        state["k_new"], state["v_new"] = new(B, extra, G, D), new(B, extra, G, D)
        state["counts"] = _shuffled(_counts(case), g)
        state["first"] = state["lengths"] + 7                     # earlier evictions have left slots behind positions
        state["mass"] = torch.rand(B, G, cap, generator=g, device=DEV)
        state["positions"] = torch.randint(0, 1 << 20, (B, G, cap), generator=g, device=DEV, dtype=torch.int32)
    else:
        # weights over many orders of size; slots in the order that earlier evictions left them in
        state["mass"] = torch.empty(B, G, cap, device=DEV).log_normal_(-2.0, 2.0, generator=g)
        order = torch.rand(B, G, cap, generator=g, device=DEV)
        order += (torch.arange(cap, device=DEV) >= state["lengths"].view(-1, 1, 1)) * 2.0
        positions = torch.empty(B, G, cap, dtype=torch.int64, device=DEV)
        positions.scatter_(2, order.argsort(-1), torch.arange(cap, device=DEV).expand(B, G, cap))
        state["positions"] = positions.to(torch.int32)
    return state


# ------------------------------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    return {"append": _append, "attn": _attn, "evict": _evict, "logprobs": _logprobs}[case["kind"]](case, state)


def _rows(pool, table):
    """[B, G, cap, D]: the rows of every sequence in slot order."""
    return pool[table.long()].permute(0, 2, 1, 3, 4).flatten(2, 3)


def _places(table, slots, page):
    """Page and row of slots [B, n]."""
    return table.long().gather(1, slots // page), slots % page


def _append(case, s):
    if own:
        from socket_b200 import paged
        paged.append(s["k_new"], s["v_new"], s["k"], s["v"], s["table"], s["lengths"], counts=s["counts"], first=s["first"],
                     positions=s["positions"], mass=s["mass"])
    else:
        S, page = case["S"], case["page"]
        at = torch.arange(S, device=DEV)
        b, t = (at < s["counts"].view(-1, 1)).nonzero(as_tuple=True)
        slot = s["lengths"].long()[b] + t
        pages, rows = s["table"].long()[b, slot // page], slot % page
        s["k"][pages, :, rows] = s["k_new"][b, t]
        s["v"][pages, :, rows] = s["v_new"][b, t]
        s["mass"][b, :, slot] = 0.0
        s["positions"][b, :, slot] = (s["first"][b] + t.to(torch.int32)).unsqueeze(1)
    return {"k": s["k"], "v": s["v"], "positions": s["positions"], "mass": s["mass"]}


def _attn(case, s):
    if own:
        from socket_b200 import paged
        out = paged.attn(s["q"], s["k"], s["v"], s["table"], s["lengths"], mass=s["mass"])
    else:
        B, G, D = case["B"], case["G"], case["D"]
        k, v = _rows(s["k"], s["table"]).float(), _rows(s["v"], s["table"]).float()
        live = torch.arange(k.shape[2], device=DEV) < s["lengths"].view(-1, 1, 1, 1)
        x = torch.matmul(s["q"].float().view(B, G, -1, D), k.transpose(2, 3)) * D ** -0.5
        x = x.masked_fill(~live, -torch.inf)
        top = x.amax(-1, keepdim=True)
        w = torch.exp(x - torch.where(top == -torch.inf, 0.0, top))
        w = w / w.sum(-1, keepdim=True).clamp_min(1e-30)
        out = torch.matmul(w, v.masked_fill(~live.transpose(2, 3), 0.0)).view(B, -1, D).to(s["q"].dtype)
        if s["mass"] is not None:
            s["mass"] += w.sum(2)
    return {"out": out} if s["mass"] is None else {"out": out, "mass": s["mass"]}


def _evict(case, s):
    budget, recent, sink, page = case["budget"], case["recent"], case["sink"], case["page"]
    if own:
        from socket_b200 import paged
        mass, positions, lengths = paged.evict(s["k"], s["v"], s["table"], s["lengths"], s["mass"], s["positions"], budget=budget,
                                               recent=recent, sink=sink)
    else:
        B, G, cap = s["mass"].shape
        slot = torch.arange(cap, device=DEV)
        live = (slot < s["lengths"].view(-1, 1, 1)).expand(B, G, cap)
        newest = s["positions"].masked_fill(~live, -1).amax(-1, keepdim=True)
        kept_for_sure = (s["positions"] < sink) | (s["positions"] > newest - recent)
        rank = torch.where(live, torch.where(kept_for_sure, torch.inf, s["mass"]), -torch.inf)
        order = rank.argsort(dim=-1, descending=True, stable=True)
        keep = torch.zeros_like(live).scatter_(2, order[..., :budget], True) & live
        hole, mover = ~keep & (slot < budget) & live, keep & (slot >= budget)
        # the i-th mover goes to the i-th hole
        place = torch.where(hole, hole.cumsum(-1) - 1, cap)
        source = torch.zeros(B, G, cap + 1, dtype=torch.long, device=DEV)
        source.scatter_(2, torch.where(mover, mover.cumsum(-1) - 1, cap), slot.expand(B, G, cap))
        hole = hole & (place < mover.sum(-1, keepdim=True))
        b, g, to = hole.nonzero(as_tuple=True)
        frm = source[b, g, place[b, g, to]]
        mass, positions = s["mass"].clone(), s["positions"].clone()
        mass[b, g, to], positions[b, g, to] = s["mass"][b, g, frm], s["positions"][b, g, frm]
        lengths = s["lengths"].clamp(max=budget)
        gone = slot >= lengths.view(-1, 1, 1)
        mass.masked_fill_(gone, 0.0)
        positions.masked_fill_(gone, -1)
        table = s["table"].long()
        for pool in (s["k"], s["v"]):
            pool[table[b, to // page], g, to % page] = pool[table[b, frm // page], g, frm % page]
    return {"k": s["k"], "v": s["v"], "mass": mass, "positions": positions, "lengths": lengths}


def _logprobs(case, s):
    if own:
        from socket_b200 import few_rows
        r = few_rows.token_logprobs(s["logits"], s["tokens"], top=case["top"], library="step")
        out = {"logprobs": r.logprobs, "entropy": r.entropy, "top_logprobs": r.top_logprobs, "top_tokens": r.top_tokens}
    else:
        vocab, k = case["vocab"], min(case["top"], case["vocab"])
        x = s["logits"].float()
        top = x.amax(-1, keepdim=True)
        d = x - top
        e = torch.exp(d)
        z = e.sum(-1, keepdim=True)
        log_z = torch.log(z)
        entropy = (log_z - (e * d).sum(-1, keepdim=True) / z).view(-1)
        logprobs = (d.gather(1, s["tokens"].view(-1, 1)) - log_z).view(-1)
        # equal logits: the lower index first, so order and index are ranked as one number
        bits = x.view(torch.int32).long()
        order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits) * vocab + (vocab - 1 - torch.arange(vocab, device=DEV))
        best = order.topk(k, dim=-1).indices if k else order[:, :0]
        out = {"logprobs": logprobs, "entropy": entropy, "top_logprobs": d.gather(1, best) - log_z, "top_tokens": best}
    if case["top"] == 0:
        del out["top_logprobs"], out["top_tokens"]
    return out


# ------------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    es = BYTES[case["dtype"]]
    if case["kind"] == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * es + case["rows"] * (16 + 12 * case["top"]), "flops": 5 * n}
    G, D, row = case["G"], case["D"], case["D"] * es
    lengths = _lengths(case)
    if case["kind"] == "append":
        n = sum(_counts(case)) * G
        return {"bytes": n * (4 * row + 8), "flops": 0}
    n = sum(lengths) * G
    if case["kind"] == "attn":
        rep = case["H"] // G
        return {"bytes": n * (2 * row + (8 if case["mass"] else 0)) + 2 * case["B"] * case["H"] * row + 4 * sum(lengths) // case["page"],
                "flops": 4 * n * rep * D}
    cap = -(-max(lengths) // case["page"]) * case["page"]
    moves = 0.0
    for L in lengths:                              # kept keys among those behind the budget, in random order
        moves += min(L, case["budget"]) * max(0, L - case["budget"]) / L * G
    return {"bytes": 8 * n + 8 * cap * case["B"] * G + moves * 4 * row, "flops": 0}


# ------------------------------------------------------------------------------------------- the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attn": _exact_attn, "evict": _exact_evict, "logprobs": _exact_logprobs}[case["kind"]](case, s)


def _exact_append(case, s):
    table, page = s["table"].tolist(), case["page"]
    for b, (n, count, first) in enumerate(zip(s["lengths"].tolist(), s["counts"].tolist(), s["first"].tolist())):
        done = 0
        while done < count:                        # what is left of a page at a time
            slot = n + done
            r, m = slot % page, min(page - slot % page, count - done)
            p = table[b][slot // page]
            s["k"][p, :, r:r + m] = s["k_new"][b, done:done + m].transpose(0, 1)
            s["v"][p, :, r:r + m] = s["v_new"][b, done:done + m].transpose(0, 1)
            done += m
        s["mass"][b, :, n:n + count] = 0.0
        s["positions"][b, :, n:n + count] = torch.arange(first, first + count, device=DEV)
    return {"k": s["k"], "v": s["v"], "positions": s["positions"], "mass": s["mass"]}


def _exact_attn(case, s):
    G, D, page = case["G"], case["D"], case["page"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    mass = None if s["mass"] is None else s["mass"].double()
    for b, n in enumerate(s["lengths"].tolist()):
        pages = s["table"][b, :-(-n // page)].long()
        for g in range(G):
            heads = slice(g * case["H"] // G, (g + 1) * case["H"] // G)
            k = s["k"][pages, g].reshape(-1, D)[:n].double()
            w = torch.softmax(s["q"][b, heads].double() @ k.T / math.sqrt(D), -1)
            out[b, heads] = w @ s["v"][pages, g].reshape(-1, D)[:n].double()
            if mass is not None:
                mass[b, g, :n] += w.sum(0)
    return {"out": out} if mass is None else {"out": out, "mass": mass}


def _exact_evict(case, s):
    budget, recent, sink, page = case["budget"], case["recent"], case["sink"], case["page"]
    mass, positions, table = s["mass"].cpu().numpy(), s["positions"].cpu().numpy(), s["table"].cpu().numpy()
    B, G, cap = mass.shape
    to_all, from_all = [], []
    for b, n in enumerate(s["lengths"].tolist()):
        for g in range(G):
            m, p = mass[b, g], positions[b, g]
            if n > budget:
                live = np.arange(n)
                safe = (p[:n] < sink) | (p[:n] > p[:n].max() - recent)
                by = np.lexsort((live, -m[:n].astype(np.float64), ~safe))       # safe ones, then by weight, then by slot
                keep = np.zeros(n, bool)
                keep[by[:budget]] = True
                to, frm = live[:budget][~keep[:budget]], live[budget:][keep[budget:]]
                m[to], p[to] = m[frm], p[frm]
                to_all += [(table[b, i // page], g, i % page) for i in to]
                from_all += [(table[b, i // page], g, i % page) for i in frm]
            m[min(n, budget):], p[min(n, budget):] = 0.0, -1
    if to_all:
        to, frm = (torch.tensor(np.array(x), device=DEV, dtype=torch.long).T for x in (to_all, from_all))
        for pool in (s["k"], s["v"]):
            pool[to[0], to[1], to[2]] = pool[frm[0], frm[1], frm[2]].clone()
    return {"k": s["k"], "v": s["v"], "mass": torch.from_numpy(mass).to(DEV), "positions": torch.from_numpy(positions).to(DEV),
            "lengths": s["lengths"].clamp(max=budget)}


def _exact_logprobs(case, s):
    parts = []
    for x, t in zip(s["logits"].split(64), s["tokens"].split(64)):
        x = x.double()
        lp = x - torch.logsumexp(x, -1, keepdim=True)
        found = {"logprobs": lp.gather(1, t.view(-1, 1)).view(-1), "entropy": -(lp.exp() * lp).sum(-1)}
        if case["top"]:
            value, index = torch.sort(lp, dim=-1, descending=True, stable=True)
            found["top_logprobs"], found["top_tokens"] = value[:, :case["top"]], index[:, :case["top"]]
        parts.append(found)
    return {name: torch.cat([p[name] for p in parts]) for name in parts[0]}
