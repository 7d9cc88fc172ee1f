"""What the paged cache's and the log probabilities' entry points refuse before anything is launched."""
import ctypes as C
import os
import re

import pytest
import torch

from socket_b200 import _lib, few_rows, paged

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
A = 1 << 20                                                   # an address nothing on the host reads


def _cache(**over):
    p = _lib.PagedCacheParams()
    for i, name in enumerate(("k", "v", "table", "lengths", "mass", "positions", "status")):
        setattr(p, name, A * (i + 1))
    p.k_rs = p.v_rs = 128
    p.k_hs = p.v_hs = 64 * 128
    p.k_ps = p.v_ps = 8 * 64 * 128
    p.table_ld = p.width = 16
    p.n_pages, p.dtype, p.B, p.G, p.D, p.page = 100, _lib.SK_BF16, 2, 8, 128, 64
    p.mass_hs = p.pos_hs = 1024
    p.mass_bs = p.pos_bs = 8192
    for k, v in over.items():
        setattr(p, k, v)
    return p


def _attn(c, q=A, out=2 * A, H=32, extra=0, ws=4 * A, ws_bytes=1 << 40, q_hs=128, o_hs=128):
    return _lib.lib().sk_paged_attn(C.byref(c), q, 32 * 128, q_hs, out, 32 * 128, o_hs, H, extra, 0.1, ws, ws_bytes, None)


def _append(c, k=A, v=A, S=4, ss=1024):
    return _lib.lib().sk_paged_append(C.byref(c), k, 4096, ss, 128, v, 4096, 1024, 128, S, None, None, None)


def _evict(c, budget=512, recent=64, sink=4, mo=A, ws=A, ws_bytes=1 << 40):
    return _lib.lib().sk_paged_evict(C.byref(c), budget, recent, sink, mo, 8192, 1024, A, 8192, 1024, A, ws, ws_bytes, None)


def test_params_struct_matches_header_fields():
    text = open(os.path.join(ROOT, "include", "socket_b200.h")).read()
    body = text[text.index("typedef struct sk_paged_cache"):text.index("} sk_paged_cache;")]
    fields = []
    for decl in body.split("{", 1)[1].split(";"):
        if decl.strip():
            fields += [re.findall(r"(\w+)\s*$", name.strip())[0] for name in decl.strip().split(",")]
    assert fields == [f[0] for f in _lib.PagedCacheParams._fields_]


@pytest.mark.parametrize("call", [_attn, _append, _evict])
@pytest.mark.parametrize("over,status", [
    (dict(dtype=3), -1), (dict(page=8), -1), (dict(page=48), -1), (dict(page=0), -1), (dict(B=-1), -1), (dict(G=0), -1), (dict(D=0), -1),
    (dict(width=-1), -1), (dict(table_ld=15), -1), (dict(k=None), -1), (dict(v=None), -1), (dict(table=None), -1), (dict(lengths=None), -1),
    (dict(width=1 << 25, table_ld=1 << 25), -1), (dict(D=264), -2), (dict(D=100), -2), (dict(k=A + 8), -3), (dict(v=A + 2), -3), (dict(k_rs=132), -3),
    (dict(v_hs=4), -3), (dict(k_ps=12), -3), (dict(dtype=0, D=66), -2), (dict(dtype=0, k_rs=130), -3)])
def test_caches_that_are_refused(call, over, status):
    assert call(_cache(**over)) == status, _lib.lib().sk_last_error()
    assert _lib.lib().sk_last_error()


def test_calls_that_are_refused():
    lib = _lib.lib()
    c = _cache()
    assert _attn(c, q=None) == -1 and _attn(c, out=None) == -1 and _attn(c, H=30) == -1 and _attn(c, H=0) == -1 and _attn(c, extra=-1) == -1
    assert _attn(c, q=A + 2) == -3 and _attn(c, out=A + 8) == -3 and _attn(c, q_hs=132) == -3 and _attn(c, o_hs=4) == -3
    assert _append(c, k=None) == -1 and _append(c, S=-1) == -1 and _append(c, v=A + 4) == -3 and _append(c, ss=1020) == -3
    assert _evict(c, budget=0) == -1 and _evict(c, recent=-1) == -1 and _evict(c, sink=-1) == -1 and _evict(c, budget=67) == -1
    assert _evict(c, mo=None) == -1 and _evict(_cache(mass=None)) == -1 and _evict(_cache(positions=None)) == -1
    assert _evict(c, recent=2 ** 31 - 1, sink=2 ** 31 - 1) == -1
    need = lib.sk_paged_attn_workspace_bytes(C.byref(c), 32)
    if need:
        assert _attn(c, ws=None) == -4 and _attn(c, ws_bytes=need - 1) == -4 and _attn(c, ws=A + 8) == -3
    need = lib.sk_paged_evict_workspace_bytes(C.byref(c), 512)
    if need:
        assert _evict(c, ws=None) == -4 and _evict(c, ws_bytes=need - 1) == -4 and _evict(c, ws=A + 8) == -3
    assert lib.sk_paged_attn_workspace_bytes(C.byref(_cache(page=5)), 32) == 0 and lib.sk_paged_attn_workspace_bytes(C.byref(c), 31) == 0
    assert lib.sk_paged_evict_workspace_bytes(C.byref(c), 0) == 0
    for call in (_attn, _append, _evict):                     # nothing to do is no error
        assert call(_cache(B=0, lengths=None, table=None, k=None, v=None)) == 0
    assert _append(c, S=0, k=None, v=None) == 0


@pytest.mark.parametrize("library", ["step", "blocks"])
def test_log_probabilities_that_are_refused(library):
    def call(logits=A, dtype=1, ld=100, rows=4, vocab=100, token=A, top=3, lp=A, tl=A, tt=A):
        args = (logits, dtype, ld, rows, vocab, token, top, lp, A, tl, tt, None, None)
        return _lib.lib().sk_token_logprobs(*args) if library == "step" else _lib.blocks().skb_token_logprobs(*args)

    for bad in (dict(logits=None), dict(dtype=7), dict(ld=99), dict(rows=-1), dict(vocab=0), dict(lp=None), dict(top=-1), dict(top=65),
                dict(top=5, vocab=4), dict(tl=None), dict(tt=None)):
        assert call(**bad) == -1, bad
    assert call(rows=0, logits=None) == 0


def test_cpu_tensors_are_refused():
    k = torch.zeros(4, 2, 16, 64)
    table, n = torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged.attn(torch.zeros(1, 4, 64), k, k, table, n)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged.append(torch.zeros(1, 1, 2, 64), torch.zeros(1, 1, 2, 64), k, k, table, n)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged.evict(k, k, table, n, torch.zeros(1, 2, 64), torch.zeros(1, 2, 64, dtype=torch.int32), budget=8)
    with pytest.raises(RuntimeError, match="CUDA"):
        few_rows.token_logprobs(torch.zeros(2, 10))


def test_page_tables_hand_out_and_take_back_pages():
    t = paged.PageTable(2, 100, 16, 9)
    assert t.width == 7 and t.table.tolist() == [[-1] * 7] * 2
    t.reserve(33)
    held = [x[:3] for x in t.table.tolist()]
    assert sorted(held[0] + held[1]) == list(range(6)) and all(x[3:] == [-1] * 4 for x in t.table.tolist()) and len(t.free) == 3
    t.reserve(48)                                             # still three pages each
    assert [x[:3] for x in t.table.tolist()] == held
    t.advance(48)
    assert t.lengths.tolist() == t.positions.tolist() == [48, 48] and t.length == t.position == 48
    with pytest.raises(RuntimeError, match="out of pages"):
        t.reserve(81)                                         # six pages each
    assert [x[:3] for x in t.table.tolist()] == held and len(t.free) == 3
    with pytest.raises(RuntimeError, match="113 slots"):
        t.reserve(113)
    t.hide()
    assert (t.table == -1).all()
    t.show()
    t.cut(17)
    assert t.length == 17 and t.position == 48 and [x[:2] for x in t.table.tolist()] == [x[:2] for x in held] and len(t.free) == 5
    t.reserve(64)
    pages = [p for x in t.table.tolist() for p in x if p >= 0]
    assert len(pages) == len(set(pages)) == 8
    t.reset()
    assert len(t.free) == 9 and t.lengths.tolist() == [0, 0] and (t.table == -1).all()


@pytest.mark.parametrize("over", [dict(page=8), dict(page=48), dict(budget=-1), dict(budget=10, recent=8, sink=3), dict(pages=-1),
                                  dict(budget=10, every=0), dict(recent=-1)])
def test_paging_that_is_refused(over):
    with pytest.raises(ValueError):
        paged.Paging(**over)
