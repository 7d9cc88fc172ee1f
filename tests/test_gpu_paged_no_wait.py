"""Page bookkeeping and evictions between decoded tokens never wait for the device."""
import pytest
import torch

from socket_b200 import paged
from socket_b200.model import ModelArgs, Transformer

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture
def no_waits():
    """Calls that wait for the device raise."""
    def switch(on):
        torch.cuda.set_sync_debug_mode("error" if on else "default")
    yield switch
    switch(False)


def test_page_tables_are_shown_without_waiting(no_waits):
    t = paged.PageTable(3, 400, 16, device=DEV)
    seen = []
    no_waits(True)
    for length in range(1, 400, 7):                           # table behind table, none of them waited for
        t.reserve(length)
        seen.append((t.table.clone(), [list(h) for h in t.held]))
    t.hide()
    t.cut(33)
    seen.append((t.table.clone(), [list(h) for h in t.held]))
    t.advance(5)
    t.reset()
    seen.append((t.table.clone(), [[], [], []]))
    no_waits(False)
    for table, held in seen:
        assert table.tolist() == [h + [-1] * (t.width - len(h)) for h in held]


def test_tokens_and_evictions_do_not_wait(no_waits):
    model = Transformer(ModelArgs.from_name("tiny")).to(device=DEV, dtype=torch.bfloat16).init_random(seed=3, std=0.05)
    model.use_pages(paged.Paging(page=16, budget=64, recent=16, sink=4, every=8))
    prompt = torch.randint(0, 512, (2, 50), generator=torch.Generator().manual_seed(0)).to(DEV)
    model.setup_caches(2, 150)
    model.setup_decode(2, "paged")
    tok = torch.argmax(model.prefill(prompt), -1, keepdim=True)
    model.start_decode(tok, 50)
    for _ in range(30):                                       # through a first eviction
        model.decode_one_token()
    no_waits(True)
    for _ in range(40):
        model.decode_one_token()
    no_waits(False)
    assert model.pages.position == 120 and model.pages.lengths.tolist() == [model.pages.length] * 2 and model.pages.length < 72
    assert all(int(layer.attention.kv_cache.status) == 0 for layer in model.layers)
