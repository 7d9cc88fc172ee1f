"""Which caches a Transformer keeps for the mode a generation asks for: the paging that a caller chose outlives calls in other modes."""
import pytest
import torch

from socket_b200.model import ModelArgs, Transformer
from socket_b200.paged import Paging

CHOSEN = Paging(page=16, budget=96, recent=8, sink=2, every=4)


def _model():
    return Transformer(ModelArgs.from_name("tiny", n_layer=2)).float().init_random(seed=0, std=0.05)


@pytest.mark.parametrize("between", [["dense"], ["sparse", "dense"], ["dense", "paged", "sparse"]])
@pytest.mark.parametrize("again", ["paged", None])
def test_chosen_paging_outlives_calls_in_other_modes(between, again):
    model = _model().use_pages(CHOSEN)
    for mode in between:
        model.choose_mode(mode)
        assert model.paging == (CHOSEN if mode == "paged" else None)
    model.choose_mode(again)
    assert model.paging == CHOSEN and model.default_mode == "paged"
    model.setup_caches(2, 200)
    assert model.pages.page == 16 and all(layer.attention.kv_cache.mass is not None for layer in model.layers)


def test_a_mode_of_one_call_is_not_the_next_ones():
    model = _model()
    model.choose_mode("paged")
    assert model.paging == Paging() and model.default_mode == "sparse"
    model.choose_mode(None)
    assert model.paging is None and model.default_mode == "sparse"


def test_caches_are_kept_where_the_mode_fits_them():
    for model, modes in ((_model().use_pages(CHOSEN), (None, "paged")), (_model(), (None, "sparse", "dense"))):
        model.setup_caches(1, 64)
        caches = [layer.attention.kv_cache for layer in model.layers]
        for mode in modes:
            model.choose_mode(mode)
            model.setup_caches(1, 64)
            assert [layer.attention.kv_cache for layer in model.layers] == caches


def test_paging_is_given_up():
    model = _model().use_pages(CHOSEN)
    model.use_pages(None)
    assert model.paging is None and model.default_mode == "sparse"
    model.choose_mode("paged")
    assert model.paging == Paging()


def test_caches_in_pages_decode_with_their_own_mode():
    """No mode named: that of the caches that are there, whoever chose them."""
    model = _model()
    model.choose_mode("paged")
    model.setup_caches(1, 64)
    model.setup_decode(1, use_graph=False)
    assert model._mode == "paged"
    model = _model().use_pages(CHOSEN)
    model.choose_mode("dense")
    model.setup_caches(1, 64)
    with pytest.raises(RuntimeError, match="not in pages"):
        model.setup_decode(1, use_graph=False)
