"""Rotary tables that a captured decode graph may read stay allocated when larger ones replace them."""

import gc
import weakref

import pytest
import torch

import economize_b200 as eco
from economize_b200.techniques.eagle3 import Eagle3Config

from .helpers import tiny_model


def _alive(refs):
    gc.collect()
    return all(r() is not None for r in refs)


@pytest.mark.parametrize("of", ["model", "local", "none", "draft layer"])
def test_outgrown_tables_stay(of):
    overrides = {"local": dict(local_rope={"rope_theta": 500.0}), "none": dict(nope_layers=(0,))}.get(of, {})
    model = tiny_model(max_position_embeddings=64, **overrides)
    if of == "draft layer":
        layer = eco.apply(model, Eagle3Config()).techniques["eagle3"].layer
        tables = layer.rope
    elif of == "none":
        tables = lambda n=0: model._layer_rope(0, *model.rope_tables(n))  # noqa: E731
    else:
        tables = lambda n=0: model.rope_tables(n, local=of == "local")  # noqa: E731
    first = tables()
    values = [t.clone() for t in first]
    refs = [weakref.ref(t) for t in first]
    del first
    larger = tables(100)
    refs += [weakref.ref(t) for t in larger]
    assert larger[0].shape[0] == 100 and all(torch.equal(t[:64], v) for t, v in zip(larger, values))
    del larger
    assert tables(300)[0].shape[0] == 300
    assert _alive(refs)
    assert all(torch.equal(r(), v) for r, v in zip(refs, values))
