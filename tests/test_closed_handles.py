"""Closed pools, plans and contexts are refused by the binding before the library is called: no device."""
from types import SimpleNamespace

import pytest

import gguf_runner_b200 as g


def plan(ctx, pages, handle):
    batch = g.Batch.__new__(g.Batch)
    batch._L, batch.ctx, batch.pages, batch._h = None, ctx, pages, handle
    return batch


@pytest.mark.parametrize("ctx,pages,handle", [(1, None, 1), (None, 1, 1), (1, 1, None)])
def test_set_refuses_what_has_been_closed(ctx, pages, handle):
    batch = plan(SimpleNamespace(_h=ctx), SimpleNamespace(_h=pages, page_size=16), handle)
    try:
        with pytest.raises(ValueError):
            batch.set([1], [1], [[0]])
    finally:
        batch._h = None


def test_a_plan_on_a_closed_pool_is_not_a_plan_without_pages():
    with pytest.raises(ValueError):
        g.Batch(SimpleNamespace(_h=None), SimpleNamespace(_h=None, page_size=16), "bf16", 1, 1, 1)
