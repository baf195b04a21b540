"""Sizes and strides at the limits of the page and beam calls."""

from __future__ import annotations

import importlib

import numpy as np
import pytest
import torch

from test_gpu_beam import DEV, P, _random, check, plain_select
from test_gpu_pages import _i32, _pool

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def beam(fi):
    return importlib.import_module("llm-inference-runtime_b200.beam")


@pytest.fixture(scope="module")
def pages(fi):
    return importlib.import_module("llm-inference-runtime_b200.pages")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("batch", [65535, 65536, 70001])
def test_select_for_many_requests(beam, dtype, batch):
    """Seven requests' logits over and over: every copy gets its request's
    choice, in rows of its own."""
    few, scores = _random(7, 2, 9, dtype, seed=1)
    which = torch.arange(batch, device=DEV) % 7
    best, parents, tokens = beam.beam_search_select(few[which], scores[which], 3)
    check(beam, few, scores, 3)
    want, want_p, want_t = beam.beam_search_select(few, scores, 3)
    shift = (2 * (torch.arange(batch, device=DEV) - which)).int()
    assert torch.equal(best, want[which]) and torch.equal(tokens, want_t[which])
    assert torch.equal(parents, want_p[which] + shift[:, None])


def test_tensors_of_one_entry_have_any_stride(pages):
    """One sequence, one page: views whose only entry has no neighbour."""
    one = lambda v: torch.tensor([[v, 9], [9, 9]], dtype=torch.int32, device=DEV)[:1, 0]  # noqa: E731
    assert one(3).stride() == (2,)
    tables, lens, refs = _i32([[0]]), one(P), one(1)
    counts = pages.free_sequences(tables, lens, refs)
    assert counts.tolist() == [1, 1, 0] and tables.tolist() == [[-1]]
    assert lens.tolist() == [0] and refs.tolist() == [0]
    # a column of a table, row after row
    wide = _i32([[0, 5], [1, 5], [2, 5]])
    t, n, c = wide[:, :1], _i32([P, 3, 0]), _i32([1, 1, 1])
    assert pages.evict_window_pages(t, n, c, 0).tolist() == [0, 0, 0]
    refs = one(1)
    remap, counts = pages.compact_pages(_pool(1), _i32([[0]]), one(P), refs)
    assert remap.tolist() == [0] and counts.tolist() == [1, 0, 0]
    t, n, counts = pages.fork_sequences(_pool(1), _i32([[0]]), one(5), one(0), one(1))
    assert t.tolist() == [[0]] and n.tolist() == [5] and counts.tolist() == [0, 0, 0]
    with pytest.raises(ValueError, match="contiguous"):
        pages.free_sequences(_i32([[0], [1]]), _i32([[1, 0], [1, 0]])[:, 0], _i32([1, 1]))


def test_beams_at_their_limits(beam, pages):
    """32 beams step, 256 beams select, one more of each is refused."""
    logits, scores = _random(1, 256, 40, torch.float32, seed=3)
    check(beam, logits, scores, 32)
    x, s = logits[:, :32], scores[:, :32].contiguous()
    t = _i32(np.arange(32)[:, None])
    c, n, pool = _i32(np.ones(96)), _i32(np.full(32, 7)), _pool(96, 1, 1, 8)
    c[32:] = 0
    _, want_p, want_t, _ = plain_select(x, s, 32)
    got = beam.beam_search_step(x, s, pool, t, n, c)
    assert np.array_equal(got["parents"].cpu().numpy(), want_p)
    assert np.array_equal(got["tokens"].cpu().numpy(), want_t) and got["counts"][2] == 0
    for beams in (33, 257):
        x, s = torch.zeros(1, beams, 300, device=DEV), torch.zeros(1, beams, device=DEV)
        with pytest.raises(NotImplementedError, match="at most 32"):
            beam.beam_search_step(x, s, pool, _i32(np.zeros((beams, 1))), _i32(np.zeros(beams)), c)
