"""Rows that calls on pages meet at the ends of their life: tables that are
full, sequences that have ended, pages that ran out. Whole numbers are equal,
pools are bit-identical."""

from __future__ import annotations

import contextlib
import importlib

import numpy as np
import pytest
import torch

from test_gpu_pages import DEV, P, _bits, _copied, _i32, _pool, plain_compact, plain_release

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def pages(fi):
    return importlib.import_module("llm-inference-runtime_b200.pages")


@contextlib.contextmanager
def _status(fi, lir, want):
    """The device status that the calls inside leave."""
    saved, fi._CHECK = fi._CHECK, False
    try:
        yield
        assert lir._lib.device_status() == want
    finally:
        fi._CHECK = saved


# ------------------------------------------------------- rows that fill their table
@pytest.mark.parametrize("extra", [1, 16, 1000])
def test_compact_follows_the_entries_of_a_row_past_its_table(pages, fi, lir, extra):
    """The length is reported, once, and the entries point at the same tokens
    as before; beside it a row whose table has room."""
    tables = np.array([[9, 7, 5], [8, 2, -1]])
    refs = np.array([0, 0, 1, 0, 0, 2, 0, 1, 1, 1])
    lens = np.array([3 * P + extra, 2 * P])
    full = np.minimum(lens, 3 * P)
    want_t, want_r, want_m, want_c, copies = plain_compact(tables, full, refs)
    pool = _pool(len(refs), 2)
    want_pool, t, c = _copied(pool, copies), _i32(tables), _i32(refs)
    with _status(fi, lir, lir._lib.PA_ERR_DEVICE_CHECK):
        remap, counts = pages.compact_pages(pool, t, _i32(lens), c)
        assert counts.tolist() == [want_c[0], want_c[1], 1]
    assert np.array_equal(t.cpu().numpy(), want_t) and np.array_equal(c.cpu().numpy(), want_r)
    assert np.array_equal(remap.cpu().numpy(), want_m)
    assert torch.equal(_bits(pool), _bits(want_pool))


def test_compact_and_free_after_a_fork_that_found_a_full_table(pages, fi, lir):
    """As the calls' documentation has it: lengths that count the token to come
    as far as the table has room."""
    tables = _i32([[6, 7], [4, 5]])
    lens, refs = _i32([2 * P, P + 3]), _i32([0, 0, 0, 0, 1, 1, 1, 1])
    pool = _pool(8, 1)
    fresh = pool.clone()
    with _status(fi, lir, lir._lib.PA_ERR_DEVICE_CHECK):
        t, n, counts = pages.fork_sequences(pool, tables, lens, _i32([0, 1]), refs)
        assert counts.tolist() == [0, 0, 1]  # no room for row 0's next token
    held = (n + 1).clamp(max=P * t.shape[1])
    with _status(fi, lir, 0):
        remap, counts = pages.compact_pages(pool, t, held, refs)
        assert counts.tolist() == [4, 4, 0] and t.tolist() == [[2, 3], [0, 1]]
        for new, old in ((2, 6), (3, 7), (0, 4), (1, 5)):
            assert torch.equal(_bits(pool[:, new]), _bits(fresh[:, old]))
        assert pages.free_sequences(t, held, refs).tolist() == [4, 4, 0]
    assert (refs == 0).all() and (t == -1).all()


def test_release_leaves_a_row_past_its_table(pages, fi, lir):
    tables, refs = np.array([[0, 1], [2, 3]]), np.array([1, 1, 1, 1])
    for call in (lambda t, n, c: pages.free_sequences(t, n, c),
                 lambda t, n, c: pages.evict_window_pages(t, n, c, 0)):
        t, n, c = _i32(tables), _i32([2 * P + 1, 2 * P]), _i32(refs)
        with _status(fi, lir, lir._lib.PA_ERR_DEVICE_CHECK):
            assert call(t, n, c)[2] == 1
        assert t[0].tolist() == [0, 1] and n[0] == 2 * P + 1 and c[:2].tolist() == [1, 1]
    want_t, want_r, _ = plain_release(tables[1:], np.array([2 * P]), refs, 0, 0)
    assert t[1].tolist() == want_t[0].tolist() and c.tolist() == want_r.tolist()
