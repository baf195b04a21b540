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


# ---------------------------------------------------------- sequences that have ended
def plain_fork(tables, lens, refs, parents, all_held=False):
    """(tables, lens, refs, counts, copies), with -1 for a parent of none."""
    rows, width = tables.shape
    lens, refs, out = lens.copy(), refs.copy(), np.full_like(tables, -1)
    out_lens, lost = np.zeros_like(lens), set()
    for s in range(rows):
        if all_held and lens[s] % P and tables[s, lens[s] // P] < 0:
            lost.add(s)
            lens[s] = lens[s] // P * P
    for r in range(rows):
        for page in tables[r, :-(-lens[r] // P)]:
            if page >= 0:
                refs[page] -= 1
    alive = [r for r in range(rows) if parents[r] != -1]
    for r in alive:
        s = parents[r]
        out_lens[r] = lens[s]
        for j in range(lens[s] // P):
            out[r, j] = tables[s, j]
            if out[r, j] >= 0:
                refs[out[r, j]] += 1
    last = {r: int(tables[parents[r], out_lens[r] // P]) for r in alive if out_lens[r] % P}
    held = {page for page in last.values() if refs[page] > 0}
    kept, wants, missing = set(), [], 0
    for r in alive:
        at = out_lens[r] // P
        if parents[r] in lost or at >= width:
            missing += 1
        elif r in last and last[r] not in held | kept:
            kept.add(last[r])
            refs[last[r]] += 1
            out[r, at] = last[r]
        else:
            wants.append(r)
    free = [i for i in range(len(refs)) if refs[i] == 0]
    copies = []
    for r, page in zip(wants, free):
        out[r, out_lens[r] // P] = page
        refs[page] = 1
        if r in last:
            copies.append((last[r], page))
    for r in wants[len(free):]:
        missing += 1
        if all_held:
            out_lens[r] = out_lens[r] // P * P
    return out, out_lens, refs, [len(copies), min(len(wants), len(free)), missing], copies


def _fork(pages, pool, t, n, parents, c):
    """One fork against the plain one; returns the new state."""
    tables, lens, refs = (x.cpu().numpy().astype(np.int64) for x in (t, n, c))
    want_t, want_l, want_r, want_c, copies = plain_fork(tables, lens, refs, parents)
    want_pool = _copied(pool, copies)
    t, n, counts = pages.fork_sequences(pool, t, n, _i32(parents), c)
    assert counts.tolist() == want_c
    assert np.array_equal(t.cpu().numpy(), want_t) and np.array_equal(n.cpu().numpy(), want_l)
    assert np.array_equal(c.cpu().numpy(), want_r)
    assert torch.equal(_bits(pool), _bits(want_pool))
    return t, n


def _references(tables, total):
    live = tables[tables >= 0].long()
    return torch.zeros(total, dtype=torch.int32, device=DEV).index_add_(
        0, live, torch.ones_like(live, dtype=torch.int32))


@pytest.mark.parametrize("seed", range(6))
@pytest.mark.parametrize("rows", [1, 5, 40, 1300])
def test_fork_of_rows_that_end(pages, seed, rows):
    """Any rows end, with and without rows that continue them, and stay ended."""
    rng = np.random.RandomState(100 * seed + rows)
    lens = rng.randint(0, 70, rows)
    total = 10 * rows
    tables = np.full((rows, 6), -1, dtype=np.int64)
    ids = rng.permutation(total).tolist()
    for r in range(rows):
        for j in range(-(-lens[r] // P)):
            tables[r, j] = ids.pop()
    t, n, pool = _i32(tables), _i32(lens), _pool(total, 1, 1, 8)
    c = _references(t, total)
    for step in range(3):
        parents = rng.randint(0, rows, rows)
        parents[rng.rand(rows) < (1.0 if seed == 0 and step == 1 else 0.4)] = -1
        t, n = _fork(pages, pool, t, n, parents, c)
        # (the token to come of the rows that go on is appended)
        n += _i32(parents >= 0)
        assert torch.equal(c, _references(t, total))
    pages.free_sequences(t, n, c)
    assert (c == 0).all()


@pytest.mark.parametrize("how", ["freed", "stopped", "ended with its pages"])
def test_beam_search_steps_beside_a_request_that_has_ended(pages, fi, how):
    """Of three requests the second ends; in every later step the counts are
    the tables' own, and the pool does not drain."""
    beam = importlib.import_module("llm-inference-runtime_b200.beam")
    batch, beams, vocab, total, prompt = 3, 4, 60, 64, 2 * P
    rows = batch * beams
    g = torch.Generator().manual_seed(7)
    pool = _pool(total, 2, 1, 8)
    t = torch.full((rows, 8), -1, dtype=torch.int32, device=DEV)
    t[:, :2] = torch.arange(rows * 2, device=DEV).view(rows, 2).int()
    n = torch.full((rows,), prompt, dtype=torch.int32, device=DEV)
    c = _references(t, total)
    scores = -torch.rand(batch, beams, generator=g).to(DEV)
    active = torch.ones(batch, dtype=torch.bool, device=DEV)
    most = 0
    for step in range(40):
        if step == 5:
            mine = slice(beams, 2 * beams)
            if how == "freed":  # (the step's tokens are in: lengths are what the rows hold)
                pages.free_sequences(t[mine], n[mine], c)
            elif how == "stopped":
                scores[1] = -float("inf")
            active[1] = False
        if how == "stopped":
            active = (scores > -float("inf")).any(1)
        logits = (torch.randn(batch, beams, vocab, generator=g) * 2).to(DEV)
        got = beam.beam_search_step(logits, scores, pool, t, n, c, active=active)
        assert got["counts"][2] == 0
        t, n, scores = got["block_tables"], got["seq_lens"], got["scores"]
        on = active.repeat_interleave(beams)
        if step >= 5:
            assert (got["parents"][1] == -1).all() and (t[~on] == -1).all() and (n[~on] == 0).all()
            if how == "stopped":
                scores[1] = -float("inf")
        assert torch.equal(got["parents"].view(-1)[on] // beams,
                           torch.arange(batch, device=DEV).int().repeat_interleave(beams)[on])
        n = n + on
        assert (n[on] == prompt + step + 1).all() and (t[on, (prompt + step) // P] >= 0).all()
        assert torch.equal(c, _references(t, total))
        most = max(most, int((c > 0).sum()))
    assert most < total
    assert int((c > 0).sum()) <= 2 * beams * 5


def test_active_is_checked(fi):
    beam = importlib.import_module("llm-inference-runtime_b200.beam")
    x, s = torch.zeros(2, 3, 10, device=DEV), torch.zeros(2, 3, device=DEV)
    n, t, c = _i32(np.zeros(6)), _i32(np.zeros((6, 2))), _i32(np.ones(4))
    for bad in (torch.ones(2, device=DEV), torch.ones(3, dtype=torch.bool, device=DEV),
                torch.ones(2, 3, dtype=torch.bool, device=DEV), torch.ones(2, dtype=torch.bool)):
        with pytest.raises(ValueError, match="active"):
            beam.beam_search_step(x, s, _pool(4), t, n, c, active=bad)


# ------------------------------------------------------------- pages that ran out
def _fork_held(pages, fi, lir, pool, t, n, parents, c):
    tables, lens, refs = (x.cpu().numpy().astype(np.int64) for x in (t, n, c))
    want_t, want_l, want_r, want_c, copies = plain_fork(tables, lens, refs, parents, True)
    want_pool = _copied(pool, copies)
    with _status(fi, lir, lir._lib.PA_ERR_DEVICE_CHECK if want_c[2] else 0):
        t, n, counts = pages.fork_sequences(pool, t, n, _i32(parents), c, all_held=True)
        assert counts.tolist() == want_c
    assert np.array_equal(t.cpu().numpy(), want_t) and np.array_equal(n.cpu().numpy(), want_l)
    assert np.array_equal(c.cpu().numpy(), want_r)
    assert torch.equal(_bits(pool), _bits(want_pool))
    return t, n, want_c


def test_forks_after_a_fork_that_found_no_page(pages, fi, lir):
    """The lost tokens are counted in every fork, never replaced by the tokens
    of a free page."""
    t, n, c = _i32([[0, 1, -1], [2, 3, -1]]), _i32([20, 20]), _i32([1, 1, 1, 1])
    pool = _pool(4, 2, 1, 8)
    c[1] += 1  # row 0's unfinished page has another holder: it needs a copy
    t, n, counts = _fork_held(pages, fi, lir, pool, t, n, np.array([0, 1]), c)
    assert counts == [0, 0, 1] and n.tolist() == [16, 20] and t.tolist()[0] == [0, -1, -1]
    # pages are free again, the caller counts a token that had no page
    c = torch.cat([c, torch.zeros(4, dtype=torch.int32, device=DEV)])
    pool = torch.cat([pool, _pool(4, 2, 1, 8, seed=1)], 1)
    for _ in range(2):
        t, n, counts = _fork_held(pages, fi, lir, pool, t, n + 1, np.array([0, 1]), c)
        assert counts[2] == 1 and n[0] == 16 and t[0].tolist() == [0, -1, -1]
    # not counted, the row goes on from its full pages
    n[1] += 1
    t, n, counts = _fork_held(pages, fi, lir, pool, t, n, np.array([0, 1]), c)
    assert counts == [0, 1, 0] and n[0] == 16 and t[0, 1] >= 0
    # another row continues a lost one: it shares the full page and is counted
    t[0, 1] = -1
    n[0] = 18
    t, n, counts = _fork_held(pages, fi, lir, pool, t, n, np.array([0, 0]), c)
    assert counts[2] == 2 and n.tolist() == [16, 16] and c[0] == 2


def crowded(seed, rows, steps=5):
    """Tables, lengths, counts, the pages that others hold (half of them), and
    for each step parents and which rows have a token counted for which there
    was no page."""
    rng = np.random.RandomState(1000 * seed + rows)
    lens = rng.randint(0, 60, rows)
    need = sum(-(-x // P) for x in lens)
    tables = np.full((rows, 6), -1, dtype=np.int64)
    ids = rng.permutation(need + rows // 16).tolist()
    for r in range(rows):
        for j in range(-(-lens[r] // P)):
            tables[r, j] = ids.pop()
    others = (rng.rand(need + rows // 16) < 0.5).astype(np.int64)
    others[ids] = 0
    refs = others.copy()
    np.add.at(refs, tables[tables >= 0], 1)
    plan = []
    for _ in range(steps):
        parents = np.where(rng.rand(rows) < 0.8, np.arange(rows), rng.randint(0, rows, rows))
        parents[rng.rand(rows) < 0.05] = -1
        plan.append((parents, rng.rand(rows) < 0.5))
    return tables, lens, refs, others, plan


def tokens_to_come(tables, lens, parents, anyway):
    """Which rows' lengths grow after a fork."""
    width = tables.shape[1]
    at = np.minimum(lens // P, width - 1)
    has = tables[np.arange(len(lens)), at] >= 0
    return (has | anyway) & (parents >= 0) & (lens < P * width)


@pytest.mark.parametrize("seed", range(6))
@pytest.mark.parametrize("rows", [12, 60, 1100])
def test_forks_in_a_pool_that_is_too_small(pages, fi, lir, seed, rows):
    """Random steps, some rows ending, more pages wanted than there are; what
    the lengths count is always in pages that the counts hold."""
    tables, lens, refs, others, plan = crowded(seed, rows)
    t, n, c, pool = _i32(tables), _i32(lens), _i32(refs), _pool(len(refs), 1, 1, 8)
    short = 0
    for parents, anyway in plan:
        t, n, counts = _fork_held(pages, fi, lir, pool, t, n, parents, c)
        short += counts[2]
        assert torch.equal(c, _references(t, len(refs)) + _i32(others))
        tables, lens = t.cpu().numpy(), n.cpu().numpy()
        for r in range(rows):
            assert (tables[r, :-(-lens[r] // P)] >= 0).all()
        n = n + _i32(tokens_to_come(tables, lens, parents, anyway))
    assert short > 0


def test_a_beam_search_step_reports_a_lost_page_until_the_beam_ends(fi, lir):
    beam = importlib.import_module("llm-inference-runtime_b200.beam")
    t, n = _i32([[0, 1, -1], [0, 2, -1]]), _i32([20, 20])
    c, pool = _i32([2, 2, 1]), _pool(3, 1, 1, 8)
    scores = torch.zeros(1, 2, device=DEV)
    # (apart by far: each beam goes on with itself)
    logits = torch.zeros(1, 2, 50, device=DEV)
    logits[0, 0, 7] = logits[0, 1, 9] = 60.0
    for step in range(3):
        with _status(fi, lir, lir._lib.PA_ERR_DEVICE_CHECK):
            got = beam.beam_search_step(logits, scores, pool, t, n, c)
            assert got["parents"].tolist() == [[0, 1]] and got["counts"].tolist() == [0, 0, 1]
        t, n, scores = got["block_tables"], got["seq_lens"], got["scores"]
        assert n.tolist() == [16, 20 + step] and t[0].tolist() == [0, -1, -1]
        n = n + 1
        if step == 0:  # there would be a page now
            c = torch.cat([c, torch.zeros(2, dtype=torch.int32, device=DEV)])
            pool = torch.cat([pool, _pool(2, 1, 1, 8, seed=1)], 1)
    with _status(fi, lir, 0):
        got = beam.beam_search_step(logits, scores, pool, t, n, c,
                                    active=torch.tensor([False], device=DEV))
        assert (got["block_tables"] == -1).all() and c.tolist() == [0, 1, 0, 0, 0]


def test_steps_captured_and_replayed_while_requests_end(fi, lir):
    """One graph of a step; which requests go on changes between replays."""
    beam = importlib.import_module("llm-inference-runtime_b200.beam")
    batch, beams, vocab, total = 4, 2, 300, 40
    rows, length = batch * beams, P + 5
    tables = torch.arange(rows * 2, device=DEV).view(rows, 2).int()
    t, n = torch.cat([tables, torch.full_like(tables, -1)], 1), _i32(np.full(rows, length))
    refs = _references(t, total)
    g = torch.Generator().manual_seed(9)
    x = torch.randn(batch, beams, vocab, generator=g).to(DEV)
    s = -torch.rand(batch, beams, generator=g).to(DEV)
    active = torch.ones(batch, dtype=torch.bool, device=DEV)
    c, fresh = refs.clone(), _pool(total, 2, 1, 8)
    pool = fresh.clone()
    with _status(fi, lir, 0):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            beam.beam_search_step(x, s, fresh.clone(), t, n, refs.clone(), active=active)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = beam.beam_search_step(x, s, pool, t, n, c, active=active)
        for on in ([1, 1, 1, 1], [1, 0, 1, 0], [0, 0, 0, 0], [0, 1, 1, 1]):
            active.copy_(torch.tensor(on, dtype=torch.bool))
            x.copy_(torch.randn(batch, beams, vocab, generator=g))
            c.copy_(refs)
            pool.copy_(fresh)
            graph.replay()
            _, choice, _ = beam.beam_search_select(x, s, beams)
            parents = choice.masked_fill(~active[:, None], -1).view(-1).cpu().numpy()
            want_t, want_l, want_r, want_c, copies = plain_fork(
                t.cpu().numpy().astype(np.int64), n.cpu().numpy().astype(np.int64),
                refs.cpu().numpy().astype(np.int64), parents, True)
            assert got["parents"].view(-1).tolist() == parents.tolist()
            assert got["counts"].tolist() == want_c
            assert np.array_equal(got["block_tables"].cpu().numpy(), want_t)
            assert np.array_equal(got["seq_lens"].cpu().numpy(), want_l)
            assert np.array_equal(c.cpu().numpy(), want_r)
            assert torch.equal(_bits(pool), _bits(_copied(fresh, copies)))
