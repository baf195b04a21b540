"""Pages on the device (evict, free, fork, compact) against plain Python.

Whole numbers throughout: tables, counts and lengths are equal, and the pool is
bit-identical."""

from __future__ import annotations

import importlib

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
P = 16


@pytest.fixture(scope="module")
def pages(fi):
    return importlib.import_module("llm-inference-runtime_b200.pages")


def _i32(a):
    return torch.as_tensor(np.ascontiguousarray(np.asarray(a, dtype=np.int32))).to(DEV)


def _held(length):
    return -(-length // P)


def _random_state(seed, rows, max_len, spare=7, shared=0.5, external=0.2, gone=0.1, lens=None):
    """Tables whose rows share pages, counts with holders outside the tables."""
    rng = np.random.RandomState(seed)
    if lens is None:
        lens = rng.randint(0, max_len + 1, rows)
    lens = np.asarray(lens)
    width = int(_held(lens.max()) + 1 + rng.randint(0, 3)) if rows else 1
    need = int(sum(_held(n) for n in lens))
    ids = rng.permutation(need + spare).tolist()
    tables = np.full((rows, width), -1, dtype=np.int64)
    for r in range(rows):
        n = _held(lens[r])
        if r and rng.rand() < shared:  # the head of an earlier row, at times all of it
            s = rng.randint(r)
            m = rng.randint(0, min(n, _held(lens[s])) + 1)
            if m == _held(lens[s]) and lens[s] % P and (lens[r] < lens[s]):
                m -= 1
            tables[r, :m] = tables[s, :m]
        else:
            m = 0
        for j in range(m, n):
            tables[r, j] = ids.pop()
        full = lens[r] // P
        tables[r, :full][rng.rand(full) < gone] = -1
        tables[r, n:] = rng.choice([-1, 10 ** 6])  # what lies behind is not read
    refs = np.zeros(need + spare, dtype=np.int64)
    for r in range(rows):
        held = tables[r, :_held(lens[r])]
        np.add.at(refs, held[held >= 0], 1)
    refs[rng.rand(len(refs)) < external] += 1
    return tables, lens.astype(np.int64), refs, rng


# ------------------------------------------------------------------ plain forms
def plain_release(tables, lens, refs, window, sinks):
    tables, refs = tables.copy(), refs.copy()
    gone = freed = 0
    for r, n in enumerate(lens):
        lo, hi = (0, _held(n)) if window is None else (_held(sinks), max(n - 1 - window, 0) // P)
        for j in range(lo, hi):
            page = tables[r, j]
            if page >= 0:
                refs[page] -= 1
                gone += 1
                freed += refs[page] == 0
                tables[r, j] = -1
    return tables, refs, [gone, freed, 0]


def plain_fork(tables, lens, refs, parents):
    """(tables, lens, refs, counts, copies)"""
    rows, width = tables.shape
    refs = refs.copy()
    for r in range(rows):
        held = tables[r, :_held(lens[r])]
        for page in held[held >= 0]:
            refs[page] -= 1
    out = np.full_like(tables, -1)
    for r, s in enumerate(parents):
        for j in range(lens[s] // P):
            out[r, j] = tables[s, j]
            if out[r, j] >= 0:
                refs[out[r, j]] += 1
    last = [tables[s, lens[s] // P] if lens[s] % P else -1 for s in parents]
    taken_by_others = {page for page in last if page >= 0 and refs[page] > 0}
    kept, wants = set(), []
    for r, page in enumerate(last):
        if page >= 0 and page not in taken_by_others and page not in kept:
            kept.add(page)
            refs[page] += 1
            out[r, lens[parents[r]] // P] = page
        elif lens[parents[r]] // P < width:
            wants.append(r)
    free = [i for i in range(len(refs)) if refs[i] == 0]
    copies, missing = [], sum(lens[s] // P >= width for s in parents)
    for k, r in enumerate(wants):
        if k >= len(free):
            missing += 1
            continue
        out[r, lens[parents[r]] // P] = free[k]
        refs[free[k]] = 1
        if last[r] >= 0:
            copies.append((last[r], free[k]))
    return out, lens[list(parents)], refs, [len(copies), min(len(wants), len(free)), missing], copies


def plain_compact(tables, lens, refs):
    n = int((refs > 0).sum())
    holes = [i for i in range(n) if refs[i] <= 0]
    movers = [i for i in range(n, len(refs)) if refs[i] > 0]
    remap = np.where(refs > 0, np.arange(len(refs)), -1)
    new = np.where(refs > 0, refs, 0)
    for s, d in zip(movers, holes):
        remap[s] = d
        new[d], new[s] = refs[s], 0
    out = tables.copy()
    for r, length in enumerate(lens):
        for j in range(_held(length)):
            if out[r, j] >= 0:
                out[r, j] = remap[out[r, j]]
    return out, new, remap, [n, len(movers), 0], list(zip(movers, holes))


def _pool(pages, layers=3, heads=2, d=64, dtype=torch.bfloat16, seed=0):
    g = torch.Generator().manual_seed(seed)
    n = layers * pages * 2 * heads * P * d
    x = torch.randint(-2 ** 15, 2 ** 15, (n,), generator=g, dtype=torch.int32).to(torch.int16)
    return x.view(dtype).view(layers, pages, 2, heads, P, d).to(DEV)


def _bits(t):
    return t.contiguous().view(torch.int16)


def _copied(pool, copies):
    want = pool.clone()
    for s, d in copies:
        if pool.dim() == 5:  # one layer
            want[d] = pool[s]
        else:
            want[:, d] = pool[:, s]
    return want


# -------------------------------------------------------------------- releasing
@pytest.mark.parametrize("window,sinks", [(0, 0), (15, 0), (16, 1), (17, 16), (100, 17), (40, 200),
                                          (5000, 4), (2 ** 31 - 1, 0), (0, 2 ** 31 - 1)])
@pytest.mark.parametrize("rows,max_len", [(1, 40), (9, 3000), (300, 200)])
def test_evict(pages, window, sinks, rows, max_len):
    tables, lens, refs, _ = _random_state(window % 83 + sinks % 7 + rows, rows, max_len)
    t, c = _i32(tables), _i32(refs)
    counts = pages.evict_window_pages(t, _i32(lens), c, window, sinks)
    want_t, want_r, want_c = plain_release(tables, lens, refs, window, sinks)
    assert np.array_equal(t.cpu().numpy(), want_t)
    assert np.array_equal(c.cpu().numpy(), want_r)
    assert counts.tolist() == want_c
    # a second call finds nothing more
    assert pages.evict_window_pages(t, _i32(lens), c, window, sinks).tolist() == [0, 0, 0]
    assert np.array_equal(c.cpu().numpy(), want_r)


def test_evict_long_rows(pages):
    tables, lens, refs, _ = _random_state(3, 5, 0, lens=[100000, 70000, 16, 99999, 33], shared=0.9)
    t, c = _i32(tables), _i32(refs)
    counts = pages.evict_window_pages(t, _i32(lens), c, 1000, 4)
    want_t, want_r, want_c = plain_release(tables, lens, refs, 1000, 4)
    assert np.array_equal(t.cpu().numpy(), want_t) and np.array_equal(c.cpu().numpy(), want_r)
    assert counts.tolist() == want_c


def test_free_some_rows_of_a_wider_table(pages):
    tables, lens, refs, _ = _random_state(8, 40, 900)
    wide = torch.full((40, tables.shape[1] + 5), 77, dtype=torch.int32, device=DEV)
    wide[:, :tables.shape[1]] = _i32(tables)
    t, n, c = wide[:, :tables.shape[1]], _i32(lens), _i32(refs)
    counts = pages.free_sequences(t[7:21], n[7:21], c)
    want_t, want_r, want_c = plain_release(tables[7:21], lens[7:21], refs, None, 0)
    tables[7:21], lens[7:21] = want_t, 0
    assert np.array_equal(t.cpu().numpy(), tables) and (wide[:, tables.shape[1]:] == 77).all()
    assert np.array_equal(c.cpu().numpy(), want_r) and np.array_equal(n.cpu().numpy(), lens)
    assert counts.tolist() == want_c
    assert pages.free_sequences(t[:0], n[:0], c).tolist() == [0, 0, 0]


def test_release_reports_what_it_cannot_do(pages, fi, lir):
    """A page outside the pool, one that nobody holds, a length past the
    table: reported, left as they are, the rest done."""
    tables = _i32([[0, 9, 2], [1, 3, 0], [4, 4, 4]])
    lens, refs = _i32([48, 48, 49]), _i32([2, 1, 1, 0, 5])
    fi._CHECK, saved = False, fi._CHECK
    try:
        counts = pages.free_sequences(tables, lens, refs)
        assert lir._lib.device_status() == lir._lib.PA_ERR_DEVICE_CHECK
    finally:
        fi._CHECK = saved
    assert counts.tolist() == [4, 3, 3]
    assert tables.tolist() == [[-1, 9, -1], [-1, 3, -1], [4, 4, 4]]
    assert lens.tolist() == [0, 0, 49] and refs.tolist() == [0, 0, 0, 0, 5]
    with pytest.raises(RuntimeError, match="device"):
        pages.free_sequences(_i32([[3]]), _i32([1]), refs)


# ------------------------------------------------------------------------- fork
def _check_fork(pages, tables, lens, refs, parents, pool=None, layers=3):
    pool = _pool(len(refs), layers) if pool is None else pool
    want_t, want_l, want_r, want_c, copies = plain_fork(tables, lens, refs, parents)
    want_pool = _copied(pool, copies)
    c = _i32(refs)
    old = _i32(tables)
    # a state may have too few free pages: the counts say so, and the status
    api = importlib.import_module("llm-inference-runtime_b200.flashinfer_api")
    api._CHECK, saved = False, api._CHECK
    try:
        t, n, counts = pages.fork_sequences(pool, old, _i32(lens), _i32(parents), c)
        status = api._lib.device_status()
    finally:
        api._CHECK = saved
    assert status == (api._lib.PA_ERR_DEVICE_CHECK if want_c[2] else 0)
    assert np.array_equal(old.cpu().numpy(), tables)
    assert counts.tolist() == want_c
    assert np.array_equal(t.cpu().numpy(), want_t)
    assert np.array_equal(n.cpu().numpy(), want_l)
    assert np.array_equal(c.cpu().numpy(), want_r)
    assert torch.equal(_bits(pool), _bits(want_pool))
    return t, n, c, pool


@pytest.mark.parametrize("seed", range(12))
@pytest.mark.parametrize("rows,max_len", [(1, 33), (4, 64), (37, 500), (200, 90)])
def test_fork_random(pages, seed, rows, max_len):
    tables, lens, refs, rng = _random_state(seed * 31 + rows, rows, max_len, spare=2 * rows)
    kind = seed % 4
    if kind == 0:
        parents = np.arange(rows)
    elif kind == 1:
        parents = np.zeros(rows, dtype=np.int64) + rng.randint(rows)
    else:
        parents = rng.randint(0, rows, rows)
    _check_fork(pages, tables, lens, refs, parents)


def test_fork_more_rows_than_one_pass(pages):
    tables, lens, refs, rng = _random_state(5, 2500, 60, spare=5000)
    _check_fork(pages, tables, lens, refs, rng.randint(0, 2500, 2500), layers=1)


@pytest.mark.parametrize("length", [0, 1, 15, 16, 17, 32, 33])
def test_fork_of_one_prompt_shared_by_all_rows(pages, length):
    """Beams of a first step: every row has the same table, unfinished page
    included; a prefix cache may hold that page too."""
    n = _held(length)
    for outside in (0, 1):
        tables = np.full((5, n + 1), -1, dtype=np.int64)
        tables[:, :n] = np.arange(n)[::-1]
        refs = np.zeros(n + 8, dtype=np.int64)
        refs[:n] = 5
        if n:
            refs[tables[0, n - 1]] += outside
        _check_fork(pages, tables, np.full(5, length), refs, np.zeros(5, dtype=np.int64))
        _check_fork(pages, tables, np.full(5, length), refs, np.array([4, 3, 3, 1, 4]))


def test_fork_pool_shapes(pages):
    """One layer, fp16, heads of 128, a pool whose layers and pages have gaps,
    and page blocks that are no multiple of the copy's slice."""
    tables, lens, refs, rng = _random_state(77, 12, 200, spare=24)
    parents = rng.randint(0, 12, 12)
    n = len(refs)
    _check_fork(pages, tables, lens, refs, parents, _pool(n, 1)[0])
    _check_fork(pages, tables, lens, refs, parents, _pool(n, 2, 8, 128, torch.float16))
    _check_fork(pages, tables, lens, refs, parents, _pool(n, 2, 5, 72))
    big = _pool(2 * n, 4, 3, 64)
    before = big.clone()
    _check_fork(pages, tables, lens, refs, parents, big[::2, ::2])
    assert torch.equal(_bits(big[1::2]), _bits(before[1::2]))
    assert torch.equal(_bits(big[:, 1::2]), _bits(before[:, 1::2]))


def test_nhd_pools(pages):
    """A page is a block of bytes in either layout; its tokens are counted
    along the layout's own dimension."""
    tables, lens, refs, rng = _random_state(78, 12, 200, spare=24)
    parents = rng.randint(0, 12, 12)
    pool = _pool(len(refs), 2, 8, 64).permute(0, 1, 2, 4, 3, 5).contiguous()
    want_t, want_l, want_r, want_c, copies = plain_fork(tables, lens, refs, parents)
    want_pool, c = _copied(pool, copies), _i32(refs)
    t, n, counts = pages.fork_sequences(pool, _i32(tables), _i32(lens), _i32(parents), c,
                                        kv_layout="NHD")
    assert np.array_equal(t.cpu().numpy(), want_t) and counts.tolist() == want_c
    assert np.array_equal(c.cpu().numpy(), want_r) and np.array_equal(n.cpu().numpy(), want_l)
    assert torch.equal(_bits(pool), _bits(want_pool))
    want_t, want_r, want_m, want_c, copies = plain_compact(want_t, want_l + 1, want_r)
    want_pool = _copied(pool, copies)
    remap, counts = pages.compact_pages(pool, t, n + 1, c, kv_layout="NHD")
    assert np.array_equal(t.cpu().numpy(), want_t) and counts.tolist() == want_c
    assert np.array_equal(c.cpu().numpy(), want_r) and torch.equal(_bits(pool), _bits(want_pool))
    assert np.array_equal(remap.cpu().numpy(), want_m)
    for call in (lambda: pages.fork_sequences(pool, t, n, n, c, kv_layout="DNH"),
                 lambda: pages.compact_pages(pool, t, n, c, "hnd")):
        with pytest.raises(ValueError, match="kv_layout"):
            call()


def test_fork_between_the_halves_of_one_buffer(pages):
    tables, lens, refs, rng = _random_state(79, 10, 100, spare=30)
    parents = rng.randint(0, 10, 10)
    both = torch.full((2,) + tables.shape, -7, dtype=torch.int32, device=DEV)
    both[1] = _i32(tables)
    pool, c = _pool(len(refs), 1), _i32(refs)
    t, _, counts = pages.fork_sequences(pool, both[1], _i32(lens), _i32(parents), c, out=both[0])
    want_t, _, want_r, want_c, _ = plain_fork(tables, lens, refs, parents)
    assert t.data_ptr() == both.data_ptr() and np.array_equal(both[0].cpu().numpy(), want_t)
    assert np.array_equal(both[1].cpu().numpy(), tables) and counts.tolist() == want_c
    flat = both.view(-1, tables.shape[1])
    for k in (0, 2, 4, 5, 10):
        with pytest.raises(ValueError, match="share memory"):
            pages.fork_sequences(pool, flat[5:15], _i32(lens), _i32(parents), c,
                                 out=flat[k:k + 10])
    assert np.array_equal(c.cpu().numpy(), want_r)


@pytest.mark.parametrize("length", [0, 16, 31, 32, 33])
def test_free_and_compact_between_a_fork_and_its_append(pages, length):
    """The page of the token to come is held once lengths count that token."""
    n = _held(length)
    tables = np.full((3, n + 2), -1, dtype=np.int64)
    tables[:, :n] = np.arange(n) + 20
    refs = np.zeros(40, dtype=np.int64)
    refs[20:20 + n] = 3
    refs[0] = 1  # held elsewhere
    t, ln, c, pool = _check_fork(pages, tables, np.full(3, length), refs, np.array([1, 1, 2]))
    own = t.cpu().numpy()[:, length // P]
    assert len(set(own.tolist())) == 3 and (own >= 0).all()
    fresh = pool.clone()
    pages.compact_pages(pool, t, ln + 1, c)
    moved = t.cpu().numpy()[:, length // P]
    for a, b in zip(own, moved):
        assert torch.equal(_bits(pool[:, b]), _bits(fresh[:, a]))
    assert c[moved.tolist()].tolist() == [1] * 3
    pages.free_sequences(t, ln + 1, c)
    assert c.sum() == 1 and (t == -1).all()


def test_fork_with_no_page_left(pages):
    tables = np.array([[0, 1, -1], [2, 3, -1], [4, 5, 6]])
    lens, refs = np.array([20, 32, 48]), np.ones(7, dtype=np.int64)
    # two pages come free with row 1; row 2's table has no room for more
    _check_fork(pages, tables, lens, refs, np.array([0, 0, 2]))
    # no page free at all
    _check_fork(pages, tables[:2], lens[:2], refs[:4], np.array([0, 1]))


def test_fork_reports_unsound_rows(pages, fi, lir):
    """Parents and lengths out of range, an unfinished page that is not one:
    those rows come back empty, the others are forked."""
    tables = np.array([[0, 1, -1], [2, 9, -1], [3, 4, -1], [5, -1, -1]])
    refs = np.array([1, 1, 1, 1, 1, 1, 0, 0])
    fi._CHECK, saved = False, fi._CHECK
    try:
        c = _i32(refs)
        t, n, counts = pages.fork_sequences(_pool(8), _i32(tables), _i32([20, 20, 64, -1]),
                                            _i32([0, 1, 2, 7]), c)
        assert lir._lib.device_status() == lir._lib.PA_ERR_DEVICE_CHECK
    finally:
        fi._CHECK = saved
    assert counts.tolist() == [0, 0, 3]
    assert t.tolist() == [[0, 1, -1], [-1] * 3, [-1] * 3, [-1] * 3] and n.tolist() == [20, 0, 0, 0]
    assert c.tolist() == [1, 1, 0, 1, 1, 1, 0, 0]


@pytest.mark.parametrize("length", [32, 20])
def test_fork_reports_counts_below_zero(pages, length):
    """A row that nobody continues gives up pages that no count holds."""
    tables, lens = _i32([[0, 1, -1], [2, 3, -1]]), _i32([length, length])
    refs = _i32([1, 1, 0, 0, 0, 0])
    with pytest.raises(RuntimeError, match="device"):
        pages.fork_sequences(_pool(6), tables, lens, _i32([0, 0]), refs)


def test_evict_and_compact_captured_and_replayed(pages, fi, lir):
    tables, lens, refs, _ = _random_state(95, 20, 600, spare=50, external=0.0, gone=0.0)
    pool = _pool(len(refs), 2)
    fresh, t, n, c = pool.clone(), _i32(tables), _i32(lens), _i32(refs)
    fi._CHECK, saved = False, fi._CHECK
    try:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            pages.evict_window_pages(t, n, c, 2 ** 31 - 1)
            pages.compact_pages(fresh.clone(), t.clone(), n, c.clone())
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            evicted = pages.evict_window_pages(t, n, c, 100, 4)
            remap, counts = pages.compact_pages(pool, t, n, c)
        for seed in (1, 2):
            lens = np.maximum(lens - seed, 0)
            n.copy_(_i32(lens))
            t.copy_(_i32(tables))
            c.copy_(_i32(refs))
            pool.copy_(fresh)
            graph.replay()
            torch.cuda.synchronize()
            want_t, want_r, want_e = plain_release(tables, lens, refs, 100, 4)
            want_t, want_r, want_m, want_c, copies = plain_compact(want_t, lens, want_r)
            assert evicted.tolist() == want_e and counts.tolist() == want_c
            assert np.array_equal(t.cpu().numpy(), want_t)
            assert np.array_equal(c.cpu().numpy(), want_r)
            assert np.array_equal(remap.cpu().numpy(), want_m)
            assert torch.equal(_bits(pool), _bits(_copied(fresh, copies)))
        assert lir._lib.device_status() == 0
    finally:
        fi._CHECK = saved


def test_fork_captured_and_replayed(pages, fi, lir):
    tables, lens, refs, rng = _random_state(91, 30, 300, spare=60)
    pool = _pool(len(refs), 2)
    fresh = pool.clone()
    t, n, c, par = _i32(tables), _i32(lens), _i32(refs), _i32(np.arange(30))
    out = torch.empty_like(t)
    fi._CHECK, saved = False, fi._CHECK
    try:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            pages.fork_sequences(pool, t, n, par, c, out=out)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            _, lens_out, counts = pages.fork_sequences(pool, t, n, par, c, out=out)
        for k in range(3):
            parents = rng.randint(0, 30, 30)
            par.copy_(_i32(parents))
            c.copy_(_i32(refs))
            pool.copy_(fresh)
            graph.replay()
            torch.cuda.synchronize()
            want_t, want_l, want_r, want_c, copies = plain_fork(tables, lens, refs, parents)
            assert np.array_equal(out.cpu().numpy(), want_t)
            assert np.array_equal(c.cpu().numpy(), want_r) and counts.tolist() == want_c
            assert np.array_equal(lens_out.cpu().numpy(), want_l)
            assert torch.equal(_bits(pool), _bits(_copied(fresh, copies)))
        assert lir._lib.device_status() == 0
    finally:
        fi._CHECK = saved


# ------------------------------------------------------------------- compaction
def _check_compact(pages, tables, lens, refs, pool=None):
    pool = _pool(len(refs), 2) if pool is None else pool
    want_t, want_r, want_m, want_c, copies = plain_compact(tables, lens, refs)
    want_pool = _copied(pool, copies)
    t, c = _i32(tables), _i32(refs)
    remap, counts = pages.compact_pages(pool, t, _i32(lens), c)
    assert counts.tolist() == want_c
    assert np.array_equal(t.cpu().numpy(), want_t)
    assert np.array_equal(c.cpu().numpy(), want_r)
    assert np.array_equal(remap.cpu().numpy(), want_m)
    assert torch.equal(_bits(pool), _bits(want_pool))


@pytest.mark.parametrize("seed", range(6))
@pytest.mark.parametrize("rows,max_len,spare", [(1, 40, 30), (20, 700, 400), (3, 10, 0), (60, 100, 3000)])
def test_compact_random(pages, seed, rows, max_len, spare):
    tables, lens, refs, _ = _random_state(seed, rows, max_len, spare=spare, external=0.1)
    _check_compact(pages, tables, lens, refs)


@pytest.mark.parametrize("live", ["none", "all", "last", "first", "every other"])
def test_compact_extremes(pages, live):
    n = 70001  # more pages than one step of the scan takes, no multiple of four
    refs = np.zeros(n, dtype=np.int64)
    if live == "all":
        refs[:] = 1
    elif live == "last":
        refs[-5:] = [1, 2, 3, 4, 5]
    elif live == "first":
        refs[:5] = 2
    elif live == "every other":
        refs[1::2] = 1
    held = np.nonzero(refs)[0][:50]
    tables = np.full((1, 60), -1, dtype=np.int64)
    tables[0, :len(held)] = held
    _check_compact(pages, tables, np.array([len(held) * P]), refs, _pool(n, 1, 1, 8))


def test_compact_without_tables_and_unaligned_counts(pages):
    refs = np.array([0, 1, 0, 0, 2, 1, 0, 3, 0, 0, 1])
    buf = torch.zeros(12, dtype=torch.int32, device=DEV)
    buf[1:] = _i32(refs)
    pool = _pool(11, 2)
    want_t, want_r, want_m, want_c, copies = plain_compact(np.zeros((0, 1), dtype=np.int64), [], refs)
    want_pool = _copied(pool, copies)
    remap, counts = pages.compact_pages(pool, _i32(np.zeros((0, 1))), _i32(np.zeros(0)), buf[1:])
    assert np.array_equal(buf[1:].cpu().numpy(), want_r) and np.array_equal(remap.cpu().numpy(), want_m)
    assert counts.tolist() == want_c and torch.equal(_bits(pool), _bits(want_pool))


def test_compact_reports_dead_entries(pages, fi, lir):
    tables, refs = _i32([[3, 1, 8], [2, 0, 0]]), _i32([0, 0, 0, 1])
    fi._CHECK, saved = False, fi._CHECK
    try:
        remap, counts = pages.compact_pages(_pool(4), tables, _i32([48, 100]), refs)
        assert lir._lib.device_status() == lir._lib.PA_ERR_DEVICE_CHECK
    finally:
        fi._CHECK = saved
    assert counts.tolist() == [1, 1, 3] and tables.tolist() == [[0, 1, 8], [2, 0, 0]]
    assert refs.tolist() == [1, 0, 0, 0] and remap.tolist() == [-1, -1, -1, 0]


def test_pages_on_another_stream(pages, fi, lir):
    """Two states worked on at the same time, each on its own stream."""
    fi._CHECK, saved = False, fi._CHECK
    try:
        states = []
        for k in range(2):
            tables, lens, refs, rng = _random_state(200 + k, 50, 400, spare=100)
            states.append((tables, lens, refs, rng.randint(0, 50, 50), _pool(len(refs), 3, seed=k)))
        got, streams = [], [torch.cuda.Stream() for _ in states]
        inputs = [(_i32(a), _i32(b), _i32(d), _i32(c)) for a, b, c, d, _ in states]
        fresh = [s[4].clone() for s in states]
        torch.cuda.synchronize()
        for (t, n, par, c), st, stream in zip(inputs, states, streams):
            with torch.cuda.stream(stream):
                got.append(pages.fork_sequences(st[4], t, n, par, c))
        torch.cuda.synchronize()
        for (tables, lens, refs, parents, pool), (t, n, counts), start, (_, _, _, c) in zip(
                states, got, fresh, inputs):
            want_t, want_l, want_r, want_c, copies = plain_fork(tables, lens, refs, parents)
            assert np.array_equal(t.cpu().numpy(), want_t) and counts.tolist() == want_c
            assert np.array_equal(c.cpu().numpy(), want_r)
            assert torch.equal(_bits(pool), _bits(_copied(start, copies)))
        assert lir._lib.device_status() == 0
    finally:
        fi._CHECK = saved


def test_offsets_past_32_bits(pages):
    """Pages whose bytes lie more than 4 GiB into the pool, and layers too."""
    n, layers = 1300, 60  # 64 KB pages: 5.1 GB, 85 MB a layer
    pool = torch.empty((layers, n, 2, 8, P, 128), dtype=torch.bfloat16, device=DEV)
    bits = pool.view(torch.int16)
    bits[:] = torch.arange(n, dtype=torch.int16, device=DEV)[None, :, None, None, None, None]
    bits += (torch.arange(layers, device=DEV) * 500).to(torch.int16)[:, None, None, None, None, None]
    refs = np.zeros(n, dtype=np.int64)
    refs[[0, 5, n - 1, n - 2]] = [1, 2, 1, 1]
    tables = np.array([[0, n - 1, -1], [5, n - 2, -1], [5, -1, -1]])
    lens = np.array([20, 32, 16])
    want_t, _, want_r, want_c, copies = plain_fork(tables, lens, refs, [0, 0, 1])
    c = _i32(refs)
    t, _, counts = pages.fork_sequences(pool, _i32(tables), _i32(lens), _i32([0, 0, 1]), c)
    assert counts.tolist() == want_c and copies == [(n - 1, 1)]
    assert np.array_equal(t.cpu().numpy(), want_t) and np.array_equal(c.cpu().numpy(), want_r)
    layer = (torch.arange(layers, device=DEV) * 500).to(torch.int16)
    same = lambda page, was: (bits[:, page].flatten(1) == (layer + was).to(torch.int16)[:, None]).all()  # noqa: E731
    assert same(1, n - 1) and same(2, 2) and same(n - 1, n - 1)
    lens = np.array([20, 20, 32])
    want_t, want_r, want_m, want_c, copies = plain_compact(want_t, lens, want_r)
    remap, counts = pages.compact_pages(pool, t, _i32(lens), c)
    assert counts.tolist() == want_c and np.array_equal(remap.cpu().numpy(), want_m)
    for s, d in copies:
        assert same(d, s)
