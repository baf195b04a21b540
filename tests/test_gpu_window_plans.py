"""Plans of several wrappers over one workspace: a window decode runs on the
plan that was made for it, and on no other.

What a refused call leaves behind is compared bit for bit: the output and the
pool stay as they were."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from test_gpu_window import DEV, HUGE, P, _decode_problem, _decode_wrapper, _t, _ws

pytestmark = pytest.mark.gpu


def _plan_other(fi, kind, ws, pr):
    """A plan of another kind over the same tables and workspace."""
    args = (_t(pr.indptr), _t(pr.indices), _t(pr.last), pr.hq, pr.hkv, pr.d, P)
    qo = _t(range(len(pr.kv) + 1))
    if kind == "decode":
        w = fi.BatchDecodeWithPagedKVCacheWrapper(ws, "HND")
        w.plan(*args, q_data_type=pr.dtype)
    elif kind == "prefill":
        w = fi.BatchPrefillWithPagedKVCacheWrapper(ws, "HND")
        w.plan(qo, *args, causal=True, q_data_type=pr.dtype, total_qo=len(pr.kv))
    elif kind == "window prefill":
        w = fi.BatchPrefillWithSlidingWindowWrapper(ws, "HND", window_left=pr.window,
                                                    num_sink_tokens=pr.sinks)
        w.plan(qo, *args, causal=True, q_data_type=pr.dtype, total_qo=len(pr.kv))
    else:
        w = fi.MultiLevelCascadeAttentionWrapper(2, ws, "HND")
        shared = [_t([0, 2]), _t([0, 1]), _t([P])]
        w.plan([_t([0, len(pr.kv)]), qo], [shared[0], args[0]], [shared[1], args[1]],
               [shared[2], args[2]], pr.hq, pr.hkv, pr.d, P, q_data_type=pr.dtype)
    return w


def _assert_refused(w, pr, q, pool):
    out = torch.full_like(q, 7)
    before = pool.clone()
    with pytest.raises(RuntimeError, match="plan"):
        w.run(q, pool, out=out)
    k = torch.ones((len(pr.kv), pr.hkv, pr.d), dtype=pr.dtype, device=DEV)
    with pytest.raises(RuntimeError, match="plan"):
        w.run_with_append(q, pool, k, k, _t(np.array(pr.kv) - 1), out=out)
    assert (out == 7).all()
    assert torch.equal(pool.view(torch.int16), before.view(torch.int16))


@pytest.mark.parametrize("kind", ["decode", "prefill", "window prefill", "cascade"])
@pytest.mark.parametrize("rows", [1, 2, 256, 1500])
def test_a_window_run_refuses_the_plan_that_replaced_its_own(fi, kind, rows):
    """Whatever the other plan leaves standing of the window's tables."""
    kv = np.random.RandomState(rows).randint(1, 150, rows).tolist()
    pr = _decode_problem(kv, 8, 2, 64, 63, 4, seed=rows, poison=False, evict=False)
    ws, q, pool = _ws(), pr.q.to(DEV), pr.device_pool()
    w = _decode_wrapper(fi, pr, ws)
    want, lse = w.run(q, pool, return_lse=True)
    pr.check(want, lse)
    _plan_other(fi, kind, ws, pr)
    _assert_refused(w, pr, q, pool)
    # planned again it runs again
    w.plan(_t(pr.indptr), _t(pr.indices), _t(pr.last), pr.hq, pr.hkv, pr.d, P, q_data_type=pr.dtype)
    assert torch.equal(w.run(q, pool), want)


@pytest.mark.parametrize("other", [(20, 4), (40, 0), (HUGE, 4), (40, HUGE)])
@pytest.mark.parametrize("lens", [[100, 50], [9, 3]])
def test_two_windows_do_not_run_on_one_anothers_plan(fi, other, lens):
    """Also where both windows hold every key and the tables are alike."""
    a = _decode_problem(lens, 8, 2, 64, 40, 4, seed=1, poison=False, evict=False)
    b = _decode_problem(lens, 8, 2, 64, *other, seed=1, poison=False, evict=False)
    ws, q, pool = _ws(), a.q.to(DEV), a.device_pool()
    wa = _decode_wrapper(fi, a, ws)
    wb = _decode_wrapper(fi, b, ws)
    _assert_refused(wa, a, q, pool)
    b.check(wb.run(q, pool))
    wa.plan(_t(a.indptr), _t(a.indices), _t(a.last), 8, 2, 64, P, q_data_type=a.dtype)
    _assert_refused(wb, b, q, pool)
    a.check(wa.run(q, pool))


def test_a_table_of_another_size_is_another_plan(fi):
    """One window, one batch size, as many visible pages at most, but more
    page ids in one of the tables."""
    a = _decode_problem([400, 390], 8, 2, 64, 20, 0, seed=2, poison=False, evict=False)
    b = _decode_problem([900, 390], 8, 2, 64, 20, 0, seed=3, poison=False, evict=False)
    ws = _ws()
    wa = _decode_wrapper(fi, a, ws)
    _decode_wrapper(fi, b, ws)
    _assert_refused(wa, a, a.q.to(DEV), a.device_pool())


def test_refused_runs_in_a_graph_report_the_plan(fi, lir):
    """Replayed after another plan, a captured run reports and writes nothing."""
    pr = _decode_problem([300, 17, 80], 8, 2, 64, 60, 2, seed=5, poison=False, evict=False)
    fi._CHECK, saved = False, fi._CHECK
    try:
        ws, q, pool = _ws(), pr.q.to(DEV), pr.device_pool()
        w = _decode_wrapper(fi, pr, ws)
        out = torch.empty_like(q)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            w.run(q, pool, out=out)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            w.run(q, pool, out=out)
        out.zero_()
        graph.replay()
        pr.check(out)
        assert lir._lib.device_status() == 0
        for kind in ("prefill", "decode"):
            _plan_other(fi, kind, ws, pr)
            out.fill_(7)
            graph.replay()
            assert lir._lib.device_status() == lir._lib.PA_ERR_NOT_PLANNED
            assert (out == 7).all()
    finally:
        fi._CHECK = saved


def test_an_append_stays_inside_the_rows_of_the_callers_table(fi):
    """Two tables of one size whose rows have other lengths, one workspace: a
    run of the first on the plan of the second takes a position that only the
    planned row has. It is reported and not written to the next row's pages."""
    a = _decode_problem([40, 400], 8, 2, 64, 40, 4, seed=11, poison=False, evict=False)
    b = _decode_problem([400, 40], 8, 2, 64, 40, 4, seed=11, poison=False, evict=False)
    ws, q, pool = _ws(), a.q.to(DEV), a.device_pool()
    w = _decode_wrapper(fi, a, ws)
    _decode_wrapper(fi, b, ws)
    before = pool.clone()
    k = torch.ones((2, 2, 64), dtype=a.dtype, device=DEV)
    with pytest.raises(RuntimeError, match="device"):
        w.run_with_append(q, pool, k, k, _t([100, 2]))  # page 6 of a row of three
    beyond = a.tables[1][6 - 3]
    assert torch.equal(pool[beyond].view(torch.int16), before[beyond].view(torch.int16))
    # on its own plan the position is refused by the row's length
    w.plan(_t(a.indptr), _t(a.indices), _t(a.last), 8, 2, 64, P, q_data_type=a.dtype)
    with pytest.raises(RuntimeError, match="device"):
        w.run_with_append(q, pool, k, k, _t([100, 2]))
    assert torch.equal(pool[beyond].view(torch.int16), before[beyond].view(torch.int16))
