"""Sliding-window attention with sinks against a plain 64-bit implementation.

Tolerance, element by element: the kernels round the probabilities to the
cache's type before P V (half a step u relative to each, u = eps / 2: at most
u * A off, A = sum_j p_j |v_j|), the output once more (u * |o|), and work in
fp32 otherwise. fp32 leaves each score off by at most D 2^-24 sum_i |q_i k_i|
scale < 2e-4 for these inputs (|q|, |k| below 6, D <= 128, scale 1/sqrt(D):
the sum is below 128 * 1.2 with room to spare), which moves p by as much
relative to itself, numerator and denominator both: 4e-4 * A. fp16
probabilities below 2^-14 are subnormal, half a step 2^-25 each: 2^-25 *
sum_j |v_j|. LSE: 2e-4 * log2(e) for the scores and fp32 roundings: 4e-4.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
P = 16
HUGE = 2 ** 31 - 1


def visible(n, length, window, sinks, causal=True):
    """[n, length] bool: which keys the last n positions see."""
    pos = np.arange(length - n, length)[:, None]
    key = np.arange(length)[None]
    seen = (pos - key <= window) | (key < sinks)
    return seen & (key <= pos) if causal else seen


class Problem:
    """Requests of qo[b] new rows over kv[b] keys in a pool of permuted pages."""

    def __init__(self, qo, kv, hq, hkv, d, window, sinks, dtype=torch.bfloat16, seed=0,
                 causal=True, layout="HND", poison=True, evict=True):
        g = torch.Generator().manual_seed(seed)
        self.qo, self.kv, self.hq, self.hkv, self.d = list(qo), list(kv), hq, hkv, d
        self.window, self.sinks, self.dtype, self.causal = window, sinks, dtype, causal
        self.layout = layout
        npages = [-(-n // P) for n in kv]
        total = sum(npages) + 3
        ids = torch.randperm(total, generator=g).tolist()
        self.tables, at = [], 0
        for n in npages:
            self.tables.append(ids[at:at + n])
            at += n
        self.pool = torch.randn((total, 2, hkv, P, d), generator=g).to(dtype)
        self.q = torch.randn((max(sum(qo), 0), hq, d), generator=g).to(dtype)
        self.k64, self.v64 = [], []
        for b in range(len(kv)):
            pages = self.pool[self.tables[b]].double()
            self.k64.append(pages[:, 0].permute(1, 0, 2, 3).reshape(hkv, -1, d)[:, :kv[b]])
            self.v64.append(pages[:, 1].permute(1, 0, 2, 3).reshape(hkv, -1, d)[:, :kv[b]])
        # what no query sees holds garbage; a page of nothing else may be gone
        bad = torch.tensor([math.nan, math.inf, -math.inf])
        for b in range(len(kv)):
            seen = (visible(qo[b], kv[b], window, sinks, causal).any(0) if qo[b]
                    else np.zeros(kv[b], dtype=bool))
            seen = np.concatenate([seen, np.zeros(npages[b] * P - kv[b], dtype=bool)])
            for j, page in enumerate(list(self.tables[b])):
                hid = np.nonzero(~seen[j * P:(j + 1) * P])[0]
                if poison and len(hid):
                    self.pool[page, :, :, hid] = bad[torch.randint(0, 3, (1,), generator=g)].to(dtype)
                if evict and len(hid) == P and j + 1 < npages[b]:
                    self.tables[b][j] = -1
        self.indptr = np.concatenate([[0], np.cumsum(npages)])
        self.indices = np.array([p for t in self.tables for p in t] or [0])
        self.last = np.array([(n - 1) % P + 1 if n else 0 for n in kv])
        self.qo_indptr = np.concatenate([[0], np.cumsum(qo)])

    def device_pool(self):
        pool = self.pool if self.layout == "HND" else self.pool.permute(0, 1, 3, 2, 4).contiguous()
        return pool.to(DEV)

    def want(self):
        """(out, lse base 2, A, sum |v|) in float64."""
        n, g = sum(self.qo), self.hq // self.hkv
        out = torch.zeros((n, self.hq, self.d), dtype=torch.float64)
        lse = torch.full((n, self.hq), -math.inf, dtype=torch.float64)
        near, total = torch.zeros_like(out), torch.zeros_like(out)
        for b, rows in enumerate(self.qo):
            if not rows or not self.kv[b]:
                continue
            r0 = int(self.qo_indptr[b])
            seen = torch.from_numpy(visible(rows, self.kv[b], self.window, self.sinks, self.causal))
            q = self.q[r0:r0 + rows].double().view(rows, self.hkv, g, self.d)
            s = torch.einsum("rhgd,hkd->hgrk", q, self.k64[b]) / math.sqrt(self.d)
            s = s.masked_fill(~seen, -math.inf)
            p = torch.softmax(s, -1)
            put = lambda x: torch.einsum("hgrk,hkd->rhgd", *x).reshape(rows, self.hq, self.d)  # noqa: E731
            out[r0:r0 + rows] = put((p, self.v64[b]))
            near[r0:r0 + rows] = put((p, self.v64[b].abs()))
            total[r0:r0 + rows] = put((seen.double().expand_as(p), self.v64[b].abs()))
            lse[r0:r0 + rows] = (torch.logsumexp(s, -1) / math.log(2)).permute(2, 0, 1).reshape(rows, -1)
        return out, lse, near, total

    def check(self, got, lse=None):
        out, want_lse, near, total = self.want()
        u = torch.finfo(self.dtype).eps / 2
        tol = (u + 4e-4) * near * (1 + u) + u * out.abs()
        if self.dtype == torch.float16:
            tol = tol + 2.0 ** -25 * total
        off = (got.double().cpu() - out).abs()
        assert torch.isfinite(got).all()
        worst = float((off - tol).max()) if off.numel() else 0.0
        assert worst <= 0, f"{worst:.3e} over; largest difference {float(off.max()):.3e}"
        if lse is not None:
            fin = torch.isfinite(want_lse)
            assert torch.equal(torch.isfinite(lse.cpu()), fin)
            assert (lse.cpu()[fin].double() - want_lse[fin]).abs().max() <= 4e-4


def _t(a):
    return torch.as_tensor(np.ascontiguousarray(np.asarray(a, dtype=np.int32))).to(DEV)


def _ws():
    return torch.empty(128 << 20, dtype=torch.uint8, device=DEV)


def _decode_wrapper(fi, pr, ws=None):
    w = fi.BatchDecodeWithSlidingWindowWrapper(_ws() if ws is None else ws, pr.layout,
                                               window_left=pr.window, num_sink_tokens=pr.sinks)
    w.plan(_t(pr.indptr), _t(pr.indices), _t(pr.last), pr.hq, pr.hkv, pr.d, P,
           q_data_type=pr.dtype)
    return w


def _decode_problem(kv, *args, **kw):
    return Problem([1] * len(kv), kv, *args, **kw)


MIXED = [1, 2, 15, 16, 17, 31, 32, 33, 100, 255, 256, 257, 1000, 0, 700]


@pytest.mark.parametrize("window", [0, 1, 14, 15, 16, 17, 31, 100, 512, HUGE])
@pytest.mark.parametrize("sinks", [0, 1, 4, 16, 17, 130, HUGE])
def test_decode_windows_and_sinks(fi, window, sinks):
    pr = _decode_problem(MIXED, 8, 2, 64, window, sinks, seed=window % 97 + sinks % 31)
    w = _decode_wrapper(fi, pr)
    out, lse = w.run(pr.q.to(DEV), pr.device_pool(), return_lse=True)
    pr.check(out, lse)


@pytest.mark.parametrize("hq,hkv,d,dtype,layout", [
    (32, 4, 64, torch.bfloat16, "HND"), (32, 8, 128, torch.float16, "HND"),
    (8, 8, 128, torch.bfloat16, "NHD"), (16, 1, 64, torch.float16, "NHD"),
    (16, 16, 64, torch.bfloat16, "HND"), (32, 16, 128, torch.bfloat16, "HND"),
    (5, 5, 64, torch.bfloat16, "HND")])
def test_decode_geometries(fi, hq, hkv, d, dtype, layout):
    pr = _decode_problem([3000, 40, 1, 517, 2048], hq, hkv, d, 333, 5, dtype, seed=hq + hkv,
                         layout=layout)
    out, lse = _decode_wrapper(fi, pr).run(pr.q.to(DEV), pr.device_pool(), return_lse=True)
    pr.check(out, lse)


@pytest.mark.parametrize("window,sinks", [(1023, 4), (63, 0)])
def test_decode_batch_larger_than_the_grid(fi, window, sinks):
    """More requests than one scan of the plan takes (1024 threads) and than
    there are SMs; every request's segment is cut somewhere."""
    rng = np.random.RandomState(5)
    kv = rng.randint(0, 200, 1500).tolist()
    kv[7] = 5000
    pr = _decode_problem(kv, 4, 1, 64, window, sinks, seed=9)
    out, lse = _decode_wrapper(fi, pr).run(pr.q.to(DEV), pr.device_pool(), return_lse=True)
    pr.check(out, lse)


def test_decode_agrees_with_the_full_wrapper_when_all_is_visible(fi):
    """The window plan cuts segments into other pieces than the full one, and
    each piece rounds its probabilities against its own maximum: each of the
    two is within the tolerance, so they are within twice that of each other
    (not bit-identical, as they would be on one partition)."""
    pr = _decode_problem(MIXED, 32, 4, 64, HUGE, 0, seed=3)
    pool, q = pr.device_pool(), pr.q.to(DEV)
    got, glse = _decode_wrapper(fi, pr).run(q, pool, return_lse=True)
    w = fi.BatchDecodeWithPagedKVCacheWrapper(_ws(), "HND")
    w.plan(_t(pr.indptr), _t(pr.indices), _t(pr.last), 32, 4, 64, P, q_data_type=pr.dtype)
    out, lse = w.run(q, pool, return_lse=True)
    pr.check(got, glse)
    pr.check(out, lse)


@pytest.mark.parametrize("hq,hkv,d,layout,dtype", [(8, 2, 64, "HND", torch.bfloat16),
                                                   (32, 8, 128, "NHD", torch.float16),
                                                   (16, 16, 64, "HND", torch.bfloat16)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (20, 3), (100, 17)])
def test_decode_with_append_equals_append_then_decode(fi, hq, hkv, d, layout, dtype, window, sinks):
    kv = [1, 16, 17, 33, 400, 1000]
    pr = _decode_problem(kv, hq, hkv, d, window, sinks, dtype, seed=11, layout=layout)
    g = torch.Generator().manual_seed(1)
    # rows of a wider tensor: strided, as views of a projection are
    kvq = torch.randn((len(kv), 2 * hkv + 1, d), generator=g).to(dtype).to(DEV)
    k, v = kvq[:, :hkv], kvq[:, hkv:2 * hkv]
    pos = _t(np.array(kv) - 1)
    q = pr.q.to(DEV)
    one, two = pr.device_pool(), pr.device_pool()
    w = _decode_wrapper(fi, pr)
    out1, lse1 = w.run_with_append(q, one, k, v, pos, return_lse=True)
    fi.append_paged_kv_cache(k, v, _t(range(len(kv))), pos, two, _t(pr.indices), _t(pr.indptr),
                             _t(pr.last), kv_layout=layout)
    out2, lse2 = w.run(q, two, return_lse=True)
    assert torch.equal(one.view(torch.int16), two.view(torch.int16))
    assert torch.equal(out1, out2) and torch.equal(lse1, lse2)


def test_append_to_a_hidden_position_reaches_the_pool_only(fi):
    """Positions that the window hides: in a page that is not visible, in the
    hidden part of a sink page and of the window's first page, and a sink."""
    kv, window, sinks = [400] * 4, 40, 4
    pr = _decode_problem(kv, 8, 2, 64, window, sinks, seed=21, poison=False, evict=False)
    q = pr.q.to(DEV)
    w = _decode_wrapper(fi, pr)
    pos = _t([100, 9, 399 - 40 - 3, 2])
    k = torch.randn(4, 2, 64, device=DEV).to(torch.bfloat16)
    k[:3] = math.nan
    one, two = pr.device_pool(), pr.device_pool()
    out1 = w.run_with_append(q, one, k, k, pos)
    fi.append_paged_kv_cache(k, k, _t(range(4)), pos, two, _t(pr.indices), _t(pr.indptr),
                             _t(pr.last), kv_layout="HND")
    out2 = w.run(q, two)
    assert torch.equal(one.view(torch.int16), two.view(torch.int16))
    assert torch.equal(out1, out2) and torch.isfinite(out1).all()


def test_append_to_a_page_that_was_given_back_is_reported(fi, lir):
    pr = _decode_problem([400], 8, 2, 64, 40, 4, seed=22)
    w = _decode_wrapper(fi, pr)
    k = torch.ones(1, 2, 64, device=DEV, dtype=torch.bfloat16)
    pool = pr.device_pool()
    before = pool.clone()
    with pytest.raises(RuntimeError, match="device"):
        w.run_with_append(pr.q.to(DEV), pool, k, k, _t([100]))
    assert torch.equal(pool.view(torch.int16), before.view(torch.int16))
    with pytest.raises(RuntimeError, match="device"):
        w.run_with_append(pr.q.to(DEV), pool, k, k, _t([400]))


def test_decode_captured_and_replayed_with_new_lengths(fi, lir):
    """Plan and run in one graph; the tables change between replays."""
    fa, saved = fi, fi._CHECK
    a = _decode_problem([50, 300, 17], 8, 2, 64, 60, 2, seed=31, poison=False, evict=False)
    fa._CHECK = False
    try:
        pool, q, ws = a.device_pool(), a.q.to(DEV), _ws()
        w = fi.BatchDecodeWithSlidingWindowWrapper(ws, "HND", window_left=60, num_sink_tokens=2)
        indptr, indices, last = _t(a.indptr), _t(a.indices), _t(a.last)
        out = torch.empty_like(q)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            w.plan(indptr, indices, last, 8, 2, 64, P, q_data_type=q.dtype)
            w.run(q, pool, out=out)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            w.plan(indptr, indices, last, 8, 2, 64, P, q_data_type=q.dtype)
            w.run(q, pool, out=out)
        for kv in ([50, 300, 17], [49, 290, 30], [64, 304, 32]):
            # same number of pages in all, other lengths
            last.copy_(_t([(n - 1) % P + 1 for n in kv]))
            graph.replay()
            torch.cuda.synchronize()
            # the same pages with the new lengths
            a.kv = [(int(a.indptr[i + 1] - a.indptr[i]) - 1) * P + (kv[i] - 1) % P + 1 for i in range(3)]
            a.k64, a.v64 = [], []
            for b in range(3):
                pages = a.pool[a.tables[b]].double()
                a.k64.append(pages[:, 0].permute(1, 0, 2, 3).reshape(2, -1, 64)[:, :a.kv[b]])
                a.v64.append(pages[:, 1].permute(1, 0, 2, 3).reshape(2, -1, 64)[:, :a.kv[b]])
            a.check(out)
        assert lir._lib.device_status() == 0
    finally:
        fa._CHECK = saved


def test_two_runs_on_one_plan_are_bit_identical(fi):
    pr = _decode_problem([9000, 20, 4000] * 7, 32, 8, 128, 2047, 16, seed=41)
    w, q, pool = _decode_wrapper(fi, pr), pr.q.to(DEV), pr.device_pool()
    a, b = w.run(q, pool), w.run(q, pool)
    assert torch.equal(a, b)
    pr.check(a)


def test_pages_past_32_bits_of_the_pool(fi):
    """The visible pages are the last ones of a pool of more than 4 GiB."""
    pr = _decode_problem([700, 90], 32, 8, 128, 200, 4, seed=43)
    n = 70000  # 64 KB pages
    pool = torch.full((n, 2, 8, P, 128), math.nan, dtype=torch.bfloat16, device=DEV)
    held = pr.pool.shape[0]
    pool[n - held:] = pr.pool.to(DEV)
    pr.indices = np.where(pr.indices >= 0, pr.indices + n - held, -1)
    q = pr.q.to(DEV)
    w = _decode_wrapper(fi, pr)
    pr.check(*w.run(q, pool, return_lse=True))
    pos = _t([699, 89])
    k = torch.randn((2, 8, 128), generator=torch.Generator().manual_seed(45)).to(pr.dtype).to(DEV)
    out = w.run_with_append(q, pool, k, k, pos)
    for b, at in enumerate((699, 89)):
        page = int(pr.indices[int(pr.indptr[b]) + at // P])
        assert page > 65536 and torch.equal(pool[page, 0, :, at % P], k[b])
        pr.k64[b][:, at] = k[b].double().cpu()
        pr.v64[b][:, at] = k[b].double().cpu()
    pr.check(out)
    pre = Problem([70, 3], [700, 90], 32, 8, 128, 200, 4, seed=44)
    pool[:] = math.nan
    held = pre.pool.shape[0]
    pool[n - held:] = pre.pool.to(DEV)
    pre.indices = np.where(pre.indices >= 0, pre.indices + n - held, -1)
    pre.device_pool = lambda: pool
    pre.check(*_prefill(fi, pre))


# ---------------------------------------------------------------------- prefill
def _prefill(fi, pr, return_lse=True):
    w = fi.BatchPrefillWithSlidingWindowWrapper(_ws(), pr.layout, window_left=pr.window,
                                                num_sink_tokens=pr.sinks)
    w.plan(_t(pr.qo_indptr), _t(pr.indptr), _t(pr.indices), _t(pr.last), pr.hq, pr.hkv, pr.d, P,
           causal=pr.causal, q_data_type=pr.dtype)
    return w.run(pr.q.to(DEV), pr.device_pool(), return_lse=return_lse)


RAGGED_QO = [1, 37, 0, 16, 300, 5, 64]
RAGGED_KV = [1, 100, 33, 16, 700, 1500, 64]


@pytest.mark.parametrize("window", [0, 1, 15, 16, 17, 127, 128, 200, HUGE])
@pytest.mark.parametrize("sinks", [0, 1, 4, 16, 17, 130, HUGE])
def test_prefill_windows_and_sinks(fi, window, sinks):
    pr = Problem(RAGGED_QO, RAGGED_KV, 8, 2, 64, window, sinks, seed=window % 89 + sinks % 37)
    pr.check(*_prefill(fi, pr))


@pytest.mark.parametrize("hq,hkv,d,dtype,layout", [
    (32, 4, 64, torch.bfloat16, "HND"), (32, 8, 128, torch.float16, "HND"),
    (8, 8, 128, torch.bfloat16, "NHD"), (16, 1, 64, torch.float16, "NHD"),
    (32, 16, 128, torch.bfloat16, "HND")])
def test_prefill_geometries(fi, hq, hkv, d, dtype, layout):
    pr = Problem([200, 1, 333], [900, 1200, 333], hq, hkv, d, 250, 9, dtype, seed=hq, layout=layout)
    pr.check(*_prefill(fi, pr))


@pytest.mark.parametrize("window,sinks", [(50, 0), (50, 20), (0, 0), (HUGE, 0)])
def test_prefill_not_causal(fi, window, sinks):
    pr = Problem(RAGGED_QO, RAGGED_KV, 8, 2, 64, window, sinks, seed=51, causal=False)
    pr.check(*_prefill(fi, pr))


def test_prefill_equals_the_full_wrapper_when_all_is_visible(fi):
    pr = Problem(RAGGED_QO, RAGGED_KV, 32, 8, 128, HUGE, 0, seed=52)
    got, glse = _prefill(fi, pr)
    w = fi.BatchPrefillWithPagedKVCacheWrapper(_ws(), "HND")
    w.plan(_t(pr.qo_indptr), _t(pr.indptr), _t(pr.indices), _t(pr.last), 32, 8, 128, P,
           causal=True, q_data_type=pr.dtype)
    out, lse = w.run(pr.q.to(DEV), pr.device_pool(), return_lse=True)
    assert torch.equal(got, out) and torch.equal(glse, lse)


def test_prefill_long_chunk_runs_many_items(fi):
    pr = Problem([1500, 700], [6000, 3000], 8, 2, 64, 511, 4, seed=53)
    out, lse = _prefill(fi, pr)
    pr.check(out, lse)
    again, _ = _prefill(fi, pr)
    assert torch.equal(out, again)


def test_chunks_then_decode_agree_with_one_prefill(fi):
    """A sequence prefilled in chunks and then decoded sees what it would see
    as the last rows of one prefill."""
    pr = Problem([600], [600], 8, 2, 64, 90, 5, seed=54, poison=False, evict=False)
    whole, _ = _prefill(fi, pr)
    tail = Problem([1], [600], 8, 2, 64, 90, 5, seed=54, poison=False, evict=False)
    tail.q = pr.q[-1:]
    out = _decode_wrapper(fi, tail).run(tail.q.to(DEV), tail.device_pool())
    tail.check(out)
    tail.check(whole[-1:])


# ---------------------------------------------------------------------- refusals
def test_wrong_tables_are_reported(fi, lir):
    pr = _decode_problem([100, 50], 8, 2, 64, 20, 0, seed=61, evict=False)
    w = fi.BatchDecodeWithSlidingWindowWrapper(_ws(), "HND", window_left=20)
    bad = [(_t([0, 20, 11]), _t(pr.indices), _t(pr.last)),       # past the page ids, backwards
           (_t([1, 7, 11]), _t(pr.indices), _t(pr.last)),        # does not start at 0
           (_t([0, 7, 900]), _t(pr.indices), _t(pr.last)),       # past the page ids
           (_t(pr.indptr), _t(pr.indices), _t([4, 17])),         # last page too long
           (_t(pr.indptr), _t(pr.indices), _t([0, 2]))]          # last page empty
    for indptr, indices, last in bad:
        with pytest.raises(RuntimeError, match="device"):
            w.plan(indptr, indices, last, 8, 2, 64, P, q_data_type=pr.dtype)
    # a visible page that is not one
    indices = pr.indices.copy()
    indices[int(pr.indptr[1]) - 1] = -1
    w.plan(_t(pr.indptr), _t(indices), _t(pr.last), 8, 2, 64, P, q_data_type=pr.dtype)
    with pytest.raises(RuntimeError, match="device"):
        w.run(pr.q.to(DEV), pr.device_pool())


def test_rows_that_claim_the_same_entries_again_are_reported(fi, lir):
    """The visible pages of such a table add up past 32 bits."""
    n, rows = 1 << 20, 6000
    indptr = np.zeros(rows + 1, dtype=np.int64)
    indptr[1::2] = n
    buf = torch.full((96 << 20,), 7, dtype=torch.uint8, device=DEV)
    w = fi.BatchDecodeWithSlidingWindowWrapper(buf[32 << 20:64 << 20], "HND", window_left=HUGE)
    fi._CHECK, saved = False, fi._CHECK
    try:
        w.plan(_t(indptr), _t(np.zeros(n)), _t(np.full(rows, P)), 8, 2, 64, P,
               q_data_type=torch.bfloat16)
        assert lir._lib.device_status() == lir._lib.PA_ERR_DEVICE_CHECK
    finally:
        fi._CHECK = saved
    assert (buf[:32 << 20] == 7).all() and (buf[64 << 20:] == 7).all()


def test_plans_are_not_exchanged(fi):
    """A full plan's workspace is not a window plan's, and the other way round."""
    pr = _decode_problem([100, 50], 8, 2, 64, 20, 0, seed=62, evict=False, poison=False)
    ws = torch.zeros(128 << 20, dtype=torch.uint8, device=DEV)
    full = fi.BatchDecodeWithPagedKVCacheWrapper(ws, "HND")
    full.plan(_t(pr.indptr), _t(pr.indices), _t(pr.last), 8, 2, 64, P, q_data_type=pr.dtype)
    _decode_wrapper(fi, pr, ws)
    with pytest.raises(RuntimeError, match="plan"):
        full.run(pr.q.to(DEV), pr.device_pool())
