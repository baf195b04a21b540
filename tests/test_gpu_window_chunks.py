"""A sequence that reaches the window kernels piece by piece, and selections
whose scores are looked at for the largest batches. The oracles and tolerances
are those of test_gpu_window.py and test_gpu_beam.py."""

from __future__ import annotations

import importlib
import math

import numpy as np
import pytest
import torch

from test_gpu_beam import _random, plain_select
from test_gpu_window import DEV, P, Problem, _prefill, _t, _ws

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hq,hkv,d,dtype,layout", [(8, 2, 64, torch.bfloat16, "HND"),
                                                   (32, 8, 128, torch.float16, "NHD"),
                                                   (16, 16, 64, torch.bfloat16, "HND")])
@pytest.mark.parametrize("window,sinks", [(90, 5), (0, 0), (16, 17), (300, 0)])
def test_chunks_and_decoded_tokens_give_the_rows_of_one_prefill(fi, hq, hkv, d, dtype, layout,
                                                                window, sinks):
    """Prefilled in chunks of 1 to 200 tokens and then decoded token by token,
    each appended to a cache that holds nothing else; pages behind the window
    are given back after each piece and overwritten."""
    pages = importlib.import_module("llm-inference-runtime_b200.pages")
    chunks, steps = (1, 37, 130, 16, 200, 65), 37
    n = sum(chunks) + steps
    pr = Problem([n], [n], hq, hkv, d, window, sinks, dtype, seed=window + d, layout=layout,
                 poison=False, evict=False)
    whole, lse = _prefill(fi, pr)
    pr.check(whole, lse)
    k, v = (x[0].transpose(0, 1).to(dtype).to(DEV) for x in (pr.k64, pr.v64))
    q = pr.q.to(DEV)
    held = -(-n // P)
    shape = (held, 2, hkv, P, d) if layout == "HND" else (held, 2, P, hkv, d)
    pool = torch.full(shape, math.nan, dtype=dtype, device=DEV)
    order = np.random.RandomState(window).permutation(held)
    table = _t(order[None])
    refs = torch.ones(held, dtype=torch.int32, device=DEV)
    ws, got, got_lse = _ws(), [], []
    kw = dict(window_left=window, num_sink_tokens=sinks)
    prefill = fi.BatchPrefillWithSlidingWindowWrapper(ws, layout, **kw)
    decode = fi.BatchDecodeWithSlidingWindowWrapper(ws, layout, **kw)
    done = 0
    for rows in chunks + (1,) * steps:
        new = slice(done, done + rows)
        done += rows
        used = -(-done // P)
        tables = (_t([0, used]), table[0, :used].contiguous(), _t([(done - 1) % P + 1]))
        pos = _t(np.arange(done - rows, done))
        if len(got) < len(chunks):
            fi.append_paged_kv_cache(k[new], v[new], _t(np.zeros(rows)), pos, pool, tables[1],
                                     tables[0], tables[2], kv_layout=layout)
            prefill.plan(_t([0, rows]), *tables, hq, hkv, d, P, causal=True, q_data_type=dtype)
            out, s = prefill.run(q[new], pool, return_lse=True)
        else:
            decode.plan(*tables, hq, hkv, d, P, q_data_type=dtype)
            out, s = decode.run_with_append(q[new], pool, k[new], v[new], pos, return_lse=True)
        got.append(out)
        got_lse.append(s)
        # (the first of the next rows is the one after the last of these)
        pages.evict_window_pages(table, _t([done]), refs, window, sinks)
        pool[refs == 0] = math.nan
    pr.check(torch.cat(got), torch.cat(got_lse))
    first, end = -(-sinks // P), max(n - 1 - window, 0) // P
    assert int((table == -1).sum()) == max(end - first, 0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("batch,beams,vocab", [(64, 8, 128256), (150, 4, 128256), (100, 8, 50257)])
def test_scores_of_full_batches(fi, dtype, batch, beams, vocab):
    beam = importlib.import_module("llm-inference-runtime_b200.beam")
    logits, scores = _random(batch, beams, vocab, dtype, seed=batch + vocab)
    best, parents, tokens = beam.beam_search_select(logits, scores, 2 * beams)
    some = [0, batch // 3, batch - 1]
    want, want_p, want_t, near = plain_select(logits[some], scores[some], 2 * beams)
    shift = torch.tensor([(b - i) * beams for i, b in enumerate(some)])[:, None]
    assert np.array_equal((parents[some].cpu() - shift).numpy(), want_p)
    assert np.array_equal(tokens[some].cpu().numpy(), want_t)
    off = np.abs(best[some].cpu().double().numpy() - want)
    assert (off <= near + 2.0 ** -24 * np.abs(want)).all()


@pytest.mark.parametrize("rows", [2047, 2048, 2049, 5000])
def test_decode_plans_of_more_requests_than_the_plan_keeps_at_hand(fi, rows):
    """The plan's own table is read back from memory past its first entries."""
    kv = np.random.RandomState(rows).randint(0, 60, rows).tolist()
    kv[-1], kv[rows // 2] = 700, 333
    pr = Problem([1] * rows, kv, 4, 1, 64, 24, 3, seed=rows)
    w = fi.BatchDecodeWithSlidingWindowWrapper(_ws(), "HND", window_left=24, num_sink_tokens=3)
    w.plan(_t(pr.indptr), _t(pr.indices), _t(pr.last), 4, 1, 64, P, q_data_type=pr.dtype)
    pr.check(*w.run(pr.q.to(DEV), pr.device_pool(), return_lse=True))


@pytest.mark.parametrize("rows", [63, 64, 65, 300, 1100])
@pytest.mark.parametrize("causal", [True, False])
def test_prefill_of_many_requests(fi, rows, causal):
    """Around the number of requests from which the plan gives a thread, not a
    warp, to each."""
    rng = np.random.RandomState(rows)
    qo = rng.randint(0, 4, rows)
    kv = qo + rng.randint(0, 60, rows)
    qo[rows // 3], kv[rows // 3] = 260, 900
    pr = Problem(qo.tolist(), kv.tolist(), 8, 2, 64, 33, 5, seed=rows, causal=causal)
    pr.check(*_prefill(fi, pr))
