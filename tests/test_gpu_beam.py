"""Beam selection against a plain 64-bit implementation, and a beam search
over the paged cache against one that keeps every beam's keys.

Choices are whole numbers and are equal. Scores: a summand exp(x - ref)
carries the roundings of its exponent (below 8 for the summands that matter:
2^-22 ln 2 relative), of log2(e) and of the exponential (2^-22 each), its
thread's four fp32 additions (2^-24 each) and the exponential that joins the
thread to the others (2^-22): together below 1.2e-6 of the sum, which is as much
in its logarithm. That is rounded to fp32 (2^-24 |lse|), and so is the score
(2^-24 |score|).
"""

from __future__ import annotations

import importlib
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
P = 16


@pytest.fixture(scope="module")
def beam(fi):
    return importlib.import_module("llm-inference-runtime_b200.beam")


def plain_select(logits, scores, n):
    """(scores, parents, tokens, tolerance) as numpy arrays."""
    x = logits.cpu().double().numpy()
    x = np.where(np.isnan(x), -np.inf, np.minimum(x, torch.finfo(logits.dtype).max))
    c = scores.cpu().double().numpy()
    batch, beams, vocab = x.shape
    out = [np.zeros((batch, n)) for _ in range(4)]
    for b in range(batch):
        flat, near = [], []
        for w in range(beams):
            top = x[b, w].max()
            if not c[b, w] > -np.inf or top == -np.inf:
                x[b, w] = -np.inf
                flat.append(np.full(vocab, -np.inf))
                near.append(0.0)
                continue
            lse = np.float32(top + math.log(np.exp(x[b, w] - top).sum()))
            flat.append(c[b, w] + (x[b, w] - np.float64(lse)))
            near.append(1.2e-6 + 2.0 ** -24 * abs(float(lse)) * 2)
        flat = np.concatenate(flat)
        # best score, lowest beam, largest logit, lowest token
        index = np.arange(beams * vocab)
        order = np.lexsort((index, -x[b].reshape(-1), index // vocab, -flat))[:n]
        out[0][b] = flat[order]
        out[1][b] = b * beams + order // vocab
        out[2][b] = order % vocab
        out[3][b] = np.array(near)[order // vocab]
    return out


def check(beam, logits, scores, n):
    best, parents, tokens = beam.beam_search_select(logits, scores, n)
    want, want_p, want_t, near = plain_select(logits, scores, n)
    got = best.cpu().double().numpy()
    assert np.array_equal(parents.cpu().numpy(), want_p)
    assert np.array_equal(tokens.cpu().numpy(), want_t)
    fin = np.isfinite(want)
    assert np.array_equal(np.isfinite(got), fin) and np.array_equal(got[~fin], want[~fin])
    assert (np.abs(got[fin] - want[fin]) <= near[fin] + 2.0 ** -24 * np.abs(want[fin])).all()


def _random(batch, beams, vocab, dtype, seed, spread=2.5):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(batch, beams, vocab, generator=g) * spread).to(dtype).to(DEV)
    return logits, (-20 * torch.rand(batch, beams, generator=g)).to(DEV)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("batch,beams,vocab,n", [
    (1, 1, 1, 1), (1, 1, 7, 7), (2, 3, 2, 6), (1, 4, 100, 32), (3, 5, 2047, 10), (1, 4, 2048, 8),
    (2, 1, 2049, 32), (1, 4, 32000, 8), (5, 8, 32003, 16), (1, 16, 50257, 32), (40, 8, 16385, 8),
    (2, 200, 33, 32)])
def test_select(beam, dtype, batch, beams, vocab, n):
    check(beam, *_random(batch, beams, vocab, dtype, seed=vocab + n), n)


@pytest.mark.parametrize("batch,beams,vocab", [(64, 8, 128256), (150, 4, 128256)])
def test_select_full_batches(beam, batch, beams, vocab):
    logits, scores = _random(batch, beams, vocab, torch.bfloat16, seed=batch)
    best, parents, tokens = beam.beam_search_select(logits, scores, 2 * beams)
    some = [0, batch // 2, batch - 1]
    want, want_p, want_t, _ = plain_select(logits[some], scores[some], 2 * beams)
    shift = torch.tensor([(b - i) * beams for i, b in enumerate(some)])[:, None]
    assert np.array_equal((parents[some].cpu() - shift).numpy(), want_p)
    assert np.array_equal(tokens[some].cpu().numpy(), want_t)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_equal_logits_go_by_their_index(beam, dtype):
    for vocab in (5, 3000, 40000):
        logits = torch.zeros(2, 3, vocab, dtype=dtype, device=DEV)
        logits[1, 2, vocab // 2:] = 1
        scores = torch.tensor([[-1.0, -1.0, -1.0], [-2.0, -1.5, -1.5]], device=DEV)
        check(beam, logits, scores, 9)
    # -0 and +0 are equal
    logits = torch.zeros(1, 1, 64, dtype=dtype, device=DEV)
    logits[0, 0, ::2] = -0.0
    check(beam, logits, torch.zeros(1, 1, device=DEV), 8)


def test_equal_beams_whatever_their_alignment(beam):
    """Rows of an odd vocabulary start at every alignment; equal rows score
    equally, so the lower beam comes first, token by token."""
    g = torch.Generator().manual_seed(4)
    for dtype in (torch.bfloat16, torch.float32):
        row = (torch.randn(32003, generator=g) * 3).to(dtype)
        logits = row.expand(1, 8, -1).contiguous().to(DEV)
        check(beam, logits, torch.full((1, 8), -3.0, device=DEV), 24)
        # a broadcast beam dimension
        check(beam, row.to(DEV).expand(1, 8, -1), torch.full((1, 8), -3.0, device=DEV), 24)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_strided_logits(beam, dtype):
    """A vocabulary cut out of padded rows, at odd offsets."""
    g = torch.Generator().manual_seed(5)
    wide = (torch.randn(3, 9, 5013, generator=g) * 3).to(dtype).to(DEV)
    for off in range(0, 10, 3):
        x = wide[:, 1::2, off:off + 5000 - off]
        check(beam, x, -torch.rand(3, 8, generator=g).to(DEV)[:, ::2], 8)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_masked_logits(beam, dtype):
    """Vocabularies masked to a few tokens, by -inf and by the type's lowest
    value, rows without any, NaN and +inf."""
    logits, scores = _random(4, 4, 3001, dtype, seed=6)
    logits[0, :, 3:] = -math.inf
    logits[1, :, 5:] = torch.finfo(dtype).min
    logits[2, 1] = -math.inf
    logits[2, 2] = torch.finfo(dtype).min
    logits[2, 3, ::2] = math.nan
    logits[3, 0] = math.nan
    logits[3, 1, 77] = math.inf
    logits[3, 2, 2990] = math.nan
    check(beam, logits, scores, 16)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("vocab", [136, 50000])
def test_certain_tokens_score_their_beam_exactly(beam, dtype, vocab):
    """A token of probability 1 adds 0, so beams of equal scores that are each
    certain of one tie, whatever its logit."""
    g = torch.Generator().manual_seed(31)
    logits = torch.full((4, 16, vocab), -90.0)
    where = torch.randint(0, vocab, (4, 16), generator=g)
    logits.scatter_(2, where[..., None], 20 * torch.randn(4, 16, 1, generator=g).clamp(-2, 2))
    scores = torch.full((4, 16), -10.737407684326172, device=DEV)
    best, parents, tokens = beam.beam_search_select(logits.to(dtype).to(DEV), scores, 16)
    assert (best == scores).all()
    assert torch.equal(parents.cpu().view(-1), torch.arange(64, dtype=torch.int32))
    assert torch.equal(tokens.cpu(), where.int())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("apart", [1, 256, 512, 4096])
@pytest.mark.parametrize("many", [1, 2, 3, 9, 40])
def test_best_logits_near_one_another(beam, dtype, many, apart):
    """The best ones sit in one vector, in neighbouring vectors or in several
    steps of one thread, in ascending and descending order."""
    logits, scores = _random(2, 3, 50000, dtype, 23)
    n = 16 // dtype.itemsize
    for w, start in ((0, 3), (1, 20000), (2, 0)):
        at = start + torch.arange(many) * (apart * n if apart > 1 else 1)
        at = at[at < 50000]
        up = 20 + torch.arange(len(at), dtype=torch.float32)
        logits[0, w, at] = up.to(dtype).to(DEV)
        logits[1, w, at] = up.flip(0).to(dtype).to(DEV)
    check(beam, logits, scores, 8)
    check(beam, logits, scores, 32)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("mask", ["lowest", -1e30, -1e20, -1e12, -3e9, -1e9, -math.inf])
def test_low_logits_among_masked_ones(beam, dtype, mask):
    """Log probabilities far below zero, most tokens masked: whole threads,
    steps and chunks hold masked logits only."""
    logits, scores = _random(3, 2, 30000, torch.float32, 19)
    logits -= 300
    g = torch.Generator().manual_seed(20)
    keep = (torch.rand(logits.shape, generator=g) < 0.002).to(DEV)
    keep[1, :, 4096:] = False
    keep[2, 1] = False
    low = torch.finfo(dtype).min
    value = low if mask == "lowest" else max(mask, low) if math.isfinite(mask) else mask
    check(beam, logits.masked_fill(~keep, value).to(dtype), scores, 8)


def test_beams_that_do_not_continue(beam):
    logits, scores = _random(5, 4, 2500, torch.bfloat16, seed=7)
    scores[0, 1:] = -math.inf           # a first step
    scores[1] = -math.inf               # a request that has ended
    scores[2, 0] = math.nan
    scores[3, 0] = -math.inf
    scores[3, 2:] = -math.inf
    logits[3, 1, 3:] = -math.inf        # three continuations in all
    scores[4] = -1e30
    check(beam, logits, scores, 8)


def test_scores_far_apart(beam):
    logits, scores = _random(3, 4, 5000, torch.float32, seed=8, spread=100.0)
    scores[0] = torch.tensor([-1e4, -2e4, -1e5, 0.0])
    scores[1] = torch.tensor([1e4, -2e4, 3e4, 0.0])
    check(beam, logits, scores, 8)


def test_layouts_against_the_threshold(beam):
    """In every warp's share of a chunk one thread holds low values only, so
    that nearly every element passes the threshold of 32 candidates; the same
    for the beams that the join looks at."""
    g = torch.Generator().manual_seed(9)
    for vocab, dtype in ((16384, torch.bfloat16), (40001, torch.bfloat16), (20000, torch.float32)):
        n = 128 // torch.finfo(dtype).bits  # logits in one 16-byte load
        x = 1 + torch.rand(600, 1, vocab, generator=g)
        idx = torch.arange(vocab)
        x[..., (idx // n) % 32 == 5] = 0
        logits = x.to(dtype).to(DEV)
        best, parents, tokens = beam.beam_search_select(logits, torch.zeros(600, 1, device=DEV), 32)
        some = [0, 311, 599]
        want, _, want_t, _ = plain_select(logits[some], torch.zeros(3, 1), 32)
        assert np.array_equal(tokens[some].cpu().numpy(), want_t)
        check(beam, logits[:1], torch.zeros(1, 1, device=DEV), 32)
    logits, scores = _random(2, 256, 100, torch.bfloat16, seed=10, spread=0.1)
    scores[:] = torch.arange(256) * 1e-3
    scores[:, 5::32] = -1e4
    check(beam, logits, scores, 32)


@pytest.mark.parametrize("order", ["up", "down"])
def test_sorted_logits(beam, order):
    x = torch.arange(70000, dtype=torch.float32, device=DEV) * 1e-3
    x = x if order == "up" else x.flip(0)
    check(beam, x.expand(2, 2, -1), torch.zeros(2, 2, device=DEV), 32)


def test_select_captured_and_replayed(beam, fi):
    logits, scores = _random(3, 4, 9000, torch.bfloat16, seed=11)
    fi._CHECK, saved = False, fi._CHECK
    try:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            beam.beam_search_select(logits, scores, 8)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            best, parents, tokens = beam.beam_search_select(logits, scores, 8)
        for seed in (12, 13):
            a, b = _random(3, 4, 9000, torch.bfloat16, seed=seed)
            logits.copy_(a)
            scores.copy_(b)
            graph.replay()
            torch.cuda.synchronize()
            _, want_p, want_t, _ = plain_select(a, b, 8)
            assert np.array_equal(parents.cpu().numpy(), want_p)
            assert np.array_equal(tokens.cpu().numpy(), want_t)
    finally:
        fi._CHECK = saved


# ------------------------------------------------- the operators as they run together
class TinyModel:
    """One attention layer over the cache with an embedding and a vocabulary."""

    def __init__(self, seed, vocab=50, hq=8, hkv=2, d=64):
        g = torch.Generator().manual_seed(seed)
        r = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16).to(DEV)  # noqa: E731
        self.q, self.k, self.v = r(vocab, hq, d), r(vocab, hkv, d), r(vocab, hkv, d)
        self.head = (torch.randn(hq * d, vocab, generator=g) / 8).to(DEV)
        self.hq, self.hkv, self.d, self.vocab = hq, hkv, d, vocab

    def logits(self, attended):
        return attended.float().reshape(attended.shape[0], -1) @ self.head

    def attend(self, tokens, window, sinks):
        """The attention of each row's last token over its own tokens, plainly."""
        n = tokens.shape[1]
        key = torch.arange(n, device=DEV)
        seen = (n - 1 - key <= window) | (key < sinks)
        q = self.q[tokens[:, -1]].double().view(-1, self.hkv, self.hq // self.hkv, self.d)
        s = torch.einsum("rhgd,rnhd->rhgn", q, self.k[tokens].double()) / math.sqrt(self.d)
        p = torch.softmax(s.masked_fill(~seen, -math.inf), -1)
        return torch.einsum("rhgn,rnhd->rhgd", p, self.v[tokens].double()).flatten(1, 2)


def test_beam_search_over_a_window_with_eviction_and_compaction(beam, fi):
    """Prefill of a prompt, then steps of select, fork, append and window
    decode, giving pages back on the way and moving the pool together: every
    beam's attention is that over its own tokens, and no page leaks."""
    pages = importlib.import_module("llm-inference-runtime_b200.pages")
    tables_mod = importlib.import_module("llm-inference-runtime_b200.tables")
    batch, beams, prompt, steps, window, sinks = 3, 4, 37, 45, 24, 2
    rows, width, total = batch * beams, 8, 80
    m = TinyModel(1)
    g = torch.Generator().manual_seed(2)
    text = torch.randint(0, m.vocab, (batch, prompt), generator=g).to(DEV)
    pool = torch.full((1, total, 2, m.hkv, P, m.d), math.nan, dtype=torch.bfloat16, device=DEV)
    refs = torch.zeros(total, dtype=torch.int32, device=DEV)
    tables = torch.full((rows, width), -1, dtype=torch.int32, device=DEV)
    held = _held(prompt)
    for b in range(batch):
        ids = torch.arange(b * held, (b + 1) * held, device=DEV)
        tables[b * beams:(b + 1) * beams, :held] = ids.int()
        refs[ids] = beams
    ws = torch.empty(128 << 20, dtype=torch.uint8, device=DEV)
    # the prompts, prefilled once per request through its first row
    lens = torch.full((rows,), prompt, dtype=torch.int32, device=DEV)
    first = tables[::beams]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    t = tables_mod.build_prefill_tables(first.contiguous(), i32([held] * batch), i32([prompt] * batch),
                                        i32([0] * batch), i32([prompt] * batch), P, batch * prompt)
    n_idx = batch * held
    fi.append_paged_kv_cache(m.k[text.flatten()], m.v[text.flatten()], t["batch_indices"],
                             t["positions"], pool[0], t["kv_indices"][:n_idx], t["kv_indptr"],
                             t["kv_last_page_len"], "HND")
    pw = fi.BatchPrefillWithSlidingWindowWrapper(ws, "HND", window_left=window, num_sink_tokens=sinks)
    pw.plan(t["qo_indptr"], t["kv_indptr"], t["kv_indices"][:n_idx], t["kv_last_page_len"], m.hq,
            m.hkv, m.d, P, causal=True, q_data_type=torch.bfloat16)
    out = pw.run(m.q[text.flatten()], pool[0])
    last = out.view(batch, prompt, m.hq, m.d)[:, -1].repeat_interleave(beams, 0)
    tokens = text.repeat_interleave(beams, 0)
    scores = torch.full((batch, beams), -math.inf, device=DEV)
    scores[:, 0] = 0
    dw = fi.BatchDecodeWithSlidingWindowWrapper(ws, "HND", window_left=window, num_sink_tokens=sinks)
    for step in range(steps):
        want = m.attend(tokens, window, sinks)
        assert (last.double() - want).abs().max() < 2e-2
        logits = m.logits(last).view(batch, beams, -1)
        _, want_p, want_t, _ = plain_select(logits, scores, beams)
        got = beam.beam_search_step(logits, scores, pool, tables, lens, refs)
        assert got["counts"][2] == 0
        assert np.array_equal(got["parents"].cpu().numpy(), want_p)
        assert np.array_equal(got["tokens"].cpu().numpy(), want_t)
        scores, tables, lens = got["scores"], got["block_tables"], got["seq_lens"]
        new = got["tokens"].view(-1).long()
        tokens = torch.cat([tokens[got["parents"].view(-1).long()], new[:, None]], 1)
        positions = lens.clone()
        lens = lens + 1
        assert (lens == tokens.shape[1]).all()
        d = tables_mod.build_decode_tables(tables, (lens + P - 1) // P, lens, P)
        count = int(((lens + P - 1) // P).sum())
        dw.plan(d["kv_indptr"], d["kv_indices"][:count], d["kv_last_page_len"], m.hq, m.hkv, m.d, P,
                q_data_type=torch.bfloat16)
        last = dw.run_with_append(m.q[new], pool[0], m.k[new], m.v[new], positions)
        if step % 4 == 1:
            pages.evict_window_pages(tables, lens, refs, window, sinks)
        if step % 10 == 7:
            remap, counts = pages.compact_pages(pool, tables, lens, refs)
            assert counts[2] == 0 and (refs[int(counts[0]):] == 0).all()
        # the counts are the tables' own
        want_refs = torch.zeros_like(refs)
        live = tables[tables >= 0].long()
        want_refs.index_add_(0, live, torch.ones_like(live, dtype=torch.int32))
        assert torch.equal(refs, want_refs)
    pages.free_sequences(tables, lens, refs)
    assert (refs == 0).all() and (tables == -1).all()


def _held(n):
    return -(-n // P)
