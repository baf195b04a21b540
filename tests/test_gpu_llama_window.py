"""The patched LLaMA model with a sliding window, and in a beam search, against
transformers' eager attention on the same weights (the tolerances of
test_gpu_llama.py: bf16 logits of a two-layer model)."""

from __future__ import annotations

import copy
import importlib
import math

import numpy as np
import pytest
import torch

from test_gpu_beam import plain_select
from test_gpu_llama import DEV, P, _close, _model, _tables

pytestmark = pytest.mark.gpu
HD = 512 // 8


def _t(a):
    return torch.as_tensor(np.asarray(a)).to(DEV)


def _window_mask(n, window, sinks):
    pos, key = np.arange(n)[:, None], np.arange(n)[None]
    seen = (key <= pos) & ((pos - key <= window) | (key < sinks))
    mask = torch.where(torch.from_numpy(seen), 0.0, torch.finfo(torch.bfloat16).min)
    return mask[None, None].to(torch.bfloat16).to(DEV)


def _eager(ref, ids, window=None, sinks=0):
    kw = {} if window is None else {"attention_mask": _window_mask(len(ids), window, sinks)}
    with torch.no_grad():
        return ref(input_ids=_t([ids]), use_cache=False, **kw).logits[0]


def test_patched_model_with_a_window_and_evicted_pages(fi):
    """Chunked prefill and decode steps past the window; between the steps the
    pages behind it go back to the pool and are overwritten."""
    llama = importlib.import_module("llm-inference-runtime_b200.llama")
    pages = importlib.import_module("llm-inference-runtime_b200.pages")
    window, sinks = 40, 3
    ref = _model()
    ours = copy.deepcopy(ref)
    llama.patch_llama_model(ours)
    pool = torch.zeros((2, 40, 2, 2, P, HD), dtype=torch.bfloat16, device=DEV)
    rng = np.random.default_rng(2)
    ids = rng.integers(0, 512, 150).tolist()
    table = torch.full((1, 12), -1, dtype=torch.int32, device=DEV)
    need = math.ceil((len(ids) + 5) / P)
    table[0, :need] = _t(rng.permutation(40)[:need]).int()
    refs = torch.zeros(40, dtype=torch.int32, device=DEV)
    refs[table[0, :need].long()] = 1
    try:
        llama.init_flashinfer_state(kv_pool=pool, page_size=P, device=DEV, window_left=window,
                                    num_sink_tokens=sinks)
        done = 0
        for chunk in (70, 17, 63):
            n = done + chunk
            held = math.ceil(n / P)
            indptr, _, last = _tables([n], [held], [np.arange(held)])
            llama.build_batch_indices_positions(_t(np.array([0, chunk], dtype=np.int32)),
                                                _t(np.array([n], dtype=np.int32)), nnz=chunk)
            llama.plan_prefill(qo_indptr=_t(np.array([0, chunk], dtype=np.int32)),
                               kv_indptr=_t(indptr), kv_indices=table[0, :held].contiguous(),
                               kv_last_page_len=_t(last), num_qo_heads=8, num_kv_heads=2,
                               head_dim=HD)
            with torch.no_grad():
                logits = ours(input_ids=_t([ids[done:n]]),
                              position_ids=_t([list(range(done, n))]), use_cache=False).logits[0]
            rel, cos = _close(logits, _eager(ref, ids[:n], window, sinks)[done:])
            assert rel < 0.05 and cos > 0.999, (n, rel, cos)
            done = n
            pages.evict_window_pages(table, _t(np.array([n], dtype=np.int32)), refs, window, sinks)
            pool[:, refs == 0] = math.nan
        assert (table[0, :need] == -1).sum() == (150 - 1 - window) // P - 1
        for _ in range(5):
            ids.append(int(rng.integers(0, 512)))
            n = len(ids)
            held = math.ceil(n / P)
            indptr, _, last = _tables([n], [held], [np.arange(held)])
            llama.PagedAttnState.batch_indices = _t(np.zeros(1, dtype=np.int32))
            llama.PagedAttnState.positions = _t(np.array([n - 1], dtype=np.int32))
            llama.plan_decode(kv_indptr=_t(indptr), kv_indices=table[0, :held].contiguous(),
                              kv_last_page_len=_t(last), num_qo_heads=8, num_kv_heads=2,
                              head_dim=HD)
            with torch.no_grad():
                logits = ours(input_ids=_t([[ids[-1]]]), position_ids=_t([[n - 1]]),
                              use_cache=False).logits[0, -1]
            rel, cos = _close(logits, _eager(ref, ids, window, sinks)[-1])
            assert rel < 0.05 and cos > 0.999, (n, rel, cos)
    finally:
        llama.init_flashinfer_state(kv_pool=pool, page_size=P, device=DEV)
    assert isinstance(llama.PagedAttnState.decode_wrapper, fi.BatchDecodeWithPagedKVCacheWrapper)
    assert not isinstance(llama.PagedAttnState.decode_wrapper, fi.BatchDecodeWithSlidingWindowWrapper)


def test_sinks_without_a_window_are_refused(fi):
    llama = importlib.import_module("llm-inference-runtime_b200.llama")
    pool = torch.zeros((2, 4, 2, 2, P, HD), dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError, match="window_left"):
        llama.init_flashinfer_state(kv_pool=pool, page_size=P, device=DEV, num_sink_tokens=3)


def test_patched_model_in_a_beam_search(fi):
    """Prompts of two requests, prefilled once each, then steps of three beams:
    the choice is the plain one on the model's logits, and each beam's logits
    are those of its own tokens."""
    llama = importlib.import_module("llm-inference-runtime_b200.llama")
    beam = importlib.import_module("llm-inference-runtime_b200.beam")
    tables_mod = importlib.import_module("llm-inference-runtime_b200.tables")
    ref = _model()
    ours = copy.deepcopy(ref)
    llama.patch_llama_model(ours)
    pool = torch.zeros((2, 48, 2, 2, P, HD), dtype=torch.bfloat16, device=DEV)
    llama.init_flashinfer_state(kv_pool=pool, page_size=P, device=DEV)
    rng = np.random.default_rng(5)
    prompts = [rng.integers(0, 512, n).tolist() for n in (29, 48)]
    beams, width = 3, 6
    held = [math.ceil(len(p) / P) for p in prompts]
    table = torch.full((2 * beams, width), -1, dtype=torch.int32, device=DEV)
    refs = torch.zeros(48, dtype=torch.int32, device=DEV)
    ids, at = rng.permutation(48), 0
    for b, n in enumerate(held):
        table[b * beams:(b + 1) * beams, :n] = _t(ids[at:at + n]).int()
        refs[_t(ids[at:at + n]).long()] = beams
        at += n
    lens = _t(np.repeat([len(p) for p in prompts], beams).astype(np.int32))
    indptr, indices, last = _tables([len(p) for p in prompts], held, [ids[:held[0]], ids[held[0]:at]])
    qo = np.concatenate([[0], np.cumsum([len(p) for p in prompts])]).astype(np.int32)
    llama.build_batch_indices_positions(_t(qo), lens[::beams].contiguous(), nnz=int(qo[-1]))
    llama.plan_prefill(qo_indptr=_t(qo), kv_indptr=_t(indptr), kv_indices=_t(indices),
                       kv_last_page_len=_t(last), num_qo_heads=8, num_kv_heads=2, head_dim=HD)
    with torch.no_grad():
        logits = ours(input_ids=_t([prompts[0] + prompts[1]]),
                      position_ids=_t([list(range(29)) + list(range(48))]), use_cache=False).logits[0]
    logits = logits[_t(qo[1:] - 1).long()].repeat_interleave(beams, 0)
    scores = torch.full((2, beams), -math.inf, device=DEV)
    scores[:, 0] = 0
    texts = [list(prompts[b]) for b in range(2) for _ in range(beams)]
    for step in range(20):
        x = logits.view(2, beams, -1)
        _, want_p, want_t, _ = plain_select(x, scores, beams)
        got = beam.beam_search_step(x, scores, pool, table, lens, refs)
        assert np.array_equal(got["parents"].cpu().numpy(), want_p)
        assert np.array_equal(got["tokens"].cpu().numpy(), want_t) and got["counts"][2] == 0
        new = got["tokens"].view(-1)
        texts = [texts[p] + [int(n)] for p, n in zip(got["parents"].view(-1).tolist(), new.tolist())]
        scores, table = got["scores"], got["block_tables"]
        lens = got["seq_lens"] + 1
        d = tables_mod.build_decode_tables(table, (lens + P - 1) // P, lens, P)
        count = int(((lens + P - 1) // P).sum())
        llama.PagedAttnState.batch_indices = d["batch_indices"]
        llama.PagedAttnState.positions = d["positions"]
        llama.plan_decode(kv_indptr=d["kv_indptr"], kv_indices=d["kv_indices"][:count],
                          kv_last_page_len=d["kv_last_page_len"], num_qo_heads=8, num_kv_heads=2,
                          head_dim=HD)
        with torch.no_grad():
            logits = ours(input_ids=new[:, None].long(), position_ids=d["positions"][:, None].long(),
                          use_cache=False).logits[:, -1]
        if step % 6 == 5:
            for r, text in enumerate(texts):
                rel, cos = _close(logits[r], _eager(ref, text)[-1])
                assert rel < 0.05 and cos > 0.999, (step, r, rel, cos)
