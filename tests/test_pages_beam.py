"""Arguments of the page and beam-search calls, on the CPU: each returns or
raises before any launch."""

from __future__ import annotations

import ctypes
import importlib

import pytest
import torch


@pytest.fixture(scope="module")
def lib(lir):
    lir.build.build()
    return lir._lib.load()


D = ctypes.c_void_p(0x1000)
OTHER = ctypes.c_void_p(0x2000)
ODD = ctypes.c_void_p(0x1008)


def test_release_arguments(lib, lir):
    E = lir._lib

    def call(tables=D, stride=4, width=4, lens=D, batch=2, page=16, sinks=0, refs=D, n=10, counts=D):
        return lib.pa_release_pages(tables, stride, width, lens, batch, page, 5, sinks, refs, n,
                                    counts, None)

    assert call(stride=3) == call(width=-1) == call(batch=-1) == call(page=0) == call(sinks=-1) == \
        call(refs=None) == call(n=0) == call(counts=None) == call(lens=None) == \
        call(tables=None) == E.PA_ERR_INVALID_ARGUMENT


def test_fork_arguments(lib, lir):
    E = lir._lib

    def call(pool=D, ls=1 << 20, layers=2, ps=4096, pb=4096, n=10, tables=D, width=4, stride=4,
             lens=D, parents=D, rows=2, page=16, refs=D, out=OTHER, out_stride=4, out_lens=D,
             counts=D, ws=D):
        return lib.pa_fork_sequences(pool, ls, layers, ps, pb, n, tables, stride, width, lens,
                                     parents, rows, page, refs, out, out_stride, out_lens, counts,
                                     ws, None)

    bad = [dict(pool=None), dict(pool=ODD), dict(ls=8), dict(layers=-1), dict(ps=4095), dict(pb=24),
           dict(pb=8192), dict(n=0), dict(n=1 << 31), dict(tables=None), dict(width=0),
           dict(stride=3), dict(lens=None), dict(parents=None), dict(rows=-1), dict(page=0),
           dict(refs=None), dict(out=D), dict(out=None), dict(out_stride=3), dict(out_lens=None),
           dict(counts=None), dict(ws=None)]
    for kw in bad:
        assert call(**kw) == E.PA_ERR_INVALID_ARGUMENT, kw


def test_compact_arguments(lib, lir):
    E = lir._lib

    def call(pool=D, pb=4096, n=10, tables=D, width=4, stride=4, lens=D, batch=2, page=16, refs=D,
             remap=D, counts=D, ws=D):
        return lib.pa_compact_pages(pool, 1 << 20, 2, 4096, pb, n, tables, stride, width, lens,
                                    batch, page, refs, remap, counts, ws, None)

    for kw in (dict(pool=ODD), dict(pb=-16), dict(n=0), dict(tables=None), dict(stride=1),
               dict(lens=None), dict(batch=-1), dict(page=0), dict(refs=None), dict(remap=None),
               dict(counts=None), dict(ws=None)):
        assert call(**kw) == E.PA_ERR_INVALID_ARGUMENT, kw


def test_beam_arguments(lib, lir):
    E = lir._lib

    def call(logits=D, scores=D, batch=2, beams=4, vocab=100, k=8, dtype=1, out=D, ws=D, size=1 << 30):
        return lib.pa_beam_select(logits, 400, 100, scores, 4, batch, beams, vocab, k, dtype, out, out,
                                  out, ws, size, None)

    for kw in (dict(logits=None), dict(scores=None), dict(batch=-1), dict(beams=0), dict(vocab=0),
               dict(k=0), dict(k=401), dict(out=None), dict(ws=None), dict(ws=ODD),
               dict(logits=ctypes.c_void_p(0x1001)), dict(logits=ctypes.c_void_p(0x1002), dtype=2)):
        assert call(**kw) == E.PA_ERR_INVALID_ARGUMENT, kw
    for kw in (dict(k=33), dict(beams=257), dict(dtype=3), dict(vocab=(1 << 24) + 1)):
        assert call(**kw) == E.PA_ERR_UNSUPPORTED, kw
    assert call(batch=0) == E.PA_OK
    assert call(size=100) == E.PA_ERR_WORKSPACE_TOO_SMALL
    assert lib.pa_beam_select_workspace_bytes(2, 4, 100, 33, 1) == 0


def test_python_checks(lir):
    pages = importlib.import_module("llm-inference-runtime_b200.pages")
    beam = importlib.import_module("llm-inference-runtime_b200.beam")
    t = torch.zeros((2, 4), dtype=torch.int32)
    n = torch.zeros(2, dtype=torch.int32)
    pool = torch.zeros((1, 4, 2, 1, 16, 8), dtype=torch.bfloat16)
    # host tensors, and types that are not int32, are refused
    for call in (lambda t: pages.evict_window_pages(t, n, n, 4), lambda t: pages.free_sequences(t, n, n),
                 lambda t: pages.fork_sequences(pool, t, n, n, n),
                 lambda t: pages.compact_pages(pool, t, n, n)):
        with pytest.raises(ValueError, match="GPU"):
            call(t)
        with pytest.raises(TypeError):
            call(t.long())
    for kw in (dict(window_left=-1), dict(window_left=2 ** 31), dict(window_left=3, num_sink_tokens=-1)):
        with pytest.raises(ValueError, match="window_left"):
            pages.evict_window_pages(t, n, n, **kw)
    x, s = torch.zeros(2, 3, 10), torch.zeros(2, 3)
    with pytest.raises(ValueError, match="GPU"):
        beam.beam_search_select(x, s, 3)
    with pytest.raises(ValueError):
        beam.beam_search_select(x[0], s, 3)
    with pytest.raises(NotImplementedError):
        beam.beam_search_select(x.double(), s, 3)
    with pytest.raises(TypeError):
        beam.beam_search_select(x, s.double(), 3)
