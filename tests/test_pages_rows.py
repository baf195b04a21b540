"""Arguments of the calls on rows at the ends of their life, on the CPU: each
returns or raises before any launch."""

from __future__ import annotations

import ctypes
import importlib

import pytest
import torch

D = ctypes.c_void_p(0x1000)
OTHER = ctypes.c_void_p(0x2000)


@pytest.fixture(scope="module")
def lib(lir):
    lir.build.build()
    return lir._lib.load()


@pytest.mark.parametrize("name", ["pa_fork_sequences", "pa_fork_held_sequences"])
def test_both_forks_check_the_same_arguments(lib, lir, name):
    E = lir._lib

    def call(pool=D, pb=4096, n=10, tables=D, width=4, lens=D, parents=D, rows=2, page=16, refs=D,
             out=OTHER, out_lens=D, counts=D, ws=D):
        return getattr(lib, name)(pool, 1 << 20, 2, 4096, pb, n, tables, 4, width, lens, parents,
                                  rows, page, refs, out, 4, out_lens, counts, ws, None)

    for kw in (dict(pool=None), dict(pb=24), dict(n=0), dict(tables=None), dict(width=0),
               dict(width=5), dict(lens=None), dict(parents=None), dict(rows=-1), dict(page=0),
               dict(refs=None), dict(out=D), dict(out=None), dict(out_lens=None), dict(counts=None),
               dict(ws=None)):
        assert call(**kw) == E.PA_ERR_INVALID_ARGUMENT, kw


def test_a_step_checks_which_requests_go_on(lir):
    beam = importlib.import_module("llm-inference-runtime_b200.beam")
    t, n = torch.zeros((6, 4), dtype=torch.int32), torch.zeros(6, dtype=torch.int32)
    pool = torch.zeros((1, 4, 2, 1, 16, 8), dtype=torch.bfloat16)
    x, s = torch.zeros(2, 3, 10), torch.zeros(2, 3)
    for bad in (torch.ones(2), torch.ones(3, dtype=torch.bool), torch.ones(2, 3, dtype=torch.bool)):
        with pytest.raises(ValueError, match="active"):
            beam.beam_search_step(x, s, pool, t, n, n, active=bad)


def test_rows_of_a_selection_are_counted_together(lib, lir):
    """As many requests as give 2^31 - 1 beams pass (the workspace is looked at
    next), one more beam is refused."""
    E = lir._lib

    def call(batch, beams):
        return lib.pa_beam_select(D, 400, 100, D, 4, batch, beams, 100, 8, E.PA_DTYPE_F32, D, D, D, D,
                                  100, None)

    for batch, beams in ((65536, 4), (2 ** 31 - 1, 1), (2 ** 23 - 1, 256)):
        assert call(batch, beams) == E.PA_ERR_WORKSPACE_TOO_SMALL, (batch, beams)
    for batch, beams in ((2 ** 23, 256), (2 ** 30, 2)):
        assert call(batch, beams) == E.PA_ERR_UNSUPPORTED, (batch, beams)
