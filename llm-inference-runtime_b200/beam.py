"""Beam search over the paged cache: selection and the reordering of states.

The reference decodes greedily or by sampling, one sequence per request
(src/engine/runtime/step_executor.py:204-260). These calls add what a step of
beam search needs between the model's logits and the next forward: the best
continuations of each request's beams, and the cache following them
(``pages.fork_sequences``), on the device without a synchronisation.
"""

from __future__ import annotations

import functools
from typing import Dict, Optional, Tuple

import torch

from . import _lib, pages
from .flashinfer_api import _after, _device_guard, _stream

_DTYPES = {torch.float16: _lib.PA_DTYPE_F16, torch.bfloat16: _lib.PA_DTYPE_BF16,
           torch.float32: _lib.PA_DTYPE_F32}
MAX_CANDIDATES = 32
MAX_BEAMS = 256
MAX_VOCAB = 2 ** 24
MAX_ROWS = 2 ** 31 - 1  # of all requests' beams


@functools.lru_cache(maxsize=256)
def _workspace_bytes(device_index: int, *sizes: int) -> int:
    """A function of the sizes and the device's SM count alone."""
    return _lib.load().pa_beam_select_workspace_bytes(*sizes)


def beam_search_select(logits: torch.Tensor, scores: torch.Tensor, num_candidates: int
                       ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The ``num_candidates`` best continuations of each request.

    logits [batch, beams, vocab] (float16 / bfloat16 / float32, last dim
    contiguous), scores [batch, beams] float32: accumulated log probabilities
    (-inf: a beam that does not continue, as all but the first of a request
    have before the first step). A continuation scores ``scores[b, w] +
    log_softmax(logits[b, w])[v]``. Returns (scores, parents, tokens), each
    [batch, num_candidates], best first; equal scores by the lowest beam,
    inside a beam by the larger logit, then the lowest token. parents are
    rows ``b * beams + w``, as ``pages.fork_sequences`` takes them. A NaN
    logit counts as -inf. At most 32 candidates of 256 beams."""
    if logits.dim() != 3 or scores.dim() != 2 or logits.shape[:2] != scores.shape:
        raise ValueError("logits must be [batch, beams, vocab] and scores [batch, beams]")
    if logits.dtype not in _DTYPES:
        raise NotImplementedError(f"logits of {logits.dtype} are not supported")
    if scores.dtype != torch.float32:
        raise TypeError("scores must be float32")
    if not logits.is_cuda or scores.device != logits.device:
        raise ValueError("logits and scores must be on one GPU")
    batch, beams, vocab = logits.shape
    n = int(num_candidates)
    if beams == 0 or vocab == 0 or not 1 <= n <= beams * vocab:
        raise ValueError("num_candidates must be in [1, beams * vocab]")
    if (n > MAX_CANDIDATES or beams > MAX_BEAMS or vocab > MAX_VOCAB
            or batch * beams > MAX_ROWS):
        raise NotImplementedError(f"at most {MAX_CANDIDATES} candidates of {MAX_BEAMS} beams and "
                                  f"{MAX_VOCAB} tokens, {MAX_ROWS} beams in all")
    if vocab > 1 and logits.stride(2) != 1:
        raise ValueError("the vocabulary dimension of logits must be contiguous")
    if scores.size(1) > 1 and scores.stride(1) != 1:
        scores = scores.contiguous()
    device = logits.device
    dtype = _DTYPES[logits.dtype]
    best = torch.empty((batch, n), dtype=torch.float32, device=device)
    parents = torch.empty((batch, n), dtype=torch.int32, device=device)
    tokens = torch.empty_like(parents)
    if batch == 0:
        return best, parents, tokens
    with _device_guard(device):
        size = _workspace_bytes(device.index, batch, beams, vocab, n, dtype)
        ws = torch.empty(size, dtype=torch.uint8, device=device)
        _lib.check(_lib.load().pa_beam_select(
            logits.data_ptr(), logits.stride(0), logits.stride(1), scores.data_ptr(),
            scores.stride(0), batch, beams, vocab, n, dtype, best.data_ptr(), parents.data_ptr(),
            tokens.data_ptr(), ws.data_ptr(), size, _stream()), "beam_search_select")
        _after("beam_search_select")
    return best, parents, tokens


def beam_search_step(logits: torch.Tensor, scores: torch.Tensor, kv_pool: torch.Tensor,
                     block_tables: torch.Tensor, seq_lens: torch.Tensor,
                     ref_counts: torch.Tensor, kv_layout: str = "HND",
                     active: Optional[torch.Tensor] = None) -> Dict[str, torch.Tensor]:
    """One step of beam search: each request's beams are replaced by its
    ``beams`` best continuations and their cache follows. As many candidates
    as beams are selected, so there are at most 32 beams here.

    Row ``b * beams + w`` of ``block_tables`` / ``seq_lens`` is beam w of
    request b. Returns scores, parents and tokens [batch, beams] and the new
    block_tables, seq_lens and counts (``pages.fork_sequences``): every beam
    owns the page that its token, to be fed to the model next, is appended
    to, at position seq_lens[r] (the lengths to pass to the next step are these
    plus one). A beam for which the pool had no page is counted in counts[2] and
    keeps its full pages only (``all_held`` there): until it is ended, each step
    counts it again.

    ``active`` [batch] bool: requests that go on. The rows of the others end,
    in this step and in every later one that names them: they give up their
    pages, take none, and come back with parent -1, length 0 (which stays 0)
    and a table of -1. Their scores and tokens mean nothing. Without it every
    row takes the page of its next token, a row without a continuation (score
    -inf) or of length 0 too, so a request that has ended has to be named:
    ``active=(scores > -inf).any(1)``, where its scores say so."""
    batch, beams = scores.shape
    if seq_lens.numel() != batch * beams:
        raise ValueError("block_tables must hold one row per beam of each request")
    if active is not None and (active.dtype != torch.bool or active.shape != (batch,)
                               or active.device != logits.device):
        raise ValueError("active must be a bool tensor of one entry per request, on the same GPU")
    best, parents, tokens = beam_search_select(logits, scores, beams)
    if active is not None:
        parents = parents.masked_fill(~active[:, None], -1)
    tables, lens, counts = pages.fork_sequences(kv_pool, block_tables, seq_lens,
                                                parents.view(-1), ref_counts,
                                                kv_layout=kv_layout, all_held=True)
    return {"scores": best, "parents": parents, "tokens": tokens, "block_tables": tables,
            "seq_lens": lens, "counts": counts}
