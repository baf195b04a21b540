"""The patched model's state when a window is refused, on the CPU."""

from __future__ import annotations

import importlib

import pytest
import torch

FIELDS = ("kv_pool", "page_size", "dtype", "window_left", "num_sink_tokens", "workspace_buffer",
          "prefill_wrapper", "decode_wrapper")


def test_a_refused_window_leaves_the_state_as_it_was(lir):
    llama = importlib.import_module("llm-inference-runtime_b200.llama")
    state = llama.PagedAttnState
    saved = {name: getattr(state, name) for name in FIELDS}
    try:
        pool = torch.zeros((1, 2, 2, 1, 16, 64), dtype=torch.bfloat16)
        llama.init_flashinfer_state(kv_pool=pool, page_size=16, device="cpu", window_left=40,
                                    num_sink_tokens=3)
        before = {name: getattr(state, name) for name in FIELDS}
        assert before["window_left"] == 40 and before["kv_pool"] is pool
        other = torch.zeros((1, 4, 2, 1, 8, 64), dtype=torch.float16)
        for kw in (dict(num_sink_tokens=3), dict(window_left=-1), dict(window_left=2 ** 31),
                   dict(window_left=4, num_sink_tokens=-1)):
            with pytest.raises(ValueError):
                llama.init_flashinfer_state(kv_pool=other, page_size=8, device="cpu", **kw)
            for name in FIELDS:
                assert getattr(state, name) is before[name], name
        llama.init_flashinfer_state(kv_pool=other, page_size=8, device="cpu")
        assert state.window_left is None and state.kv_pool is other and state.page_size == 8
    finally:
        for name in FIELDS:
            setattr(state, name, saved[name])
