"""Arguments of the sliding-window entry points, on the CPU: each call returns
or raises before any launch."""

from __future__ import annotations

import ctypes
import importlib

import pytest
import torch


@pytest.fixture(scope="module")
def api(lir):
    lir.build.build()
    return importlib.import_module("llm-inference-runtime_b200.flashinfer_api")


@pytest.mark.parametrize("name", ["BatchDecodeWithSlidingWindowWrapper",
                                  "BatchPrefillWithSlidingWindowWrapper"])
def test_constructor_checks_the_window(api, name):
    cls = getattr(api, name)
    ws = torch.empty(16, dtype=torch.uint8)
    with pytest.raises(TypeError):
        cls(ws, "HND")
    for kw in ({"window_left": -1}, {"window_left": 2 ** 31}, {"window_left": 4, "num_sink_tokens": -1},
               {"window_left": 4, "num_sink_tokens": 2 ** 31}):
        with pytest.raises(ValueError):
            cls(ws, "HND", **kw)
    with pytest.raises(KeyError):
        cls(ws, "DHN", window_left=4)
    w = cls(ws, "HND", window_left=0, num_sink_tokens=3)
    with pytest.raises(RuntimeError, match="plan"):
        w.run(torch.zeros(1, 8, 64, dtype=torch.bfloat16),
              torch.zeros(4, 2, 2, 16, 64, dtype=torch.bfloat16))
    t = torch.zeros(2, dtype=torch.int32)
    for kw in ({"window_left": 5}, {"logits_soft_cap": 1.0}, {"pos_encoding_mode": "ROPE_LLAMA"}):
        with pytest.raises(NotImplementedError):
            args = (t, t, t, t) if "Prefill" in name else (t, t, t)
            w.plan(*args, 8, 2, 64, 16, **kw)


def test_window_calls_check_their_arguments(lir):
    lib = lir._lib.load()
    E = lir._lib
    d = ctypes.c_void_p(0x1000)

    def plan(batch=4, n=10, hq=32, hkv=4, dim=64, page=16, window=7, sinks=0, indices=d, ws=d):
        return lib.pa_window_decode_plan(d, indices, d, batch, n, hq, hkv, dim, page, window, sinks,
                                         ws, 1 << 30, None)

    assert plan(window=-1) == plan(sinks=-1) == plan(batch=0) == plan(hq=30) == \
        plan(indices=None) == plan(ws=ctypes.c_void_p(0x1008)) == E.PA_ERR_INVALID_ARGUMENT
    assert plan(dim=96) == plan(page=8) == plan(hq=128) == E.PA_ERR_UNSUPPORTED

    def prefill(window=7, sinks=0, hq=32, dim=64):
        return lib.pa_window_prefill_plan(d, d, d, 4, 100, 10, hq, 4, dim, 16, window, sinks, d,
                                          1 << 30, None)

    assert prefill(window=-1) == prefill(sinks=-1) == prefill(hq=30) == E.PA_ERR_INVALID_ARGUMENT
    assert prefill(dim=32) == prefill(hq=12) == E.PA_ERR_UNSUPPORTED

    desc = E.PagedKVCache()
    desc.k_base, desc.v_base = 0x1000, 0x2000
    desc.page_stride, desc.head_stride, desc.token_stride = 2 * 4 * 16 * 64, 16 * 64, 64
    desc.num_pages, desc.num_kv_heads, desc.page_size, desc.head_dim = 8, 4, 16, 64
    desc.dtype = E.PA_DTYPE_BF16

    def run(window=7, sinks=0, q=d):
        return lib.pa_window_decode_run(q, 2048, 64, ctypes.byref(desc), d, d, d, 4, 10, 32, window,
                                        sinks, 0.0, d, 1 << 30, d, None, None)

    assert run(window=-1) == run(sinks=-1) == E.PA_ERR_INVALID_ARGUMENT
    odd = ctypes.c_void_p(0x1008)
    assert lib.pa_window_decode_append_run(
        d, 2048, 64, odd, 256, 64, d, 256, 64, d, ctypes.byref(desc), d, d, d, 4, 10, 32, 7, 0, 0.0,
        d, 1 << 30, d, None, None) == E.PA_ERR_INVALID_ARGUMENT
    assert lib.pa_window_prefill_run(
        d, 2048, 64, ctypes.byref(desc), d, d, d, d, 4, 100, 32, 1, -1, 0, 0.0, d, 1 << 30, d, None,
        None) == E.PA_ERR_INVALID_ARGUMENT
    desc.head_dim = 96
    assert run() == E.PA_ERR_UNSUPPORTED


class _OnGpu:
    """A stand-in for a tensor of GPU 0, where there is none."""

    device = "cuda:0"

    def __init__(self, like):
        self._like = like

    def __getattr__(self, name):
        return getattr(self._like, name)

    def get_device(self):
        return 0


@pytest.mark.parametrize("name", ["BatchDecodeWithSlidingWindowWrapper",
                                  "BatchPrefillWithSlidingWindowWrapper"])
def test_run_refuses_tensors_that_do_not_fit(api, name):
    """Other devices than the workspace's, outputs of another type or shape."""
    w = getattr(api, name)(_OnGpu(torch.empty(16, dtype=torch.uint8)), "HND", window_left=4)
    w._planned = True  # as after a plan
    q = torch.zeros(2, 8, 64, dtype=torch.bfloat16)
    pool = torch.zeros(4, 2, 2, 16, 64, dtype=torch.bfloat16)
    halves = (pool[:, 0], pool[:, 1])
    lse = torch.zeros(2, 8)
    on = _OnGpu
    for bad in ((q, pool), (on(q), pool), (on(q), halves), (on(q), (on(halves[0]), halves[1])),
                (q, (on(halves[0]), on(halves[1])))):
        with pytest.raises(ValueError, match="device"):
            w.run(*bad)
    cache = (on(halves[0]), on(halves[1]))
    for out in (on(q.float()), q):
        with pytest.raises(ValueError, match="out"):
            w.run(on(q), cache, out=out)
    for bad in (lse.double(), lse[:1], lse.t().contiguous().t(), lse[0]):
        with pytest.raises(ValueError, match="lse"):
            w.run(on(q), cache, lse=on(bad))
    with pytest.raises(ValueError, match="lse"):
        w.run(on(q), cache, lse=lse)
