"""The operators around the paged cache that are measured, with their plain forms.

Six operators that serve long contexts and beams from one paged KV cache:

* ``window_decode``   one new token per request attends the last keys of its context and a few
                      first ones (sinks); with or without the append of that token
* ``window_prefill``  the same for chunks of new tokens over cached prefixes
* ``evict``           pages that lie wholly behind the window lose their reference
* ``compact``         the live pages of the pool move to its front, tables follow
* ``beam_select``     the best continuations over beams and vocabulary
* ``fork``            sequences continue from chosen parents: full pages are shared, the page that
                      the next token goes to is made private

Cache layout: pool [layers, pages, 2, kv heads, 16, head dim]; a sequence's pages are a row of a
block table or a run of a CSR list; an entry of -1 is a page that was given back.
"""

import importlib
import math
import random

import numpy as np
import torch

own = False

PAGE = 16
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
# q heads, kv heads, head dim of the two attention geometries that the configurations use
GEOMETRY = {"tinyllama": (32, 4, 64), "llama3": (32, 8, 128)}


def _package(name):
    return importlib.import_module("llm-inference-runtime_b200." + name)


# ------------------------------------------------------------------------------- cases
def listed():
    return [
        # one user's chat: a single request far past its window, one layer's call and its plan
        {"name": "decode, one request", "op": "window_decode", "geometry": "llama3", "batch": 1,
         "lo": 5000, "hi": 5000, "window": 1023, "sinks": 4, "layers": 1, "dtype": "bf16",
         "append": False, "mix": 1},
        # a serving step: a full batch with pages behind the window given back, the step's tokens
        # appended in the same call, four layers on one plan
        {"name": "decode, full batch", "op": "window_decode", "geometry": "tinyllama", "batch": 256,
         "lo": 1024, "hi": 4096, "window": 1023, "sinks": 4, "layers": 4, "dtype": "bf16",
         "append": True, "mix": 2},
        # a short follow-up prompt over a cached conversation
        {"name": "prefill, short prompt", "op": "window_prefill", "geometry": "tinyllama", "batch": 1,
         "qo_lo": 37, "qo_hi": 37, "pre_lo": 2001, "pre_hi": 2001, "window": 511, "sinks": 4,
         "dtype": "bf16", "mix": 4},
        # chunked prefill: sixteen chunks of 512 over prefixes of up to 2048 tokens
        {"name": "prefill, sixteen chunks", "op": "window_prefill", "geometry": "llama3", "batch": 16,
         "qo_lo": 512, "qo_hi": 512, "pre_lo": 0, "pre_hi": 2048, "window": 1023, "sinks": 4,
         "dtype": "bf16", "mix": 5},
        # one request's first beams, small vocabulary
        {"name": "select, four beams", "op": "beam_select", "batch": 1, "beams": 4, "vocab": 32000,
         "candidates": 8, "dtype": "bf16", "mix": 6},
        # a batch of requests with eight beams each, large vocabulary
        {"name": "select, full batch", "op": "beam_select", "batch": 64, "beams": 8,
         "vocab": 128256, "candidates": 16, "dtype": "bf16", "mix": 7},
        # beams of one request continue after a selection
        {"name": "fork, eight beams", "op": "fork", "geometry": "tinyllama", "layers": 22, "batch": 1,
         "beams": 8, "lo": 333, "hi": 333, "mix": 8},
        # every request of a batch reorders its beams
        {"name": "fork, full batch", "op": "fork", "geometry": "tinyllama", "layers": 22,
         "batch": 64, "beams": 8, "lo": 256, "hi": 2047, "mix": 9},
        # pages given back by a whole batch of long sequences at once
        {"name": "evict, full batch", "op": "evict", "batch": 512, "lo": 8192, "hi": 32768,
         "window": 4095, "sinks": 4, "mix": 10},
        # pages given back by a few sequences
        {"name": "evict, few sequences", "op": "evict", "batch": 3, "lo": 500, "hi": 2000,
         "window": 255, "sinks": 16, "mix": 11},
        # a pool that is two thirds full moves together, before a snapshot or a resize
        {"name": "compact, large pool", "op": "compact", "geometry": "llama3", "layers": 8,
         "pages": 6000, "batch": 64, "live": 0.66, "mix": 12},
        # a small pool with few holes
        {"name": "compact, small pool", "op": "compact", "geometry": "tinyllama", "layers": 2,
         "pages": 500, "batch": 8, "live": 0.9, "mix": 13},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case; its batch (or pool) is halved until it costs no more than the largest listed
    one of its operator."""
    c = _drawn(rng)
    most = [work(x) for x in listed() if x["op"] == c["op"]]
    size = "pages" if c["op"] == "compact" else "batch"
    while c[size] > 1 and any(work(c)[k] > max(w[k] for w in most) for k in ("bytes", "flops")):
        c[size] //= 2
    return c


def _drawn(rng):
    op = rng.choice(["window_decode", "window_decode", "window_prefill", "window_prefill",
                     "beam_select", "fork", "evict", "compact"])
    c = {"op": op, "mix": rng.randrange(1 << 30)}
    if op == "window_decode":
        c["geometry"] = rng.choice(sorted(GEOMETRY))
        c["batch"] = _log_int(rng, 1, 160)
        c["hi"] = _log_int(rng, 16, 16384)
        c["lo"] = rng.randint(1, c["hi"])
        c["window"] = _log_int(rng, 1, 3500) - 1
        c["sinks"] = rng.choice([0, 1, 4, 16, rng.randint(0, 130)])
        c["layers"] = rng.choice([1, 1, 2])
        c["dtype"] = rng.choice(["bf16", "fp16"])
        c["append"] = rng.random() < 0.4
    elif op == "window_prefill":
        c["geometry"] = rng.choice(sorted(GEOMETRY))
        c["batch"] = _log_int(rng, 1, 14)
        c["qo_hi"] = _log_int(rng, 1, 512)
        c["qo_lo"] = rng.randint(1, c["qo_hi"])
        c["pre_hi"] = _log_int(rng, 1, 4096)
        c["pre_lo"] = rng.randint(0, c["pre_hi"])
        c["window"] = _log_int(rng, 1, 1024) - 1
        c["sinks"] = rng.choice([0, 1, 4, 16, rng.randint(0, 130)])
        c["dtype"] = rng.choice(["bf16", "fp16"])
    elif op == "beam_select":
        c["batch"] = _log_int(rng, 1, 60)
        c["beams"] = rng.randint(1, 8)
        c["vocab"] = _log_int(rng, 100, 128000)
        c["candidates"] = min(32, c["vocab"], rng.choice([c["beams"], 2 * c["beams"]]))
        c["dtype"] = rng.choice(["bf16", "fp16", "fp32"])
    elif op == "fork":
        c["geometry"] = rng.choice(sorted(GEOMETRY))
        c["layers"] = rng.randint(1, 10)
        c["batch"] = _log_int(rng, 1, 40)
        c["beams"] = rng.randint(1, 8)
        c["hi"] = _log_int(rng, 16, 1200)
        c["lo"] = rng.randint(1, c["hi"])
    elif op == "evict":
        c["batch"] = _log_int(rng, 1, 500)
        c["hi"] = _log_int(rng, 64, 30000)
        c["lo"] = rng.randint(1, c["hi"])
        c["window"] = _log_int(rng, 1, 8192) - 1
        c["sinks"] = rng.choice([0, 1, 4, 16, rng.randint(0, 130)])
    else:
        c["geometry"] = rng.choice(sorted(GEOMETRY))
        c["layers"] = rng.randint(1, 8)
        c["pages"] = _log_int(rng, 100, 5500)
        c["batch"] = rng.randint(1, 64)
        c["live"] = rng.uniform(0.3, 0.95)
    return c


# -------------------------------------------------------------------- shapes from a case
def _lengths(case, n, lo, hi, salt=0):
    """n lengths in [lo, hi], the same for every seed (the work of a case does not change)."""
    rng = random.Random(case["mix"] * 7 + salt)
    return np.array([rng.randint(lo, hi) for _ in range(n)], dtype=np.int64)


def _pages(length):
    return (length + PAGE - 1) // PAGE


def _visible_from(first_query, window):
    """First key that a query at position first_query sees through the window."""
    return np.maximum(first_query - window, 0)


def _dead_pages(first_query, case):
    """[begin, end) of the pages that no query from first_query on can see."""
    begin = np.full_like(first_query, _pages(case["sinks"]))
    return begin, np.maximum(begin, _visible_from(first_query, case["window"]) // PAGE)


def _attention_shape(case):
    if case["op"] == "window_decode":
        kv = _lengths(case, case["batch"], case["lo"], case["hi"])
        return np.ones_like(kv), kv
    qo = _lengths(case, case["batch"], case["qo_lo"], case["qo_hi"], 1)
    return qo, qo + _lengths(case, case["batch"], case["pre_lo"], case["pre_hi"], 2)


def _seen(case, qo, kv):
    """(query, key) pairs that are seen, and keys that some query sees, over the batch."""
    pairs = keys = 0
    for n, length in zip(qo.tolist(), kv.tolist()):
        pos = np.arange(length - n, length)
        start = _visible_from(pos, case["window"])
        pairs += int((pos + 1 - start + np.minimum(case["sinks"], start)).sum())
        keys += int(length - start[0] + min(case["sinks"], start[0]))
    return pairs, keys


def _fork_shape(case):
    """Lengths of the rows, parents (whole rows' numbers), and how many last pages are shared."""
    rng = random.Random(case["mix"])
    rows, beams = case["batch"] * case["beams"], case["beams"]
    lens = np.repeat(_lengths(case, case["batch"], case["lo"], case["hi"]), beams)
    parents = [b * beams + min(int(rng.expovariate(1.0) * beams / 3), beams - 1)
               for b in range(case["batch"]) for _ in range(beams)]
    shared = [min(beams, 1 + rng.randrange(beams)) for _ in range(case["batch"])]
    return rows, lens, np.array(parents, dtype=np.int64), shared


def _fork_copies(case):
    rows, lens, parents, _ = _fork_shape(case)
    seen, n = set(), 0
    for r in range(rows):
        p = int(parents[r])
        if lens[p] % PAGE:
            n += p in seen
            seen.add(p)
    return n


def work(case):
    op = case["op"]
    if op in ("window_decode", "window_prefill"):
        hq, hkv, d = GEOMETRY[case["geometry"]]
        layers = case.get("layers", 1)
        qo, kv = _attention_shape(case)
        pairs, keys = _seen(case, qo, kv)
        rows = int(qo.sum())
        moved = keys * hkv * d * 2 * 2 + rows * hq * d * 2 * 2
        if case.get("append"):
            moved += rows * hkv * d * 2 * 2
        return {"bytes": layers * moved, "flops": layers * pairs * hq * d * 4}
    if op == "beam_select":
        n = case["batch"] * case["beams"] * case["vocab"]
        size = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": n * size + case["batch"] * case["candidates"] * 12, "flops": 4 * n}
    if op == "fork":
        _, hkv, d = GEOMETRY[case["geometry"]]
        rows, lens, _, _ = _fork_shape(case)
        entries = int(_pages(lens).sum())
        page = 2 * hkv * PAGE * d * 2 * case["layers"]
        return {"bytes": 2 * _fork_copies(case) * page + 4 * (4 * entries + 4 * rows), "flops": entries}
    if op == "evict":
        lens = _lengths(case, case["batch"], case["lo"], case["hi"])
        begin, end = _dead_pages(lens - 1, case)
        n = int((end - begin).sum())
        return {"bytes": 16 * n + 4 * case["batch"], "flops": n + case["batch"]}
    _, hkv, d = GEOMETRY[case["geometry"]]
    page = 2 * hkv * PAGE * d * 2 * case["layers"]
    live = _compact_live(case)
    moves = int(live[int(live.sum()):].sum())
    return {"bytes": 2 * moves * page + 12 * case["pages"] + 8 * int(live.sum()), "flops": case["pages"]}


def _compact_live(case):
    rng = np.random.RandomState(case["mix"] % (1 << 31))
    return rng.random_sample(case["pages"]) < case["live"]


# ----------------------------------------------------------------------------- prepare
def _i32(a):
    return torch.as_tensor(np.ascontiguousarray(a).astype(np.int32)).cuda()


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    rng = np.random.RandomState(seed % (1 << 31))
    state = {"case": dict(case)}
    op = case["op"]
    if op in ("window_decode", "window_prefill"):
        _prepare_attention(case, state, gen, rng)
    elif op == "beam_select":
        rows = case["batch"] * case["beams"]
        # the spread of a language model's logits, and sums of log probabilities so far
        logits = torch.randn(rows, case["vocab"], device="cuda", generator=gen) * 2.5
        state["logits"] = logits.to(DTYPES[case["dtype"]]).view(case["batch"], case["beams"], -1)
        state["scores"] = -20 * torch.rand(case["batch"], case["beams"], device="cuda", generator=gen)
    elif op == "fork":
        _prepare_fork(case, state, gen, rng)
    elif op == "evict":
        lens = _lengths(case, case["batch"], case["lo"], case["hi"])
        # a quarter of the sequences share their pages with the one before them
        stride = int(_pages(lens).max())
        tables = np.full((case["batch"], stride), -1, dtype=np.int64)
        pages = int(_pages(lens).sum())
        ids, at = rng.permutation(pages), 0
        refs = np.zeros(pages, dtype=np.int64)
        for b, n in enumerate(_pages(lens).tolist()):
            tables[b, :n] = ids[at:at + n]
            at += n
            if b % 4 == 3:
                m = min(n, int(_pages(lens[b - 1])) - 1)
                tables[b, :m] = tables[b - 1, :m]
            np.add.at(refs, tables[b, :n], 1)
        state["tables"], state["lens"], state["refs"] = _i32(tables), _i32(lens), _i32(refs)
    else:
        _prepare_compact(case, state, gen, rng)
    torch.cuda.synchronize()
    return state


def _normal(shape, dtype, gen):
    return torch.randn(shape, device="cuda", dtype=dtype, generator=gen)


def _prepare_attention(case, state, gen, rng):
    hq, hkv, d = GEOMETRY[case["geometry"]]
    dtype = DTYPES[case["dtype"]]
    layers = case.get("layers", 1)
    qo, kv = _attention_shape(case)
    order = rng.permutation(case["batch"])
    qo, kv = qo[order], kv[order]
    begin, end = _dead_pages(kv - qo, case)
    indptr = np.concatenate([[0], np.cumsum(_pages(kv))])
    used = int(indptr[-1] - (end - begin).sum())
    pool_pages = used + 7
    ids, at = rng.permutation(pool_pages), 0
    indices = np.full(int(indptr[-1]), -1, dtype=np.int64)
    for b in range(case["batch"]):
        mask = np.ones(int(indptr[b + 1] - indptr[b]), dtype=bool)
        mask[begin[b]:end[b]] = False
        n = int(mask.sum())
        indices[indptr[b]:indptr[b + 1]][mask] = ids[at:at + n]
        at += n
    rows = int(qo.sum())
    state["indptr"], state["indices"] = _i32(indptr), _i32(indices)
    state["last"] = _i32((kv - 1) % PAGE + 1)
    state["lens"], state["positions"] = _i32(kv), _i32(kv - 1)
    state["qo_indptr"] = _i32(np.concatenate([[0], np.cumsum(qo)]))
    state["rows"], state["longest"] = rows, int(qo.max())
    # the most keys that one request's queries see together
    state["keys"] = int(np.max(kv - np.maximum(_visible_from(kv - qo, case["window"]) - case["sinks"], 0)))
    state["pool"] = _normal((layers, pool_pages, 2, hkv, PAGE, d), dtype, gen)
    state["q"] = _normal((layers, rows, hq, d), dtype, gen)
    if case.get("append"):
        state["k"] = _normal((layers, rows, hkv, d), dtype, gen)
        state["v"] = _normal((layers, rows, hkv, d), dtype, gen)
    state["workspace"] = torch.empty(128 << 20, dtype=torch.uint8, device="cuda")


def _prepare_fork(case, state, gen, rng):
    _, hkv, d = GEOMETRY[case["geometry"]]
    rows, lens, parents, shared = _fork_shape(case)
    stride = int(lens.max()) // PAGE + 2
    tables = np.full((rows, stride), -1, dtype=np.int64)
    counts = _pages(lens)
    total = 2 * rows  # room for the pages that the fork hands out
    for b in range(case["batch"]):
        total += int(counts[b * case["beams"]]) + 2 * case["beams"]
    ids, at = rng.permutation(total), 0
    refs = np.zeros(total, dtype=np.int64)
    for b in range(case["batch"]):
        r0, n = b * case["beams"], int(counts[b * case["beams"]])
        common = max(n - 2, 0)  # beams share all but their last pages
        tables[r0:r0 + case["beams"], :common] = ids[at:at + common]
        at += common
        for w in range(case["beams"]):
            tail = n - common
            if w < shared[b] or w == 0 or tail == 0 or common == 0:
                tables[r0 + w, common:n] = ids[at:at + tail]
                at += tail
            else:  # a beam that also shares its last full page with beam 0
                tables[r0 + w, common:n - 1] = tables[r0, common:n - 1]
                tables[r0 + w, n - 1] = ids[at]
                at += 1
            np.add.at(refs, tables[r0 + w, :n], 1)
    state["tables"], state["lens"] = _i32(tables), _i32(lens)
    state["parents"], state["refs"] = _i32(parents), _i32(refs)
    state["pool"] = _normal((case["layers"], total, 2, hkv, PAGE, d), torch.bfloat16, gen)


def _prepare_compact(case, state, gen, rng):
    _, hkv, d = GEOMETRY[case["geometry"]]
    live = _compact_live(case)
    ids = np.nonzero(live)[0]
    ids = ids[rng.permutation(len(ids))]
    batch = min(case["batch"], max(1, len(ids)))
    cuts = np.linspace(0, len(ids), batch + 1).astype(np.int64)
    lens = (cuts[1:] - cuts[:-1]) * PAGE - rng.randint(0, PAGE, batch)
    lens = np.maximum(lens, 0)
    tables = np.full((batch, max(1, int((cuts[1:] - cuts[:-1]).max()))), -1, dtype=np.int64)
    for b in range(batch):
        tables[b, :cuts[b + 1] - cuts[b]] = ids[cuts[b]:cuts[b + 1]]
    state["tables"], state["lens"], state["refs"] = _i32(tables), _i32(lens), _i32(live)
    state["pool"] = _normal((case["layers"], case["pages"], 2, hkv, PAGE, d), torch.bfloat16, gen)


# --------------------------------------------------------------------------------- run
def run(state):
    op = state["case"]["op"]
    if own:
        return _OWN[op](state, state["case"])
    return _PLAIN[op](state, state["case"])


def _own_window_decode(s, case):
    hq, hkv, d = GEOMETRY[case["geometry"]]
    w = _package("flashinfer_api").BatchDecodeWithSlidingWindowWrapper(
        s["workspace"], "HND", window_left=case["window"], num_sink_tokens=case["sinks"])
    w.plan(s["indptr"], s["indices"], s["last"], hq, hkv, d, PAGE, q_data_type=s["q"].dtype)
    out = torch.empty_like(s["q"])
    lse = torch.empty(out.shape[:3], dtype=torch.float32, device="cuda")
    for i in range(case["layers"]):
        if case["append"]:
            w.run_with_append(s["q"][i], s["pool"][i], s["k"][i], s["v"][i], s["positions"],
                              out=out[i], lse=lse[i], return_lse=True)
        else:
            w.run(s["q"][i], s["pool"][i], out=out[i], lse=lse[i], return_lse=True)
    return (out, lse, s["pool"]) if case["append"] else (out, lse)


def _own_window_prefill(s, case):
    hq, hkv, d = GEOMETRY[case["geometry"]]
    w = _package("flashinfer_api").BatchPrefillWithSlidingWindowWrapper(
        s["workspace"], "HND", window_left=case["window"], num_sink_tokens=case["sinks"])
    w.plan(s["qo_indptr"], s["indptr"], s["indices"], s["last"], hq, hkv, d, PAGE, causal=True,
           q_data_type=s["q"].dtype, total_qo=s["rows"])
    return w.run(s["q"][0], s["pool"][0], return_lse=True)


def _own_beam_select(s, case):
    return _package("beam").beam_search_select(s["logits"], s["scores"], case["candidates"])


def _own_fork(s, case):
    refs = s["refs"].clone()
    tables, lens, counts = _package("pages").fork_sequences(
        s["pool"], s["tables"], s["lens"], s["parents"], refs)
    return tables, lens, counts, refs, s["pool"]


def _own_evict(s, case):
    tables, refs = s["tables"].clone(), s["refs"].clone()
    counts = _package("pages").evict_window_pages(tables, s["lens"], refs, case["window"],
                                                  case["sinks"])
    return tables, refs, counts


def _own_compact(s, case):
    tables, refs = s["tables"].clone(), s["refs"].clone()
    remap, counts = _package("pages").compact_pages(s["pool"], tables, s["lens"], refs)
    return tables, refs, remap, counts, s["pool"]


_OWN = {"window_decode": _own_window_decode, "window_prefill": _own_window_prefill,
        "beam_select": _own_beam_select, "fork": _own_fork, "evict": _own_evict,
        "compact": _own_compact}


# ------------------------------------------------------------------------- plain forms
def _keys_of(s, first_query, case):
    """Positions of the keys that a request's queries see, [batch, keys] with -1 behind the last:
    the sinks, then the window of the first query up to the last key."""
    start = (first_query - case["window"]).clamp(min=0)
    sinks = start.clamp(max=case["sinks"])
    m = torch.arange(s["keys"], device="cuda")[None]
    pos = torch.where(m < sinks[:, None], m, m - sinks[:, None] + start[:, None])
    return torch.where(pos < s["lens"].long()[:, None], pos, -1)


def _gather(s, pos):
    """K and V at those positions of every layer, float32 [batch, keys, layers, kv heads, dim]."""
    at = pos.clamp(min=0)
    page = s["indices"].long()[s["indptr"].long()[:-1, None] + at // PAGE].clamp(min=0)
    kv = s["pool"][:, page, :, :, at % PAGE]  # [batch, keys, layers, 2, kv heads, dim]
    kv = kv.masked_fill((pos < 0)[..., None, None, None, None], 0)
    return kv[:, :, :, 0].float(), kv[:, :, :, 1].float()


def _attend(scores, v_product):
    """exp(scores - max) @ V / sum, and the base-2 log of the sum; rows that see nothing give 0."""
    top = scores.amax(-1, keepdim=True)
    weight = (scores - torch.where(top == -math.inf, torch.zeros_like(top), top)).exp()
    total = weight.sum(-1, keepdim=True)
    out = v_product(weight) / total.clamp(min=1e-37)
    return out, (top + total.log())[..., 0] * math.log2(math.e)


def _plain_window_decode(s, case):
    hq, hkv, d = GEOMETRY[case["geometry"]]
    lens, table = s["lens"].long(), s["indices"].long()
    if case["append"]:
        at = s["positions"].long()
        page = table[s["indptr"].long()[:-1] + at // PAGE]
        new = torch.stack([s["k"], s["v"]], 3).transpose(0, 1)  # [batch, layers, heads, 2, dim]
        s["pool"][:, page, :, :, at % PAGE] = new.transpose(2, 3)
    pos = _keys_of(s, lens - 1, case)
    k, v = _gather(s, pos)
    q = s["q"].float().view(case["layers"], case["batch"], hkv, hq // hkv, d)
    scores = torch.einsum("lbhgd,bmlhd->lbhgm", q, k) / math.sqrt(d)
    scores = scores.masked_fill((pos < 0)[None, :, None, None], -math.inf)
    out, lse = _attend(scores, lambda w: torch.einsum("lbhgm,bmlhd->lbhgd", w, v))
    out = out.reshape(s["q"].shape).to(s["q"].dtype)
    lse = lse.reshape(out.shape[:3])
    return (out, lse, s["pool"]) if case["append"] else (out, lse)


def _plain_window_prefill(s, case):
    hq, hkv, d = GEOMETRY[case["geometry"]]
    lens, first = s["lens"].long(), s["qo_indptr"].long()
    qo = first[1:] - first[:-1]
    pos = _keys_of(s, lens - qo, case)
    k, v = _gather(s, pos)
    i = torch.arange(s["longest"], device="cuda")[None]
    row = (first[:-1, None] + i).clamp(max=s["rows"] - 1)
    q = s["q"][0][row].float().view(case["batch"], s["longest"], hkv, hq // hkv, d)
    at = (lens - qo)[:, None] + i  # a query's position
    sees = (pos[:, None] >= 0) & (pos[:, None] <= at[..., None])
    sees &= (pos[:, None] >= at[..., None] - case["window"]) | (pos[:, None] < case["sinks"])
    scores = torch.einsum("bqhgd,bmhd->bhgqm", q, k[:, :, 0]) / math.sqrt(d)
    scores = scores.masked_fill(~sees[:, None, None], -math.inf)
    out, lse = _attend(scores, lambda w: torch.einsum("bhgqm,bmhd->bhgqd", w, v[:, :, 0]))
    out = out.permute(0, 3, 1, 2, 4).reshape(case["batch"], s["longest"], hq, d)
    lse = lse.permute(0, 3, 1, 2).reshape(case["batch"], s["longest"], hq)
    owner = torch.bucketize(torch.arange(s["rows"], device="cuda"), first[1:], right=True)
    local = torch.arange(s["rows"], device="cuda") - first[owner]
    return out[owner, local].to(s["q"].dtype), lse[owner, local]


def _plain_beam_select(s, case):
    batch, beams, vocab, n = case["batch"], case["beams"], case["vocab"], case["candidates"]
    x = s["logits"].double()
    top = x.amax(-1, keepdim=True)
    norm = (top + (x - top).exp().sum(-1, keepdim=True).log()).float()
    score = (s["scores"].double()[..., None] + (x - norm.double())).view(batch, -1)
    # the n best, equal ones by the lowest index: all above the n-th value, then the first equal ones
    least = score.topk(n).values[:, -1:]
    above, equal = score > least, score == least
    left = n - above.sum(-1, keepdim=True)
    take = above | (equal & (equal.cumsum(-1) <= left))
    place = torch.arange(score.shape[1], 0, -1, device="cuda")[None]
    index = (take * place).topk(n).indices  # in the order of their index
    value, order = score.gather(1, index).sort(dim=-1, descending=True, stable=True)
    index = index.gather(1, order)
    row = torch.arange(batch, device="cuda")[:, None] * beams + index // vocab
    return value.float(), row.int(), (index % vocab).int()


def _plain_fork(s, case):
    tables, lens, parents = s["tables"].long(), s["lens"].long(), s["parents"].long()
    pool, refs = s["pool"], s["refs"].long()
    rows, stride = tables.shape
    n = refs.numel()
    full, part = lens // PAGE, lens % PAGE > 0
    j = torch.arange(stride, device="cuda")[None]
    children = torch.zeros(rows, dtype=torch.long, device="cuda").index_add_(0, parents, torch.ones_like(parents))
    held = (j < full[:, None]) & (tables >= 0)
    refs.index_add_(0, tables.clamp(min=0).view(-1), torch.where(held, children[:, None] - 1, 0).view(-1))
    last = tables.gather(1, full[:, None])[:, 0]
    refs.index_add_(0, last.clamp(min=0), torch.where(part, -1, 0))
    # of the rows that continue one unfinished page the first keeps it, unless others hold it too
    mine, full, part = last[parents], full[parents], part[parents]
    r = torch.arange(rows, device="cuda")
    first = torch.full((n,), rows, device="cuda").scatter_reduce_(
        0, torch.where(part, mine, 0), torch.where(part, r, rows), "amin")
    keep = part & (refs[mine.clamp(min=0)] == 0) & (first[mine.clamp(min=0)] == r)
    refs.index_add_(0, mine.clamp(min=0), keep.long())
    # the others take free pages, lowest number first
    free = (refs == 0).long()
    slot = torch.full((n + rows + 1,), -1, device="cuda")
    slot.scatter_(0, torch.where(free > 0, free.cumsum(0) - 1, n + rows), torch.arange(n, device="cuda"))
    wants = (~keep).long()
    new = torch.where(keep, mine, slot[wants.cumsum(0) - 1])
    got = ~keep & (new >= 0)
    refs.index_add_(0, new.clamp(min=0), got.long())
    source = (got & part).nonzero()[:, 0]
    pool[:, new[source]] = pool[:, mine[source]]
    out = torch.where(j < full[:, None], tables[parents], -1)
    out.scatter_(1, full[:, None], new[:, None])
    missing = (~keep & (new < 0)).sum()
    counts = torch.stack([(got & part).sum(), got.sum(), missing])
    return out.int(), lens[parents].int(), counts.int(), refs.int(), pool


def _plain_evict(s, case):
    tables, lens, refs = s["tables"].long(), s["lens"].long(), s["refs"].long()
    j = torch.arange(tables.shape[1], device="cuda")[None]
    end = (lens - 1 - case["window"]).clamp(min=0) // PAGE
    gone = (j >= -(-case["sinks"] // PAGE)) & (j < end[:, None]) & (tables >= 0)
    left = refs.index_add(0, tables.clamp(min=0).view(-1), -gone.long().view(-1))
    freed = ((refs > 0) & (left == 0)).sum()
    counts = torch.stack([gone.sum(), freed, torch.zeros_like(freed)])
    return torch.where(gone, -1, tables).int(), left.int(), counts.int()


def _plain_compact(s, case):
    tables, lens, refs, pool = s["tables"].long(), s["lens"].long(), s["refs"], s["pool"]
    live = refs > 0
    count = live.sum()
    i = torch.arange(refs.numel(), device="cuda")
    source = (live & (i >= count)).nonzero()[:, 0]
    target = (~live & (i < count)).nonzero()[:, 0]
    remap = torch.where(live, i, -1)
    remap[source] = target
    pool[:, target] = pool[:, source]
    new = torch.zeros_like(refs)
    new[remap[live]] = refs[live]
    j = torch.arange(tables.shape[1], device="cuda")[None]
    held = (j < (lens[:, None] + PAGE - 1) // PAGE) & (tables >= 0)
    tables = torch.where(held, remap[tables.clamp(min=0)], tables)
    counts = torch.stack([count, torch.full_like(count, source.numel()), torch.zeros_like(count)])
    return tables.int(), new, remap.int(), counts.int(), pool


_PLAIN = {"window_decode": _plain_window_decode, "window_prefill": _plain_window_prefill,
          "beam_select": _plain_beam_select, "fork": _plain_fork, "evict": _plain_evict,
          "compact": _plain_compact}


# ------------------------------------------------------------------------------- exact
def exact(case, seed):
    """What run() returns, from the definitions, in 64 bits, one request after the other."""
    s = prepare(case, seed)
    op = case["op"]
    if op in ("window_decode", "window_prefill"):
        return _exact_attention(case, s)
    if op == "beam_select":
        logp = torch.log_softmax(s["logits"].double(), -1) + s["scores"].double()[..., None]
        best = logp.flatten(1).topk(case["candidates"]).values
        return best, None, None
    if op == "fork":
        pool = s["pool"]
        tables, parents = s["tables"].cpu().tolist(), s["parents"].cpu().tolist()
        lens, refs = s["lens"].cpu().tolist(), s["refs"].cpu().tolist()
        for r, length in enumerate(lens):
            for page in tables[r][:-(-length // PAGE)]:
                refs[page] -= 1
        last, claimed = {}, set()
        for p in parents:
            for page in tables[p][:lens[p] // PAGE]:
                refs[page] += 1
        for r, p in enumerate(parents):
            if lens[p] % PAGE:
                last[r] = tables[p][lens[p] // PAGE]
        outside = {page for page in last.values() if refs[page] > 0}
        todo = []
        for r in range(len(parents)):
            if r in last and last[r] not in outside and last[r] not in claimed:
                claimed.add(last[r])
                refs[last[r]] += 1
            else:
                todo.append(r)
        free = [i for i, n in enumerate(refs) if n == 0]
        for r, page in zip(todo, free):
            if r in last:
                pool[:, page] = pool[:, last[r]]
        return None, None, None, None, pool
    if op == "compact":
        pool, refs = s["pool"], s["refs"].cpu().tolist()
        count = sum(n > 0 for n in refs)
        holes = iter([i for i in range(count) if refs[i] == 0])
        for i in range(count, len(refs)):
            if refs[i] > 0:
                pool[:, next(holes)] = pool[:, i]
        return None, None, None, None, pool
    return None


def _exact_attention(case, s):
    hq, hkv, d = GEOMETRY[case["geometry"]]
    indptr, kv = s["indptr"].cpu().tolist(), s["lens"].cpu().tolist()
    rows, pool = s["qo_indptr"].cpu().tolist(), s["pool"]
    layers = pool.shape[0]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(out.shape[:3], dtype=torch.float64, device="cuda")
    if case.get("append"):
        for b, length in enumerate(kv):
            page = int(s["indices"][indptr[b] + (length - 1) // PAGE])
            pool[:, page, 0, :, (length - 1) % PAGE] = s["k"][:, b]
            pool[:, page, 1, :, (length - 1) % PAGE] = s["v"][:, b]
    for b, length in enumerate(kv):
        n = rows[b + 1] - rows[b]
        at = torch.arange(length - n, length, device="cuda")
        key = torch.arange(length, device="cuda")
        sees = (key[None] <= at[:, None]) & ((at[:, None] - key[None] <= case["window"])
                                             | (key[None] < case["sinks"]))
        key = key[sees.any(0)]
        sees = sees[:, sees.any(0)]
        page = s["indices"][indptr[b]:indptr[b + 1]].long()[key // PAGE]
        for i in range(layers):
            k = pool[i][page, 0, :, key % PAGE].double().repeat_interleave(hq // hkv, 1)
            v = pool[i][page, 1, :, key % PAGE].double().repeat_interleave(hq // hkv, 1)
            q = s["q"][i, rows[b]:rows[b + 1]].double()
            score = torch.einsum("qhd,khd->hqk", q, k) / math.sqrt(d)
            score = torch.where(sees[None], score, -math.inf)
            lse[i, rows[b]:rows[b + 1]] = torch.logsumexp(score, -1).T / math.log(2)
            out[i, rows[b]:rows[b + 1]] = torch.einsum("hqk,khd->qhd", torch.softmax(score, -1), v)
    if case["op"] == "window_prefill":
        return out[0], lse[0]
    return (out, lse, pool) if case.get("append") else (out, lse)
