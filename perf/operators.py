"""The operators of a generation step that are measured: what is run, on which inputs, and what it costs.

Three operators meet in the single-token step of a language model: the new keys and values are quantised into the
cache (and read back where a long prompt continues), attention reads the quantised cache, and a token is drawn from
the logits.  ``run`` computes each in its plain form out of elementary torch operations, or, with ``own`` set, through
this package's entry points.

* cache row (one token of one head, ``x[d]``): ``a = max|x|``; int8: ``scale = a / 127``, ``code = rint(x * 127 / a)``
  with ties to even; e4m3: ``scale = a / 448``, ``code = e4m3(x * 448 / a)``.  The row stands for ``code * scale``.
* attention: query ``i`` of ``n`` stands at ``p = length - n + i`` and sees slots ``max(first, p - window + 1) .. p``
  (``window`` 0: from ``first``); a query that sees nothing gives zeros.  Query head ``h`` uses key head ``h // group``.
* sampling: tokens ordered by logit (descending, then index); top-k keeps the first k, top-p those before which less
  than ``top_p`` of the top-k mass lies, min-p those with at least ``min_p`` of the largest probability; the result is
  the lowest index at which the running mass of the kept tokens, in index order, exceeds ``uniform`` times their sum.
  ``temperature`` 0 is arg-max.
"""
import math

import torch

own = False

FULL = 8 * 131072 * 128           # elements of K (and of V) in the largest cache that is listed


def listed():
    return [
        # -- attention over the quantised cache ------------------------------------------------------------------
        # a few words of a chat with a small model: pure latency
        dict(name="attend_few_tokens", op="attend", batch=1, kv_heads=2, group=4, queries=1, dim=64, slots=64, shortest=37,
             longest=37, fmt="int8", dtype="float16", window=0, padded=False),
        # batch-1 generation with the 8B shapes (32 query heads on 8 key heads), a kilobyte prompt
        dict(name="attend_one_sequence", op="attend", batch=1, kv_heads=8, group=4, queries=1, dim=128, slots=4096,
             shortest=1151, longest=1151, fmt="int8", dtype="bfloat16", window=0, padded=False),
        # a serving batch at the decoder's default cache length, every sequence at another position, left-padded
        dict(name="attend_batch", op="attend", batch=32, kv_heads=8, group=4, queries=1, dim=128, slots=4096,
             shortest=2048, longest=4096, fmt="int8", dtype="bfloat16", window=0, padded=True),
        # one very long context
        dict(name="attend_long", op="attend", batch=1, kv_heads=8, group=4, queries=1, dim=128, slots=131072,
             shortest=131071, longest=131071, fmt="e4m3", dtype="bfloat16", window=0, padded=False),
        # five drafted tokens verified at once, wide heads, a sliding window
        dict(name="attend_draft", op="attend", batch=8, kv_heads=4, group=2, queries=5, dim=256, slots=8192,
             shortest=3001, longest=8192, fmt="e4m3", dtype="float16", window=2500, padded=False),
        # -- the cache written and read back ---------------------------------------------------------------------
        # the single-token step of a batch
        dict(name="cache_one_token", op="cache", batch=32, kv_heads=8, tokens=1, dim=128, slots=4096, shortest=2048,
             longest=4095, fmt="int8", dtype="bfloat16", read="new"),
        # a prompt's next chunk: written, then everything so far read back for an ordinary attention
        dict(name="cache_chunk", op="cache", batch=2, kv_heads=8, tokens=517, dim=128, slots=8192, shortest=6001,
             longest=6517, fmt="e4m3", dtype="bfloat16", read="all"),
        # a batch of whole prompts
        dict(name="cache_prompts", op="cache", batch=32, kv_heads=8, tokens=2048, dim=128, slots=4096, shortest=0,
             longest=0, fmt="int8", dtype="float16", read="new"),
        # -- sampling --------------------------------------------------------------------------------------------
        # a small vocabulary, FP32 logits, min-p
        dict(name="sample_small", op="sample", rows=3, vocab=5003, dtype="float32", temperature=1.0, top_k=0, top_p=1.0,
             min_p=0.05, mixed=False, masked=False),
        # batch-1 generation with the 8B shape's head, the usual settings
        dict(name="sample_one_row", op="sample", rows=1, vocab=151936, dtype="bfloat16", temperature=0.6, top_k=20,
             top_p=0.95, min_p=0.0, mixed=False, masked=False),
        # a serving batch in which every request brings its own settings, some constrained by a grammar
        dict(name="sample_mixed_rows", op="sample", rows=64, vocab=151936, dtype="bfloat16", temperature=0.8, top_k=50,
             top_p=0.9, min_p=0.02, mixed=True, masked=True),
        # a large batch, nucleus only: nothing but the whole row's mass tells where the cut lies
        dict(name="sample_nucleus", op="sample", rows=256, vocab=128256, dtype="bfloat16", temperature=1.0, top_k=0,
             top_p=0.9, min_p=0.0, mixed=False, masked=False),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(("attend", "attend", "cache", "sample"))
    if op == "sample":
        vocab = _log_int(rng, 1000, 152000)
        kind = rng.choice(("plain", "top_k", "top_p", "min_p", "all"))
        return dict(op=op, rows=_log_int(rng, 1, 256 * 128256 // max(vocab, 128256)), vocab=vocab,
                    dtype=rng.choice(("bfloat16", "float16", "float32")), temperature=rng.choice((0.3, 0.7, 1.0, 1.5)),
                    top_k=_log_int(rng, 1, 600) if kind in ("top_k", "all") else 0,
                    top_p=round(rng.uniform(0.1, 0.99), 3) if kind in ("top_p", "all") else 1.0,
                    min_p=round(rng.uniform(0.005, 0.3), 3) if kind in ("min_p", "all") else 0.0,
                    mixed=rng.random() < 0.3, masked=rng.random() < 0.3)
    kv_heads = rng.choice((1, 2, 4, 8, 16))
    dim = rng.choice((64, 64, 80, 96, 128, 128, 128, 192, 256))
    fmt, dtype = rng.choice(("int8", "e4m3")), rng.choice(("bfloat16", "float16"))
    if op == "cache":
        batch = _log_int(rng, 1, 32)
        slots = _log_int(rng, 16, max(16, FULL // (2 * batch * kv_heads * dim)))
        tokens = 1 if rng.random() < 0.3 else _log_int(rng, 1, slots)
        shortest = rng.randint(0, slots - tokens)
        return dict(op=op, batch=batch, kv_heads=kv_heads, tokens=tokens, dim=dim, slots=slots,
                    shortest=shortest, longest=rng.randint(shortest, slots - tokens), fmt=fmt, dtype=dtype, read=rng.choice(("new", "all")))
    batch = _log_int(rng, 1, 64)
    slots = _log_int(rng, 16, max(16, min(131072, FULL // (batch * kv_heads * dim))))
    queries = 1 if rng.random() < 0.6 else rng.randint(2, 8)
    group = rng.choice((1, 2, 3, 4, 4, 5, 7, 8, 16))
    if slots * batch * kv_heads * dim * queries * group > 8 * FULL:
        queries, group = 1, min(group, 8)
    shortest = rng.randint(queries, slots)
    return dict(op=op, batch=batch, kv_heads=kv_heads, group=group, queries=queries, dim=dim, slots=slots,
                shortest=shortest, longest=rng.randint(shortest, slots), fmt=fmt, dtype=dtype,
                window=_log_int(rng, 1, slots) if rng.random() < 0.25 else 0, padded=rng.random() < 0.25)


# ---------------------------------------------------------------------------------------------------- inputs
def _top(fmt):
    return 127.0 if fmt == "int8" else 448.0


def _quantise(x, fmt):
    """Codes and scales of the rows of ``x`` (last dimension); the code is decided in 64 bits."""
    a = x.abs().amax(-1, keepdim=True).float()
    finite = torch.isfinite(a)
    scale = torch.where(finite, a / _top(fmt), torch.full_like(a, math.nan))
    q = x.double() * _top(fmt) / a.double()
    q = torch.where(finite & (a > 0), q, torch.zeros_like(q))
    codes = q.round().to(torch.int8) if fmt == "int8" else q.float().to(torch.float8_e4m3fn)
    return codes, scale.squeeze(-1)


def _keys(gen, shape, dtype):
    """Key-like rows: a few channels are much larger than the rest, as in trained models."""
    x = torch.randn(shape, generator=gen, device="cuda")
    channel = 1 + 5 * (torch.rand(shape[1], 1, shape[-1], generator=gen, device="cuda") < 0.03).float()
    return x.mul_(channel).to(dtype)


def _places(case, gen):
    """One position per sequence, spread evenly from the case's shortest to its longest, in any order."""
    span = case["longest"] - case["shortest"] + 1
    u = torch.rand(case["batch"], generator=gen, device="cuda", dtype=torch.float64)
    order = torch.randperm(case["batch"], generator=gen, device="cuda")
    return case["shortest"] + ((order + u) / case["batch"] * span).floor().long().clamp_(max=span - 1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = getattr(torch, case["dtype"])
    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        # a broad bulk, and per row a handful of tokens that the context suggests
        logits = torch.randn(rows, vocab, generator=gen, device="cuda") * 2.0
        hot = torch.randint(0, vocab, (rows, 24), generator=gen, device="cuda")
        logits.scatter_(1, hot, 8 + 4 * torch.rand(rows, 24, generator=gen, device="cuda"))
        if case["masked"]:                         # a grammar that allows a part of the vocabulary, in every other row
            allowed = torch.rand(rows, vocab, generator=gen, device="cuda") < 0.2
            allowed[::2] = True
            logits.masked_fill_(~allowed, -math.inf)
        uniform = torch.rand(rows, generator=gen, device="cuda")
        given = {k: torch.full((rows,), float(case[k]), device="cuda") for k in ("temperature", "top_p", "min_p")}
        given["top_k"] = torch.full((rows,), case["top_k"], dtype=torch.int32, device="cuda")
        if case["mixed"]:                          # requests with settings of their own; some switch a filter off
            r = torch.rand(4, rows, generator=gen, device="cuda")
            given["temperature"] = torch.where(r[0] < 0.15, 0.0, given["temperature"] * (0.5 + r[0]))
            given["top_k"] = torch.where(r[1] < 0.4, 0, 1 + (r[1] * max(case["top_k"], 50)).int()).int()
            given["top_p"] = torch.where(r[2] < 0.4, 1.0, r[2])
            given["min_p"] = torch.where(r[3] < 0.6, 0.0, 0.1 * r[3])
        return dict(case=case, logits=logits.to(dtype), uniform=uniform, **given)

    batch, heads, slots, dim = case["batch"], case["kv_heads"], case["slots"], case["dim"]
    state = dict(case=case)
    for name in ("k", "v"):
        codes = torch.empty(batch, heads, slots, dim, device="cuda",
                            dtype=torch.int8 if case["fmt"] == "int8" else torch.float8_e4m3fn)
        scales = torch.empty(batch, heads, slots, device="cuda")
        for b in range(batch):                     # one sequence at a time: the 64-bit copies stay small
            shape = (1, heads, slots, dim)
            x = _keys(gen, shape, dtype) if name == "k" else torch.randn(shape, generator=gen, device="cuda").to(dtype)
            c, s = _quantise(x, case["fmt"])
            codes[b], scales[b] = c[0], s[0]
        state[name + "_codes"], state[name + "_scales"] = codes, scales
    if case["op"] == "cache":
        tokens = case["tokens"]
        # projections give [batch, tokens, heads, dim]; the cache sees them transposed
        for name in ("k", "v"):
            x = _keys(gen, (batch, heads, tokens, dim), dtype)
            state[name] = x.transpose(1, 2).contiguous().transpose(1, 2)
        state["positions"] = _places(case, gen)
        # what is read back: the new tokens' slots (of a batch that moves together), or all slots that a sequence of
        # the batch may have filled
        if case["read"] == "new":
            state["positions"] = state["positions"][:1].expand(batch).contiguous()
            state["range"] = (int(state["positions"][0]), tokens)
        else:
            state["range"] = (0, case["longest"] + tokens)
        return state
    q = torch.randn(batch, case["queries"], heads * case["group"], dim, generator=gen, device="cuda") * 1.5
    state["q"] = q.to(dtype).transpose(1, 2)
    state["lengths"] = _places(case, gen)
    state["first"] = None
    if case["padded"]:
        u = torch.rand(batch, generator=gen, device="cuda")
        state["first"] = (u * u * state["lengths"] * 0.5).long()
    return state


# ---------------------------------------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if case["op"] == "sample":
        return _sample(state)
    cache = (state["k_codes"], state["k_scales"], state["v_codes"], state["v_scales"])
    if case["op"] == "cache":
        return _write_and_read(state, cache)
    return _attend(state, cache)


def _write_and_read(state, cache):
    case, (first, count) = state["case"], state["range"]
    if own:
        from dfloat11_b200 import ops
        ops.kv_append(state["k"], state["v"], *cache, state["positions"])
        return ops.kv_read(*cache, first, count, dtype=state["k"].dtype)
    outputs = []
    at = state["positions"][:, None] + torch.arange(case["tokens"], device="cuda")          # [batch, tokens]
    sequence = torch.arange(case["batch"], device="cuda")[:, None]
    for x, codes, scales in ((state["k"], cache[0], cache[1]), (state["v"], cache[2], cache[3])):
        new_codes, new_scales = _quantise(x, case["fmt"])
        # bytes are moved as integers: torch indexes no 8-bit floats
        codes.view(torch.int8).transpose(1, 2)[sequence, at] = new_codes.view(torch.int8).transpose(1, 2)
        scales.transpose(1, 2)[sequence, at] = new_scales.transpose(1, 2)
        window = slice(first, first + count)
        outputs.append((codes[:, :, window].float() * scales[:, :, window, None]).to(x.dtype))
    return tuple(outputs)


def _attend(state, cache):
    case, q = state["case"], state["q"]
    if own:
        from dfloat11_b200 import ops
        return ops.kv_attention(q, *cache, state["lengths"], first=state["first"], window=case["window"])
    k_codes, k_scales, v_codes, v_scales = cache
    batch, heads, group, queries, dim = (case[k] for k in ("batch", "kv_heads", "group", "queries", "dim"))
    slots = int(k_codes.shape[2])
    k = k_codes.float() * k_scales[..., None]
    v = v_codes.float() * v_scales[..., None]
    rows = q.float().reshape(batch, heads, group * queries, dim)
    scores = torch.matmul(rows, k.transpose(2, 3)) / math.sqrt(dim)
    slot = torch.arange(slots, device="cuda")
    place = state["lengths"][:, None] - queries + torch.arange(queries, device="cuda")       # [batch, queries]
    low = torch.zeros_like(place) if state["first"] is None else state["first"][:, None].expand_as(place)
    if case["window"]:
        low = torch.maximum(low, place - case["window"] + 1)
    seen = (slot >= low[..., None]) & (slot <= place[..., None])                             # [batch, queries, slots]
    seen = seen[:, None].expand(batch, group, queries, slots).reshape(batch, 1, group * queries, slots)
    scores = scores.masked_fill(~seen, -math.inf)
    peak = scores.amax(-1, keepdim=True)
    weights = torch.where(seen, torch.exp(scores - peak), 0.0)
    total = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights, v) / total
    out = torch.where(total > 0, out, 0.0)
    return out.view(batch, heads * group, queries, dim).transpose(1, 2).to(q.dtype).contiguous()


def _sample(state):
    if own:
        from dfloat11_b200 import ops
        return ops.sample(state["logits"], state["uniform"], temperature=state["temperature"], top_k=state["top_k"],
                          top_p=state["top_p"], min_p=state["min_p"])
    # 64 bits: with 10^5 tokens, sums in 32 decide some borders wrongly
    z = state["logits"].double()
    vocab = z.shape[1]
    z = torch.where(torch.isnan(z), -math.inf, z)
    t = state["temperature"].double()[:, None]
    z, index = torch.sort(z, dim=1, descending=True, stable=True)
    w = torch.exp((z - z[:, :1]) / torch.where(t > 0, t, 1.0))
    rank = torch.arange(vocab, device="cuda")
    k = state["top_k"][:, None]
    w = torch.where((k <= 0) | (rank < k), w, 0.0)
    running = torch.cumsum(w, 1)
    top_p = state["top_p"].double()[:, None]
    in_p = (top_p >= 1) | (running - w < top_p * running[:, -1:])
    keep = in_p & (w >= state["min_p"].double()[:, None])
    keep[:, 0] = True
    kept = torch.zeros_like(w).scatter_(1, index, torch.where(keep, w, 0.0))
    running = torch.cumsum(kept, 1)
    drawn = (running <= state["uniform"].double()[:, None] * running[:, -1:]).sum(1)
    return torch.where(t[:, 0] > 0, drawn, index[:, 0])


# ---------------------------------------------------------------------------------------------------- cost
def work(case):
    size = {"bfloat16": 2, "float16": 2, "float32": 4}[case["dtype"]]
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        # one scaling, one exponential (counted as one) and one sum per token
        return {"bytes": n * size + case["rows"] * (4 + 4 * 4 + 8), "flops": 3 * n}
    batch, heads, dim = case["batch"], case["kv_heads"], case["dim"]
    row = dim + 4                                                                 # codes and scale of a token
    if case["op"] == "cache":
        tokens = batch * heads * case["tokens"]
        span = case["tokens"] if case["read"] == "new" else case["longest"] + case["tokens"]
        old = batch * heads * (span - case["tokens"])                             # read back, but not written here
        total = 2 * (tokens * (dim * size + row) + old * row + (tokens + old) * dim * size)
        return {"bytes": total, "flops": 2 * dim * (4 * tokens + (tokens + old))}
    length = (case["shortest"] + case["longest"]) / 2
    if case["padded"]:
        length *= 5 / 6                            # a sixth of the slots on average lies before the first token
    if case["window"]:
        length = min(length, case["window"] + case["queries"] - 1)
    seen = batch * heads * length
    rows = case["group"] * case["queries"]
    return {"bytes": int(2 * seen * row + 2 * batch * heads * rows * dim * size), "flops": int(4 * seen * rows * dim)}


# ---------------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "sample":
        return _exact_sample(case, state)
    if case["op"] == "cache":
        return _exact_cache(case, state)
    return _exact_attend(case, state)


def _exact_sample(case, state):
    tokens = []
    for r in range(case["rows"]):
        z = torch.nan_to_num(state["logits"][r].to(torch.float64), nan=-math.inf, posinf=math.inf, neginf=-math.inf)
        best = float(z.max())
        t = float(state["temperature"][r])
        if t <= 0:
            tokens.append(int((z == best).nonzero()[0]))
            continue
        alive = (z > -math.inf).nonzero()[:, 0]                                   # ascending indices
        p = ((z[alive] - best) / t).exp_()
        order = torch.argsort(-z[alive], stable=True)
        k = int(state["top_k"][r])
        if k > 0:
            order = order[:k]
        limit = float(state["top_p"][r])
        if limit < 1:
            before = torch.cat([p.new_zeros(1), p[order].cumsum(0)])
            n = int(torch.searchsorted(before[:-1].contiguous(), limit * before[-1:], right=False))
            order = order[:max(n, 1)]
        order = order[p[order] >= min(float(state["min_p"][r]), 1.0)]
        chosen = order.sort().values
        mass = p[chosen].cumsum(0)
        place = int(torch.searchsorted(mass, float(state["uniform"][r]) * mass[-1:], right=True))
        tokens.append(int(alive[chosen[min(place, len(chosen) - 1)]]))
    return torch.tensor(tokens, device="cuda")


def _exact_cache(case, state):
    first, count = state["range"]
    results = []
    for name in ("k", "v"):
        stored = state[name + "_codes"][:, :, first:first + count].to(torch.float32).to(torch.float64)
        stored = stored * state[name + "_scales"][:, :, first:first + count].to(torch.float64).unsqueeze(-1)
        for b in range(case["batch"]):
            x = state[name][b].to(torch.float64)                                  # [heads, tokens, dim]
            largest, top = x.abs().max(dim=-1, keepdim=True).values, 127 if case["fmt"] == "int8" else 448
            y = torch.where(largest > 0, x * top / largest, torch.zeros_like(x))  # the product is exact: ties stay ties
            step = torch.ones_like(y)
            if case["fmt"] == "e4m3":                                             # 3 fraction bits, smallest exponent -6
                exponent = torch.frexp(y.abs()).exponent.clamp(min=-5) - 1
                step = torch.ldexp(step, exponent - 3)
            value = torch.round(y / step) * step * largest / top
            start = int(state["positions"][b]) - first
            stored[b, :, start:start + case["tokens"]] = value
        results.append(stored)
    return tuple(results)


def _exact_attend(case, state):
    heads, group, queries, dim = case["kv_heads"], case["group"], case["queries"], case["dim"]
    out = torch.zeros(case["batch"], queries, heads * group, dim, dtype=torch.float64, device="cuda")
    for b in range(case["batch"]):
        length = int(state["lengths"][b])
        begin = 0 if state["first"] is None else int(state["first"][b])
        for i in range(queries):
            here = length - queries + i
            low = max(begin, here - case["window"] + 1) if case["window"] else begin
            if here < low:
                continue
            for h in range(heads):
                k = state["k_codes"][b, h, low:here + 1].to(torch.float32).to(torch.float64)
                v = state["v_codes"][b, h, low:here + 1].to(torch.float32).to(torch.float64)
                q = state["q"][b, h * group:(h + 1) * group, i].to(torch.float64)
                s = (q @ k.T) * state["k_scales"][b, h, low:here + 1].to(torch.float64) / dim ** 0.5
                p = torch.softmax(s, dim=-1) * state["v_scales"][b, h, low:here + 1].to(torch.float64)
                out[b, i, h * group:(h + 1) * group] = p @ v
    return out
