"""The 8-bit key/value cache (ops.kv_append, ops.kv_read, ops.kv_attention) against its definition in 64 bits.

Codes and scales are compared bit for bit.  The bound for attention, per output with A = sum p|v| / sum p, is
  eps/2 |ref|            the result's rounding (eps/2: half a step of its type)
  + A 2^-11              weights rounded to fp16 before they meet the values
  + A 2 ds               a score off by ds moves its weight by a factor 1 + ds, and the denominator as much;
                         ds = (d + 8) 2^-22 S with S the largest scale * sum |q k| : d fp32 products summed one after
                         the other, each step rounded by at most 2^-22 of the running sum (truncating adders included)
  + A (n/16 + 64) 2^-22  the sums over n slots, 16 of which meet in one step, and the joins of parts
plus 2^-24 of the row's largest query entry per product for entries that fp16 holds as subnormals.
The int8 kernel multiplies code + 128 and takes 128 times the other operand's sum off again, so what its sums round
are steps of size |code| + 128: in the two terms with 2^-22, |k| and |v| are |k| + 128 k_scale and |v| + 128 v_scale.
(With one slot seen the result is the value itself and A = |v|; a code of 1 then carries 129 2^-22 = 2^-15 of itself,
which is beside the 2^-11 of the weight but not nothing.)
"""
import numpy as np
import pytest
import torch

from dfloat11_b200 import _lib, ops

DEV = "cuda:0"
gpu = pytest.mark.gpu
FORMATS = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
TOP = {"int8": 127.0, "e4m3": 448.0}
DTYPES = [torch.bfloat16, torch.float16]


def reference_rows(x, fmt):
    """(code values, scales) of the rows of a CPU tensor, the code from the quotient in 64 bits."""
    x = x.double()
    a = x.abs().amax(-1, keepdim=True)
    fine = torch.isfinite(a) & (a > 0)
    q = torch.where(fine, x * TOP[fmt] / torch.where(fine, a, torch.ones_like(a)), torch.zeros_like(x))
    if fmt == "int8":
        code = torch.round(q)
    else:
        step = torch.exp2(torch.floor(torch.log2(q.abs().clamp(min=2.0 ** -6))) - 3)
        code = torch.round(q / step) * step
    scale = torch.where(torch.isfinite(a), a.float() / TOP[fmt], torch.full_like(a, float("nan")).float())
    return code, scale.squeeze(-1)


def new_cache(batch, heads, slots, dim, fmt, fill=None):
    """Four cache tensors; `fill` is the byte that codes (and the bytes of the scales) are filled with."""
    codes = [torch.zeros(batch, heads, slots, dim, dtype=torch.uint8, device=DEV) for _ in range(2)]
    scales = [torch.zeros(batch, heads, slots, dtype=torch.float32, device=DEV) for _ in range(2)]
    if fill is not None:
        for c in codes:
            c.fill_(fill)
        for s in scales:
            s.view(torch.uint8).fill_(fill)
    k, v = (c.view(FORMATS[fmt]) for c in codes)
    return k, scales[0], v, scales[1]


def random_rows(shape, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * torch.exp2(torch.randint(-6, 7, (*shape[:-1], 1), generator=g).float())
    return x.to(dtype)


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,tokens,layout", [(16, 1, "plain"), (64, 3, "projection"), (80, 7, "plain"), (96, 5, "odd"),
                                               (128, 1, "projection"), (128, 33, "projection"), (192, 2, "odd"),
                                               (256, 9, "projection")])
def test_append_and_read_back(fmt, dtype, dim, tokens, layout):
    batch, heads, slots = 3, 2, 41
    k, v = (random_rows((batch, heads, tokens, dim), dtype, s) for s in (1, 2))
    if layout == "projection":                      # [batch, tokens, heads, dim] seen transposed
        kd, vd = (x.to(DEV).transpose(1, 2).contiguous().transpose(1, 2) for x in (k, v))
    elif layout == "odd":                           # rows that start at any element
        kd, vd = (torch.zeros(batch, heads, tokens, dim + 3, dtype=dtype, device=DEV)[..., 1:1 + dim] for _ in range(2))
        kd.copy_(k), vd.copy_(v)
    else:
        kd, vd = k.to(DEV), v.to(DEV)
    cache = new_cache(batch, heads, slots, dim, fmt, fill=0x5A)
    before = [t.clone() for t in cache]
    positions = torch.tensor([0, slots - tokens, 2], device=DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    ops.kv_append(kd, vd, *cache, positions, status=status)
    assert status.item() == 0
    for x, codes, scales, codes0, scales0 in ((k, cache[0], cache[1], before[0], before[1]),
                                              (v, cache[2], cache[3], before[2], before[3])):
        want, want_scale = reference_rows(x, fmt)
        written = torch.zeros(batch, slots, dtype=torch.bool)
        for b, p in enumerate(positions.tolist()):
            got = codes[b, :, p:p + tokens].float().cpu().double()
            assert torch.equal(got, want[b])
            assert torch.equal(scales[b, :, p:p + tokens].cpu(), want_scale[b])
            written[b, p:p + tokens] = True
        untouched = ~written[:, None].expand(batch, heads, slots).to(DEV)
        assert torch.equal(codes.view(torch.uint8)[untouched], codes0.view(torch.uint8)[untouched])
        assert torch.equal(scales.view(torch.int32)[untouched], scales0.view(torch.int32)[untouched])
    first = 2
    for out_dtype in DTYPES:
        for got, codes, scales in zip(ops.kv_read(*cache, first, tokens, dtype=out_dtype), cache[::2], cache[1::2]):
            want = (codes[:, :, first:first + tokens].float() * scales[:, :, first:first + tokens, None]).to(out_dtype)
            assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want)) and got.is_contiguous()


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_append_rows_that_are_special(fmt, dtype):
    """Ties, zeros, the type's extremes and subnormals, infinities and NaN."""
    dim, top, info = 32, TOP[fmt], torch.finfo(dtype)
    rows = torch.zeros(9, dim, dtype=torch.float64)
    rows[1] = torch.arange(dim) - 15.5                                   # int8: halves exactly between codes below
    rows[1, 0] = top
    rows[2] = torch.linspace(-1, 1, dim)
    rows[2, 3], rows[2, 4] = info.max, info.max / 2
    rows[3] = info.smallest_normal * torch.linspace(-1, 1, dim)          # subnormals of the type
    rows[4, 5] = float("inf")
    rows[5, 31] = float("nan")
    rows[6, 0] = -info.max
    rows[7, 7] = info.smallest_normal * info.eps                         # the smallest positive number
    rows[8] = torch.exp2(-torch.arange(dim).double())                    # e4m3: down to its subnormals and below
    x = rows.to(dtype).view(1, 1, 9, dim)
    cache = new_cache(1, 1, 16, dim, fmt, fill=0x11)
    ops.kv_append(x.to(DEV), x.to(DEV), *cache, torch.tensor([4], device=DEV))
    want, scale = reference_rows(x, fmt)
    for codes, scales in (cache[:2], cache[2:]):
        assert torch.equal(codes[:, :, 4:13].float().cpu().double(), want)
        assert torch.equal(torch.nan_to_num(scales[:, :, 4:13].cpu(), nan=-1), torch.nan_to_num(scale, nan=-1))
    k, _ = ops.kv_read(*cache, 4, 9, dtype=dtype)
    nan = torch.isnan(k[0, 0]).cpu()
    assert nan[4].all() and nan[5].all() and int(nan.sum()) == 2 * dim
    assert torch.equal(k[0, 0, 0].cpu(), torch.zeros(dim, dtype=dtype))


@gpu
@pytest.mark.parametrize("start,tokens", [(-2, 4), (6, 4), (8, 1), (-1, 1), (2 ** 62, 2), (-2 ** 63, 3), (2 ** 63 - 1, 2)])
def test_append_leaves_out_slots_that_are_not_there(start, tokens):
    dim, slots = 64, 8
    x = random_rows((2, 1, tokens, dim), torch.bfloat16, 3).to(DEV)
    cache = new_cache(2, 1, slots, dim, "int8", fill=0x33)
    before = [t.clone() for t in cache]
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    ops.kv_append(x, x, *cache, torch.tensor([start, 3], device=DEV), status=status)
    assert status.item() == _lib.STATUS_BAD_POSITIONS
    fits = [t for t in range(tokens) if 0 <= start + t < slots]
    for now, old in zip(cache, before):
        now, old = (t.view(torch.uint8).view(2, slots, -1).cpu() for t in (now, old))
        other = [s for s in range(slots) if s - start not in fits]
        assert torch.equal(now[0, other], old[0, other])
        assert torch.equal(now[1, 3 + tokens:], old[1, 3 + tokens:]) and not torch.equal(now[1, 3], old[1, 3])
    want, _ = reference_rows(x.cpu(), "int8")
    for t in fits:
        assert torch.equal(cache[0][0, 0, start + t].cpu().double(), want[0, 0, t])


# ------------------------------------------------------------------ attention
def reference_attention(q, cache, lengths, first, scale, window):
    """(result, bound without the result's rounding), both [batch, queries, heads, dim] in 64 bits on the CPU."""
    kc, ks, vc, vs = (t.float().cpu().double() for t in cache)
    q = q.cpu().double()
    batch, heads, queries, dim = q.shape
    kv_heads, slots = kc.shape[1], kc.shape[2]
    out = torch.zeros(batch, queries, heads, dim, dtype=torch.float64)
    bound = torch.zeros_like(out)
    for b in range(batch):
        for i in range(queries):
            place = lengths[b] - queries + i
            low = max(first[b], 0)
            if window:
                low = max(low, place - window + 1)
            high = min(place, slots - 1)
            if high < low:
                continue
            for h in range(heads):
                g = h // (heads // kv_heads)
                k = kc[b, g, low:high + 1] * ks[b, g, low:high + 1, None]
                v = vc[b, g, low:high + 1] * vs[b, g, low:high + 1, None]
                p = torch.softmax(k @ q[b, h, i] * scale, 0)
                out[b, i, h] = p @ v
                magnitude, shift = p @ v.abs(), 128 * (cache[0].dtype == torch.int8)
                stepped = magnitude + shift * (p @ vs[b, g, low:high + 1])
                score = float(((k.abs() + shift * ks[b, g, low:high + 1, None]) @ q[b, h, i].abs()).max()) * abs(scale)
                small = dim * 2.0 ** -24 * float(q[b, h, i].abs().max() * k.abs().max()) * abs(scale)
                ds = (dim + 8) * 2.0 ** -22 * score + small
                bound[b, i, h] = magnitude * (2.0 ** -11 + 2 * ds) + stepped * ((high - low + 1) / 16 + 64) * 2.0 ** -22
    return out, bound


def check_attention(q, cache, lengths, first=None, scale=None, window=0, **kw):
    batch = q.shape[0]
    as_list = lambda t: [0] * batch if t is None else (t.tolist() * batch if t.numel() == 1 else t.tolist())  # noqa: E731
    got = ops.kv_attention(q, *cache, lengths, first=first, scale=scale, window=window, **kw)
    want, bound = reference_attention(q, cache, as_list(lengths), as_list(first),
                                      q.shape[3] ** -0.5 if scale is None else scale, window)
    assert got.shape == want.shape and got.dtype == q.dtype and got.is_contiguous()
    bound = bound + want.abs() * (torch.finfo(q.dtype).eps / 2) + 2.0 ** -25     # fp16's subnormal results
    error = (got.cpu().double() - want).abs()
    worst = float((error - bound).max())
    assert worst <= 0, f"{worst} above the bound, at {int((error > bound).sum())} of {error.numel()}"
    return got


def filled_cache(batch, heads, slots, dim, fmt, seed, dtype=torch.bfloat16):
    cache = new_cache(batch, heads, slots, dim, fmt)
    g = torch.Generator().manual_seed(seed)
    k = torch.randn(batch, heads, slots, dim, generator=g) * (1 + 5 * (torch.rand(heads, 1, dim, generator=g) < 0.05))
    v = torch.randn(batch, heads, slots, dim, generator=g) * torch.exp2(torch.randint(-3, 4, (batch, heads, slots, 1), generator=g))
    ops.kv_append(k.to(dtype).to(DEV), v.to(dtype).to(DEV), *cache, torch.zeros(1, dtype=torch.int64, device=DEV))
    return cache


def query(batch, heads, queries, dim, dtype, seed, size=1.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(batch, queries, heads, dim, generator=g) * size).to(dtype)
    return x.to(DEV).transpose(1, 2)


def poison(cache, lengths, first=None):
    """Slots that no query may see: codes of the highest byte values, scales that are NaN."""
    kc, ks, vc, vs = cache
    for b, n in enumerate(lengths):
        ranges = [slice(max(n, 0), None)] + ([slice(0, max(first[b], 0))] if first else [])
        for r in ranges:
            for codes, scales in ((kc, ks), (vc, vs)):
                codes[b].view(torch.uint8)[:, r] = 0x7F
                scales[b][:, r] = float("nan")


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,group", [(16, 1), (64, 4), (80, 3), (96, 8), (128, 4), (128, 16), (192, 5), (256, 2), (256, 9)])
def test_attention_single_token(fmt, dtype, dim, group):
    lengths = [1, 2, 15, 16, 17, 0, 63, 64, 65, 130]
    cache = filled_cache(len(lengths), 2, 130, dim, fmt, seed=dim + group, dtype=dtype)
    poison(cache, lengths)
    got = check_attention(query(len(lengths), 2 * group, 1, dim, dtype, 7), cache, torch.tensor(lengths, device=DEV))
    assert not got[5].any()                                             # nothing to see: zeros


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("queries,group,dim", [(2, 4, 128), (3, 1, 64), (5, 2, 256), (8, 7, 80), (17, 4, 128), (40, 1, 128)])
def test_attention_several_tokens(fmt, queries, group, dim):
    lengths = [queries, 1, 0, 33, 100, 64]                              # shorter than the queries: the first see nothing
    cache = filled_cache(len(lengths), 2, 100, dim, fmt, seed=queries)
    poison(cache, lengths)
    q = query(len(lengths), 2 * group, queries, dim, torch.bfloat16, 8)
    got = check_attention(q, cache, torch.tensor(lengths, device=DEV))
    assert not got[2].any() and not got[1, :queries - 1].any()


@gpu
@pytest.mark.parametrize("window", [0, 1, 2, 16, 33, 500, 2 ** 31 - 1])
@pytest.mark.parametrize("queries", [1, 4])
def test_attention_window_and_padding(window, queries):
    lengths, first = [200, 200, 77, 50, 120, 9], [0, 150, 77, 90, -5, 4]
    cache = filled_cache(len(lengths), 1, 200, 128, "int8", seed=5)
    if queries == 1 and not window:
        poison(cache, lengths, first)
    q = query(len(lengths), 4, queries, 128, torch.bfloat16, 9)
    check_attention(q, cache, torch.tensor(lengths, device=DEV), first=torch.tensor(first, device=DEV), window=window)


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("batch,heads,slots,queries", [(1, 1, 20011, 1), (300, 2, 40, 1), (2, 4, 8000, 2), (1, 2, 9000, 3), (7, 3, 2500, 1), (40, 4, 700, 1), (3, 8, 5000, 1)])
def test_attention_long(fmt, batch, heads, slots, queries):
    cache = filled_cache(batch, heads, slots, 64, fmt, seed=11)
    lengths = torch.tensor([slots - (b * 977) % slots for b in range(batch)], device=DEV)
    check_attention(query(batch, heads * 4, queries, 64, torch.float16, 10, size=3.0), cache, lengths)


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dim,group,queries,kv_heads,slots,lengths", [
    (128, 4, 1, 4, 13000, [0, 8999, 1, 0, 0, 17, 300, 13000, 0]),       # one sequence among CTAs, many in one CTA
    (128, 4, 1, 4, 40000, [39999]),
    (128, 4, 1, 8, 13000, [0] * 3),                                     # nothing at all
    (64, 2, 3, 4, 25000, [5, 2500, 0, 2, 4000, 33, 25000]),
    (256, 5, 4, 2, 9000, [700, 3, 0, 1111]),                            # three row groups
    (80, 16, 2, 2, 13000, [64, 1000, 0, 2]),
    (128, 1, 1, 2, 3300, [(37 * b) % 600 for b in range(75)]),           # more sequences than a warp has lanes
    (96, 3, 1, 16, 1700, [300 - b % 2 for b in range(70)]),
])
@pytest.mark.parametrize("windowed", [False, True])
def test_attention_shared_out(fmt, dim, group, queries, kv_heads, slots, lengths, windowed):
    """Caches so large that the tiles of all sequences are shared out evenly; lengths of any kind in them."""
    batch, window = len(lengths), slots - 100 if windowed else 0
    shape = (batch, kv_heads, slots, dim)
    need = _lib.lib.df11_kv_attention_workspace_bytes(batch, kv_heads * group, kv_heads, queries, dim, slots, window)
    assert need > 0, "this case is meant to take the shared-out kernel"
    cache = new_cache(*shape, fmt)
    g = torch.Generator(device=DEV).manual_seed(40)
    for c in cache[::2]:
        for b in range(batch):
            c[b].copy_((torch.randn(shape[1:], generator=g, device=DEV) * 40).clamp(-127, 127).to(c.dtype))
    for s in cache[1::2]:
        s.copy_(torch.rand(s.shape, generator=g, device=DEV) * 0.02)
    poison(cache, lengths)
    at = torch.tensor(lengths, device=DEV)
    q = query(batch, kv_heads * group, queries, dim, torch.bfloat16, 41)
    got = check_attention(q, cache, at, window=window)
    assert torch.equal(got, ops.kv_attention(q, *cache, at, window=window))
    first = torch.tensor([(b * 29) % 50 for b in range(batch)], device=DEV)
    check_attention(q, cache, at, first=first, window=window)


@gpu
@pytest.mark.parametrize("size", [0.0, 1e-6, 30.0, 1e4])
@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_flat_and_peaked(size, dtype):
    """Scores that are all alike, and scores so far apart that one slot takes all."""
    cache = filled_cache(2, 2, 333, 128, "e4m3", seed=12)
    check_attention(query(2, 8, 1, 128, dtype, 13, size=size), cache, torch.tensor([333, 300], device=DEV))


@gpu
def test_attention_flat_over_values_of_very_different_size():
    """Weights times value scales over 40 powers of two: none of the small ones may be lost against its own kind."""
    cache = filled_cache(1, 1, 4000, 128, "int8", seed=14)
    cache[3][0, 0] *= torch.exp2(torch.linspace(-20, 20, 4000, device=DEV))
    q = query(1, 4, 1, 128, torch.bfloat16, 15)
    for n in (4000, 1000, 16):
        check_attention(q, cache, torch.tensor([n], device=DEV))


@gpu
def test_attention_values_that_start_with_zeros():
    """A sequence whose first values are zeros and whose others are tiny or huge; and one that is all zeros."""
    cache = filled_cache(3, 1, 500, 64, "e4m3", seed=30)
    for b, size in ((0, 2.0 ** -40), (1, 2.0 ** 40), (2, 0.0)):
        cache[3][b, :, :100] = 0
        cache[3][b, :, 100:] *= size
    q = query(3, 4, 1, 64, torch.bfloat16, 31)
    lengths = torch.tensor([500, 480, 300], device=DEV)
    got = ops.kv_attention(q, *cache, lengths).double().cpu()
    want, bound = reference_attention(q, cache, lengths.tolist(), [0] * 3, 0.125, 0)
    assert ((got - want).abs() <= bound + want.abs() * 2.0 ** -8).all() and not got[2].any() and got[0].any()


@gpu
def test_attention_lengths_beyond_the_cache_and_shared_ones():
    cache = filled_cache(3, 2, 96, 128, "int8", seed=16)
    q = query(3, 8, 1, 128, torch.bfloat16, 17)
    one = torch.tensor([64], device=DEV)
    got = check_attention(q, cache, one, first=torch.tensor([3], device=DEV))
    many = ops.kv_attention(q, *cache, one.expand(3).contiguous(), first=torch.tensor([3, 3, 3], device=DEV))
    assert torch.equal(got, many)
    check_attention(q, cache, torch.tensor([97, 120, 10 ** 6], device=DEV))
    check_attention(q, cache, torch.tensor([-1, -2 ** 63, 50], device=DEV))
    for first in (2 ** 62, 2 ** 63 - 1):
        for length in (one, torch.tensor([-5], device=DEV), torch.tensor([2 ** 63 - 1], device=DEV)):
            assert not ops.kv_attention(q, *cache, length, first=torch.tensor([first], device=DEV)).any()
    check_attention(q, cache, one, first=torch.tensor([-2 ** 63], device=DEV))


@gpu
def test_attention_query_layouts_and_scale():
    cache = filled_cache(2, 2, 50, 128, "e4m3", seed=18)
    lengths = torch.tensor([50, 31], device=DEV)
    q = query(2, 8, 2, 128, torch.bfloat16, 19)
    want = check_attention(q, cache, lengths, scale=0.3)
    odd = torch.zeros(2, 8, 2, 131, dtype=torch.bfloat16, device=DEV)[..., 2:130]
    odd.copy_(q)
    same = q[:, :1].expand(2, 8, 2, 128)                                # one query for all heads: stride 0
    assert torch.equal(ops.kv_attention(q.contiguous(), *cache, lengths, scale=0.3), want)
    assert torch.equal(ops.kv_attention(odd, *cache, lengths, scale=0.3), want)
    check_attention(same, cache, lengths)
    check_attention(q, cache, lengths, scale=0.0)
    check_attention(q, cache, lengths, scale=-0.05)


@gpu
def test_attention_a_nan_row_that_is_seen_spoils_its_sequence_only():
    cache = filled_cache(2, 1, 40, 64, "int8", seed=20)
    cache[1][0, 0, 7] = float("nan")
    q = query(2, 4, 1, 64, torch.bfloat16, 21)
    got = ops.kv_attention(q, *cache, torch.tensor([40, 40], device=DEV))
    assert torch.isnan(got[0]).all() and torch.isfinite(got[1]).all()
    got = ops.kv_attention(q, *cache, torch.tensor([7, 40], device=DEV))
    assert torch.isfinite(got).all()


@gpu
def test_step_in_a_graph_beside_another_stream():
    """Append, attention and the position's advance captured once and replayed; a second sequence of calls runs on
    another stream at the same time.  Both give what the calls one by one give."""
    batch, heads, group, dim, slots, steps = 2, 2, 4, 128, 900, 12
    start = 700
    rows = [[random_rows((batch, heads, 1, dim), torch.bfloat16, 100 * s + i).to(DEV) for i in range(steps)] for s in (1, 2)]
    qs = [query(batch, heads * group, 1, dim, torch.bfloat16, 300 + i) for i in range(steps)]

    def fresh():
        return filled_cache(batch, heads, slots, dim, "int8", seed=22)

    cache, want = fresh(), []
    for i in range(steps):
        ops.kv_append(rows[0][i], rows[1][i], *cache, torch.tensor([start + i], device=DEV))
        want.append(ops.kv_attention(qs[i], *cache, torch.tensor([start + i + 1], device=DEV)))
    final = [t.clone() for t in cache]

    cache, other = fresh(), fresh()
    pos = torch.tensor([start], device=DEV)
    k, v, q = (torch.zeros_like(t) for t in (rows[0][0], rows[1][0], qs[0]))
    out = torch.empty_like(want[0])

    def step():
        ops.kv_append(k, v, *cache, pos)
        pos.add_(1)
        ops.kv_attention(q, *cache, pos, out=out)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    pos.fill_(start)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    got, beside = [], []
    for i in range(steps):
        k.copy_(rows[0][i]), v.copy_(rows[1][i]), q.copy_(qs[i])
        graph.replay()
        got.append(out.clone())
        with torch.cuda.stream(side):
            ops.kv_append(rows[0][i], rows[1][i], *other, torch.tensor([start + i], device=DEV))
            beside.append(ops.kv_attention(qs[i], *other, torch.tensor([start + i + 1], device=DEV)))
    torch.cuda.synchronize()
    for i in range(steps):
        assert torch.equal(got[i], want[i]) and torch.equal(beside[i], want[i])
    for a, b, c in zip(cache, other, final):
        assert torch.equal(a.view(torch.uint8), c.view(torch.uint8)) and torch.equal(b.view(torch.uint8), c.view(torch.uint8))


@gpu
def test_offsets_beyond_32_bits():
    """A cache of more than 2^32 codes: its last slots are written, read and attended to like any others."""
    slots, dim, n = (1 << 26) + 40, 64, 40
    cache = new_cache(1, 1, slots, dim, "int8")
    x, y = (random_rows((1, 1, n, dim), torch.bfloat16, s) for s in (50, 51))
    ops.kv_append(x.to(DEV), y.to(DEV), *cache, torch.tensor([slots - n], device=DEV))
    for got, rows in zip(ops.kv_read(*cache, slots - n, n), (x, y)):
        want, scale = reference_rows(rows, "int8")
        assert torch.equal(got.cpu(), (want.float() * scale[..., None]).to(torch.bfloat16))
    assert not cache[0][:, :, :1000].any() and not cache[1][:, :, :slots - n].any()
    tail = tuple(t[:, :, slots - n:].clone() for t in cache)
    q = query(1, 4, 1, dim, torch.bfloat16, 52)
    want, bound = reference_attention(q, tail, [n], [0], dim ** -0.5, 0)
    for window, first in ((0, slots - n), (n, 0)):
        got = ops.kv_attention(q, *cache, torch.tensor([slots], device=DEV), first=torch.tensor([first], device=DEV), window=window)
        assert ((got.cpu().double() - want).abs() <= bound + want.abs() * 2.0 ** -8).all()
    del cache, tail
    torch.cuda.empty_cache()


@gpu
def test_nothing_to_do():
    cache = filled_cache(2, 1, 8, 64, "int8", seed=23)
    none = torch.empty(2, 1, 0, 64, dtype=torch.bfloat16, device=DEV)
    pos = torch.zeros(1, dtype=torch.int64, device=DEV)
    before = [t.clone() for t in cache]
    ops.kv_append(none, none, *cache, pos)
    assert all(torch.equal(a, b) for a, b in zip(cache, before))
    k, v = ops.kv_read(*cache, 8, 0)
    assert k.shape == v.shape == (2, 1, 0, 64)
    assert ops.kv_attention(torch.empty(2, 4, 0, 64, dtype=torch.bfloat16, device=DEV), *cache, pos).shape == (2, 0, 4, 64)


@gpu
def test_refusals_on_the_gpu():
    cache = filled_cache(2, 2, 8, 64, "int8", seed=24)
    x = random_rows((2, 2, 1, 64), torch.bfloat16, 25).to(DEV)
    q = query(2, 8, 1, 64, torch.bfloat16, 26)
    pos = torch.zeros(1, dtype=torch.int64, device=DEV)
    e4m3 = new_cache(2, 2, 8, 64, "e4m3")
    bad_append = [(x.float(), x.float(), *cache, pos), (x, x.half(), *cache, pos), (x[:1], x[:1], *cache, pos),
                  (x, x.transpose(2, 3), *cache, pos), (x, x, *cache, pos.int()), (x, x, *cache, pos.expand(3)),
                  (x, x, *cache, torch.zeros(3, dtype=torch.int64, device=DEV)), (x.cpu(), x, *cache, pos),
                  (x, x, *cache, pos.cpu()), (x, x, cache[0], cache[1], e4m3[2], cache[3], pos),
                  (x, x, cache[0].transpose(1, 2), cache[1], cache[2].transpose(1, 2), cache[3], pos),
                  (x, x, cache[0], cache[1].double(), cache[2], cache[3], pos),
                  (x.repeat(1, 1, 1, 2)[..., ::2], x, *cache, pos), (x.clone().requires_grad_(), x, *cache, pos)]
    for args in bad_append:
        with pytest.raises(RuntimeError):
            ops.kv_append(*args)
    for dim in (8, 24, 272):                                            # head sizes the kernels do not have
        c, y = new_cache(1, 1, 4, dim, "int8"), torch.zeros(1, 1, 1, dim, dtype=torch.bfloat16, device=DEV)
        for call in (lambda: ops.kv_append(y, y, *c, pos), lambda: ops.kv_attention(y, *c, pos), lambda: ops.kv_read(*c, 0, 1)):
            with pytest.raises(_lib.DF11Error, match="head_dim"):
                call()
    for args in ((-1, 2), (7, 2), (0, 9)):
        with pytest.raises(RuntimeError):
            ops.kv_read(*cache, *args)
    with pytest.raises(RuntimeError):
        ops.kv_read(*cache, 0, 2, dtype=torch.float32)
    with pytest.raises(RuntimeError):
        ops.kv_read(*cache, 0, 2, out=(x, x))
    for bad in (dict(window=-1), dict(out=torch.empty_like(q)), dict(first=pos.int()), dict(lengths=pos.int()), dict(q=q[:, :3]),
                dict(q=q.float()), dict(q=q[..., :32])):
        args = dict(q=q, lengths=pos, **{})
        args.update(bad)
        with pytest.raises(RuntimeError):
            ops.kv_attention(args.pop("q"), *cache, args.pop("lengths"), **args)


# ------------------------------------------------------------------ without a GPU
def test_refusals_without_a_gpu():
    x = torch.zeros(1, 1, 1, 64, dtype=torch.bfloat16)
    cache = (torch.zeros(1, 1, 4, 64, dtype=torch.int8), torch.zeros(1, 1, 4), torch.zeros(1, 1, 4, 64, dtype=torch.int8),
             torch.zeros(1, 1, 4))
    pos = torch.zeros(1, dtype=torch.int64)
    for call in (lambda: ops.kv_append(x, x, *cache, pos), lambda: ops.kv_read(*cache, 0, 1), lambda: ops.kv_attention(x, *cache, pos)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_argument_errors_of_the_c_entry_points():
    buf = np.zeros(4096 + 16, np.uint8)
    p = (buf.ctypes.data + 15) // 16 * 16
    lib = _lib.lib

    def append(**kw):
        a = dict(k=p, v=p, kc=p, ks=p, vc=p, vs=p, pos=p, n_pos=1, batch=1, heads=1, tokens=1, dim=64, slots=4, t=0, f=0)
        a.update(kw)
        return lib.df11_kv_append(a["k"], a["v"], 64, 64, 64, 64, 64, 64, a["kc"], a["ks"], a["vc"], a["vs"], a["pos"],
                                  a["n_pos"], a["batch"], a["heads"], a["tokens"], a["dim"], a["slots"], a["t"], a["f"], None, 0, None)

    def read(**kw):
        a = dict(kc=p, ko=p, batch=1, dim=64, slots=4, first=0, n=1, t=0, f=0)
        a.update(kw)
        return lib.df11_kv_read(a["kc"], p, p, p, a["ko"], p, a["batch"], 1, a["slots"], a["dim"], a["first"], a["n"], a["t"], a["f"], 0, None)

    def attention(**kw):
        a = dict(q=p, kc=p, lengths=p, n_len=1, first=None, n_first=0, out=p, batch=1, heads=2, kv=1, queries=1, dim=64, slots=4,
                 window=0, t=0, f=0, ws=p, ws_bytes=1 << 40)
        a.update(kw)
        return lib.df11_kv_attention(a["q"], 64, 64, 64, a["kc"], p, p, p, a["lengths"], a["n_len"], a["first"], a["n_first"],
                                     a["out"], a["ws"], a["ws_bytes"], a["batch"], a["heads"], a["kv"], a["queries"], a["dim"],
                                     a["slots"], a["window"], 0.1, a["t"], a["f"], 0, None)

    bad = _lib.DF11_ERR_BADARG
    for kw in (dict(k=None), dict(kc=None), dict(pos=None), dict(kc=p + 8), dict(ks=p + 2), dict(k=p + 1), dict(pos=p + 4),
               dict(n_pos=2), dict(batch=-1), dict(heads=0), dict(tokens=-1), dict(dim=72), dict(dim=272), dict(dim=0),
               dict(slots=0), dict(t=2), dict(f=2), dict(batch=2 ** 31), dict(tokens=2 ** 33)):
        assert append(**kw) == bad, kw
        assert lib.df11_last_error()
    for kw in (dict(kc=None), dict(ko=None), dict(ko=p + 8), dict(first=-1), dict(n=-1), dict(first=4, n=1), dict(n=5),
               dict(first=2 ** 62, n=2 ** 62), dict(t=2), dict(dim=8)):
        assert read(**kw) == bad, kw
    for kw in (dict(q=None), dict(lengths=None), dict(out=None), dict(out=p + 8), dict(q=p + 1), dict(lengths=p + 4), dict(n_len=2),
               dict(first=p, n_first=2), dict(heads=3, kv=2), dict(heads=0), dict(queries=-1), dict(window=-1), dict(dim=40),
               dict(t=2), dict(f=-1), dict(queries=2 ** 31)):
        assert attention(**kw) == bad, kw
    assert append(tokens=0) == append(batch=0, n_pos=0) == read(n=0) == attention(queries=0) == _lib.DF11_OK
