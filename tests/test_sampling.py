"""ops.sample against its definition in 64 bits.  Tokens are compared exactly: there is no tolerance."""
import numpy as np
import pytest
import torch

from dfloat11_b200 import _lib, ops

DEV = "cuda:0"
gpu = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def reference_row(z, u, temperature, top_k, top_p, min_p):
    """One row (numpy float64); settings are the numbers the kernel gets (fp32 values where they came as tensors)."""
    z = np.where(np.isnan(z), -np.inf, z)
    best = z.max()
    if best == -np.inf:
        return 0
    if not temperature > 0:
        return int(np.argmax(z))
    alive = np.flatnonzero(z > -np.inf)
    with np.errstate(invalid="ignore"):
        d = np.where(z[alive] == best, 0.0, z[alive] - best)
    w = np.where(d == -np.inf, 0.0, np.exp(np.where(d == -np.inf, 0.0, d) / temperature))
    order = np.argsort(-z[alive], kind="stable")
    if top_k > 0:
        order = order[:top_k]
    if top_p < 1:
        mass = np.cumsum(w[order])
        before = np.concatenate([[0.0], mass[:-1]])
        order = order[:max(1, int((before < top_p * mass[-1]).sum()))]
    order = order[w[order] >= min(min_p, 1.0)]
    kept = np.sort(order)
    mass = np.cumsum(w[kept])
    return int(alive[kept[min(int((mass <= u * mass[-1]).sum()), len(kept) - 1)]])


def reference(logits, uniform, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    z = logits.double().cpu().numpy()
    per_row = [x.double().cpu().numpy() if isinstance(x, torch.Tensor) else np.full(len(z), float(x))
               for x in (uniform, temperature, top_k, top_p, min_p)]
    return torch.tensor([reference_row(z[r], per_row[0][r], per_row[1][r], int(per_row[2][r]), per_row[3][r], per_row[4][r])
                         for r in range(len(z))])


def check(logits, uniform, **settings):
    got = ops.sample(logits, uniform, **settings)
    assert got.dtype == torch.int64 and got.shape == (logits.shape[0],)
    want = reference(logits, uniform, **settings)
    assert torch.equal(got.cpu(), want), (got.cpu() != want).nonzero().flatten().tolist()
    return got


def rows_of(rows, vocab, dtype, seed, spread=2.5, peaks=5):
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(rows, vocab, generator=g) * spread
    z.scatter_(1, torch.randint(0, vocab, (rows, peaks), generator=g), 9 + 3 * torch.rand(rows, peaks, generator=g))
    return z.to(dtype).to(DEV), torch.rand(rows, generator=g).to(DEV)


SETTINGS = {
    "plain": {}, "cold": dict(temperature=0.3), "hot": dict(temperature=5.0), "greedy": dict(temperature=0.0),
    "top_1": dict(top_k=1), "top_5": dict(top_k=5), "top_40": dict(top_k=40, temperature=0.8), "top_700": dict(top_k=700),
    "top_4000": dict(top_k=4000, temperature=3.0), "top_all": dict(top_k=2 ** 31 - 1), "p_small": dict(top_p=0.01),
    "p_half": dict(top_p=0.5), "p_most": dict(top_p=0.95, temperature=1.3), "p_almost": dict(top_p=0.99999, temperature=2.0),
    "min_p": dict(min_p=0.05), "min_p_1": dict(min_p=1.0), "min_p_tiny": dict(min_p=1e-6, temperature=2.0),
    "all": dict(temperature=0.7, top_k=50, top_p=0.9, min_p=0.02), "all_wide": dict(temperature=4.0, top_k=900, top_p=0.97, min_p=1e-3),
}


@gpu
@pytest.mark.parametrize("name", SETTINGS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab", [(5, 1), (5, 2), (9, 33), (17, 1000), (6, 5003), (3, 32001), (2, 151936)])
def test_settings(name, dtype, rows, vocab):
    logits, uniform = rows_of(rows, vocab, dtype, seed=vocab + rows, peaks=min(5, vocab))
    check(logits, uniform, **SETTINGS[name])


@gpu
@pytest.mark.parametrize("rows", [1, 2, 5, 19, 40, 80, 150, 300])
def test_row_counts(rows):
    """Every way the kernel spreads rows over the GPU, with settings that differ row by row."""
    vocab = 20000
    logits, uniform = rows_of(rows, vocab, torch.bfloat16, seed=rows)
    g = torch.Generator().manual_seed(rows)
    r = torch.rand(4, rows, generator=g)
    check(logits, uniform, temperature=torch.where(r[0] < 0.2, torch.zeros(rows), r[0] * 2).to(DEV),
          top_k=torch.where(r[1] < 0.3, 0.0, r[1] * 300).int().to(DEV), top_p=torch.where(r[2] < 0.3, torch.ones(rows), r[2]).to(DEV),
          min_p=torch.where(r[3] < 0.5, torch.zeros(rows), r[3] * 0.1).to(DEV))


@gpu
@pytest.mark.parametrize("name", ["plain", "greedy", "top_5", "top_700", "p_half", "p_most", "min_p", "all", "all_wide"])
@pytest.mark.parametrize("levels", [1, 2, 6])
def test_ties(name, levels):
    """Few distinct logits: every border falls among equal tokens, and the lowest indices win."""
    g = torch.Generator().manual_seed(levels)
    logits = torch.randint(0, levels, (12, 6001), generator=g).to(torch.bfloat16).to(DEV)
    check(logits, torch.rand(12, generator=g).to(DEV), **SETTINGS[name])


@gpu
@pytest.mark.parametrize("name", SETTINGS)
def test_flat_distribution(name):
    """Nothing stands out: with top-p the cut lies deep in the row."""
    logits, uniform = rows_of(4, 40009, torch.float32, seed=3, spread=0.3, peaks=0)
    check(logits, uniform, **SETTINGS[name])


@gpu
@pytest.mark.parametrize("name", SETTINGS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_tokens(name, dtype):
    """-inf, the type's lowest value and NaN in the row; rows with one token left, and with none."""
    logits, uniform = rows_of(8, 3001, dtype, seed=4)
    g = torch.Generator().manual_seed(5)
    off = (torch.rand(8, 3001, generator=g) < 0.9).to(DEV)
    logits[0].masked_fill_(off[0], float("-inf"))
    logits[1].masked_fill_(off[1], torch.finfo(dtype).min)
    logits[2].masked_fill_(off[2], float("nan"))
    logits[3] = float("-inf")
    logits[3, 2017] = -3.0
    logits[4] = torch.finfo(dtype).min
    logits[4, 3000] = float("nan")
    logits[5] = float("-inf")
    logits[5, ::7] = float("nan")
    logits[6, 100:110] = float("inf")
    logits[6, 105] = float("-inf")
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = ops.sample(logits, uniform, status=status, **SETTINGS[name])
    assert torch.equal(got.cpu(), reference(logits, uniform, **SETTINGS[name]))
    assert got[5] == 0 and got[3] == 2017 and status.item() == _lib.STATUS_EMPTY_ROW


@gpu
@pytest.mark.parametrize("name", ["plain", "top_40", "p_most", "min_p", "all"])
def test_extreme_random_numbers(name):
    u = torch.tensor([0.0, 2.0 ** -24, 2.0 ** -40, 1 - 2.0 ** -24, 0.5], device=DEV)
    logits, _ = rows_of(5, 4099, torch.float32, seed=6)
    check(logits, u, **SETTINGS[name])
    same = logits[:1].expand(5, 4099)                                       # one row for all: stride 0
    got = check(same, u, **SETTINGS[name])
    assert got[0] <= got[1] and got[2] <= got[1] <= got[4] <= got[3]
    outside = torch.tensor([-1.0, float("nan"), 1.0, 7.0, float("inf")], device=DEV)
    first, last = got[0], check(same, torch.full((5,), 1 - 2.0 ** -24, device=DEV), **SETTINGS[name])
    clamped = ops.sample(same, outside, **SETTINGS[name])
    assert clamped[0] == first and clamped[1] == first
    assert all(int(t) >= int(last[0]) for t in clamped[2:])


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offset,stride", [(0, 5003), (1, 5010), (3, 5007), (8, 5056)])
def test_rows_that_start_anywhere(dtype, offset, stride):
    logits, uniform = rows_of(7, 5003, dtype, seed=7)
    wide = torch.full((7, stride + offset), 99.0, dtype=dtype, device=DEV)   # large logits all around: none may be read
    view = wide[:, offset:offset + 5003] if stride + offset > 5003 else wide
    view.copy_(logits)
    for name in ("plain", "greedy", "top_40", "p_most", "all"):
        assert torch.equal(check(view, uniform, **SETTINGS[name]), ops.sample(logits, uniform, **SETTINGS[name]))


@gpu
def test_last_position_of_a_sequence_of_logits():
    logits = torch.randn(3, 4, 1000, generator=torch.Generator().manual_seed(8)).to(torch.bfloat16).to(DEV)
    check(logits[:, -1], torch.tensor([0.1, 0.5, 0.9], device=DEV), top_k=20)


@gpu
def test_extreme_temperatures():
    logits, uniform = rows_of(6, 2003, torch.float32, seed=9)
    for t in (1e-38, 1e-9, 3e-8, 1e-7, 1e-6, 1e6, 1e30, 1e37, 3e38):
        check(logits, uniform, temperature=t)
        check(logits, uniform, temperature=torch.full((6,), t, device=DEV), top_p=0.7)
    greedy = ops.sample(logits, uniform, temperature=0.0)
    for t in (-1.0, float("nan")):                                          # what a tensor may hold but a number may not
        assert torch.equal(ops.sample(logits, uniform, temperature=torch.full((6,), t, device=DEV)), greedy)
    for p in (0.0, -1.0):
        assert torch.equal(ops.sample(logits, uniform, top_p=torch.full((6,), p, device=DEV)), greedy)


@gpu
@pytest.mark.parametrize("temperature", [1e-7, 1e-6, 1e-5, 1.0, 1e36, 1e37, 3e38])
def test_neighbouring_and_outermost_logits(temperature):
    """Logits one float apart (a temperature of their spacing tells them apart), and the type's ends, beside -inf."""
    z = torch.full((4, 3000), float("-inf"))
    near = torch.tensor([10.0]).repeat(40)
    for i in range(1, 40):
        near[i] = torch.nextafter(near[i - 1], torch.tensor(0.0))
    z[0, 100:140] = near
    z[1, ::50] = torch.finfo(torch.float32).max
    z[1, 7] = torch.finfo(torch.float32).min
    z[2, ::70] = torch.finfo(torch.float32).min
    z[3, ::3] = torch.finfo(torch.float32).min
    z[3, 5], z[3, 9] = 0.0, torch.finfo(torch.float32).max
    z = z.to(DEV)
    for u in (0.1, 0.5, 0.93):
        for settings in ({}, dict(top_p=0.6), dict(min_p=0.3), dict(top_k=300, top_p=0.9), dict(top_k=5)):
            check(z, torch.full((4,), u, device=DEV), temperature=temperature, **settings)


@gpu
def test_repeated_and_captured_calls_agree():
    logits, uniform = rows_of(20, 50021, torch.bfloat16, seed=10)
    want = check(logits, uniform, temperature=1.2, top_p=0.98)
    for _ in range(5):
        assert torch.equal(ops.sample(logits, uniform, temperature=1.2, top_p=0.98), want)
    z, u, out = torch.zeros_like(logits), torch.zeros_like(uniform), torch.full((20,), -1, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.sample(z, u, temperature=1.2, top_p=0.98, out=out)
    z.copy_(logits), u.copy_(uniform)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        beside = ops.sample(logits, uniform, temperature=1.2, top_p=0.98)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(beside, want)


@gpu
def test_frequencies():
    """Random numbers on an even grid draw every kept token as often as its probability says, to one grid step."""
    p = torch.tensor([0.4, 0.3, 0.2, 0.1])
    n = 4000
    logits = p.log().float().to(DEV).expand(n, 4)
    u = ((torch.arange(n) + 0.5) / n).to(DEV)
    for settings, want in (({}, p), (dict(top_k=2), torch.tensor([4 / 7, 3 / 7, 0, 0])),
                           (dict(top_p=0.75), torch.tensor([4 / 9, 3 / 9, 2 / 9, 0])), (dict(min_p=0.7), torch.tensor([4 / 7, 3 / 7, 0, 0]))):
        counts = torch.bincount(ops.sample(logits, u, **settings).cpu(), minlength=4)
        assert (counts - want * n).abs().max() <= 1.01


@gpu
def test_refusals():
    logits, uniform = rows_of(3, 50, torch.float32, seed=11)
    for bad in (dict(temperature=-1), dict(temperature=float("inf")), dict(temperature=float("nan")), dict(top_k=-1), dict(top_p=0),
                dict(top_p=1.5), dict(min_p=-0.1), dict(min_p=2), dict(top_k=torch.ones(3, device=DEV)),
                dict(top_p=torch.ones(2, device=DEV)), dict(min_p=torch.ones(3)), dict(temperature=torch.ones(3, device=DEV).half()),
                dict(out=torch.empty(3, device=DEV)), dict(out=torch.empty(2, dtype=torch.int64, device=DEV))):
        with pytest.raises(RuntimeError):
            ops.sample(logits, uniform, **bad)
    for z, u in ((logits.double(), uniform), (logits[0], uniform), (logits, uniform[:2]), (logits, uniform.double()),
                 (logits.t(), uniform), (logits[:, :0], uniform), (logits, uniform.cpu())):
        with pytest.raises(RuntimeError):
            ops.sample(z, u)
    assert ops.sample(logits[:0], uniform[:0]).shape == (0,)


def test_refusals_without_a_gpu():
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.sample(torch.zeros(1, 4), torch.zeros(1))


def test_argument_errors_of_the_c_entry_point():
    buf = np.zeros(1024, np.uint8)
    p = (buf.ctypes.data + 15) // 16 * 16

    def call(**kw):
        a = dict(z=p, stride=10, t=2, rows=1, vocab=10, u=p, temp=None, out=p)
        a.update(kw)
        return _lib.lib.df11_sample(a["z"], a["stride"], a["t"], a["rows"], a["vocab"], a["u"], a["temp"], 1.0, None, 0, None, 1.0,
                                    None, 0.0, a["out"], None, 0, None)

    for kw in (dict(z=None), dict(u=None), dict(out=None), dict(t=3), dict(t=-1), dict(rows=-1), dict(vocab=0), dict(vocab=2 ** 31),
               dict(stride=-1), dict(z=p + 2), dict(out=p + 4), dict(u=p + 1), dict(temp=p + 2)):
        assert call(**kw) == _lib.DF11_ERR_BADARG, kw
        assert _lib.lib.df11_last_error()
    assert call(rows=0) == _lib.DF11_OK
