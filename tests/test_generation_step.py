"""The quantised cache, the attention over it and sampling together, as a generation step uses them: through a model's
layers, in the graph decoder, eagerly and replayed."""
import pytest
import torch
import torch.nn as nn

import dfloat11_b200 as df11
from dfloat11_b200 import kv_cache, ops
from tests.test_kv_cache import reference_attention, reference_rows
from tests.test_model_api import tiny_llama

gpu = pytest.mark.gpu
DEV = "cuda:0"


def prompt(batch, n, seed):
    return torch.randint(0, 1024, (batch, n), generator=torch.Generator().manual_seed(seed)).to(DEV)


def eager(model, ids, n_new, fmt, chunk=None, choose=None, max_len=64):
    """The decoder's loop without a graph: (ids, cache).  choose(logits [b, vocab], step) gives the next tokens."""
    from transformers import StaticCache
    cache = kv_cache.for_model(model.config, max_len, fmt) if fmt else StaticCache(config=model.config, max_cache_len=max_len)
    choose = choose or (lambda z, step: z.argmax(-1))
    before = model.config._attn_implementation
    if fmt:
        model.set_attn_implementation(kv_cache.ATTENTION_NAME)
    try:
        with torch.no_grad():
            out, n = [ids], ids.shape[1]
            for start in range(0, n, chunk or n):
                stop = min(start + (chunk or n), n)
                logits = model(input_ids=ids[:, start:stop], past_key_values=cache, use_cache=True,
                               cache_position=torch.arange(start, stop, device=ids.device)).logits
            for step in range(n_new):
                out.append(choose(logits[:, -1], step).view(-1, 1))
                if step < n_new - 1:
                    logits = model(input_ids=out[-1], past_key_values=cache, use_cache=True,
                                   cache_position=torch.tensor([n + step], device=ids.device)).logits
    finally:
        model.set_attn_implementation(before)
    return torch.cat(out, dim=1), cache


@gpu
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_what_the_layers_get(fmt, monkeypatch):
    """Every layer's rows reach the cache in their slots, and every later token attends to exactly those."""
    model = tiny_llama(seed=3).to(DEV)
    rows, seen, checked = {}, [], []
    append, attend = ops.kv_append, ops.kv_attention

    def spy_append(k, v, k_codes, *rest, **kw):
        rows.setdefault(k_codes.data_ptr(), []).append((k.clone().cpu(), v.clone().cpu()))
        return append(k, v, k_codes, *rest, **kw)

    def spy_attend(q, *cache_and_lengths, **kw):
        cache, lengths = cache_and_lengths[:4], cache_and_lengths[4]
        k, v = (torch.cat([r[i] for r in rows[cache[0].data_ptr()]], dim=2) for i in (0, 1))
        n = k.shape[2]
        assert lengths.tolist() == [n] and kw["scale"] == pytest.approx(q.shape[3] ** -0.5)
        for x, codes, scales in ((k, cache[0], cache[1]), (v, cache[2], cache[3])):
            want, want_scale = reference_rows(x, fmt)
            assert torch.equal(codes[:, :, :n].float().cpu().double(), want) and torch.equal(scales[:, :, :n].cpu(), want_scale)
            assert not codes[:, :, n:].float().any()
        got = attend(q, *cache_and_lengths, **kw)
        want, bound = reference_attention(q, cache, [n] * q.shape[0], [0] * q.shape[0], kw["scale"], 0)
        assert ((got.cpu().double() - want).abs() <= bound + want.abs() * 2.0 ** -8 + 1e-12).all()
        seen.append((q.shape[2], n))
        checked.append(cache[0].data_ptr())
        return got

    monkeypatch.setattr(ops, "kv_append", spy_append)
    monkeypatch.setattr(ops, "kv_attention", spy_attend)
    ids, cache = eager(model, prompt(2, 9, 1), 5, fmt)
    assert ids.shape == (2, 14)
    # the prompt attends to itself without the codes; each of the 4 steps asks all 3 layers
    assert seen == [(1, n) for n in (10, 11, 12, 13) for _ in range(3)] and len(set(checked)) == 3
    assert int(cache.get_seq_length()) == 13 and cache.store.host_seen == 13
    bf16 = 2 * 2 * 2 * 64 * 32 * 3 * 2                                  # K and V, batch, heads, slots, dims, layers, bytes
    assert cache.store.nbytes == bf16 // 2 * (32 + 4) // 32


@gpu
def test_the_first_tokens_attend_exactly():
    """The prompt's logits are those of the same model with its own attention and cache."""
    model = tiny_llama(seed=4).to(DEV)
    ids = prompt(2, 11, 2)
    captured = {}

    def choose(name):
        def f(z, step):
            captured.setdefault(name, z.clone())
            return z.argmax(-1)
        return f

    eager(model, ids, 1, None, choose=choose("own"))
    eager(model, ids, 1, "int8", choose=choose("df11"))
    a, b = captured["own"].float(), captured["df11"].float()
    # two bf16 attentions in 3 layers differ by roundings only: far below the spread of the logits
    assert (a - b).abs().max() <= 0.05 * a.std() and model.config._attn_implementation != kv_cache.ATTENTION_NAME


@gpu
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("batch,chunk", [(1, None), (3, None), (2, 20), (1, 1)])
def test_decoder_with_a_quantised_cache(fmt, batch, chunk):
    """One graph per token gives the ids of the same loop run eagerly, on repeated calls and other prompts."""
    model = tiny_llama(seed=5).to(DEV)
    ids, other = prompt(batch, 45, 3), prompt(batch, 23, 4)
    decoder = df11.GraphedGreedyDecoder(model, max_cache_len=64, kv_format=fmt, prefill_chunk=chunk)
    want, _ = eager(model, ids, 16, fmt, chunk)
    want_other, _ = eager(model, other, 30, fmt, chunk)
    assert torch.equal(decoder.generate(ids, 16), want)
    assert torch.equal(decoder.generate(ids, 16), want)
    assert torch.equal(decoder.generate(other, 30), want_other)
    assert torch.equal(decoder.generate(ids, 1), want[:, :46])
    assert torch.equal(decoder.generate(ids, 16), want)
    assert model.config._attn_implementation != kv_cache.ATTENTION_NAME
    with pytest.raises(ValueError):
        decoder.generate(ids, 20)
    df11.check_status()


@gpu
@pytest.mark.parametrize("fmt", [None, "int8"])
@pytest.mark.parametrize("batch", [1, 3])
def test_decoder_that_samples(fmt, batch):
    """Replayed steps draw what the same settings and random numbers give step by step; settings may change between calls."""
    model = tiny_llama(seed=6).to(DEV)
    ids = prompt(batch, 9, 5)
    decoder = df11.GraphedGreedyDecoder(model, max_cache_len=64, kv_format=fmt)
    greedy, _ = eager(model, ids, 12, fmt)
    for settings in (dict(temperature=0.9, top_k=40, top_p=0.95), dict(temperature=[0.0, 1.5, 0.7][:batch], min_p=0.01),
                     dict(temperature=torch.full((batch,), 3.0))):
        uniform = torch.rand(12, batch, generator=torch.Generator(DEV).manual_seed(7), device=DEV)
        per_row = dict(temperature=torch.as_tensor(settings["temperature"], dtype=torch.float32).expand(batch).contiguous().to(DEV),
                       **{k: v for k, v in settings.items() if k != "temperature"})
        if "top_p" in per_row:                              # the decoder keeps settings as float32
            per_row["top_p"] = torch.full((batch,), per_row["top_p"], device=DEV)
        if "min_p" in per_row:
            per_row["min_p"] = torch.full((batch,), per_row["min_p"], device=DEV)
        want, _ = eager(model, ids, 12, fmt, choose=lambda z, step: ops.sample(z, uniform[step].contiguous(), **per_row))
        for _ in range(2):
            got = decoder.generate(ids, 12, generator=torch.Generator(DEV).manual_seed(7), **settings)
            assert torch.equal(got, want)
        assert torch.equal(decoder.generate(ids, 12), greedy)              # and back: the other kind of step
    assert torch.equal(decoder.generate(ids, 12, temperature=0.0), greedy)
    a, b = (decoder.generate(ids, 40, temperature=5.0, generator=torch.Generator().manual_seed(s)) for s in (1, 2))
    assert not torch.equal(a, b)
    eos = int(a[0, 9 + 8])
    if batch == 1:
        got = decoder.generate(ids, 40, eos_token_id=eos, eos_check_every=4, temperature=5.0, generator=torch.Generator().manual_seed(1))
        first = int((a[0, 9:] == eos).nonzero()[0])
        assert torch.equal(got, a[:, :9 + first + 1])
    df11.check_status()


@gpu
def test_compressed_weights_with_the_whole_step(tmp_path):
    """A compressed model, the quantised cache and sampling in one graph: the ids of the uncompressed model."""
    import copy
    path = str(tmp_path / "m")
    reference = tiny_llama(seed=8)
    df11.compress_model(copy.deepcopy(reference), {r"model\.embed_tokens": [], r"lm_head": [],
                                                   r"model\.layers\.\d+": ["self_attn.q_proj", "self_attn.k_proj", "self_attn.v_proj",
                                                                           "self_attn.o_proj", "mlp.gate_proj", "mlp.up_proj", "mlp.down_proj"]},
                        path, check_correctness=False)
    model = df11.DFloat11Model.from_pretrained(path, device=DEV, bfloat16_model=tiny_llama(seed=9))
    ids = prompt(2, 13, 6)
    got = [df11.GraphedGreedyDecoder(m, max_cache_len=64, kv_format="int8").generate(
        ids, 20, temperature=0.8, top_p=0.9, generator=torch.Generator(DEV).manual_seed(11)) for m in (model, reference.to(DEV))]
    assert torch.equal(got[0], got[1]) and got[0].shape == (2, 33)


@gpu
def test_cache_by_hand():
    """QuantizedKVCache without a model: what a layer of one's own does with it."""
    store = df11.QuantizedKVCache(2, 3, 2, 64, 40, "e4m3", DEV)
    g = torch.Generator(DEV).manual_seed(12)
    rows = torch.randn(2, 2, 3, 2, 7, 64, generator=g, device=DEV).to(torch.bfloat16)
    q = torch.randn(3, 8, 3, 64, generator=g, device=DEV).to(torch.bfloat16)
    for start, stop in ((0, 4), (4, 7)):
        store.begin(stop - start)
        for layer in range(2):
            store.append(layer, rows[0, layer, :, :, start:stop], rows[1, layer, :, :, start:stop])
            out = store.attend(layer, q[:, :, :stop - start])
        store.end(stop - start)
    assert store.host_seen == 7 and store.seen.item() == 7
    k, v = store.read(1, 0, 7)
    want, scale = reference_rows(rows[0, 1].cpu(), "e4m3")
    assert torch.equal(k.cpu(), (want.float() * scale[..., None]).to(torch.bfloat16)) and v.shape == (3, 2, 7, 64)
    want, bound = reference_attention(q, store.layers[1], [7] * 3, [0] * 3, 64 ** -0.5, 0)
    assert ((out.cpu().double() - want).abs() <= bound + want.abs() * 2.0 ** -8 + 1e-12).all()
    with pytest.raises(ValueError, match="exceed"):
        store.begin(34)
    store.reset()
    assert store.seen.item() == 0


@gpu
def test_refusals_on_the_gpu():
    model = tiny_llama(seed=13).to(DEV)
    ids = prompt(2, 5, 8)
    decoder = df11.GraphedGreedyDecoder(model, max_cache_len=32, kv_format="int8")
    for bad in (dict(temperature=-1.0), dict(temperature=float("nan")), dict(temperature=1.0, top_k=-1), dict(temperature=1.0, top_p=0.0),
                dict(temperature=1.0, top_p=1.1), dict(temperature=1.0, min_p=2.0), dict(temperature=[1.0, 1.0, 1.0])):
        with pytest.raises(ValueError):
            decoder.generate(ids, 4, **bad)
    cache = kv_cache.for_model(model.config, 32)
    model.set_attn_implementation(kv_cache.ATTENTION_NAME)
    with torch.no_grad():
        with pytest.raises(NotImplementedError):                           # left padding
            model(input_ids=ids, past_key_values=cache, use_cache=True, attention_mask=(ids > 300).long())
        with pytest.raises(RuntimeError, match="for_model"):               # another cache
            model(input_ids=ids, use_cache=True)


def test_refusals_without_a_gpu():
    with pytest.raises(ValueError, match="format"):
        df11.GraphedGreedyDecoder(nn.Linear(2, 2), kv_format="int4")
    with pytest.raises(ValueError, match="chunk"):
        df11.GraphedGreedyDecoder(nn.Linear(2, 2), prefill_chunk=0)
    with pytest.raises(RuntimeError, match="CUDA"):
        df11.GraphedGreedyDecoder(nn.Linear(2, 2), kv_format="int8")
    with pytest.raises(ValueError, match="format"):
        df11.QuantizedKVCache(1, 1, 1, 64, 8, "bf16")
    for bad in (dict(n_layers=0), dict(batch=0), dict(kv_heads=0), dict(max_slots=0), dict(head_dim=24), dict(head_dim=512)):
        sizes = dict(n_layers=1, batch=1, kv_heads=1, head_dim=64, max_slots=8)
        sizes.update(bad)
        with pytest.raises(ValueError):
            df11.QuantizedKVCache(**sizes)
    with pytest.raises(RuntimeError, match="CUDA"):
        df11.QuantizedKVCache(1, 1, 1, 64, 8, device="cpu")


def test_models_with_other_attention_are_refused():
    from transformers import LlamaConfig
    config = LlamaConfig(num_hidden_layers=2, hidden_size=64, num_attention_heads=2)
    config.layer_types = ["full_attention", "sliding_attention"]
    with pytest.raises(ValueError, match="full attention"):
        kv_cache.for_model(config, 16)
    with pytest.raises(ValueError, match="format"):
        kv_cache.for_model(LlamaConfig(num_hidden_layers=1), 16, "int2")
    assert len(kv_cache.for_model(LlamaConfig(num_hidden_layers=3), 16).layers) == 3
