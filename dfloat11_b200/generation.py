"""Generation with the host taken out of the loop: one CUDA graph per single-token step.

The reference measures generation through Hugging Face ``generate`` (inference.py:45-95), where
every token pays the Python cost of a whole forward pass -- some 30 ms for a 36-layer model,
several times what the GPU needs.  Here the single-token step (forward over a static KV cache,
arg-max, position update) is captured once into a CUDA graph and replayed per token.  The DF11
decode hooks run at capture time; their launches through the C ABI are recorded like any other
kernel, so a replay decompresses (or, with ``DF11_FUSED_GEMV=1``, multiplies straight from the
compressed weights) exactly as an eager step would.

The next token is the arg-max or, with a temperature, drawn by ``ops.sample`` from random numbers that are
made before the loop.  With ``kv_format`` the keys and values are kept in 8 bits (``kv_cache.py``) instead of
in a ``StaticCache``: half the memory, and attention reads the filled part of the codes only.

Works for any ``transformers`` causal LM whose forward accepts ``past_key_values`` /
``cache_position`` with a ``StaticCache`` -- compressed or not, whole or tensor-parallel (every
rank runs the same loop; the collectives of the partitioned mode are captured with the rest).
Prompts of one batch have the same length; the graph is captured per batch size.
"""
from __future__ import annotations

from contextlib import contextmanager
from typing import Optional

import torch

from . import kv_cache, ops


class GraphedGreedyDecoder:
    """``decoder = GraphedGreedyDecoder(model, max_cache_len=4096); ids = decoder.generate(prompt, 256)``

    ``kv_format``: ``"int8"`` or ``"e4m3"`` keeps the cache in 8 bits; None in the activations' precision.
    ``prefill_chunk``: tokens of a prompt that go through the model at once (None: all), which bounds the memory of
    a long prompt's activations."""

    def __init__(self, model, max_cache_len: int = 4096, kv_format: Optional[str] = None, prefill_chunk: Optional[int] = None):
        if kv_format is not None and kv_format not in kv_cache.FORMATS:
            raise ValueError(f"unknown cache format {kv_format!r}: {', '.join(kv_cache.FORMATS)} are supported")
        if prefill_chunk is not None and prefill_chunk < 1:
            raise ValueError("prefill_chunk must be at least 1")
        self.model = model
        self.max_cache_len = int(max_cache_len)
        self.kv_format = kv_format
        self.prefill_chunk = prefill_chunk
        self.device = next(model.parameters()).device
        if self.device.type != "cuda":
            raise RuntimeError("GraphedGreedyDecoder needs the model on a CUDA device")
        import inspect
        try:
            self._keeps_logits = "logits_to_keep" in inspect.signature(model.forward).parameters
        except (TypeError, ValueError):
            self._keeps_logits = False
        self._cache = None
        self._graph = None
        self._graph_samples = False
        self._tok = self._pos = self._count = self._produced = None
        self._uniform = self._settings = None

    # -- one single-token step on static tensors -------------------------------------------------
    def _choose(self, logits: torch.Tensor, uniform: Optional[torch.Tensor]) -> None:
        """The next token of every sequence: arg-max, or drawn with the settings and these random numbers."""
        if uniform is None:
            self._tok.copy_(logits[:, -1:].argmax(-1))
        else:
            last = logits[:, -1]
            if last.stride(1) != 1:
                last = last.contiguous()
            self._tok.copy_(ops.sample(last, uniform, **self._settings, status=self._status()).view(-1, 1))

    def _status(self) -> torch.Tensor:
        from .dfloat11 import _status_word
        return _status_word(self._tok.device)

    def _step(self, samples: bool):
        self._produced.index_copy_(0, self._count, self._tok.view(1, -1))
        logits = self.model(input_ids=self._tok, past_key_values=self._cache, cache_position=self._pos,
                            use_cache=True).logits
        # the prompt's token was drawn with row 0, the token after the one at `count` is drawn with row count + 1
        self._choose(logits, self._uniform[1:].index_select(0, self._count).view(-1) if samples else None)
        self._pos.add_(1)
        self._count.add_(1)

    def _prepare(self, batch: int):
        from transformers import StaticCache
        dev = self.device
        if self._cache is None or self._tok.shape[0] != batch:
            self._graph = None                            # static tensors change: the old capture is void
            self._cache = None
            if self.kv_format is None:
                self._cache = StaticCache(config=self.model.config, max_cache_len=self.max_cache_len)
            self._tok = torch.zeros(batch, 1, dtype=torch.int64, device=dev)
            self._pos = torch.zeros(1, dtype=torch.int64, device=dev)
            self._count = torch.zeros(1, dtype=torch.int64, device=dev)
            self._produced = torch.zeros(self.max_cache_len + 8, batch, dtype=torch.int64, device=dev)
            self._uniform = torch.zeros(self.max_cache_len + 8, batch, dtype=torch.float32, device=dev)
            self._settings = dict(temperature=torch.ones(batch, device=dev), top_k=torch.zeros(batch, dtype=torch.int32, device=dev),
                                  top_p=torch.ones(batch, device=dev), min_p=torch.zeros(batch, device=dev))
            if self.kv_format is not None:
                self._cache = kv_cache.for_model(self.model.config, self.max_cache_len, self.kv_format, status=self._status())
        else:
            self._cache.reset()

    @contextmanager
    def _attention(self):
        """The model's attention while the cache is quantised, put back afterwards."""
        if self.kv_format is None:
            yield
            return
        before = self.model.config._attn_implementation
        self.model.set_attn_implementation(kv_cache.ATTENTION_NAME)
        try:
            yield
        finally:
            self.model.set_attn_implementation(before)

    def _prefill(self, input_ids: torch.Tensor) -> torch.Tensor:
        """The prompt through the model, chunk by chunk; returns the logits of its last chunk."""
        n_prompt = input_ids.shape[1]
        chunk = self.prefill_chunk or n_prompt
        # only the last position's logits are needed: models whose forward can skip the others
        # (`logits_to_keep`) do not multiply the whole prompt with the output head
        extra = {"logits_to_keep": 1} if self._keeps_logits else {}
        for start in range(0, n_prompt, chunk):
            stop = min(start + chunk, n_prompt)
            logits = self.model(input_ids=input_ids[:, start:stop], past_key_values=self._cache,
                                cache_position=torch.arange(start, stop, device=input_ids.device), use_cache=True, **extra).logits
        return logits

    def _set_sampling(self, batch: int, max_new_tokens: int, temperature, top_k, top_p, min_p, generator) -> None:
        for name, value, low, high in (("temperature", temperature, 0.0, 3.4e38), ("top_k", top_k, 0, 2 ** 31 - 1),
                                       ("top_p", top_p, 1e-45, 1.0), ("min_p", min_p, 0.0, 1.0)):
            value = torch.as_tensor(value, dtype=torch.float64).reshape(-1).cpu()
            if value.numel() not in (1, batch) or not bool(((value >= low) & (value <= high)).all()):
                raise ValueError(f"{name} must be a number or one per sequence, from {low} to {high}")
            self._settings[name].copy_(value.expand(batch))
        rows = self._uniform[:max_new_tokens]
        if generator is None or generator.device == rows.device:
            torch.rand(rows.shape, generator=generator, out=rows)
        else:
            rows.copy_(torch.rand(rows.shape, generator=generator))

    def generate(self, input_ids: torch.Tensor, max_new_tokens: int, eos_token_id: Optional[int] = None,
                 eos_check_every: int = 32, temperature=None, top_k=0, top_p=1.0, min_p=0.0,
                 generator: Optional[torch.Generator] = None) -> torch.Tensor:
        """Prompts ``[b, n]`` -> ``[b, n + new]`` ids.  With one sequence, stops early at
        ``eos_token_id`` (looked for every ``eos_check_every`` tokens, the only host synchronisation
        in the loop).

        Greedy unless ``temperature`` is given; ``temperature``, ``top_k``, ``top_p`` and ``min_p`` are numbers or one per
        sequence, as ``ops.sample`` has them (a temperature of 0 is greedy for its sequence).  The random numbers come
        from ``generator`` (ranks of a tensor-parallel group need generators of one seed each)."""
        with torch.no_grad(), self._attention():
            return self._generate(input_ids, max_new_tokens, eos_token_id, eos_check_every, temperature, top_k, top_p, min_p, generator)

    def _generate(self, input_ids, max_new_tokens, eos_token_id, eos_check_every, temperature, top_k, top_p, min_p, generator):
        if input_ids.dim() != 2 or input_ids.shape[0] < 1:
            raise ValueError("input_ids must be [batch, n]")
        if eos_token_id is not None and input_ids.shape[0] != 1:
            raise ValueError("early stopping at an end-of-sequence id is for one sequence at a time")
        n_prompt = input_ids.shape[1]
        if n_prompt + max_new_tokens > self.max_cache_len:
            raise ValueError(f"{n_prompt} + {max_new_tokens} tokens exceed max_cache_len = {self.max_cache_len}")
        if max_new_tokens <= 0:
            return input_ids
        dev = self.device
        input_ids = input_ids.to(dev)
        self._prepare(input_ids.shape[0])
        samples = temperature is not None
        if samples:
            self._set_sampling(input_ids.shape[0], max_new_tokens, temperature, top_k, top_p, min_p, generator)
        if samples != self._graph_samples:
            self._graph = None                             # the captured step chooses its token the other way
            self._graph_samples = samples
        self._choose(self._prefill(input_ids), self._uniform[0] if samples else None)
        self._pos.fill_(n_prompt)
        self._count.zero_()

        steps = max_new_tokens - 1                         # the prefill gave the first new token
        done = 0
        if self._graph is None and steps > 0:
            # two eager steps on a side stream (allocations, lazy initialisation, the hooks' one-time
            # work) advance the generation like any other step; the capture records a step
            # without running it
            side = torch.cuda.Stream(device=dev)
            side.wait_stream(torch.cuda.current_stream(dev))
            with torch.cuda.stream(side):
                while done < min(2, steps):
                    self._step(samples)
                    done += 1
            torch.cuda.current_stream(dev).wait_stream(side)
            if done < steps:
                torch.cuda.synchronize(dev)
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    self._step(samples)
                self._graph = graph
        if self.kv_format is not None and done < steps:
            self._cache.store.host_seen = None             # replays move the cache without the host's knowledge
        while done < steps:
            self._graph.replay()
            done += 1
            if eos_token_id is not None and done % eos_check_every == 0:
                if bool((self._produced[:done, 0] == eos_token_id).any()):
                    break
        # the token of the last step is still in `tok`
        self._produced.index_copy_(0, self._count, self._tok.view(1, -1))
        new = self._produced[:done + 1]
        if eos_token_id is not None:
            hit = (new[:, 0] == eos_token_id).nonzero()
            if hit.numel():
                new = new[:int(hit[0]) + 1]
        return torch.cat([input_ids, new.t()], dim=1)

    def reset(self) -> None:
        """Forget the captured graph (after changing the model or the DF11 environment switches)."""
        self._graph = None
