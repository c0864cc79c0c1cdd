"""The key/value cache of a generating model in 8 bits, and its place in ``transformers``.

The reference keeps weights small and leaves the cache to its caller's library, in BF16; once the weights are 30 %
smaller it is the cache that limits batch and context (a 36-layer model with 8 key heads of 128: 144 KB per token).
``QuantizedKVCache`` holds it as int8 or e4m3 codes with one scale per row -- 0.52 of the BF16 bytes -- and offers what a
layer needs: ``append`` quantises new rows as they are written, ``attend`` is attention straight over the codes for a few
new tokens, ``read`` gives rows back for an ordinary attention.  ``for_model`` makes a ``transformers`` cache of it; the
model's attention then goes through the function registered as ``df11_kv``:

* the first tokens (an empty cache) attend to one another exactly, in the precision of the activations, while their rows are
  quantised for those that follow;
* up to ``FEW_TOKENS`` later ones attend straight to the codes;
* longer ones (the next chunk of a long prompt) attend to the rows read back, and exactly to one another.

Device-side state only: the number of tokens seen is a tensor, so a single-token step can be captured into a CUDA graph
and replayed.
"""
from __future__ import annotations

from typing import List, Optional, Tuple

import torch

from . import ops

FORMATS = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
FEW_TOKENS = 16          # tokens per sequence that attend straight to the codes
ATTENTION_NAME = "df11_kv"


class QuantizedKVCache:
    """Codes and scales of ``n_layers`` layers for sequences of one batch that move together.

    ``seen`` (int64 ``[1]`` on the device) is the number of tokens in the cache.  A forward of ``n`` tokens calls
    ``begin(n)``, then ``append`` / ``attend`` per layer, then ``end()``; ``filled`` is ``seen + n`` meanwhile.  Where the
    number is known on the host (no graph replay has moved it since ``reset``), ``host_seen`` has it."""

    def __init__(self, n_layers: int, batch: int, kv_heads: int, head_dim: int, max_slots: int, fmt: str = "int8",
                 device="cuda"):
        if fmt not in FORMATS:
            raise ValueError(f"unknown cache format {fmt!r}: {', '.join(FORMATS)} are supported")
        if min(n_layers, batch, kv_heads, max_slots) < 1:
            raise ValueError("a cache needs at least one layer, sequence, head and slot")
        if head_dim < 16 or head_dim > 256 or head_dim % 16:
            raise ValueError(f"head_dim {head_dim}: multiples of 16 up to 256 are supported")
        device = torch.device(device)
        if device.type != "cuda":
            raise RuntimeError("QuantizedKVCache needs a CUDA device")
        self.fmt, self.max_slots = fmt, int(max_slots)
        shape = (batch, kv_heads, self.max_slots, head_dim)
        # zeros, so that slots that were never written hold numbers
        self.layers: List[Tuple[torch.Tensor, ...]] = [
            tuple(t for _ in range(2) for t in (torch.zeros(shape, dtype=torch.uint8, device=device).view(FORMATS[fmt]),
                                                torch.zeros(shape[:3], dtype=torch.float32, device=device)))
            for _ in range(n_layers)]
        self.seen = torch.zeros(1, dtype=torch.int64, device=device)
        self.filled = torch.zeros(1, dtype=torch.int64, device=device)
        self.host_seen: Optional[int] = 0

    @property
    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for layer in self.layers for t in layer)

    def reset(self) -> None:
        """Forget all tokens.  The bytes stay; nothing reads them before they are written again."""
        self.seen.zero_()
        self.filled.zero_()
        self.host_seen = 0

    def begin(self, n_tokens: int) -> None:
        if self.host_seen is not None and self.host_seen + n_tokens > self.max_slots:
            raise ValueError(f"{self.host_seen} + {n_tokens} tokens exceed the cache's {self.max_slots} slots")
        torch.add(self.seen, n_tokens, out=self.filled)

    def end(self, n_tokens: int) -> None:
        self.seen.copy_(self.filled)
        if torch.cuda.is_current_stream_capturing():
            self.host_seen = None                       # replays move the cache without the host's knowledge
        elif self.host_seen is not None:
            self.host_seen += n_tokens

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, status: Optional[torch.Tensor] = None) -> None:
        """New rows ``[batch, kv_heads, n, head_dim]`` to the slots from ``seen`` on."""
        ops.kv_append(k, v, *self.layers[layer], self.seen, status=status)

    def attend(self, layer: int, q: torch.Tensor, scale: Optional[float] = None) -> torch.Tensor:
        """``q`` ``[batch, heads, n, head_dim]``, the last ``n`` of the ``filled`` tokens -> ``[batch, n, heads, head_dim]``."""
        return ops.kv_attention(q, *self.layers[layer], self.filled, scale=scale)

    def read(self, layer: int, first_slot: int, n_slots: int, dtype: torch.dtype = torch.bfloat16):
        """``(k, v)`` rows of these slots, each ``[batch, kv_heads, n_slots, head_dim]``."""
        return ops.kv_read(*self.layers[layer], first_slot, n_slots, dtype=dtype)


def _attention(module, query, key, value, attention_mask, scaling=None, dropout=0.0, **kwargs):
    """The attention function behind ``df11_kv``; ``key`` carries the cache layer that it was appended to."""
    layer = getattr(key, "df11_cache_layer", None)
    if layer is None:
        raise RuntimeError("the df11_kv attention needs a cache made by kv_cache.for_model")
    if dropout or any(kwargs.get(name) is not None for name in ("sliding_window", "softcap", "s_aux", "head_mask")):
        raise NotImplementedError("the quantised cache has no dropout, sliding window, soft-capping, sinks or head masks")
    if attention_mask is not None:
        raise NotImplementedError("the quantised cache takes prompts of one length, without an attention mask")
    store, past, n = layer.store, layer.past, query.shape[2]
    if past != 0 and (n <= FEW_TOKENS or past is None):
        return store.attend(layer.index, query, scale=scaling), None
    mask = None
    if past:
        k, v = store.read(layer.index, 0, past, dtype=key.dtype)
        key, value = torch.cat([k, key], dim=2), torch.cat([v, value], dim=2)
        mask = torch.ones(n, past + n, dtype=torch.bool, device=query.device).tril_(past)
    out = torch.nn.functional.scaled_dot_product_attention(query, key, value, attn_mask=mask, is_causal=mask is None, scale=scaling,
                                                           enable_gqa=query.shape[1] != key.shape[1])
    return out.transpose(1, 2).contiguous(), None


def _no_mask(*args, **kwargs):
    if kwargs.get("attention_mask") is not None and not bool(kwargs["attention_mask"].all()):
        raise NotImplementedError("the quantised cache takes prompts of one length, without padding")
    return None


_cache_class = None


def _cache_type():
    """The cache class; made on first use, since it derives from ``transformers``' and registers the attention there."""
    global _cache_class
    if _cache_class is not None:
        return _cache_class
    from transformers import AttentionInterface, AttentionMaskInterface, Cache
    from transformers.cache_utils import CacheLayerMixin

    class QuantizedLayer(CacheLayerMixin):
        is_compileable = True
        is_sliding = False

        def __init__(self, cache, index: int):
            super().__init__()
            self.cache, self.index = cache, index
            self.past: Optional[int] = 0

        @property
        def store(self) -> QuantizedKVCache:
            return self.cache.store

        def lazy_initialization(self, key_states, value_states):
            cache = self.cache
            if cache.store is None:
                batch, heads, _, dim = key_states.shape
                cache.store = QuantizedKVCache(len(cache.layers), batch, heads, dim, cache.max_slots, cache.fmt, key_states.device)
            self.is_initialized = True

        def update(self, key_states, value_states, *args, **kwargs):
            if not self.is_initialized:
                self.lazy_initialization(key_states, value_states)
            store, n = self.store, key_states.shape[2]
            if self.index == 0:
                store.begin(n)
            self.past = store.host_seen
            store.append(self.index, key_states, value_states, status=self.cache.status)
            if self.index == len(store.layers) - 1:
                store.end(n)
            key_states.df11_cache_layer = self
            return key_states, value_states

        def get_mask_sizes(self, query_length):
            return self.cache.max_slots, 0

        def get_seq_length(self):
            return 0 if self.store is None else self.store.seen

        def get_max_cache_shape(self):
            return self.cache.max_slots

        def reset(self):
            if self.index == 0 and self.store is not None:
                self.store.reset()

    class QuantizedModelCache(Cache):
        def __init__(self, n_layers: int, max_slots: int, fmt: str, status: Optional[torch.Tensor]):
            self.store: Optional[QuantizedKVCache] = None
            self.max_slots, self.fmt, self.status = int(max_slots), fmt, status
            super().__init__(layers=[QuantizedLayer(self, i) for i in range(n_layers)])

    AttentionInterface.register(ATTENTION_NAME, _attention)
    AttentionMaskInterface.register(ATTENTION_NAME, _no_mask)
    _cache_class = QuantizedModelCache
    return QuantizedModelCache


def for_model(config, max_slots: int, fmt: str = "int8", status: Optional[torch.Tensor] = None):
    """A ``transformers`` cache over a ``QuantizedKVCache`` for a decoder of this configuration.

    The codes are allocated with the first tokens, for their batch, heads (of a tensor-parallel shard: its own) and device;
    ``.store`` is then the ``QuantizedKVCache``; all of the model's layers are on that device.  The model has to run with ``set_attn_implementation("df11_kv")``, for
    which ``GraphedGreedyDecoder(kv_format=...)`` cares.  ``status``: int32 word for ``STATUS_BAD_POSITIONS``."""
    if fmt not in FORMATS:
        raise ValueError(f"unknown cache format {fmt!r}: {', '.join(FORMATS)} are supported")
    text = config.get_text_config(decoder=True) if hasattr(config, "get_text_config") else config
    kinds = set(getattr(text, "layer_types", None) or ["full_attention"])
    if kinds != {"full_attention"}:
        raise ValueError(f"the quantised cache is for full attention in every layer, not {sorted(kinds)}")
    return _cache_type()(text.num_hidden_layers, max_slots, fmt, status)
