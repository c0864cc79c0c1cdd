"""Torch-facing launchers of the libdf11 entry points.

These stand where the reference calls its cupy kernel object
(``_decode(grid=..., block=..., shared_mem=..., args=[...])``, dfloat11/dfloat11.py:142-151
and :576-585): same tensors, same meaning, but the launch goes through the C ABI of
``libdf11.so`` onto torch's current CUDA stream of the tensors' device.  There is no
CPU or pure-PyTorch fallback: tensors that are not on a CUDA device raise.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib


def _require_cuda(_pinned_ok=(), **tensors: torch.Tensor) -> torch.device:
    """The CUDA device all the tensors are on.  Names listed in ``_pinned_ok`` may instead be pinned
    host tensors: page-locked memory has the same address on the device (unified addressing), so a
    kernel can read the few bytes it needs of them over PCIe without a staging copy."""
    device = None
    for name, t in tensors.items():
        if t is None:
            continue
        if not t.is_cuda and name in _pinned_ok and t.is_pinned():
            if not t.is_contiguous():
                raise RuntimeError(f"`{name}` must be contiguous")
            continue
        if not t.is_cuda:
            raise RuntimeError(f"df11 decode needs CUDA tensors; `{name}` is on {t.device}")
        if not t.is_contiguous():
            raise RuntimeError(f"`{name}` must be contiguous")
        if device is None:
            device = t.device
        elif t.device != device:
            raise RuntimeError(f"`{name}` is on {t.device}, expected {device}")
    return device


def _stream(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def decode(luts: torch.Tensor, encoded_exponent: torch.Tensor, sign_mantissa: torch.Tensor,
           output_positions: torch.Tensor, gaps: torch.Tensor, out: Optional[torch.Tensor] = None,
           max_block_elems: int = 0, status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Decompress one DF11 unit into ``out`` (BF16, ``sign_mantissa.numel()`` elements).

    ``output_positions`` may be the uint8 byte view stored on disk or a uint32/int32 tensor.
    ``status`` is an optional int32 tensor of one element that receives DF11_STATUS_* bits.
    Asynchronous: returns right after the launch on the current stream.
    """
    device = _require_cuda(luts=luts, encoded_exponent=encoded_exponent, sign_mantissa=sign_mantissa,
                           output_positions=output_positions, gaps=gaps, out=out, status=status)
    n_elements = sign_mantissa.numel()
    if out is None:
        out = torch.empty(n_elements, dtype=torch.bfloat16, device=device)
    if out.dtype != torch.bfloat16 or out.numel() < n_elements:
        raise RuntimeError("`out` must be a bfloat16 tensor with at least n_elements elements")
    _lib.check(_lib.lib.df11_decode(
        luts.data_ptr(), encoded_exponent.data_ptr(), sign_mantissa.data_ptr(),
        output_positions.data_ptr(), gaps.data_ptr(), out.data_ptr(),
        luts.shape[0], encoded_exponent.numel(), n_elements, int(max_block_elems),
        status.data_ptr() if status is not None else None, device.index, _stream(device)))
    return out


def aux_bytes(n_bytes: int, n_elements: int) -> int:
    """Size in bytes of the auxiliary buffer `prepare` fills for a unit of these sizes."""
    return _lib.check(_lib.lib.df11_aux_bytes(int(n_bytes), int(n_elements)))


def prepare(luts: torch.Tensor, encoded_exponent: torch.Tensor, output_positions: torch.Tensor,
            gaps: torch.Tensor, n_elements: int, aux: Optional[torch.Tensor] = None,
            status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Fill (allocating if needed) the auxiliary buffer that ``decode_prepared`` reads."""
    device = _require_cuda(("encoded_exponent",), luts=luts, encoded_exponent=encoded_exponent,
                           output_positions=output_positions, gaps=gaps, aux=aux, status=status)
    need = aux_bytes(encoded_exponent.numel(), n_elements)
    if aux is None:
        aux = torch.empty(need, dtype=torch.uint8, device=device)
    _lib.check(_lib.lib.df11_prepare(
        luts.data_ptr(), encoded_exponent.data_ptr(), output_positions.data_ptr(), gaps.data_ptr(),
        aux.data_ptr(), aux.numel() * aux.element_size(), luts.shape[0], encoded_exponent.numel(),
        int(n_elements), status.data_ptr() if status is not None else None, device.index, _stream(device)))
    return aux


def decode_prepared(luts: torch.Tensor, encoded_exponent: torch.Tensor, sign_mantissa: torch.Tensor,
                    output_positions: torch.Tensor, gaps: torch.Tensor, aux: torch.Tensor,
                    out: Optional[torch.Tensor] = None, max_block_elems: int = 0,
                    status: Optional[torch.Tensor] = None, ctas_per_sm: int = 0) -> torch.Tensor:
    """Single-pass decode using the buffer made by ``prepare`` for the same unit.

    ``ctas_per_sm`` > 0 caps the CTAs the persistent kernel places on an SM, for a launch that
    should leave room for kernels of other streams (``df11_decode_prepared_shared``)."""
    device = _require_cuda(luts=luts, encoded_exponent=encoded_exponent, sign_mantissa=sign_mantissa,
                           output_positions=output_positions, gaps=gaps, aux=aux, out=out, status=status)
    n_elements = sign_mantissa.numel()
    if out is None:
        out = torch.empty(n_elements, dtype=torch.bfloat16, device=device)
    if out.dtype != torch.bfloat16 or out.numel() < n_elements:
        raise RuntimeError("`out` must be a bfloat16 tensor with at least n_elements elements")
    if ctas_per_sm:
        _lib.check(_lib.lib.df11_decode_prepared_shared(
            luts.data_ptr(), encoded_exponent.data_ptr(), sign_mantissa.data_ptr(),
            output_positions.data_ptr(), gaps.data_ptr(), aux.data_ptr(), out.data_ptr(),
            luts.shape[0], encoded_exponent.numel(), n_elements, int(ctas_per_sm),
            status.data_ptr() if status is not None else None, device.index, _stream(device)))
        return out
    _lib.check(_lib.lib.df11_decode_prepared(
        luts.data_ptr(), encoded_exponent.data_ptr(), sign_mantissa.data_ptr(),
        output_positions.data_ptr(), gaps.data_ptr(), aux.data_ptr(), out.data_ptr(),
        luts.shape[0], encoded_exponent.numel(), n_elements, int(max_block_elems),
        status.data_ptr() if status is not None else None, device.index, _stream(device)))
    return out


def seek_interval(elements: int = 0) -> int:
    """Elements per seek point of the prepared form (16 or 32), process-wide; a non-zero argument
    sets it.  Buffers made by ``prepare`` are only valid under the setting they were made under."""
    return _lib.check(_lib.lib.df11_seek_interval(int(elements)))


def chunk_elements() -> int:
    """Elements per independently decodable chunk of the prepared form (32 seek intervals)."""
    return 32 * seek_interval()


def decode_range_prepared(luts: torch.Tensor, encoded_exponent: torch.Tensor, sign_mantissa: torch.Tensor,
                          aux: torch.Tensor, first_element: int, range_elements: int, out: torch.Tensor,
                          status: Optional[torch.Tensor] = None, ctas_per_sm: int = 0) -> torch.Tensor:
    """Decompress elements ``[first_element, first_element + range_elements)`` of a prepared unit into
    ``out[:range_elements]``.  The range starts on a multiple of ``chunk_elements()`` and ends on one
    or at the end of the unit.  ``ctas_per_sm`` > 0 caps the CTAs per SM, as in ``decode_prepared``."""
    device = _require_cuda(luts=luts, encoded_exponent=encoded_exponent, sign_mantissa=sign_mantissa,
                           aux=aux, out=out, status=status)
    if out.dtype != torch.bfloat16 or out.numel() < range_elements:
        raise RuntimeError("`out` must be a bfloat16 tensor with at least range_elements elements")
    if ctas_per_sm:
        _lib.check(_lib.lib.df11_decode_range_prepared_shared(
            luts.data_ptr(), encoded_exponent.data_ptr(), sign_mantissa.data_ptr(), aux.data_ptr(),
            int(first_element), int(range_elements), out.data_ptr(), luts.shape[0], encoded_exponent.numel(),
            sign_mantissa.numel(), int(ctas_per_sm), status.data_ptr() if status is not None else None,
            device.index, _stream(device)))
        return out[:range_elements]
    _lib.check(_lib.lib.df11_decode_range_prepared(
        luts.data_ptr(), encoded_exponent.data_ptr(), sign_mantissa.data_ptr(), aux.data_ptr(),
        int(first_element), int(range_elements), out.data_ptr(), luts.shape[0], encoded_exponent.numel(),
        sign_mantissa.numel(), status.data_ptr() if status is not None else None, device.index, _stream(device)))
    return out[:range_elements]


def decode_rows_prepared(luts: torch.Tensor, encoded_exponent: torch.Tensor, sign_mantissa: torch.Tensor,
                         aux: torch.Tensor, rows: torch.Tensor, row_elements: int,
                         out: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Decompress only the given rows of a unit viewed as ``[n_elements / row_elements, row_elements]``.

    ``rows`` is an int64 CUDA tensor; the result has one row per entry, in that order.  Needs the
    buffer made by ``prepare`` and a row length that is a multiple of ``chunk_elements()``.
    ``encoded_exponent`` and ``sign_mantissa`` may be pinned host tensors (the kernel then reads
    just those rows' bytes over PCIe), as may ``encoded_exponent`` in ``prepare``."""
    device = _require_cuda(("encoded_exponent", "sign_mantissa"), luts=luts, encoded_exponent=encoded_exponent,
                           sign_mantissa=sign_mantissa, aux=aux, rows=rows, out=out, status=status)
    if rows.dtype != torch.int64:
        raise RuntimeError("`rows` must be an int64 tensor")
    n_rows = rows.numel()
    if out is None:
        out = torch.empty(n_rows * row_elements, dtype=torch.bfloat16, device=device)
    if out.dtype != torch.bfloat16 or out.numel() < n_rows * row_elements:
        raise RuntimeError("`out` must be a bfloat16 tensor with at least n_rows * row_elements elements")
    _lib.check(_lib.lib.df11_decode_rows_prepared(
        luts.data_ptr(), encoded_exponent.data_ptr(), sign_mantissa.data_ptr(), aux.data_ptr(),
        rows.data_ptr(), n_rows, int(row_elements), out.data_ptr(), luts.shape[0], encoded_exponent.numel(),
        sign_mantissa.numel(), status.data_ptr() if status is not None else None, device.index, _stream(device)))
    return out[:n_rows * row_elements].view(n_rows, row_elements)


_gemv_scratch = {}          # device -> float32 tensor for the partial sums


def _gemv_workspace(device: torch.device, n_rows: int, in_features: int, m: int) -> torch.Tensor:
    need = _lib.check(_lib.lib.df11_gemv_partials_bytes(n_rows, in_features, m)) // 4
    buf = _gemv_scratch.get(device)
    if buf is None or buf.numel() < need:
        buf = _gemv_scratch[device] = torch.empty(max(need, 1 << 20), dtype=torch.float32, device=device)
    return buf


def gemv_prepared(luts: torch.Tensor, encoded_exponent: torch.Tensor, sign_mantissa: torch.Tensor,
                  aux: torch.Tensor, x: torch.Tensor, first_element: int, n_rows: int, in_features: int,
                  bias: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                  status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x @ W.T (+ bias)`` for the ``[n_rows, in_features]`` matrix that starts at element
    ``first_element`` of a prepared unit, decoding the weights on the fly (never written).

    ``x`` is a contiguous BF16 tensor of 1..4 rows of ``in_features``; the result is
    ``[rows, n_rows]`` BF16.  Launches on one device share a scratch area, so they must be
    queued on one stream (or otherwise kept from overlapping)."""
    device = _require_cuda(luts=luts, encoded_exponent=encoded_exponent, sign_mantissa=sign_mantissa, aux=aux,
                           x=x, bias=bias, out=out, status=status)
    if x.dtype != torch.bfloat16 or (bias is not None and bias.dtype != torch.bfloat16):
        raise RuntimeError("`x` and `bias` must be bfloat16")
    if x.numel() % in_features:
        raise RuntimeError("`x` does not hold whole rows of in_features elements")
    m = x.numel() // in_features
    if out is None:
        out = torch.empty(m, n_rows, dtype=torch.bfloat16, device=device)
    if out.dtype != torch.bfloat16 or out.numel() < m * n_rows:
        raise RuntimeError("`out` must be a bfloat16 tensor of m * n_rows elements")
    partials = _gemv_workspace(device, n_rows, in_features, m)
    _lib.check(_lib.lib.df11_gemv_prepared(
        luts.data_ptr(), encoded_exponent.data_ptr(), sign_mantissa.data_ptr(), aux.data_ptr(), x.data_ptr(),
        out.data_ptr(), bias.data_ptr() if bias is not None else None, partials.data_ptr(),
        int(first_element), int(n_rows), int(in_features), int(m), luts.shape[0], encoded_exponent.numel(),
        sign_mantissa.numel(), status.data_ptr() if status is not None else None, device.index, _stream(device)))
    return out


# ------------------------------------------------------------------ operators of a generation step
#
# A single-token step launches these once per layer, so the host time of a call counts: each first asks in one
# expression whether everything is as it should be (some 3 microseconds), and only if not goes through the checks
# one by one, which name what is wrong.
_ELEMENT_TYPES = {torch.bfloat16: _lib.TYPE_BF16, torch.float16: _lib.TYPE_FP16, torch.float32: _lib.TYPE_FP32}
_LEAST, _MOST = 5e-324, 1.7976931348623157e308
KV_FORMATS = {torch.int8: _lib.KV_INT8, torch.float8_e4m3fn: _lib.KV_E4M3}


def _activation(name: str, t: torch.Tensor, shape, device: Optional[torch.device]) -> torch.device:
    """Checks of a ``[batch, heads, tokens, head_dim]`` activation: on ``device``, BF16 or FP16, no gradient
    asked for, any strides as long as the last dimension is contiguous."""
    if not t.is_cuda:
        raise RuntimeError(f"df11 kernels need CUDA tensors; `{name}` is on {t.device}")
    if device is not None and t.device != device:
        raise RuntimeError(f"`{name}` is on {t.device}, expected {device}")
    if t.dtype not in (torch.bfloat16, torch.float16):
        raise RuntimeError(f"`{name}` must be bfloat16 or float16, not {t.dtype}")
    if t.dim() != 4 or (shape is not None and any(want is not None and have != want for have, want in zip(t.shape, shape))):
        raise RuntimeError(f"`{name}` has shape {tuple(t.shape)}, expected {shape or '[batch, heads, tokens, head_dim]'}")
    if t.numel() and t.stride(3) != 1:
        raise RuntimeError(f"the last dimension of `{name}` must be contiguous")
    if t.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"`{name}` requires a gradient, which this inference operator does not have; "
                           "call it under torch.no_grad()")
    return t.device


def _cache(k_codes: torch.Tensor, k_scales: torch.Tensor, v_codes: torch.Tensor, v_scales: torch.Tensor):
    """Checks of the four tensors of a quantised cache; returns (device, format, batch, heads, slots, head_dim)."""
    device = _require_cuda(k_codes=k_codes, k_scales=k_scales, v_codes=v_codes, v_scales=v_scales)
    if k_codes.dtype not in KV_FORMATS or v_codes.dtype != k_codes.dtype:
        raise RuntimeError("`k_codes` and `v_codes` must both be int8 or both be float8_e4m3fn")
    if k_codes.dim() != 4 or v_codes.shape != k_codes.shape:
        raise RuntimeError("`k_codes` and `v_codes` must be [batch, kv_heads, max_slots, head_dim], of one shape")
    for name, t in (("k_scales", k_scales), ("v_scales", v_scales)):
        if t.dtype != torch.float32 or t.shape != k_codes.shape[:3]:
            raise RuntimeError(f"`{name}` must be float32 [batch, kv_heads, max_slots]")
    return (device, KV_FORMATS[k_codes.dtype], *k_codes.shape)


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream_at(index: int) -> int:
    """The current stream of CUDA device ``index``, without making a stream object where torch allows it."""
    return _raw_stream(index) if _raw_stream is not None else torch.cuda.current_stream(index).cuda_stream


def _cache_fits(at: int, k_codes: torch.Tensor, k_scales: torch.Tensor, v_codes: torch.Tensor, v_scales: torch.Tensor, shape) -> bool:
    dtype, rows = k_codes.dtype, shape[:3]
    return (at >= 0 and len(shape) == 4 and dtype in KV_FORMATS and v_codes.dtype == dtype and v_codes.shape == shape
            and k_scales.shape == rows and v_scales.shape == rows and k_scales.dtype == torch.float32
            and v_scales.dtype == torch.float32 and v_codes.get_device() == at and k_scales.get_device() == at
            and v_scales.get_device() == at and k_codes.is_contiguous() and v_codes.is_contiguous()
            and k_scales.is_contiguous() and v_scales.is_contiguous())


def _indices_fit(at: int, t: torch.Tensor, batch: int) -> bool:
    return t.get_device() == at and t.dtype == torch.int64 and t.is_contiguous() and t.numel() in (1, batch)


def _per_sequence(name: str, t: torch.Tensor, batch: int, device: torch.device) -> torch.Tensor:
    _require_cuda(**{name: t})
    if t.device != device:
        raise RuntimeError(f"`{name}` is on {t.device}, expected {device}")
    if t.dtype != torch.int64 or t.numel() not in (1, batch):
        raise RuntimeError(f"`{name}` must be an int64 tensor of 1 or {batch} elements")
    return t


def kv_append(k: torch.Tensor, v: torch.Tensor, k_codes: torch.Tensor, k_scales: torch.Tensor, v_codes: torch.Tensor,
              v_scales: torch.Tensor, positions: torch.Tensor, status: Optional[torch.Tensor] = None) -> None:
    """Quantises new keys and values into the cache: token ``i`` of sequence ``b`` goes to slot ``positions[b] + i``.

    ``k``, ``v``: ``[batch, kv_heads, tokens, head_dim]`` BF16 or FP16, any strides as long as the last dimension is
    contiguous.  ``k_codes``, ``v_codes``: ``[batch, kv_heads, max_slots, head_dim]`` int8 or float8_e4m3fn -- the
    dtype is the format --, ``k_scales``, ``v_scales``: float32 ``[batch, kv_heads, max_slots]``; ``head_dim`` is a
    multiple of 16, at most 256.  A row ``x`` of largest magnitude ``a`` gets ``scale = a / 127`` (e4m3: ``a / 448``)
    and stands for ``code * scale``, with the code nearest to ``x / scale`` (ties to even); a row with an infinity or
    a NaN stands for NaNs.  ``positions``: int64, one per sequence or one for all.  Tokens whose slot the cache does not
    have are left out and set ``STATUS_BAD_POSITIONS`` in ``status``."""
    shape, at = k_codes.shape, k_codes.get_device()
    if not (_cache_fits(at, k_codes, k_scales, v_codes, v_scales, shape) and _indices_fit(at, positions, shape[0])
            and k.get_device() == at and v.get_device() == at and k.shape == v.shape and k.dim() == 4
            and k.shape[:2] == shape[:2] and k.shape[3] == shape[3] and (k.dtype == torch.bfloat16 or k.dtype == torch.float16)
            and v.dtype == k.dtype and not (k.requires_grad or v.requires_grad)
            and (status is None or (status.get_device() == at and status.dtype == torch.int32))
            and k.stride(3) == 1 and v.stride(3) == 1):
        device, _, batch, heads, _, dim = _cache(k_codes, k_scales, v_codes, v_scales)
        _activation("k", k, (batch, heads, None, dim), device)
        _activation("v", v, (batch, heads, k.shape[2], dim), device)
        if v.dtype != k.dtype:
            raise RuntimeError("`k` and `v` must have one dtype")
        _per_sequence("positions", positions, batch, device)
        _require_cuda(k_codes=k_codes, status=status)
        if status is not None and status.dtype != torch.int32:
            raise RuntimeError("`status` must be an int32 tensor")
    batch, heads, slots, dim = shape
    tokens = k.shape[2]
    if not k.numel():
        return
    ks, vs = k.stride(), v.stride()
    rc = _lib.lib.df11_kv_append(
        k.data_ptr(), v.data_ptr(), ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], k_codes.data_ptr(), k_scales.data_ptr(),
        v_codes.data_ptr(), v_scales.data_ptr(), positions.data_ptr(), positions.numel(), batch, heads, tokens, dim,
        slots, _ELEMENT_TYPES[k.dtype], KV_FORMATS[k_codes.dtype], status.data_ptr() if status is not None else None, at,
        _stream_at(at))
    if rc:
        _lib.check(rc)


def kv_read(k_codes: torch.Tensor, k_scales: torch.Tensor, v_codes: torch.Tensor, v_scales: torch.Tensor, first_slot: int,
            n_slots: int, dtype: torch.dtype = torch.bfloat16, out=None):
    """Slots ``[first_slot, first_slot + n_slots)`` of every sequence as ``(k, v)``, each
    ``[batch, kv_heads, n_slots, head_dim]`` in ``dtype`` (BF16 or FP16): ``code * scale`` in fp32, rounded once.
    ``out`` may hold the two contiguous tensors to fill."""
    cache, at = k_codes.shape, k_codes.get_device()
    if not _cache_fits(at, k_codes, k_scales, v_codes, v_scales, cache):
        _cache(k_codes, k_scales, v_codes, v_scales)
    batch, heads, slots, dim = cache
    if dtype not in (torch.bfloat16, torch.float16):
        raise RuntimeError(f"`dtype` must be bfloat16 or float16, not {dtype}")
    first_slot, n_slots = int(first_slot), int(n_slots)
    if first_slot < 0 or n_slots < 0 or first_slot + n_slots > slots:
        raise RuntimeError(f"slots {first_slot} .. {first_slot + n_slots} are not in a cache of {slots}")
    shape = (batch, heads, n_slots, dim)
    if out is None:
        k = torch.empty(shape, dtype=dtype, device=k_codes.device)
        v = torch.empty(shape, dtype=dtype, device=k_codes.device)
    else:
        k, v = out
        _require_cuda(k_codes=k_codes, k=k, v=v)
        if any(t.dtype != dtype or tuple(t.shape) != shape for t in (k, v)):
            raise RuntimeError(f"`out` must be two {dtype} tensors of shape {shape}")
    if k.numel():
        rc = _lib.lib.df11_kv_read(
            k_codes.data_ptr(), k_scales.data_ptr(), v_codes.data_ptr(), v_scales.data_ptr(), k.data_ptr(), v.data_ptr(),
            batch, heads, slots, dim, first_slot, n_slots, _ELEMENT_TYPES[dtype], KV_FORMATS[k_codes.dtype], at,
            _stream_at(at))
        if rc:
            _lib.check(rc)
    return k, v


def kv_attention(q: torch.Tensor, k_codes: torch.Tensor, k_scales: torch.Tensor, v_codes: torch.Tensor,
                 v_scales: torch.Tensor, lengths: torch.Tensor, first: Optional[torch.Tensor] = None,
                 scale: Optional[float] = None, window: int = 0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of a few new tokens over a quantised cache, which is read in its 8-bit form.

    ``q``: ``[batch, heads, queries, head_dim]`` BF16 or FP16, any strides as long as the last dimension is contiguous;
    head ``h`` reads the keys of head ``h // (heads // kv_heads)``.  The cache is described at ``kv_append``.
    ``lengths``: int64, one per sequence or one for all: the filled slots, the new tokens' included, so that query ``i``
    stands at ``p = length - queries + i`` and sees slots ``max(first, p - window + 1) .. p`` (``window`` 0: from
    ``first``, which is 0 when it is not given; left padding lies before it).  ``scale`` defaults to
    ``head_dim ** -0.5``.  The result is ``[batch, queries, heads, head_dim]`` in ``q``'s dtype, as the projection that
    follows wants it; a query that sees nothing gives zeros.  Any number of queries works; what the kernel is made for
    is one to some sixteen rows per key head (a long prompt is better read back with ``kv_read``).
    Working memory is allocated per call, so calls may overlap on different streams."""
    cache, at, shape = k_codes.shape, k_codes.get_device(), q.shape
    if not (_cache_fits(at, k_codes, k_scales, v_codes, v_scales, cache) and _indices_fit(at, lengths, cache[0])
            and (first is None or _indices_fit(at, first, cache[0])) and q.get_device() == at and len(shape) == 4
            and shape[0] == cache[0] and shape[3] == cache[3] and (q.dtype == torch.bfloat16 or q.dtype == torch.float16)
            and not q.requires_grad and q.stride(3) == 1):
        device, _, batch, _, _, dim = _cache(k_codes, k_scales, v_codes, v_scales)
        _activation("q", q, (batch, None, None, dim), device)
        _per_sequence("lengths", lengths, batch, device)
        if first is not None:
            _per_sequence("first", first, batch, device)
    batch, kv_heads, slots, dim = cache
    heads, queries = shape[1], shape[2]
    if heads < 1 or heads % kv_heads:
        raise RuntimeError(f"{heads} query heads on {kv_heads} key heads")
    window = int(window)
    if window < 0:
        raise RuntimeError("`window` must not be negative")
    if out is None:
        out = torch.empty((batch, queries, heads, dim), dtype=q.dtype, device=q.device)
    else:
        _require_cuda(k_codes=k_codes, out=out)
        if out.dtype != q.dtype or tuple(out.shape) != (batch, queries, heads, dim):
            raise RuntimeError(f"`out` must be a {q.dtype} tensor of shape {(batch, queries, heads, dim)}")
    if not q.numel():
        return out
    need = _lib.lib.df11_kv_attention_workspace_bytes(batch, heads, kv_heads, queries, dim, slots, window)
    if need < 0:
        _lib.check(need)
    workspace = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
    qs = q.stride()
    rc = _lib.lib.df11_kv_attention(
        q.data_ptr(), qs[0], qs[1], qs[2], k_codes.data_ptr(), k_scales.data_ptr(), v_codes.data_ptr(), v_scales.data_ptr(),
        lengths.data_ptr(), lengths.numel(), first.data_ptr() if first is not None else None,
        first.numel() if first is not None else 0, out.data_ptr(), workspace.data_ptr() if need else None, need, batch,
        heads, kv_heads, queries, dim, slots, window, dim ** -0.5 if scale is None else scale,
        _ELEMENT_TYPES[q.dtype], KV_FORMATS[k_codes.dtype], at, _stream_at(at))
    if rc:
        _lib.check(rc)
    return out


def sample(logits: torch.Tensor, uniform: torch.Tensor, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0,
           out: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One token per row of ``logits`` (``[rows, vocab]`` BF16, FP16 or FP32; rows may lie apart), int64 ``[rows]``.

    ``uniform``: float32 ``[rows]`` in [0, 1), the only randomness.  The settings are numbers, or tensors of one entry
    per row (float32; ``top_k`` int32).  The tokens are ordered by logit, descending, equal ones by index: ``top_k``
    keeps the first so many (0: all), ``top_p`` those before which less than ``top_p`` of the mass that ``top_k`` left
    lies (1: all), ``min_p`` those with at least ``min_p`` of the largest probability (0: all).  The result is the lowest
    index at which the running mass of the kept tokens, in index order, exceeds ``uniform`` times their whole mass.
    ``temperature`` 0 is arg-max, the lowest index among equals.  NaN and -inf are never drawn; a row of nothing else
    gives 0 and sets ``STATUS_EMPTY_ROW`` in ``status``."""
    if not logits.is_cuda:
        raise RuntimeError(f"df11 kernels need CUDA tensors; `logits` is on {logits.device}")
    if logits.dim() != 2 or logits.shape[1] < 1 or logits.dtype not in _ELEMENT_TYPES:
        raise RuntimeError("`logits` must be [rows, vocab] in bfloat16, float16 or float32")
    at, (rows, vocab) = logits.get_device(), logits.shape
    stride = logits.stride()
    if vocab > 1 and stride[1] != 1:
        raise RuntimeError("the rows of `logits` must be contiguous")

    def fits(t, dtype):
        return t.get_device() == at and t.dtype == dtype and t.numel() == rows and t.is_contiguous()

    if not fits(uniform, torch.float32):
        raise RuntimeError(f"`uniform` must be a contiguous float32 tensor of {rows} elements on {logits.device}")
    if out is None:
        out = torch.empty(rows, dtype=torch.int64, device=logits.device)
    elif not fits(out, torch.int64):
        raise RuntimeError(f"`out` must be a contiguous int64 tensor of {rows} elements on {logits.device}")
    if status is not None and (status.get_device() != at or status.dtype != torch.int32):
        raise RuntimeError(f"`status` must be an int32 tensor on {logits.device}")
    args = []
    for name, value, dtype, low, high in (("temperature", temperature, torch.float32, 0, _MOST), ("top_k", top_k, torch.int32, 0, 2 ** 31 - 1),
                                          ("top_p", top_p, torch.float32, _LEAST, 1), ("min_p", min_p, torch.float32, 0, 1)):
        if isinstance(value, torch.Tensor):
            if not fits(value, dtype):
                raise RuntimeError(f"`{name}` must be a number or a contiguous {dtype} tensor of {rows} elements on {logits.device}")
            args.append(value.data_ptr())
            args.append(0)
        else:
            if not low <= value <= high:
                raise RuntimeError(f"`{name}` = {value} is out of range")
            args.append(None)
            args.append(int(value) if name == "top_k" else float(value))
    if rows:
        rc = _lib.lib.df11_sample(
            logits.data_ptr(), stride[0], _ELEMENT_TYPES[logits.dtype], rows, vocab, uniform.data_ptr(), *args,
            out.data_ptr(), status.data_ptr() if status is not None else None, at, _stream_at(at))
        if rc:
            _lib.check(rc)
    return out
