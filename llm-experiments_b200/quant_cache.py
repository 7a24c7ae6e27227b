"""A key / value cache held in 4 or 8 bits: quantised as it is written, read back, and attended over as it is.

Stands beside ``kv_cache.py`` and follows it: ``quant_cache_update`` is ``kv_cache_update``, ``quant_cache_gather`` is ``kv_cache_gather``,
``attention_with_quant_cache`` is ``attention_with_kv_cache``, for a cache of ``k_bits`` / ``v_bits`` per element and one bfloat16 scale
per 32 of them (the form is in include/b2kv.h).  At (4, 4) bits and heads of 128 a token takes 144 bytes per key / value head
where a bfloat16 cache takes 512, which is what decoding reads; the reference's cache is fp32 (simple-llm/src/gpu/gpu_kv_cache.py:66-78).

Heads may be grouped (``n_kv_heads`` divides the query heads), several new tokens per sequence are written and attended with in one call
(``tokens``: a prompt's rows; drafted tokens that are looked over together), and scores may be capped, biased by the distance or
limited to a window.  Prompts attend over their own rows with ``flash_attention`` and go into the cache with ``quant_cache_update``.

A decoding loop over several layers writes every layer with ``advance=False`` and attends with ``pending=tokens`` (rows that are written
but not counted yet), and advances with the last layer; a single layer advances as it writes.
"""
from __future__ import annotations

from typing import List, Optional

import torch

from . import _native
from .batch import batch_op_begin, dev_status_ptr, reference_op, validate_buffer_shape_1d, validate_buffer_shape_2d
from .buffers import gpu_buffer_2d_create, gpu_buffer_zerofy
from .kv_cache import dtype_code
from .types import GPUBuffer1D, GPUBuffer2D, GPUContext, QuantKVCache, QuantKVCacheConfig, QuantKVCacheLayer

HEAD_DIMS = (32, 64, 96, 128, 256)
BITS = ((4, 4), (8, 4), (8, 8))
LARGEST = torch.finfo(torch.float32).max
MAX_TOKENS = 64  # new tokens per sequence that attention takes in one call


def quant_cache_create(ctx: GPUContext, config: QuantKVCacheConfig) -> QuantKVCache:
    for name in ("batch_size", "max_seq_len", "n_layers", "n_kv_heads", "head_dim"):
        if getattr(config, name) <= 0:
            raise ValueError(f"{name} must be > 0, got {getattr(config, name)}")
    if config.head_dim not in HEAD_DIMS:
        raise ValueError(f"head_dim {config.head_dim} is not one of {HEAD_DIMS}")
    if (config.k_bits, config.v_bits) not in BITS:
        raise ValueError(f"(k_bits, v_bits) = ({config.k_bits}, {config.v_bits}) is not one of {BITS}")
    dtype_code(config.dtype)
    if config.max_seq_len > 1 << 30:
        raise ValueError(f"max_seq_len must be at most {1 << 30}, got {config.max_seq_len}")
    if config.block_size < 0 or config.n_blocks < 0:
        raise ValueError("block_size and n_blocks must be >= 0")
    B, T, G, D = config.batch_size, config.max_seq_len, config.n_kv_heads, config.head_dim
    block_table, n_blocks, rows = None, 0, B * G * T
    if config.block_size > 0:
        max_blocks = -(-T // config.block_size)
        n_blocks = config.n_blocks or B * max_blocks
        if n_blocks < B * max_blocks:
            raise ValueError(f"n_blocks {n_blocks} cannot hold {B} sequences of {max_blocks} blocks")
        # identity placement; callers may overwrite the table with their own allocation
        block_table = torch.arange(B * max_blocks, dtype=torch.int32, device=ctx.device).reshape(B, max_blocks)
        rows = n_blocks * G * config.block_size
    scales = _native.lib.b2kv_qcache_scale_row(D)

    def buffer(cols: int, dtype: torch.dtype) -> GPUBuffer2D:
        made = gpu_buffer_2d_create(ctx, rows, cols, dtype=dtype)
        gpu_buffer_zerofy(ctx, made)
        return made

    layers: List[QuantKVCacheLayer] = [
        QuantKVCacheLayer(k_codes=buffer(D * config.k_bits // 8, torch.uint8), v_codes=buffer(D * config.v_bits // 8, torch.uint8),
                          k_scales=buffer(scales, torch.bfloat16), v_scales=buffer(scales, torch.bfloat16)) for _ in range(config.n_layers)]
    seq_lens = torch.zeros(B, dtype=torch.int32, device=ctx.device) if config.ragged else None
    return QuantKVCache(layers=layers, batch_size=B, max_seq_len=T, current_len=0, n_kv_heads=G, head_dim=D, dtype=config.dtype,
                        k_bits=config.k_bits, v_bits=config.v_bits, seq_lens=seq_lens, block_table=block_table,
                        block_size=config.block_size, n_blocks=n_blocks)


def quant_cache_reset(cache: QuantKVCache) -> None:
    cache.current_len = 0
    if cache.seq_lens is not None:
        cache.seq_lens.zero_()


def quant_cache_set_lengths(cache: QuantKVCache, lens) -> None:
    """Installs per-sequence lengths (host list / array / tensor of B ints)."""
    host = torch.as_tensor(lens, dtype=torch.int32).reshape(cache.batch_size).cpu()
    if int(host.min()) < 0 or int(host.max()) > cache.max_seq_len:
        raise ValueError(f"lengths must lie in [0, {cache.max_seq_len}]")
    if cache.seq_lens is None:
        cache.seq_lens = host.to(cache.layers[0].k_codes.buffer.device)
    else:
        cache.seq_lens.copy_(host, non_blocking=True)
    cache.current_len = int(host.max())


def _layer(cache: QuantKVCache, layer_idx: int):
    """``b2kv_qcache`` of a layer."""
    layers = cache.layers
    if layer_idx < 0 or layer_idx >= len(layers):
        raise ValueError(f"layer_idx {layer_idx} out of range [0, {len(layers)})")
    layer, table, lens = layers[layer_idx], cache.block_table, cache.seq_lens
    return _native.qcache(
        layer.k_codes.buffer.data_ptr(), layer.v_codes.buffer.data_ptr(), layer.k_scales.buffer.data_ptr(), layer.v_scales.buffer.data_ptr(), 0 if table is None else table.data_ptr(), 0 if lens is None else lens.data_ptr(), cache.current_len,
        cache.batch_size, cache.n_kv_heads, cache.head_dim, cache.max_seq_len, 0 if table is None else table.shape[1], cache.block_size,
        cache.n_blocks, cache.k_bits, cache.v_bits, dtype_code(cache.dtype))


def _rows(buffer: GPUBuffer2D, shape, dtype: torch.dtype, name: str) -> int:
    """Checks a buffer of rows; its row pitch."""
    t = buffer.buffer
    if buffer.shape != shape:
        validate_buffer_shape_2d(buffer, shape, name)
    if t.dtype != dtype:
        raise ValueError(f"{name} dtype must match the cache dtype {dtype}")
    if t.is_contiguous():
        return shape[1]
    if t.dim() != 2 or t.stride(1) != 1:
        raise ValueError(f"the elements of a row of {name} must lie next to one another")
    return t.stride(0)


@reference_op("quant_cache_update")
def quant_cache_update(ctx: GPUContext, cache: QuantKVCache, layer_idx: int, new_k: GPUBuffer2D, new_v: GPUBuffer2D, tokens: int = 1,
                       advance: bool = True) -> None:
    """Quantises ``tokens`` rows per sequence (row ``b * tokens + i`` of ``new_k`` and ``new_v``, ``[batch * tokens, kv_heads * head_dim]``,
    rows any multiple of 16 bytes apart) into the places behind what the sequence holds, and counts them unless ``advance`` is off."""
    described = _layer(cache, layer_idx)
    if tokens <= 0:
        raise ValueError(f"tokens must be > 0, got {tokens}")
    if cache.current_len + tokens > cache.max_seq_len:
        raise ValueError(f"Cache is full: current_len={cache.current_len}, tokens={tokens}, max_seq_len={cache.max_seq_len}")
    shape = (cache.batch_size * tokens, cache.n_kv_heads * cache.head_dim)
    ld_k, ld_v = _rows(new_k, shape, cache.dtype, "new_k"), _rows(new_v, shape, cache.dtype, "new_v")
    stream = batch_op_begin(ctx)
    _native.check(_native.lib.b2kv_qcache_write(described, new_k.buffer.data_ptr(), ld_k, new_v.buffer.data_ptr(), ld_v, tokens,
                                                dev_status_ptr(ctx), stream))
    if advance:
        if cache.seq_lens is not None:
            _native.check(_native.lib.b2kv_advance_lengths(cache.seq_lens.data_ptr(), cache.batch_size, tokens, stream))
        cache.current_len += tokens


@reference_op("quant_cache_gather")
def quant_cache_gather(ctx: GPUContext, cache: QuantKVCache, layer_idx: int, which: str = "k", length: Optional[int] = None, last: bool = False,
                       pending: int = 0) -> torch.Tensor:
    """The values ``[B, length, kv_heads, head_dim]`` that one layer's K or V stands for: the first ``length`` tokens of every sequence
    (``None``: ``max_seq_len``), or with ``last`` its last ones; zeros where a sequence has no token.  ``pending`` rows behind the lengths
    count as held."""
    described = _layer(cache, layer_idx)
    if which not in ("k", "v"):
        raise ValueError(f"which must be 'k' or 'v', got {which!r}")
    n = cache.max_seq_len if length is None else int(length)
    if n <= 0 or pending < 0:
        raise ValueError(f"length must be > 0 and pending >= 0, got {n} and {pending}")
    out = torch.empty((cache.batch_size, n, cache.n_kv_heads, cache.head_dim), dtype=cache.dtype, device=cache.layers[layer_idx].k_codes.buffer.device)
    stream = batch_op_begin(ctx)
    _native.check(_native.lib.b2kv_qcache_read(described, 0 if which == "k" else 1, out.data_ptr(), n, int(last), min(pending, cache.max_seq_len), dev_status_ptr(ctx), stream))
    return out


@reference_op("attention_with_quant_cache")
def attention_with_quant_cache(ctx: GPUContext, cache: QuantKVCache, layer_idx: int, q_new: GPUBuffer2D, output: GPUBuffer2D, tokens: int = 1,
                               scale: Optional[float] = None, softcap: float = 0.0, window: int = 0, slopes: Optional[GPUBuffer1D] = None,
                               pending: int = 0) -> None:
    """Attention of the last ``tokens`` tokens of every sequence over the cache: ``q_new`` and ``output`` are ``[batch * tokens, heads *
    head_dim]``, ``heads`` a multiple of the cache's, query row ``b * tokens + i`` standing at place ``n - tokens + i`` of the ``n`` tokens
    of sequence ``b``.  A query at place p sees the tokens t <= p, with ``window`` only those with ``p - t < window``, with the scores
    ``cap(scale * q . k) - slopes[head] * (p - t)``; ``scale`` is ``head_dim ** -0.5`` unless given, ``cap(x) = softcap * tanh(x / softcap)``
    with ``softcap``.  A query that sees nothing gives zeros.  ``pending`` rows that ``quant_cache_update`` wrote without advancing count too."""
    described = _layer(cache, layer_idx)
    if not 1 <= tokens <= MAX_TOKENS:
        raise ValueError(f"tokens must lie in [1, {MAX_TOKENS}], got {tokens}")
    held = cache.current_len + pending
    if pending < 0 or held > cache.max_seq_len:
        raise ValueError(f"pending must lie in [0, {cache.max_seq_len - cache.current_len}], got {pending}")
    if held == 0 and cache.seq_lens is None:  # (with lengths of their own, sequences may be empty)
        raise ValueError("Cache is empty: current_len=0")
    if window < 0:
        raise ValueError(f"window must be >= 0, got {window}")
    if not (softcap == 0 or 1e-30 <= softcap <= LARGEST) or not (scale is None or -LARGEST <= scale <= LARGEST):
        raise ValueError(f"softcap must be 0 or at least 1e-30, and it and scale finite float32 numbers, got {softcap} and {scale}")
    D, columns = cache.head_dim, q_new.shape[1]
    heads = columns // D
    if heads * D != columns or heads == 0 or heads % cache.n_kv_heads != 0:
        raise ValueError(f"q_new has {columns} columns, not a multiple of {cache.n_kv_heads} heads of {D}")
    shape = (cache.batch_size * tokens, columns)
    ld_q, ld_out = _rows(q_new, shape, cache.dtype, "q_new"), _rows(output, shape, cache.dtype, "output")
    if slopes is not None:
        validate_buffer_shape_1d(slopes, heads, "slopes")
        if slopes.buffer.dtype != torch.float32 or not slopes.buffer.is_contiguous():
            raise ValueError("slopes must be contiguous float32")
    args = _native.qcache_attend_args(q_new.buffer.data_ptr(), output.buffer.data_ptr(), 0 if slopes is None else slopes.buffer.data_ptr(),
                                      ld_q, ld_out, heads, tokens, held, pending, min(window, held + tokens), D ** -0.5 if scale is None else scale, softcap)
    stream, lib = batch_op_begin(ctx), _native.lib
    nbytes = lib.b2kv_qcache_attend_workspace_bytes(described, args)
    # Scratch of this call alone, from the stream's (or the capture's) own memory: nothing is shared by calls that run at the same time.
    ws = torch.empty(nbytes, dtype=torch.uint8, device=q_new.buffer.device) if nbytes else None
    rc = lib.b2kv_qcache_attend(described, args, None if ws is None else ws.data_ptr(), nbytes, dev_status_ptr(ctx), stream)
    if rc != 0:
        _native.check(rc)
