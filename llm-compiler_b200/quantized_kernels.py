"""Python wrappers over the C ABI for serving in 8 bits (include/b200_serve.h, "Serving in 8 bits"): a paged KV cache of
8-bit codes with a scale for each block of tokens and KV head, copies of cache blocks, rows quantised to 8-bit integers
behind a norm, and projections in 8-bit integers. Same rules as kernels.py: preconditions raise before anything is
launched, launches go to torch's current stream and never synchronise, and there is no fallback to PyTorch."""

from __future__ import annotations

from typing import List, Optional, Sequence, Tuple, Union

import torch

from . import _lib
from .kernels import (_EPILOGUES, _check, _code, _count, _dense, _ptr, _require_cuda, _stream, runtime)

# The formats of a cache in 8 bits: the code of the C ABI and the largest code.
CACHE_CODES = {torch.int8: _lib.I8, torch.float8_e4m3fn: _lib.E4M3}
MAX_K = 131056  # (a sum of that many products of two 8-bit integers stays below 2^31)


def _cache_code(dtype: torch.dtype) -> int:
    try:
        return CACHE_CODES[dtype]
    except KeyError as error:
        raise ValueError(f"a cache in 8 bits holds int8 or float8_e4m3fn, not {dtype}") from error


def _check_cache(key_pool: torch.Tensor, value_pool: torch.Tensor, key_scales: torch.Tensor, value_scales: torch.Tensor,
                 block_table: torch.Tensor, batch: int) -> Tuple[int, int, int, int]:
    """(blocks, kv heads, block size, head dim) of a cache whose parts fit together."""

    shape = key_pool.shape
    if len(shape) != 4 or value_pool.shape != shape or not key_pool.is_contiguous() or not value_pool.is_contiguous() or \
            key_pool.dtype != value_pool.dtype:
        raise ValueError("KV pools must be contiguous blocks x H x block_size x D tensors of one shape and dtype")
    for scales in (key_scales, value_scales):
        if scales.shape != shape[:2] or scales.dtype != torch.float32 or not scales.is_contiguous():
            raise ValueError("scales must be contiguous float32 blocks x H tensors")
    if block_table.dtype != torch.int32 or block_table.ndim != 2 or block_table.shape[0] != batch or \
            not block_table.is_contiguous():
        raise ValueError("block_table must be a contiguous int32 B x max_blocks tensor")
    return shape


def b200_paged_kv_store_8bit(key_pool: torch.Tensor, value_pool: torch.Tensor, key_scales: torch.Tensor,
                             value_scales: torch.Tensor, block_table: torch.Tensor, key: torch.Tensor,
                             value: torch.Tensor, positions: torch.Tensor) -> None:
    """serve.kv.store into a paged cache in 8 bits, in place, one launch: the rows of key / value (B x H x T x D, bf16 or
    fp16, any strides) become codes of their blocks at positions[b] .. positions[b] + T - 1. A block's scale is the largest
    magnitude it has been given / 127 (int8) or / 448 (float8_e4m3fn); where a new row raises it, the rows in front of it
    are rounded anew to the larger scale. A block that is entered at its first row forgets what it held.

    Pools are blocks x H x block_size x D, scales float32 blocks x H, the table int32 B x max_blocks."""

    device = _require_cuda(key_pool, value_pool, key_scales, value_scales, block_table, key, value, positions)
    if key.ndim != 4 or key.shape != value.shape or key.dtype != value.dtype:
        raise ValueError("key/value must be B x H x T x D tensors of one shape and dtype")
    batch, heads, tokens, dim = key.shape
    blocks, pool_heads, block_size, pool_dim = _check_cache(key_pool, value_pool, key_scales, value_scales, block_table, batch)
    if heads != pool_heads or dim != pool_dim:
        raise ValueError("key/value heads or head_dim do not match the pools")
    if key.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"key/value must be bfloat16 or float16, not {key.dtype}")
    if dim % 16:
        raise ValueError("head_dim must be a multiple of 16")
    if positions.shape != (batch,) or positions.dtype != torch.int64 or not positions.is_contiguous():
        raise ValueError("positions must be a contiguous int64 batch vector")
    if batch == 0 or tokens == 0:
        return
    rt = runtime(device)
    code = _lib.load().b200_paged_kv_store_8bit(
        key_pool.data_ptr(), value_pool.data_ptr(), key_scales.data_ptr(), value_scales.data_ptr(), block_table.data_ptr(),
        key.data_ptr(), value.data_ptr(), positions.data_ptr(), batch, heads, tokens, dim, blocks, block_size,
        block_table.shape[1], _lib.i64_array(key.stride()), _lib.i64_array(value.stride()), _code(key.dtype),
        _cache_code(key_pool.dtype), rt.status.data_ptr(), _stream())
    _check(code, "b200_paged_kv_store_8bit")
    _count(rt)


def b200_paged_decode_attention_8bit(query: torch.Tensor, key_pool: torch.Tensor, value_pool: torch.Tensor,
                                     key_scales: torch.Tensor, value_scales: torch.Tensor, block_table: torch.Tensor,
                                     lengths: torch.Tensor, attention_mask: Optional[torch.Tensor], *, scale: float,
                                     split_tokens: int = 0, max_length_hint: int = 0) -> torch.Tensor:
    """serve.decode_attention over a paged cache in 8 bits: query B x Hq x 1 x D (bf16 or fp16), the first lengths[b]
    entries of each sequence, an additive B x 1 x 1 x S mask or None. Returns B x Hq x 1 x D. Scores, softmax statistics
    and sums are fp32; a sequence without tokens, or with every token masked by -inf, gives NaN."""

    device = _require_cuda(query, key_pool, value_pool, key_scales, value_scales, block_table, lengths, attention_mask)
    if query.ndim != 4 or query.shape[2] != 1:
        raise ValueError("query must be B x H x 1 x D")
    batch, q_heads, _, dim = query.shape
    blocks, kv_heads, block_size, pool_dim = _check_cache(key_pool, value_pool, key_scales, value_scales, block_table, batch)
    if pool_dim != dim or kv_heads <= 0 or q_heads % kv_heads:
        raise ValueError("query does not match the pools")
    if query.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"query must be bfloat16 or float16, not {query.dtype}")
    if dim not in (64, 128, 256):
        raise ValueError("head_dim must be 64, 128 or 256")
    if block_size % 32:
        raise ValueError("the block size must be a multiple of 32 tokens")
    if lengths.shape != (batch,) or lengths.dtype != torch.int64 or not lengths.is_contiguous():
        raise ValueError("lengths must be a contiguous int64 batch vector")
    if query.stride(3) != 1:
        query = _dense(query)
    capacity = block_table.shape[1] * block_size
    mask_len, mask_stride, mask_code = capacity, 0, _lib.F32
    if attention_mask is not None:
        if attention_mask.ndim != 4 or attention_mask.shape[:3] != (batch, 1, 1):
            raise ValueError("attention_mask must be B x 1 x 1 x S")
        mask_len = attention_mask.shape[3]
        if mask_len > capacity or mask_len <= 0:
            raise ValueError("mask length must be in [1, capacity]")
        if attention_mask.stride(3) != 1:
            attention_mask = _dense(attention_mask)
        mask_stride = attention_mask.stride(0)
        mask_code = _code(attention_mask.dtype)
    output = query.new_empty((batch, q_heads, 1, dim))
    if batch == 0:
        return output
    rt = runtime(device)
    library = _lib.load()
    longest = min(max_length_hint, mask_len) if max_length_hint > 0 else mask_len
    need = library.b200_paged_decode_attention_8bit_workspace_bytes(batch, q_heads, kv_heads, dim, longest, split_tokens)
    workspace = rt.own_workspace("decode_attention_8bit", need) if need else None
    code = library.b200_paged_decode_attention_8bit(
        query.data_ptr(), key_pool.data_ptr(), value_pool.data_ptr(), key_scales.data_ptr(), value_scales.data_ptr(),
        block_table.data_ptr(), lengths.data_ptr(), _ptr(attention_mask), output.data_ptr(), batch, q_heads, kv_heads, dim,
        blocks, block_size, block_table.shape[1], mask_len, query.stride(0), query.stride(1), mask_stride, mask_code,
        float(scale), _code(query.dtype), _cache_code(key_pool.dtype), int(split_tokens), int(max_length_hint),
        _ptr(workspace), need, rt.status.data_ptr(), _stream())
    _check(code, "b200_paged_decode_attention_8bit")
    _count(rt)
    return output


def _block_index(index: Union[torch.Tensor, Sequence[int]], what: str) -> Union[torch.Tensor, List[int]]:
    if isinstance(index, torch.Tensor):
        if index.dtype != torch.int32 or index.ndim != 1 or not index.is_contiguous():
            raise ValueError(f"{what} must be a contiguous int32 vector or a list")
        return index
    return [int(i) for i in index]


def b200_copy_kv_blocks(pools: Sequence[torch.Tensor], sources: Union[torch.Tensor, Sequence[int]],
                        destinations: Union[torch.Tensor, Sequence[int]]) -> None:
    """pool[:, destinations[i]] = pool[:, sources[i]] for every pool, in place, one launch: blocks of a paged cache, 8-bit or
    not, copied in every layer. Pools are contiguous layers x blocks x ... tensors (keys, values, their scales) that agree
    in layers and blocks, eight at most. Destinations are distinct and none is among the sources: lists are checked here
    (and copied to the device), int32 device vectors are taken at their word."""

    if not pools or len(pools) > _lib.MAX_COPY_POOLS:
        raise ValueError(f"between one and {_lib.MAX_COPY_POOLS} pools are copied at once")
    device = _require_cuda(*pools)
    layers, blocks = pools[0].shape[:2] if pools[0].ndim >= 2 else (0, 0)
    table = (_lib.BlockPool * len(pools))()
    for entry, pool in zip(table, pools):
        if pool.ndim < 2 or pool.shape[:2] != (layers, blocks) or pool.numel() == 0 or not pool.is_contiguous():
            raise ValueError("pools must be contiguous layers x blocks x ... tensors that agree in layers and blocks")
        size = pool.element_size()
        entry.base, entry.layer_stride, entry.block_bytes = pool.data_ptr(), pool.stride(0) * size, pool.stride(1) * size
    sources, destinations = _block_index(sources, "sources"), _block_index(destinations, "destinations")
    if len(sources) != len(destinations):
        raise ValueError("sources and destinations must be of one length")
    if not isinstance(sources, torch.Tensor) and not isinstance(destinations, torch.Tensor):
        if any(not 0 <= i < blocks for i in (*sources, *destinations)):
            raise ValueError(f"block indices must be in [0, {blocks})")
        if len(set(destinations)) != len(destinations) or set(destinations) & set(sources):
            raise ValueError("destinations must be distinct and none of them a source")
    if len(sources) == 0:
        return
    sources, destinations = (i if isinstance(i, torch.Tensor) else torch.tensor(i, dtype=torch.int32, device=device)
                             for i in (sources, destinations))
    _require_cuda(pools[0], sources, destinations)
    rt = runtime(device)
    code = _lib.load().b200_copy_kv_blocks(table, len(pools), sources.data_ptr(), destinations.data_ptr(),
                                           sources.numel(), layers, blocks, rt.status.data_ptr(), _stream())
    _check(code, "b200_copy_kv_blocks")
    _count(rt)


def _row_stride(tensor: torch.Tensor) -> Optional[int]:
    """Elements from row to row where `tensor` is a matrix of rows at one distance (leading dimensions merged)."""

    if tensor.is_contiguous():
        return tensor.shape[-1]
    if tensor.ndim == 2 and tensor.stride(1) == 1 and tensor.stride(0) >= tensor.shape[1]:
        return tensor.stride(0)
    return None


def _quantize(tensor: torch.Tensor, residual: Optional[torch.Tensor], weight: Optional[torch.Tensor], epsilon: float,
              what: str):
    device = _require_cuda(tensor, residual, weight)
    if tensor.ndim < 1 or tensor.shape[-1] <= 0:
        raise ValueError("the input must have rows of at least one element")
    hidden = tensor.shape[-1]
    if weight is not None and (weight.shape != (hidden,) or weight.dtype != tensor.dtype or not weight.is_contiguous()):
        raise ValueError("weight must be a contiguous vector of the row length in the input dtype")
    stride = _row_stride(tensor)
    if stride is None:
        tensor, stride = _dense(tensor), hidden
    residual_stride, total = hidden, None
    if residual is not None:
        if residual.shape != tensor.shape or residual.dtype != tensor.dtype:
            raise ValueError("residual must match the input's shape and dtype")
        residual_stride = _row_stride(residual)
        if residual_stride is None:
            residual, residual_stride = _dense(residual), hidden
        total = torch.empty(tensor.shape, dtype=tensor.dtype, device=device)
    rows = tensor.numel() // hidden
    codes = torch.empty(tensor.shape, dtype=torch.int8, device=device)
    scales = torch.empty(tensor.shape[:-1], dtype=torch.float32, device=device)
    if rows == 0:
        return codes, scales, total
    rt = runtime(device)
    code = _lib.load().b200_quantize_rows_int8(
        tensor.data_ptr(), _ptr(residual), _ptr(weight), _ptr(total), codes.data_ptr(), scales.data_ptr(), rows, hidden,
        stride, residual_stride, float(epsilon), _code(tensor.dtype), _stream())
    _check(code, what)
    _count(rt)
    return codes, scales, total


def b200_rms_norm_int8(tensor: torch.Tensor, weight: torch.Tensor, *, epsilon: float,
                       residual: Optional[torch.Tensor] = None
                       ) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]:
    """serve.rms_norm with the residual's addition in front and its output in 8-bit integers, one launch: (codes int8,
    scales float32 per row, sum). sum = round(tensor + residual) in the input dtype (None without a residual: the rows
    themselves are normalised); codes * scales stand for the normalised rows, the largest of each row being 127."""

    return _quantize(tensor, residual, weight, epsilon, "b200_rms_norm_int8")


def b200_quantize_rows_int8(tensor: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """(codes int8, scales float32 per row): rows of activations in front of a projection, or a weight's rows, which are its
    output columns."""

    codes, scales, _ = _quantize(tensor, None, None, 0.0, "b200_quantize_rows_int8")
    return codes, scales


def b200_linear_int8(values: torch.Tensor, scales: torch.Tensor, weight: torch.Tensor, weight_scales: torch.Tensor,
                     bias: Optional[torch.Tensor] = None, *, residual: Optional[torch.Tensor] = None,
                     epilogue: str = "none", out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """serve.linear in 8-bit integers: y = (values . weight) scales weight_scales (+ bias), sums exact in 32-bit integers.

    values int8 [..., K] with scales float32 [...], weight int8 N x K with weight_scales float32 [N]; bias, residual and y
    are of out_dtype. epilogue "residual": y + residual; "swiglu": weight holds gate_j and up_j alternating, the result is
    silu(gate) * up with N / 2 columns. One rounding, at the end. K must be a multiple of 16."""

    device = _require_cuda(values, scales, weight, weight_scales, bias, residual)
    if weight.ndim != 2:
        raise ValueError("weight must be N x K")
    n, k = weight.shape
    shape = values.shape
    if not shape or shape[-1] != k:
        raise ValueError("the last input dimension must equal the weight's K")
    if values.dtype != torch.int8 or weight.dtype != torch.int8:
        raise ValueError("values and weight must be int8")
    if scales.shape != shape[:-1] or weight_scales.shape != (n,) or scales.dtype != torch.float32 or \
            weight_scales.dtype != torch.float32:
        raise ValueError("scales must be float32, one per row of values and one per row of weight")
    if not (values.is_contiguous() and weight.is_contiguous() and scales.is_contiguous() and weight_scales.is_contiguous()):
        raise ValueError("values, weight and their scales must be contiguous")
    if k % 16 or k > MAX_K:
        raise ValueError(f"K must be a multiple of 16 and at most {MAX_K}")
    if epilogue not in _EPILOGUES:
        raise ValueError(f"unknown epilogue {epilogue!r}")
    if epilogue == "swiglu" and n % 2:
        raise ValueError("swiglu needs an even number of weight rows")
    if bias is not None and (bias.shape != (n,) or bias.dtype != out_dtype or not bias.is_contiguous()):
        raise ValueError("bias must be a contiguous vector of N elements in out_dtype")
    output = torch.empty((*shape[:-1], n // 2 if epilogue == "swiglu" else n), dtype=out_dtype, device=device)
    if epilogue == "residual":
        if residual is None or residual.shape != output.shape or residual.dtype != out_dtype:
            raise ValueError("residual must match the output shape and dtype")
        residual = _dense(residual)
    elif residual is not None:
        raise ValueError("residual given without the residual epilogue")
    if output.numel() == 0:
        return output
    rt = runtime(device)
    code = _lib.load().b200_linear_int8(
        values.data_ptr(), scales.data_ptr(), weight.data_ptr(), weight_scales.data_ptr(), _ptr(bias), _ptr(residual),
        output.data_ptr(), scales.numel(), k, n, _code(out_dtype), _EPILOGUES[epilogue], rt.status.data_ptr(), _stream())
    _check(code, "b200_linear_int8")
    _count(rt)
    return output
