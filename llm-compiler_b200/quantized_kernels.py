"""Python wrappers over the C ABI for serving in 8 bits (include/b200_serve.h, "Serving in 8 bits"): a paged KV cache of
8-bit codes with a scale for each block of tokens and KV head, copies of cache blocks, rows quantised to 8-bit integers
behind a norm, and projections in 8-bit integers. Same rules as kernels.py: preconditions raise before anything is
launched, launches go to torch's current stream and never synchronise, and there is no fallback to PyTorch.

Short calls are bound by the host, so the wrappers count their steps: arguments are packed into the ABI's structs by one
struct.pack (0.7 us; 27 ctypes arguments take 3.8), outputs are made like an input where they are."""

from __future__ import annotations

import functools
import struct
from typing import List, Optional, Sequence, Tuple, Union

import torch

from . import _lib
from .kernels import (_DTYPE_CODES, _EPILOGUES, _RUNTIMES, DeviceRuntime, _check, _code, _dense, _guard_current_device,
                      _stream, runtime)

# (looked up at every call otherwise)
_BFLOAT16, _FLOAT16, _FLOAT32, _INT32, _INT64 = torch.bfloat16, torch.float16, torch.float32, torch.int32, torch.int64

# The formats of a cache in 8 bits: the code of the C ABI.
CACHE_CODES = {torch.int8: _lib.I8, torch.float8_e4m3fn: _lib.E4M3}
ATTENTION_HEAD_DIMS = (64, 128, 256)
MAX_K = 131056  # (a sum of that many products of two 8-bit integers stays below 2^31)

# The ABI's structs: pointers, 64-bit integers, doubles.
_STORE_CALL = struct.Struct("=9Q17q").pack
_ATTENTION_CALL = struct.Struct("=11Q17qd").pack
_ROWS_CALL = struct.Struct("=6Q5qd").pack
_LINEAR_CALL = struct.Struct("=8Q5q").pack
_POOLS = [struct.Struct(f"={3 * count}Q").pack for count in range(_lib.MAX_COPY_POOLS + 1)]


def _runtime_of(first: torch.Tensor, *others: Optional[torch.Tensor]) -> DeviceRuntime:
    """The runtime of the operands' GPU, which is the current one; anything else is refused."""

    try:
        index = first.get_device()
        for tensor in others:
            if tensor is not None and tensor.get_device() != index:
                raise ValueError("all operands must live on the same CUDA device")
    except AttributeError as error:
        raise ValueError("operands must be CUDA tensors") from error
    if index < 0:
        raise ValueError("the B200 backend only runs CUDA tensors (there is no CPU fallback)")
    if index != torch._C._cuda_getDevice():
        _guard_current_device(first.device)
    return _RUNTIMES.get(index) or runtime(first.device)


def _cache_code(dtype: torch.dtype) -> int:
    try:
        return CACHE_CODES[dtype]
    except KeyError as error:
        raise ValueError(f"a cache in 8 bits holds int8 or float8_e4m3fn, not {dtype}") from error


def _check_cache(key_pool: torch.Tensor, value_pool: torch.Tensor, key_scales: torch.Tensor, value_scales: torch.Tensor,
                 block_table: torch.Tensor, batch: int) -> Tuple[int, int, int, int, int]:
    """(blocks, kv heads, block size, head dim, columns of the table) of a cache whose parts fit together."""

    shape = key_pool.shape
    if len(shape) != 4 or value_pool.shape != shape or not key_pool.is_contiguous() or not value_pool.is_contiguous() or \
            key_pool.dtype is not value_pool.dtype:
        raise ValueError("KV pools must be contiguous blocks x H x block_size x D tensors of one shape and dtype")
    per_block = key_scales.shape
    if per_block != shape[:2] or value_scales.shape != per_block or key_scales.dtype is not _FLOAT32 or \
            value_scales.dtype is not _FLOAT32 or not key_scales.is_contiguous() or not value_scales.is_contiguous():
        raise ValueError("scales must be contiguous float32 blocks x H tensors")
    table_shape = block_table.shape
    if block_table.dtype is not _INT32 or len(table_shape) != 2 or table_shape[0] != batch or not block_table.is_contiguous():
        raise ValueError("block_table must be a contiguous int32 B x max_blocks tensor")
    return (*shape, table_shape[1])


def b200_paged_kv_store_8bit(key_pool: torch.Tensor, value_pool: torch.Tensor, key_scales: torch.Tensor,
                             value_scales: torch.Tensor, block_table: torch.Tensor, key: torch.Tensor,
                             value: torch.Tensor, positions: torch.Tensor) -> None:
    """serve.kv.store into a paged cache in 8 bits, in place, one launch: the rows of key / value (B x H x T x D, bf16 or
    fp16, any strides) become codes of their blocks at positions[b] .. positions[b] + T - 1. A block's scale is the largest
    magnitude it has been given / 127 (int8) or / 448 (float8_e4m3fn); where a new row raises it, the rows in front of it
    are rounded anew to the larger scale. A block that is entered at its first row forgets what it held.

    Pools are blocks x H x block_size x D, scales float32 blocks x H, the table int32 B x max_blocks. No block may belong
    to two sequences of one call."""

    rt = _runtime_of(key_pool, value_pool, key_scales, value_scales, block_table, key, value, positions)
    if key.ndim != 4 or key.shape != value.shape or key.dtype != value.dtype:
        raise ValueError("key/value must be B x H x T x D tensors of one shape and dtype")
    batch, heads, tokens, dim = key.shape
    blocks, pool_heads, block_size, pool_dim, columns = _check_cache(key_pool, value_pool, key_scales, value_scales,
                                                                     block_table, batch)
    if heads != pool_heads or dim != pool_dim:
        raise ValueError("key/value heads or head_dim do not match the pools")
    dtype = key.dtype
    if dtype is not _BFLOAT16 and dtype is not _FLOAT16:
        raise ValueError(f"key/value must be bfloat16 or float16, not {key.dtype}")
    if dim % 16:
        raise ValueError("head_dim must be a multiple of 16")
    if positions.shape != (batch,) or positions.dtype is not _INT64 or not positions.is_contiguous():
        raise ValueError("positions must be a contiguous int64 batch vector")
    cache = _cache_code(key_pool.dtype)
    if batch == 0 or tokens == 0:
        return
    code = _lib.load().b200_paged_kv_store_8bit(_STORE_CALL(
        key_pool.data_ptr(), value_pool.data_ptr(), key_scales.data_ptr(), value_scales.data_ptr(), block_table.data_ptr(),
        key.data_ptr(), value.data_ptr(), positions.data_ptr(), rt.status.data_ptr(), batch, heads, tokens, dim, blocks,
        block_size, columns, *key.stride(), *value.stride(), _DTYPE_CODES[dtype], cache), _stream())
    if code:
        _check(code, "b200_paged_kv_store_8bit")
    rt.launches += 1


@functools.lru_cache(maxsize=4096)
def _attention_need(batch: int, q_heads: int, kv_heads: int, dim: int, longest: int, split_tokens: int) -> int:
    return int(_lib.load().b200_paged_decode_attention_8bit_workspace_bytes(batch, q_heads, kv_heads, dim, longest,
                                                                            split_tokens))


def b200_paged_decode_attention_8bit(query: torch.Tensor, key_pool: torch.Tensor, value_pool: torch.Tensor,
                                     key_scales: torch.Tensor, value_scales: torch.Tensor, block_table: torch.Tensor,
                                     lengths: torch.Tensor, attention_mask: Optional[torch.Tensor], *, scale: float,
                                     split_tokens: int = 0, max_length_hint: int = 0) -> torch.Tensor:
    """serve.decode_attention over a paged cache in 8 bits: query B x Hq x 1 x D (bf16 or fp16), the first lengths[b]
    entries of each sequence, an additive B x 1 x 1 x S mask or None. Returns B x Hq x 1 x D. Scores, softmax statistics
    and sums are fp32; a sequence without tokens, or with every token masked by -inf, gives NaN. max_length_hint sizes the
    split of the work and bounds nothing."""

    rt = _runtime_of(query, key_pool, value_pool, key_scales, value_scales, block_table, lengths, attention_mask)
    shape, dtype = query.shape, query.dtype
    if len(shape) != 4 or shape[2] != 1:
        raise ValueError("query must be B x H x 1 x D")
    batch, q_heads, _, dim = shape
    blocks, kv_heads, block_size, pool_dim, max_blocks = _check_cache(key_pool, value_pool, key_scales, value_scales,
                                                                      block_table, batch)
    if pool_dim != dim or kv_heads <= 0 or q_heads % kv_heads:
        raise ValueError("query does not match the pools")
    if dtype is not _BFLOAT16 and dtype is not _FLOAT16:
        raise ValueError(f"query must be bfloat16 or float16, not {query.dtype}")
    if dim not in ATTENTION_HEAD_DIMS:
        raise ValueError("head_dim must be 64, 128 or 256")
    if block_size % 32:
        raise ValueError("the block size must be a multiple of 32 tokens")
    if lengths.shape != (batch,) or lengths.dtype is not _INT64 or not lengths.is_contiguous():
        raise ValueError("lengths must be a contiguous int64 batch vector")
    q_batch_stride, q_head_stride, _, q_stride = query.stride()
    if q_stride != 1:
        query = _dense(query)
        q_batch_stride, q_head_stride = q_heads * dim, dim
    mask_pointer, mask_len, mask_stride, mask_code = 0, max_blocks * block_size, 0, _lib.F32
    if attention_mask is not None:
        if attention_mask.ndim != 4 or attention_mask.shape[:3] != (batch, 1, 1):
            raise ValueError("attention_mask must be B x 1 x 1 x S")
        if attention_mask.shape[3] > mask_len or attention_mask.shape[3] <= 0:
            raise ValueError("mask length must be in [1, capacity]")
        mask_len = attention_mask.shape[3]
        if attention_mask.stride(3) != 1:
            attention_mask = _dense(attention_mask)
        mask_pointer, mask_stride, mask_code = attention_mask.data_ptr(), attention_mask.stride(0), _code(attention_mask.dtype)
    cache = _cache_code(key_pool.dtype)
    output = torch.empty_like(query) if query.is_contiguous() else query.new_empty((batch, q_heads, 1, dim))
    if batch == 0:
        return output
    need = _attention_need(batch, q_heads, kv_heads, dim, min(max_length_hint, mask_len) if max_length_hint > 0 else mask_len,
                           split_tokens)
    workspace = rt.own_workspace("decode_attention_8bit", need).data_ptr() if need else 0
    code = _lib.load().b200_paged_decode_attention_8bit(_ATTENTION_CALL(
        query.data_ptr(), key_pool.data_ptr(), value_pool.data_ptr(), key_scales.data_ptr(), value_scales.data_ptr(),
        block_table.data_ptr(), lengths.data_ptr(), mask_pointer, output.data_ptr(), workspace, rt.status.data_ptr(), batch,
        q_heads, kv_heads, dim, blocks, block_size, max_blocks, mask_len, q_batch_stride, q_head_stride, mask_stride, mask_code,
        _DTYPE_CODES[dtype], cache, split_tokens, max_length_hint, need, scale), _stream())
    if code:
        _check(code, "b200_paged_decode_attention_8bit")
    rt.launches += 1
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
    sources, destinations = _block_index(sources, "sources"), _block_index(destinations, "destinations")
    rt = _runtime_of(*pools, *(index for index in (sources, destinations) if isinstance(index, torch.Tensor)))
    layers, blocks = pools[0].shape[:2] if pools[0].ndim >= 2 else (0, 0)
    places: List[int] = []
    for pool in pools:
        shape, size = pool.shape, pool.nbytes
        if size == 0 or len(shape) < 2 or shape[0] != layers or shape[1] != blocks or not pool.is_contiguous():
            raise ValueError("pools must be contiguous layers x blocks x ... tensors that agree in layers and blocks")
        places += (pool.data_ptr(), size // layers, size // (layers * blocks))
    count = len(sources)
    if count != len(destinations):
        raise ValueError("sources and destinations must be of one length")
    if not isinstance(sources, torch.Tensor) and not isinstance(destinations, torch.Tensor):
        if any(not 0 <= i < blocks for i in (*sources, *destinations)):
            raise ValueError(f"block indices must be in [0, {blocks})")
        if len(set(destinations)) != count or set(destinations) & set(sources):
            raise ValueError("destinations must be distinct and none of them a source")
    if count == 0:
        return
    if not isinstance(sources, torch.Tensor):
        sources = torch.tensor(sources, dtype=torch.int32, device=pools[0].device)
    if not isinstance(destinations, torch.Tensor):
        destinations = torch.tensor(destinations, dtype=torch.int32, device=pools[0].device)
    code = _lib.load().b200_copy_kv_blocks(_POOLS[len(pools)](*places), len(pools), sources.data_ptr(),
                                           destinations.data_ptr(), count, layers, blocks, rt.status.data_ptr(), _stream())
    if code:
        _check(code, "b200_copy_kv_blocks")
    rt.launches += 1


def _row_stride(tensor: torch.Tensor) -> Optional[int]:
    """Elements from row to row where `tensor` is a matrix of rows at one distance (leading dimensions merged)."""

    if tensor.is_contiguous():
        return tensor.shape[-1]
    if tensor.ndim == 2 and tensor.stride(1) == 1 and tensor.stride(0) >= tensor.shape[1]:
        return tensor.stride(0)
    return None


def _quantize(tensor: torch.Tensor, residual: Optional[torch.Tensor], weight: Optional[torch.Tensor], epsilon: float,
              what: str):
    rt = _runtime_of(tensor, residual, weight)
    shape, dtype = tensor.shape, tensor.dtype
    if not shape or shape[-1] <= 0:
        raise ValueError("the input must have rows of at least one element")
    hidden = shape[-1]
    code_dtype = _DTYPE_CODES.get(dtype)
    if code_dtype is None:
        _code(dtype)  # (raises)
    weight_pointer = residual_pointer = total_pointer = 0
    if weight is not None:
        if weight.shape != (hidden,) or weight.dtype is not dtype or not weight.is_contiguous():
            raise ValueError("weight must be a contiguous vector of the row length in the input dtype")
        weight_pointer = weight.data_ptr()
    stride = hidden if tensor.is_contiguous() else _row_stride(tensor)
    if stride is None:
        tensor, stride = _dense(tensor), hidden
    like = tensor if stride == hidden else None  # (contiguous: outputs may be made like it)
    residual_stride, total = hidden, None
    if residual is not None:
        if residual.shape != shape or residual.dtype is not dtype:
            raise ValueError("residual must match the input's shape and dtype")
        residual_stride = hidden if residual.is_contiguous() else _row_stride(residual)
        if residual_stride is None:
            residual, residual_stride = _dense(residual), hidden
        total = torch.empty_like(tensor) if like is not None else tensor.new_empty(shape)
        residual_pointer, total_pointer = residual.data_ptr(), total.data_ptr()
    codes = torch.empty_like(tensor, dtype=torch.int8) if like is not None else tensor.new_empty(shape, dtype=torch.int8)
    # (one size in place of a shape: 1 us less)
    scales = tensor.new_empty(shape[0] if len(shape) == 2 else shape[:-1], dtype=_FLOAT32)
    rows = scales.numel()
    if rows == 0:
        return codes, scales, total
    code = _lib.load().b200_quantize_rows_int8(_ROWS_CALL(
        tensor.data_ptr(), residual_pointer, weight_pointer, total_pointer, codes.data_ptr(), scales.data_ptr(), rows, hidden,
        stride, residual_stride, code_dtype, epsilon), _stream())
    if code:
        _check(code, what)
    rt.launches += 1
    return codes, scales, total


def b200_rms_norm_int8(tensor: torch.Tensor, weight: torch.Tensor, *, epsilon: float,
                       residual: Optional[torch.Tensor] = None
                       ) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]:
    """serve.rms_norm with the residual's addition in front and its output in 8-bit integers, one launch: (codes int8,
    scales float32 per row, sum). sum = round(tensor + residual) in the input dtype (None without a residual: the rows
    themselves are normalised); codes * scales stand for the normalised rows, the largest of each row being 127 (less where
    the row's largest, before the norm's factor, is below 127 * 2^-126: a scale that small would lose its bits)."""

    if weight is None:
        raise ValueError("a norm has a weight")
    return _quantize(tensor, residual, weight, epsilon, "b200_rms_norm_int8")


def b200_quantize_rows_int8(tensor: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """(codes int8, scales float32 per row): rows of activations in front of a projection, or a weight's rows, which are its
    output columns. The largest code of a row is 127, or less where its largest magnitude is below 127 * 2^-126."""

    codes, scales, _ = _quantize(tensor, None, None, 0.0, "b200_quantize_rows_int8")
    return codes, scales


def b200_linear_int8(values: torch.Tensor, scales: torch.Tensor, weight: torch.Tensor, weight_scales: torch.Tensor,
                     bias: Optional[torch.Tensor] = None, *, residual: Optional[torch.Tensor] = None,
                     epilogue: str = "none", out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """serve.linear in 8-bit integers: y = (values . weight) scales weight_scales (+ bias), sums exact in 32-bit integers.

    values int8 [..., K] with scales float32 [...], weight int8 N x K with weight_scales float32 [N]; bias, residual and y
    are of out_dtype. epilogue "residual": y + residual; "swiglu": weight holds gate_j and up_j alternating, the result is
    silu(gate) * up with N / 2 columns. One rounding, at the end. K must be a multiple of 16."""

    rt = _runtime_of(values, scales, weight, weight_scales, bias, residual)
    if weight.ndim != 2:
        raise ValueError("weight must be N x K")
    n, k = weight.shape
    shape = values.shape
    if not shape or shape[-1] != k:
        raise ValueError("the last input dimension must equal the weight's K")
    if values.dtype != torch.int8 or weight.dtype != torch.int8:
        raise ValueError("values and weight must be int8")
    leading = shape[:-1]
    if scales.shape != leading or weight_scales.shape != (n,) or scales.dtype != torch.float32 or \
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
    code_dtype = _code(out_dtype)
    bias_pointer = residual_pointer = 0
    if bias is not None:
        if bias.shape != (n,) or bias.dtype != out_dtype or not bias.is_contiguous():
            raise ValueError("bias must be a contiguous vector of N elements in out_dtype")
        bias_pointer = bias.data_ptr()
    output = values.new_empty((*leading, n // 2 if epilogue == "swiglu" else n), dtype=out_dtype)
    if epilogue == "residual":
        if residual is None or residual.shape != output.shape or residual.dtype != out_dtype:
            raise ValueError("residual must match the output shape and dtype")
        residual = _dense(residual)
        residual_pointer = residual.data_ptr()
    elif residual is not None:
        raise ValueError("residual given without the residual epilogue")
    m = scales.numel()
    if m == 0 or n == 0:
        return output
    code = _lib.load().b200_linear_int8(_LINEAR_CALL(
        values.data_ptr(), scales.data_ptr(), weight.data_ptr(), weight_scales.data_ptr(), bias_pointer, residual_pointer,
        output.data_ptr(), rt.status.data_ptr(), m, k, n, code_dtype, _EPILOGUES[epilogue]), _stream())
    if code:
        _check(code, "b200_linear_int8")
    rt.launches += 1
    return output
