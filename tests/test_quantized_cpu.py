"""Serving in 8 bits without a GPU: what the C ABI refuses before any launch, what the wrappers refuse, and the block
bookkeeping of fork, release and compact with the copies written down instead of made."""

import struct

import pytest
import torch

import llm_compiler_b200 as b200
from llm_compiler_b200 import _lib, quantized_kernels
from llm_compiler_b200.kv_state import ExecutionError, PagedKVCacheState, QuantizedPagedKVCacheState

FAKE, ODD = 256, 264  # never dereferenced: rejected on the host


def store(pool=FAKE, batch=1, heads=2, tokens=1, dim=64, blocks=4, size=32, columns=2, dtype=_lib.BF16, cache=_lib.I8,
          status=FAKE):
    call = struct.pack("=9Q17q", pool or 0, *[FAKE] * 7, status or 0, batch, heads, tokens, dim, blocks, size, columns,
                       128, 64, 64, 1, 128, 64, 64, 1, dtype, cache)
    return _lib.load().b200_paged_kv_store_8bit(call, None)


def test_store_refusals():
    assert store(pool=None) == store(status=None) == _lib.ERR_BAD_ARGUMENT
    assert store(batch=-1) == store(heads=0) == store(dim=0) == store(blocks=0) == store(columns=0) == _lib.ERR_BAD_ARGUMENT
    assert store(dim=40) == store(dtype=_lib.F32) == store(cache=_lib.BF16) == store(cache=7) == _lib.ERR_UNSUPPORTED
    assert store(pool=ODD) == _lib.ERR_ALIGNMENT
    assert store(batch=70000) == _lib.ERR_TOO_LARGE
    assert store(batch=0) == store(tokens=0) == 0


def attention(query=FAKE, pool=FAKE, mask=0, batch=1, heads=4, kv_heads=2, dim=64, blocks=4, size=32, columns=2,
              mask_len=64, mask_dtype=_lib.F32, dtype=_lib.BF16, cache=_lib.I8, split=0, workspace=0, nbytes=0):
    call = struct.pack("=11Q17qd", query or 0, pool, *[FAKE] * 5, mask, FAKE, workspace, FAKE, batch, heads, kv_heads, dim,
                       blocks, size, columns, mask_len, 256, 64, 0, mask_dtype, dtype, cache, split, 0, nbytes, 0.125)
    return _lib.load().b200_paged_decode_attention_8bit(call, None)


def test_attention_refusals():
    assert attention(query=None) == attention(heads=5) == attention(mask_len=65) == attention(mask_len=0) == \
        attention(split=-1) == attention(mask=FAKE, mask_dtype=9) == attention(blocks=0) == _lib.ERR_BAD_ARGUMENT
    assert attention(dim=96) == attention(size=48) == attention(dtype=_lib.F32) == attention(cache=_lib.F16) == \
        _lib.ERR_UNSUPPORTED
    assert attention(pool=ODD) == _lib.ERR_ALIGNMENT
    assert attention(batch=70000) == attention(blocks=1 << 31) == _lib.ERR_TOO_LARGE
    # sixteen splits of 128 tokens: more than a cluster, with partials in a workspace
    need = _lib.load().b200_paged_decode_attention_8bit_workspace_bytes(1, 4, 2, 64, 2048, 128)
    split = dict(columns=64, mask_len=2048, split=128)
    assert need > 0 and attention(**split) == attention(**split, workspace=FAKE, nbytes=need - 1) == _lib.ERR_WORKSPACE
    assert _lib.load().b200_paged_decode_attention_8bit_workspace_bytes(1, 4, 2, 64, 2048, 1024) == 0
    assert attention(batch=0) == 0


def test_copy_refusals():
    library = _lib.load()
    pools = struct.pack("=27Q", *[FAKE, 4096, 1024] * 9)

    def copy(count=1, n=2, layers=2, blocks=4, sources=FAKE, table=pools):
        return library.b200_copy_kv_blocks(table, count, sources, FAKE, n, layers, blocks, FAKE, None)

    assert copy(sources=None) == copy(count=0) == copy(n=-1) == copy(layers=0) == copy(blocks=0) == _lib.ERR_BAD_ARGUMENT
    assert copy(blocks=5) == _lib.ERR_BAD_ARGUMENT  # layers that overlap
    assert copy(table=struct.pack("=3Q", 0, 4096, 1024)) == _lib.ERR_BAD_ARGUMENT
    assert copy(count=9) == _lib.ERR_TOO_LARGE
    assert copy(n=0) == 0


def test_quantised_rows_and_linear_refusals():
    library = _lib.load()

    def rows(x=FAKE, residual=None, total=None, n=2, hidden=64, stride=64, dtype=_lib.BF16):
        return library.b200_quantize_rows_int8(struct.pack("=6Q5qd", x or 0, residual or 0, FAKE, total or 0, FAKE, FAKE, n,
                                                           hidden, stride, 64, dtype, 1e-6), None)

    assert rows(x=None) == rows(residual=FAKE) == rows(hidden=0) == rows(stride=63) == rows(dtype=_lib.I8) == \
        _lib.ERR_BAD_ARGUMENT
    assert rows(n=1 << 31) == rows(hidden=1 << 31, stride=1 << 31) == _lib.ERR_TOO_LARGE
    assert rows(n=0) == 0

    def linear(x=FAKE, weight=FAKE, residual=None, m=4, k=64, n=8, dtype=_lib.BF16, epilogue=0):
        return library.b200_linear_int8(struct.pack("=8Q5q", x or 0, FAKE, weight, FAKE, 0, residual or 0, FAKE, FAKE, m, k, n,
                                                    dtype, epilogue), None)

    assert linear(x=None) == linear(k=0) == linear(epilogue=3) == linear(epilogue=1) == linear(residual=FAKE) == \
        linear(dtype=_lib.I8) == _lib.ERR_BAD_ARGUMENT
    assert linear(k=72) == linear(n=7, epilogue=2) == _lib.ERR_UNSUPPORTED
    assert linear(weight=ODD) == _lib.ERR_ALIGNMENT
    assert linear(k=131072) == _lib.ERR_TOO_LARGE
    assert linear(m=0) == 0


def test_wrappers_refuse_cpu_tensors():
    x = torch.zeros(2, 64)
    with pytest.raises(ValueError, match="CUDA"):
        b200.b200_quantize_rows_int8(x)
    with pytest.raises(ValueError, match="CUDA"):
        b200.b200_linear_int8(x.to(torch.int8), x[:, 0], x.to(torch.int8), x[:, 0])
    with pytest.raises(ValueError, match="CUDA"):
        b200.b200_copy_kv_blocks([x], [0], [1])


@pytest.fixture
def copies(monkeypatch):
    made = []
    monkeypatch.setattr(quantized_kernels, "b200_copy_kv_blocks",
                        lambda pools, sources, destinations: made.append((list(sources), list(destinations))))
    return made


def make_state(kind=PagedKVCacheState, dtype=torch.bfloat16, batch=4, num_blocks=12):
    return kind.allocate_paged(num_layers=2, batch=batch, max_tokens=160, block_size=32, num_blocks=num_blocks, kv_heads=2,
                               head_dim=64, dtype=dtype, device="cpu")


def test_fork_shares_whole_blocks_and_copies_a_partial_one(copies):
    state = make_state()
    state.reserve([70, 33, 0, 0])
    assert state._host_table[:2] == [[0, 1, 2], [3, 4]]
    state.fork(0, 2, tokens=70)
    assert state._host_table[2] == [0, 1, 5] and copies == [([2], [5])]
    assert state.block_table[2].tolist() == [0, 1, 5, -1, -1]
    assert [row[2].item() for row in state.lengths] == [70, 70]
    state.fork(2, 3, tokens=64)
    assert state._host_table[3] == [0, 1] and len(copies) == 1 and state.blocks_in_use() == 6
    state.release(0)
    assert state._free[-1] == 2 and state.blocks_in_use() == 5  # 0 and 1 have two holders left
    state.release(2)
    state.release(3)
    assert sorted(state._free) == [0, 1, 2, 5, 6, 7, 8, 9, 10, 11] and state._sharers == {}
    state.fork(1, 0, tokens=0)
    assert state._host_table[0] == [] and state.blocks_in_use() == 2


def test_fork_keeps_the_distances_of_the_extra_length_rows(copies):
    """(an engine's positions and attention lengths stand behind the layers' rows)"""
    state = PagedKVCacheState.allocate_paged(num_layers=2, batch=3, max_tokens=160, block_size=32, num_blocks=12, kv_heads=2,
                                             head_dim=64, dtype=torch.bfloat16, device="cpu", extra_length_rows=2)
    state.reserve([70, 33, 0])
    state._length_arena.copy_(torch.tensor([[70, 33, 0], [70, 33, 0], [70, 33, 0], [71, 34, 1]]))
    state.fork(0, 2)
    assert state._length_arena[:, 2].tolist() == [70, 70, 70, 71] and state._length_arena[:, 0].tolist() == [70, 70, 70, 71]
    state.release(2)
    state.fork(0, 2, tokens=40)
    assert state._length_arena[:, 2].tolist() == [40, 40, 40, 41]


def test_a_fork_whose_copy_fails_changes_nothing(monkeypatch):
    state = make_state()
    state.reserve([70, 0, 0, 0])
    def fails(*arguments):
        raise RuntimeError("launch")
    monkeypatch.setattr(quantized_kernels, "b200_copy_kv_blocks", fails)
    with pytest.raises(RuntimeError):
        state.fork(0, 1, tokens=70)
    assert state._host_table == [[0, 1, 2], [], [], []] and state._sharers == {} and len(state._free) == 9


def test_fork_refusals_change_nothing(copies):
    state = make_state(num_blocks=5)
    state.reserve([70, 33, 0, 0])
    for arguments, tokens in (((0, 0), 10), ((0, 1), 10), ((0, 9), 10), ((-1, 2), 10), ((0, 2), 97), ((0, 2), -1), ((0, 2), 70)):
        with pytest.raises(ExecutionError):  # (the last one: no free block for the partial copy)
            state.fork(*arguments, tokens=tokens)
    assert state._host_table == [[0, 1, 2], [3, 4], [], []] and state._sharers == {} and copies == []
    state.lengths[0][0] = 64
    state.fork(0, 2)  # (the length as the device has it)
    assert state._host_table[2] == [0, 1]


def test_compact_moves_the_highest_blocks_into_the_lowest_holes(copies):
    state = make_state()
    state.reserve([70, 33, 40, 0], order=[9, 1, 7, 4, 11, 0, 5])
    state.fork(1, 3, tokens=64)
    assert state._host_table == [[9, 1, 7], [4, 11], [0, 5], [4, 11]]
    assert state.compact() == 7
    assert copies == [([7, 9, 11], [2, 3, 6])]
    assert state._host_table == [[3, 1, 2], [4, 6], [0, 5], [4, 6]]
    assert state.block_table[3, :2].tolist() == [4, 6] and state._sharers == {4: 2, 6: 2}
    assert state._free == [11, 10, 9, 8, 7] and state.compact() == 7 and len(copies) == 1
    state.release(1)
    assert sorted(state._free) == [7, 8, 9, 10, 11]
    state.release(3)
    assert sorted(state._free) == [4, 6, 7, 8, 9, 10, 11]


def test_state_in_8_bits_has_its_shapes_and_refuses_other_types(copies):
    with pytest.raises(ExecutionError, match="8 bits"):
        make_state(QuantizedPagedKVCacheState)
    state = make_state(QuantizedPagedKVCacheState, torch.int8)
    assert state.keys[0].shape == (12, 2, 32, 64) and state.key_scales[1].shape == (12, 2) and state.capacity == 160
    assert [tuple(pool.shape) for pool in state._pools] == [(2, 12, 2, 32, 64)] * 2 + [(2, 12, 2)] * 2
    assert state.keys[1].data_ptr() == state._pools[0][1].data_ptr()
    derived = state._derive(3)
    assert isinstance(derived, QuantizedPagedKVCacheState) and derived.value_scales is state.value_scales
    with pytest.raises(ExecutionError):
        state.store(0, torch.zeros(4, 3, 1, 64), torch.zeros(4, 3, 1, 64), torch.zeros(4, dtype=torch.int64))
    state.reserve([40, 0, 0, 0])
    state.keys[0].view(torch.int8)[0, 1, 3, 5] = 7
    state.key_scales[0][0, 1] = 0.5
    assert float(state.gather(0, 0, 40)[0][3, 1, 5]) == 3.5
