"""Steps of a paged KV state and of an engine that fail: a fork changes neither blocks, table, lengths nor sharers, a reservation
leaves host and device with one table, an engine is refused when it is built."""

import pytest
import torch

from llm_compiler_b200 import quantized_kernels
from llm_compiler_b200 import qwen2 as q2
from llm_compiler_b200.engine import Qwen2Engine
from llm_compiler_b200.kv_state import ExecutionError, PagedKVCacheState, QuantizedPagedKVCacheState


def make_state(kind=PagedKVCacheState, dtype=torch.bfloat16, batch=3, num_blocks=8):
    return kind.allocate_paged(num_layers=2, batch=batch, max_tokens=160, block_size=32, num_blocks=num_blocks, kv_heads=2,
                               head_dim=64, dtype=dtype, device="cpu", extra_length_rows=2)


def bookkeeping(state):
    return ([list(row) for row in state._host_table], sorted(state._free), dict(state._sharers), state.block_table.tolist(),
            state._length_arena.tolist())


@pytest.mark.parametrize("tokens,held", [([64, 96, 200], [2, 3, 1]), ([64, 160, 96], [2, 3, 1]), ([96, 200, 64], [3, 1, 1])])
def test_a_reservation_that_cannot_be_met_leaves_the_table_as_the_host_has_it(tokens, held):
    """A sequence beyond the capacity, a pool too small: the sequences in front keep what they were given, on both sides."""
    state = make_state(num_blocks=6)
    state.reserve([32, 32, 32])
    with pytest.raises(ExecutionError):
        state.reserve(tokens)
    assert [len(row) for row in state._host_table] == held
    for b, row in enumerate(state._host_table):
        assert state.block_table[b].tolist() == row + [-1] * (5 - len(row))
    assert sorted(state._free + [block for row in state._host_table for block in row]) == list(range(6))


def make_engine(num_blocks, lengths, kind=QuantizedPagedKVCacheState, dtype=torch.int8):
    """An engine between steps, without its model: what fork works on."""
    engine = Qwen2Engine.__new__(Qwen2Engine)
    engine.paged, engine.batch = True, len(lengths)
    engine.state = make_state(kind, dtype, len(lengths), num_blocks)
    engine.capacity = engine.state.capacity
    engine.input_ids = torch.arange(10, 10 + len(lengths))
    engine._host_lengths = list(lengths)
    arena = engine.state._length_arena
    arena[:3], arena[3] = torch.tensor(lengths), torch.tensor(lengths) + 1
    engine._block_slack = 0
    engine._reserve_blocks()
    return engine


def everything(engine):
    return (*bookkeeping(engine.state), list(engine._host_lengths), engine._block_slack, engine.input_ids.tolist())


@pytest.fixture
def copies(monkeypatch):
    made = []
    monkeypatch.setattr(quantized_kernels, "b200_copy_kv_blocks",
                        lambda pools, sources, destinations: made.append((list(sources), list(destinations))))
    return made


@pytest.mark.parametrize("num_blocks,lengths", [
    (9, [150, 0, 40]),   # 5 + 1 + 3 held of 9: the target's block takes the copy of the last one, four are shared
    (9, [70, 5, 40]),    # 4 + 2 + 3 of 9: two given back, for the copy and the block ahead
])
def test_a_fork_that_has_room_takes_the_targets_blocks_back(num_blocks, lengths, copies):
    engine = make_engine(num_blocks, lengths)
    engine.fork(0, 1)
    assert engine._host_lengths == [lengths[0], lengths[0], lengths[2]] and engine.input_ids.tolist() == [10, 10, 12]
    state = engine.state
    whole, partial = divmod(lengths[0], 32)
    assert state._host_table[1][:whole] == state._host_table[0][:whole]
    assert copies == [([state._host_table[0][whole]], [state._host_table[1][whole]])]
    assert state._length_arena[:, 1].tolist() == [lengths[0]] * 3 + [lengths[0] + 1]
    held = [block for row in state._host_table for block in set(row)]
    assert not set(held) & set(state._free) and len(set(held)) + len(state._free) == num_blocks
    assert all(state.block_table[b, :len(row)].tolist() == row for b, row in enumerate(state._host_table))
    assert all(len(row) * 32 > n for row, n in zip(state._host_table, engine._host_lengths))


def test_a_fork_over_a_branch_of_its_source(copies):
    engine = make_engine(9, [70, 20, 40])
    engine.fork(0, 1)
    first = bookkeeping(engine.state)
    engine.fork(0, 1)  # (shared blocks are given back and taken again, its own last ones serve once more)
    again = bookkeeping(engine.state)
    assert again[2] == first[2] and len(again[1]) == len(first[1]) and [len(row) for row in again[0]] == [len(row) for row in first[0]]


@pytest.mark.parametrize("case", ["no block for the copy", "no block ahead"])
def test_a_fork_without_room_changes_nothing(case, copies):
    engine = Qwen2Engine.__new__(Qwen2Engine)
    engine.paged, engine.batch, engine.capacity = True, 3, 160
    if case == "no block for the copy":
        state = engine.state = make_state(QuantizedPagedKVCacheState, torch.int8, 3, num_blocks=5)
        state.reserve([96, 64, 0])      # 3 + 2 of 5
        state.fork(1, 2, tokens=64)     # the target's two blocks are shared: none comes back
        lengths = [70, 64, 64]
    else:
        state = engine.state = make_state(QuantizedPagedKVCacheState, torch.int8, 3, num_blocks=7)
        state.reserve([96, 32, 96])     # 3 + 1 + 3 of 7: one comes back, the copy and the next step's block need two
        lengths = [70, 10, 90]
    engine._host_lengths, engine._block_slack = list(lengths), 3
    engine.input_ids = torch.arange(10, 13)
    state._length_arena[:3], state._length_arena[3] = torch.tensor(lengths), torch.tensor(lengths) + 1
    before = everything(engine)
    with pytest.raises(ExecutionError, match="exhausted"):
        engine.fork(0, 1)
    assert everything(engine) == before and copies == []


def test_a_fork_whose_copy_cannot_be_launched_changes_nothing(monkeypatch):
    engine = make_engine(12, [70, 20, 40])
    before = everything(engine)

    def fails(*arguments):
        raise RuntimeError("launch")

    monkeypatch.setattr(quantized_kernels, "b200_copy_kv_blocks", fails)
    with pytest.raises(RuntimeError):
        engine.fork(0, 1)
    assert everything(engine) == before


def test_an_engine_refuses_head_sizes_that_a_cache_in_8_bits_has_no_attention_for():
    """When it is built, not at its first step."""
    config = q2.Qwen2Config(hidden_size=128, intermediate_size=256, num_layers=1, num_heads=4, num_kv_heads=2, rms_norm_eps=1e-6,
                            rope_theta=1e6, vocab_size=64, tie_word_embeddings=True)
    weights = q2.make_weights(config, seed=0, dtype=torch.bfloat16)
    assert config.head_dim == 32
    with pytest.raises(ValueError, match="head sizes"):
        Qwen2Engine(config, weights, batch=2, capacity=64, kv_layout="paged", block_size=32, kv_dtype=torch.int8)
