"""Steps of a paged KV state that fail change nothing: neither blocks, table, lengths nor sharers."""

import pytest
import torch

from llm_compiler_b200.kv_state import ExecutionError, PagedKVCacheState


def make_state(kind=PagedKVCacheState, dtype=torch.bfloat16, batch=3, num_blocks=8):
    return kind.allocate_paged(num_layers=2, batch=batch, max_tokens=160, block_size=32, num_blocks=num_blocks, kv_heads=2,
                               head_dim=64, dtype=dtype, device="cpu", extra_length_rows=2)


def bookkeeping(state):
    return ([list(row) for row in state._host_table], sorted(state._free), dict(state._sharers), state.block_table.tolist(),
            state._length_arena.tolist())


@pytest.mark.parametrize("tokens", [[64, 96, 200], [64, 160, 96]])
def test_a_reservation_that_cannot_be_met_takes_no_block(tokens):
    """(a sequence beyond the capacity, a pool too small: the sequences in front of it had room)"""
    state = make_state(num_blocks=6)
    state.reserve([32, 32, 32])
    before = bookkeeping(state)
    with pytest.raises(ExecutionError):
        state.reserve(tokens)
    assert bookkeeping(state) == before
    state.reserve([64, 32, 32])
    assert state.block_table[0, :2].tolist() == state._host_table[0] and len(state._host_table[0]) == 2
