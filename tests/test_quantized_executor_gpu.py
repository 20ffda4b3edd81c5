"""The KernelIR executor on a paged state in 8 bits: the reference-compiled graphs, unchanged, in both numerical modes and as
fused decode layers."""

import json
from pathlib import Path

import pytest
import torch

import quantized_helpers as ref
from llm_compiler_b200 import kernel_ir as ir
from llm_compiler_b200 import qwen2 as q2
from llm_compiler_b200.executor import B200Executor, bind_arguments
from llm_compiler_b200.kv_state import PagedKVCacheState, QuantizedPagedKVCacheState

pytestmark = pytest.mark.gpu
GOLDEN = Path(__file__).resolve().parent / "golden"


@pytest.mark.parametrize("cache", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("form", ["fast", "pytorch_compatible", "fused"])
def test_reference_decode_graph_on_a_state_in_8_bits(form, cache, golden_tiny):
    """The same graph over a 16-bit paged state and over one in 8 bits that was given the same prompt: lengths move alike, the
    cache holds the definition's codes of the rows that the 16-bit state was given in the first step, and the logits differ by
    what codes off by half a step cost (a step is 1/127 of a block's largest, or 1/8 of a value)."""
    gold = golden_tiny["bf16"]
    config = q2.Qwen2Config(**gold["config"])
    weights = {k: v.cuda() for k, v in q2.make_weights(config, seed=0, dtype=torch.bfloat16).items()}
    inv_freq = q2.inverse_frequency(config, "cuda")
    batch, prompt, steps = gold["batch"], gold["prompt"], gold["steps"]
    mode = "pytorch_compatible" if form == "pytorch_compatible" else "fast"
    module = ir.module_from_json(json.loads((GOLDEN / f"kernel_ir_tiny_bf16_decode_{mode}.json").read_text()))
    ir.lower_to_b200(module, zero_mask_arguments=("attention_mask",) if form == "fused" else ())
    states, logits = [], [[], []]
    zeros = torch.zeros(batch, dtype=torch.int64, device="cuda")
    for kind, dtype in ((PagedKVCacheState, torch.bfloat16), (QuantizedPagedKVCacheState, cache)):
        state = kind.allocate_paged(num_layers=config.num_layers, batch=batch, max_tokens=gold["capacity"], block_size=32,
                                    num_blocks=8, kv_heads=config.num_kv_heads, head_dim=config.head_dim, dtype=dtype, device="cuda")
        state.reserve([prompt + steps] * batch, order=[5, 2, 7, 0, 3, 1, 6, 4])
        for layer in range(config.num_layers):
            state.store(layer, gold["keys"][layer][:, :prompt].transpose(1, 2).cuda(),
                        gold["values"][layer][:, :prompt].transpose(1, 2).cuda(), zeros)
            state.lengths[layer].fill_(prompt)
        states.append(state)
    before = ref.Cache(states[1].keys[0], states[1].key_scales[0])
    executor = B200Executor()
    for step in range(steps):
        for i, state in enumerate(states):
            out, states[i] = executor.run(module, bind_arguments(module.functions[0], weights, {
                "input_ids": gold["tokens"][:, step].view(batch, 1).cuda(),
                "attention_mask": torch.zeros(batch, 1, 1, prompt + step + 1, device="cuda"),
                "position_ids": torch.full((batch, 1), prompt + step, device="cuda"),
                "kv_state": state, "inv_freq": inv_freq})).outputs
            logits[i].append(out[:, 0].float())
        if step == 0:  # (layer 0 sees the same input in both)
            rows = torch.stack([states[0].gather(0, b, prompt + 1)[0][prompt] for b in range(batch)]).unsqueeze(2)
            before.store(states[1].block_table.cpu(), rows, torch.full((batch,), prompt))
            got, want = (states[1].keys[0].cpu().float() * states[1].key_scales[0].cpu()[:, :, None, None],
                         (before.codes * before.scales[:, :, None, None]).float())
            # (the fused layer of 16 bits rounds q|k|v elsewhere: a step of bf16, and the code that it may move)
            assert float((got - want).abs().max()) <= (2.0 ** -7 + 1 / 8) * float(want.abs().max())
    assert isinstance(states[1], QuantizedPagedKVCacheState)
    for state in states:
        state.check()
        assert torch.equal(torch.stack(list(state.lengths), 0).cpu(), gold["lengths"])
    for wide, narrow in zip(*logits):
        assert float((narrow - wide).norm() / wide.norm()) < (0.05 if cache == torch.int8 else 0.2)
