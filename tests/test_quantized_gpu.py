"""The operators in 8 bits against their 64-bit definitions: the store that quantises into a paged cache, decode attention
over it, copies of blocks, rows quantised behind a norm, integer projections; their refusals on the device; all of them
together as a server uses them."""

import math

import pytest
import torch

import llm_compiler_b200 as b200
import quantized_helpers as ref
from llm_compiler_b200 import _lib, kernels
from llm_compiler_b200 import qwen2 as q2
from llm_compiler_b200.engine import Qwen2Engine
from llm_compiler_b200.kv_state import ExecutionError, PagedKVCacheState, QuantizedPagedKVCacheState

pytestmark = pytest.mark.gpu
CACHES = [torch.int8, torch.float8_e4m3fn]


def make_cache(g, dtype, blocks, heads, size, dim):
    """Random codes and scales of a cache that has been in use."""
    top = ref.TOP[dtype]
    pools = [(torch.randn(blocks, heads, size, dim, generator=g) * top / 3).clamp(-top, top) for _ in range(2)]
    pools = [(p.round() if dtype == torch.int8 else p).to(dtype).cuda() for p in pools]
    scales = [((2 + 3 * torch.rand(blocks, heads, generator=g)) / top).cuda() for _ in range(2)]
    return pools, scales


def scattered(g, batch, columns, extra=3):
    order = torch.randperm(batch * columns + extra, generator=g)[:batch * columns]
    return order.to(torch.int32).view(batch, columns), batch * columns + extra


def same_codes(pool, cache):
    got, want = pool.cpu().float().double(), cache.codes
    return torch.equal(got.nan_to_num(1e9), want.nan_to_num(1e9))


# ---------------------------------------------------------------------------------------------------------------- store ----
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("size,heads,dim,tokens,positions", [
    (32, 2, 64, 1, [0, 31, 32, 70]),      # one token: a fresh block, a block's last row, the next one's first
    (128, 3, 128, 1, [5, 127, 128, 300]),
    (64, 1, 64, 63, [0, 1, 64, 37]),      # portions that end inside, at and behind a block's end
    (32, 2, 256, 100, [0, 7, 31, 32]),
    (256, 1, 128, 300, [0, 255, 1, 100]),  # more rows of a block than a thread keeps
    (96, 4, 48, 97, [0, 95, 96, 3]),
])
def test_store_gives_the_codes_and_scales_of_the_definition(dtype, cache, size, heads, dim, tokens, positions):
    g = torch.Generator().manual_seed(size + tokens + dim)
    batch, columns = len(positions), -(-(max(positions) + tokens) // size)
    table, blocks = scattered(g, batch, columns)
    (keys, values), (key_scales, value_scales) = make_cache(g, cache, blocks, heads, size, dim)
    expected = [ref.Cache(keys, key_scales), ref.Cache(values, value_scales)]
    # rows of a packed projection; magnitudes that raise some blocks' scales and not others
    packed = torch.randn(batch, tokens, 2, heads, dim, generator=g) * torch.exp2(torch.randint(-2, 3, (batch, 1, 1, heads, 1),
                                                                                             generator=g).float())
    packed = packed.to(dtype)
    key, value = packed[:, :, 0].transpose(1, 2), packed[:, :, 1].transpose(1, 2)
    positions = torch.tensor(positions)
    for cached, x in zip(expected, (key, value)):
        cached.store(table, x, positions)
    device = packed.cuda()
    b200.b200_paged_kv_store_8bit(keys, values, key_scales, value_scales, table.cuda(), device[:, :, 0].transpose(1, 2),
                                  device[:, :, 1].transpose(1, 2), positions.cuda())
    for pool, scales, cached in ((keys, key_scales, expected[0]), (values, value_scales, expected[1])):
        assert torch.equal(scales.cpu().double(), cached.scales)
        assert same_codes(pool, cached)
    kernels.runtime().check_status()


@pytest.mark.parametrize("cache", CACHES)
def test_store_takes_any_strides_and_unaligned_rows(cache):
    g = torch.Generator().manual_seed(3)
    batch, heads, tokens, dim, size = 2, 3, 40, 64, 32
    table, blocks = scattered(g, batch, 2)
    base = torch.randn(batch, heads, dim, tokens + 1, generator=g).bfloat16()
    wide = torch.randn(batch, tokens, heads, dim + 3, generator=g).bfloat16()
    results = []
    for make in (lambda x: x, lambda x: x.contiguous()):
        (keys, values), (key_scales, value_scales) = make_cache(torch.Generator().manual_seed(9), cache, blocks, heads, size, dim)
        key = make(base.cuda()[..., 1:].transpose(2, 3))             # element stride tokens + 1
        value = make(wide.cuda()[..., 1:dim + 1].transpose(1, 2))    # odd row stride, odd offset
        b200.b200_paged_kv_store_8bit(keys, values, key_scales, value_scales, table.cuda(), key, value,
                                      torch.tensor([0, 11]).cuda())
        results.append((keys.view(torch.uint8), values.view(torch.uint8), key_scales, value_scales))
    for a, b in zip(*results):
        assert torch.equal(a, b)


@pytest.mark.parametrize("cache", CACHES)
def test_store_of_zeros_tiny_and_non_finite_rows(cache):
    g = torch.Generator().manual_seed(5)
    size, dim = 32, 64
    x = torch.randn(4, 1, 3, dim, generator=g).bfloat16()
    x[0] = 0.0
    x[1] = 2.0 ** -133  # subnormal: the scale stops at the smallest normal number
    x[2, 0, 1, 5], x[2, 0, 2, 6], x[2, 0, 0, 7] = math.inf, -math.inf, math.nan
    x[3] = math.inf     # nothing finite in the block
    table, blocks = scattered(g, 4, 1)
    (keys, values), (key_scales, value_scales) = make_cache(g, cache, blocks, 1, size, dim)
    expected = ref.Cache(keys, key_scales)
    expected.store(table, x, torch.zeros(4, dtype=torch.int64))
    clean = x.clone()
    clean[2:] = 1.0
    zeros = torch.zeros(4, dtype=torch.int64, device="cuda")
    b200.b200_paged_kv_store_8bit(keys, values, key_scales, value_scales, table.cuda(), clean.cuda(), clean.cuda(), zeros)
    kernels.runtime().check_status()
    b200.b200_paged_kv_store_8bit(keys, values, key_scales, value_scales, table.cuda(), x.cuda(), clean.cuda(), zeros)
    with pytest.raises(kernels.KernelStatusError, match="8-bit format"):
        kernels.runtime().check_status()
    assert torch.equal(key_scales.cpu().double(), expected.scales)
    where = table[:3, 0].long()  # (with no finite row there is no scale for an infinity to saturate at)
    assert torch.equal(keys.cpu().float()[where][:, :, :3].nan_to_num(1e9), expected.codes[where][:, :, :3].float().nan_to_num(1e9))
    assert float(key_scales[table[3, 0].item(), 0]) == 0.0


def test_store_skips_what_has_no_place_and_says_so():
    g = torch.Generator().manual_seed(6)
    size, dim, heads = 32, 64, 2
    table, blocks = scattered(g, 4, 2)
    table[1, 0] = -1
    table[2, 1] = blocks
    (keys, values), (key_scales, value_scales) = make_cache(g, torch.int8, blocks, heads, size, dim)
    cached = ref.Cache(keys, key_scales)
    x = torch.randn(4, heads, 40, dim, generator=g).half()
    for positions, match in (([0, 0, 0, 0], "negative KV position"), ([30, -1, 0, 30], "beyond capacity"),
                             ([0, -1, 0, 2 ** 62], "beyond capacity"), ([0, -(2 ** 62), 0, 64], "beyond capacity")):
        positions = torch.tensor(positions)
        cached.store(table, x, positions)
        b200.b200_paged_kv_store_8bit(keys, values, key_scales, value_scales, table.cuda(), x.cuda(), x.cuda(), positions.cuda())
        with pytest.raises(kernels.KernelStatusError, match=match):
            kernels.runtime().check_status()
        assert torch.equal(key_scales.cpu().double(), cached.scales) and same_codes(keys, cached)


def test_token_by_token_stores_read_like_one_store_of_the_prompt_within_the_roundings_of_growth():
    """Each growth of a scale rounds what is held once more: half a step of the scale then, which is at most half a step of
    the last one; the last scale is the prompt's own."""
    g = torch.Generator().manual_seed(8)
    size, dim, tokens = 32, 64, 45
    x = (torch.randn(1, 2, tokens, dim, generator=g) * torch.linspace(0.2, 2, tokens).view(1, 1, -1, 1)).bfloat16()
    table = torch.tensor([[2, 0]], dtype=torch.int32)
    pools, scales = make_cache(g, torch.int8, 3, 2, size, dim)
    growths = torch.zeros(3, 2)
    before = scales[0].clone().cpu()
    for t in range(tokens):
        b200.b200_paged_kv_store_8bit(*pools, *scales, table.cuda(), x[:, :, t:t + 1].cuda(), x[:, :, t:t + 1].cuda(),
                                      torch.tensor([t]).cuda())
        if t % size == 0:
            growths[table[0, t // size]] = 0
        growths += (scales[0].cpu() > before).float()
        before = scales[0].cpu()
    whole = ref.Cache(*[t.clone() for t in (pools[0], scales[0])])
    whole.store(table, x, torch.tensor([0]))
    assert torch.equal(scales[0].cpu()[[2, 0]].double(), whole.scales[[2, 0]])
    for column, rows in ((0, 32), (1, 13)):
        at = int(table[0, column])
        off = pools[0].cpu()[at].double()[:, :rows] - \
            x[0, :, column * size:column * size + rows].double() / whole.scales[at][:, None, None]
        limit = 0.5 + 0.5 * growths[at].double() + 1e-4
        assert bool((off.abs() <= limit[:, None, None]).all())
    assert float(growths[2].max()) > 2  # (the case does grow)


# ------------------------------------------------------------------------------------------------------------ attention ----
def check_attention(g, cache, dtype, lengths, heads, kv_heads, dim, size, *, mask=None, spread=1.0, capacity=0, hint=0,
                    split_tokens=0, dirty=True):
    batch = len(lengths)
    columns = -(-max(capacity, max(lengths), 1) // size)
    table, blocks = scattered(g, batch, columns)
    pools, scales = make_cache(g, cache, blocks, kv_heads, size, dim)
    if dirty:  # entries behind a sequence's end: anything, NaN codes among it
        for b, length in enumerate(lengths):
            for column in range(length // size, columns):
                first = max(0, length - column * size)
                for pool in pools:
                    pool.view(torch.uint8)[table[b, column], :, first:] = 0x7f
    for s in scales:
        s.mul_(torch.exp2(spread * torch.randn(s.shape, generator=g)).cuda())
    query = torch.randn(batch, 1, heads, dim, generator=g).to(dtype).transpose(1, 2)
    lengths_ = torch.tensor(lengths)
    keys, values = ref.Cache(pools[0], scales[0]), ref.Cache(pools[1], scales[1])
    want, bound = ref.attention(query, keys, values, table, lengths_, mask, dim ** -0.5)
    got = b200.b200_paged_decode_attention_8bit(query.cuda(), *pools, *scales, table.cuda(), lengths_.cuda(),
                                                None if mask is None else mask.cuda(), scale=dim ** -0.5,
                                                max_length_hint=hint, split_tokens=split_tokens)
    assert got.shape == query.shape and got.dtype == dtype
    got = got.cpu().double()
    assert torch.equal(got.isnan(), want.isnan())
    worst = ((got - want).abs() / bound).nan_to_num(0.0).max()
    assert float(worst) <= 1.0, f"{float(worst):.2f} of the bound"
    kernels.runtime().check_status()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads,kv_heads", [(14, 2), (3, 3), (16, 1), (24, 2), (40, 2)])
def test_attention_of_heads_types_and_ragged_lengths(dtype, cache, dim, heads, kv_heads):
    g = torch.Generator().manual_seed(heads * dim)
    check_attention(g, cache, dtype, [1, 33, 0, 300, 129, 64, 31], heads, kv_heads, dim, 64)


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("size", [32, 96, 128, 256])
@pytest.mark.parametrize("lengths", [[1], [32], [2049], [5000, 17], [255, 256, 257, 511, 512, 513]])
def test_attention_of_blocks_and_splits(cache, size, lengths):
    g = torch.Generator().manual_seed(size + len(lengths))
    check_attention(g, cache, torch.bfloat16, lengths, 7, 1, 64, size, capacity=6000)
    check_attention(g, cache, torch.bfloat16, lengths, 8, 2, 128, size, hint=max(lengths))
    check_attention(g, cache, torch.bfloat16, lengths, 8, 2, 64, size, hint=10, split_tokens=64)  # a hint bounds nothing


@pytest.mark.parametrize("dim,heads", [(64, 7), (64, 16), (128, 8), (128, 13), (256, 4)])
@pytest.mark.parametrize("splits", [2, 3, 5, 6, 7, 8, 9])
def test_attention_of_any_number_of_splits(dim, heads, splits):
    """Clusters of any size, all of whose CTAs have tiles or only some, and more splits than a cluster holds."""
    g = torch.Generator().manual_seed(dim + splits)
    for cache, dtype in ((torch.int8, torch.bfloat16), (torch.float8_e4m3fn, torch.float16)):
        check_attention(g, cache, dtype, [1500, 700, 0, 129, 1], heads, 1, dim, 32, split_tokens=-(-1504 // splits))


@pytest.mark.parametrize("batch,dim", [(25, 128), (30, 128), (36, 128), (50, 128), (60, 128), (90, 128), (45, 64), (13, 256), (40, 256)])
def test_attention_of_batches_between_the_sizes_of_clusters(batch, dim):
    g = torch.Generator().manual_seed(batch)
    lengths = torch.randint(0, 1100, (batch,), generator=g).tolist()
    check_attention(g, torch.int8, torch.bfloat16, lengths, 4, 2, dim, 64, capacity=1100)


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("kind", ["padded", "lowest", "soft", "empty-row", "half", "positive-infinity"])
def test_attention_masks(cache, kind):
    g = torch.Generator().manual_seed(len(kind))
    lengths = [200, 1, 64, 777]
    mask = torch.zeros(4, 1, 1, 800)
    if kind == "padded":
        mask[:, :, :, :1] = -math.inf
        mask[3, :, :, 1:300] = -math.inf  # (whole tiles and splits with nothing left)
        mask[1] = 0
    elif kind == "lowest":  # every token at the type's lowest value: scores vanish in it and the weights are equal
        mask[:] = torch.finfo(torch.float32).min
        mask[2, :, :, ::2] = 0
    elif kind == "soft":
        mask = torch.randn(4, 1, 1, 800, generator=g).bfloat16()
    elif kind == "empty-row":
        mask[2] = -math.inf
        mask[1] = -math.inf
    elif kind == "half":
        mask = torch.randn(4, 1, 1, 800, generator=g).half()
        mask[:, :, :, 5::9] = -math.inf
        mask = torch.cat([mask, mask], 3)[..., ::2]  # an element stride of two
    else:
        mask[0, :, :, 3] = math.inf
    check_attention(g, cache, torch.bfloat16, lengths, 6, 2, 64, 32, mask=mask, capacity=800)


def test_attention_of_scales_far_apart():
    """Blocks whose scales differ by 2^-20 ... 2^20: a value block of small scale that gets all of the weight keeps its
    precision beside a large one that gets none."""
    g = torch.Generator().manual_seed(1)
    for cache in CACHES:
        check_attention(g, cache, torch.bfloat16, [500, 1000], 4, 2, 64, 32, spread=8.0)
    size, dim = 32, 64
    pools, scales = make_cache(g, torch.int8, 2, 1, size, dim)
    scales[1][0], scales[1][1] = 1e6, 1e-6
    table = torch.tensor([[0, 1]], dtype=torch.int32)
    mask = torch.zeros(1, 1, 1, 64)
    mask[..., :32] = -200.0
    query = torch.randn(1, 1, 1, dim, generator=g).half()
    got = b200.b200_paged_decode_attention_8bit(query.cuda(), *pools, *scales, table.cuda(), torch.tensor([64]).cuda(),
                                                mask.cuda(), scale=0.125).cpu().double()
    values = ref.Cache(pools[1], scales[1])
    values.scales[0] = 0.0
    want, _ = ref.attention(query, ref.Cache(pools[0], scales[0]), values, table, [64], mask, 0.125)
    # fp16 spaces its results 2^-24 apart here; 2^-10 of the largest for the probabilities
    assert float((got - want).abs().max()) <= 2.0 ** -25 + 2.0 ** -10 * 127e-6


def test_attention_of_queries_at_the_ends_of_their_range():
    """Queries beyond fp16's range and below it, and scales that bring their scores back to order one."""
    g = torch.Generator().manual_seed(2)
    size, dim = 32, 64
    for factor in (1e30, 1e-30):
        pools, scales = make_cache(g, torch.int8, 4, 1, size, dim)
        scales[0].div_(factor)
        table = torch.tensor([[3, 1, 0, 2]], dtype=torch.int32)
        query = (torch.randn(1, 4, 1, dim, generator=g) * factor).bfloat16()
        want, bound = ref.attention(query, ref.Cache(pools[0], scales[0]), ref.Cache(pools[1], scales[1]), table, [111], None, 0.125)
        got = b200.b200_paged_decode_attention_8bit(query.cuda(), *pools, *scales, table.cuda(), torch.tensor([111]).cuda(),
                                                    None, scale=0.125).cpu().double()
        assert bool(((got - want).abs() <= bound).all())


def test_attention_leaves_out_blocks_that_are_not_there_and_clamps_lengths():
    g = torch.Generator().manual_seed(4)
    size, dim = 32, 64
    table, blocks = scattered(g, 2, 4)
    pools, scales = make_cache(g, torch.int8, blocks, 1, size, dim)
    query = torch.randn(2, 4, 1, dim, generator=g).bfloat16()
    keys, values = ref.Cache(pools[0], scales[0]), ref.Cache(pools[1], scales[1])
    mask = torch.zeros(2, 1, 1, 100)
    want, bound = ref.attention(query, keys, values, table, [100, 50], mask, 0.125)
    got = b200.b200_paged_decode_attention_8bit(query.cuda(), *pools, *scales, table.cuda(), torch.tensor([128, 50]).cuda(),
                                                mask.cuda(), scale=0.125)
    with pytest.raises(kernels.KernelStatusError, match="attention mask length"):
        kernels.runtime().check_status()
    assert bool(((got.cpu().double() - want).abs() <= bound).all())
    holes = table.clone()
    holes[0, 1], holes[1, 0] = -1, blocks
    mask = torch.zeros(2, 1, 1, 128)
    mask[0, :, :, 32:64] = -math.inf
    mask[1, :, :, :32] = -math.inf
    want, bound = ref.attention(query, keys, values, table, [128, 50], mask, 0.125)
    got = b200.b200_paged_decode_attention_8bit(query.cuda(), *pools, *scales, holes.cuda(), torch.tensor([128, 50]).cuda(),
                                                None, scale=0.125)
    with pytest.raises(kernels.KernelStatusError, match="position"):
        kernels.runtime().check_status()
    assert bool(((got.cpu().double() - want).abs() <= bound).all())
    got = b200.b200_paged_decode_attention_8bit(query.cuda(), *pools, *scales, table.cuda(), torch.tensor([-5, 50]).cuda(),
                                                None, scale=0.125)
    assert bool(got[0].isnan().all()) and not bool(got[1].isnan().any())


def test_attention_is_the_same_from_run_to_run_on_streams_and_in_replayed_graphs():
    g = torch.Generator().manual_seed(11)
    lengths = torch.tensor([3000, 10, 1500]).cuda()
    table, blocks = scattered(g, 3, 24)
    pools, scales = make_cache(g, torch.float8_e4m3fn, blocks, 2, 128, 64)
    queries = [torch.randn(3, 14, 1, 64, generator=g).bfloat16().cuda() for _ in range(2)]

    def call(query):
        return b200.b200_paged_decode_attention_8bit(query, *pools, *scales, table_, lengths, None, scale=0.125)

    table_ = table.cuda()
    want = [call(q) for q in queries]
    for _ in range(3):
        assert torch.equal(call(queries[0]), want[0])
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    found = [[], []]
    for _ in range(20):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                found[i].append(call(queries[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in found[i])
    graphs, outputs = [], []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outputs.append(call(queries[i]))
        graphs.append(graph)
    for _ in range(10):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                graphs[i].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(outputs[i], want[i]) for i in range(2))


def test_wrappers_refuse_what_does_not_fit():
    state = make_state(torch.int8)
    cache = (state.keys[0], state.values[0], state.key_scales[0], state.value_scales[0], state.block_table)
    rows = torch.zeros(4, 2, 1, 64, dtype=torch.bfloat16, device="cuda")
    at = state.positions(0)
    wrong = lambda i, t: tuple(t if j == i else c for j, c in enumerate(cache))
    for arguments in ((*cache, rows.float(), rows.float(), at), (*cache, rows, rows[:, :1], at), (*cache, rows[:, :1], rows[:, :1], at),
                      (*cache, rows, rows, at.int()), (*cache, rows, rows, at[:2]), (*cache, rows, rows.half(), at),
                      (*wrong(0, cache[0].float()), rows, rows, at), (*wrong(2, cache[2].half()), rows, rows, at),
                      (*wrong(2, cache[2][:, :1]), rows, rows, at), (*wrong(4, cache[4].long()), rows, rows, at),
                      (*wrong(4, cache[4][:2]), rows, rows, at), (*cache, rows.cpu(), rows, at)):
        with pytest.raises(ValueError):
            b200.b200_paged_kv_store_8bit(*arguments)
    query = torch.zeros(4, 4, 1, 64, dtype=torch.bfloat16, device="cuda")
    lengths = state.lengths[0]
    for arguments in ((query.float(), *cache, lengths, None), (query[:, :3], *cache, lengths, None), (query[:2], *cache, lengths, None),
                      (query.expand(4, 4, 2, 64), *cache, lengths, None), (query, *cache, lengths.int(), None),
                      (query, *cache, lengths, torch.zeros(4, 1, 1, 257, device="cuda")),
                      (query, *cache, lengths, torch.zeros(4, 1, 2, 9, device="cuda"))):
        with pytest.raises(ValueError):
            b200.b200_paged_decode_attention_8bit(*arguments, scale=1.0)
    for pools, sources, destinations in (([], [0], [1]), ([at], [0], [1]), (state._pools, [0], [24]), (state._pools, [0], [-1]),
                                         (state._pools, [0, 1], [2, 2]), (state._pools, [0, 1], [1, 2]), (state._pools, [0], [1, 2]),
                                         (state._pools, torch.tensor([0], device="cuda"), [1]),
                                         ([state._pools[0], state._pools[1][:1]], [0], [1])):
        with pytest.raises(ValueError):
            b200.b200_copy_kv_blocks(pools, sources, destinations)
    x, w = torch.zeros(2, 64, device="cuda"), torch.zeros(64, device="cuda")
    for call in (lambda: b200.b200_rms_norm_int8(x, w.half(), epsilon=1e-6), lambda: b200.b200_rms_norm_int8(x, w[:5], epsilon=1e-6),
                 lambda: b200.b200_rms_norm_int8(x, None, epsilon=1e-6), lambda: b200.b200_rms_norm_int8(x, w, epsilon=1e-6, residual=x[:1]),
                 lambda: b200.b200_quantize_rows_int8(x.to(torch.int32))):
        with pytest.raises(ValueError):
            call()
    v, vs = b200.b200_quantize_rows_int8(x)
    for arguments, options in (((v, vs, v.float(), vs), {}), ((v, vs[:1], v, vs), {}), ((v[:, :40], vs, v[:, :40], vs), {}),
                               ((v, vs, v, vs, w[:2].half()), {}), ((v, vs, v, vs), dict(epilogue="gelu")),
                               ((v, vs, v, vs), dict(epilogue="residual")), ((v, vs, v, vs), dict(residual=x)),
                               ((v, vs, v[:1], vs[:1]), dict(epilogue="swiglu")), ((v, vs, v, vs), dict(out_dtype=torch.int8)),
                               ((v[:, :24].contiguous(), vs, v[:, :24].contiguous(), vs), {})):
        with pytest.raises(ValueError):
            b200.b200_linear_int8(*arguments, **options)


def test_waits_that_run_out_set_the_status_and_leave_the_next_calls_right():
    """Kernels whose copies never come: every wait gives up, the status says so, and the same calls are right afterwards."""
    g = torch.Generator().manual_seed(17)
    table, blocks = scattered(g, 2, 8)
    pools, scales = make_cache(g, torch.int8, blocks, 2, 64, 64)
    query, lengths = torch.randn(2, 4, 1, 64, generator=g).bfloat16().cuda(), torch.tensor([500, 100]).cuda()
    cases = [lambda s=s: b200.b200_paged_decode_attention_8bit(query, *pools, *scales, table.cuda(), lengths, None, scale=0.125,
                                                               split_tokens=s) for s in (0, 40, 512)]
    for m, k, n in ((8, 256, 512), (8, 1024, 128), (300, 512, 512), (300, 2048, 200), (1024, 512, 2048), (1024, 512, 2050), (250, 12000, 2500)):
        values, weight = (torch.randint(-127, 128, (r, k), generator=g, dtype=torch.int8).cuda() for r in (m, n))
        a = (values, torch.rand(m, generator=g).cuda(), weight, torch.rand(n, generator=g).cuda())
        cases.append(lambda a=a: b200.b200_linear_int8(*a))
        residual = torch.randn(m, n, generator=g).bfloat16().cuda()
        cases.append(lambda a=a, r=residual: b200.b200_linear_int8(*a, residual=r, epilogue="residual"))
    want = [case() for case in cases]
    kernels.runtime().check_status()
    library = _lib.load()
    for case, right in zip(cases, want):
        library.b200_debug_set_waits(2000, 1)
        try:
            case()
            torch.cuda.synchronize()
        finally:
            library.b200_debug_set_waits(4000000, 0)
        with pytest.raises(kernels.KernelStatusError, match="wait gave up"):
            kernels.runtime().check_status()
        assert torch.equal(case(), right)
        kernels.runtime().check_status()


def test_calls_without_rows_launch_nothing():
    state = make_state(torch.int8, batch=4)
    launches = kernels.launch_count()
    nothing = torch.zeros(4, 2, 0, 64, dtype=torch.bfloat16, device="cuda")
    state.store(0, nothing, nothing, state.positions(0))
    empty = torch.zeros(0, 4, 1, 64, dtype=torch.bfloat16, device="cuda")
    out = b200.b200_paged_decode_attention_8bit(empty, state.keys[0], state.values[0], state.key_scales[0],
                                                state.value_scales[0], state.block_table[:0], state.lengths[0][:0], None,
                                                scale=1.0)
    assert out.shape == empty.shape and kernels.launch_count() == launches


# ----------------------------------------------------------------------------------------------------------------- copy ----
@pytest.mark.parametrize("shape", [(128, 64), (32, 256), (96, 24), (37, 31), (7, 3)])
def test_copied_blocks_hold_what_their_sources_hold_and_the_others_keep_theirs(shape):
    g = torch.Generator().manual_seed(shape[0])
    layers, blocks, heads = 3, 40, 2
    pools = [torch.randint(0, 255, (layers, blocks, heads, *shape), generator=g).to(torch.uint8).cuda(),
             torch.randn(layers, blocks, shape[0], heads, shape[1], generator=g).bfloat16().cuda(),
             torch.randn(layers, blocks, heads, generator=g).cuda()]
    order = torch.randperm(blocks, generator=g)
    sources, destinations = order[:13], order[13:26]
    sources[3] = sources[4]  # one block into two
    want = [pool.clone() for pool in pools]
    for pool in want:
        pool[:, destinations.cuda()] = pool[:, sources.cuda()]
    b200.b200_copy_kv_blocks(pools, sources.to(torch.int32).cuda(), destinations.to(torch.int32).cuda())
    assert all(torch.equal(a, b) for a, b in zip(pools, want))
    again = [pool.clone() for pool in pools]
    b200.b200_copy_kv_blocks(pools, sources.tolist(), destinations.tolist())
    b200.b200_copy_kv_blocks(pools, [], [])
    assert all(torch.equal(a, b) for a, b in zip(pools, again))
    b200.b200_copy_kv_blocks(pools[2:], torch.tensor([0, blocks, -1], dtype=torch.int32).cuda(),
                             torch.tensor([-1, 1, 2], dtype=torch.int32).cuda())
    with pytest.raises(kernels.KernelStatusError, match="position"):
        kernels.runtime().check_status()
    assert all(torch.equal(a, b) for a, b in zip(pools, again))


# ----------------------------------------------------------------------------------------------------------------- norm ----
def check_rows(codes, scales, y, slack):
    """Codes within half a step of y / scale, where `slack` (relative) is what 32-bit operations put on top."""
    most = y.abs().amax(-1)
    want = most / 127.0
    assert bool(((scales.cpu().double() - want).abs() <= slack * want).all())
    exact = torch.where(most[..., None] > 0, y / want.clamp_min(1e-300)[..., None], 0.0)
    assert float((codes.cpu().double() - exact).abs().max()) <= 0.5 + 127 * 5 * 2.0 ** -24
    assert bool((codes.cpu().abs().amax(-1) == torch.where(most > 0, 127, 0)).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,hidden", [(1, 896), (5, 16), (3, 1), (64, 3584), (7, 1001), (2, 20000), (700, 136), (1300, 2050)])
@pytest.mark.parametrize("residual", [False, True])
def test_norm_gives_the_sum_and_codes_of_the_definition(dtype, rows, hidden, residual):
    g = torch.Generator().manual_seed(rows * hidden)
    x = torch.randn(rows, hidden, generator=g).to(dtype)
    res = (2 * torch.randn(rows, hidden, generator=g)).to(dtype) if residual else None
    weight = (1 + 0.2 * torch.randn(hidden, generator=g)).to(dtype)
    if rows > 2:
        x[1] = 0
        if residual:
            res[1] = 0
    total, y = ref.norm(x, res, weight, 1e-6)
    codes, scales, sums = b200.b200_rms_norm_int8(x.cuda(), weight.cuda(), epsilon=1e-6,
                                                  residual=res.cuda() if residual else None)
    assert codes.dtype == torch.int8 and scales.dtype == torch.float32 and codes.shape == x.shape
    if residual:
        assert torch.equal(sums.cpu(), total)
    else:
        assert sums is None
    # a sum of `hidden` squares is off by at most hidden u, its root by half of that; four more operations
    check_rows(codes, scales, y, (hidden / 2 + 8) * 2.0 ** -24)


def test_norm_of_strided_higher_rank_and_unaligned_inputs():
    g = torch.Generator().manual_seed(1)
    wide = torch.randn(6, 300, generator=g).bfloat16().cuda()
    weight = torch.randn(128, generator=g).bfloat16().cuda()
    deep = wide[:, :128].contiguous().view(2, 3, 128)
    for x in (wide[:, 40:168], wide[:, 41:169], wide[:, :256:2], deep, deep.transpose(0, 1)):
        _, y = ref.norm(x, None, weight, 1e-5)
        codes, scales, _ = b200.b200_rms_norm_int8(x, weight, epsilon=1e-5)
        assert codes.shape == x.shape and scales.shape == x.shape[:-1]
        check_rows(codes, scales, y, 72 * 2.0 ** -24)
    res = torch.randn(6, 300, generator=g).bfloat16().cuda()[:, 3:131]
    total, y = ref.norm(wide[:, 8:136], res, weight, 1e-5)
    codes, scales, sums = b200.b200_rms_norm_int8(wide[:, 8:136], weight, epsilon=1e-5, residual=res)
    assert torch.equal(sums.cpu(), total)
    check_rows(codes, scales, y, 72 * 2.0 ** -24)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,hidden,stride", [(5200, 1024, 1024), (1500, 3584, 3600), (450, 20000, 20000)])
def test_rows_that_a_cta_takes_in_turn(dtype, rows, hidden, stride):
    """More rows than CTAs: each row is its own, whatever was in front of it; rows of zeros and of NaN among them."""
    g = torch.Generator().manual_seed(hidden)
    x = torch.randn(rows, stride, generator=g)[:, :hidden] * torch.exp2(torch.arange(rows) % 13 - 6.0)[:, None]
    x[7::100] = 0
    x = x.to(dtype)
    weight = (1 + 0.2 * torch.randn(hidden, generator=g)).to(dtype)
    bad = list(range(11, rows, 150))
    whole = torch.zeros(rows, stride, dtype=dtype, device="cuda")
    whole[:, :hidden] = x.cuda()
    on = whole[:, :hidden]
    on[bad, 3] = math.nan
    good = torch.ones(rows, dtype=torch.bool)
    good[bad] = False
    _, y = ref.norm(x, None, weight, 1e-6)
    for (codes, scales), want, slack in ((b200.b200_rms_norm_int8(on, weight.cuda(), epsilon=1e-6)[:2], y, hidden / 2 + 8),
                                         (b200.b200_quantize_rows_int8(on), x.double(), 2)):
        assert bool(scales[bad].isnan().all()) and not bool(codes[bad].any())
        check_rows(codes.cpu()[good], scales.cpu()[good], want[good], slack * 2.0 ** -24)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_rows_without_a_norm_and_rows_that_are_not_finite(dtype):
    g = torch.Generator().manual_seed(2)
    x = (torch.randn(9, 272, generator=g) * torch.exp2(torch.arange(9.0) * 2 - 8)[:, None]).to(dtype)
    codes, scales = b200.b200_quantize_rows_int8(x.cuda())
    check_rows(codes, scales, x.double(), 2.0 ** -23)
    x[1, 5], x[2, 6], x[3, 7] = math.inf, -math.inf, math.nan
    codes, scales = b200.b200_quantize_rows_int8(x.cuda())
    assert bool(scales[1:4].isnan().all()) and not bool(codes[1:4].any())
    check_rows(codes[4:], scales[4:], x[4:].double(), 2.0 ** -23)
    assert b200.b200_quantize_rows_int8(x.cuda()[:0])[0].shape == (0, 272)


# --------------------------------------------------------------------------------------------------------------- linear ----
def check_linear(g, m, k, n, epilogue="none", bias=False, dtype=torch.bfloat16, extreme=False):
    values = torch.randint(-127, 128, (m, k), generator=g, dtype=torch.int8)
    weight = torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int8)
    if extreme:  # the largest sums there are
        values[:] = -128
        weight[:] = torch.where(torch.arange(n)[:, None] % 2 == 0, -128, 127)
    scales = (torch.rand(m, generator=g) + 0.5) / 70
    weight_scales = (torch.rand(n, generator=g) + 0.5) / 70 / math.sqrt(k)
    b = torch.randn(n, generator=g).to(dtype) if bias else None
    res = torch.randn(m, n, generator=g).to(dtype) if epilogue == "residual" else None
    on = [t.cuda() if t is not None else None for t in (values, scales, weight, weight_scales, b, res)]
    got = b200.b200_linear_int8(*on[:5], residual=on[5], epilogue=epilogue, out_dtype=dtype)
    want, off = ref.linear(values, scales, weight, weight_scales, b, res, epilogue)
    got = got.cpu().double()
    bound = off + ref.HALF_STEP[dtype] * (want.abs() + off) + 2.0 ** -25
    worst = ((got - want).abs() / bound).max()
    assert float(worst) <= 1.0, f"{float(worst):.2f} of the bound"
    kernels.runtime().check_status()


@pytest.mark.parametrize("epilogue,bias", [("none", False), ("none", True), ("residual", False), ("residual", True),
                                           ("swiglu", False), ("swiglu", True)])
@pytest.mark.parametrize("m,k,n", [(1, 16, 2), (1, 896, 1152), (7, 144, 130), (16, 4864, 896), (33, 1024, 514), (64, 896, 9728),
                                   (65, 256, 62), (129, 208, 386), (200, 2048, 1000)])
def test_linear_of_sizes_and_epilogues(epilogue, bias, m, k, n):
    check_linear(torch.Generator().manual_seed(m + k + n), m, k, n, epilogue, bias)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m,k,n", [(1, 64, 1), (3, 80, 33), (40, 3584, 301), (128, 512, 255), (515, 304, 1027), (1100, 128, 777)])
def test_linear_of_types_and_odd_columns(dtype, m, k, n):
    g = torch.Generator().manual_seed(m + n)
    check_linear(g, m, k, n, dtype=dtype, bias=True)
    if n % 2 == 0 or n > 1:
        check_linear(g, m, k, n - n % 2, "swiglu", dtype=dtype)
        check_linear(g, m, k, n, "residual", dtype=dtype)


@pytest.mark.parametrize("m", [2, 100, 700])
def test_linear_sums_are_exact_up_to_the_largest(m):
    check_linear(torch.Generator().manual_seed(0), m, 131056, 40, dtype=torch.float32, extreme=True)


@pytest.mark.parametrize("m,k,n", [(2048, 896, 1152), (1300, 4864, 896), (4100, 144, 2000), (1025, 3584, 520)])
@pytest.mark.parametrize("epilogue", ["none", "residual", "swiglu"])
def test_linear_of_prompts(m, k, n, epilogue):
    check_linear(torch.Generator().manual_seed(m), m, k, n, epilogue, bias=epilogue != "residual")


@pytest.mark.parametrize("m,k,n", [(300, 2048, 200), (900, 4096, 37), (1025, 3584, 520), (3068, 1424, 106), (258, 18944, 130)])
@pytest.mark.parametrize("epilogue", ["none", "residual", "swiglu"])
def test_linear_of_many_rows_against_a_narrow_weight(m, k, n, epilogue):
    """(rows in chunks, K slices of a chunk where that fills the GPU)"""
    n -= n % 2 if epilogue == "swiglu" else 0
    check_linear(torch.Generator().manual_seed(m + n), m, k, n, epilogue, bias=True, dtype=torch.float16 if n % 4 else torch.bfloat16)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("epilogue", ["none", "residual", "swiglu"])
@pytest.mark.parametrize("m,k,n", [(260, 256, 20000), (260, 256, 20008), (260, 80, 20004), (260, 80, 20006), (260, 80, 20003),
                                   (2600, 144, 7976), (2600, 144, 7970)])
def test_linear_whose_pairs_take_several_tiles(m, k, n, epilogue, dtype):
    """Rows of y on multiples of 16, 8, 4 and 2 bytes, each pair of SMs with a few tiles, rows and columns that end inside one."""
    n -= n % 2 if epilogue == "swiglu" else 0
    check_linear(torch.Generator().manual_seed(m + n), m, k, n, epilogue, bias=epilogue != "none", dtype=dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("epilogue", ["none", "residual", "swiglu"])
@pytest.mark.parametrize("m,k,n", [(512, 4864, 896), (458, 9136, 1213), (520, 9136, 1800), (600, 9136, 1500), (250, 12000, 2500)])
def test_linear_whose_k_is_cut_between_pairs(m, k, n, epilogue, dtype):
    """Few tiles and a long K: two, three or four pairs of a cluster share a tile's products."""
    n -= n % 2 if epilogue == "swiglu" else 0
    check_linear(torch.Generator().manual_seed(m + n), m, k, n, epilogue, bias=epilogue != "none", dtype=dtype)


def test_linear_cut_between_pairs_sums_exactly_up_to_the_largest():
    check_linear(torch.Generator().manual_seed(0), 200, 131056, 1500, dtype=torch.float32, extreme=True)


def test_linear_of_a_prompt_sums_exactly_up_to_the_largest():
    check_linear(torch.Generator().manual_seed(0), 300, 131056, 1040, dtype=torch.float32, extreme=True)


@pytest.mark.parametrize("m,k,n,epilogue", [(64, 896, 9728, "swiglu"), (16, 4864, 896, "residual"), (8, 256, 40000, "none"),
                                            (48, 3584, 37888, "swiglu"), (1, 64, 64, "none"), (256, 1024, 3584, "residual")])
def test_linear_whose_weight_is_read_ahead(m, k, n, epilogue):
    """Chained launches that may read the weight while the kernel in front, which writes the rows, still runs: the results
    of launches one after another, whatever the rows were before."""
    g = torch.Generator().manual_seed(m + n)
    weight, scales = b200.b200_quantize_rows_int8(torch.randn(n, k, generator=g).bfloat16().cuda())
    norm = torch.ones(k, dtype=torch.bfloat16, device="cuda")
    rows = [torch.randn(m, k, generator=g).bfloat16().cuda() for _ in range(6)]
    residual = torch.randn(m, n, generator=g).bfloat16().cuda() if epilogue == "residual" else None
    def run(x):
        codes, row_scales, _ = b200.b200_rms_norm_int8(x, norm, epsilon=1e-6)
        return b200.b200_linear_int8(codes, row_scales, weight, scales, residual=residual, epilogue=epilogue)
    want = [run(x) for x in rows]
    torch.cuda.synchronize()
    with kernels.launch_mode(programmatic=True, constant_weights=True, keep_variants=True):
        got = [run(x) for x in rows]
        codes, row_scales, _ = b200.b200_rms_norm_int8(rows[0], norm, epsilon=1e-6)
        again = [b200.b200_linear_int8(codes, row_scales, weight, scales, residual=residual, epilogue=epilogue) for _ in range(3)]
    assert all(torch.equal(a, b) for a, b in zip(got + again, want + 3 * want[:1]))
    kernels.runtime().check_status()


@pytest.mark.parametrize("rows", [8, 600])
@pytest.mark.parametrize("offset", [1, 2, 4, 8])
def test_linear_residual_that_starts_anywhere(rows, offset):
    """A residual that is a slice of a longer vector: the result does not depend on where it starts."""
    g = torch.Generator().manual_seed(offset)
    values, weight = (torch.randint(-127, 128, (r, 256), generator=g, dtype=torch.int8).cuda() for r in (rows, 1024))
    scales = [torch.rand(r, generator=g).cuda() for r in (rows, 1024)]
    whole = torch.randn(rows * 1024 + 16, generator=g).bfloat16().cuda()
    part = whole[offset:offset + rows * 1024].view(rows, 1024)
    one, other = (b200.b200_linear_int8(values, scales[0], weight, scales[1], residual=residual, epilogue="residual")
                  for residual in (part, part.clone()))
    assert torch.equal(one, other)


def test_linear_keeps_leading_dimensions_and_passes_nan_scales_on():
    g = torch.Generator().manual_seed(0)
    values = torch.randint(-127, 128, (2, 3, 64), generator=g, dtype=torch.int8).cuda()
    weight = torch.randint(-127, 128, (10, 64), generator=g, dtype=torch.int8).cuda()
    scales = torch.rand(2, 3, generator=g).cuda()
    scales[1, 1] = math.nan
    y = b200.b200_linear_int8(values, scales, weight, torch.ones(10, device="cuda"))
    assert y.shape == (2, 3, 10)
    assert bool(y[1, 1].isnan().all()) and not bool(y[0].isnan().any())
    assert b200.b200_linear_int8(values[:0], scales[:0], weight, torch.ones(10, device="cuda")).shape == (0, 3, 10)


# ------------------------------------------------------------------------------------------------------------- together ----
def make_state(cache, *, batch=4, max_tokens=256, block_size=32, num_blocks=24, layers=2, kv_heads=2, dim=64):
    kind = QuantizedPagedKVCacheState if cache in CACHES else PagedKVCacheState
    return kind.allocate_paged(num_layers=layers, batch=batch, max_tokens=max_tokens, block_size=block_size,
                               num_blocks=num_blocks, kv_heads=kv_heads, head_dim=dim, dtype=cache, device="cuda")


@pytest.mark.parametrize("cache", [*CACHES, torch.bfloat16])
def test_a_server_stores_forks_appends_releases_and_compacts(cache):
    """Prompts, a fork in the middle of a block, appends to both branches, one released, the pool compacted: what every
    sequence reads stays its own."""
    g = torch.Generator().manual_seed(21)
    state = make_state(cache)
    state.reserve([70, 70, 0, 0], order=torch.randperm(24, generator=g).tolist())

    def rows(tokens):
        return torch.randn(4, 2, tokens, 64, generator=g).bfloat16().cuda()

    prompt = [rows(70), rows(70)]
    positions = torch.tensor([0, 0, -1, -1]).cuda()  # (the empty places take no part)
    for slot in range(2):
        state.store(slot, *prompt, positions)
    with pytest.raises(ExecutionError):
        state.check()
    state._length_arena[:, :2] = 70

    def read(sequence, tokens):
        return [[x.float() for x in state.gather(slot, sequence, tokens)] for slot in range(2)]

    def same(a, b):
        return all(torch.equal(x, y) for p, q in zip(a, b) for x, y in zip(p, q))

    first, second = read(0, 70), read(1, 70)
    assert state.blocks_in_use() == 6
    state.fork(0, 2, tokens=70)     # two whole blocks shared, the third copied
    assert state.blocks_in_use() == 7 and state._host_table[2][:2] == state._host_table[0][:2]
    state.fork(0, 3, tokens=64)     # whole blocks alone: nothing to copy
    assert state.blocks_in_use() == 7 and state.lengths[1].tolist() == [70, 70, 70, 64]
    assert same(read(2, 70), first)
    with pytest.raises(ExecutionError, match="still holds"):
        state.fork(0, 2)
    state.release(3)
    with pytest.raises(ExecutionError, match="does not hold"):
        state.fork(1, 3, tokens=999)
    state.fork(0, 3, tokens=64)
    state.reserve([71, 71, 71, 65])
    new = [rows(1), rows(1)]
    lengths = torch.tensor([70, 70, 70, 64])
    for slot in range(2):
        state.store(slot, *new, lengths.cuda())
    state.check()
    # the appended rows differ; the shared blocks, and sequence 1, are as they were
    whole = [[x[:64] for x in pair] for pair in first]
    for sequence in (0, 2, 3):
        assert same(read(sequence, 64), whole)
    before = [read(s, n) for s, n in enumerate((71, 71, 71, 65))]
    assert not torch.equal(before[0][0][0][70], before[2][0][0][70])
    state.release(0)
    assert state.blocks_in_use() == 7  # three of 1, the two that 2 and 3 share, one of each: 0's own last block is free
    assert state.compact() == 7
    assert max(b for row in state._host_table for b in row) == 6
    assert all(same(read(s, n), before[s]) for s, n in ((1, 71), (2, 71), (3, 65)))
    assert state._host_table[2][:2] == state._host_table[3][:2]
    state._length_arena[:2] = torch.tensor([0, 71, 71, 65]).cuda()
    query = torch.randn(4, 14, 1, 64, generator=g).bfloat16()
    out = state.decode_attention(1, query.cuda(), None, groups=7, scale=0.125).cpu().double()
    table = state.block_table.cpu()
    if cache in CACHES:
        caches = [ref.Cache(state.keys[1], state.key_scales[1]), ref.Cache(state.values[1], state.value_scales[1])]
        want, bound = ref.attention(query, *caches, table, [0, 71, 71, 65], None, 0.125)
        assert bool(((out - want).abs()[1:] <= bound[1:]).all()) and bool(out[0].isnan().all())
    state.release(2)
    state.release(3)
    state.release(1)
    assert state.blocks_in_use() == 0 and len(state._free) == 24 and state.compact() == 0


def test_a_layer_in_8_bits_step_by_step():
    """norm -> q|k|v -> RoPE -> store -> attention -> o onto the residual -> norm -> gate|up -> down, each step against its
    definition on what the step before left, over a prompt and three decode steps."""
    g = torch.Generator().manual_seed(31)
    hidden, heads, kv_heads, dim, inter, batch = 256, 4, 2, 64, 512, 3
    weights = {name: b200.b200_quantize_rows_int8((torch.randn(n, k, generator=g) / math.sqrt(k)).bfloat16().cuda())
               for name, n, k in (("qkv", (heads + 2 * kv_heads) * dim, hidden), ("o", hidden, heads * dim),
                                  ("gate_up", 2 * inter, hidden), ("down", hidden, inter))}
    bias = torch.randn((heads + 2 * kv_heads) * dim, generator=g).bfloat16().cuda()
    norms = [(1 + 0.1 * torch.randn(hidden, generator=g)).bfloat16().cuda() for _ in range(2)]
    state = make_state(torch.int8, batch=batch, layers=1, block_size=32, num_blocks=16)
    inv_freq = (10000.0 ** (-torch.arange(0, dim, 2).float() / dim)).cuda()
    cached = None

    def project(name, codes, scales, *args, **kwargs):
        y = b200.b200_linear_int8(codes, scales, *weights[name], *args, **kwargs)
        want, off = ref.linear(codes, scales, *weights[name], args[0] if args else None, kwargs.get("residual"),
                               kwargs.get("epilogue", "none"))
        got = y.cpu().double().flatten(0, -2)
        assert bool(((got - want).abs() <= off + 2.0 ** -8 * (want.abs() + off) + 1e-30).all())
        return y

    position = 0
    for tokens in (40, 1, 1, 1):
        x = torch.randn(batch, tokens, hidden, generator=g).bfloat16().cuda()
        state.reserve([position + tokens] * batch)
        if cached is None:
            cached = [ref.Cache(state.keys[0], state.key_scales[0]), ref.Cache(state.values[0], state.value_scales[0])]
        codes, scales, _ = b200.b200_rms_norm_int8(x, norms[0], epsilon=1e-6)
        check_rows(codes, scales, ref.norm(x, None, norms[0], 1e-6)[1], 136 * 2.0 ** -24)
        qkv = project("qkv", codes, scales, bias)
        q, k, v = (part.view(batch, tokens, -1, dim).transpose(1, 2)
                   for part in qkv.split([heads * dim, kv_heads * dim, kv_heads * dim], dim=2))
        ids = torch.arange(position, position + tokens).expand(batch, tokens).contiguous().cuda()
        cosine, sine = b200.b200_rope_table(ids, inv_freq, torch.bfloat16)
        q, k = b200.b200_rope(q, k, cosine, sine)
        table = state.block_table.cpu()
        at = torch.full((batch,), position, dtype=torch.int64)
        state.store(0, k, v, at.cuda())
        for cache, new in zip(cached, (k, v)):
            cache.store(table, new, at)
        assert same_codes(state.keys[0], cached[0]) and same_codes(state.values[0], cached[1])
        position += tokens
        state = state.advance(0, delta=tokens)
        if tokens > 1:
            continue
        attended = state.decode_attention(0, q, None, groups=heads // kv_heads, scale=dim ** -0.5)
        want, bound = ref.attention(q, *cached, table, [position] * batch, None, dim ** -0.5)
        assert bool(((attended.cpu().double() - want).abs() <= bound).all())
        rows = attended.view(batch, heads * dim)
        o = project("o", *b200.b200_quantize_rows_int8(rows))
        codes, scales, x = b200.b200_rms_norm_int8(o, norms[1], epsilon=1e-6, residual=x.view(batch, hidden))
        gated = project("gate_up", codes, scales, epilogue="swiglu")
        x = project("down", *b200.b200_quantize_rows_int8(gated), residual=x, epilogue="residual")
        assert bool(x.isfinite().all())
    state.check()


@pytest.mark.parametrize("weights_dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cache", CACHES)
def test_an_engine_serves_from_a_cache_in_8_bits(cache, weights_dtype):
    """The prompt's cache is the definition's of the keys and values that the 16-bit engine caches; a captured step gives the
    launched one's tokens; attention over the quantised prompt keeps the logits near the 16-bit engine's."""
    config = q2.Qwen2Config(hidden_size=256, intermediate_size=512, num_layers=2, num_heads=4, num_kv_heads=2, rms_norm_eps=1e-6,
                            rope_theta=1e6, vocab_size=512, tie_word_embeddings=True)
    weights = {k: v.cuda() for k, v in q2.make_weights(config, seed=1, dtype=weights_dtype).items()}
    prompt = q2.make_prompt_ids(config, 3, 77, seed=2)
    make = lambda **options: Qwen2Engine(config, weights, batch=3, capacity=160, **options)
    plain = make()
    engine, other = (make(kv_layout="paged", block_size=32, kv_dtype=cache) for _ in range(2))
    assert isinstance(engine.state, QuantizedPagedKVCacheState) and engine.state.keys[0].dtype == cache
    empty = [ref.Cache(engine.state.keys[0], engine.state.key_scales[0]), ref.Cache(engine.state.values[0], engine.state.value_scales[0])]
    wide, logits = plain.prefill(prompt), engine.prefill(prompt)
    assert torch.equal(logits, wide)  # (a prompt attends in 16 bits)
    # layer 0, whose inputs are the same whatever the launches: what the 16-bit engine caches, quantised
    table = engine.state.block_table.cpu()
    for cached, buffer, pool, scales in zip(empty, (plain.state.keys[0], plain.state.values[0]),
                                            (engine.state.keys[0], engine.state.values[0]),
                                            (engine.state.key_scales[0], engine.state.value_scales[0])):
        cached.store(table, buffer[:, :77].transpose(1, 2), torch.zeros(3, dtype=torch.int64))
        assert torch.equal(scales.cpu().double(), cached.scales) and same_codes(pool, cached)
    tokens = engine.generate(prompt, 40)            # captured
    assert torch.equal(other.generate(prompt, 40, use_graph=False), tokens)
    for b in range(3):  # (the blocks themselves lie elsewhere: one engine has given its own back and taken new ones)
        for mine, theirs in zip(engine.state.gather(1, b, 116), other.state.gather(1, b, 116)):
            assert torch.equal(mine, theirs)
    engine.state.check()
    # one step behind the prompt: scores and values off by at most half a code each of their block's largest
    engine.prefill(prompt)
    plain.prefill(prompt)
    plain.decode_step(feed_back=False)
    engine.decode_step(feed_back=False)
    off = (engine.logits.float() - plain.logits.float()).norm() / plain.logits.float().norm()
    assert float(off) < (0.05 if cache == torch.int8 else 0.2)
    with pytest.raises(ValueError, match="8 bits"):
        make(kv_dtype=cache)
    with pytest.raises(ValueError, match="8 bits"):
        make(kv_layout="paged", kv_dtype=torch.int16)


@pytest.mark.parametrize("cache", [None, torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("tokens", [64, 77])
def test_an_engine_forks_a_sequence(cache, tokens):
    """A branch gives the tokens of the sequence it comes from while its input does, another input moves it alone; capturing
    a step stores nothing in an 8-bit cache."""
    config = q2.Qwen2Config(hidden_size=256, intermediate_size=512, num_layers=2, num_heads=4, num_kv_heads=2, rms_norm_eps=1e-6,
                            rope_theta=1e6, vocab_size=512, tie_word_embeddings=True)
    weights = {k: v.cuda() for k, v in q2.make_weights(config, seed=1, dtype=torch.bfloat16).items()}
    prompt = q2.make_prompt_ids(config, 3, tokens, seed=2)
    make = lambda: Qwen2Engine(config, weights, batch=3, capacity=160, kv_layout="paged", block_size=32, kv_dtype=cache)
    engine, apart = make(), make()
    expected = apart.generate(prompt, 24)
    engine.prefill(prompt)
    if cache is not None:
        pools = [pool.clone() for pool in engine.state._pools]
        engine.capture()
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(pools, engine.state._pools))
    else:
        engine.capture()
    rows = [engine.input_ids.clone()]  # (next_ids holds the warm-up's)
    for step in range(24):
        if step == 5:
            engine.fork(0, 2)
        rows.append(engine.decode_step().clone())
    rows = torch.stack(rows, dim=1)
    assert torch.equal(rows[:2], expected[:2])                                  # the others go on as they would have
    assert torch.equal(rows[2, :6], expected[2, :6]) and torch.equal(rows[2, 6:], expected[0, 6:])
    assert engine.state.blocks_in_use() < sum(len(row) for row in engine.state._host_table)
    engine.prefill(prompt)                                                      # shared blocks are given back
    assert engine.state._sharers == {}
    engine.fork(1, 0)
    engine.input_ids[0] = (engine.input_ids[1] + 1) % 512
    rows = torch.stack([engine.decode_step().clone() for _ in range(8)], dim=1)
    assert torch.equal(rows[1], expected[1, 1:9])
    engine.state.check()
    for arguments in ((1, 1), (0, 9), (0, -1)):
        with pytest.raises(ExecutionError):
            engine.fork(*arguments)
    with pytest.raises(ExecutionError, match="paged"):
        Qwen2Engine(config, weights, batch=2, capacity=64).fork(0, 1)


@pytest.mark.parametrize("layout", [{}, dict(kv_layout="paged", block_size=32), dict(kv_layout="paged", block_size=32, kv_dtype=torch.int8)])
@pytest.mark.parametrize("weights_dtype", [torch.bfloat16, torch.float16])
def test_an_engine_projects_in_8_bit_integers(layout, weights_dtype):
    """It runs on every layout, captured as launched, and its logits stay near the 16-bit engine's: weights and rows are
    each off by at most half a code of their row's largest, a few tenths of a percent of the sums."""
    config = q2.Qwen2Config(hidden_size=256, intermediate_size=512, num_layers=2, num_heads=4, num_kv_heads=2, rms_norm_eps=1e-6,
                            rope_theta=1e6, vocab_size=512, tie_word_embeddings=True)
    if weights_dtype == torch.float16 and layout and "kv_dtype" not in layout:
        pytest.skip("the 16-bit paged layout holds bf16")
    weights = {k: v.cuda() for k, v in q2.make_weights(config, seed=1, dtype=weights_dtype).items()}
    prompt = q2.make_prompt_ids(config, 3, 77, seed=2)
    make = lambda **options: Qwen2Engine(config, weights, batch=3, capacity=160, **layout, **options)
    plain, engine, other = make(), make(weight_dtype=torch.int8), make(weight_dtype=torch.int8)
    assert engine.layers[0]["o_w"][0].dtype == torch.int8
    assert torch.equal(engine.generate(prompt, 30), other.generate(prompt, 30, use_graph=False))
    wide, logits = plain.prefill(prompt).float(), engine.prefill(prompt).float()
    assert float((logits - wide).norm() / wide.norm()) < 0.1
    plain.decode_step(feed_back=False)
    engine.decode_step(feed_back=False)
    assert float((engine.logits.float() - plain.logits.float()).norm() / plain.logits.float().norm()) < 0.1
    engine.state.check()
    with pytest.raises(ValueError, match="8-bit projections"):
        make(weight_dtype=torch.int16)
