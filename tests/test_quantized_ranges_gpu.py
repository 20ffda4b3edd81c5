"""Operators in 8 bits over the whole range of what they may be given: values of any size, value blocks any distance apart, tails of small
probabilities behind a token that dominates, tables of more than 2^24 tiles, rows of tiny numbers."""

import math

import pytest
import torch

import llm_compiler_b200 as b200
import quantized_helpers as ref
from llm_compiler_b200 import kernels

pytestmark = pytest.mark.gpu
CACHES = [torch.int8, torch.float8_e4m3fn]


def attention(query, keys, values, table, length, mask, scale):
    """(result, bound on the kernel's distance from it) of one sequence, 1 x Hq x 1 x D, in 64 bits.

    With A = sum p|v|, an element of the result is off by
     - its own rounding;
     - a probability's rounding to fp16: 2^-11 of it (fp16 results, two numbers: 2^-22), or, where that is less, half of
       fp16's smallest step, which is 2^-34 of the largest probability (2^-25 on numbers that are carried 2^11 higher, a block's
       scale at least a quarter of its reference), and never more than the probability itself;
     - the scores: products of D terms in 32 bits, (D + 4) u of the sum of magnitudes, 2^-25 of the query's largest times the
       keys' sum, a mask's addition; twice, for the normalisation;
     - exponentials good to 2^-21 of arguments (in units of log 2) of up to 64, rounded to u: 2^-18;
     - sums in 32 bits: a warp of four adds a product of 16 tokens at a time, four roundings each, and its lanes' sums of
       probabilities one of 8 tokens at a time; merges and rescalings 64 u."""
    u = 2.0 ** -24
    half = ref.HALF_STEP[query.dtype]
    probability = 2.0 ** -11 if query.dtype == torch.bfloat16 else 2.0 ** -22
    smallest = 2.0 ** -25 if query.dtype == torch.float16 else 2.0 ** -133
    q = query.double()
    _, heads, _, dim = q.shape
    out, bound = torch.empty_like(q), torch.empty_like(q)
    k, v = keys.rows(table[0], length), values.rows(table[0], length)
    group = heads // k.shape[0]
    for h in range(heads):
        kk, vv, one = k[h // group], v[h // group], q[0, h, 0]
        scores = kk @ one * scale
        slack = ((dim + 4) * u * (kk.abs() @ one.abs()) + 2.0 ** -25 * one.abs().max() * kk.abs().sum(1)) * scale
        if mask is not None:
            scores = scores + mask[0, 0, 0, :length].double()
            slack = slack + u * scores.abs().nan_to_num(0.0, 0.0, 0.0)
        p = torch.softmax(scores, 0)
        out[0, h, 0] = p @ vv
        a = p @ vv.abs()
        rounding = torch.maximum(probability * p, torch.minimum(p, 2.0 ** -34 * p.max())) @ vv.abs()
        off = 2 * float(torch.where(p > 0, slack, 0.0).max())
        sums = u * (length / 64 * 4 + length / 32 + 64)
        bound[0, h, 0] = half * out[0, h, 0].abs() + rounding + a * (off + 2.0 ** -18 + sums) + smallest
    return out, bound


def check(query, pools, scales, table, length, mask, scale, **options):
    want, bound = attention(query, ref.Cache(pools[0], scales[0]), ref.Cache(pools[1], scales[1]), table, length, mask, scale)
    got = b200.b200_paged_decode_attention_8bit(query.cuda(), *pools, *scales, table.cuda(), torch.tensor([length]).cuda(),
                                                None if mask is None else mask.cuda(), scale=scale, **options)
    got = got.cpu().double()
    assert bool(want.isfinite().all()) and bool(got.isfinite().all())
    worst = float(((got - want).abs() / bound).max())
    assert worst <= 1.0, f"{worst:.3g} of the bound"
    kernels.runtime().check_status()


def random_codes(g, cache, blocks, heads, size, dim):
    top = ref.TOP[cache]
    codes = (torch.randn(blocks, heads, size, dim, generator=g) * top / 3).clamp(-top, top)
    return (codes.round() if cache == torch.int8 else codes).to(cache).cuda()


# what the blocks' value scales are, 2^x, four blocks (a tile for each warp) at a time
PATTERNS = {
    "tiny-first": [-73, -6], "tinier-first": [-100, -6], "tiny-last": [-6, -100], "zero-like": [-126, -5, -126, -6],
    "70-up": [-40, 30], "70-down": [30, -40], "120-up": [-90, 30], "120-down": [30, -90],
    "down-and-down": [0, -58, -116], "down-down-up": [0, -59, -118, 20, -20], "up-and-up": [-118, -59, 0],
    "sawtooth": [-10, 60, -30, 90, -110, 5],
}


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("dtype,dim,heads", [(torch.bfloat16, 64, 4), (torch.bfloat16, 128, 12), (torch.bfloat16, 256, 3)])
@pytest.mark.parametrize("pattern", PATTERNS)
@pytest.mark.parametrize("visible", ["all", "smallest", "largest"])
def test_attention_of_value_blocks_any_distance_apart(cache, dtype, dim, heads, pattern, visible):
    """All blocks weigh alike, or those of the smallest (largest) scale alone: the others are masked out, in front and behind.
    (bf16 values, whose scales lie between 2^-126 and 2^121.)"""
    g = torch.Generator().manual_seed(dim)
    exponents = [e for e in PATTERNS[pattern] for _ in range(4)]
    blocks, size = len(exponents), 32
    pools = [random_codes(g, cache, blocks, 1, size, dim) for _ in range(2)]
    top = ref.TOP[cache]
    scales = [torch.full((blocks, 1), 3.0 / top), (1 + torch.rand(blocks, 1, generator=g)) * torch.tensor(
        [[2.0 ** e] for e in exponents])]
    table = torch.randperm(blocks, generator=g).to(torch.int32).view(1, blocks)
    scales[1][table[0].long()] = scales[1].clone()  # (block i of the sequence has the i-th scale)
    scales = [s.cuda() for s in scales]
    length = blocks * size - 5
    mask = None
    if visible != "all":
        keep = min(exponents) if visible == "smallest" else max(exponents)
        mask = torch.full((1, 1, 1, length), -math.inf)
        for i, e in enumerate(exponents):
            if e == keep:
                mask[..., i * size:(i + 1) * size] = 0.0
    query = torch.randn(1, heads, 1, dim, generator=g).to(dtype)
    for split_tokens in (0, blocks * size):  # a tile a warp, and all of them in turn
        check(query, pools, scales, table, length, mask, dim ** -0.5, split_tokens=split_tokens)


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("seed", range(6))
def test_attention_of_value_blocks_at_random_distances_and_probabilities(cache, seed):
    """Scales anywhere in bf16's range, scores from a few units to a hundred apart."""
    g = torch.Generator().manual_seed(seed)
    blocks, size, dim, heads = 40, 32, 64, 6
    pools = [random_codes(g, cache, blocks, 2, size, dim) for _ in range(2)]
    scales = [torch.full((blocks, 2), 3.0 / ref.TOP[cache]).cuda(),
              torch.exp2(-126 + 226 * torch.rand(blocks, 2, generator=g)).cuda()]
    table = torch.randperm(blocks, generator=g).to(torch.int32).view(1, blocks)
    query = (torch.randn(1, heads, 1, dim, generator=g) * [0.1, 1.0, 10.0][seed % 3]).bfloat16()
    for split_tokens in (0, 320, blocks * size):
        check(query, pools, scales, table, blocks * size - 3, None, 0.125, split_tokens=split_tokens)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("above", [8, 14, 18])
@pytest.mark.parametrize("ratio", [1.0, 3.9, 12.0, 0.1])
@pytest.mark.parametrize("masked", [False, True])
def test_attention_of_a_long_tail_behind_a_token_that_dominates(dtype, cache, above, ratio, masked):
    """One token `above` the others' scores whose value is zero, in a block of `ratio` times the others' value scale: the
    result is the tail's alone, each probability of it some e^-above of the largest."""
    g = torch.Generator().manual_seed(above)
    length, size, dim, heads = 30100, 128, 64, 4
    blocks = -(-length // size)
    top = ref.TOP[cache]
    keys = torch.zeros(blocks, 1, size, dim)
    values = 40 + (top - 40) * torch.rand(blocks, 1, size, dim, generator=g)  # of one sign
    at = 1000
    keys[at // size, 0, at % size, 0] = 100.0
    values[at // size, 0, at % size] = 0.0
    pools = [(x.round() if cache == torch.int8 else x).to(cache).cuda() for x in (keys, values)]
    scales = [torch.full((blocks, 1), 0.01).cuda(), torch.full((blocks, 1), 1.0 / top).cuda()]
    scales[1][at // size] *= ratio
    query = torch.zeros(1, heads, 1, dim)
    query[..., 0] = above / 0.125
    query[:, :, :, 1:] = torch.randn(1, heads, 1, dim - 1, generator=g)
    table = torch.arange(blocks, dtype=torch.int32).view(1, blocks)
    mask = torch.zeros(1, 1, 1, length) if masked else None
    check(query.to(dtype), pools, scales, table, length, mask, 0.125)
    check(query.to(dtype), pools, scales, table, length, mask, 0.125, split_tokens=length)


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("dtype,dim,heads", [(torch.bfloat16, 64, 4), (torch.bfloat16, 128, 12), (torch.bfloat16, 256, 3)])
@pytest.mark.parametrize("largest", [2.0 ** 127, 2.0 ** -120])
def test_attention_of_values_at_the_ends_of_their_range(cache, dtype, dim, heads, largest):
    """Values up to half of fp32's largest number, thousands of them of one sign and of one weight, and down to its smallest: the
    result lies among them, though their sum does not."""
    g = torch.Generator().manual_seed(dim)
    length, size = 5000, 32
    blocks = -(-length // size)
    top = ref.TOP[cache]
    pools = [random_codes(g, cache, blocks, 1, size, dim) for _ in range(2)]
    pools[1] = pools[1].float().abs().to(cache)
    scales = [torch.full((blocks, 1), 1.0 / top).cuda(), (largest / top * (0.5 + 0.5 * torch.rand(blocks, 1, generator=g))).cuda()]
    table = torch.randperm(blocks, generator=g).to(torch.int32).view(1, blocks)
    query = torch.randn(1, heads, 1, dim, generator=g).to(dtype)
    for split_tokens in (0, length, 800, 256):  # the library's choice, one CTA, a cluster, partials in the workspace
        check(query, pools, scales, table, length, None, dim ** -0.5, split_tokens=split_tokens)


@pytest.mark.parametrize("size,columns", [(32, (1 << 24) + 2), (96, 5592406 + 3)])
def test_attention_behind_the_first_half_billion_tokens(size, columns):
    """A table of more than 2^24 tiles whose entries share a block, all but the last two: their tokens' scores are 40 above the
    others', so that the e^20 of those weigh e^-20 of them, and the result is those two blocks' mean."""
    g = torch.Generator().manual_seed(0)
    dim = 64
    keys = torch.zeros(3, 1, size, dim, dtype=torch.int8)
    keys[1:, :, :, 0] = 100
    pools = [keys.cuda(), torch.randint(-127, 128, (3, 1, size, dim), generator=g, dtype=torch.int8).cuda()]
    scales = [torch.full((3, 1), 0.01).cuda(), torch.full((3, 1), 1 / 127).cuda()]
    table = torch.zeros(1, columns, dtype=torch.int32, device="cuda")
    table[0, -2:] = torch.tensor([1, 2], dtype=torch.int32)
    query = torch.zeros(1, 2, 1, dim, dtype=torch.bfloat16, device="cuda")
    query[..., 0] = 320.0
    got = b200.b200_paged_decode_attention_8bit(query, *pools, *scales, table, torch.tensor([columns * size - 7]).cuda(), None,
                                                scale=0.125).cpu().double()
    values = torch.cat([pools[1][1, 0], pools[1][2, 0, :-7]]).cpu().double() / 127
    want = values.mean(0)
    # the result's rounding, a probability's, and the others' weight: e^-40 each of some 2^29 tokens, against 57 and more
    others = columns * size * math.exp(-40) / values.shape[0]
    bound = 2.0 ** -8 * want.abs() + 2.0 ** -10 * values.abs().mean(0) + 2 * others + 2.0 ** -18
    assert bool(((got - want).abs() <= bound).all())
    kernels.runtime().check_status()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,hidden", [(12, 136), (12, 1001), (900, 2048)])
def test_rows_of_tiny_numbers(dtype, rows, hidden):
    """Rows whose largest magnitude is 2^-112 .. 2^-149, fp32's end, without a norm and behind one: codes * scales stand for
    the row to half a step of its scale, which is the largest magnitude / 127 and no less than the smallest normal number
    (behind a norm: times the row's factor)."""
    g = torch.Generator().manual_seed(hidden)
    lowest = -149 if dtype == torch.float32 else -133
    x = 2 * torch.rand(rows, hidden, generator=g, dtype=torch.float64) - 1
    x = (x * torch.exp2(torch.linspace(-112, lowest, rows, dtype=torch.float64))[:, None]).to(dtype)
    weight = (1 + 0.2 * torch.randn(hidden, generator=g)).to(dtype)
    zeros = torch.zeros_like(x)
    r = x.double()
    weighted = r * weight.double()
    factor = 1.0 / torch.sqrt((r * r).mean(-1) + 1e-6)
    plain = b200.b200_quantize_rows_int8(x.cuda())
    normed = b200.b200_rms_norm_int8(x.cuda(), weight.cuda(), epsilon=1e-6)[:2]
    behind = b200.b200_rms_norm_int8(zeros.cuda(), weight.cuda(), epsilon=1e-6, residual=x.cuda())[:2]
    for (codes, scales), y, by in ((plain, r, torch.ones(rows, dtype=torch.float64)), (normed, weighted, factor), (behind, weighted, factor)):
        codes, scales = codes.cpu().double(), scales.cpu().double()
        most = y.abs().amax(-1)
        step = torch.where(most > 0, (most / 127).clamp_min(ref.SMALLEST), 0.0)
        # a product with a weight is rounded to 2^-149 here, half of that off; 1 / 127, the product with it, the sum of squares,
        # its root and the last product: 8 u
        assert bool(((scales - step * by).abs() <= by * (8 * 2.0 ** -24 * step + 2.0 ** -150)).all())
        off = (codes - y / step.clamp_min(1e-300)[:, None]).abs()
        assert float(torch.where(most[:, None] > 0, off, 0.0).max()) <= 0.5 + 127 * 5 * 2.0 ** -24 + 2.0 ** -150 / ref.SMALLEST
        assert not bool(codes[most == 0].any())
