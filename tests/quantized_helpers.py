"""64-bit forms of the operators in 8 bits, from their definitions, on the CPU."""

import math

import torch

TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
SMALLEST = 2.0 ** -126
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def f32(x):
    """A 64-bit number rounded to 32 bits: one IEEE operation on 32-bit operands is that of its 64-bit result."""
    return x.float().double()


def code(x, dtype):
    """The nearest code, ties to even, saturating; NaN becomes 0 as an integer and stays NaN as e4m3."""
    if dtype == torch.int8:
        return torch.round(x.nan_to_num(0.0, math.inf, -math.inf).clamp(-127, 127))
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6).clamp_max(2.0 ** 100))) - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


class Cache:
    """A cache in 8 bits of one kind (keys or values): codes as 64-bit numbers, scales."""

    def __init__(self, pool, scales):
        self.dtype = pool.dtype
        self.codes, self.scales = pool.cpu().float().double(), scales.cpu().double()

    def store(self, table, x, positions):
        """x: B x H x T x D."""
        x = x.cpu().double()
        size = self.codes.shape[2]
        inverse_top = f32(torch.tensor(1.0 / TOP[self.dtype], dtype=torch.float64))
        for b, position in enumerate(positions.tolist()):
            if position < 0:
                continue
            for column in range(position // size, -(-(position + x.shape[2]) // size)):
                if column >= table.shape[1] or not 0 <= int(table[b, column]) < self.codes.shape[0]:
                    continue
                at = int(table[b, column])
                lo, hi = max(position, column * size), min(position + x.shape[2], (column + 1) * size)
                new = x[b, :, lo - position:hi - position]
                most = torch.where(new.isfinite(), new.abs(), 0.0).amax((1, 2))
                scale = torch.where(most > 0, f32(most * inverse_top).clamp_min(SMALLEST), 0.0)
                held = lo - column * size
                if held:
                    before = self.scales[at].clone()
                    scale = torch.maximum(scale, before)
                    grown = scale > before
                    ratio = f32(before / scale.clamp_min(SMALLEST))
                    anew = code(f32(self.codes[at, :, :held] * ratio[:, None, None]), self.dtype)
                    self.codes[at, :, :held] = torch.where(grown[:, None, None], anew, self.codes[at, :, :held])
                inverse = torch.where(scale > 0, f32(1.0 / scale.clamp_min(SMALLEST)), 0.0)
                self.codes[at, :, held:hi - column * size] = code(f32(new * inverse[:, None, None]), self.dtype)
                self.scales[at] = scale

    def rows(self, table_row, length):
        """H x length x D values."""
        blocks = table_row[:-(-length // self.codes.shape[2])].long()
        x = self.codes[blocks] * self.scales[blocks][:, :, None, None]
        return x.transpose(0, 1).flatten(1, 2)[:, :length]


def attention(query, keys, values, table, lengths, mask, scale):
    """(result, bound on the kernels' distance from it): B x Hq x 1 x D.

    The bound, with A = sum p|v| / sum p and u = 2^-24: the result's own rounding; a probability rounded to fp16 (2^-11 of
    it; 2^-22 for fp16 results, where two numbers hold it), or to 2^-25 of the largest where that is coarser (times 16: block
    scales up to 16 apart share an accumulator); scores from products of D terms in 32 bits, each off by at most (D + 4) u of
    the sum of magnitudes, and by 2^-25 of the query's largest times the keys' sum (its smallest elements in fp16), which
    moves a probability by that much and its normalisation by as much again; sums of `length` terms; an exponential good to
    2^-21."""
    query = query.cpu()
    half = HALF_STEP[query.dtype]
    probability = 2.0 ** -11 if query.dtype == torch.bfloat16 else 2.0 ** -22
    q = query.double()
    batch, heads, _, dim = q.shape
    out, bound = torch.empty_like(q), torch.empty_like(q)
    u = 2.0 ** -24
    for b in range(batch):
        length = int(lengths[b])
        k, v = keys.rows(table[b], length), values.rows(table[b], length)
        group = heads // k.shape[0]
        for h in range(heads):
            kk, vv = k[h // group], v[h // group]
            scores = kk @ q[b, h, 0] * scale
            slack = ((dim + 4) * u * (kk.abs() @ q[b, h, 0].abs()) + 2.0 ** -25 * q[b, h, 0].abs().max() * kk.abs().sum(1)) * scale
            if mask is not None:
                extra = mask[b, 0, 0, :length].double()
                scores = scores + extra
                slack = slack + u * scores.abs().nan_to_num(0.0, 0.0, 0.0)
            p = torch.softmax(scores, 0) if length else scores
            out[b, h, 0] = (p[:, None] * vv).sum(0) if length else math.nan
            a = (p[:, None] * vv.abs()).sum(0)
            largest = vv.abs().max() if length else 0.0
            off = 2 * slack.nan_to_num(0.0, 0.0, 0.0).max() if length else 0.0
            peak = p.max() if length else 0.0
            bound[b, h, 0] = half * out[b, h, 0].abs() + a * (probability + 2.0 ** -21 + 2 * u * length + off) + \
                16 * 2.0 ** -25 * length * largest * peak + 1e-30
    return out, bound


def norm(x, residual, weight, epsilon):
    """(rows behind the sum, y): x in its own type, y in 64 bits."""
    total = x.cpu()
    if residual is not None:
        total = (total.float() + residual.cpu().float()).to(x.dtype)
    r = total.double()
    y = r if weight is None else r / torch.sqrt((r * r).mean(-1, keepdim=True) + epsilon) * weight.cpu().double()
    return total, y


def linear(values, scales, weight, weight_scales, bias, residual, epilogue):
    """(result, bound without the output's rounding) in 64 bits. An integer sum becomes 32 bits, is scaled twice and takes
    the bias: four roundings of u. SwiGLU: silu moves by at most 1.1 of a change of its argument; its exponential, quotient
    and product add 8 u (an exponential good to 4 u of a result the exponent of which is off by u |gate|)."""
    u = 2.0 ** -24
    y = values.cpu().double().flatten(0, -2) @ weight.cpu().double().T
    y = y * scales.cpu().double().flatten()[:, None] * weight_scales.cpu().double()[None]
    off = 3 * u * y.abs()
    if bias is not None:
        y = y + bias.cpu().double()
        off = off + u * y.abs()
    if epilogue == "swiglu":
        gate, up = y[:, 0::2], y[:, 1::2]
        g_off, u_off = off[:, 0::2], off[:, 1::2]
        silu = gate / (1.0 + torch.exp(-gate))
        y = silu * up
        off = 1.1 * g_off * up.abs() + silu.abs() * u_off + (8 + 2 * gate.abs()) * u * y.abs()
    elif epilogue == "residual":
        y = y + residual.cpu().double().flatten(0, -2)
        off = off + u * y.abs()
    return y, off
