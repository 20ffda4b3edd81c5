"""Operators of serving in 8 bits, as measurable cases: a paged cache held in 8 bits with a scale for each block of tokens
and KV head, the attention that reads it, copies of its blocks, and projections in 8-bit integers behind a norm that
quantises its output.

Five kinds of case:
  attention  one query token a sequence over the cached keys and values of that sequence, read through a block table
  store      new tokens' keys and values, quantised into their blocks; a block that is half full keeps what it holds, and
             its scale only grows
  copy       blocks copied to other blocks in every layer's pool (a sequence that is forked, a pool that is compacted)
  norm       residual sum, RMS norm and quantisation of each row to 8-bit integers
  linear     product of such rows with a weight in 8-bit integers, scaled per row and per output column

Pools are [blocks, kv_heads, block_size, head_dim] in int8 or e4m3 and stand for code * scale[block, kv_head].
"""

from __future__ import annotations

import math
from typing import Dict, List, Optional

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
CACHE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn, "bf16": torch.bfloat16}
TOP = {"int8": 127.0, "e4m3": 448.0}
EPSILON = 1e-6
SMALLEST = 1.1754943508222875e-38  # the smallest normal number of 32 bits: no scale but zero is below it


# ------------------------------------------------------------------------------------------------------------- cases ----
def _attention(batch, context, heads, kv_heads, dim, *, cache="int8", dtype="bf16", block=128, ragged=False, mask=False):
    return dict(kind="attention", batch=batch, context=context, heads=heads, kv_heads=kv_heads, dim=dim, cache=cache,
                dtype=dtype, block=block, ragged=ragged, mask=mask)


def _store(batch, tokens, kv_heads, dim, *, first=0, cache="int8", dtype="bf16", block=128):
    return dict(kind="store", batch=batch, tokens=tokens, kv_heads=kv_heads, dim=dim, first=first, cache=cache, dtype=dtype,
                block=block)


def _copy(layers, moved, kv_heads, dim, *, cache="e4m3", block=128):
    return dict(kind="copy", layers=layers, moved=moved, kv_heads=kv_heads, dim=dim, cache=cache, block=block)


def _norm(rows, width, *, dtype="bf16", residual=True):
    return dict(kind="norm", rows=rows, width=width, dtype=dtype, residual=residual)


def _linear(rows, width, columns, *, form="none", bias=False, dtype="bf16"):
    return dict(kind="linear", rows=rows, width=width, columns=columns, form=form, bias=bias, dtype=dtype)


def listed() -> List[dict]:
    return [
        # one user's conversation: a single short context, a call that is all latency
        dict(_attention(1, 1000, 14, 2, 64), name="attention-single"),
        # a serving batch of equal contexts, heads of 64 in groups of seven
        dict(_attention(64, 4096, 14, 2, 64, cache="e4m3"), name="attention-batch"),
        # a server's sequences of very different ages, heads of 128: the largest read of the cache
        dict(_attention(64, 8192, 28, 4, 128, ragged=True, block=64), name="attention-ragged"),
        # a few long documents with padding masked out, fp16 queries, small blocks, an odd context
        dict(_attention(3, 30001, 16, 8, 128, cache="e4m3", dtype="fp16", block=32, mask=True), name="attention-long-masked"),
        # a decode step's append of one token for each sequence of a batch, into blocks that are partly full
        dict(_store(64, 1, 4, 128, first=77, cache="e4m3"), name="store-step"),
        # prompts of a batch into empty caches
        dict(_store(4, 4096, 4, 128), name="store-prompt"),
        # a sequence forked for a second answer: the last, partly filled block in each layer
        dict(_copy(24, 1, 2, 64), name="copy-fork"),
        # a pool of 16-bit keys and values compacted: hundreds of blocks to lower places
        dict(_copy(28, 150, 4, 128, cache="bf16"), name="copy-compact"),
        # one row between two projections of a decode step
        dict(_norm(1, 896), name="norm-single"),
        # the rows of long prompts
        dict(_norm(16384, 3584), name="norm-prompt"),
        # a decode batch through gate and up of a feed-forward layer: a stream of the weight
        dict(_linear(48, 3584, 37888, form="swiglu"), name="linear-step"),
        # prompts of a batch through the way down, onto the residual: the largest product
        dict(_linear(8191, 18944, 3584, form="residual"), name="linear-prompt"),
    ]


def _spread(rng, low: int, high: int) -> int:
    """A whole number whose logarithm is spread evenly."""

    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49))))))


def draw(rng) -> dict:
    kind = rng.choice(["attention", "attention", "store", "copy", "norm", "linear", "linear"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    kv_heads, dim, block = rng.choice([1, 2, 3, 4, 8]), rng.choice([64, 64, 128, 128, 256]), rng.choice([32, 64, 96, 128, 256])
    if kind == "attention":
        batch = _spread(rng, 1, 200)
        context = _spread(rng, 1, min(60000, 64 * 4096 * 4 * 128 // (batch * kv_heads * dim)))
        group = rng.choice([1, 2, 3, 4, 6, 7, 8, 12, 16, 20])
        return _attention(batch, context, group * kv_heads, kv_heads, dim, cache=rng.choice(["int8", "e4m3"]), dtype=dtype,
                          block=block, ragged=rng.random() < 0.6, mask=rng.random() < 0.25)
    if kind == "store":
        batch = _spread(rng, 1, 128)
        tokens = 1 if rng.random() < 0.4 else _spread(rng, 2, max(2, 4 * 4096 * 4 * 128 // (batch * kv_heads * dim)))
        tokens = min(tokens, 20000)
        return _store(batch, tokens, kv_heads, dim, first=rng.choice([0, rng.randrange(3 * block)]),
                      cache=rng.choice(["int8", "e4m3"]), dtype=dtype, block=block)
    if kind == "copy":
        layers = rng.randint(1, 32)
        cache = rng.choice(["e4m3", "e4m3", "bf16"])
        most = 28 * 150 * 4 * 128 * 128 * 2 // (layers * kv_heads * dim * block * CACHE[cache].itemsize)
        return _copy(layers, _spread(rng, 1, max(1, min(3000, most))), kv_heads, dim, cache=cache, block=block)
    if kind == "norm":
        width = _spread(rng, 64, 9000)
        if rng.random() < 0.7:
            width = -(-width // 16) * 16
        return _norm(_spread(rng, 1, min(16384, 16384 * 3584 // (2 * width))), width, dtype=rng.choice(["bf16", "fp16", "fp32"]),
                     residual=rng.random() < 0.6)
    width, columns = 16 * _spread(rng, 4, 1200), _spread(rng, 17, 38000)
    form = rng.choice(["none", "residual", "swiglu"])
    columns += columns % 2 if form == "swiglu" else 0
    rows = _spread(rng, 1, max(1, min(9000, 8191 * 18944 * 3584 // (width * columns))))
    return _linear(rows, width, columns, form=form, bias=rng.random() < 0.5,
                   dtype=rng.choice(["bf16", "fp16", "fp32"]) if form == "none" else dtype)


def _lengths(case: dict) -> List[int]:
    """Cached tokens of each sequence, the new one counted: all alike, or spread from one to the longest."""

    batch, context = case["batch"], case["context"]
    if not case["ragged"] or batch == 1:
        return [context] * batch
    return [1 + (context - 1) * ((b * 37 + 5) % batch) // max(1, batch - 1) for b in range(batch)]


# ------------------------------------------------------------------------------------------------------------ inputs ----
def _generator(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, *shape, dtype=torch.float32, scale=1.0) -> torch.Tensor:
    x = torch.empty(shape, dtype=dtype, device="cuda")
    x.normal_(0.0, scale, generator=g)
    return x


def _codes(g, cache: str, *shape) -> torch.Tensor:
    """Codes as a quantised cache or weight holds them: bell-shaped, up to the type's largest."""

    x = torch.empty(shape, dtype=torch.float16, device="cuda").normal_(0.0, 1.0, generator=g)
    if cache == "bf16":
        return x.to(torch.bfloat16)
    x.mul_(TOP[cache] / 3.4).clamp_(-TOP[cache], TOP[cache])
    return x.round_().to(torch.int8) if cache == "int8" else x.to(torch.float8_e4m3fn)


def _scales(g, cache: str, *shape) -> torch.Tensor:
    """Scales of blocks whose largest values lie between 2 and 5."""

    return torch.empty(shape, dtype=torch.float32, device="cuda").uniform_(2.0, 5.0, generator=g).div_(TOP[cache])


def _table(g, batch: int, columns: int) -> torch.Tensor:
    """Every sequence's blocks, scattered over the pool."""

    return torch.randperm(batch * columns, device="cuda", generator=g).to(torch.int32).view(batch, columns)


def prepare(case: dict, seed: int) -> dict:
    g = _generator(seed)
    s = dict(case)
    kind = case["kind"]
    if kind == "attention":
        batch, kv_heads, dim, block = case["batch"], case["kv_heads"], case["dim"], case["block"]
        columns = -(-case["context"] // block)
        blocks = batch * columns
        s["table"] = _table(g, batch, columns)
        for name in ("keys", "values"):
            s[name] = _codes(g, case["cache"], blocks, kv_heads, block, dim)
            s[name + "_scales"] = _scales(g, case["cache"], blocks, kv_heads)
        s["lengths"] = torch.tensor(_lengths(case), dtype=torch.int64).cuda()
        s["query"] = _normal(g, batch, 1, case["heads"], dim, dtype=TYPES[case["dtype"]]).transpose(1, 2)
        s["scale"] = dim ** -0.5
        s["additive"] = None
        if case["mask"]:  # padding in front of each prompt, as a server that pads on the left masks it out
            at = torch.arange(columns * block, device="cuda").view(1, 1, 1, -1)
            pad = (s["lengths"] // 7).view(batch, 1, 1, 1)
            s["additive"] = torch.zeros(batch, 1, 1, columns * block, device="cuda").masked_fill(at < pad, -math.inf)
        s["longest"] = case["context"]
    elif kind == "store":
        batch, tokens, kv_heads, dim, block = (case[k] for k in ("batch", "tokens", "kv_heads", "dim", "block"))
        columns = -(-(case["first"] + tokens) // block)
        s["table"] = _table(g, batch, columns)
        for name in ("keys", "values"):
            s[name] = _codes(g, case["cache"], batch * columns, kv_heads, block, dim)
            s[name + "_scales"] = _scales(g, case["cache"], batch * columns, kv_heads)
            # new rows as a packed projection lays them out: [batch, tokens, heads, dim]
            s["new_" + name] = _normal(g, batch, tokens, kv_heads, dim, dtype=TYPES[case["dtype"]]).transpose(1, 2)
        s["positions"] = torch.full((batch,), case["first"], dtype=torch.int64, device="cuda")
    elif kind == "copy":
        layers, moved, kv_heads, dim, block = (case[k] for k in ("layers", "moved", "kv_heads", "dim", "block"))
        blocks = 2 * moved + 3
        s["pools"] = [_codes(g, case["cache"], layers, blocks, kv_heads, block, dim) for _ in range(2)]
        if case["cache"] != "bf16":
            s["pools"] += [_scales(g, case["cache"], layers, blocks, kv_heads) for _ in range(2)]
        order = torch.randperm(blocks, device="cuda", generator=g).to(torch.int32)
        s["sources"], s["destinations"] = order[:moved].clone(), order[moved:2 * moved].clone()
    elif kind == "norm":
        dtype = TYPES[case["dtype"]]
        s["x"] = _normal(g, case["rows"], case["width"], dtype=dtype)
        s["residual_rows"] = _normal(g, case["rows"], case["width"], dtype=dtype, scale=2.0) if case["residual"] else None
        s["weight"] = (1.0 + 0.2 * _normal(g, case["width"])).to(dtype)
    else:
        rows, width, columns, dtype = case["rows"], case["width"], case["columns"], TYPES[case["dtype"]]
        s["x"] = _codes(g, "int8", rows, width)
        s["x_scales"] = _scales(g, "int8", rows)
        s["weight"] = _codes(g, "int8", columns, width)
        s["weight_scales"] = _scales(g, "int8", columns).div_(math.sqrt(width))
        s["bias_row"] = _normal(g, columns, dtype=dtype) if case["bias"] else None
        s["residual_rows"] = _normal(g, rows, columns, dtype=dtype, scale=2.0) if case["form"] == "residual" else None
    return s


# --------------------------------------------------------------------------------------------- the framework's calls ----
def _run_own(s: dict):
    import llm_compiler_b200 as b200

    kind = s["kind"]
    if kind == "attention":
        return b200.b200_paged_decode_attention_8bit(
            s["query"], s["keys"], s["values"], s["keys_scales"], s["values_scales"], s["table"], s["lengths"], s["additive"],
            scale=s["scale"], max_length_hint=s["longest"])
    if kind == "store":
        b200.b200_paged_kv_store_8bit(s["keys"], s["values"], s["keys_scales"], s["values_scales"], s["table"], s["new_keys"],
                                      s["new_values"], s["positions"])
        return _held(s)
    if kind == "copy":
        b200.b200_copy_kv_blocks(s["pools"], s["sources"], s["destinations"])
        return tuple(s["pools"])
    if kind == "norm":
        values, scales, total = b200.b200_rms_norm_int8(s["x"], s["weight"], epsilon=EPSILON, residual=s["residual_rows"])
        out = torch.empty(values.shape, dtype=torch.bfloat16, device="cuda")
        torch.mul(values, scales.unsqueeze(1), out=out)
        return (out, scales, total) if s["residual"] else (out, scales)
    return b200.b200_linear_int8(s["x"], s["x_scales"], s["weight"], s["weight_scales"], s["bias_row"], epilogue=s["form"],
                                 residual=s["residual_rows"], out_dtype=TYPES[s["dtype"]])


# ------------------------------------------------------------------------------------------------------- plain forms ----
def _held(s: dict):
    """What a cache holds: e4m3 codes and their scales, or the values that 8-bit integers stand for and their scales."""

    if s["cache"] == "e4m3":
        return s["keys"], s["values"], s["keys_scales"], s["values_scales"]
    return (s["keys"] * s["keys_scales"][:, :, None, None], s["values"] * s["values_scales"][:, :, None, None],
            s["keys_scales"], s["values_scales"])


def _attention_plain(s: dict) -> torch.Tensor:
    batch, heads, kv_heads, dim, block = (s[k] for k in ("batch", "heads", "kv_heads", "dim", "block"))
    table = s["table"].long()
    columns = table.shape[1]

    def rows(name):  # [batch, kv_heads, tokens, dim] in 32 bits
        x = s[name][table].float() * s[name + "_scales"][table][..., None, None]
        return x.transpose(1, 2).reshape(batch, kv_heads, columns * block, dim)

    valid = torch.arange(columns * block, device="cuda").view(1, 1, 1, -1) < s["lengths"].view(batch, 1, 1, 1)
    keys, values = rows("keys"), rows("values")
    query = s["query"].float().reshape(batch, kv_heads, heads // kv_heads, dim)
    scores = torch.matmul(query, keys.transpose(2, 3)) * s["scale"]
    if s["additive"] is not None:
        scores = scores + s["additive"]
    scores = torch.where(valid, scores, -math.inf)
    values = torch.where(valid.transpose(2, 3), values, 0.0)
    weights = torch.exp(scores - scores.amax(-1, keepdim=True))
    out = torch.matmul(weights, values) / weights.sum(-1, keepdim=True)
    return out.reshape(batch, heads, 1, dim).to(s["query"].dtype)


def _store_plain(s: dict):
    """Every sequence's touched blocks at once: rows in front of `first` stay, and are rounded anew where the scale grows."""

    batch, tokens, kv_heads, dim, block, first, cache = (
        s[k] for k in ("batch", "tokens", "kv_heads", "dim", "block", "first", "cache"))
    top, low = TOP[cache], first // block
    columns = -(-(first + tokens) // block)
    where = s["table"][:, low:columns].long()  # [batch, touched]
    touched = columns - low
    span = touched * block
    at = torch.arange(span, device="cuda").view(1, 1, touched, block, 1) + low * block
    old, fresh = at < first, (at >= first) & (at < first + tokens)
    grown = torch.arange(touched, device="cuda").view(1, touched, 1) * block + low * block < first  # blocks that hold rows already

    def code(x):
        return torch.clamp(torch.round(x), -top, top).to(torch.int8) if cache == "int8" else \
            torch.clamp(x, -top, top).to(torch.float8_e4m3fn)

    for name in ("keys", "values"):  # keys, then values
        pool, scales = s[name], s[name + "_scales"]
        new = torch.zeros(batch, kv_heads, span, dim, device="cuda")
        new[:, :, first - low * block:first - low * block + tokens] = s["new_" + name]
        new = new.view(batch, kv_heads, touched, block, dim)
        most = torch.where(fresh, new.abs(), 0.0).amax((3, 4)).transpose(1, 2)  # [batch, touched, kv_heads]
        scale = most * torch.full((), 1.0 / top, device="cuda")
        scale = torch.where(most > 0, scale.clamp_min(SMALLEST), 0.0)
        before = torch.where(grown, scales[where], 0.0)
        scale = torch.maximum(scale, before)
        inverse = torch.where(scale > 0, scale.reciprocal(), 0.0)
        ratio = torch.where(scale > 0, before / scale, 0.0)
        held = pool[where]  # [batch, touched, kv_heads, block, dim]
        kept = code(held.float() * ratio[..., None, None])
        written = code(new.transpose(1, 2) * inverse[..., None, None])
        old_t, fresh_t = old.transpose(1, 2), fresh.transpose(1, 2)
        if cache == "int8":
            pool[where] = torch.where(fresh_t, written, torch.where(old_t, kept, held))
        else:  # (selection of bytes)
            pool.view(torch.uint8)[where] = torch.where(
                fresh_t, written.view(torch.uint8), torch.where(old_t, kept.view(torch.uint8), held.view(torch.uint8)))
        scales[where] = scale
    return _held(s)


def _norm_plain(s: dict):
    x = s["x"].float()
    total = s["x"]
    if s["residual"]:
        total = (x + s["residual_rows"].float()).to(s["x"].dtype)
        x = total.float()
    y = x * torch.rsqrt(x.square().mean(1, keepdim=True) + EPSILON) * s["weight"].float()
    scales = y.abs().amax(1) / torch.full((), 127.0, device="cuda")
    codes = torch.where(scales[:, None] > 0, torch.round(y / scales[:, None]), 0.0)
    out = (codes * scales[:, None]).to(torch.bfloat16)
    return (out, scales, total) if s["residual"] else (out, scales)


def _linear_plain(s: dict) -> torch.Tensor:
    y = torch.matmul(s["x"].float(), s["weight"].float().t())
    y = y * s["x_scales"][:, None] * s["weight_scales"][None, :]
    if s["bias"]:
        y = y + s["bias_row"].float()
    if s["form"] == "swiglu":  # columns 2 j and 2 j + 1 are gate j and up j
        gate, up = y[:, 0::2], y[:, 1::2]
        y = gate / (1.0 + torch.exp(-gate)) * up
    elif s["form"] == "residual":
        y = y + s["residual_rows"].float()
    return y.to(TYPES[s["dtype"]])


def run(s: dict):
    if own:
        return _run_own(s)
    kind = s["kind"]
    if kind == "attention":
        return _attention_plain(s)
    if kind == "store":
        return _store_plain(s)
    if kind == "copy":
        for pool in s["pools"]:
            bits = pool.view(torch.uint8) if pool.dtype == torch.float8_e4m3fn else pool
            bits[:, s["destinations"].long()] = bits[:, s["sources"].long()]
        return tuple(s["pools"])
    if kind == "norm":
        return _norm_plain(s)
    return _linear_plain(s)


# -------------------------------------------------------------------------------------------------------------- work ----
def work(case: dict) -> Dict[str, float]:
    """Inputs read once, outputs written once. A store reads and writes again what its blocks hold only where a scale grows;
    that is not counted."""

    kind = case["kind"]
    if kind == "attention":
        tokens = sum(_lengths(case))
        blocks = sum(-(-n // case["block"]) for n in _lengths(case))
        rows = case["batch"] * case["heads"] * case["dim"]
        size = 2 * tokens * case["kv_heads"] * case["dim"] + 8 * blocks * case["kv_heads"] + 4 * blocks + 8 * case["batch"]
        size += 2 * rows * TYPES[case["dtype"]].itemsize + (4 * tokens if case["mask"] else 0)
        return {"bytes": size, "flops": 4 * tokens * case["heads"] * case["dim"]}
    if kind == "store":
        new = 2 * case["batch"] * case["tokens"] * case["kv_heads"] * case["dim"]
        columns = -(-(case["first"] + case["tokens"]) // case["block"])
        size = new * (TYPES[case["dtype"]].itemsize + 1) + 16 * case["batch"] * columns * case["kv_heads"]
        if case["cache"] == "int8":  # the values that it stands for are an output
            size += 2 * case["batch"] * columns * case["kv_heads"] * case["block"] * case["dim"] * 4
        return {"bytes": size, "flops": 2 * new}
    if kind == "copy":
        one = case["kv_heads"] * case["block"] * case["dim"] * CACHE[case["cache"]].itemsize * 2
        one += 0 if case["cache"] == "bf16" else 8 * case["kv_heads"]
        size = 2 * case["layers"] * case["moved"] * one
        return {"bytes": size, "flops": 0}
    if kind == "norm":
        held = case["rows"] * case["width"]
        size = TYPES[case["dtype"]].itemsize * (held * (3 if case["residual"] else 1) + case["width"]) + 2 * held + 4 * case["rows"]
        return {"bytes": size, "flops": 6 * held}
    rows, width, columns = case["rows"], case["width"], case["columns"]
    outputs = rows * columns // (2 if case["form"] == "swiglu" else 1) * (2 if case["form"] == "residual" else 1)
    size = (rows + columns) * (width + 4) + outputs * TYPES[case["dtype"]].itemsize
    size += columns * TYPES[case["dtype"]].itemsize if case["bias"] else 0
    return {"bytes": size, "flops": 2 * rows * width * columns}


# ------------------------------------------------------------------------------------------------------------- exact ----
def _e4m3(x: torch.Tensor) -> torch.Tensor:
    """The nearest e4m3 number (four exponent bits of bias 7, three of mantissa, 448 the largest), in 64 bits."""

    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)
    return (torch.round(x / step) * step).clamp(-448.0, 448.0)


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "copy":
        return None  # (nothing is computed)
    if kind == "attention":
        batch, heads, kv_heads, dim, block = (case[k] for k in ("batch", "heads", "kv_heads", "dim", "block"))
        group = heads // kv_heads
        out = torch.empty(batch, heads, 1, dim, dtype=torch.float64, device="cuda")
        for b, length in enumerate(_lengths(case)):
            blocks = s["table"][b, :-(-length // block)].long()
            for h in range(kv_heads):
                k, v = (torch.cat(list(s[n][blocks, h].double() * s[n + "_scales"][blocks, h].double()[:, None, None]))[:length]
                        for n in ("keys", "values"))
                q = s["query"][b, h * group:(h + 1) * group, 0].double()
                logits = q @ k.T * s["scale"]
                if s["additive"] is not None:
                    logits += s["additive"][b, 0, :, :length].double()
                out[b, h * group:(h + 1) * group, 0] = torch.softmax(logits, 1) @ v
        return out
    if kind == "store":
        block, first, tokens, int8 = case["block"], case["first"], case["tokens"], case["cache"] == "int8"
        top = torch.tensor(1.0 / TOP[case["cache"]], dtype=torch.float32).double().item()
        pools = []
        for name in ("keys", "values"):
            pool, scales = s[name].double(), s[name + "_scales"].double()
            for column in range(first // block, -(-(first + tokens) // block)):
                at = s["table"][:, column].long()
                lo, hi = max(first, column * block), min(first + tokens, (column + 1) * block)
                new = s["new_" + name][:, :, lo - first:hi - first].double()
                need = (new.abs().amax((2, 3)) * top).float().double().clamp_min(SMALLEST)
                scale = need
                if lo > column * block:
                    before = scales[at]
                    scale = torch.maximum(need, before)
                    ratio = (before / scale).float().double()[..., None, None]
                    held = (pool[at][:, :, :lo - column * block] * ratio).float().double()
                    pool[at, :, :lo - column * block] = torch.round(held) if int8 else _e4m3(held)
                inverse = (1.0 / scale).float().double()[..., None, None]
                codes = (new * inverse).float().double()
                pool[at, :, lo - column * block:hi - column * block] = torch.round(codes).clamp(-127, 127) if int8 else _e4m3(codes)
                scales[at] = scale
            pools.append((pool * scales[..., None, None] if int8 else pool, scales))
        return pools[0][0], pools[1][0], pools[0][1], pools[1][1]
    if kind == "norm":
        x = s["x"].double()
        if case["residual"]:
            total = (x + s["residual_rows"].double()).to(s["x"].dtype)
            x = total.double()
        y = x / torch.sqrt((x * x).mean(1, keepdim=True) + EPSILON) * s["weight"].double()
        scales = y.abs().amax(1) / 127.0
        out = torch.round(y / scales[:, None]) * scales[:, None]
        return (out, scales, total.double()) if case["residual"] else (out, scales)
    y = s["x"].double() @ s["weight"].double().T
    y *= s["x_scales"].double()[:, None] * s["weight_scales"].double()[None]
    if case["bias"]:
        y += s["bias_row"].double()
    if case["form"] == "swiglu":
        y = torch.nn.functional.silu(y[:, 0::2]) * y[:, 1::2]
    elif case["form"] == "residual":
        y += s["residual_rows"].double()
    return y
