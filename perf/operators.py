"""Measured cases of the serving operators around an 8-bit paged K/V cache.

Four operators make one decode or prefill step: ``paged_slots`` says where the new tokens of
each request go, ``rotary_embedding`` turns their queries and keys by their positions,
``paged_cache_append_8bit`` stores keys and values in 8 bits, and
``paged_attention_decode_8bit`` reads them back.  ``run`` computes each in elementary torch
operations (``own`` false) or through ``radeon_kernels`` (``own`` true); ``exact`` is the
definition in 64 bits.
"""

from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
_INDEX = {"int32": torch.int32, "int64": torch.int64}
_LARGEST = {"e4m3": 448.0, "int8": 127.0}
_rk = None


def _package():
    global _rk
    if _rk is None:
        root = str(Path(__file__).resolve().parents[1] / "radeon-kernels_b200")
        if root not in sys.path:
            sys.path.insert(0, root)
        import radeon_kernels

        _rk = radeon_kernels
    return _rk


# ------------------------------------------------------------------------------ cases
def listed():
    return [
        # One decode step of a small batch: queries and keys of 16 tokens are rotated.
        dict(name="rotary decode", op="rotary", tokens=16, query_heads=32, kv_heads=8, head_dim=128, rotary_dim=128,
             dtype="bf16", interleaved=False, scaling="none", train=False, index="int32"),
        # A prompt chunk of a model whose positions were stretched to 128 Ki.
        dict(name="rotary prefill", op="rotary", tokens=8192, query_heads=32, kv_heads=8, head_dim=128, rotary_dim=128,
             dtype="bf16", interleaved=False, scaling="yarn", train=False, index="int64"),
        # A training step: adjacent pairs, half of each head, an odd number of tokens, with gradients.
        dict(name="rotary train", op="rotary", tokens=4099, query_heads=16, kv_heads=16, head_dim=128, rotary_dim=64,
             dtype="fp16", interleaved=True, scaling="linear", train=True, index="int64"),
        # Decode: 256 requests with one new token each.
        dict(name="slots decode", op="slots", requests=256, longest=8000, new_longest=1, padding=0, block_size=16,
             max_blocks=512, index="int32", shape=11),
        # Chunked prefill of 61 prompts of mixed lengths, the token buffer padded at its end.
        dict(name="slots prefill", op="slots", requests=61, longest=4096, new_longest=2048, padding=777, block_size=32,
             max_blocks=256, index="int64", shape=12),
        # Decode: one token of each of 128 requests joins its last block.
        dict(name="append decode", op="append", requests=128, longest=2048, new_longest=1, kv_heads=8, head_dim=128,
             block_size=16, dtype="bf16", cache="e4m3", shape=13),
        # Prompts of 37 requests, 8-bit integers, small heads.
        dict(name="append prefill int8", op="append", requests=37, longest=300, new_longest=700, kv_heads=4, head_dim=64,
             block_size=32, dtype="fp16", cache="int8", shape=14),
        # A long-prompt batch.
        dict(name="append prefill e4m3", op="append", requests=21, longest=1000, new_longest=4000, kv_heads=8,
             head_dim=128, block_size=16, dtype="bf16", cache="e4m3", shape=15),
        # One user, a context of about a thousand tokens: latency.
        dict(name="attention one request", op="attention", requests=1, shortest=1003, longest=1003, query_heads=32,
             kv_heads=8, head_dim=128, block_size=16, dtype="bf16", cache="e4m3", index="int32", shape=16),
        # Sixteen users at 2048 tokens.
        dict(name="attention batch", op="attention", requests=16, shortest=2048, longest=2048, query_heads=32, kv_heads=8,
             head_dim=128, block_size=16, dtype="bf16", cache="e4m3", index="int32", shape=17),
        # A busy server: lengths from one token to 16 Ki.
        dict(name="attention ragged int8", op="attention", requests=61, shortest=1, longest=16384, query_heads=32,
             kv_heads=4, head_dim=128, block_size=32, dtype="fp16", cache="int8", index="int64", shape=18),
        # Four documents of 128 Ki tokens.
        dict(name="attention long", op="attention", requests=4, shortest=131072, longest=131072, query_heads=32, kv_heads=8,
             head_dim=128, block_size=64, dtype="bf16", cache="e4m3", index="int32", shape=19),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["rotary", "slots", "append", "attention", "attention"])
    shape = rng.randrange(1 << 20)
    dtype, index, cache = rng.choice(["fp16", "bf16"]), rng.choice(["int32", "int64"]), rng.choice(["e4m3", "int8"])
    if op == "rotary":
        head_dim = rng.choice([64, 80, 96, 128, 192, 256])
        return dict(op=op, tokens=_spread(rng, 1, 6000), query_heads=rng.choice([4, 8, 20, 28, 32]),
                    kv_heads=rng.choice([1, 2, 4, 8]), head_dim=head_dim,
                    rotary_dim=rng.choice([head_dim, head_dim // 2, head_dim // 4]), dtype=dtype,
                    interleaved=rng.random() < 0.5, scaling=rng.choice(["none", "linear", "ntk", "yarn"]),
                    train=rng.random() < 0.4, index=index)
    if op == "slots":
        new = rng.choice([1, 1, 5, 300, 2000])
        longest, block_size = _spread(rng, 1, 8000), rng.choice([8, 16, 32, 48, 64])
        return dict(op=op, requests=_spread(rng, 1, 400 if new > 5 else 1000), longest=longest, new_longest=new,
                    padding=rng.choice([0, 0, 1, 100]), block_size=block_size,
                    max_blocks=-(-(longest + new) // block_size) + rng.choice([0, 1, 100]), index=index, shape=shape)
    block_size = rng.choice([8, 16, 24, 32, 64, 128])
    kv_heads, head_dim = rng.choice([1, 2, 3, 4, 8]), rng.choice([64, 128, 256])
    if op == "append":
        new = rng.choice([1, 1, 9, 200, 1500])
        return dict(op=op, requests=_spread(rng, 1, 400 if new < 200 else 24), longest=_spread(rng, 1, 1000),
                    new_longest=new, kv_heads=kv_heads, head_dim=head_dim, block_size=block_size, dtype=dtype,
                    cache=cache, shape=shape)
    requests = _spread(rng, 1, 128)
    longest = _spread(rng, 1, 1_000_000 // (requests * kv_heads) * 128 // head_dim + 1)
    return dict(op=op, requests=requests, shortest=rng.choice([1, longest]), longest=longest,
                query_heads=kv_heads * rng.choice([1, 2, 4, 5, 7, 8, 16]), kv_heads=kv_heads, head_dim=head_dim,
                block_size=block_size, dtype=dtype, cache=cache, index=index, shape=shape)


# ------------------------------------------------------------------------------ sizes
def _lengths(case):
    """(tokens that each request has, tokens that it gets), the same for every seed."""
    rng = random.Random(case["shape"])
    n = case["requests"]
    if case["op"] == "attention":
        low, high = case["shortest"], case["longest"]
        return [_spread(rng, low, high) for _ in range(n)], [0] * n
    has = [rng.randint(0, case["longest"]) for _ in range(n)]
    most = case["new_longest"]
    new = [1 if most == 1 else rng.randint(0, most) for _ in range(n)]
    return has, new if sum(new) else [1] * n


def _blocks(length, block_size):
    return -(-length // block_size)


def work(case):
    if case["op"] == "rotary":
        heads = case["query_heads"] + case["kv_heads"]
        values = case["tokens"] * heads * case["head_dim"]
        pairs = case["tokens"] * heads * (case["rotary_dim"] // 2)
        passes = 2 if case["train"] else 1
        index = 4 if case["index"] == "int32" else 8
        return {"bytes": passes * (4 * values + index * case["tokens"]), "flops": passes * 6 * pairs}
    has, new = _lengths(case)
    if case["op"] == "slots":
        index = 4 if case["index"] == "int32" else 8
        b = case["block_size"]
        added = sum(_blocks(h + n, b) - _blocks(h, b) for h, n in zip(has, new))
        joined = sum(1 for h, n in zip(has, new) if n and h % b)
        tokens = sum(new) + case["padding"]
        return {"bytes": index * (3 * len(has) + 2 * added + joined + 1) + (8 + index) * tokens, "flops": 2 * tokens}
    row = case["kv_heads"] * case["head_dim"]
    b = case["block_size"]
    if case["op"] == "append":
        tokens = sum(new)
        touched = sum(_blocks(h + n, b) - h // b for h, n in zip(has, new) if n)
        return {"bytes": tokens * (2 * row * 3 + 8) + touched * case["kv_heads"] * 16, "flops": 6 * tokens * row}
    blocks = sum(_blocks(h, b) for h in has)
    index = 4 if case["index"] == "int32" else 8
    wide = case["query_heads"] * case["head_dim"]
    return {"bytes": 2 * row * sum(has) + blocks * (8 * case["kv_heads"] + index) + len(has) * (4 * wide + index),
            "flops": 4 * wide * sum(has)}


# ----------------------------------------------------------------------------- inputs
def _frequencies(case):
    """Radians per position of each pair, in 64 bits: what a program computes once."""
    dim, base, factor, original = case["rotary_dim"], 10000.0, 8.0, 16384
    if case["scaling"] == "ntk":
        base *= factor ** (dim / (dim - 2))
    freq = [base ** (-2.0 * i / dim) for i in range(dim // 2)]
    if case["scaling"] == "linear":
        freq = [f / factor for f in freq]
    if case["scaling"] == "yarn":
        at = [dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base)) for turns in (32.0, 1.0)]
        low, high = max(math.floor(at[0]), 0), min(math.ceil(at[1]), dim - 1)
        share = [min(max((i - low) / max(high - low, 1e-3), 0.0), 1.0) for i in range(dim // 2)]
        freq = [f / factor * s + f * (1 - s) for f, s in zip(freq, share)]
    return freq


def _amplitude(case):
    return 0.1 * math.log(8.0) + 1.0 if case["scaling"] == "yarn" else 1.0


def _values(gen, rows, heads, dim, dtype):
    """Activations: normal, with a few channels of each head several times as large."""
    wide = torch.exp(0.7 * torch.randn((1, heads, dim), generator=gen, device="cuda"))
    return (torch.randn((rows, heads, dim), generator=gen, device="cuda") * wide).to(dtype)


def _tables(case, gen, held, max_blocks, index):
    """Block tables that hold `held` tokens of each request in blocks of a shuffled pool; the rest -1."""
    b = case["block_size"]
    counts = torch.tensor([_blocks(h, b) for h in held], device="cuda")
    total = int(counts.sum())
    pool = total + total // 8 + 3
    order = torch.randperm(pool, generator=gen, device="cuda")
    col = torch.arange(max_blocks, device="cuda")
    first = (torch.cumsum(counts, 0) - counts)[:, None]
    table = torch.where(col < counts[:, None], order[(first + col).clamp(max=pool - 1)], -1)
    return table.to(index), pool, order[total:].to(index)


def _stored(case, gen, pool):
    """A filled cache in 8 bits: values normal within a block and head, with one scale each."""
    shape = (pool, case["block_size"], case["kv_heads"], case["head_dim"])
    largest = _LARGEST[case["cache"]]
    x = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float16)
    x *= largest / 5.0
    x.clamp_(-largest, largest)
    return x.round_().to(torch.int8) if case["cache"] == "int8" else x.to(torch.float8_e4m3fn)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": case}
    if case["op"] == "rotary":
        dtype, tokens = _DTYPES[case["dtype"]], case["tokens"]
        wide = case["query_heads"] + 2 * case["kv_heads"]
        # Queries, keys and values leave one projection side by side; the operator reads the
        # first two where they are.
        joint = _values(gen, tokens, wide, case["head_dim"], dtype)
        state["query"] = joint[:, : case["query_heads"]]
        state["key"] = joint[:, case["query_heads"] : case["query_heads"] + case["kv_heads"]]
        start = torch.randint(0, 131072 - tokens, (), generator=gen, device="cuda")
        state["positions"] = (start + torch.arange(tokens, device="cuda")).to(_INDEX[case["index"]])
        state["frequencies"] = torch.tensor(_frequencies(case), dtype=torch.float64, device="cuda")
        state["amplitude"] = _amplitude(case)
        if case["train"]:
            state["query"].requires_grad_(True)
            state["key"].requires_grad_(True)
            state["grads"] = (_values(gen, tokens, case["query_heads"], case["head_dim"], dtype),
                              _values(gen, tokens, case["kv_heads"], case["head_dim"], dtype))
        return state
    has, new = _lengths(case)
    b = case["block_size"]
    if case["op"] == "slots":
        index = _INDEX[case["index"]]
        ends = [h + n for h, n in zip(has, new)]
        state["block_tables"], _, _ = _tables(case, gen, has, case["max_blocks"], index)
        wanted = sum(_blocks(e, b) - _blocks(h, b) for e, h in zip(ends, has))
        state["free_blocks"] = torch.randperm(wanted + 64, generator=gen, device="cuda").to(index)
        state["context_lengths"] = torch.tensor(has, dtype=index, device="cuda")
        state["new_lengths"] = torch.tensor(new, dtype=index, device="cuda")
        state["tokens"] = sum(new) + case["padding"]
        return state
    if case["op"] == "append":
        dtype, tokens = _DTYPES[case["dtype"]], sum(new)
        ends = [h + n for h, n in zip(has, new)]
        table, pool, _ = _tables(case, gen, ends, max(1, max(_blocks(e, b) for e in ends)), torch.int64)
        counts = torch.tensor(new, device="cuda")
        request = torch.repeat_interleave(torch.arange(len(new), device="cuda"), counts)
        at = torch.arange(tokens, device="cuda") - (torch.cumsum(counts, 0) - counts)[request]
        position = torch.tensor(has, device="cuda")[request] + at
        state["slot_mapping"] = table[request, position // b] * b + position % b
        heads = case["kv_heads"]
        state["key"] = _values(gen, tokens, heads, case["head_dim"], dtype)
        state["value"] = _values(gen, tokens, heads, case["head_dim"], dtype)
        state["key_cache"], state["value_cache"] = _stored(case, gen, pool), _stored(case, gen, pool)
        # Scales of earlier appends: powers of two around what such values need.
        exponent = 8 if case["cache"] == "e4m3" else 6
        for name in ("key_scales", "value_scales"):
            power = torch.randint(0, 4, (pool, heads), generator=gen, device="cuda") - exponent
            state[name] = torch.exp2(power.float())
        return state
    dtype, index = _DTYPES[case["dtype"]], _INDEX[case["index"]]
    max_blocks = max(_blocks(h, b) for h in has) + 1
    state["block_tables"], pool, _ = _tables(case, gen, has, max_blocks, index)
    state["context_lengths"] = torch.tensor(has, dtype=index, device="cuda")
    state["query"] = _values(gen, len(has), case["query_heads"], case["head_dim"], dtype)
    state["key_cache"], state["value_cache"] = _stored(case, gen, pool), _stored(case, gen, pool)
    largest = _LARGEST[case["cache"]]
    for name in ("key_scales", "value_scales"):
        spread = 0.3 * torch.randn((pool, case["kv_heads"]), generator=gen, device="cuda")
        state[name] = torch.exp(spread) * (5.0 / largest)
    return state


# ------------------------------------------------------------------------------- runs
def run(state):
    return {"rotary": _run_rotary, "slots": _run_slots, "append": _run_append, "attention": _run_attention}[
        state["case"]["op"]](state)


def _rotate(x, cos, sin, interleaved):
    """The rotated head, in 32 bits, rounded once: pairs are neighbours or a half apart."""
    half = cos.shape[-1]
    f = x.float()
    a, b = (f[..., 0 : 2 * half : 2], f[..., 1 : 2 * half : 2]) if interleaved else (f[..., :half], f[..., half : 2 * half])
    c, d = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([c, d], dim=-1).flatten(-2) if interleaved else torch.cat([c, d], dim=-1)
    return torch.cat([turned, f[..., 2 * half :]], dim=-1).to(x.dtype)


def _run_rotary(s):
    case = s["case"]
    if own:
        out = _package().rotary_embedding(s["query"], s["key"], s["positions"], s["frequencies"],
                                          interleaved=case["interleaved"], amplitude=s["amplitude"])
        if not case["train"]:
            return out
        return (*out, *torch.autograd.grad(out, (s["query"], s["key"]), s["grads"]))
    angle = s["positions"].double()[:, None] * s["frequencies"]
    cos = (torch.cos(angle) * s["amplitude"]).float()[:, None]
    sin = (torch.sin(angle) * s["amplitude"]).float()[:, None]
    out = [_rotate(x.detach(), cos, sin, case["interleaved"]) for x in (s["query"], s["key"])]
    if case["train"]:
        # The gradient of a rotation is the rotation back.
        out += [_rotate(g, cos, -sin, case["interleaved"]) for g in s["grads"]]
    return tuple(out)


def _run_slots(s):
    case = s["case"]
    b, tokens, tables = case["block_size"], s["tokens"], s["block_tables"]
    if own:
        slots, positions, lengths, used = _package().paged_slots(
            tables, s["context_lengths"], s["new_lengths"], s["free_blocks"], num_tokens=tokens, block_size=b)
        return slots, positions, lengths, used, tables
    has, new = s["context_lengths"].long(), s["new_lengths"].long()
    ends = has + new
    old, want = (has + b - 1) // b, (ends + b - 1) // b
    after = torch.cumsum(want - old, 0)
    col = torch.arange(tables.shape[1], device=tables.device)
    fresh = (col >= old[:, None]) & (col < want[:, None])
    at = (after - (want - old))[:, None] + col - old[:, None]
    block = s["free_blocks"][at.clamp(0, s["free_blocks"].shape[0] - 1)]
    tables.copy_(torch.where(fresh, block, tables))
    last = torch.cumsum(new, 0)
    token = torch.arange(tokens, device=tables.device)
    marks = torch.zeros(tokens + 1, dtype=torch.int64, device=tables.device)
    marks.index_add_(0, last, torch.ones_like(last))
    request = torch.cumsum(marks, 0)[:tokens].clamp(max=has.shape[0] - 1)
    live = token < last[-1]
    position = torch.where(live, has[request] + token - (last - new)[request], 0)
    slot = tables[request, (position // b).clamp(max=tables.shape[1] - 1)].long() * b + position % b
    return torch.where(live, slot, -1), position.to(tables.dtype), ends.to(tables.dtype), after[-1:].to(tables.dtype), tables


def _store(rows, cache, scales, slots, block_size, kind):
    """One cache's append: the scale of a block and head is the least power of two that its
    values fit, and never falls while the block lives; a scale that grows re-rounds the rows
    that stay."""
    largest = _LARGEST[kind]
    touched, member = torch.unique(slots // block_size, return_inverse=True)
    offset = slots % block_size
    x = rows.float()
    was = scales[touched]
    most = torch.zeros_like(was).index_reduce_(0, member, x.abs().amax(-1), "amax")
    mantissa, exponent = torch.frexp(most / largest)
    exponent = torch.where(most > 0, exponent - (mantissa == 0.5).int(), -126)
    need = torch.exp2(exponent.clamp(min=-126).float())
    new = torch.zeros(touched.shape, dtype=torch.bool, device=x.device)
    new[member[offset == 0]] = True
    last = torch.zeros_like(touched).index_reduce_(0, member, offset, "amax")
    now = torch.maximum(torch.where(new[:, None], 0.0, was), need)
    keep = (torch.arange(block_size, device=x.device) < last[:, None]) & ~new[:, None]
    grown = keep[:, :, None, None] & (now > was)[:, None, :, None]
    bits = cache.view(torch.uint8)
    held = bits[touched]
    moved = held.view(cache.dtype).float() * was[:, None, :, None] * (1.0 / now)[:, None, :, None]
    held = torch.where(grown, _to8(moved, kind).view(torch.uint8), held)
    held[member, offset] = _to8(x * (1.0 / now)[member][:, :, None], kind).view(torch.uint8)
    bits[touched] = held
    scales[touched] = now


def _to8(x, kind):
    """Rounded to the nearest 8-bit value, ties to even."""
    largest = _LARGEST[kind]
    x = x.clamp(-largest, largest)
    return torch.round(x).to(torch.int8) if kind == "int8" else x.to(torch.float8_e4m3fn)


def _run_append(s):
    case = s["case"]
    if own:
        _package().paged_cache_append_8bit(s["key"], s["value"], s["key_cache"], s["value_cache"], s["key_scales"],
                                           s["value_scales"], s["slot_mapping"])
    else:
        _store(s["key"], s["key_cache"], s["key_scales"], s["slot_mapping"], case["block_size"], case["cache"])
        _store(s["value"], s["value_cache"], s["value_scales"], s["slot_mapping"], case["block_size"], case["cache"])
    return s["key_cache"], s["value_cache"], s["key_scales"], s["value_scales"]


def _run_attention(s):
    case = s["case"]
    if own:
        return _package().paged_attention_decode_8bit(s["query"], s["key_cache"], s["value_cache"], s["key_scales"],
                                                      s["value_scales"], s["block_tables"], s["context_lengths"])
    n, heads, dim, b = case["requests"], case["kv_heads"], case["head_dim"], case["block_size"]
    table = s["block_tables"].long().clamp(min=0)
    span = table.shape[1] * b
    live = torch.arange(span, device=table.device) < s["context_lengths"].long()[:, None]

    def read(cache, scales):
        x = cache.view(torch.uint8)[table].view(cache.dtype)
        return (x.float() * scales[table][:, :, None, :, None]).view(n, span, heads, dim).permute(0, 2, 1, 3)

    query = s["query"].float().view(n, heads, -1, dim) / math.sqrt(dim)
    score = torch.matmul(query, read(s["key_cache"], s["key_scales"]).transpose(2, 3))
    score = torch.where(live[:, None, None], score, float("-inf"))
    weight = torch.exp(score - score.amax(-1, keepdim=True))
    weight = weight / weight.sum(-1, keepdim=True)
    out = torch.matmul(weight, read(s["value_cache"], s["value_scales"]))
    return out.view(n, case["query_heads"], dim).to(s["query"].dtype)


# ------------------------------------------------------------------- the definition
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        return _exact_rotary(s)
    if case["op"] == "append":
        return tuple(
            x for pair in zip(*(_exact_append(s, which) for which in ("key", "value"))) for x in pair)
    if case["op"] == "attention":
        return _exact_attention(s)
    return None


def _exact_rotary(s):
    """Each pair as a complex number times amplitude * e^(i * position * frequency)."""
    case = s["case"]
    turn = torch.polar(torch.full((), s["amplitude"], dtype=torch.float64, device="cuda"),
                       s["positions"].double()[:, None] * s["frequencies"])[:, None]

    def turned(x, by):
        out, half = x.detach().double().clone(), case["rotary_dim"] // 2
        i = torch.arange(half, device="cuda")
        first, second = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + half)
        z = torch.complex(out[..., first], out[..., second]) * by
        out[..., first], out[..., second] = z.real, z.imag
        return out

    out = [turned(s["query"], turn), turned(s["key"], turn)]
    if case["train"]:
        out += [turned(g, turn.conj()) for g in s["grads"]]
    return tuple(out)


def _exact_append(s, which):
    """The append, from sorted slots: (cache values, scales)."""
    case = s["case"]
    b, kind = case["block_size"], case["cache"]
    stored, scales = s[which + "_cache"].double(), s[which + "_scales"].double()
    slots, order = torch.sort(s["slot_mapping"])
    x = s[which].double()[order]
    touched, member = torch.unique_consecutive(slots // b, return_inverse=True)
    peak = torch.zeros((touched.shape[0], x.shape[1]), dtype=torch.float64, device="cuda")
    peak.scatter_reduce_(0, member[:, None].expand(-1, x.shape[1]), x.abs().amax(-1), "amax")
    # The least k with peak <= largest * 2^k, found from the logarithm and put right by one.
    k = torch.floor(torch.log2(peak.clamp(min=1e-300) / _LARGEST[kind]))
    k = torch.where(peak > _LARGEST[kind] * torch.exp2(k), k + 1, k)
    k = torch.where(peak > _LARGEST[kind] * torch.exp2(k), k + 1, k).clamp(min=-126)
    first = torch.full((touched.shape[0],), b, device="cuda").scatter_reduce_(0, member, slots % b, "amin")
    last = torch.zeros((touched.shape[0],), dtype=torch.int64, device="cuda").scatter_reduce_(0, member, slots % b, "amax")
    was = scales[touched]
    now = torch.where(first[:, None] == 0, torch.exp2(k), torch.maximum(was, torch.exp2(k)))
    rows = stored[touched]
    again = _nearest(rows * (was / now)[:, None, :, None], kind)
    inside = (torch.arange(b, device="cuda") < last[:, None]) & (first > 0)[:, None]
    change = inside[:, :, None, None] & (now != was)[:, None, :, None]
    rows = torch.where(change, again, rows)
    rows[member, slots % b] = _nearest(x / now[member][:, :, None], kind)
    stored[touched] = rows
    scales[touched] = now
    return stored if kind == "e4m3" else None, scales


def _nearest(x, kind):
    """The nearest 8-bit value: whole numbers, or 3 bits behind the leading one and no step under 2^-9."""
    if kind == "int8":
        return torch.round(x).clamp(-127, 127)
    power = torch.floor(torch.log2(x.abs().clamp(min=2.0**-20))).clamp(min=-6)
    step = torch.exp2(power - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def _exact_attention(s):
    """One request after the other, head by head, over its own tokens only."""
    case = s["case"]
    n, heads, dim, b = case["requests"], case["kv_heads"], case["head_dim"], case["block_size"]
    group = case["query_heads"] // heads
    out = torch.zeros((n, case["query_heads"], dim), dtype=torch.float64, device="cuda")
    scale = dim**-0.5
    for i, length in enumerate(s["context_lengths"].tolist()):
        blocks = s["block_tables"][i, : _blocks(length, b)].long()
        kept = {}
        for name in ("key", "value"):
            cache = s[name + "_cache"]
            part = cache.view(torch.uint8)[blocks].view(cache.dtype).double() * s[name + "_scales"][blocks].double()[:, None, :, None]
            kept[name] = part.reshape(-1, heads, dim)[:length]
        q = s["query"][i].double().view(heads, group, dim)
        p = torch.softmax(torch.einsum("hgd,thd->hgt", q, kept["key"]) * scale, -1)
        out[i] = torch.einsum("hgt,thd->hgd", p, kept["value"]).reshape(-1, dim)
    return out
