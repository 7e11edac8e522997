"""Plain 64-bit forms of the rotary, slot map, 8-bit append and 8-bit attention operators,
written from their definitions (numpy on the CPU, loops where they are clearest), and the
error bounds that a correct kernel keeps."""

from __future__ import annotations

import math

import numpy as np

LARGEST = {"e4m3": 448.0, "int8": 127.0}
HALF_STEP = {"bf16": 2.0**-8, "fp16": 2.0**-11}  # half a step, relative to the value
TINY = {"bf16": 2.0**-133, "fp16": 2.0**-24}  # the smallest step (of subnormals)


# --------------------------------------------------------------------------- rotary
def rotary(x, positions, frequencies, interleaved, amplitude, inverse=False):
    """x [tokens, heads, head_dim] float64; (result, bound of the fp32 arithmetic)."""
    out, slack = x.copy(), np.zeros_like(x)
    n = len(frequencies)
    angle = positions.astype(np.float64)[:, None] * frequencies
    cos, sin = amplitude * np.cos(angle)[:, None], amplitude * np.sin(angle)[:, None]
    if inverse:
        sin = -sin
    i = np.arange(n)
    first, second = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
    a, b = x[..., first], x[..., second]
    out[..., first], out[..., second] = a * cos - b * sin, b * cos + a * sin
    # fp32: cosine and sine are good to 2^-22 absolutely (the fraction of a turn is rounded to
    # 2^-25 turns, 2^-22.3 radians; sincospi adds 2 ulp), two products, one sum; the angle
    # itself is good to 2^-52 of its turns.
    turns = np.abs(angle)[:, None] * 2.0**-50
    slack[..., first] = slack[..., second] = abs(amplitude) * (np.abs(a) + np.abs(b)) * (2.0**-21 + turns)
    return out, slack


def rounding(reference, dtype):
    return np.abs(reference) * HALF_STEP[dtype] * (1 + 2.0**-10) + TINY[dtype]


# --------------------------------------------------------------------------- slots
def slots(block_tables, has, gets, free, num_tokens, block_size):
    """(slot_mapping, positions, lengths, blocks_used, block_tables, whether all was well)."""
    tables = block_tables.copy()
    room = tables.shape[1] * block_size
    slot, position = np.full(num_tokens, -1, np.int64), np.zeros(num_tokens, np.int64)
    lengths, used, token, well = [], 0, 0, True
    for b, (h, n) in enumerate(zip(has.tolist(), gets.tolist())):
        well = well and h >= 0 and n >= 0 and h + n <= room
        h, n = min(max(h, 0), room), max(n, 0)
        end = min(h + n, room)
        for j in range(-(-h // block_size), -(-end // block_size)):
            well = well and used < len(free)
            tables[b, j] = free[used] if used < len(free) else -1
            used += 1
        for i in range(max(0, min(n, num_tokens - token))):
            p = h + i
            block = tables[b, p // block_size] if p < room else -1
            position[token + i] = p
            slot[token + i] = block * block_size + p % block_size if block >= 0 else -1
            well = well and block >= 0
        token += n
        lengths.append(end)
    return slot, position, np.array(lengths), used, tables, well and token <= num_tokens


# --------------------------------------------------------------------------- append
def nearest(x, kind):
    """The nearest 8-bit value of each x (float64 in, the values out), ties to even, saturating."""
    x = np.clip(x, -LARGEST[kind], LARGEST[kind])
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        if kind == "int8":
            return np.nan_to_num(np.rint(x), nan=0.0)
        magnitude = np.maximum(np.abs(x), 2.0**-20)
        step = 2.0 ** (np.maximum(np.floor(np.log2(magnitude)), -6) - 3)
        return np.rint(x / step) * step


def least_power(peak, kind):
    k = -126
    while peak > LARGEST[kind] * 2.0**k:
        k += 1
    return 2.0**k


def append(rows, cache, scales, slot_mapping, kind):
    """One cache: rows [T, H, D] float64, cache [N, B, H, D] values, scales [N, H]; new (cache,
    scales, whether all was well)."""
    cache, scales = cache.copy(), scales.copy()
    blocks, size = cache.shape[:2]
    runs, well = [], True
    for t, s in enumerate(slot_mapping.tolist()):
        if s >= blocks * size:
            well = False
        if s < 0 or s >= blocks * size:
            continue
        last = runs[-1][-1] if runs else None
        if last is not None and last[0] == t - 1 and last[1] < s and last[1] // size == s // size:
            runs[-1].append((t, s))
        else:
            runs.append([(t, s)])
    seen = set()
    for run in runs:
        block = run[0][1] // size
        if block in seen:
            well = False
            continue
        seen.add(block)
        tokens, offsets = [t for t, _ in run], [s % size for _, s in run]
        for h in range(cache.shape[2]):
            x = rows[tokens, h]
            finite = np.abs(x[np.isfinite(x)])
            need = least_power(finite.max() if finite.size else 0.0, kind)
            was = 0.0 if offsets[0] == 0 else scales[block, h]
            was = was if was > 0 and np.isfinite(was) else 0.0
            now = max(was, need)
            if offsets[0] > 0 and now != was:
                for o in range(offsets[-1]):
                    if o not in offsets:
                        cache[block, o, h] = nearest(cache[block, o, h] * was / now, kind)
            with np.errstate(invalid="ignore"):
                cache[block, offsets, h] = nearest(x / now, kind)
            scales[block, h] = now
    return cache, scales, well


# ------------------------------------------------------------------------- attention
def attention(query, key_cache, value_cache, key_scales, value_scales, tables, lengths, scale, dtype):
    """float64 inputs (caches: the stored values); (result, bound of the kernel's error).

    With A = sum_t p_t |vs_t v_t| and B = max_t scale * |ks_t| * sum_i |q_i k_ti|, the kernel's
    output differs from the result by at most the sum of
      * A * 2^-10: the weights of V rounded to fp16 (half a step, 2^-11, and as much again for
        what lies below fp16's normal range: N values of at most 2^-25 of the largest weight);
      * A * 2 * (B * (D + 16) * 2^-24 + 2^-18): fp32 scores, exponentials (2^-22 each), sums and
        rescaling, in the numerator and in the denominator;
      * A * 2 * max_t scale * |ks_t| * 2^-25 * max|q| * sum_i |k_ti|: queries brought to fp16;
      * the rounding of the output.
    """
    batch, heads, dim = query.shape
    blocks, size, kv_heads, _ = key_cache.shape
    out, slack = np.full(query.shape, np.nan), np.zeros(query.shape)
    room = tables.shape[1] * size
    for b in range(batch):
        n = min(max(int(lengths[b]), 0), room)
        t = np.arange(n)
        block = tables[b, t // size] if n else np.zeros(0, np.int64)
        good = (block >= 0) & (block < blocks)
        t, block = t[good], block[good]
        for h in range(heads):
            g = h // (heads // kv_heads)
            ks, vs = key_scales[block, g], value_scales[block, g]
            k, v = key_cache[block, t % size, g], value_cache[block, t % size, g]
            if not len(t):
                continue
            with np.errstate(invalid="ignore"):
                s = scale * ks * (k @ query[b, h])
                p = np.exp(s - s.max())
                p /= p.sum()
                out[b, h] = (p * vs) @ v
                a = (p * np.abs(vs)) @ np.abs(v)
                near = (scale * np.abs(ks) * (np.abs(k) @ np.abs(query[b, h]))).max()
                down = (scale * np.abs(ks) * np.abs(k).sum(1)).max() * 2.0**-25 * np.abs(query[b, h]).max()
                largest = (p * np.abs(vs)).max() * np.abs(v).max()
                slack[b, h] = a * (2.0**-10 + 2 * (near * (dim + 16) * 2.0**-24 + 2.0**-18 + down))
                slack[b, h] += len(t) * 2.0**-25 * largest
    return out, slack + rounding(np.nan_to_num(out), dtype)


def default_scale(dim):
    return 1.0 / math.sqrt(dim)
