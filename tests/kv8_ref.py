"""Plain statements of the jl_kv8_* operators in 64 bits (numpy), sequence by sequence and token by token."""
import math

import numpy as np

UNMAPPED = -1


def map_ref(held, added, table, free, cursor, block, capacity, token_slots, positions, slot_map):
    """Returns (lengths, offsets, cursor, result); table and the token arrays are changed in place."""
    n, per = table.shape
    left = len(free) - cursor if 0 <= cursor <= len(free) else 0
    tokens = asked = taken = refused = 0
    lengths, offsets = [], [0]
    for r in range(n):
        h, a = int(held[r]), int(added[r])
        start = tokens
        tokens += max(a, 0)
        bad = h < 0 or a < 0 or h + a > min(per * block, 2**31 - 1) or tokens > capacity
        have = 0 if bad else -(-h // block)
        need = 0 if bad else -(-(h + a) // block) - have
        asked += need
        served = not bad and (need == 0 or asked <= left)
        if served:
            for j in range(need):
                table[r, have + j] = free[cursor + asked - need + j]
            taken += need
        else:
            refused += 1
        lengths.append(h + a if served else h)
        offsets.append(min(tokens, 2**31 - 1))
        for t in range(start, min(tokens, capacity)):
            p = h + t - start if served else -1
            b = int(table[r, p // block]) if p >= 0 else -1
            token_slots[t], positions[t] = r, p
            slot_map[t] = b * block + p % block if b >= 0 else -1
    return (np.array(lengths, np.int32), np.array(offsets, np.int32), cursor + taken,
            np.array([min(tokens, capacity), taken, refused, min(asked, 2**31 - 1)], np.int32))


def rotate(x, cos, sin):
    """Pairs (2i, 2i + 1) of the last axis."""
    a, b = x[..., 0::2], x[..., 1::2]
    out = np.empty_like(x)
    out[..., 0::2], out[..., 1::2] = a * cos - b * sin, a * sin + b * cos
    return out


def quantise(x):
    """codes and scales of the rows of x (last axis), from their 64-bit values."""
    x = x.astype(np.float64)
    with np.errstate(invalid="ignore", over="ignore"):
        most = np.max(np.abs(x), -1)
    good = np.isfinite(x).all(-1)
    some = good & (most >= 2.0 ** -100)
    with np.errstate(invalid="ignore"):
        codes = np.rint(np.where(some[..., None], x, 0) * 127 / np.where(some, most, 1)[..., None]).astype(np.int8)
    return codes, np.where(good, np.where(some, most / 127, 0), np.nan)


def append_ref(codes, scales, k, v, slot_map, count, positions=None, cos=None, sin=None):
    """codes [2, blocks, heads, block, size] and 64-bit scales [2, blocks, heads, block], in place."""
    _, blocks, heads, block, d = codes.shape
    k = k.astype(np.float64).reshape(-1, heads, d)
    v = v.astype(np.float64).reshape(-1, heads, d)
    for t in range(count):
        place = int(slot_map[t])
        if not 0 <= place < blocks * block:
            continue
        for which, x in ((0, k[t]), (1, v[t])):
            if which == 0 and cos is not None:
                p = int(positions[t])
                with np.errstate(invalid="ignore"):
                    x = rotate(x, cos[p].astype(np.float64), sin[p].astype(np.float64)) if 0 <= p < len(cos) else np.full_like(x, np.nan)
            codes[which, place // block, :, place % block], scales[which, place // block, :, place % block] = quantise(x)


def attention_ref(codes, scales, q, table, kv_slots, positions, scale, window=0, cos=None, sin=None, count=None):
    """(out [rows, heads, size], lse [rows, heads], largest |score| per row) in 64 bits; rows from `count` on are None there: NaN."""
    _, blocks, kv_heads, block, d = codes.shape
    rows, heads = q.shape[:2]
    out, lse, most = np.zeros((rows, heads, d)), np.full((rows, heads), -np.inf), np.zeros(rows)
    group = heads // kv_heads
    for r in range(rows if count is None else min(rows, count)):
        slot = int(kv_slots[r]) if kv_slots is not None else r
        n, p = int(positions[r]) + 1, int(positions[r])
        if not 0 <= slot < len(table):
            continue
        j = np.arange(max(0, n - window) if window else 0, max(0, min(n, table.shape[1] * block)))
        b = table[slot][j // block].astype(np.int64)
        there = (b >= 0) & (b < blocks)
        j, b = j[there], b[there]
        if len(j) == 0:
            continue
        x = q[r].astype(np.float64)
        if cos is not None:
            x = rotate(x, cos[p].astype(np.float64), sin[p].astype(np.float64)) if p < len(cos) else np.full_like(x, np.nan)
        for h in range(kv_heads):
            mine = slice(h * group, (h + 1) * group)
            k, v = (codes[w, b, h, j % block].astype(np.float64) * scales[w, b, h, j % block].astype(np.float64)[:, None] for w in (0, 1))
            with np.errstate(all="ignore"):
                s = x[mine] @ k.T * scale
                m = np.max(s, -1, keepdims=True)
                base = np.where(m == -np.inf, 0.0, m)
                w = np.exp(s - base)
                total = w.sum(-1, keepdims=True)
                out[r, mine] = np.where(total == 0, 0, (w @ v) / np.where(total == 0, 1, total))
                lse[r, mine] = (base + np.log(total))[:, 0]
                most[r] = max(most[r], float(np.max(np.abs(s))))
    return out, lse, most


def rope_tables(rows, d, theta=500000.0):
    angle = np.arange(rows)[:, None] * theta ** (-np.arange(0, d, 2) / d)[None]
    return np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)


def score_tolerance(d, most):
    """How far a score of |score| <= most may be off: d products, their sum in binary32, each rounding at most 2^-23 of the partial
    sums (a matrix instruction may cut instead of round), which walk at random, and a few roundings of factors."""
    return 2.0 ** -22 * (8 + math.sqrt(d) * most)
