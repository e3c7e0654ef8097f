"""CPU oracle of what a serving decoder adds: norms into 8 bits, pages and
slots, the 4-bit cache, sampling; in numpy's 64 bits.

TEST INFRASTRUCTURE ONLY, written from the formulas in include/kk.h, one
row, token or sequence at a time; pinned in tests/test_oracle_serve.py."""
import math

import numpy as np


def rms_norm(x, residual, weight, eps):
    """(y, h) of rows x [rows, N]."""
    h = np.asarray(x, np.float64)
    if residual is not None:
        h = h + np.asarray(residual, np.float64)
    y = h / np.sqrt((h * h).sum(-1, keepdims=True) / h.shape[-1] + eps)
    return (y if weight is None else y * np.asarray(weight, np.float64)), h


def rms_codes(x, residual, weight):
    """Codes of rms_norm_quant: rint(127 h w / max |h w|)."""
    h = np.asarray(x, np.float64)
    if residual is not None:
        h = h + np.asarray(residual, np.float64)
    z = h if weight is None else h * np.asarray(weight, np.float64)
    top = np.abs(z).max(-1, keepdims=True)
    return np.where(top > 0, np.rint(127.0 * z / np.where(top > 0, top, 1)), 0).astype(np.int8)


def plan(table, starts, counts, free, used, tokens, block):
    """(slots, positions, lengths, granted, used, table), all copies."""
    table = table.copy()
    B, columns = table.shape
    slots, positions = np.full((B, tokens), -1, np.int64), np.full((B, tokens), -1, np.int32)
    lengths, granted = np.zeros(B, np.int32), np.zeros(B, np.int32)
    used = min(max(int(used), 0), len(free))
    short, left = False, len(free) - used
    for b in range(B):
        start = int(starts[b])
        if not 0 <= start <= columns * block:
            continue
        count = tokens if counts is None else min(max(int(counts[b]), 0), tokens)
        lengths[b] = start
        if start + count > columns * block:
            continue
        have = -(-start // block)
        need = -(-(start + count) // block) - have
        if need:
            short = short or need > left
            if short:
                continue
            table[b, have:have + need] = free[used:used + need]
            used, left = used + need, left - need
        for t in range(count):
            p = start + t
            page = int(table[b, p // block])
            slots[b, t] = page * block + p % block if page >= 0 else -1
            positions[b, t] = p
        granted[b], lengths[b] = count, start + count
    return slots, positions, lengths, granted, used, table


def release(table, lengths, ended, free, used, block):
    """(table, free, used), copies."""
    table, free = table.copy(), free.copy()
    used = min(max(int(used), 0), len(free))
    back = []
    for b in range(table.shape[0]):
        if ended[b]:
            n = min(-(-max(int(lengths[b]), 0) // block), table.shape[1])
            back += [int(p) for p in table[b, :n] if p >= 0]
            table[b, :n] = -1
    back = back[:used]
    free[used - len(back):used] = back
    return table, free, used - len(back)


def append4(codes, scales, new, slots):
    """codes uint8 [pages, Hk, block, D / 2], scales f16 [pages, Hk, block, 2] (copied); new [N, Hk, D], slots [N]."""
    codes, scales = codes.copy(), scales.copy()
    pages, heads, block, half = codes.shape
    for n, slot in enumerate(slots):
        slot = int(slot)
        if not 0 <= slot < pages * block:
            continue
        for h in range(heads):
            x = np.clip(np.nan_to_num(new[n, h].astype(np.float64), nan=0.0), -65504.0, 65504.0)
            low = np.float16(np.float32(x.min()))
            step = np.float16(np.float32((x.max() - float(low)) / 15.0))
            code = np.zeros(2 * half, np.uint8)
            if step > 0:
                code = np.clip(np.rint((x - float(low)) / float(step)), 0, 15).astype(np.uint8)
            else:
                step = np.float16(0)
            codes[slot // block, h, slot % block] = code[:half] | code[half:] << 4
            scales[slot // block, h, slot % block] = step, low
    return codes, scales


def values4(codes, scales):
    """What the codes stand for [pages, Hk, block, D], in 64 bits."""
    both = np.concatenate([codes & 15, codes >> 4], -1).astype(np.float64)
    return both * scales[..., :1].astype(np.float64) + scales[..., 1:].astype(np.float64)


def cached4(codes, scales, table, length, tokens_last=False):
    """The `length` rows [S, Hk, D] of one sequence's cache, and whether each lies in a page of the pool."""
    if tokens_last:
        codes = codes.swapaxes(2, 3)
    pages, heads, block, half = codes.shape
    rows, there = np.zeros((length, heads, 2 * half)), np.zeros(length, bool)
    for j in range(length):
        page = int(table[j // block])
        if 0 <= page < pages:
            there[j] = True
            rows[j] = values4(codes[page, :, j % block], scales[page, :, j % block])
    return rows, there


def sample(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, log-probability, border) of one row x [V]; border: how near, relative to all that is kept, a running
    sum comes to where it would decide otherwise."""
    x = np.asarray(x, np.float64)
    live = np.flatnonzero(x > -np.inf)
    if not live.size:
        return -1, -math.inf, 1.0
    order = live[np.argsort(-x[live], kind="stable")]
    if not temperature > 0:
        return int(order[0]), 0.0, 1.0
    top = x[order[0]]
    w = np.array([1.0 if x[i] == top else math.exp((x[i] - top) / temperature) for i in order])
    border = 1.0
    if 0 < top_k < len(w):
        w = w[:top_k]
    if top_p < 1:
        upto = np.cumsum(w)
        want = max(float(top_p), 0.0) * upto[-1]
        keep = int(np.searchsorted(upto, want)) + 1
        border = min(border, np.abs(upto - want).min() / upto[-1] if top_p > 0 else 1.0)
        w = w[:keep]
    if min_p > 0:
        border = min(border, np.abs(w / min(float(min_p), 1.0) - 1).min() if min_p < 1 else 1.0)
        w = w[w >= min(float(min_p), 1.0)]
    upto = np.cumsum(w)
    want = min(max(float(u), 0.0), 1.0 - 2.0 ** -24) * upto[-1]
    at = min(int(np.searchsorted(upto, want, side="right")), len(w) - 1)
    border = min(border, np.abs(upto - want).min() / upto[-1] if u > 0 else 1.0)
    return int(order[at]), math.log(w[at] / upto[-1]), border
