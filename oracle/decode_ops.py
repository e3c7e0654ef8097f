"""CPU oracle of the token decoder's operators, in numpy's 64 bits.

TEST INFRASTRUCTURE ONLY, written from the formulas in include/kk.h, one
head, query or token at a time; pinned in tests/test_oracle_decode.py."""
import math

import numpy as np


def rotated(x, weight, positions, turns, eps=1e-6, interleaved=False, amplitude=1.0):
    """x [B, T, H, D]; positions [B, T]; turns whole numbers [R]."""
    x = np.asarray(x, np.float64)
    if weight is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(weight, np.float64)
    y = x.copy()
    n = len(turns)
    for b in range(x.shape[0]):
        for t in range(x.shape[1]):
            for i in range(n):
                part = int(positions[b][t]) * int(turns[i]) % (1 << 64)
                angle = 2 * math.pi * (part / 2.0 ** 64)
                c, s = math.cos(angle), math.sin(angle)
                j, k = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
                y[b, t, :, j] = amplitude * (x[b, t, :, j] * c - x[b, t, :, k] * s)
                y[b, t, :, k] = amplitude * (x[b, t, :, k] * c + x[b, t, :, j] * s)
    return y


def append(codes, scales, new, table, starts, counts):
    """codes [pages, Hk, block, D] (copied), scales [pages, Hk]; new [B, T, Hk, D]."""
    codes, scales = codes.copy(), scales.copy()
    pages, heads, block, _ = codes.shape
    for b in range(new.shape[0]):
        start, end = int(starts[b]), int(starts[b]) + min(int(counts[b]), new.shape[1])
        if start < 0:
            continue
        end = min(end, table.shape[1] * block)
        for column in range(start // block, -(-end // block)) if end > start else ():
            page = int(table[b, column])
            if not 0 <= page < pages:
                continue
            lo, hi = max(start, column * block), min(end, (column + 1) * block)
            held = lo - column * block
            for h in range(heads):
                rows = new[b, lo - start:hi - start, h].astype(np.float64)
                finite = np.abs(rows[np.isfinite(rows)])
                top = np.float32(finite.max() if finite.size else 0)
                s = np.float32(0) if top == 0 else max(top / np.float32(127), np.float32(2.0 ** -126))
                before = scales[page, h]
                if held:
                    s = max(s, before)
                    if s != before:
                        codes[page, h, :held] = np.rint(codes[page, h, :held] * (float(before) / float(s)))
                scales[page, h] = s
                if s == 0:
                    q = np.zeros_like(rows)
                else:
                    q = np.clip(np.rint(np.nan_to_num(rows / float(s), nan=0.0, posinf=127, neginf=-127)), -127, 127)
                codes[page, h, held:held + hi - lo] = q
    return codes, scales


def attention(q, k, v, seen, scale):
    """q [T, Hq, D]; k, v [S, Hk, D]; seen(t) -> the places that query t sees."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    y = np.zeros(q.shape)
    group = q.shape[1] // k.shape[1]
    for t in range(q.shape[0]):
        at = np.asarray(seen(t), int)
        if not at.size:
            continue
        for h in range(q.shape[1]):
            s = k[at, h // group] @ q[t, h] * scale
            p = np.exp(s - s.max())
            y[t, h] = p @ v[at, h // group] / p.sum()
    return y


def cached(codes, scales, table, length, tokens_last=False):
    """The `length` rows [S, Hk, D] of one sequence's cache, and whether each lies in a page of the pool."""
    if tokens_last:
        codes = codes.swapaxes(2, 3)
    pages, heads, block, dim = codes.shape
    rows, there = np.zeros((length, heads, dim)), np.zeros(length, bool)
    for j in range(length):
        page = int(table[j // block])
        if 0 <= page < pages:
            there[j] = True
            rows[j] = codes[page, :, j % block].astype(np.float64) * scales[page].astype(np.float64)[:, None]
    return rows, there


def logits(x, history, lengths, repetition, presence, frequency, bias, allowed):
    """x [B, V]; one value a row of the penalties; bias [B, V]; allowed bool [B, V]."""
    y = np.asarray(x, np.float64).copy()
    for b in range(y.shape[0]):
        count = {}
        for token in history[b][:max(0, int(lengths[b]))]:
            count[int(token)] = count.get(int(token), 0) + 1
        for token, n in count.items():
            if 0 <= token < y.shape[1]:
                z = y[b, token]
                y[b, token] = (z / repetition[b] if z > 0 else z * repetition[b]) - frequency[b] * n - presence[b]
        y[b] += bias[b]
        y[b, ~allowed[b]] = -np.inf
    return y
