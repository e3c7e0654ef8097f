"""Attention over the 4-bit cache against the 64-bit oracle, where its
kernels' ways part: few queries and many, sequences cut over blocks and joined,
holes in the table, windows, values of far sizes, what is not finite.

The bounds go by what a query weighs.  Score j is step_j (q . c_j) + low_j sum(q):
D products and sums each in fp32 of a size A_j = |scale| sum_d |q_d| (15 step_j +
|low_j|), so that its power of two is off by e_j = 2 (D + 8) U A_j of itself, and the
quotient by their mean as well; sums over the tokens in parts of 16 at the least,
powers and quotient 16 U; a weight times its value's step in two halves keeps 2^-22
of itself and 2^-32 of the largest such product; of fp16 queries in one half 2^-11 and
2^-31.  fp32 queries are the sum of two halves: 2^-22 of a score's size A_j."""
import ctypes

import numpy as np
import pytest

from conftest import assert_bitexact, rng
from oracle import decode_ops as D
from oracle import serve_ops as S
from test_parity_decode import U, half_step, within
from test_parity_serve import DTYPES, cache4

pytestmark = pytest.mark.gpu


def filled(r, pages, Hk, dim, block, step=0.3):
    """Parts of a cache whose steps and lowest values are those of rows around 0."""
    parts = [r.integers(0, 256, (pages, Hk, block, dim // 2)).astype(np.uint8), None,
             r.integers(0, 256, (pages, Hk, dim // 2, block)).astype(np.uint8), None]
    for i in (1, 3):
        steps = step * r.uniform(0.7, 1.3, (pages, Hk, block))
        parts[i] = np.stack([steps, -7.5 * steps * r.uniform(0.8, 1.2, steps.shape)], -1).astype(np.float16)
    return parts


def on_device(kk, parts):
    return kk.KVCache4(*(kk.to_device(x) for x in parts))


def pool(r, B, columns):
    pages = B * columns + 3
    return r.permutation(pages)[:B * columns].reshape(B, columns).astype(np.int32), pages


def run(kk, q, parts, table, lengths, counts=None, scale=None, window=0):
    dev = kk.to_device
    return kk.to_host(kk.ops.cache4_attention(dev(q), parts if isinstance(parts, kk.KVCache4) else on_device(kk, parts),
                                              dev(table), dev(lengths), None if counts is None else dev(counts), scale, window))


def check(out, q, parts, table, n, scale, window=0, count=None, queries=None, what=""):
    """Queries of one sequence [T, Hq, D] of n cached tokens, the newest `count` q's own."""
    T, t = q.shape[0], q.dtype.type
    count = T if count is None else count
    n = min(n, table.size * parts[0].shape[2])
    queries = np.arange(T) if queries is None else queries
    k, there = S.cached4(parts[0], parts[1], table, n)
    v, _ = S.cached4(parts[2], parts[3], table, n, tokens_last=True)

    def size(scales):  # 15 step + |low| of each token and head
        pages, block = scales.shape[0], scales.shape[2]
        x = np.abs(scales.astype(np.float64)) @ np.array([15.0, 1.0])
        page = np.repeat(table, block)[:n]
        return np.where(there[:, None], x[np.clip(page, 0, pages - 1), :, np.arange(n) % block], 0)
    ks, vs = size(parts[1]), size(parts[3])

    def seen(i):
        place = n - count + queries[i]
        if queries[i] >= count or place < 0:
            return np.zeros(0, int)
        at = np.arange(max(0, place - window + 1) if window else 0, min(place + 1, n))
        return at[there[at]]
    some = q[queries]
    want = D.attention(some, k, v, seen, scale)
    q64, group, tol = some.astype(np.float64), q.shape[1] // k.shape[1], np.zeros(want.shape)
    for i in range(len(queries)):
        at = seen(i)
        if not at.size:
            continue
        for h in range(q.shape[1]):
            g = h // group
            s = k[at, g] @ q64[i, h] * scale
            p = np.exp(s - s.max())
            p /= p.sum()
            A = abs(scale) * np.abs(q64[i, h]).sum() * ks[at, g]
            off = (2 * (q.shape[-1] + 8) * U + 2.0 ** -22 * (t == np.float32)) * A
            share = p @ off + (at.size / 16 + 16) * U + 2.0 ** -22 + (half_step(t) if t == np.float16 else 0)
            floor = at.size * (2.0 ** -31 if t == np.float16 else 2.0 ** -32) * (p * vs[at, g]).max()
            tol[i, h] = p @ (off * vs[at, g]) + 2 * share * (p @ vs[at, g]) + floor
    tol += half_step(t) * np.abs(want) + 2.0 ** -25 * (t == np.float16)
    within(out[queries], want, tol, what)


CASES = [  # B, T, Hq, Hk, D, block, longest, window
    (1, 1, 12, 12, 64, 32, 1, 0),
    (1, 1, 12, 12, 64, 32, 389, 0),
    (3, 1, 8, 2, 128, 64, 700, 0),
    (2, 1, 7, 1, 96, 16, 333, 50),
    (1, 1, 40, 2, 64, 16, 257, 0),
    (2, 5, 4, 2, 64, 128, 300, 0),
    (1, 17, 8, 2, 128, 64, 130, 0),
    (2, 70, 2, 1, 96, 32, 201, 33),
    (1, 130, 3, 3, 256, 256, 260, 0),
    (1, 64, 6, 1, 32, 16, 64, 0),
    (1, 3, 1, 1, 224, 64, 3000, 0),
    (2, 2, 2, 2, 160, 32, 1500, 1),
    (2, 33, 4, 1, 192, 128, 515, 0),
    (1, 32, 1, 1, 128, 16, 77, 0),
]


@pytest.mark.parametrize("case", CASES, ids=str)
@pytest.mark.parametrize("t", DTYPES)
def test_cache4_attention(gpu, case, t):
    kk = gpu
    B, T, Hq, Hk, dim, block, longest, window = case
    r = rng(longest + T)
    table, pages = pool(r, B, -(-longest // block))
    lengths = r.integers(longest // 2, longest + 1, B).astype(np.int32)
    lengths[0] = longest
    counts = r.integers(0, T + 1, B).astype(np.int32)
    counts[0] = T
    parts = filled(r, pages, Hk, dim, block)
    for b in range(B):  # what lies behind the last token is anybody's
        last = -(-int(lengths[b]) // block)
        table[b, last:] = -7
        if last and lengths[b] % block:
            parts[1][table[b, last - 1], :, lengths[b] % block:] = np.nan
            parts[3][table[b, last - 1], :, lengths[b] % block:] = np.inf
    q = (1.5 * r.normal(size=(B, T, Hq, dim))).astype(t)
    scale = 1.3 / dim ** 0.5
    out = run(kk, q, parts, table, lengths, counts, scale, window)
    for b in range(B):
        check(out[b], q[b], parts, table[b], int(lengths[b]), scale, window, int(counts[b]), what=f"sequence {b}")
        assert not out[b, counts[b]:].any()


@pytest.mark.parametrize("t", DTYPES)
@pytest.mark.parametrize("window", [0, 70, 2 ** 62])
def test_a_batch_past_a_waves_lanes(gpu, t, window):
    """150 sequences, lengths from 0."""
    kk = gpu
    r = rng(150)
    B, block, dim, longest = 150, 16, 32, 900
    lengths = np.where(r.random(B) < 0.1, 0, (longest * r.random(B) ** 3).astype(int)).astype(np.int32)
    lengths[[0, 64, 149]] = longest, 0, longest - 3
    table, pages = pool(r, B, -(-longest // block))
    parts = filled(r, pages, 2, dim, block)
    q = r.normal(size=(B, 1, 6, dim)).astype(t)
    out = run(kk, q, parts, table, lengths, scale=0.2, window=window)
    assert not out[lengths == 0].any()
    for b in [*range(0, 8), 62, 63, 64, 65, 127, 128, 129, 148, 149]:
        if lengths[b]:
            check(out[b], q[b], parts, table[b], int(lengths[b]), 0.2, min(window, 2 ** 20), what=f"sequence {b}")


@pytest.mark.parametrize("t", DTYPES)
@pytest.mark.parametrize("B,T,Hq,Hk,dim,block,longest,window", [
    (35, 70, 4, 4, 64, 16, 700, 0), (70, 40, 8, 4, 128, 64, 300, 40), (50, 130, 3, 3, 96, 32, 530, 0),
    (9, 600, 16, 8, 32, 128, 900, 0), (33, 520, 2, 2, 128, 16, 521, 0), (2, 9, 6, 2, 256, 64, 900, 0),
    (3, 25, 2, 1, 160, 16, 400, 70), (2, 12, 8, 2, 128, 16, 2100, 0), (80, 40, 4, 4, 64, 32, 500, 0),
    (1, 11, 9, 3, 224, 256, 5000, 0)])
def test_many_tiles_of_queries(gpu, t, B, T, Hq, Hk, dim, block, longest, window):
    """Batches whose tiles of queries fill the GPU once, nearly, or several times over."""
    kk = gpu
    r = rng(B * T)
    table, pages = pool(r, B, -(-longest // block))
    lengths = r.integers(1, longest + 1, B).astype(np.int32)
    lengths[[0, B - 1]] = longest, longest - 1
    counts = np.minimum(r.integers(0, T + 1, B), lengths).astype(np.int32)
    counts[0] = min(T, longest)
    parts = filled(r, pages, Hk, dim, block)
    q = (1.5 * r.normal(size=(B, T, Hq, dim))).astype(t)
    scale = 1.3 / dim ** 0.5
    out = run(kk, q, parts, table, lengths, counts, scale, window)
    for b in range(B):
        assert not out[b, counts[b]:].any()
    for b in sorted({0, min(1, B - 1), B // 2, B - 1}):
        some = np.unique(r.integers(0, T, 24))
        check(out[b], q[b], parts, table[b], int(lengths[b]), scale, window, int(counts[b]), some, f"sequence {b}")


@pytest.mark.parametrize("t", DTYPES)
@pytest.mark.parametrize("T", [1, 33])
def test_more_sequences_than_a_grids_axis(gpu, t, T):
    """33000 sequences of two heads that share their pages."""
    kk = gpu
    r = rng(33000)
    B, block, dim, at = 33000, 16, 32, [0, 1, 255, 32767, 32768, 32999]
    lengths = r.integers(0, 33, B).astype(np.int32)
    lengths[at] = [32, 1, 0, 17, 16, 31]
    table = np.broadcast_to(np.array([4, 1], np.int32), (B, 2))
    parts = filled(r, 5, 2, dim, block)
    q = np.broadcast_to(r.normal(size=(1, T, 2, dim)).astype(t), (B, T, 2, dim))
    out = run(kk, q, parts, table, lengths, scale=0.2)
    assert not out[lengths == 0].any()
    for b in at:
        if lengths[b]:
            check(out[b], q[b], parts, table[b], int(lengths[b]), 0.2, what=f"sequence {b}")


@pytest.mark.parametrize("t", DTYPES)
@pytest.mark.parametrize("T,Hq,Hk,dim,block,longest,window", [
    (1, 2, 1, 128, 64, 20011, 0), (1, 7, 1, 96, 32, 9000, 0), (1, 24, 1, 64, 16, 7001, 5000), (3, 8, 1, 64, 256, 6000, 0),
    (2, 12, 1, 96, 64, 4100, 130), (1, 16, 2, 192, 64, 5003, 0)])
def test_long_sequences_are_cut_and_joined(gpu, t, T, Hq, Hk, dim, block, longest, window):
    kk = gpu
    r = rng(longest)
    table, pages = pool(r, 2, -(-longest // block))
    lengths = np.array([longest, longest // 3], np.int64)
    parts = filled(r, pages, Hk, dim, block)
    q = (1.5 * r.normal(size=(2, T, Hq, dim))).astype(t)
    cache = on_device(kk, parts)
    out = run(kk, q, cache, table, lengths, scale=0.05, window=window)
    for b in range(2):
        check(out[b], q[b], parts, table[b], int(lengths[b]), 0.05, window, what=f"sequence {b}")
    for _ in range(3):
        assert_bitexact(run(kk, q, cache, table, lengths, scale=0.05, window=window), out)


@pytest.mark.parametrize("t", DTYPES)
@pytest.mark.parametrize("T,Hq,Hk,dim,block,longest,window", [
    (40, 7, 1, 64, 32, 1500, 0), (33, 4, 1, 96, 16, 700, 100), (300, 2, 1, 128, 64, 1111, 0), (17, 8, 2, 96, 128, 900, 0),
    (130, 3, 1, 256, 64, 600, 0), (700, 1, 1, 64, 64, 700, 33), (65, 2, 2, 160, 16, 333, 0)])
def test_chunks_of_tokens_over_a_cache(gpu, t, T, Hq, Hk, dim, block, longest, window):
    """Parts of the tokens joined where there are few queries; counts that leave queries without a place."""
    kk = gpu
    r = rng(T + longest)
    table, pages = pool(r, 2, -(-longest // block))
    lengths, counts = np.array([longest, longest - 7], np.int32), np.array([T, T - T // 3], np.int32)
    parts = filled(r, pages, Hk, dim, block)
    q = r.normal(size=(2, T, Hq, dim)).astype(t)
    cache = on_device(kk, parts)
    out = run(kk, q, cache, table, lengths, counts, 0.1, window)
    for b in range(2):
        some = np.unique(np.concatenate([[0, 1, T - 1, T // 2, int(counts[b]) - 1], r.integers(0, T, 12)]))
        check(out[b], q[b], parts, table[b], int(lengths[b]), 0.1, window, int(counts[b]), some, f"sequence {b}")
        assert not out[b, counts[b]:].any()
    assert_bitexact(run(kk, q, cache, table, lengths, counts, 0.1, window), out)


@pytest.mark.parametrize("t", DTYPES)
@pytest.mark.parametrize("T", [1, 3, 40])
def test_what_lies_outside_is_left_out(gpu, t, T):
    """Lengths below 0, of 0 and past the table, pages outside the pool, scales that are NaN where nothing is cached."""
    kk = gpu
    r = rng(12)
    B, Hq, Hk, dim, block, columns = 6, 4, 2, 64, 16, 5
    table, pages = pool(r, B, columns)
    parts = filled(r, pages, Hk, dim, block)
    lengths = np.array([0, -9, 2 ** 40, 77, 50, 33], np.int64)
    table[3, 1], table[3, 3], table[4, :] = pages, -2 ** 31, -1
    for i in (1, 3):
        parts[i][table[5, 3:]] = np.nan
    q = r.normal(size=(B, T, Hq, dim)).astype(t)
    out = run(kk, q, parts, table, lengths)
    assert not out[[0, 1, 4]].any()
    for b in (3, 5):
        check(out[b], q[b], parts, table[b], int(lengths[b]), dim ** -0.5, what=f"sequence {b}")
    for i in range(T):  # (sequence 2's queries lie past the table: all see all)
        check(out[2, i:i + 1], q[2, i:i + 1], parts, table[2], columns * block, dim ** -0.5)


@pytest.mark.parametrize("t", DTYPES)
@pytest.mark.parametrize("T,group", [(3, 2), (20, 2), (90, 1)])
@pytest.mark.parametrize("part,at", [(1, 0), (1, 1), (3, 0), (3, 1)])
def test_scales_that_are_not_finite_stay_with_the_queries_that_see_them(gpu, t, T, group, part, at):
    """A step or a lowest value of NaN or infinity near the end: what comes before it does not know it."""
    kk = gpu
    r = rng(T)
    block, dim, n = 16, 64, 400
    table, pages = pool(r, 1, n // block)
    parts = filled(r, pages, 2, dim, block)
    bad = n - T + T // 3
    parts[part][table[0, bad // block], :, bad % block, at] = np.inf if T == 90 else np.nan
    q = r.normal(size=(1, T, 2 * group, dim)).astype(t)
    out = run(kk, q, parts, table, np.array([n], np.int32), scale=0.1)
    place = n - T + np.arange(T)
    clean = np.flatnonzero(place < bad)
    clean_parts = [np.nan_to_num(x, nan=0.0, posinf=0.0) if x.dtype == np.float16 else x for x in parts]
    if clean.size:
        check(out[0], q[0], clean_parts, table[0], n, 0.1, queries=clean)
    # (a value of a code 0 times an infinite step is NaN as well: all of the row is poisoned)
    assert not np.isfinite(out[0][place >= bad]).any()


@pytest.mark.parametrize("t", DTYPES)
@pytest.mark.parametrize("T", [1, 30, 96])
@pytest.mark.parametrize("jump", [4, 8, 12])
def test_values_of_far_sizes(gpu, t, T, jump):
    """Tokens of large steps that few queries see, or that get no weight, take no bits from the others."""
    kk = gpu
    r = rng(100 * jump + T)
    dim, block, window, n = 64, 16, 200, 409
    table, pages = pool(r, 1, -(-n // block))
    parts = filled(r, pages, 2, dim, block)
    factor = np.where(r.random((pages, 2, block)) < 0.1, 2.0 ** jump, 1.0)
    parts[3] = (parts[3].astype(np.float64) * 0.01 * factor[..., None]).astype(np.float16)
    q = (1.5 * r.normal(size=(1, T, 4, dim))).astype(t)
    out = run(kk, q, parts, table, np.array([n], np.int32), scale=0.15, window=window)
    check(out[0], q[0], parts, table[0], n, 0.15, window)
    # keys of large steps whose scores lose, beside values of all sizes
    parts[1][..., 1] -= (factor > 1) * np.float16(60)
    q = np.abs(q)
    out = run(kk, q, parts, table, np.array([n], np.int32), scale=0.15, window=window)
    check(out[0], q[0], parts, table[0], n, 0.15, window)


@pytest.mark.parametrize("t", DTYPES)
@pytest.mark.parametrize("T", [2, 70])
def test_steps_of_nothing(gpu, t, T):
    """Rows of one value have a step of 0; fp16's smallest steps keep their bits."""
    kk = gpu
    r = rng(31)
    dim, block, n = 96, 32, 300
    table, pages = pool(r, 1, -(-n // block))
    parts = filled(r, pages, 1, dim, block)
    parts[3][..., 0] = 0
    q = r.normal(size=(1, T, 4, dim)).astype(t)
    out = run(kk, q, parts, table, np.array([n], np.int32), scale=0.1)
    check(out[0], q[0], parts, table[0], n, 0.1)
    if t == np.float32:
        parts[3] = np.stack([np.full(parts[3].shape[:-1], 2.0 ** -24), 0 * parts[3][..., 0]], -1).astype(np.float16)
        out = run(kk, q, parts, table, np.array([n], np.int32), scale=0.1)
        check(out[0], q[0], parts, table[0], n, 0.1)
    parts[1][..., 0] = 0
    out = run(kk, q, parts, table, np.array([n], np.int32), scale=0.1)
    check(out[0], q[0], parts, table[0], n, 0.1)


@pytest.mark.parametrize("t", DTYPES)
@pytest.mark.parametrize("T", [1, 50])
@pytest.mark.parametrize("scale", [20.0, -0.2, 0.0])
def test_scores_of_any_size_and_sign(gpu, t, T, scale):
    kk = gpu
    r = rng(32)
    dim, block, n = 64, 64, 200
    table, pages = pool(r, 1, -(-n // block))
    parts = filled(r, pages, 2, dim, block)
    q = r.normal(size=(1, T, 4, dim)).astype(t)
    out = run(kk, q, parts, table, np.array([n], np.int32), scale=scale)
    check(out[0], q[0], parts, table[0], n, scale)


@pytest.mark.parametrize("T", [1, 40])
@pytest.mark.parametrize("size", [2.0 ** -60, 2.0 ** 60])
def test_fp32_queries_of_any_size(gpu, T, size):
    kk = gpu
    r = rng(33)
    dim, block, n = 64, 16, 120
    table, pages = pool(r, 1, -(-n // block))
    parts = filled(r, pages, 2, dim, block)
    q = (r.normal(size=(1, T, 2, dim)) * size).astype(np.float32)
    out = run(kk, q, parts, table, np.array([n], np.int32), scale=0.2 / size)
    check(out[0], q[0], parts, table[0], n, 0.2 / size)


@pytest.mark.parametrize("t", DTYPES)
@pytest.mark.parametrize("T", [1, 44])
def test_queries_that_are_not_finite_or_zero(gpu, t, T):
    """A query's own row alone: its neighbours in the block keep theirs."""
    kk = gpu
    r = rng(34)
    dim, block, n = 64, 32, 150
    table, pages = pool(r, 1, -(-n // block))
    parts = filled(r, pages, 2, dim, block)
    q = r.normal(size=(1, T, 6, dim)).astype(t)
    q[0, T - 1, 1, 3], q[0, 0, 4, 9] = np.nan, np.inf
    q[0, T - 1, 5] = 0
    out = run(kk, q, parts, table, np.array([n], np.int32), scale=0.1)
    assert np.isnan(out[0, T - 1, 1]).all() and np.isnan(out[0, 0, 4]).all()
    fine = q.copy()
    fine[~np.isfinite(fine).all(-1)] = 0
    got = out.copy()
    got[0, T - 1, 1] = got[0, 0, 4] = 0
    for h in (0, 2, 3, 5):
        one = fine[0][:, [h]]
        head = [x[:, [h // 3]] for x in parts]
        check(got[0][:, [h]], one, head, table[0], n, 0.1, what=f"head {h}")


@pytest.mark.parametrize("t", DTYPES)
@pytest.mark.parametrize("T", [1, 37])
def test_views_and_rows_that_start_anywhere(gpu, t, T):
    kk = gpu
    r = rng(35)
    dim, block, n, B = 96, 16, 90, 2
    table, pages = pool(r, B, -(-n // block))
    parts = filled(r, pages, 3, dim, block)
    base = r.normal(size=(B, 6, T, dim + 3)).astype(t)
    view = kk.to_device(base).transpose([0, 2, 1, 3]).slice_axis(3, 1, dim + 1)
    wide = kk.to_device(np.full((B, 11), -1, np.int32))
    kk.ops.copy_into(wide.slice_axis(1, 2, 2 + table.shape[1]), kk.to_device(table))
    lengths = np.array([n, n - 17], np.int64)
    out = kk.to_host(kk.ops.cache4_attention(view, on_device(kk, parts), wide.slice_axis(1, 2, 2 + table.shape[1]),
                                             kk.to_device(lengths), scale=0.1))
    q = np.ascontiguousarray(base.transpose(0, 2, 1, 3)[..., 1:dim + 1])
    assert_bitexact(out, run(kk, q, parts, table, lengths, scale=0.1))
    for b in range(B):
        check(out[b], q[b], parts, table[b], int(lengths[b]), 0.1)


def test_past_32_bit_offsets(gpu):
    """A pool of 2.3 billion bytes a side, the sequence in its last and first pages, written there and read."""
    kk = gpu
    r = rng(13)
    Hk, dim, block = 8, 128, 64
    pages = 2_300_000_000 // (Hk * dim // 2 * block) + 1
    empty = kk.DeviceTensor.empty
    cache = kk.KVCache4(empty((pages, Hk, block, dim // 2), np.uint8), empty((pages, Hk, block, 2), np.float16),
                        empty((pages, Hk, dim // 2, block), np.uint8), empty((pages, Hk, block, 2), np.float16))
    table = np.array([[pages - 1, 0, pages - 2]], np.int32)
    n = 150
    x = r.normal(size=(2, 1, n, Hk, dim)).astype(np.float32)
    j = np.arange(n)
    slots = (table[0][j // block].astype(np.int64) * block + j % block)[None]
    kk.ops.cache4_append(cache, kk.to_device(x[0]), kk.to_device(x[1]), kk.to_device(slots))
    small = [np.zeros((3, Hk, block, dim // 2), np.uint8), np.zeros((3, Hk, block, 2), np.float16)]
    kc, ks = S.append4(*small, x[0, 0], j)
    vc, vs = S.append4(*small, x[1, 0], j)
    parts = [kc, ks, vc.swapaxes(2, 3), vs]
    for T in (1, 60):
        q = r.normal(size=(1, T, 16, dim)).astype(np.float32)
        out = run(kk, q, cache, table, np.array([n], np.int32))
        check(out[0], q[0], parts, np.arange(3), n, dim ** -0.5, what=f"T {T}")
    del cache
    kk.pool_trim(0)


def test_two_recorded_calls_share_no_state(gpu):
    """Graphs of calls whose parts lie in the library's scratch, replayed in turn and between eager calls."""
    kk = gpu
    r = rng(36)
    block, graphs = 32, []
    for T, dim, n in ((1, 64, 5000), (60, 128, 1800), (2, 96, 3100)):
        table, pages = pool(r, 1, -(-n // block))
        parts = filled(r, pages, 1, dim, block)
        cache, q = on_device(kk, parts), kk.to_device(r.normal(size=(1, T, 2, dim)).astype(np.float32))
        out, dt, ln = kk.DeviceTensor.empty(q.shape), kk.to_device(table), kk.to_device(np.array([n], np.int32))

        def step(out=out, q=q, c=cache, dt=dt, ln=ln):
            kk._lib.call("kk_cache4_attention", out.desc(), q.desc(), c.k.desc(), c.k_scale.desc(), c.v.desc(),
                         c.v_scale.desc(), dt.desc(), ln.desc(), None, 0.1, 0)
        step()
        want = kk.to_host(out)
        check(want[0], kk.to_host(q)[0], parts, table[0], n, 0.1)
        kk._lib.call("kk_graph_begin")
        step()
        g = ctypes.c_int(-1)
        kk._lib.call("kk_graph_end", ctypes.byref(g))
        graphs.append((g, out, want, step))
    for i in range(6):
        for g, out, want, step in graphs if i % 2 else graphs[::-1]:
            kk.ops.copy_into(out, kk.ops.fill(out.shape, float("nan")))
            if i == 3:
                step()
            kk._lib.call("kk_graph_launch", g.value)
        for g, out, want, _ in graphs:
            assert_bitexact(kk.to_host(out), want)
    for g, *_ in graphs:
        kk._lib.call("kk_graph_destroy", g.value)


def test_pages_appended_and_read_as_a_server_does(gpu):
    """Pages planned, tokens appended by their slots, attended over, released and used again, for some steps."""
    kk = gpu
    r = rng(37)
    B, Hq, Hk, dim, block, columns = 4, 4, 2, 64, 16, 6
    pages = 14
    cache, _ = cache4(kk, pages, Hk, dim, block)
    dev = kk.to_device
    table, free, used = dev(np.full((B, columns), -1, np.int32)), dev(r.permutation(pages).astype(np.int32)), dev(np.zeros(1, np.int32))
    rows = [[np.zeros((0, Hk, dim), np.float32) for _ in range(2)] for _ in range(B)]
    starts = np.zeros(B, np.int32)
    for T in (20, 1, 1, 30, 5, 1, 17):
        counts = r.integers(1, T + 1, B).astype(np.int32)
        slots, _, lengths, granted, used = kk.ops.plan_pages(table, dev(starts), dev(counts), free, used, T, block)
        k, v, q = (r.normal(size=(B, T, h, dim)).astype(np.float32) for h in (Hk, Hk, Hq))
        kk.ops.cache4_append(cache, dev(k), dev(v), slots)
        out = kk.to_host(kk.ops.cache4_attention(dev(q), cache, table, lengths, granted, 0.2))
        given, ends = kk.to_host(granted), kk.to_host(lengths)
        assert ((given == counts) | (given == 0)).all()
        for b in range(B):
            rows[b] = [np.concatenate([old, new[b, :given[b]]]) for old, new in zip(rows[b], (k, v))]
            assert len(rows[b][0]) == ends[b]
            # the same rows in a cache of their own
            n, small = int(ends[b]), [np.zeros((columns, Hk, block, dim // 2), np.uint8), np.zeros((columns, Hk, block, 2), np.float16)]
            kc, ks = S.append4(*small, rows[b][0], np.arange(n))
            vc, vs = S.append4(*small, rows[b][1], np.arange(n))
            check(out[b], q[b], [kc, ks, vc.swapaxes(2, 3), vs], np.arange(columns), n, 0.2, 0, int(given[b]), what=f"{T} {b}")
        starts = ends.copy()
        ended = (starts > 50) | (given == 0)
        kk.ops.release_pages(table, dev(starts), dev(ended), free, used, block)
        for b in np.flatnonzero(ended):
            rows[b], starts[b] = [x[:0] for x in rows[b]], 0
    held = sum(-(-int(s) // block) for s in starts)
    assert int(kk.to_host(used)[0]) == held
