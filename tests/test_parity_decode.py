"""The token decoder's operators against their 64-bit oracle.

Tolerances, from the operations counted at each test: a result rounded to
type t is off by half a step of it, finfo(t).eps / 2 of its value; U = 2^-24 is
fp32's."""
import ctypes

import numpy as np
import pytest

from conftest import assert_bitexact, rng
from oracle import decode_ops as D

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DTYPES = [np.float32, np.float16]


def half_step(t):
    return float(np.finfo(t).eps) / 2


def within(got, want, tol, what=""):
    got = np.asarray(got, np.float64)
    assert got.shape == want.shape, what
    assert np.array_equal(np.isfinite(got), np.isfinite(want)), what
    ok = np.isfinite(want)
    assert np.array_equal(got[~ok], want[~ok]), what
    err, tol = np.abs(got[ok] - want[ok]), np.broadcast_to(tol, want.shape)[ok]
    assert np.all(err <= tol), f"{what}: {int((err > tol).sum())} of {err.size}, worst {(err / tol).max():.3g} of its bound"


# ------------------------------------------------------- norm and rotation
def rotary_tol(want, x, weight, amplitude, t):
    """The norm: a sum of D squares (D / 4 + 8 additions in a row at most), a
    mean, a root, a division, two products; the rotation: sine and cosine
    within 2 U, amplitude, two products and a sum of values of at most the row's
    largest; half a step of the result."""
    top = np.abs(x.astype(np.float64))
    if weight is not None:
        top = top / np.sqrt((top * top).mean(-1, keepdims=True) + 1e-6) * np.abs(weight)
    top = top.max(-1, keepdims=True) * max(1.0, abs(amplitude))
    return (x.shape[-1] / 8 + 4 + 6 + 8) * U * 2 * top + half_step(t) * np.abs(want) + 2.0 ** -25 * (t == np.float16)


ROTARY = [  # B, T, Hq, Hk, D, R, interleaved, norm, far
    (1, 1, 12, 12, 64, 64, False, True, 10),
    (2, 7, 8, 2, 128, 128, False, True, 100000),
    (1, 300, 4, 1, 128, 64, False, True, 2 ** 30),
    (3, 5, 3, 3, 80, 32, True, False, 10 ** 6),
    (2, 9, 2, 1, 96, 96, True, True, 5000),
    (1, 4, 2, 2, 256, 256, False, True, 5000),
    (1, 3, 5, 1, 50, 50, False, True, 99),
    (1, 3, 5, 1, 33, 12, True, True, 99),
    (2, 3, 1, 1, 1, 0, False, True, 9),
    (1, 2, 2, 1, 2, 2, True, True, 9),
    (1, 2, 1, 1, 256, 34, False, True, 9),
    (5, 1000, 2, 1, 64, 32, True, True, 9),
]


@pytest.mark.parametrize("case", ROTARY, ids=str)
@pytest.mark.parametrize("t", DTYPES)
def test_qk_norm_rotary(gpu, case, t):
    kk = gpu
    B, T, Hq, Hk, dim, R, inter, norm, far = case
    r = rng(hash(case) % 1000)
    qkv = (1.5 * r.normal(size=(B, T, Hq + 2 * Hk, dim))).astype(t)
    pos = (r.integers(0, far, (B, 1)) + np.arange(T)).astype(np.int64 if far > 2 ** 20 else np.int32)
    turns = kk.rotary_turns(R, factor=4.0)
    wq, wk = ((1 + 0.2 * r.normal(size=dim)).astype(np.float32), (1 + 0.2 * r.normal(size=dim)).astype(np.float16)) \
        if norm else (None, None)
    dev = kk.to_device(qkv)
    q, k = dev.slice_axis(2, 0, Hq), dev.slice_axis(2, Hq, Hq + Hk)
    D_ = kk.to_device
    oq, ok = kk.ops.qk_norm_rotary(q, k, D_(pos), D_(turns) if R else None, None if wq is None else D_(wq),
                                   None if wk is None else D_(wk), interleaved=inter, amplitude=1.25)
    for out, x, w in ((oq, qkv[:, :, :Hq], wq), (ok, qkv[:, :, Hq:Hq + Hk], wk)):
        want = D.rotated(x, w, pos, turns.tolist(), interleaved=inter, amplitude=1.25)
        assert out.dtype == t
        within(kk.to_host(out), want, rotary_tol(want, x, w, 1.25, t), str(case))


def test_rotary_far_and_negative_positions_lose_nothing(gpu):
    kk = gpu
    r = rng(5)
    x = r.normal(size=(1, 6, 2, 64)).astype(np.float32)
    pos = np.array([0, -1, 2 ** 31, -2 ** 40, 2 ** 62, 123456789012345], np.int64)
    turns = kk.rotary_turns(64)
    got = kk.to_host(kk.ops.rotary(kk.to_device(x), kk.to_device(pos), kk.to_device(turns)))
    want = D.rotated(x, None, pos[None], turns.tolist())
    within(got, want, rotary_tol(want, x, None, 1.0, np.float32))


@pytest.mark.parametrize("t", DTYPES)
def test_rotary_strides_in_place_and_misaligned(gpu, t):
    """Head-major operands, an offset of one value, the output over its input."""
    kk = gpu
    r = rng(6)
    turns, pos = kk.rotary_turns(64), np.arange(3, 14, dtype=np.int32)
    base = r.normal(size=(2, 4, 11, 65)).astype(t)
    dev = kk.to_device(base)
    x = dev.transpose([0, 2, 1, 3]).slice_axis(3, 1, 65)
    host = base.transpose(0, 2, 1, 3)[..., 1:]
    want = D.rotated(host, None, np.broadcast_to(pos, (2, 11)), turns.tolist())
    dpos, dturns = kk.to_device(pos), kk.to_device(turns)
    kk._lib.call("kk_qk_norm_rotary", x.desc(), None, x.desc(), None, None, None, dpos.desc(), dturns.desc(), 1e-6, 0,
                 1.0)
    within(kk.to_host(x), want, rotary_tol(want, host, None, 1.0, t))
    assert_bitexact(kk.to_host(dev)[..., 0], base[..., 0])


def test_rotary_empty_and_zero_rows(gpu):
    kk = gpu
    turns = kk.to_device(kk.rotary_turns(64))
    pos = kk.to_device(np.zeros(1, np.int32))
    for shape in ((0, 1, 2, 64), (2, 0, 2, 64), (2, 1, 0, 64)):
        assert kk.ops.rotary(kk.DeviceTensor.empty(shape), pos, turns).shape == shape
    z = kk.ops.qk_norm_rotary(kk.to_device(np.zeros((1, 1, 2, 64), np.float32)), None, pos, turns,
                              kk.to_device(np.ones(64, np.float32)))[0]
    assert not kk.to_host(z).any()


# ------------------------------------------------------------------- cache
def pool(r, B, columns, pages=None):
    """A table whose sequences share no page, unused entries of a pool mixed among them."""
    pages = pages or B * columns + 3
    return r.permutation(pages)[:B * columns].reshape(B, columns).astype(np.int32), pages


def random_cache(r, pages, Hk, block, dim):
    return (r.integers(-127, 128, (pages, Hk, block, dim)).astype(np.int8),
            r.uniform(0.01, 0.03, (pages, Hk)).astype(np.float32),
            r.integers(-127, 128, (pages, Hk, dim, block)).astype(np.int8),
            r.uniform(0.01, 0.03, (pages, Hk)).astype(np.float32))


def on_device(kk, parts):
    return kk.KVCache(*(kk.to_device(x) for x in parts))


def check_append(kk, parts, k, v, table, starts, counts, **views):
    cache = on_device(kk, parts)
    kk.ops.cache_append(cache, views.get("dev_k", kk.to_device(k)), views.get("dev_v", kk.to_device(v)), kk.to_device(table),
                        kk.to_device(starts), None if counts is None else kk.to_device(counts))
    n = np.full(len(starts), k.shape[1]) if counts is None else counts
    wk, wks = D.append(parts[0], parts[1], k, table, starts, n)
    wv, wvs = D.append(parts[2].swapaxes(2, 3), parts[3], v, table, starts, n)
    assert_bitexact(kk.to_host(cache.k_scale), wks, "key scales")
    assert_bitexact(kk.to_host(cache.v_scale), wvs, "value scales")
    assert_bitexact(kk.to_host(cache.k), wk, "keys")
    assert_bitexact(kk.to_host(cache.v), wv.swapaxes(2, 3), "values")
    return cache


@pytest.mark.parametrize("t", DTYPES)
@pytest.mark.parametrize("B,T,Hk,dim,block,held", [
    (1, 1, 1, 16, 16, 0), (5, 1, 2, 64, 32, 31), (3, 2, 1, 128, 16, 15), (2, 70, 2, 96, 32, 40), (1, 300, 3, 64, 64, 5),
    (2, 33, 1, 256, 128, 100), (1, 513, 1, 80, 256, 1), (40, 1, 8, 128, 64, 63)])
def test_cache_append(gpu, t, B, T, Hk, dim, block, held):
    kk = gpu
    r = rng(B + T)
    columns = (held + T) // block + 1
    table, pages = pool(r, B, columns)
    starts = r.integers(0, held + 1, B).astype(np.int32)
    starts[-1] = held
    counts = r.integers(0, T + 1, B).astype(np.int64)
    counts[0] = T
    # some rows far larger than a page's scale holds, some far smaller
    size = 10.0 ** r.uniform(-3, 1, (B, T, 1, 1))
    k, v = ((size * r.normal(size=(B, T, Hk, dim))).astype(t) for _ in range(2))
    check_append(kk, random_cache(r, pages, Hk, block, dim), k, v, table, starts, counts)


def test_cache_append_token_by_token_is_what_attention_reads(gpu):
    """Steps of one token: the scales grow as the page fills, and what it holds stays within its steps."""
    kk = gpu
    r = rng(8)
    x = (np.linspace(0.1, 3, 40)[None, :, None, None] * r.normal(size=(1, 40, 2, 32))).astype(np.float32)
    table = np.array([[1, 0, 2]], np.int32)
    cache = kk.KVCache.zeros(3, 2, 32, 16)
    parts = [kk.to_host(t) for t in (cache.k, cache.k_scale, cache.v, cache.v_scale)]
    for i in range(40):
        at = np.array([i], np.int32)
        cache = check_append(kk, parts, x[:, i:i + 1], x[:, i:i + 1], table, at, None)
        parts = [kk.to_host(t) for t in (cache.k, cache.k_scale, cache.v, cache.v_scale)]
    rows, there = D.cached(parts[0], parts[1], table[0], 40)
    values, _ = D.cached(parts[2], parts[3], table[0], 40, tokens_last=True)
    assert there.all() and np.array_equal(rows, values)
    # each change of the scale rounds once more: sixteen roundings of half a step at most
    step = np.repeat(parts[1][table[0, :3]], 16, axis=0)[:40, :, None]
    assert np.all(np.abs(rows - x[0]) <= 8.001 * step)
    k, v = cache.values()
    assert_bitexact(kk.to_host(k), parts[0].astype(np.float32) * parts[1][:, :, None, None])
    assert_bitexact(kk.to_host(v), parts[2].astype(np.float32) * parts[3][:, :, None, None])


def test_cache_append_ties_infinities_nan_and_tiny_values(gpu):
    kk = gpu
    r = rng(9)
    block, dim = 16, 16
    k = np.zeros((4, 3, 1, dim), np.float32)
    k[0, :, 0] = (r.integers(-253, 254, (3, dim)) / 2.0)  # halves of a step, once a row of 127 sets it to 1
    k[0, 0, 0, :2] = 127.0, -126.5
    k[1, :, 0] = r.normal(size=(3, dim))
    k[1, 0, 0, :4] = np.inf, -np.inf, np.nan, 3.0e38
    k[2, :, 0] = 1e-42 * r.normal(size=(3, dim))
    k[3, 1, 0] = np.nan
    table = np.arange(4, dtype=np.int32).reshape(4, 1)
    parts = random_cache(r, 4, 1, block, dim)
    starts = np.array([0, 5, 0, 0], np.int32)
    check_append(kk, parts, k, -k, table, starts, None)


def test_cache_append_leaves_out_what_lies_outside(gpu):
    """Negative and far starts, tokens past the table, pages outside the pool, counts past T and below 0."""
    kk = gpu
    r = rng(10)
    B, T, block, dim = 8, 20, 16, 32
    table, pages = pool(r, B, 2)
    table[3, 1], table[4, 0], table[5, 0] = -1, pages, 2 ** 31 - 1
    starts = np.array([-1, 2 ** 62, 25, 3, 3, 3, 0, 0], np.int64)
    counts = np.array([T, T, T, T, T, T, 1000, -5], np.int32)
    k, v = (r.normal(size=(B, T, 2, dim)).astype(np.float16) for _ in range(2))
    check_append(kk, random_cache(r, pages, 2, block, dim), k, v, table, starts, counts)


def test_cache_append_strided_rows(gpu):
    """Keys and values as views of a fused projection, head-major, at an odd offset."""
    kk = gpu
    r = rng(11)
    base = r.normal(size=(2, 3, 21, 2, 65)).astype(np.float32)
    dev = kk.to_device(base)
    views = {"dev_" + n: dev.transpose([0, 2, 1, 3, 4]).slice_axis(3, i, i + 1).squeeze([3]).slice_axis(3, 1, 65)
             for i, n in enumerate("kv")}
    k, v = (np.ascontiguousarray(base.transpose(0, 2, 1, 3, 4)[:, :, :, i, 1:]) for i in range(2))
    table, pages = pool(r, 2, 3)
    check_append(kk, random_cache(r, pages, 3, 16, 64), k, v, table, np.array([7, 0], np.int32), None, **views)


# --------------------------------------------------------------- attention
def attention_tol(q, k, v, want, scale, t, tokens):
    """Scores: D products and sums in fp32 of |q||k| in size, so each power of two is off by twice its share; sums over
    `tokens` in parts of 16 at the least; the powers and the quotient 8 U.  With fp16 operands a weight may be
    rounded to fp16 before its product with v."""
    q, k, v = (np.abs(np.asarray(x, np.float64)) for x in (q, k, v))
    if not k.size:
        return half_step(t) * np.abs(want)
    group = q.shape[-2] // k.shape[-2]
    most = max(float((q[..., h, :].reshape(-1, q.shape[-1]) @ k[:, h // group].T).max()) for h in range(q.shape[-2]))
    share = 2 * (q.shape[-1] + 8) * U * most * abs(scale) + (tokens / 16 + 16) * U
    if t == np.float16:
        share += half_step(t)
    return 2 * share * v.max() + half_step(t) * np.abs(want) + 2.0 ** -25 * (t == np.float16)


CACHE = [  # B, T, Hq, Hk, D, block, longest, window
    (1, 1, 12, 12, 64, 32, 1, 0),
    (1, 1, 12, 12, 64, 32, 389, 0),
    (3, 1, 8, 2, 128, 64, 700, 0),
    (2, 1, 7, 1, 96, 16, 333, 50),
    (1, 1, 40, 2, 64, 16, 257, 0),
    (2, 5, 4, 2, 64, 128, 300, 0),
    (1, 17, 8, 2, 128, 64, 130, 0),
    (2, 70, 2, 1, 80, 32, 201, 33),
    (1, 130, 3, 3, 256, 256, 260, 0),
    (1, 64, 6, 1, 16, 16, 64, 0),
    (1, 3, 1, 1, 240, 64, 5000, 0),
    (2, 2, 2, 2, 48, 32, 2500, 1),
]


@pytest.mark.parametrize("case", CACHE, ids=str)
@pytest.mark.parametrize("t", DTYPES)
def test_cache_attention(gpu, case, t):
    kk = gpu
    B, T, Hq, Hk, dim, block, longest, window = case
    r = rng(longest + T)
    columns = -(-longest // block)
    table, pages = pool(r, B, columns)
    lengths = r.integers(longest // 2, longest + 1, B).astype(np.int32)
    lengths[0] = longest
    counts = r.integers(0, T + 1, B).astype(np.int32)
    counts[0] = T
    parts = random_cache(r, pages, Hk, block, dim)
    for b in range(B):  # what lies behind the last token is anybody's
        table[b, -(-int(lengths[b]) // block):] = -7
    q = (1.5 * r.normal(size=(B, T, Hq, dim))).astype(t)
    scale = 1.3 / dim ** 0.5
    out = kk.to_host(kk.ops.cache_attention(kk.to_device(q), on_device(kk, parts), kk.to_device(table),
                                            kk.to_device(lengths), kk.to_device(counts), scale, window))
    for b in range(B):
        n = int(lengths[b])
        k, _ = D.cached(parts[0], parts[1], table[b], n)
        v, _ = D.cached(parts[2], parts[3], table[b], n, tokens_last=True)
        place = n - int(counts[b]) + np.arange(T)

        def seen(i):
            if i >= counts[b] or place[i] < 0:
                return []
            return np.arange(max(0, place[i] - window + 1) if window else 0, place[i] + 1)
        want = D.attention(q[b], k, v, seen, scale)
        within(out[b], want, attention_tol(q[b], k, v, want, scale, t, n), f"{case} sequence {b}")
        assert not out[b, counts[b]:].any()


@pytest.mark.parametrize("T", [1, 40])
def test_cache_attention_leaves_out_what_lies_outside(gpu, T):
    """Lengths below 0, of 0 and past the table, pages outside the pool, scales that are NaN where nothing is cached."""
    kk = gpu
    r = rng(12)
    B, Hq, Hk, dim, block, columns = 6, 4, 2, 64, 16, 5
    table, pages = pool(r, B, columns)
    parts = list(random_cache(r, pages, Hk, block, dim))
    lengths = np.array([0, -9, 2 ** 40, 77, 50, 33], np.int64)
    table[3, 1], table[3, 3], table[4, :] = pages, -2 ** 31, -1
    for i in (1, 3):
        parts[i][table[5, 3:]] = np.nan
    q = r.normal(size=(B, T, Hq, dim)).astype(np.float32)
    out = kk.to_host(kk.ops.cache_attention(kk.to_device(q), on_device(kk, parts), kk.to_device(table),
                                            kk.to_device(lengths)))
    assert not out[[0, 1, 4]].any()
    for b in (2, 3, 5):
        n = min(int(lengths[b]), columns * block)
        k, there = D.cached(parts[0], parts[1], table[b], n)
        v, _ = D.cached(parts[2], parts[3], table[b], n, tokens_last=True)

        def seen(i):
            return [j for j in range(min(n, int(lengths[b]) - T + i + 1)) if there[j]]
        want = D.attention(q[b], k, v, seen, dim ** -0.5)
        within(out[b], want, attention_tol(q[b], k, v, want, dim ** -0.5, np.float32, n), f"sequence {b}")


def test_cache_attention_past_32_bit_offsets(gpu):
    """A pool of 2.3 billion codes a side, the sequence in its last and first pages."""
    kk = gpu
    r = rng(13)
    Hk, dim, block = 8, 128, 64
    pages = 2_300_000_000 // (Hk * dim * block) + 1
    cache = kk.KVCache(kk.DeviceTensor.empty((pages, Hk, block, dim), np.int8), kk.DeviceTensor.empty((pages, Hk)),
                       kk.DeviceTensor.empty((pages, Hk, dim, block), np.int8), kk.DeviceTensor.empty((pages, Hk)))
    table = np.array([[pages - 1, 0, pages - 2]], np.int32)
    n = 150
    x = r.normal(size=(2, 1, n, Hk, dim)).astype(np.float32)
    kk.ops.cache_append(cache, kk.to_device(x[0]), kk.to_device(x[1]), kk.to_device(table),
                        kk.to_device(np.zeros(1, np.int32)))
    small = [np.zeros((3, Hk, block, dim), np.int8), np.zeros((3, Hk), np.float32)]
    kc, ks = D.append(*small, x[0], np.arange(3)[None], [0], [n])
    vc, vs = D.append(*small, x[1], np.arange(3)[None], [0], [n])
    k, _ = D.cached(kc, ks, [0, 1, 2], n)
    v, _ = D.cached(vc, vs, [0, 1, 2], n)
    for T in (1, 60):
        q = r.normal(size=(1, T, 16, dim)).astype(np.float32)
        out = kk.to_host(kk.ops.cache_attention(kk.to_device(q), cache, kk.to_device(table),
                                                kk.to_device(np.array([n], np.int32))))
        want = D.attention(q[0], k, v, lambda i: np.arange(n - T + i + 1), dim ** -0.5)
        within(out[0], want, attention_tol(q[0], k, v, want, dim ** -0.5, np.float32, n), f"T {T}")
    del cache
    kk.pool_trim(0)


CROSS = [  # B, T, S, Hq, Hk, D, mask's axes
    (1, 1, 1, 1, 1, 64, 0),
    (4, 1, 130, 12, 12, 64, 0),
    (2, 1, 1500, 8, 2, 128, 2),
    (2, 33, 65, 4, 1, 64, 3),
    (1, 150, 201, 6, 3, 80, 2),
    (1, 129, 512, 2, 2, 64, 0),
    (2, 20, 100, 2, 1, 33, 3),
    (1, 3, 70, 1, 1, 1, 2),
    (1, 40, 70, 2, 1, 256, 3),
    (1, 7, 300, 14, 2, 72, 0),
    (3, 2, 0, 2, 1, 64, 0),
]


@pytest.mark.parametrize("case", CROSS, ids=str)
@pytest.mark.parametrize("t", DTYPES)
def test_cross_attention(gpu, case, t):
    """Lengths from 0, masked states of NaN and infinities, masks that leave rows empty, fused keys and values."""
    kk = gpu
    B, T, S, Hq, Hk, dim, axes = case
    r = rng(S + T)
    kv = r.normal(size=(B, S, 2, Hk, dim)).astype(t)
    q = (1.5 * r.normal(size=(B, T, Hq, dim))).astype(t)
    lengths = r.integers(0, S + 1, B).astype(np.int32)
    lengths[0] = S
    mask = np.ones((B, T, S), bool)
    if axes == 2:
        mask &= (r.random((B, S)) < 0.7)[:, None]
    if axes == 3:
        mask &= r.random((B, T, S)) < 0.6
        mask[0, T // 2] = False
    clean = kv.copy()
    for b in range(B):
        hidden = ~mask[b].any(0) | (np.arange(S) >= lengths[b])
        kv[b, hidden] = np.array([np.nan, np.inf, -np.inf, np.finfo(t).min], t)[r.integers(0, 4, int(hidden.sum()))][
            :, None, None, None]
        clean[b, hidden] = 0
    dev = kk.to_device(kv)
    k, v = (dev.slice_axis(2, i, i + 1).squeeze([2]) for i in range(2))
    m = None if not axes else kk.to_device(mask if axes == 3 else mask[:, 0])
    out = kk.to_host(kk.ops.cross_attention(kk.to_device(q), k, v, kk.to_device(lengths), m, 0.2))
    assert out.dtype == t
    for b in range(B):
        def seen(i):
            return np.flatnonzero(mask[b, i] & (np.arange(S) < lengths[b]))
        want = D.attention(q[b], clean[b, :, 0], clean[b, :, 1], seen, 0.2)
        within(out[b], want, attention_tol(q[b], clean[b, :, 0], clean[b, :, 1], want, 0.2, t, S), f"{case} {b}")


@pytest.mark.parametrize("t", DTYPES)
@pytest.mark.parametrize("T", [1, 50])
def test_cross_attention_strides_and_broadcasts(gpu, t, T):
    """Head-major operands at an odd offset, one sequence's states for all, a mask broadcast over sequences."""
    kk = gpu
    r = rng(15)
    base = r.normal(size=(1, 3, 90, 65)).astype(t)
    q = r.normal(size=(2, 6, T, 64)).astype(t)
    mask = r.random((1, T, 90)) < 0.5
    x = kk.to_device(base).transpose([0, 2, 1, 3]).slice_axis(3, 1, 65).broadcast_to((2, 90, 3, 64))
    out = kk.to_host(kk.ops.cross_attention(kk.to_device(q).transpose([0, 2, 1, 3]), x, x, None, kk.to_device(mask)))
    k = base[0].transpose(1, 0, 2)[..., 1:]
    for b in range(2):
        qb = q[b].transpose(1, 0, 2)
        want = D.attention(qb, k, k, lambda i: np.flatnonzero(mask[0, i]), 0.125)
        within(out[b], want, attention_tol(qb, k, k, want, 0.125, t, 90))


@pytest.mark.parametrize("size", [1e-18, 1e-3, 1.0, 1e4, 1e18])
def test_cross_attention_over_fp32s_range(gpu, size):
    """States far larger and smaller than fp16 holds, rows of mixed sizes; scores of order one throughout."""
    kk = gpu
    r = rng(16)
    q = r.normal(size=(1, 40, 2, 64)).astype(np.float32)
    k = (size * r.normal(size=(1, 77, 2, 64))).astype(np.float32)
    v = (size * 10.0 ** r.uniform(-2, 2, (1, 77, 1, 1)) * r.normal(size=(1, 77, 2, 64))).astype(np.float32)
    out = kk.to_host(kk.ops.cross_attention(kk.to_device(q), kk.to_device(k), kk.to_device(v), scale=0.2 / size))
    want = D.attention(q[0], k[0], v[0], lambda i: np.arange(77), 0.2 / size)
    within(out[0], want, attention_tol(q[0], k[0], v[0], want, 0.2 / size, np.float32, 77))


@pytest.mark.parametrize("t", DTYPES)
def test_attention_of_large_scores(gpu, t):
    """Scores in the thousands: one state takes all the weight, none overflows."""
    kk = gpu
    r = rng(17)
    q, k, v = (r.normal(size=s).astype(t) for s in ((1, 20, 2, 64), (1, 90, 2, 64), (1, 90, 2, 64)))
    out = kk.to_host(kk.ops.cross_attention(kk.to_device(q), kk.to_device(k), kk.to_device(v), scale=100.0))
    want = D.attention(q[0], k[0], v[0], lambda i: np.arange(90), 100.0)
    within(out[0], want, attention_tol(q[0], k[0], v[0], want, 100.0, t, 90))


def test_attention_repeats_its_bits(gpu):
    """No order of parts shows: calls of the same inputs agree to the last bit."""
    kk = gpu
    r = rng(18)
    parts, table = random_cache(r, 64, 2, 64, 128), np.arange(64, dtype=np.int32)[None]
    cache, q = on_device(kk, parts), kk.to_device(r.normal(size=(1, 1, 8, 128)).astype(np.float32))
    length = kk.to_device(np.array([4000], np.int32))
    first = kk.to_host(kk.ops.cache_attention(q, cache, kk.to_device(table), length))
    for _ in range(5):
        assert_bitexact(kk.to_host(kk.ops.cache_attention(q, cache, kk.to_device(table), length)), first)


# ------------------------------------------------------------------ logits
@pytest.mark.parametrize("t", DTYPES)
@pytest.mark.parametrize("B,V,L", [(1, 1, 1), (3, 70, 9), (2, 1025, 350), (2, 8192, 3000), (5, 20001, 64), (1, 40000, 0)])
def test_process_logits(gpu, t, B, V, L):
    kk = gpu
    r = rng(V)
    x = (3 * r.normal(size=(B, V))).astype(t)
    x[0, 0] = np.inf
    # outside the vocabulary too
    history = np.where(r.random((B, L)) < 0.1, r.integers(-2 ** 31, 2 ** 31, (B, L)), r.integers(0, V, (B, L)) // 3)
    history = history.astype(np.int32 if V < 2000 else np.int64)
    lengths = r.integers(-1, L + 3, B).astype(np.int64)
    rep, pres, freq = (r.uniform(1, 2, B).astype(np.float32) for _ in range(3))
    bias, allowed = r.normal(size=(B, V)).astype(np.float32), r.random((B, V)) < 0.5
    allowed[-1] = B == 1  # a row that allows nothing
    dev = kk.to_device
    got = kk.to_host(kk.ops.process_logits(dev(x), dev(history), dev(lengths), dev(rep), dev(pres), dev(freq), dev(bias),
                                           dev(kk.allowed_bits(allowed))))
    want = D.logits(x, history, np.minimum(lengths, L), rep, pres, freq, bias, allowed)
    # quotient or product, two products' and three sums' roundings of values of this size
    n = max(1, L)
    size = np.where(np.isfinite(x.astype(np.float64)), np.abs(x.astype(np.float64)), 0) * 2 + 2 * n + 2 + np.abs(bias)
    within(got, want, 5 * U * size)


def test_process_logits_absent_parts_and_one_for_all(gpu):
    kk = gpu
    r = rng(20)
    dev = kk.to_device
    x = r.normal(size=(3, 50)).astype(np.float32)
    assert_bitexact(kk.to_host(kk.ops.process_logits(dev(x))), x)
    bias, allowed = r.normal(size=50).astype(np.float32), r.random((1, 50)) < 0.5
    got = kk.to_host(kk.ops.process_logits(dev(x), bias=dev(bias), allowed=dev(kk.allowed_bits(allowed))))
    assert_bitexact(got, np.where(allowed, x + bias, np.float32(-np.inf)))
    history = np.tile(np.arange(0, 40, 2, dtype=np.int32), (3, 1))
    got = kk.to_host(kk.ops.process_logits(dev(x), dev(history), presence=dev(np.array([0.5], np.float32))))
    want = x.copy()
    want[:, 0:40:2] -= np.float32(0.5)
    assert_bitexact(got, want)
    wide = dev(r.normal(size=(6, 101)).astype(np.float32))
    view = wide.slice_axis(0, 0, 6, 2).slice_axis(1, 1, 51)
    assert_bitexact(kk.to_host(kk.ops.process_logits(view)), kk.to_host(wide)[::2, 1:51])


# ------------------------------------------------------------------ graphs
def test_a_recorded_step_replays(gpu):
    """The whole step recorded with resident buffers, replayed between eager work, each replay as the eager call."""
    kk = gpu
    r = rng(21)
    B, H, dim, block = 2, 4, 64, 16
    table = kk.to_device(np.arange(8, dtype=np.int32).reshape(2, 4))
    cache = kk.KVCache.zeros(8, H, dim, block)
    turns = kk.to_device(kk.rotary_turns(dim))
    pos, lengths = kk.to_device(np.zeros((B, 1), np.int32)), kk.to_device(np.ones(B, np.int32))
    x = [kk.to_device(np.zeros((B, 1, H, dim), np.float32)) for _ in range(3)]
    enc = [kk.to_device(r.normal(size=(B, 600, H, dim)).astype(np.float32)) for _ in range(2)]
    outs = [kk.DeviceTensor.empty((B, 1, H, dim)) for _ in range(4)]
    logits, history = kk.DeviceTensor.empty((B, H * dim)), kk.to_device(np.zeros((B, 5), np.int32))
    freq = kk.to_device(np.ones(1, np.float32))

    def step():
        call = kk._lib.call
        call("kk_qk_norm_rotary", outs[0].desc(), outs[1].desc(), x[0].desc(), x[1].desc(), None, None, pos.desc(),
             turns.desc(), 1e-6, 0, 1.0)
        call("kk_cache_append", cache.k.desc(), cache.k_scale.desc(), cache.v.desc(), cache.v_scale.desc(),
             outs[1].desc(), x[2].desc(), table.desc(), starts.desc(), None)
        call("kk_cache_attention", outs[2].desc(), outs[0].desc(), cache.k.desc(), cache.k_scale.desc(),
             cache.v.desc(), cache.v_scale.desc(), table.desc(), lengths.desc(), None, 0.125, 0)
        call("kk_cross_attention", outs[3].desc(), outs[2].desc(), enc[0].desc(), enc[1].desc(), None, None, 0.125)
        call("kk_process_logits", logits.desc(), flat.desc(), history.desc(), None, None,
             None, freq.desc(), None, None)

    def load(i):
        for t in x:
            kk.ops.copy_into(t, kk.to_device(r.normal(size=t.shape).astype(np.float32)))
        kk.ops.copy_into(pos, kk.to_device(np.full((B, 1), i, np.int32)))
        kk.ops.copy_into(lengths, kk.to_device(np.full(B, i + 1, np.int32)))

    state = [cache.k, cache.k_scale, cache.v, cache.v_scale]
    load(0)
    starts, flat = pos.squeeze([1]), outs[3].reshape((B, H * dim))
    step()
    kk.sync()
    kk._lib.call("kk_graph_begin")
    step()
    g = ctypes.c_int(-1)
    kk._lib.call("kk_graph_end", ctypes.byref(g))
    for i in range(20):
        load(i)
        before = [t.astype(t.dtype) for t in state]
        step()
        eager = [kk.to_host(t) for t in outs + [logits] + state]
        for t, b in zip(state, before):
            kk.ops.copy_into(t, b)
        for t in outs + [logits]:
            kk.ops.copy_into(t, kk.ops.fill(t.shape, float("nan")))
        kk.sync()
        kk._lib.call("kk_graph_launch", g.value)
        for got, want in zip(outs + [logits] + state, eager):
            assert_bitexact(kk.to_host(got), want, f"replay {i}")
    kk._lib.call("kk_graph_destroy", g.value)
