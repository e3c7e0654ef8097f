"""The serving decoder's operators against their 64-bit oracle.

Tolerances, from the operations counted at each test: a result rounded to
type t is off by half a step of it, finfo(t).eps / 2 of its value; U = 2^-24 is
fp32's.  Codes, slots, tokens and cached values are equal."""
import ctypes

import numpy as np
import pytest

from conftest import assert_bitexact, rng
from oracle import serve_ops as S
from test_parity_decode import U, half_step, within

pytestmark = pytest.mark.gpu
DTYPES = [np.float32, np.float16]


# -------------------------------------------------------------------- norms
def norm_tol(y, t, N):
    """A sum of N squares: a thread's in a row (64 of rows over a wave, 16 of longer ones), each square and addition
    U, then 16 levels at most, halved by the root; the addition of the residual U (twice in its square, once itself);
    mean, eps, root, quotient 3 U, two products 2 U; half a step of the result, fp16's smallest step."""
    return np.abs(y) * ((64 + 17 + 2) / 2 + 1 + 3 + 2) * U + half_step(t) * np.abs(y) + 2.0 ** -25 * (t == np.float16)


NORMS = [(1, 1), (1, 7), (5, 64), (4, 768), (3, 255), (2, 257), (7, 1000), (130, 513), (2, 2049), (3, 4096), (2, 5121),
         (3, 8192), (2, 16384), (1, 16383)]


@pytest.mark.parametrize("rows,N", NORMS)
@pytest.mark.parametrize("tx", DTYPES)
@pytest.mark.parametrize("tr", DTYPES + [None])
def test_rms_norm(gpu, rows, N, tx, tr):
    kk = gpu
    r = rng(N)
    x = (r.normal(size=(rows, N)) * np.where(r.random(N) < 0.05, 30, 1)).astype(tx)
    res = None if tr is None else (2 * r.normal(size=(rows, N))).astype(tr)
    w = (1 + 0.2 * r.normal(size=N)).astype(tx if N % 2 else np.float32)
    dev = kk.to_device
    got = kk.ops.rms_norm(dev(x), dev(w), None if res is None else dev(res), 1e-5)
    want, h = S.rms_norm(x, res, w, 1e-5)
    if res is None:
        y = kk.to_host(got)
    else:
        y, total = (kk.to_host(t) for t in got)
        assert total.dtype == tr
        within(total, h, (U + half_step(tr)) * np.abs(h) + 2.0 ** -25 * (tr == np.float16), "sum")
    assert y.dtype == tx
    within(y, want, norm_tol(want, tx, N), "norm")


@pytest.mark.parametrize("rows,N", NORMS)
@pytest.mark.parametrize("tx", DTYPES)
@pytest.mark.parametrize("tr", DTYPES + [None])
def test_rms_norm_quant(gpu, rows, N, tx, tr):
    kk = gpu
    r = rng(N + 1)
    x = (r.normal(size=(rows, N)) * np.where(r.random(N) < 0.05, 30, 1)).astype(tx)
    res = None if tr is None else (2 * r.normal(size=(rows, N))).astype(tr)
    if rows > 1:
        x[1] = 0
        if res is not None:
            res[1] = 0
    w = (1 + 0.2 * r.normal(size=N)).astype(np.float32)
    dev = kk.to_device
    got = kk.ops.rms_norm_quant(dev(x), dev(w), None if res is None else dev(res), 1e-5)
    codes, scales = (kk.to_host(t) for t in got[:2])
    y, h = S.rms_norm(x, res, w, 1e-5)
    assert np.array_equal(codes, S.rms_codes(x, res, w))
    want = np.abs(y).max(-1, keepdims=True) / 127
    within(scales, want, 1.001 * U * want, "scales")  # (formed in 64 bits)
    if res is not None:
        within(kk.to_host(got[2]), h, (U + half_step(tr)) * np.abs(h) + 2.0 ** -25 * (tr == np.float16), "sum")


def test_rms_norm_quant_ties_go_to_the_even_code(gpu):
    """Values that are halves of steps exactly, for largest values of any size."""
    kk = gpu
    for top in (127.0, 254.0, 3.0, 1.0, 0.7, 1000.0):
        top = float(np.float32(top))
        x = np.concatenate([[top], np.arange(-126.5, 127) / 127 * top, [top / 2, -top / 2]]).astype(np.float32)[None]
        codes, _ = kk.ops.rms_norm_quant(kk.to_device(x))
        assert np.array_equal(kk.to_host(codes), S.rms_codes(x, None, None)), top


def test_rms_norm_rows_that_are_not_finite(gpu):
    kk = gpu
    r = rng(3)
    x = r.normal(size=(6, 300)).astype(np.float32)
    clean = kk.to_host(kk.ops.rms_norm(kk.to_device(x)))
    c0, s0 = (kk.to_host(t) for t in kk.ops.rms_norm_quant(kk.to_device(x)))
    x[1, 17], x[4, 299] = np.nan, np.inf
    y = kk.to_host(kk.ops.rms_norm(kk.to_device(x)))
    c1, s1 = (kk.to_host(t) for t in kk.ops.rms_norm_quant(kk.to_device(x)))
    rest = [0, 2, 3, 5]
    assert_bitexact(y[rest], clean[rest])
    assert np.isnan(y[1]).all() and np.isnan(y[4, 299])
    assert np.array_equal(c1[rest], c0[rest]) and np.isnan(s1[[1, 4]]).all()
    assert_bitexact(s1[rest], s0[rest])


@pytest.mark.parametrize("t", DTYPES)
def test_rms_norm_views_in_place_and_misaligned(gpu, t):
    kk = gpu
    r = rng(4)
    base = r.normal(size=(4, 9, 203)).astype(t)
    dev = kk.to_device(base)
    views = [(dev.slice_axis(2, 1, 102), base[:, :, 1:102]), (dev.slice_axis(1, 0, 9, 3), base[:, ::3]),
             (dev.slice_axis(0, 1, 2).slice_axis(2, 3, 4), base[1:2, :, 3:4])]
    for view, x in views:
        y = kk.to_host(kk.ops.rms_norm(view))
        want, _ = S.rms_norm(x.reshape(-1, x.shape[-1]), None, None, 1e-6)
        within(y.reshape(want.shape), want, norm_tol(want, t, x.shape[-1]))
    # the sum in the residual's place, the norm in x's
    x, res = (r.normal(size=(5, 1000)).astype(t) for _ in range(2))
    dx, dr = kk.to_device(x), kk.to_device(res)
    y, total = (kk.to_host(z) for z in kk.ops.rms_norm(dx, residual=dr))
    kk._lib.call("kk_rms_norm", dx.desc(), dr.desc(), dx.desc(), dr.desc(), None, 1e-6)
    assert_bitexact(kk.to_host(dx), y)
    assert_bitexact(kk.to_host(dr), total)
    # rows broadcast, and none
    one = kk.to_device(x[:1])
    rows = kk.to_host(kk.ops.rms_norm(one.broadcast_to((3, 1000))))
    assert_bitexact(rows, np.repeat(rows[:1], 3, 0))
    assert kk.to_host(kk.ops.rms_norm(kk.to_device(np.zeros((0, 5), t)))).shape == (0, 5)


@pytest.mark.parametrize("shape,scale", [
    ((1, 256), (1, 1)), ((3, 260), (3, 1)), ((5, 4096), (5, 1)), ((2, 3, 1028), (2, 3, 1)), ((2, 3, 1028), (1, 3, 1)),
    ((7, 8196), ()), ((70000, 256), (70000, 1)), ((3, 255), (3, 1)), ((4, 12), (4, 1))])
def test_dequantize_rows(gpu, shape, scale):
    """Codes of tokens with their scales: products of fp32, equal to the last bit."""
    kk = gpu
    r = rng(shape[-1])
    q = r.integers(-127, 128, shape).astype(np.int8)
    s = np.asarray(r.uniform(-1e-2, 1e-2, scale), np.float32)
    s[(0,) * s.ndim] = 3e38
    with np.errstate(over="ignore"):
        want = q.astype(np.float32) * s
    dev = kk.to_device
    assert_bitexact(kk.to_host(kk.ops.dequantize(dev(q), dev(s))), want, "rows")
    if q.ndim == 2:  # views of rows of another length, and codes at an odd address
        wide = np.zeros((shape[0], shape[1] + 8), np.int8)
        for at in (4, 3):
            wide[:, at:at + shape[1]] = q
            view = dev(wide).slice_axis(1, at, at + shape[1])
            assert_bitexact(kk.to_host(kk.ops.dequantize(view, dev(s))), want, "views")


def test_rms_norm_quant_feeds_the_8_bit_product(gpu):
    """Codes and scales as matmul_integer_scaled takes them: its rows times the scales."""
    kk = gpu
    r = rng(5)
    x, w = r.normal(size=(33, 768)).astype(np.float32), r.integers(-127, 128, (768, 96)).astype(np.int8)
    ws = r.uniform(0.001, 0.002, 96).astype(np.float32)
    codes, scales = kk.ops.rms_norm_quant(kk.to_device(x))
    y = kk.ops.matmul_integer_scaled(codes, kk.to_device(w), None, None, kk.to_device(ws))
    y = kk.to_host(kk.ops.binary("Mul", y, scales))
    c, s = kk.to_host(codes).astype(np.int64), kk.to_host(scales).astype(np.float64)
    want = (c @ w.astype(np.int64)) * ws.astype(np.float64) * s
    within(y, want, 3 * U * np.abs(want))  # (a sum of whole numbers, exact; its rounding to fp32 and two products)


# -------------------------------------------------------------------- pages
def run_plan(kk, table, starts, counts, free, used, tokens, block, alias=False):
    dev = kk.to_device
    t, u = dev(table), dev(np.array([used], np.int32))
    out = kk.ops.plan_pages(t, dev(starts), None if counts is None else dev(counts), dev(free), u, tokens, block,
                            u if alias else None)
    slots, positions, lengths, granted, left = (kk.to_host(x) for x in out)
    return slots, positions, lengths, granted, int(left[0]), kk.to_host(t)


def check_plan(kk, table, starts, counts, free, used, tokens, block, alias=False):
    got = run_plan(kk, table, starts, counts, free, used, tokens, block, alias)
    want = S.plan(table, starts, counts, free, used, tokens, block)
    for name, g, w in zip(("slots", "positions", "lengths", "granted", "used", "table"), got, want):
        assert np.array_equal(g, w), name
    return got


@pytest.mark.parametrize("B,T,block,held", [
    (1, 1, 16, 0), (1, 0, 16, 5), (3, 1, 64, 700), (32, 1, 64, 2000), (300, 1, 16, 100), (700, 3, 32, 90), (5, 40, 16, 33),
    (257, 7, 256, 300), (4, 2047, 16, 50), (3, 2048, 32, 0), (3, 2049, 128, 1), (2, 6000, 64, 999)])
@pytest.mark.parametrize("t", [np.int32, np.int64])
@pytest.mark.parametrize("short", [False, True])
def test_plan_pages(gpu, B, T, block, held, t, short):
    kk = gpu
    r = rng(B + T + held)
    columns = -(-(held + T) // block) or 1
    table = r.integers(-3, 10 * B * columns, (B, columns)).astype(np.int32)
    starts, counts = r.integers(0, held + 1, B).astype(t), r.integers(-1, T + 2, B).astype(t)
    if B > 4:
        starts[3], counts[2] = -5, 2 ** 31 - 1 if t == np.int32 else 2 ** 62
        starts[1] = columns * block + 1
        starts[0], counts[0] = columns * block, 0
    wanted = int(sum(-(-(int(s) + min(max(int(c), 0), T)) // block) - -(-int(s) // block) for s, c in zip(starts, counts)))
    free = r.permutation(20 + (max(wanted // 2, 0) if short else wanted + 5)).astype(np.int32)
    free[::7] -= 1  # (negative pages among them)
    check_plan(kk, table, starts, counts, free, 17, T, block, alias=bool(B % 2))
    check_plan(kk, table, starts[:1], None, free, 0, T, block) if B == 1 else None


def test_plan_pages_odd_lists(gpu):
    kk = gpu
    table = np.full((2, 4), -1, np.int32)
    none = np.zeros(0, np.int32)
    two = np.array([5, 20], np.int64)
    for free, used in ((none, 0), (none, 3), (np.array([7], np.int32), -2), (np.array([7], np.int32), 9)):
        check_plan(kk, table, two, None, free, used, 12, 16)
    # one start for all, rows of a wider table, outputs that are views
    wide = kk.to_device(np.full((3, 9), -1, np.int32))
    slots, positions = kk.DeviceTensor.empty((3, 11), np.int64), kk.DeviceTensor.empty((3, 12), np.int32)
    kk.ops.copy_into(slots, kk.ops.fill(slots.shape, 77, np.int64))
    lengths, granted, used = (kk.DeviceTensor.empty((n,), np.int32) for n in (3, 3, 1))
    free = kk.to_device(np.arange(10, dtype=np.int32))
    kk._lib.call("kk_plan_pages", wide.slice_axis(1, 2, 7).desc(), slots.slice_axis(1, 1, 11).desc(),
                 positions.slice_axis(1, 2, 12).desc(), lengths.desc(), granted.desc(), used.desc(),
                 kk.to_device(np.zeros(1, np.int32)).desc(), None, free.desc(), kk.to_device(np.zeros(1, np.int32)).desc(), 16)
    got = kk.to_host(wide)
    assert got[:, 2].tolist() == [0, 1, 2] and (np.delete(got, 2, 1) == -1).all()
    s = kk.to_host(slots)
    assert (s[:, 0] == 77).all() and np.array_equal(s[:, 1:], np.arange(3)[:, None] * 16 + np.arange(10))


@pytest.mark.parametrize("B,columns,block", [(1, 1, 16), (7, 5, 32), (3, 2500, 16), (90, 40, 64), (1024, 3, 16), (2500, 7, 32)])
def test_release_pages(gpu, B, columns, block):
    kk = gpu
    r = rng(B * columns)
    table = r.integers(-2, 1000, (B, columns)).astype(np.int32)
    lengths = r.integers(-4, columns * block + 40, B).astype(np.int64)
    ended = r.random(B) < 0.6
    ended[0] = True
    for used in (B * columns, 3, 0, 2 ** 30, -1):
        free = r.integers(0, 1000, B * columns + 10).astype(np.int32)
        dev = kk.to_device
        t, f, u = dev(table), dev(free), dev(np.array([used], np.int32))
        kk.ops.release_pages(t, dev(lengths), dev(ended), f, u, block)
        wt, wf, wu = S.release(table, lengths, ended, free, used, block)
        assert np.array_equal(kk.to_host(t), wt) and np.array_equal(kk.to_host(f), wf) and int(kk.to_host(u)[0]) == wu


# --------------------------------------------------------------- 4-bit cache
def cache4(kk, pages, Hk, dim, block, r=None):
    """A KVCache4 and its parts on the host; anything in it where r is given."""
    def some(shape, t):
        if r is None:
            return np.zeros(shape, t)
        return r.integers(0, 256, shape).astype(t) if t == np.uint8 else r.normal(size=shape).astype(t)
    parts = [some((pages, Hk, block, dim // 2), np.uint8), some((pages, Hk, block, 2), np.float16),
             some((pages, Hk, dim // 2, block), np.uint8), some((pages, Hk, block, 2), np.float16)]
    return kk.KVCache4(*(kk.to_device(x) for x in parts)), parts


def check_append(kk, cache, parts, k, v, slots, dk=None, dv=None):
    dev = kk.to_device
    kk.ops.cache4_append(cache, dev(k) if dk is None else dk, dev(v) if dv is None else dv, dev(slots))
    flat = slots.reshape(-1)
    kc, ks = S.append4(parts[0], parts[1], k.reshape((-1,) + k.shape[2:]), flat)
    vc, vs = S.append4(parts[2].swapaxes(2, 3), parts[3], v.reshape((-1,) + v.shape[2:]), flat)
    want = [kc, ks, vc.swapaxes(2, 3), vs]
    for name, g, w in zip(("keys", "key scales", "values", "value scales"), (cache.k, cache.k_scale, cache.v, cache.v_scale), want):
        g = kk.to_host(g)
        if g.dtype == np.float16:
            assert np.array_equal(g.view(np.uint16) & 0x7fff, np.abs(w).view(np.uint16)), name  # (a lowest value may be -0)
        assert np.array_equal(g, w), name
    return want


@pytest.mark.parametrize("t", DTYPES)
@pytest.mark.parametrize("B,T,Hk,dim,block", [
    (1, 1, 1, 32, 16), (32, 1, 8, 128, 64), (3, 33, 2, 64, 32), (2, 70, 3, 96, 16), (1, 95, 1, 256, 256), (2, 31, 2, 224, 128),
    (5, 7, 12, 64, 64)])
def test_cache4_append_and_values(gpu, t, B, T, Hk, dim, block):
    """Slots in any order, some left out, over a cache that holds something."""
    kk = gpu
    r = rng(T + dim)
    pages = -(-B * T // block) + 2
    cache, parts = cache4(kk, pages, Hk, dim, block, r)
    slots = r.permutation(pages * block)[:B * T].astype(np.int64)
    if B * T > 4:
        slots[[0, 2]] = -1, pages * block
        slots[4] = 2 ** 40
    k, v = ((1.5 * r.normal(size=(B, T, Hk, dim))).astype(t) for _ in range(2))
    slots = slots.reshape(B, T) if T % 2 else np.clip(slots, -1, 2 ** 31 - 1).astype(np.int32).reshape(B, T)
    want = check_append(kk, cache, parts, k, v, slots)
    got_k, got_v = (kk.to_host(x) for x in cache.values())
    assert_bitexact(got_k, S.values4(want[0], want[1]).astype(np.float32) + np.float32(0))
    assert np.array_equal(got_v, S.values4(want[2].swapaxes(2, 3), want[3]).astype(np.float32).swapaxes(2, 3))


@pytest.mark.parametrize("t", DTYPES)
def test_cache4_append_odd_values(gpu, t):
    """Rows of one value, of ties, of infinities and NaN, of fp16's smallest and largest values."""
    kk = gpu
    top = float(np.finfo(t).max)
    rows = [np.zeros(64), np.full(64, -3.25), np.arange(64) % 31 / 2.0, 100 + np.arange(64) % 31 / 2.0,
            np.where(np.arange(64) % 5 == 0, np.nan, 1.0), np.full(64, np.nan), np.linspace(-top, top, 64),
            np.where(np.arange(64) == 7, np.inf, 0.5), np.where(np.arange(64) == 9, -np.inf, np.arange(64.0)),
            np.arange(64) * 2.0 ** -24, np.arange(64) * 2.0 ** -22, 1 + np.arange(64) * 2.0 ** -10, -np.arange(64) * 1e-3,
            np.where(np.arange(64) % 2 == 0, np.inf, -np.inf)]
    with np.errstate(over="ignore", invalid="ignore"):
        x = np.array(rows).astype(t)[None, :, None, :]
    cache, parts = cache4(kk, 2, 1, 64, 16)
    check_append(kk, cache, parts, x, x[:, ::-1], np.arange(len(rows), dtype=np.int32)[None])


def test_cache4_append_views(gpu):
    """Keys and values as views of a fused projection, head-major, at an odd offset; slots of strides."""
    kk = gpu
    r = rng(11)
    base = r.normal(size=(2, 3, 21, 2, 65)).astype(np.float32)
    dev = kk.to_device(base)
    dk, dv = (dev.transpose([0, 2, 1, 3, 4]).slice_axis(3, i, i + 1).squeeze([3]).slice_axis(3, 1, 65) for i in range(2))
    k, v = (np.ascontiguousarray(base.transpose(0, 2, 1, 3, 4)[:, :, :, i, 1:]) for i in range(2))
    cache, parts = cache4(kk, 4, 3, 64, 16)
    slots = r.permutation(64)[:42].reshape(21, 2)
    dslots = kk.to_device(slots).transpose()
    kk.ops.cache4_append(cache, dk, dv, dslots)
    second, _ = cache4(kk, 4, 3, 64, 16)
    want = check_append(kk, second, parts, k, v, np.ascontiguousarray(slots.T))
    assert np.array_equal(kk.to_host(cache.k), want[0]) and np.array_equal(kk.to_host(cache.v), want[2])


# ----------------------------------------------------------------- sampling
def check_sample(kk, x, u, temperature=None, top_k=None, top_p=None, min_p=None, device=None, most=0):
    """Tokens equal the oracle's but for at most `most` rows within 1e-9 of a border; logarithms within their rounding
    and what a sum in parts of 2^-34 leaves."""
    dev = kk.to_device
    args = [None if a is None else dev(a) for a in (temperature, top_k, top_p, min_p)]
    tokens, logs = (kk.to_host(z) for z in kk.ops.sample(dev(x) if device is None else device, dev(u), *args))
    near = 0
    for b in range(x.shape[0]):
        def of(a, default):
            return default if a is None else a[b if a.size > 1 else 0]
        token, log, border = S.sample(x[b], of(u, 0), of(temperature, 1.0), int(of(top_k, 0)), of(top_p, 1.0), of(min_p, 0.0))
        if tokens[b] != token:
            assert border < 1e-9, f"row {b}: {tokens[b]}, not {token}; border {border}"
            near += 1
            continue
        assert logs[b] == log or abs(logs[b] - log) <= U * abs(log) + 2.0 ** -33 + 1e-9, f"row {b}"
    assert near <= most
    return tokens


@pytest.mark.parametrize("t", DTYPES)
@pytest.mark.parametrize("B,V", [(1, 1), (3, 2), (4, 50), (6, 1025), (5, 4096), (5, 4097), (3, 20000), (3, 50257), (2, 131071),
                                 (2, 131072)])
@pytest.mark.parametrize("spread", [0.02, 1.0, 8.0])
def test_sample(gpu, t, B, V, spread):
    kk = gpu
    r = rng(V + B)
    f = np.float32
    for i in range(6):
        x = (spread * r.normal(size=(B, V))).astype(t)
        if i % 2:
            x[r.random((B, V)) < 0.3] = -np.inf
            x[:, V // 2] = 0
        u = r.random(B).astype(f)
        u[0] = (0.0, 1 - 2.0 ** -24, 0.5, u[0], 1.0, -1.0)[i]
        limits = dict(temperature=r.choice([0.0, 0.3, 1.0, 1.7, 50.0], B).astype(f),
                      top_k=r.choice([0, -1, 1, 2, 40, V // 2, V, 2 * V], B).astype(np.int32 if i % 2 else np.int64),
                      top_p=r.choice([1.0, 0.0, 0.1, 0.9, 0.999, 2.0], B).astype(f),
                      min_p=r.choice([0.0, 0.0, 0.01, 0.3, 1.0, 2.0], B).astype(f))
        if i:
            limits.pop(list(limits)[(i - 1) % 4])
        check_sample(kk, x, u, **limits)


@pytest.mark.parametrize("V", [60, 5000, 100000])
def test_sample_many_equal_logits(gpu, V):
    """More equal logits than are put in order: the lowest index first, by count and by weight."""
    kk = gpu
    r = rng(V)
    u = r.random(8).astype(np.float32)
    for levels in (1, 2, 3, 17):
        x = r.integers(0, levels, (8, V)).astype(np.float16) / 4
        for limits in (dict(), dict(top_k=np.array([V // 3], np.int32)), dict(top_p=np.array([0.7], np.float32)),
                       dict(min_p=np.array([0.9], np.float32)),
                       dict(top_k=np.array([V // 2 + 1], np.int64), top_p=np.array([0.6], np.float32),
                            min_p=np.array([0.5], np.float32), temperature=np.array([0.5], np.float32))):
            check_sample(kk, x, u, **limits)


def test_sample_rows_of_nothing_and_of_infinities(gpu):
    kk = gpu
    inf, low = np.inf, np.finfo(np.float32).min
    x = np.full((9, 70), -inf, np.float32)
    x[1, 33] = 5
    x[2, [3, 60]] = inf
    x[2, 5] = 1e30
    x[3] = np.nan
    x[4] = low
    x[5, 7], x[5, 9] = np.nan, 0.0
    x[6], x[6, 50] = low, 2.0
    x[7, [1, 2]] = -0.0, 0.0
    x[8, [4, 5]] = 3e38, -3e38
    for u in (0.0, 0.4, 0.6, 1 - 2.0 ** -24):
        tokens = check_sample(kk, np.where(np.isnan(x), -inf, x), np.full(9, u, np.float32), device=kk.to_device(x))
        assert tokens[[0, 3]].tolist() == [-1, -1] and tokens[[1, 5, 6, 8]].tolist() == [33, 9, 50, 4]
        assert tokens[2] == (3 if u < 0.5 else 60) and tokens[7] == (1 if u < 0.5 else 2)
        greedy = kk.to_host(kk.ops.sample(kk.to_device(x), kk.to_device(np.full(1, u, np.float32)),
                                          kk.to_device(np.array([np.nan], np.float32)))[0])
        assert greedy.tolist() == [-1, 33, 3, -1, 0, 9, 50, 1, 4]


def test_sample_views_and_no_logarithms(gpu):
    kk = gpu
    r = rng(21)
    base = r.normal(size=(6, 1501)).astype(np.float16)
    view = kk.to_device(base).slice_axis(0, 0, 6, 2).slice_axis(1, 1, 1501)
    u = r.random(3).astype(np.float32)
    tokens = check_sample(kk, base[::2, 1:], u, device=view)
    alone = kk.DeviceTensor.empty((3,), np.int32)
    kk._lib.call("kk_sample", alone.desc(), None, view.desc(), kk.to_device(u).desc(), None, None, None, None)
    assert np.array_equal(kk.to_host(alone), tokens)
    assert kk.to_host(kk.ops.sample(kk.to_device(base[:0]), kk.to_device(u[:0]))[0]).shape == (0,)


def test_sample_repeats_itself(gpu):
    """Nothing hangs on the order in which a row's blocks and lanes come."""
    kk = gpu
    r = rng(22)
    x, u = kk.to_device((3 * r.normal(size=(4, 131072))).astype(np.float32)), kk.to_device(r.random(4).astype(np.float32))
    p = kk.to_device(np.array([0.95], np.float32))
    first = [kk.to_host(z) for z in kk.ops.sample(x, u, top_p=p)]
    for _ in range(5):
        for g, w in zip(kk.ops.sample(x, u, top_p=p), first):
            assert_bitexact(kk.to_host(g), w)


@pytest.mark.parametrize("B,V", [(150, 60000), (330, 33000)])
def test_sample_many_long_rows(gpu, B, V):
    """More rows than there is room to cut as often as one, or at all."""
    r = rng(V)
    x = (2 * r.normal(size=(B, V))).astype(np.float16)
    check_sample(gpu, x, r.random(B).astype(np.float32), top_k=r.choice([0, 1, 50, 1000], B).astype(np.int32),
                 top_p=r.choice([1.0, 0.9, 0.5], B).astype(np.float32))


# ------------------------------------------------------------------- graphs
def test_recorded_draws_of_long_rows_replay(gpu):
    """Two recorded calls over rows cut into blocks, with rows of nothing, of equal logits and without a temperature
    among them, replayed by turns between eager calls, share no state."""
    kk = gpu
    r = rng(24)
    f = np.float32
    graphs = []
    for B, V, t in ((5, 50257, np.float32), (7, 20001, np.float16)):
        x, u, temperature, top_p = (kk.to_device(np.ones(s, d)) for s, d in (((B, V), t), ((B,), f), ((B,), f), ((B,), f)))
        tokens, logs = kk.DeviceTensor.empty((B,), np.int32), kk.DeviceTensor.empty((B,))
        args = [z.desc() for z in (tokens, logs, x, u, temperature)] + [None, top_p.desc(), None]
        kk._lib.call("kk_sample", *args)
        kk.sync()
        kk._lib.call("kk_graph_begin")
        kk._lib.call("kk_sample", *args)
        g = ctypes.c_int(-1)
        kk._lib.call("kk_graph_end", ctypes.byref(g))
        graphs.append((g.value, B, V, t, x, u, temperature, top_p, tokens, logs))
    for i in range(4):
        want = []
        for g, B, V, t, x, u, temperature, top_p, tokens, logs in graphs:
            host = (3 * r.normal(size=(B, V))).astype(t)
            host[1], host[2] = -np.inf, 0.25
            hu, ht, hp = r.random(B).astype(f), r.choice([0.5, 1.0], B).astype(f), r.choice([0.9, 1.0], B).astype(f)
            ht[0] = 0
            for to, of in ((x, host), (u, hu), (temperature, ht), (top_p, hp), (tokens, np.full(B, -7, np.int32))):
                kk.ops.copy_into(to, kk.to_device(of))
            want.append([kk.to_host(z) for z in kk.ops.sample(x, u, temperature, top_p=top_p)])
            check_sample(kk, host, hu, ht, top_p=hp)
        kk.sync()
        for g, *_ in graphs:
            kk._lib.call("kk_graph_launch", g)
        for (*_, tokens, logs), w in zip(graphs, want):
            assert_bitexact(kk.to_host(tokens), w[0], f"replay {i}")
            assert_bitexact(kk.to_host(logs), w[1], f"replay {i}")
    for g, *_ in graphs:
        kk._lib.call("kk_graph_destroy", g)


def test_a_recorded_serving_step_replays(gpu):
    """Pages, norm, append, attention and a token, recorded with resident buffers and replayed between eager work, each
    replay as the eager call."""
    kk = gpu
    r = rng(23)
    call = kk._lib.call
    B, H, dim, block, columns, width = 3, 4, 64, 16, 4, 256
    cache, _ = cache4(kk, 40, H, dim, block)
    table = kk.to_device(np.full((B, columns), -1, np.int32))
    free, used = kk.to_device(r.permutation(40).astype(np.int32)), kk.to_device(np.zeros(1, np.int32))
    starts, u = kk.to_device(np.zeros(B, np.int32)), kk.to_device(np.zeros(B, np.float32))
    x, res = (kk.to_device(np.zeros((B, 1, width), np.float32)) for _ in range(2))
    empty = kk.DeviceTensor.empty
    slots, positions = empty((B, 1), np.int64), empty((B, 1), np.int32)
    lengths, granted, tokens = (empty((B,), np.int32) for _ in range(3))
    y, total, out, codes = empty((B, 1, width)), empty((B, 1, width)), empty((B, 1, H, dim)), empty((B, 1, width), np.int8)
    scales, logs = empty((B, 1, 1)), empty((B,))
    q, logits = y.reshape((B, 1, H, dim)), out.reshape((B, width))

    def step():
        call("kk_plan_pages", table.desc(), slots.desc(), positions.desc(), lengths.desc(), granted.desc(), used.desc(),
             starts.desc(), None, free.desc(), used.desc(), block)
        call("kk_rms_norm", y.desc(), total.desc(), x.desc(), res.desc(), None, 1e-6)
        call("kk_rms_norm_quant", codes.desc(), scales.desc(), None, x.desc(), None, None, 1e-6)
        call("kk_cache4_append", cache.k.desc(), cache.k_scale.desc(), cache.v.desc(), cache.v_scale.desc(), q.desc(),
             q.desc(), slots.desc())
        call("kk_cache4_attention", out.desc(), q.desc(), cache.k.desc(), cache.k_scale.desc(), cache.v.desc(),
             cache.v_scale.desc(), table.desc(), lengths.desc(), granted.desc(), 0.125, 0)
        call("kk_sample", tokens.desc(), logs.desc(), logits.desc(), u.desc(), None, None, None, None)

    state = [cache.k, cache.k_scale, cache.v, cache.v_scale, table, used]
    made = [slots, positions, lengths, granted, tokens, y, total, out, codes, scales, logs]
    step()
    kk.sync()
    call("kk_graph_begin")
    step()
    g = ctypes.c_int(-1)
    call("kk_graph_end", ctypes.byref(g))
    kk.ops.copy_into(used, kk.to_device(np.zeros(1, np.int32)))
    kk.ops.copy_into(table, kk.ops.fill(table.shape, -1, np.int32))
    for i in range(columns * block):
        for t in (x, res):
            kk.ops.copy_into(t, kk.to_device(r.normal(size=t.shape).astype(np.float32)))
        kk.ops.copy_into(starts, kk.to_device(np.full(B, i, np.int32)))
        kk.ops.copy_into(u, kk.to_device(r.random(B).astype(np.float32)))
        before = [t.astype(t.dtype) for t in state]
        step()
        eager = [kk.to_host(t) for t in made + state]
        for t, b in zip(state, before):
            kk.ops.copy_into(t, b)
        for t in made:
            kk.ops.copy_into(t, kk.ops.fill(t.shape, 7, t.dtype))
        kk.sync()
        call("kk_graph_launch", g.value)
        for got, want in zip(made + state, eager):
            assert_bitexact(kk.to_host(got), want, f"replay {i}")
    assert int(kk.to_host(used)[0]) == B * columns
    call("kk_graph_destroy", g.value)
