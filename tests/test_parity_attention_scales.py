"""Attention whose values are of far sizes: pages and rows that are large
beside the others, seen by some queries only, or seen and given no weight.

The bounds go by what a query weighs, sum_j p_j |v_j| from the 64-bit oracle
(|v_j| a row's largest), not by the largest value that it sees.  Score j is D
products and sums in fp32 of |q| |k_j| in size, so that its power of two is off
by e_j = 2 (D + 8) U |scale| |q| |k_j| of itself, and the quotient by their mean as
well; sums over the tokens in parts of 16 at the least; powers and quotient 8 U; a
weight in two halves keeps 2^-24 of itself and 2^-38 of the largest weight times
size, in one half (fp16 operands) 2^-11 and 2^-31."""
import numpy as np
import pytest

from conftest import rng
from oracle import decode_ops as D
from test_parity_attention import run_cache
from test_parity_decode import U, half_step, pool, random_cache, within

pytestmark = pytest.mark.gpu
DTYPES = [np.float32, np.float16]


def check(out, q, k, v, seen, scale, what=""):
    """out, q [T, Hq, D]; k, v [S, Hk, D]."""
    t = q.dtype.type
    q64, k64, v64 = (np.asarray(x, np.float64) for x in (q, k, v))
    want = D.attention(q64, k64, v64, seen, scale)
    group, tol = q.shape[1] // k.shape[1], np.zeros(want.shape)
    for i in range(q.shape[0]):
        at = np.asarray(seen(i), int)
        if not at.size:
            continue
        for h in range(q.shape[1]):
            g = h // group
            s = k64[at, g] @ q64[i, h] * scale
            p = np.exp(s - s.max())
            p /= p.sum()
            top = np.abs(v64[at, g]).max(-1)
            off = 2 * (q.shape[-1] + 8) * U * abs(scale) * (np.abs(k64[at, g]) @ np.abs(q64[i, h]))
            share = p @ off + (at.size / 16 + 16) * U + at.size * 2.0 ** -38
            if t == np.float16:
                share += half_step(t) + at.size * 2.0 ** -31
            tol[i, h] = p @ (off * top) + 2 * share * (p @ top)
    tol += half_step(t) * np.abs(want) + 2.0 ** -25 * (t == np.float16)
    within(out, want, tol, what)


def check_cache(out, q, parts, table, n, scale, window=0, what=""):
    """One sequence of n cached tokens, the newest q's own."""
    k, _ = D.cached(parts[0], parts[1], table, n)
    v, _ = D.cached(parts[2], parts[3], table, n, tokens_last=True)
    place = n - q.shape[0] + np.arange(q.shape[0])
    check(out, q, k, v, lambda i: np.arange(max(0, place[i] - window + 1) if window else 0, place[i] + 1), scale, what)


@pytest.mark.parametrize("t", DTYPES)
@pytest.mark.parametrize("block", [16, 32])
@pytest.mark.parametrize("group", [1, 2])
@pytest.mark.parametrize("jump", [4, 8, 12])
def test_windows_over_pages_whose_scales_jump(gpu, t, block, group, jump):
    """Large pages leave the windows of a wave's last queries as those before them still see them."""
    kk = gpu
    r = rng(100 * jump + block + group)
    T, dim, window = 96, 64, 200
    for n in (408, 409, 410):  # (the window passes a page's end at a wave's queries 31, 30, 29)
        table, pages = pool(r, 1, -(-n // block))
        parts = list(random_cache(r, pages, 8, block, dim))
        parts[1][table[0]] = np.linspace(0.005, 0.03, table.shape[1], dtype=np.float32)[:, None]
        parts[3] = (0.01 * np.where(r.random((pages, 8)) < 0.1, 2.0 ** jump, 1.0)).astype(np.float32)
        q = (1.5 * r.normal(size=(1, T, 8 * group, dim))).astype(t)
        out = run_cache(kk, q, parts, table, np.array([n], np.int32), scale=0.3, window=window)
        check_cache(out[0], q[0], parts, table[0], n, 0.3, window, f"{n} tokens")


@pytest.mark.parametrize("t", DTYPES)
@pytest.mark.parametrize("n", [360, 361, 362])
def test_one_large_page_behind_another_that_a_window_left(gpu, t, n):
    """Two pages of 100 among pages of 0.01: a query that has left the first behind meets the second."""
    kk = gpu
    r = rng(n)
    T, dim, block, window = 64, 64, 16, 200
    table, pages = pool(r, 1, -(-n // block))
    parts = list(random_cache(r, pages, 1, block, dim))
    parts[1] = np.full((pages, 1), 0.01, np.float32)
    for first in range(5, 12):
        for apart in range(4, 10):
            parts[3] = np.full((pages, 1), 0.01, np.float32)
            parts[3][table[0, [first, first + apart]], 0] = 100.0
            q = r.normal(size=(1, T, 1, dim)).astype(t)
            out = run_cache(kk, q, parts, table, np.array([n], np.int32), scale=0.1, window=window)
            check_cache(out[0], q[0], parts, table[0], n, 0.1, window, f"pages {first} and {first + apart}")


@pytest.mark.parametrize("t", DTYPES)
@pytest.mark.parametrize("T,group,dim,block,n", [
    (1, 1, 64, 16, 300), (1, 7, 128, 64, 900), (3, 2, 96, 32, 200), (20, 1, 48, 16, 150), (1, 4, 240, 128, 500), (40, 1, 64, 16, 300), (40, 2, 128, 64, 300), (70, 1, 96, 32, 200), (33, 1, 240, 16, 150), (90, 1, 64, 256, 700)])
@pytest.mark.parametrize("ratio", [1e3, 1e6, 1e9, 1e12, 1e30])
def test_a_page_of_large_scale_without_weight_takes_no_bits(gpu, t, T, group, dim, block, n, ratio):
    """Values `ratio` times the others', whose scores lie so far below that they weigh nothing, or (in a second head) as
    much as all the others together."""
    kk = gpu
    r = rng(T + dim)
    table, pages = pool(r, 1, -(-n // block))
    parts = list(random_cache(r, pages, 2, block, dim))
    parts[0] = r.integers(-12, 13, parts[0].shape).astype(np.int8)
    sign = np.where(r.random(dim) < 0.5, 1, -1)
    q = ((1 + 0.05 * r.random((1, T, 2 * group, dim))) * sign).astype(t)
    parts[1] = np.full((pages, 2), 0.01, np.float32)
    parts[3] = r.uniform(0.01, 0.02, (pages, 2)).astype(np.float32)
    for page in table[0, [0, (n - T) // block // 2]] if block < 256 else table[0, 1:2]:
        parts[0][page] = -127 * sign
        parts[1][page] = np.float32((np.log(ratio) + np.array([60, 0])) / (127 * dim))
        parts[3][page] *= np.float32(ratio)
    out = run_cache(kk, q, parts, table, np.array([n], np.int32), scale=1.0)
    at = np.unique(np.clip([0, 1, T // 2, T - 2, T - 1], 0, T - 1))  # (the queries that the oracle forms)
    k, _ = D.cached(parts[0], parts[1], table[0], n)
    v, _ = D.cached(parts[2], parts[3], table[0], n, tokens_last=True)
    check(out[0][at], q[0][at], k, v, lambda i: np.arange(n - T + at[i] + 1), 1.0)


def run_states(kk, q, k, v, mask=None, scale=1.0):
    dev = kk.to_device
    return kk.to_host(kk.ops.cross_attention(dev(q), dev(k), dev(v), mask=None if mask is None else dev(mask), scale=scale))


@pytest.mark.parametrize("T,group,dim,S", [(1, 1, 64, 300), (8, 1, 128, 90), (40, 2, 64, 300), (33, 1, 128, 1000), (200, 1, 96, 130),
                                           (40, 1, 200, 90), (50, 2, 33, 260)])
@pytest.mark.parametrize("by_query", [False, True])
@pytest.mark.parametrize("ratio", [1e3, 1e6, 1e9, 1e12, 1e30])
def test_states_of_large_values_without_weight_take_no_bits(gpu, T, group, dim, S, by_query, ratio):
    """As for pages: the rows that weigh nothing in one head weigh as much as all the others together in another."""
    kk = gpu
    r = rng(T + dim)
    sign = np.where(r.random(dim) < 0.5, 1.0, -1.0)
    q = ((1 + 0.05 * r.random((1, T, 2 * group, dim))) * sign).astype(np.float32)
    k = (0.1 * r.normal(size=(1, S, 2, dim))).astype(np.float32)
    v = r.normal(size=(1, S, 2, dim)).astype(np.float32)
    for row in (3, S // 2, S - 1):
        k[0, row] = -sign * (np.log(ratio) + np.array([[60], [0]])) / dim
        v[0, row] *= np.float32(ratio)
    mask = r.random((1, T, S)) < 0.8 if by_query else None
    if by_query:
        mask[:, :, [3, S // 2, S - 1]] = True
    out = run_states(kk, q, k, v, mask)
    at = np.unique(np.clip([0, 1, T // 2, T - 2, T - 1], 0, T - 1))
    check(out[0][at], q[0][at], k[0], v[0], lambda i: np.flatnonzero(mask[0, at[i]]) if by_query else np.arange(S), 1.0)


@pytest.mark.parametrize("T", [1, 40, 300])
def test_channels_of_mixed_sizes_keep_their_own_bits(gpu, T):
    """Channels of values 1e-9 to 1e9 in one row, queries' and keys' channels of opposite sizes: an output's bound goes
    by its own channel's values."""
    kk = gpu
    r = rng(T)
    dim, S = 64, 200
    size = 10.0 ** r.permutation(np.linspace(-9, 9, dim))
    q = (size * r.normal(size=(1, T, 1, dim))).astype(np.float32)
    k = (0.2 / size * r.normal(size=(1, S, 1, dim))).astype(np.float32)
    v = (r.permutation(size) * r.normal(size=(1, S, 1, dim))).astype(np.float32)
    out = run_states(kk, q, k, v)
    q64, k64, v64 = (np.asarray(x[0], np.float64) for x in (q, k, v))
    for i in np.unique([0, T // 2, T - 1]):
        s = k64[:, 0] @ q64[i, 0]
        p = np.exp(s - s.max())
        p /= p.sum()
        off = 2 * (dim + 8) * U * (np.abs(k64[:, 0]) @ np.abs(q64[i, 0]))
        share = p @ off + (S / 16 + 16) * U
        tol = (p * off) @ np.abs(v64[:, 0]) + 2 * share * (p @ np.abs(v64[:, 0]))
        within(out[0, i, 0], p @ v64[:, 0], tol, f"query {i}")


@pytest.mark.parametrize("t", DTYPES)
@pytest.mark.parametrize("T,by_query", [(1, False), (5, False), (40, False), (40, True), (200, True)])
def test_an_infinite_key_weighs_nothing_where_its_score_is_minus_infinity(gpu, t, T, by_query):
    """One value of one key is infinite: queries whose own value there is negative do as if it were not there, the
    others have no softmax."""
    kk = gpu
    r = rng(T)
    S, dim = 150, 64
    q = r.normal(size=(1, T, 1, dim)).astype(t)
    q[0, ::2, 0, 7] = -np.abs(q[0, ::2, 0, 7]) - t(0.1)
    q[0, 1::2, 0, 7] = np.abs(q[0, 1::2, 0, 7]) + t(0.1)
    k, v = (r.normal(size=(1, S, 1, dim)).astype(t) for _ in range(2))
    k[0, 100, 0, 7] = np.inf
    mask = r.random((1, T, S)) < 0.8 if by_query else np.ones((1, T, S), bool)
    mask[0, :, 100] = True
    out = run_states(kk, q, k, v, mask if by_query else None, 0.3)
    at = np.arange(0, T, 2)
    k[0, 100] = 0
    check(out[0][at], q[0][at], k[0], v[0], lambda i: [j for j in np.flatnonzero(mask[0, at[i]]) if j != 100], 0.3)
    assert np.isnan(out[0, 1::2]).all()
