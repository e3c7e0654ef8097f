"""Attention over the 4-bit cache at the ends of its types: scales near fp16's
largest, queries of nothing, batches that a block's threads go through."""
import numpy as np
import pytest

from conftest import rng
from test_parity_attention4 import check, filled, pool, run
from test_parity_serve import DTYPES

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", DTYPES)
@pytest.mark.parametrize("T", [1, 60, 200])
@pytest.mark.parametrize("step,low", [(9000, 0), (8200, -30), (65000, 65504), (7000, 60000), (9000, -65504), (4094, 0)])
def test_keys_of_fp16s_largest_sizes(gpu, t, T, step, low):
    """Some keys' middles, low + 8 step, pass fp16's range: they are values like others, to the bits of fp32."""
    kk = gpu
    r = rng(abs(step + low) + T)
    dim, block, n = 64, 16, 300
    table, pages = pool(r, 1, -(-n // block))
    parts = filled(r, pages, 2, dim, block)
    far = r.random(parts[1].shape[:3]) < 0.2
    parts[1][far] = step, low
    q = r.normal(size=(1, T, 4, dim)).astype(t)
    scale = 1e-6
    out = run(kk, q, parts, table, np.array([n], np.int32), scale=scale)
    check(out[0], q[0], parts, table[0], n, scale)


@pytest.mark.parametrize("t", DTYPES)
@pytest.mark.parametrize("T,group", [(1, 2), (5, 2), (40, 1), (300, 2)])
@pytest.mark.parametrize("scale", [1e-3, 1e-6, 1e-10, 1e-30, -1e-10])
def test_queries_of_nothing_under_a_small_scale(gpu, t, T, group, scale):
    """A query of zeros, or of fp32's smallest values, weighs what it sees alike, whatever the scale is."""
    kk = gpu
    r = rng(T)
    dim, block, n = 64, 32, 437
    table, pages = pool(r, 1, -(-n // block))
    parts = filled(r, pages, 2, dim, block)
    q = r.normal(size=(1, T, 2 * group, dim)).astype(t)
    q[:, ::2, 0] = 0
    q[:, -1] = 0
    if t == np.float32:
        q[:, T // 2, 1] = 1e-44
    for window in (0, 130):
        out = run(kk, q, parts, table, np.array([n], np.int32), scale=scale, window=window)
        some = np.unique(np.concatenate([[0, T - 1, T // 2], r.integers(0, T, 12)]))
        check(out[0], q[0], parts, table[0], n, scale, window, queries=some)


@pytest.mark.parametrize("t", DTYPES)
def test_a_batch_past_a_blocks_threads(gpu, t):
    """600 sequences, some of several parts, where a thread of the block goes through three of them."""
    kk = gpu
    r = rng(600)
    B, block, dim, longest = 600, 64, 64, 6000
    lengths = np.where(r.random(B) < 0.1, 0, r.integers(1, 90, B)).astype(np.int32)
    far = [0, 1, 2, 5, 191, 192, 383, 384, 597, 599]
    lengths[far] = longest - np.arange(len(far)) * 401
    # pages are shared: what a sequence reads is checked, not who owns it
    pages = 200
    table = r.integers(0, pages, (B, -(-longest // block))).astype(np.int32)
    parts = filled(r, pages, 1, dim, block)
    q = r.normal(size=(B, 1, 3, dim)).astype(t)
    out = run(kk, q, parts, table, lengths, scale=0.2)
    assert not out[lengths == 0].any()
    for b in sorted({*far, *r.integers(0, B, 20).tolist()}):
        if lengths[b]:
            check(out[b], q[b], parts, table[b], int(lengths[b]), 0.2, what=f"sequence {b}")


@pytest.mark.parametrize("T", [1, 20, 60, 200])
@pytest.mark.parametrize("step,low", [(9000, 0), (65000, 65504), (65504, -65504), (2.0 ** -24, 60000), (0, -65504)])
def test_values_of_fp16s_largest_sizes(gpu, T, step, low):
    kk = gpu
    r = rng(T)
    dim, block, n = 96, 32, 333
    table, pages = pool(r, 1, -(-n // block))
    parts = filled(r, pages, 2, dim, block)
    parts[3][r.random(parts[3].shape[:3]) < 0.2] = step, low
    q = r.normal(size=(1, T, 4, dim)).astype(np.float32)
    out = run(kk, q, parts, table, np.array([n], np.int32), scale=0.1)
    check(out[0], q[0], parts, table[0], n, 0.1)
