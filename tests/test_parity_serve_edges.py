"""The serving decoder's norms at the ends of their types, its pages in a program's
own buffers, its draws under masks that are numbers."""
import numpy as np
import pytest

from conftest import assert_bitexact, rng
from oracle import serve_ops as S
from test_parity_serve import DTYPES, check_sample

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tw", DTYPES)
@pytest.mark.parametrize("rows,N", [(3, 60), (4, 300), (2, 1500), (3, 4000), (2, 16384)])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_rms_norm_quant_of_weights_that_are_not_finite(gpu, rows, N, tw, bad):
    """A row whose norm is not finite says so by its scale, whichever side that comes from."""
    kk = gpu
    r = rng(N)
    x = r.normal(size=(rows, N)).astype(np.float32)
    w = (1 + 0.2 * r.normal(size=N)).astype(tw)
    w[N * 2 // 3] = bad
    codes, scales = (kk.to_host(t) for t in kk.ops.rms_norm_quant(kk.to_device(x), kk.to_device(w)))
    assert np.isnan(scales).all() and not codes.any()


@pytest.mark.parametrize("N", [60, 300, 4000, 9000])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_rms_norm_quant_of_infinite_values_under_weights_of_0(gpu, N, bad):
    kk = gpu
    r = rng(N + 1)
    x, w = r.normal(size=(4, N)).astype(np.float32), np.ones(N, np.float32)
    w[N // 2] = 0
    c0, s0 = (kk.to_host(t) for t in kk.ops.rms_norm_quant(kk.to_device(x), kk.to_device(w)))
    x[2, N // 2] = bad
    codes, scales = (kk.to_host(t) for t in kk.ops.rms_norm_quant(kk.to_device(x), kk.to_device(w)))
    rest = [0, 1, 3]
    assert np.isnan(scales[2]).all() and not codes[2].any()
    assert np.array_equal(codes[rest], c0[rest])
    assert_bitexact(scales[rest], s0[rest])


@pytest.mark.parametrize("t", DTYPES)
@pytest.mark.parametrize("N", [60, 300, 4000, 16384])
def test_rms_norm_quant_of_a_row_of_zeros_without_eps(gpu, t, N):
    kk = gpu
    r = rng(N + 2)
    x = r.normal(size=(3, N)).astype(t)
    x[1] = 0
    codes, scales = (kk.to_host(v) for v in kk.ops.rms_norm_quant(kk.to_device(x), eps=0.0))
    assert scales[1] == 0 and not codes[1].any()
    assert (scales[[0, 2]] > 0).all() and (np.abs(codes[[0, 2]]).max(-1) == 127).all()


def test_plan_pages_between_the_starts_of_a_wider_buffer(gpu):
    """Outputs that lie between the strided starts and counts share no memory with them."""
    kk = gpu
    r = rng(9)
    B, T, block, columns = 5, 7, 16, 6
    starts, counts = r.integers(0, 60, B).astype(np.int32), r.integers(0, T + 1, B).astype(np.int32)
    host = np.full((B, 20), -9, np.int32)
    host[:, 3], host[:, 18] = starts, counts
    wide = kk.to_device(host.reshape(-1))
    table = r.permutation(B * columns).reshape(B, columns).astype(np.int32)
    free = r.permutation(40).astype(np.int32)
    of = dict(starts=wide.slice_axis(0, 3, B * 20, 20), counts=wide.slice_axis(0, 18, B * 20, 20),
              lengths=wide.slice_axis(0, 4, 4 + B), granted=wide.slice_axis(0, 24, 24 + B))
    t, slots, positions = kk.to_device(table), kk.DeviceTensor.empty((B, T), np.int64), kk.DeviceTensor.empty((B, T), np.int32)
    used = kk.to_device(np.array([2], np.int32))
    kk._lib.call("kk_plan_pages", t.desc(), slots.desc(), positions.desc(), of["lengths"].desc(), of["granted"].desc(),
                 used.desc(), of["starts"].desc(), of["counts"].desc(), kk.to_device(free).desc(), used.desc(), block)
    want = S.plan(table, starts, counts, free, 2, T, block)
    for g, w in zip((slots, positions, of["lengths"], of["granted"], used, t), want):
        assert np.array_equal(kk.to_host(g).reshape(np.shape(w)), w)
    assert np.array_equal(kk.to_host(of["starts"]), starts) and np.array_equal(kk.to_host(of["counts"]), counts)


@pytest.mark.parametrize("t", DTYPES)
@pytest.mark.parametrize("V", [3000, 50257, 131072])
@pytest.mark.parametrize("spread", [0.05, 0.5, 2.0])
def test_sample_under_a_finite_mask(gpu, t, V, spread):
    """Some logits of the type's lowest value, or of -1e4, as masks put them: the others then lie in few bins, of more
    tokens than are put in order."""
    r = rng(V)
    f = np.float32
    for low in (np.finfo(t).min, -1e4):
        x = (spread * r.normal(size=(5, V))).astype(t)
        x[r.random((5, V)) < 0.1] = low
        u = r.random(5).astype(f)
        for limits in (dict(), dict(top_p=np.array([0.9], f)), dict(top_k=np.array([V // 3], np.int32)),
                       dict(min_p=np.array([0.2], f), temperature=np.array([0.6], f)),
                       dict(top_k=np.array([V // 2], np.int64), top_p=np.array([0.7], f), min_p=np.array([0.05], f),
                            temperature=np.array([1.3], f))):
            check_sample(gpu, x, u, **limits)
