"""The serving decoder's norms at the ends of their types."""
import numpy as np
import pytest

from conftest import assert_bitexact, rng
from test_parity_serve import DTYPES

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
