"""The token decoder's oracle against what does not retype it: rotations as
complex powers and their invariants, torch's attention in float64, closed
forms of the cache's rounding, counting by hand."""
import numpy as np
import torch

from conftest import load_pkg, rng
from oracle import decode_ops as D


def test_rotation_keeps_lengths_and_differences():
    """Norms are kept, and products depend on the difference of positions alone."""
    kk = load_pkg()
    r = rng(1)
    turns = kk.rotary_turns(16).tolist()
    x, y = r.normal(size=(1, 1, 1, 16)), r.normal(size=(1, 1, 1, 16))
    for inter in (False, True):
        def at(z, p):
            return D.rotated(z, None, [[p]], turns, interleaved=inter)[0, 0, 0]
        assert np.allclose(np.linalg.norm(at(x, 12345)), np.linalg.norm(x))
        assert np.allclose(at(x, 7) @ at(y, 5), at(x, 1000007) @ at(y, 1000005))
        assert np.allclose(at(x, 0), x[0, 0, 0])
        z = x[0, 0, 0].reshape(8, 2) if inter else x[0, 0, 0].reshape(2, 8).T
        w = (z[:, 0] + 1j * z[:, 1]) * np.exp(1j * 9 * 10000.0 ** (-np.arange(8) / 8))
        got = at(x, 9).reshape(8, 2) if inter else at(x, 9).reshape(2, 8).T
        assert np.allclose(got[:, 0] + 1j * got[:, 1], w)


def test_norm_is_torchs():
    r = rng(2)
    x, w = r.normal(size=(2, 3, 4, 10)), r.normal(size=10)
    want = torch.nn.functional.rms_norm(torch.from_numpy(x), (10,), torch.from_numpy(w), eps=1e-6).numpy()
    assert np.allclose(D.rotated(x, w, np.zeros((2, 3)), []), want)


def test_attention_is_torchs():
    r = rng(3)
    q, k, v = r.normal(size=(5, 6, 8)), r.normal(size=(9, 2, 8)), r.normal(size=(9, 2, 8))
    got = D.attention(q, k, v, lambda t: np.arange(5 + t), 0.3)
    mask = torch.arange(9) < 5 + torch.arange(5)[:, None]
    want = torch.nn.functional.scaled_dot_product_attention(
        *(torch.from_numpy(np.repeat(x, n, 1)).transpose(0, 1) for x, n in ((q, 1), (k, 3), (v, 3))), attn_mask=mask,
        scale=0.3).transpose(0, 1).numpy()
    assert np.allclose(got, want)
    assert not D.attention(q, k, v, lambda t: [], 0.3).any()


def test_append_rounds_within_half_a_step_and_keeps_scales():
    r = rng(4)
    codes, scales = np.zeros((4, 1, 16, 16), np.int8), np.zeros((4, 1), np.float32)
    table = np.array([[2, 0]])
    x = r.normal(size=(1, 20, 1, 16)).astype(np.float32)
    c1, s1 = D.append(codes, scales, x, table, [0], [20])
    rows, there = D.cached(c1, s1, table[0], 20)
    assert there.all()
    step = np.repeat(np.array([s1[2, 0], s1[0, 0]]), [16, 4])[:, None, None]
    assert np.all(np.abs(rows - x[0]) <= 0.5000001 * step)
    assert np.abs(c1[2]).max() == 127 and np.abs(c1[0]).max() == 127 and not c1[[1, 3]].any()
    # a larger row raises the scale of its page alone, a smaller one leaves all
    c2, s2 = D.append(c1, s1, 10 * x[:, :1], table, [20], [1])
    assert s2[0, 0] > s1[0, 0] and s2[2, 0] == s1[2, 0] and np.array_equal(c2[2], c1[2])
    c3, s3 = D.append(c1, s1, 0.1 * x[:, :1], table, [20], [1])
    assert np.array_equal(s3, s1) and np.array_equal(c3[0, :, :4], c1[0, :, :4])


def test_logits_by_hand():
    x = np.array([[1.0, -1.0, 2.0, 0.5]])
    got = D.logits(x, [[0, 0, 1, 9, 3]], [4], [2.0], [0.25], [0.5], np.array([[0, 0, 0, 1.0]]),
                   np.array([[True, True, False, True]]))
    assert got.tolist() == [[0.5 - 1.0 - 0.25, -2.0 - 0.5 - 0.25, -np.inf, 1.5]]
