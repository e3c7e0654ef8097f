"""The serving decoder's oracle against what does not retype it: torch's norm,
closed forms of the codes' rounding, pages counted by hand, frequencies."""
import math

import numpy as np
import torch

from conftest import rng
from oracle import serve_ops as S


def test_norm_is_torchs():
    r = rng(1)
    x, res, w = r.normal(size=(5, 33)), r.normal(size=(5, 33)), r.normal(size=33)
    y, h = S.rms_norm(x, res, w, 1e-5)
    want = torch.nn.functional.rms_norm(torch.from_numpy(x + res), (33,), torch.from_numpy(w), eps=1e-5).numpy()
    assert np.allclose(y, want) and np.array_equal(h, x + res)


def test_codes_are_within_half_a_step_of_the_norm():
    r = rng(2)
    x, w = r.normal(size=(7, 50)), r.normal(size=50)
    y, _ = S.rms_norm(x, None, w, 1e-6)
    codes = S.rms_codes(x, None, w)
    scale = np.abs(y).max(-1, keepdims=True) / 127
    assert np.abs(codes * scale - y).max() <= 0.5000001 * scale.max()
    assert (np.abs(codes).max(-1) == 127).all()
    assert not S.rms_codes(np.zeros((1, 4)), None, None).any()


def test_plan_by_hand():
    table = np.full((4, 3), -1, np.int32)
    table[0, 0], table[1, :2] = 9, (7, 8)
    out = S.plan(table, [3, 32, 0, 0], [2, 3, 40, 16], np.array([1, 2, 3, 4], np.int32), 1, 40, 16)
    slots, positions, lengths, granted, used, table = out
    assert granted.tolist() == [2, 3, 0, 0] and lengths.tolist() == [5, 35, 0, 0] and used == 2
    assert slots[0, :3].tolist() == [9 * 16 + 3, 9 * 16 + 4, -1] and slots[1, :3].tolist() == [32, 33, 34] + []
    assert positions[1, :4].tolist() == [32, 33, 34, -1] and (slots[2:] == -1).all()
    # (page 2 of the list's first free place went to sequence 1; the third wanted 3 of the 2 left, and the fourth came after)
    assert table.tolist() == [[9, -1, -1], [7, 8, 2], [-1, -1, -1], [-1, -1, -1]]


def test_release_is_plans_reverse():
    table = np.array([[4, 5, -1], [6, -3, 7], [8, 9, 2]], np.int32)
    free = np.array([4, 5, 6, 7, 8, 9, 1], np.int32)
    t, f, used = S.release(table, [17, 48, 33], [1, 1, 0], free, 6, 16)
    assert used == 2 and f.tolist() == [4, 5, 4, 5, 6, 7, 1]
    assert t.tolist() == [[-1, -1, -1], [-1, -1, -1], [8, 9, 2]]


def test_append_rounds_within_half_a_step():
    r = rng(3)
    codes, scales = np.zeros((2, 1, 16, 32), np.uint8), np.zeros((2, 1, 16, 2), np.float16)
    x = r.normal(size=(3, 1, 64)).astype(np.float32)
    c, s = S.append4(codes, scales, x, [17, -1, 4])
    v = S.values4(c, s)
    for slot, row in ((17, 0), (4, 2)):
        step, low = (float(z) for z in s[slot // 16, 0, slot % 16])
        # half a step, and what the roundings of low and step to fp16 move
        assert np.abs(v[slot // 16, 0, slot % 16] - x[row, 0]).max() <= 0.5 * step + 2.0 ** -11 * (abs(low) + 15 * step)
        assert low == np.float16(x[row].min())
    assert not c[0, 0, 5].any() and not s[1, 0, 0].any()
    rows, there = S.cached4(c, s, np.array([1, 5]), 20)
    assert there.tolist() == [True] * 16 + [False] * 4 and np.array_equal(rows[1], v[1, :, 1])


def test_sampling_has_the_softmaxs_frequencies():
    x = np.array([0.0, 2.0, -1.0, 2.0, -np.inf])
    p = np.exp((x - 2) / 0.7)
    p /= p.sum()
    got = np.bincount([S.sample(x, (i + 0.5) / 1000, 0.7)[0] for i in range(1000)], minlength=5) / 1000
    assert np.abs(got - p).max() < 1.5e-3 and got[4] == 0
    assert abs(S.sample(x, 0.0, 0.7)[1] - math.log(p[1])) < 1e-12
    assert [S.sample(x, u, top_k=1)[0] for u in (0.0, 0.99)] == [1, 1]
    assert {S.sample(x, u / 50, top_k=2)[0] for u in range(50)} == {1, 3}
    # 1, 1, e^-2, e^-3 of 2.185 in all: 0.915 comes before the third, 0.977 before the fourth
    assert {S.sample(x, u / 400, top_p=0.9)[0] for u in range(400)} == {1, 3}
    assert {S.sample(x, u / 400, top_p=0.95)[0] for u in range(400)} == {1, 3, 0}
    assert {S.sample(x, u / 400, min_p=0.1)[0] for u in range(400)} == {1, 3, 0}
    assert {S.sample(x, u / 400, min_p=0.2)[0] for u in range(400)} == {1, 3}
    assert S.sample(x, 0.99, 0.0)[:2] == (1, 0.0)
    assert S.sample(np.full(3, -np.inf), 0.5)[:2] == (-1, -math.inf)
