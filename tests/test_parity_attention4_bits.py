"""Attention over the 4-bit cache of fp16 queries, held to the bits of its output's
type: which bits a query keeps does not hang on how many others are in the call.

The bounds are those of fp32 queries in test_parity_attention4 without the split of the
query (fp16 ones are multiplied as they are): scores, powers and sums in fp32, a weight
times its value's step in two halves, which keep 2^-22 of it and 2^-32 of the largest
such product; then half a step of fp16."""
import numpy as np
import pytest

from conftest import rng
from oracle import decode_ops as D
from oracle import serve_ops as S
from test_parity_attention4 import filled, pool, run
from test_parity_decode import U, half_step, within

pytestmark = pytest.mark.gpu
F16 = np.float16


def check_bits(out, q, parts, table, n, scale, window, queries, what):
    """The queries' rows [some, Hq, D] of q [T, Hq, D], the newest of n cached tokens."""
    T, some = q.shape[0], q[queries]
    k, _ = S.cached4(parts[0], parts[1], table, n)
    v, _ = S.cached4(parts[2], parts[3], table, n, tokens_last=True)
    block, at_row = parts[0].shape[2], np.arange(n)

    def size(scales):  # 15 step + |low| of each token and head
        x = np.abs(scales.astype(np.float64)) @ np.array([15.0, 1.0])
        return x[table[at_row // block], :, at_row % block]
    ks, vs = size(parts[1]), size(parts[3])

    def seen(i):
        place = n - T + queries[i]
        return np.arange(max(0, place - window + 1) if window else 0, place + 1)
    want = D.attention(some, k, v, seen, scale)
    tol, group = np.zeros(want.shape), q.shape[1] // k.shape[1]
    for i in range(len(queries)):
        at = seen(i)
        for h in range(q.shape[1]):
            g, q64 = h // group, some[i, h].astype(np.float64)
            s = k[at, g] @ q64 * scale
            p = np.exp(s - s.max())
            p /= p.sum()
            off = 2 * (q.shape[-1] + 8) * U * abs(scale) * np.abs(q64).sum() * ks[at, g]
            share = p @ off + (at.size / 16 + 16) * U + 2.0 ** -22
            floor = at.size * 2.0 ** -32 * (p * vs[at, g]).max()
            tol[i, h] = p @ (off * vs[at, g]) + 2 * share * (p @ vs[at, g]) + floor
    within(out[queries], want, tol + half_step(F16) * np.abs(want) + 2.0 ** -25, what)


@pytest.mark.parametrize("T,Hq,Hk,dim,block,longest,window", [
    (1, 8, 1, 32, 16, 5, 0), (1, 300, 1, 32, 16, 5, 0), (1, 512, 1, 64, 64, 6, 0), (1, 520, 1, 32, 16, 5, 0),
    (1, 1100, 1, 128, 64, 4, 0), (2, 600, 2, 96, 16, 7, 0), (2, 600, 2, 96, 64, 7, 3), (30, 20, 1, 64, 32, 40, 9),
    (520, 1, 1, 32, 64, 523, 5), (40, 16, 1, 128, 128, 50, 8), (1, 600, 1, 160, 64, 5, 0)])
def test_fp16_queries_keep_their_outputs_bits(gpu, T, Hq, Hk, dim, block, longest, window):
    """Scores of small sizes from keys of one value each, values around 0: what is left of the bound is the output's
    own rounding."""
    kk = gpu
    r = rng(T + Hq)
    table, pages = pool(r, 1, -(-longest // block))
    parts = filled(r, pages, Hk, dim, block)
    parts[1][..., 0], parts[1][..., 1] = 0, r.uniform(-1, 1, parts[1].shape[:3])
    q = np.broadcast_to(r.uniform(0.1, 1, (1, T, Hq, 1)), (1, T, Hq, dim)).astype(F16)
    out = run(kk, q, parts, table, np.array([longest], np.int32), scale=1 / dim, window=window)
    some = np.arange(T) if T < 40 else np.unique(r.integers(0, T, 40))
    check_bits(out[0], q[0], parts, table[0], longest, 1 / dim, window, some, "outputs")
