"""What a token decoder's program keeps: the paged cache of 8-bit keys and
values, the table of its rotation, a grammar's mask as bits."""
import math

import numpy as np

from . import ops

BLOCKS = (16, 32, 64, 128, 256)


class KVCache:
    """Keys and values of one layer in 8 bits, in pages of `block` tokens with
    a scale for each page and head (include/kk.h, kk_cache_append); which
    pages a sequence has, and how many of its tokens are cached, is the
    program's to keep."""

    __slots__ = ("k", "k_scale", "v", "v_scale")

    def __init__(self, k, k_scale, v, v_scale):
        pages, heads, block, dim = k.shape
        if block not in BLOCKS:
            raise ValueError(f"pages of {block} tokens (one of {BLOCKS})")
        if dim % 16 or not 16 <= dim <= 256:
            raise ValueError(f"heads of {dim} values (16 to 256 in steps of 16)")
        if v.shape != (pages, heads, dim, block):
            raise ValueError(f"values {v.shape} do not fit keys {k.shape}")
        if k_scale.shape != (pages, heads) or v_scale.shape != (pages, heads):
            raise ValueError(f"scales {k_scale.shape}, {v_scale.shape} do not fit keys {k.shape}")
        if k.dtype != np.int8 or v.dtype != np.int8 or k_scale.dtype != np.float32 or v_scale.dtype != np.float32:
            raise TypeError("codes are int8, scales float32")
        self.k, self.k_scale, self.v, self.v_scale = k, k_scale, v, v_scale

    @classmethod
    def zeros(cls, pages, heads, dim, block=64):
        """An empty cache."""
        pages, heads, dim, block = int(pages), int(heads), int(dim), int(block)
        return cls(ops.fill((pages, heads, block, dim), 0, np.int8), ops.fill((pages, heads), 0),
                   ops.fill((pages, heads, dim, block), 0, np.int8), ops.fill((pages, heads), 0))

    def values(self):
        """What the codes stand for, as float32: keys [pages, heads, block, D]
        and values [pages, heads, D, block]."""
        return ops.cache_values(self)


def rotary_turns(dim, base=10000.0, factor=1.0, old_length=None, low=1.0, high=4.0):
    """The rotation's table (int64 [dim / 2], host) for kk_qk_norm_rotary:
    pair i turns base^(-2 i / dim) a position, as 2^64ths of a turn.

    For contexts longer than the model was trained on: `factor` divides the
    positions.  With `old_length`, the length it was trained on, only slow
    pairs are divided: those of fewer than `low` turns over that length wholly,
    those of more than `high` not at all, those between in proportion."""
    dim = int(dim)
    if dim < 0 or dim % 2:
        raise ValueError(f"an even number of values turns, not {dim}")
    if not base > 0 or not factor >= 1:
        raise ValueError("base must be above 0 and factor 1 or more")
    if old_length is not None and not 0 < low < high:
        raise ValueError("low and high must be above 0 and in order")
    out = []
    for i in range(dim // 2):
        turn = float(base) ** (-2.0 * i / dim) / (2 * math.pi)
        if old_length is None:
            turn /= factor
        else:
            keep = min(1.0, max(0.0, (old_length * turn - low) / (high - low)))
            turn *= keep + (1.0 - keep) / factor
        out.append(int(turn * 2.0 ** 64) % (1 << 64))
    return np.array(out, np.uint64).astype(np.int64)


def allowed_bits(allowed):
    """bool [.., V] (tokens a grammar allows, host) as the int32 words
    [.., ceil(V / 32)] of kk_process_logits."""
    allowed = np.asarray(allowed, bool)
    pad = -allowed.shape[-1] % 32
    bits = np.packbits(np.pad(allowed, [(0, 0)] * (allowed.ndim - 1) + [(0, pad)]), axis=-1, bitorder="little")
    return np.ascontiguousarray(bits).view("<i4")
