"""The token decoder's operators without a GPU: what they refuse (each check
precedes all GPU work), the rules that name a cache's rows, the host tables."""
import os
import shutil
import subprocess

import numpy as np
import pytest

from conftest import ROOT, load_pkg

F32, F16, I8, I32, I64 = np.float32, np.float16, np.int8, np.int32, np.int64


class _Memory:
    ptr, nbytes = 1 << 20, 1 << 30


def T(shape, dtype=F32, strides=None, offset=0):
    return load_pkg().DeviceTensor(_Memory(), shape, dtype, strides, offset)


def refused(name, args, code, match):
    kk = load_pkg()
    with pytest.raises(kk._lib.KKError, match=match) as e:
        kk._lib.call(name, *[a.desc() if isinstance(a, kk.DeviceTensor) else a for a in args])
    assert e.value.code == code


def rotary_args(**over):
    a = dict(out_q=T((2, 5, 4, 64)), out_k=T((2, 5, 2, 64)), q=T((2, 5, 4, 64)), k=T((2, 5, 2, 64)), wq=T((64,)),
             wk=T((64,)), pos=T((2, 5), I32), turns=T((32,), I64), eps=1e-6, inter=0, amp=1.0)
    a.update(over)
    return list(a.values())


ARG, UNSUPPORTED = -1, -5


@pytest.mark.parametrize("over,code,match", [
    (dict(q=T((2, 5, 4, 64), I32)), ARG, "q must be f32 or f16"),
    (dict(q=T((5, 4, 64))), ARG, "q must be"),
    (dict(q=T((2, 5, 4, 300))), UNSUPPORTED, "heads of 300"),
    (dict(q=T((2, 5, 4, 64), F32, (1280, 256, 1, 4))), ARG, "next to each other"),
    (dict(out_q=T((2, 5, 4, 64), F16)), ARG, "dtype"),
    (dict(out_q=T((2, 5, 3, 64))), ARG, "shape"),
    (dict(out_q=T((2, 5, 4, 64), F32, (0, 256, 64, 1))), ARG, "broadcast"),
    (dict(out_q=None), ARG, "NULL"),
    (dict(k=None), ARG, "without k"),
    (dict(k=T((2, 4, 2, 64))), ARG, "k must have"),
    (dict(k=T((2, 5, 2, 64), F16)), ARG, "dtype"),
    (dict(wq=T((32,))), ARG, "q_weight"),
    (dict(wk=T((64,), I32)), ARG, "k_weight"),
    (dict(turns=T((33,), I64)), ARG, "do not fit"),
    (dict(turns=T((32,), I32)), ARG, "turns must"),
    (dict(pos=None), ARG, "NULL"),
    (dict(pos=T((2, 5))), ARG, "positions must be int"),
    (dict(pos=T((2, 6), I32)), ARG, "positions must be \\["),
    (dict(eps=-1.0), ARG, "eps"),
    (dict(eps=float("nan")), ARG, "eps")])
def test_qk_norm_rotary_refuses(over, code, match):
    refused("kk_qk_norm_rotary", rotary_args(**over), code, match)


def cache_args(**over):
    a = dict(k=T((7, 2, 32, 64), I8), ks=T((7, 2)), v=T((7, 2, 64, 32), I8), vs=T((7, 2)))
    a.update({n: x for n, x in over.items() if n in a})
    return list(a.values())


BAD_CACHES = [
    (dict(k=T((7, 2, 32, 64), np.uint8)), ARG, "k_codes must be int8"),
    (dict(k=T((7, 2, 32, 64), I8, (8192, 4096, 128, 1))), ARG, "k_codes must be int8"),
    (dict(k=T((7, 2, 32, 64), I8, None, 8)), ARG, "16-byte aligned"),
    (dict(v=T((7, 2, 32, 64), I8)), ARG, "v_codes must be"),
    (dict(ks=T((7, 3))), ARG, "k_scales must be"),
    (dict(vs=T((7, 2), F16)), ARG, "v_scales must be"),
    (dict(k=T((7, 2, 48, 64), I8), v=T((7, 2, 64, 48), I8)), UNSUPPORTED, "pages of 48"),
    (dict(k=T((7, 2, 32, 40), I8), v=T((7, 2, 40, 32), I8)), UNSUPPORTED, "heads of 40"),
    (dict(k=None), ARG, "NULL")]


def append_args(**over):
    a = dict(nk=T((3, 4, 2, 64)), nv=T((3, 4, 2, 64)), table=T((3, 5), I32), starts=T((3,), I32), counts=T((3,), I64))
    a.update({n: x for n, x in over.items() if n in a})
    return cache_args(**over) + list(a.values())


@pytest.mark.parametrize("over,code,match", BAD_CACHES + [
    (dict(nk=T((3, 4, 2, 64), F16)), ARG, "one dtype"),
    (dict(nv=T((3, 5, 2, 64))), ARG, "one shape"),
    (dict(nk=T((3, 4, 3, 64)), nv=T((3, 4, 3, 64))), ARG, "holds 2 heads"),
    (dict(table=T((2, 5), I32)), ARG, "a row a sequence"),
    (dict(table=T((3, 5), I64)), ARG, "table must be int32"),
    (dict(table=T((3, 5), I32, (10, 2))), ARG, "one piece"),
    (dict(starts=T((2,), I32)), ARG, "starts must"),
    (dict(starts=T((3,))), ARG, "starts must be int"),
    (dict(counts=T((3, 1), I32)), ARG, "counts must"),
    (dict(starts=None), ARG, "NULL")])
def test_cache_append_refuses(over, code, match):
    refused("kk_cache_append", append_args(**over), code, match)


def attention_args(**over):
    a = dict(table=T((3, 5), I32), lengths=T((3,), I32), counts=None, scale=0.125, window=0)
    a.update({n: x for n, x in over.items() if n in a})
    head = [over.get("out", T((3, 4, 6, 64))), over.get("q", T((3, 4, 6, 64)))]
    return head + cache_args(**over) + list(a.values())


@pytest.mark.parametrize("over,code,match", BAD_CACHES + [
    (dict(q=T((3, 4, 5, 64)), out=T((3, 4, 5, 64))), ARG, "not a multiple"),
    (dict(q=T((3, 4, 6, 32)), out=T((3, 4, 6, 32))), ARG, "over keys of"),
    (dict(q=T((2, 4, 6, 64)), out=T((2, 4, 6, 64))), ARG, "a row a sequence"),
    (dict(out=T((3, 4, 6, 64), F16)), ARG, "dtype"),
    (dict(out=T((3, 4, 6, 64), F32, (0, 384, 64, 1))), ARG, "broadcast"),
    (dict(lengths=T((4,), I32)), ARG, "lengths must"),
    (dict(counts=T((3,))), ARG, "counts must be int"),
    (dict(window=-1), ARG, "window"),
    (dict(scale=float("inf")), ARG, "finite")])
def test_cache_attention_refuses(over, code, match):
    refused("kk_cache_attention", attention_args(**over), code, match)


def cross_args(**over):
    a = dict(out=T((2, 3, 4, 64)), q=T((2, 3, 4, 64)), k=T((2, 9, 2, 64)), v=T((2, 9, 2, 64)), lengths=T((2,), I32),
             mask=T((2, 3, 9), np.bool_), scale=0.125)
    a.update(over)
    return list(a.values())


@pytest.mark.parametrize("over,code,match", [
    (dict(k=T((2, 9, 3, 64)), v=T((2, 9, 3, 64))), ARG, "not a multiple"),
    (dict(k=T((2, 9, 0, 64)), v=T((2, 9, 0, 64))), ARG, "not a multiple"),
    (dict(v=T((2, 8, 2, 64))), ARG, "one shape"),
    (dict(v=T((2, 9, 2, 64), F16)), ARG, "one dtype"),
    (dict(k=T((1, 9, 2, 64)), v=T((1, 9, 2, 64))), ARG, "sequences"),
    (dict(q=T((2, 3, 4, 260)), out=T((2, 3, 4, 260)), k=T((2, 9, 2, 260)), v=T((2, 9, 2, 260))), UNSUPPORTED,
     "heads of 260"),
    (dict(lengths=T((2,))), ARG, "lengths must be int"),
    (dict(mask=T((2, 3, 8), np.bool_)), ARG, "mask must"),
    (dict(mask=T((2, 3, 9))), ARG, "mask must"),
    (dict(mask=T((9,), np.bool_)), ARG, "mask must"),
    (dict(scale=float("nan")), ARG, "finite"),
    (dict(q=None), ARG, "NULL")])
def test_cross_attention_refuses(over, code, match):
    refused("kk_cross_attention", cross_args(**over), code, match)


def logits_args(**over):
    a = dict(out=T((2, 70)), x=T((2, 70), F16), history=T((2, 9), I32), lengths=T((2,), I32), rep=T((2,)),
             pres=T((1,)), freq=None, bias=T((70,)), allowed=T((1, 3), I32))
    a.update(over)
    return list(a.values())


@pytest.mark.parametrize("over,code,match", [
    (dict(x=T((2, 70), I32)), ARG, "logits must"),
    (dict(out=T((2, 70), F16)), ARG, "out must"),
    (dict(out=T((2, 70), F32, (0, 1))), ARG, "broadcast"),
    (dict(x=T((2, 70), F32, (1, 2))), ARG, "one piece"),
    (dict(history=None), ARG, "need the history"),
    (dict(history=T((2, 9))), ARG, "history must"),
    (dict(lengths=T((3,), I32)), ARG, "history_lengths must"),
    (dict(rep=T((3,))), ARG, "repetition must"),
    (dict(pres=T((2,), F16)), ARG, "presence must"),
    (dict(bias=T((69,))), ARG, "bias must"),
    (dict(allowed=T((2, 2), I32)), ARG, "allowed must"),
    (dict(allowed=T((2, 3), I64)), ARG, "allowed must")])
def test_process_logits_refuses(over, code, match):
    refused("kk_process_logits", logits_args(**over), code, match)


def test_a_sound_call_gets_as_far_as_the_device():
    kk = load_pkg()
    if kk.tensor._state["device"] is not None:
        pytest.skip("library already initialised in this process")
    for name, args in [("kk_qk_norm_rotary", rotary_args()), ("kk_cache_append", append_args()),
                       ("kk_cache_attention", attention_args()), ("kk_cross_attention", cross_args()),
                       ("kk_process_logits", logits_args())]:
        refused(name, args, -4, "kk_init")


def test_cache_rows_stay_in_range(tmp_path):
    cc = shutil.which("g++")
    if not cc:
        pytest.skip("no C++ compiler")
    exe = str(tmp_path / "check")
    subprocess.run([cc, "-O2", "-std=c++17", "-I", os.path.join(ROOT, "best-tts-godot_amd", "csrc"),
                    os.path.join(ROOT, "tests", "cache_index_check.cpp"), "-o", exe], check=True)
    out = subprocess.run([exe], capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout == "ok\n", out.stdout


def test_kv_cache_checks_its_parts():
    kk = load_pkg()
    kk.KVCache(*cache_args())
    for over, _, _ in BAD_CACHES:
        if set(over) == {"k"} and over["k"] is not None and over["k"].dtype == I8:
            continue  # (strides and alignment are the library's to check)
        with pytest.raises((ValueError, TypeError, AttributeError)):
            kk.KVCache(*cache_args(**over))


def test_rotary_turns():
    kk = load_pkg()
    t = kk.rotary_turns(64).astype(np.float64) / 2.0 ** 64 * 2 * np.pi
    assert np.allclose(t, 10000.0 ** (-np.arange(32) / 32.0), rtol=1e-12)
    assert np.allclose(kk.rotary_turns(64, factor=4.0) * 4.0, kk.rotary_turns(64), rtol=1e-9)
    whole, some = kk.rotary_turns(64), kk.rotary_turns(64, factor=8.0, old_length=4096, low=1.0, high=4.0)
    turns = whole / 2.0 ** 64 * 4096
    assert np.array_equal(some[turns > 4], whole[turns > 4]) and (turns > 4).any() and (turns < 1).any()
    assert np.allclose(some[turns < 1] * 8.0, whole[turns < 1], rtol=1e-6)
    between = (turns > 1) & (turns < 4)
    assert between.any() and np.all(some[between] < whole[between]) and np.all(some[between] * 8.0 > whole[between])
    assert kk.rotary_turns(0).shape == (0,)
    for bad in (dict(dim=3), dict(dim=4, base=0), dict(dim=4, factor=0.5), dict(dim=4, old_length=9, low=2, high=1)):
        with pytest.raises(ValueError):
            kk.rotary_turns(**bad)


def test_allowed_bits():
    kk = load_pkg()
    a = np.random.default_rng(0).random((3, 70)) < 0.5
    words = kk.allowed_bits(a)
    assert words.shape == (3, 3) and words.dtype == np.int32
    for v in range(70):
        assert np.array_equal((words[:, v >> 5] >> (v & 31)) & 1, a[:, v])
