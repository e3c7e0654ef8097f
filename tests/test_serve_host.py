"""The serving decoder's operators without a GPU: what they refuse (each check
precedes all GPU work)."""
import numpy as np
import pytest

from conftest import load_pkg
from test_decode_host import ARG, UNSUPPORTED, T, refused

F32, F16, I8, U8, I32, I64, BOOL = np.float32, np.float16, np.int8, np.uint8, np.int32, np.int64, np.bool_


def norm_args(quant=False, **over):
    a = dict(out=T((3, 5, 64), I8 if quant else F32))
    if quant:
        a["scales"] = T((3, 5, 1))
    a.update(sum=T((3, 5, 64)), x=T((3, 5, 64)), residual=T((3, 5, 64)), weight=T((64,)), eps=1e-6)
    a.update(over)
    return list(a.values())


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("over,code,match", [
    (dict(x=None), ARG, "NULL"),
    (dict(x=T(())), ARG, "axis"),
    (dict(x=T((3, 5, 64), I32)), ARG, "x must be f32 or f16"),
    (dict(x=T((3, 5, 64), F32, (640, 128, 2))), ARG, "next to each other"),
    (dict(x=T((3, 5, 64), F32, (1000, 64, 1))), ARG, "evenly spaced"),
    (dict(out=T((3, 5, 64), U8)), ARG, "out must be"),
    (dict(out=T((3, 5, 63))), ARG, "shape"),
    (dict(residual=T((15, 64))), ARG, "shape"),
    (dict(residual=T((3, 5, 64), I8)), ARG, "residual must be f32 or f16"),
    (dict(residual=None), ARG, "sum without residual"),
    (dict(sum=T((3, 5, 64), F16)), ARG, "residual's dtype"),
    (dict(sum=T((3, 5, 64), F32, (0, 0, 1))), ARG, "broadcast"),
    (dict(weight=T((63,))), ARG, "weight"),
    (dict(weight=T((64,), I8)), ARG, "weight"),
    (dict(weight=T((64,), F32, (2,))), ARG, "weight"),
    (dict(eps=-1e-6), ARG, "eps"),
    (dict(eps=float("nan")), ARG, "eps"),
    (dict(), ARG, "must not be the same")])
def test_rms_norm_refuses(quant, over, code, match):
    refused("kk_rms_norm_quant" if quant else "kk_rms_norm", norm_args(quant, **over), code, match)


def test_rms_norm_refuses_sizes_and_scales():
    wide = dict(out=T((2, 16385)), sum=None, x=T((2, 16385)), residual=None, weight=None)
    refused("kk_rms_norm", norm_args(**wide), UNSUPPORTED, "16385")
    empty = dict(out=T((2, 0)), sum=None, x=T((2, 0)), residual=None, weight=None)
    refused("kk_rms_norm", norm_args(**empty), UNSUPPORTED, "of 0")
    refused("kk_rms_norm_quant", norm_args(True, scales=None), ARG, "scales")
    refused("kk_rms_norm_quant", norm_args(True, scales=T((3, 5, 1), F16)), ARG, "scales")
    refused("kk_rms_norm_quant", norm_args(True, scales=T((3, 4))), ARG, "scales")
    refused("kk_rms_norm_quant", norm_args(True, out=T((3, 5, 64))), ARG, "out must be int8")


def plan_args(**over):
    a = dict(table=T((4, 9), I32), slots=T((4, 7), I64), positions=T((4, 7), I32, None, 64), lengths=T((4,), I32, None, 1000),
             granted=T((4,), I32, None, 2000), used_out=T((1,), I32), starts=T((4,), I32, None, 3000),
             counts=T((4,), I64, None, 4000), free=T((30,), I32), used=T((1,), I32), block=32)
    a.update(over)
    return list(a.values())


@pytest.mark.parametrize("over,code,match", [
    (dict(table=None), ARG, "NULL"),
    (dict(table=T((4, 9), I64)), ARG, "table must be int32"),
    (dict(table=T((4, 9), I32, (1, 4))), ARG, "row of table"),
    (dict(table=T((4, 9), I32, (0, 1))), ARG, "broadcast"),
    (dict(table=T((4, 2 ** 27), I32)), UNSUPPORTED, "columns"),
    (dict(block=48), UNSUPPORTED, "pages of 48"),
    (dict(slots=T((4, 7), I32)), ARG, "slots must be int64"),
    (dict(slots=T((3, 7), I64)), ARG, "slots must be"),
    (dict(slots=T((4, 7), I64, (1, 4))), ARG, "rows in one piece"),
    (dict(positions=T((4, 6), I32)), ARG, "positions must be"),
    (dict(positions=T((4, 7), I64)), ARG, "positions must be int32"),
    (dict(lengths=T((4,), I64)), ARG, "lengths must be int32"),
    (dict(granted=T((3,), I32)), ARG, "granted must be"),
    (dict(granted=T((4,), I32, None, 3000)), ARG, "must not be starts"),
    (dict(lengths=T((4,), I32, None, 3000)), ARG, "must not be starts"),
    (dict(starts=T((4,))), ARG, "starts must be int"),
    (dict(starts=T((3,), I32)), ARG, "starts must have"),
    (dict(counts=T((4,))), ARG, "counts must be int"),
    (dict(free=T((30,), I64)), ARG, "free must be int32"),
    (dict(used=T((2,), I32)), ARG, "used must be"),
    (dict(used_out=T((), I32)), ARG, "used_out must be")])
def test_plan_pages_refuses(over, code, match):
    refused("kk_plan_pages", plan_args(**over), code, match)


@pytest.mark.parametrize("over,code,match", [
    (dict(table=T((4, 9))), ARG, "table must be int32"),
    (dict(lengths=T((3,), I32)), ARG, "lengths must"),
    (dict(ended=T((4,), I32)), ARG, "ended must be bool"),
    (dict(ended=T((1,), BOOL)), ARG, "ended must be bool"),
    (dict(free=None), ARG, "NULL"),
    (dict(used=T((1,), I64)), ARG, "used must be int32"),
    (dict(block=0), UNSUPPORTED, "pages of 0")])
def test_release_pages_refuses(over, code, match):
    a = dict(table=T((4, 9), I32), lengths=T((4,), I64), ended=T((4,), BOOL), free=T((30,), I32), used=T((1,), I32), block=16)
    refused("kk_release_pages", list(dict(a, **over).values()), code, match)


def cache4_args(**over):
    a = dict(k=T((7, 2, 32, 32), U8), ks=T((7, 2, 32, 2), F16), v=T((7, 2, 32, 32), U8), vs=T((7, 2, 32, 2), F16))
    a.update({n: x for n, x in over.items() if n in a})
    return list(a.values())


BAD_CACHES4 = [
    (dict(k=T((7, 2, 32, 32), I8)), ARG, "k_codes must be uint8"),
    (dict(k=T((7, 2, 32, 32), U8, (4096, 2048, 64, 1))), ARG, "k_codes must be uint8"),
    (dict(k=T((7, 2, 32, 32), U8, None, 8)), ARG, "16-byte aligned"),
    (dict(v=T((7, 2, 32, 64), U8)), ARG, "v_codes must be"),
    (dict(v=T((6, 2, 32, 32), U8)), ARG, "v_codes must be"),
    (dict(ks=T((7, 2, 32, 2))), ARG, "k_scales must be"),
    (dict(vs=T((7, 2, 32), F16)), ARG, "v_scales must be"),
    (dict(vs=T((7, 2, 32, 2), F16, None, 4)), ARG, "v_scales must be"),
    (dict(k=T((7, 2, 48, 32), U8), v=T((7, 2, 32, 48), U8), ks=T((7, 2, 48, 2), F16), vs=T((7, 2, 48, 2), F16)),
     UNSUPPORTED, "pages of 48"),
    (dict(k=T((7, 2, 32, 40), U8), v=T((7, 2, 40, 32), U8)), UNSUPPORTED, "heads of 80"),
    (dict(k=T((7, 2, 32, 144), U8), v=T((7, 2, 144, 32), U8)), UNSUPPORTED, "heads of 288"),
    (dict(k=None), ARG, "NULL")]


@pytest.mark.parametrize("over,code,match", BAD_CACHES4 + [
    (dict(x=T((2, 5, 2, 64), I32)), ARG, "k must be f32 or f16"),
    (dict(x=T((2, 5, 3, 64))), ARG, "one shape"),
    (dict(x=T((2, 5, 2, 64), F16)), ARG, "one dtype"),
    (dict(x=T((2, 5, 3, 64)), y=T((2, 5, 3, 64))), ARG, "do not fit"),
    (dict(x=T((2, 5, 2, 32)), y=T((2, 5, 2, 32))), ARG, "do not fit"),
    (dict(x=T((2, 5, 2, 64), F32, (1280, 256, 128, 2))), ARG, "next to each other"),
    (dict(slots=T((2, 5))), ARG, "slots must be"),
    (dict(slots=T((10,), I64)), ARG, "slots must be")])
def test_cache4_append_refuses(over, code, match):
    a = dict(x=T((2, 5, 2, 64)), y=T((2, 5, 2, 64)), slots=T((2, 5), I64))
    a.update({n: x for n, x in over.items() if n in a})
    refused("kk_cache4_append", cache4_args(**over) + list(a.values()), code, match)


@pytest.mark.parametrize("over,code,match", BAD_CACHES4 + [
    (dict(out_k=T((7, 2, 32, 64), F16)), ARG, "out_k must be f32"),
    (dict(out_k=T((7, 2, 32, 32))), ARG, "out_k must be"),
    (dict(out_v=T((7, 2, 32, 64))), ARG, "out_v must be"),
    (dict(out_v=T((7, 2, 64, 32), F32, None, 1)), ARG, "16-byte aligned")])
def test_cache4_values_refuses(over, code, match):
    a = dict(out_k=T((7, 2, 32, 64)), out_v=T((7, 2, 64, 32)))
    a.update({n: x for n, x in over.items() if n in a})
    refused("kk_cache4_values", list(a.values()) + cache4_args(**over), code, match)


@pytest.mark.parametrize("over,code,match", BAD_CACHES4 + [
    (dict(q=T((2, 5, 4, 64), I32)), ARG, "q must be f32 or f16"),
    (dict(q=T((2, 5, 3, 64)), out=T((2, 5, 3, 64))), ARG, "not a multiple"),
    (dict(q=T((2, 5, 4, 32)), out=T((2, 5, 4, 32))), ARG, "over keys of 64"),
    (dict(out=T((2, 5, 4, 64), F16)), ARG, "q's dtype"),
    (dict(out=T((2, 5, 4, 64), F32, (0, 256, 64, 1))), ARG, "broadcast"),
    (dict(table=T((2, 6), I64)), ARG, "table must be int32"),
    (dict(table=T((3, 6), I32)), ARG, "row a sequence"),
    (dict(lengths=T((2,))), ARG, "lengths must be int"),
    (dict(counts=T((3,), I32)), ARG, "counts must have"),
    (dict(scale=float("inf")), ARG, "scale must be finite"),
    (dict(window=-1), ARG, "window")])
def test_cache4_attention_refuses(over, code, match):
    a = dict(out=T((2, 5, 4, 64)), q=T((2, 5, 4, 64)))
    b = dict(table=T((2, 6), I32), lengths=T((2,), I32), counts=T((2,), I64), scale=0.1, window=0)
    for d in (a, b):
        d.update({n: x for n, x in over.items() if n in d})
    refused("kk_cache4_attention", list(a.values()) + cache4_args(**over) + list(b.values()), code, match)


@pytest.mark.parametrize("over,code,match", [
    (dict(logits=T((3, 50), I32)), ARG, "logits must be f32 or f16"),
    (dict(logits=T((3, 5, 10))), ARG, "logits must be"),
    (dict(logits=T((3, 50), F32, (100, 2))), ARG, "one piece"),
    (dict(logits=T((3, 131073))), UNSUPPORTED, "131073"),
    (dict(logits=T((3, 0))), UNSUPPORTED, "rows of 0"),
    (dict(tokens=T((3,), I64)), ARG, "tokens must be int32"),
    (dict(tokens=T((2,), I32)), ARG, "tokens must be"),
    (dict(logs=T((3,), F16)), ARG, "logs must be f32"),
    (dict(uniforms=None), ARG, "NULL"),
    (dict(uniforms=T((3,), F16)), ARG, "uniforms must be f32"),
    (dict(temperature=T((2,))), ARG, "temperature must have"),
    (dict(top_k=T((3,))), ARG, "top_k must be int"),
    (dict(top_p=T((3, 1))), ARG, "top_p must have"),
    (dict(min_p=T((3,), I32)), ARG, "min_p must be f32")])
def test_sample_refuses(over, code, match):
    a = dict(tokens=T((3,), I32), logs=T((3,)), logits=T((3, 50)), uniforms=T((3,)), temperature=T((3,)),
             top_k=T((1,), I64), top_p=T((3,)), min_p=T((3,)))
    refused("kk_sample", list(dict(a, **over).values()), code, match)


@pytest.mark.parametrize("over,error,match", [
    (dict(k=T((7, 2, 48, 32), U8)), ValueError, "pages of 48"),
    (dict(k=T((7, 2, 32, 24), U8)), ValueError, "heads of 48"),
    (dict(v=T((7, 2, 32, 16), U8)), ValueError, "do not fit"),
    (dict(ks=T((7, 2, 32), F16)), ValueError, "scales"),
    (dict(k=T((7, 2, 32, 32), I8)), TypeError, "uint8"),
    (dict(vs=T((7, 2, 32, 2))), TypeError, "float16")])
def test_a_4_bit_cache_that_does_not_fit_is_refused(over, error, match):
    k, ks, v, vs = cache4_args(**over)
    with pytest.raises(error, match=match):
        load_pkg().KVCache4(k, ks, v, vs)


def test_rows_that_are_not_evenly_spaced_are_copied():
    ops = load_pkg().ops
    even = T((3, 5, 64), F32, (10 * 64, 2 * 64, 1))
    assert ops._rows(even) is even and ops._rows(None) is None
    one = T((1, 5, 64), F32, (7, 128, 1))
    assert ops._rows(one) is one
