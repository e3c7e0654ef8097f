"""The cut of long sequences over blocks, and the cache's values, without a GPU."""
import os
import shutil
import subprocess

import pytest

from conftest import ROOT
from test_decode_host import ARG, BAD_CACHES, F16, T, attention_args, cache_args, refused


def test_chunks_fit_their_grid(tmp_path):
    cc = shutil.which("g++")
    if not cc:
        pytest.skip("no C++ compiler")
    exe = str(tmp_path / "check")
    subprocess.run([cc, "-O2", "-std=c++17", "-I", os.path.join(ROOT, "best-tts-godot_amd", "csrc"),
                    os.path.join(ROOT, "tests", "chunk_check.cpp"), "-o", exe], check=True)
    out = subprocess.run([exe], capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout == "ok\n", out.stdout


def values_args(**over):
    parts = dict(zip(("k", "ks", "v", "vs"), cache_args(**{n: x for n, x in over.items() if n in ("k", "ks", "v", "vs")})))
    a = dict(out_k=T(cache_args()[0].shape), out_v=T(cache_args()[2].shape))
    a.update({n: x for n, x in over.items() if n in a})
    return list(a.values()) + list(parts.values())


@pytest.mark.parametrize("over,code,match", BAD_CACHES + [
    (dict(out_k=None), ARG, "NULL"),
    (dict(out_k=T(cache_args()[0].shape, F16)), ARG, "out_k must be f32"),
    (dict(out_v=T(cache_args()[0].shape)), ARG, "out_v must have the shape"),
    (dict(out_v=T(cache_args()[2].shape, offset=1)), ARG, "aligned")])
def test_cache_values_refuses(over, code, match):
    refused("kk_cache_values", values_args(**over), code, match)


def test_a_missing_table_is_refused():
    refused("kk_cache_attention", attention_args(table=None), ARG, "NULL")
