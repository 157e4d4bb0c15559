"""The paged cache without a GPU: what its kernels touch, walked on the host, and the calls that its entry points refuse."""
import ctypes
import os
import shutil
import subprocess

import pytest
import torch

from intrasm_engine_amd import _lib

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def check(tmp_path_factory):
    compiler = shutil.which("g++")
    assert compiler, "needs a host C++ compiler"
    exe = str(tmp_path_factory.mktemp("paged") / "check")
    subprocess.run([compiler, "-O2", "-std=c++17", "-Wall", "-Werror", os.path.join(HERE, "paged_cache_check.cpp"), "-o", exe], check=True)
    return lambda *args: subprocess.run([exe, *map(str, args)], stdout=subprocess.PIPE, text=True)


@pytest.mark.parametrize("seed", range(4))
@pytest.mark.parametrize("what", ["append", "attend", "keys"])
def test_nothing_outside_the_arrays_and_every_token_once(check, what, seed):
    got = check(what, seed)
    assert got.returncode == 0, got.stdout


# ---- refusals: no launch, so addresses that nothing stands behind will do ------------------------------------------------
A, ODD = 4096, 4096 + 2      # aligned, and not
STRIDES = (ctypes.c_longlong * 3)(256, 128, 1)


def cache(**other):
    c = _lib.PagedCache(dtype=_lib.F16, eight_bits=0, pages=10, page_size=64, kv_heads=2, head_dim=128, key_page_stride=2 * 64 * 128, value_page_stride=2 * 64 * 128,
                        keys=A, values=A, table=A, seqs=3, table_width=4, table_stride=4, lengths=A)
    for name, value in other.items():
        setattr(c, name, value)
    return c


def append(c, tokens=3, offsets=None, heads=2, k=A, v=A, q=A, out=A, rotation=A, positions=256, rotary=128):
    return _lib.load().iex_kv_append(ctypes.byref(c) if c else None, tokens, offsets, heads, k, STRIDES, v, STRIDES, q, STRIDES, out, STRIDES, rotation, positions, rotary, 0, None)


def attend(c, heads=4, q=A, scale=0.1, listed=None, count=0, out=A, ws=A, ws_bytes=1 << 40):
    return _lib.load().iex_paged_attention(ctypes.byref(c) if c else None, heads, q, STRIDES, scale, listed, count, out, STRIDES, ws, ws_bytes, None)


def select(c, heads=4, q=A, count=3, first=1, last=1, out=A, ws=A, ws_bytes=1 << 40):
    return _lib.load().iex_select_pages(ctypes.byref(c) if c else None, heads, q, STRIDES, count, first, last, out, ws, ws_bytes, None)


BAD_CACHES = [(dict(dtype=_lib.F32), -2, "fp16 or bf16"), (dict(head_dim=96), -2, "heads of 64"), (dict(page_size=48), -2, "pages of 16"), (dict(page_size=512), -2, "pages of 16"),
              (dict(page_size=8), -2, "pages of 16"), (dict(pages=-1), -1, "negative"), (dict(seqs=-1), -1, "negative"), (dict(table_width=1 << 24), -3, "2^30"), (dict(lengths=None), -1, "null"),
              (dict(table=None), -1, "null"), (dict(kv_heads=5000), -3, "4096 key heads")]
BAD_PAGES = [(dict(keys=None), -1, "null"), (dict(values=None), -1, "null"), (dict(keys=ODD), -2, "16-byte aligned"), (dict(values=ODD), -2, "16-byte aligned"),
             (dict(key_page_stride=2 * 64 * 128 + 4), -2, "16-byte aligned"), (dict(value_page_stride=64 * 128), -1, "overlap"), (dict(eight_bits=1), -1, "null"),
             (dict(eight_bits=1, key_exponents=A, value_exponents=A + 4), -2, "16-byte aligned")]


@pytest.mark.parametrize("other,code,text", BAD_CACHES)
@pytest.mark.parametrize("call", [append, attend, select])
def test_caches_that_every_entry_point_refuses(call, other, code, text):
    assert call(cache(bounds=A, **other)) == code and text in _lib.last_error()


@pytest.mark.parametrize("other,code,text", BAD_PAGES)
@pytest.mark.parametrize("call", [append, attend])
def test_pages_that_are_refused(call, other, code, text):
    assert call(cache(**other)) == code and text in _lib.last_error()


@pytest.mark.parametrize("call,arguments,code,text", [
    (append, dict(tokens=-1), -1, "negative"), (append, dict(tokens=4), -1, "one token per sequence"), (append, dict(k=None), -1, "null"), (append, dict(v=None), -1, "null"),
    (append, dict(q=None), -1, "null"), (append, dict(out=None), -1, "null"), (append, dict(rotary=72), -2, "multiple of 16"), (append, dict(rotary=144), -2, "multiple of 16"),
    (append, dict(positions=255), -1, "every position"), (append, dict(rotation=None), -1, "rotation"), (append, dict(rotation=ODD), -1, "rotation"), (append, dict(k=A + 1), -2, "aligned"),
    (append, dict(heads=-2), -1, "negative"),
    (attend, dict(heads=3), -1, "multiple of key heads"), (attend, dict(heads=-2), -1, "negative"), (attend, dict(q=None), -1, "null"), (attend, dict(out=None), -1, "null"),
    (attend, dict(scale=0.0), -2, "scale"), (attend, dict(scale=-1.0), -2, "scale"), (attend, dict(scale=float("nan")), -2, "scale"), (attend, dict(scale=float("inf")), -2, "scale"),
    (attend, dict(count=3), -1, "null"), (attend, dict(listed=A), -1, "must have entries"), (attend, dict(listed=A, count=-1), -1, "must have entries"),
    (attend, dict(listed=A, count=1 << 25), -3, "2^30"), (attend, dict(q=A + 1), -2, "aligned"),
    (select, dict(heads=3), -1, "multiple of key heads"), (select, dict(count=0), -1, "at least one page"), (select, dict(count=3, first=2, last=2), -1, "among them"),
    (select, dict(first=-1), -1, "at least one page"), (select, dict(q=None), -1, "null"), (select, dict(out=None), -1, "null"),
])
def test_arguments_that_are_refused(call, arguments, code, text):
    assert call(cache(bounds=A), **arguments) == code and text in _lib.last_error()


def test_workspaces_and_null_caches():
    lib = _lib.load()
    long = cache(table_width=1 << 12, seqs=1, table_stride=1 << 12)
    need = lib.iex_paged_attention_workspace_bytes(ctypes.byref(long), 4, 0)
    assert need > 0 and attend(long, ws=None) == -1 and "workspace" in _lib.last_error()
    assert attend(long, ws_bytes=need - 1) == -1 and attend(long, ws=A + 64) == -1
    assert lib.iex_paged_attention_workspace_bytes(ctypes.byref(cache(table_width=1)), 4, 0) == 0
    many = cache(bounds=A, table_width=1 << 12, seqs=1, table_stride=1 << 12)
    assert lib.iex_select_pages_workspace_bytes(ctypes.byref(many)) == 2 * 4096 * 4 and lib.iex_select_pages_workspace_bytes(ctypes.byref(cache(bounds=A))) == 0
    for given in (dict(ws=None), dict(ws=A + 16), dict(ws_bytes=4)):
        assert select(many, **given) == -1 and "workspace" in _lib.last_error()
    assert select(cache()) == -1 and "null" in _lib.last_error()
    for call in (append, attend, select):
        assert call(None) == -1 and "null" in _lib.last_error()
    assert lib.iex_paged_attention_workspace_bytes(None, 4, 0) == 0 and lib.iex_select_pages_workspace_bytes(None) == 0


def test_calls_with_nothing_to_do():
    assert append(cache(), tokens=0, offsets=A) == 0 and attend(cache(seqs=0)) == 0 and select(cache(bounds=A, seqs=0)) == 0
    assert attend(cache(), heads=0) == 0


def test_tensors_of_the_cpu_are_refused():
    ops = torch.ops.iex_ops
    x = torch.zeros(1, 2, 64)
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="k must be a CUDA tensor"):
        ops.kv_append_(x, x, x, x, i, i)
    with pytest.raises(RuntimeError, match="q must be a CUDA tensor"):
        ops.paged_attention(x, x, x, i, i)
    with pytest.raises(RuntimeError, match="q must be a CUDA tensor"):
        ops.select_pages(x, x, i, i, 16, 1)
