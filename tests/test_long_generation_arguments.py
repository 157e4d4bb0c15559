"""Calls that the C entry points of a bounded cache refuse before anything is launched (no GPU: addresses that nothing stands behind)."""
import ctypes

import pytest
import torch

from intrasm_engine_amd import _lib

A, ODD = 4096, 4096 + 2
STRIDES = (ctypes.c_longlong * 3)(256, 128, 1)


def cache(**other):
    c = _lib.PagedCache(dtype=_lib.F16, eight_bits=0, pages=10, page_size=64, kv_heads=2, head_dim=128, key_page_stride=2 * 64 * 128, value_page_stride=2 * 64 * 128,
                        keys=A, values=A, table=A, seqs=3, table_width=4, table_stride=4, lengths=A)
    for name, value in other.items():
        setattr(c, name, value)
    return c


def rotation(**other):
    r = _lib.Rotation(table=A, rows=256, features=128, at=A, axis_stride=3, axes=3, sections=(ctypes.c_int * 3)(16, 24, 24))
    for name, value in other.items():
        setattr(r, name, (ctypes.c_int * len(value))(*value) if name == "sections" and value is not None else value)
    return r


def accumulate(c, heads=4, q=A, scale=0.1, weights=A, out=A, ws=A, ws_bytes=1 << 40):
    return _lib.load().iex_paged_attention_accumulate(ctypes.byref(c) if c else None, heads, q, STRIDES, scale, weights, out, STRIDES, ws, ws_bytes, None)


def evict(c, lengths=A, weights=A, keep=100, recent=10, first=2, kept=A, ws=A, ws_bytes=1 << 40):
    return _lib.load().iex_evict_tokens(ctypes.byref(c) if c else None, lengths, weights, keep, recent, first, kept, ws, ws_bytes, None)


def append(c, r=None, tokens=3, heads=2):
    return _lib.load().iex_kv_append_at(ctypes.byref(c) if c else None, tokens, None, heads, A, STRIDES, A, STRIDES, A, STRIDES, A, STRIDES, ctypes.byref(r) if r else None, None)


def rotate(r, dtype=_lib.F16, tokens=3, heads=2, dim=128, x=A, out=A):
    return _lib.load().iex_rotate(dtype, tokens, heads, dim, x, STRIDES, out, STRIDES, ctypes.byref(r) if r else None, 0, None)


@pytest.mark.parametrize("call", [accumulate, evict, append])
@pytest.mark.parametrize("other,code,text", [(dict(dtype=_lib.F32), -2, "fp16 or bf16"), (dict(head_dim=96), -2, "heads of 64"), (dict(page_size=48), -2, "pages of 16"),
                                             (dict(pages=-1), -1, "negative"), (dict(table_width=1 << 24), -3, "2^30"), (dict(lengths=None), -1, "null"), (dict(table=None), -1, "null"),
                                             (dict(keys=None), -1, "null"), (dict(values=ODD), -2, "16-byte aligned"), (dict(key_page_stride=64), -1, "overlap"), (dict(eight_bits=1), -1, "null"),
                                             (dict(kv_heads=5000), -3, "4096 key heads")])
def test_caches_that_are_refused(call, other, code, text):
    assert call(cache(**other)) == code and text in _lib.last_error()


@pytest.mark.parametrize("call,arguments,code,text", [
    (accumulate, dict(heads=3), -1, "multiple of key heads"), (accumulate, dict(heads=-2), -1, "negative"), (accumulate, dict(q=None), -1, "null"), (accumulate, dict(out=None), -1, "null"),
    (accumulate, dict(weights=None), -1, "null"), (accumulate, dict(weights=A + 4), -2, "16-byte aligned"), (accumulate, dict(scale=0.0), -2, "scale"),
    (accumulate, dict(scale=float("nan")), -2, "scale"), (accumulate, dict(q=A + 1), -2, "aligned"), (accumulate, dict(heads=2 * 4097), -3, "4096 query heads"),
    (accumulate, dict(ws=None), -1, "workspace"), (accumulate, dict(ws=A + 64), -1, "workspace"), (accumulate, dict(ws_bytes=16), -1, "workspace"),
    (evict, dict(keep=0), -1, "at least one token"), (evict, dict(keep=-1), -1, "at least one token"), (evict, dict(recent=99), -1, "among them"), (evict, dict(first=-1), -1, "among them"),
    (evict, dict(recent=(1 << 31) - 1, first=1, keep=(1 << 31) - 1), -1, "among them"), (evict, dict(lengths=None), -1, "null"), (evict, dict(lengths=A + 4), -1, "null"),
    (evict, dict(weights=None), -1, "null"), (evict, dict(kept=None), -1, "null"), (evict, dict(weights=ODD), -2, "aligned"), (evict, dict(ws=None), -1, "workspace"),
    (evict, dict(ws_bytes=64), -1, "workspace"),
])
def test_arguments_that_are_refused(call, arguments, code, text):
    assert call(cache(), **arguments) == code and text in _lib.last_error()


@pytest.mark.parametrize("call", [lambda r: append(cache(), r), rotate])
@pytest.mark.parametrize("other,code,text", [
    (dict(table=None), -1, "rotation"), (dict(table=A + 4), -1, "rotation"), (dict(rows=0), -1, "must have a row"), (dict(rows=-1), -1, "negative"), (dict(features=-16), -1, "negative"),
    (dict(axes=5), -2, "one to four axes"), (dict(axes=0), -2, "one to four axes"), (dict(sections=None), -1, "need sections"), (dict(sections=[16, 24, 23]), -1, "sections of 63"),
    (dict(sections=[-16, 56, 24]), -1, "a section of -16"), (dict(sections=[1 << 30, 1 << 30, 64]), -1, "a section"), (dict(features=0), -1, "without a rotation"),
    (dict(features=144, sections=[24, 24, 24]), -2, "128"), (dict(at=A + 1), -2, "aligned"), (dict(features=512, sections=[100, 100, 56]), -2, "up to 256")])
def test_rotations_that_are_refused(call, other, code, text):
    assert call(rotation(**other)) == code and text in _lib.last_error()


def test_evictions_that_are_too_large():
    many = cache(seqs=100, table_width=1 << 22)
    assert evict(many, keep=1 << 27, recent=0, first=0) == -3 and "too many" in _lib.last_error()
    assert evict(cache(pages=(1 << 25) + 1), keep=10, recent=0, first=0) == -3 and "2^31 tokens" in _lib.last_error()
    assert evict(cache(seqs=1 << 21), keep=10, recent=0, first=0) == -3 and "too many" in _lib.last_error()
    # a table that holds no more than is kept: what is kept takes no room
    assert _lib.load().iex_evict_tokens_workspace_bytes(ctypes.byref(cache()), 1 << 30) == _lib.load().iex_evict_tokens_workspace_bytes(ctypes.byref(cache()), 256) < 256


def test_more_refusals_of_rotations():
    assert append(cache(), rotation(at=None)) == -1 and "several axes without positions" in _lib.last_error()
    assert append(cache(), rotation(at=None, axes=1, sections=None, rows=255)) == -1 and "every position" in _lib.last_error()
    assert append(cache(), rotation(features=72, sections=[12, 12, 12])) == -2 and "multiple of 16" in _lib.last_error()
    assert rotate(None) == -1 and "null" in _lib.last_error()
    assert rotate(rotation(at=None)) == -1 and "null" in _lib.last_error()
    for arguments, code, text in ((dict(dtype=7), -2, "fp32, fp16 or bf16"), (dict(tokens=-1), -1, "negative"), (dict(x=None), -1, "null"), (dict(out=None), -1, "null"), (dict(x=A + 1), -2, "aligned"),
                                  (dict(dtype=_lib.F32, out=ODD), -2, "aligned"), (dict(tokens=1 << 27), -3, "too many"), (dict(heads=1 << 16), -3, "too many"), (dict(dim=1 << 16), -3, "too many"),
                                  (dict(dim=120), -2, "even number")):
        assert rotate(rotation(), **arguments) == code and text in _lib.last_error(), arguments


def test_workspaces_and_calls_with_nothing_to_do():
    lib = _lib.load()
    c = cache()
    scores, parts = 3 * 4 * 256 * 4, 0
    assert lib.iex_paged_attention_accumulate_workspace_bytes(ctypes.byref(c), 4) == 256 + scores + parts      # 12 statistics, rounded up
    assert lib.iex_paged_attention_accumulate_workspace_bytes(None, 4) == 0 and lib.iex_paged_attention_accumulate_workspace_bytes(ctypes.byref(c), 3) == 0
    assert lib.iex_evict_tokens_workspace_bytes(ctypes.byref(c), 0) == 0 and lib.iex_evict_tokens_workspace_bytes(None, 5) == 0
    assert accumulate(cache(seqs=0)) == 0 and accumulate(c, heads=0) == 0 and evict(cache(seqs=0)) == 0 and evict(cache(kv_heads=0)) == 0
    assert append(c, None, tokens=0, heads=0) == -1 and rotate(rotation(), tokens=0) == 0 and rotate(rotation(), heads=0) == 0
    assert rotate(rotation(rows=0, at=None, axes=1, sections=None), tokens=0) == 0 and rotate(rotation(at=None, table=None), tokens=0, x=None, out=None) == 0
    for call in (accumulate, evict, append):
        assert call(None) == -1 and "null" in _lib.last_error()


def test_tensors_of_the_cpu_are_refused():
    ops = torch.ops.iex_ops
    x, i = torch.zeros(1, 2, 64), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="q must be a CUDA tensor"):
        ops.paged_attention_accumulate_(x, x, x, i, i, x)
    with pytest.raises(RuntimeError, match="keys must be a CUDA tensor"):
        ops.evict_tokens_(x, x, i, i, x, 1, 0)
    with pytest.raises(RuntimeError, match="x must be a CUDA tensor"):
        ops.rotate(x, x[0], i)
