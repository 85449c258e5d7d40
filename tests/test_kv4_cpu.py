"""The 4-bit paged cache without a GPU: argument checks of the C ABI, plans, and the plain forms themselves."""
import ctypes

import numpy as np
import pytest

import aihost_b200 as A
import kv4_plain as plain
from aihost_b200.kv4 import Kv4Spec
from test_kv8_cpu import BASE


def _plan(batch=4, n_tokens=4, max_new=1, max_kv=1024, **kw):
    need, kernel = ctypes.c_size_t(), ctypes.c_int32()
    d = Kv4Spec(**{**BASE, **kw}).desc()
    status = A.lib().aihost_kv4_plan(None, ctypes.byref(d), batch, n_tokens, max_new, max_kv, ctypes.byref(need), ctypes.byref(kernel))
    return status, need.value, kernel.value


@pytest.mark.parametrize("change, status, word", [
    (dict(), A.OK, b""), (dict(n_q_heads=30), A.EINVAL, b"multiple"), (dict(head_dim=96), A.EUNSUPPORTED, b"head_dim"),
    (dict(page_rows=8), A.EUNSUPPORTED, b"page_rows"), (dict(n_pages=0), A.EINVAL, b"n_pages"),
    (dict(io_dtype=A.Q8_0), A.EINVAL, b"io_dtype"), (dict(rope_mode=7), A.EINVAL, b"rope_mode"),
    (dict(score_cap=float("nan")), A.EINVAL, b"score_cap"), (dict(batch=0), A.EINVAL, b"batch"),
    (dict(max_new=9, max_kv=8), A.EINVAL, b"max_kv")])
def test_descriptions_are_checked(change, status, word):
    assert _plan(**change)[0] == status
    if status != A.OK:
        assert word in A.lib().aihost_attn_last_error()


def test_plans():
    assert _plan(batch=1, max_kv=64)[1] == 0  # a single chunk is written straight out
    assert 0 < _plan(batch=1, max_kv=4096)[1] < _plan(batch=1, max_kv=65536)[1]
    assert _plan(64, 64, 1, 8192)[2] == _plan(8, 64, 8, 8192)[2] == A.KV8_SPLIT_CACHE
    assert _plan(1, 2048, 2048, 16384)[2] == A.KV8_TENSOR
    assert _plan(1, 2048, 2048, 16384, io_dtype=A.F32)[2] == A.KV8_SPLIT_CACHE


@pytest.mark.parametrize("max_kv", [1, 127, 8193, 1 << 20, (1 << 31) - 1])
@pytest.mark.parametrize("batch, new", [(1, 1), (70000, 1), (3, 5), (1, 4000)])
def test_plans_of_every_size(batch, new, max_kv):
    """Scratch is whole parts of 8, 16 or 256 rows, head_dim + 2 floats each, within what a context can be given."""
    if max_kv < new:
        return
    status, size, kernel = _plan(batch, batch * new, new, max_kv)
    assert status == A.OK and size % ((128 + 2) * 4 * (256 if kernel == A.KV8_TENSOR else 8)) == 0 and size < 1 << 36


def test_null_arguments_are_refused():
    L = A.lib()
    d = Kv4Spec(**BASE).desc()
    r = ctypes.byref(d)
    assert L.aihost_kv4_append(None, r, 1, *[None] * 9) == A.EINVAL
    assert L.aihost_kv4_read(None, r, 1, None, None, None, None, A.F16, None) == A.EINVAL
    assert L.aihost_kv4_attention(None, r, 1, 1, 1, 1, *[None] * 13) == A.EINVAL
    assert L.aihost_kv4_plan(None, None, 1, 1, 1, 1, None, None) == A.EINVAL
    assert L.aihost_kv4_plan(None, r, 1, 1, 1, 64, None, None) == A.OK


def test_plain_codes_by_hand():
    x = np.arange(16, dtype=np.float32)[None] * 2 - 3  # -3 .. 27: step 2, codes 0 .. 15
    codes, low, step = plain.quantise(x)
    assert codes.tolist() == [list(range(16))] and low.tolist() == [-3.0] and step.tolist() == [2.0]
    packed = plain.pack(codes)
    assert packed.tolist() == [[0x20, 0x64, 0x31, 0x75, 0xa8, 0xec, 0xb9, 0xfd]]
    assert np.array_equal(plain.unpack(packed), codes)
    assert np.array_equal(plain.values(packed, np.float16([[-3, 2]])), x)
    codes, low, step = plain.quantise(np.full((1, 16), 2.5, np.float32))
    assert not codes.any() and low.tolist() == [2.5] and step.tolist() == [2.0 ** -24]
    assert np.isnan(plain.quantise(np.float32([[1, np.inf]]))[1]).all()
