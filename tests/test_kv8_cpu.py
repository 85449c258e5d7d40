"""The 8-bit paged cache without a GPU: argument checks of the C ABI, scratch sizes, and the plain page map itself."""
import ctypes

import pytest

import aihost_b200 as A
from aihost_b200.kv8 import Kv8Spec

BASE = dict(n_q_heads=32, n_kv_heads=8, head_dim=128, page_rows=64, n_pages=100, max_pages=16)


def _size(batch=4, n_tokens=4, max_new=1, max_kv=1024, **kw):
    need = ctypes.c_size_t()
    d = Kv8Spec(**{**BASE, **kw}).desc()
    return A.lib().aihost_kv8_workspace_size(ctypes.byref(d), batch, n_tokens, max_new, max_kv, ctypes.byref(need)), need.value


@pytest.mark.parametrize("change, status, word", [
    (dict(), A.OK, b""),
    (dict(n_q_heads=30), A.EINVAL, b"multiple"),
    (dict(n_kv_heads=0), A.EINVAL, b"n_kv_heads"),
    (dict(head_dim=96), A.EUNSUPPORTED, b"head_dim"),
    (dict(page_rows=48), A.EUNSUPPORTED, b"page_rows"),
    (dict(page_rows=256), A.EUNSUPPORTED, b"page_rows"),
    (dict(n_pages=0), A.EINVAL, b"n_pages"),
    (dict(max_pages=0), A.EINVAL, b"max_pages"),
    (dict(io_dtype=A.Q8_0), A.EINVAL, b"io_dtype"),
    (dict(out_dtype=3), A.EINVAL, b"out_dtype"),
    (dict(rope_mode=7), A.EINVAL, b"rope_mode"),
    (dict(rope_theta=-1.0), A.EINVAL, b"rope_theta"),
    (dict(rope_theta=-1.0, rope_mode=A.ROPE_NONE), A.OK, b""),
    (dict(scale=float("nan")), A.EINVAL, b"scale"),
    (dict(score_cap=-2.0), A.EINVAL, b"score_cap"),
    (dict(score_cap=float("inf")), A.EINVAL, b"score_cap"),
    (dict(batch=0), A.EINVAL, b"batch"),
    (dict(n_tokens=-1), A.EINVAL, b"n_tokens"),
    (dict(max_new=0), A.EINVAL, b"max_new"),
    (dict(max_new=9, max_kv=8), A.EINVAL, b"max_kv"),
])
def test_descriptions_are_checked(change, status, word):
    assert _size(**change)[0] == status
    if status != A.OK:
        assert word in A.lib().aihost_attn_last_error()


@pytest.mark.parametrize("field, value, word", [("q_token_stride", 100, b"at least"), ("kv_token_stride", 2056, b"multiples")])
def test_strides_are_checked(field, value, word):
    d = Kv8Spec(**BASE).desc()
    setattr(d, field, value)
    need = ctypes.c_size_t()
    assert A.lib().aihost_kv8_workspace_size(ctypes.byref(d), 1, 1, 1, 64, ctypes.byref(need)) == A.EINVAL
    assert word in A.lib().aihost_attn_last_error()


def test_scratch_grows_with_the_cache_and_not_for_one_chunk():
    assert _size(batch=1, max_kv=64)[1] == 0  # a single chunk is written straight out
    assert 0 < _size(batch=1, max_kv=4096)[1] < _size(batch=1, max_kv=65536)[1]


def test_of_tiles_alike_only_those_past_whole_waves_are_cut():
    """1200 new rows of 4 heads a group are 19 tiles of 256 for each of 8 heads: 148 of them, a wave, need no scratch."""
    status, size = _size(batch=1, n_tokens=1200, max_new=1200, max_kv=13200, n_pages=1000, max_pages=300)
    parts, odd = divmod(size, 256 * (128 + 2) * 4)
    assert status == A.OK and odd == 0 and parts % 4 == 0 and 2 <= parts // 4 <= 32


def test_null_context_is_refused():
    L = A.lib()
    d = Kv8Spec(**BASE).desc()
    r = ctypes.byref(d)
    assert L.aihost_page_map(None, 1, 64, 1, 1, 1, *[None] * 11) == A.EINVAL
    assert L.aihost_page_release(None, 1, 64, 1, 1, *[None] * 6) == A.EINVAL
    assert L.aihost_kv8_append(None, r, 1, *[None] * 9) == A.EINVAL
    assert L.aihost_kv8_read(None, r, 1, None, None, None, None, A.F16, None) == A.EINVAL
    assert L.aihost_kv8_attention(None, r, 1, 1, 1, 1, *[None] * 13) == A.EINVAL
    assert L.aihost_kv8_workspace_size(r, 1, 1, 1, 1, None) == A.EINVAL
    assert L.aihost_kv8_workspace_size(None, 1, 1, 1, 1, ctypes.byref(ctypes.c_size_t())) == A.EINVAL


def test_plain_page_map_by_hand():
    from kv8_plain import page_map

    # 16-row pages; sequence 0 has 15 rows in page 9 and gets 2, sequence 1 gets nothing, sequence 2 gets its first 17
    t, kv, start, slots, pos, free, refused = page_map(16, 12, 4, 20, [15, 32, 0], [2, 0, 17], [3, 1, 4, 7], 4,
                                                       [[9, -1, -1, -1], [5, 6, -1, -1], [-1] * 4])
    assert not refused and kv == [17, 32, 17] and start == [0, 2, 2, 19] and free == 1
    assert t == [[9, 7, -1, -1], [5, 6, -1, -1], [4, 1, -1, -1]]
    assert slots == [9 * 16 + 15, 7 * 16] + [4 * 16 + i for i in range(16)] + [1 * 16] + [-1]
    assert pos == [15, 16] + list(range(17)) + [0]
    assert page_map(16, 12, 4, 20, [15, 32, 0], [2, 0, 17], [3, 1], 2, [[9], [5], [0]])[-1]


def test_plan_tells_scratch_and_kernel():
    """Without a context, for the current device: the scratch of aihost_kv8_workspace_size, and the kernel by the step."""
    need, kernel = ctypes.c_size_t(), ctypes.c_int32()
    d = Kv8Spec(**BASE).desc()

    def plan(*a):
        assert A.lib().aihost_kv8_plan(None, ctypes.byref(d), *a, ctypes.byref(need), ctypes.byref(kernel)) == A.OK
        assert need.value == _size(*a)[1]
        return kernel.value

    assert plan(64, 64, 1, 8192) == A.KV8_SPLIT_CACHE
    assert plan(8, 64, 8, 8192) == A.KV8_SPLIT_CACHE
    assert plan(1, 2048, 2048, 16384) == A.KV8_TENSOR
    d.io_dtype = A.F32
    assert A.lib().aihost_kv8_plan(None, ctypes.byref(d), 1, 2048, 2048, 16384, None, ctypes.byref(kernel)) == A.OK
    assert kernel.value == A.KV8_SPLIT_CACHE
    assert A.lib().aihost_kv8_plan(None, ctypes.byref(d), 0, 1, 1, 1, None, None) == A.EINVAL


@pytest.mark.parametrize("mode, ok", [(A.ROPE_NONE, True), (A.ROPE_NEOX, True), (3, False), (-1, False), (0x200, False)])
def test_round_q_goes_with_every_rope_mode(mode, ok):
    d = Kv8Spec(**BASE, rope_mode=mode, round_q=True).desc()
    assert d.rope_mode == mode | A.KV8_ROUND_Q
    need = ctypes.c_size_t()
    got = A.lib().aihost_kv8_workspace_size(ctypes.byref(d), 1, 1, 1, 64, ctypes.byref(need))
    assert got == (A.OK if ok else A.EINVAL)
    assert Kv8Spec(**BASE, rope_mode=mode).desc().rope_mode == mode
