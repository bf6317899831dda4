"""Which caches mt_rope_append and mt_kv_copy take to overlap, without a GPU (the ones that they accept run in
test_kv_interleaved_gpu.py)."""
import pytest

import mingtts as mt
from test_f8_abi import A, MB, append, kv_struct, ref

B, HKV, LEN = 4, 2, 64
N = HKV * LEN * 64  # a sequence's codes
S = HKV * LEN       # and scale bytes


@pytest.mark.parametrize("over", [
    dict(v=A + N - 16, stride=2 * N),                      # side by side, but for the last 16 bytes
    dict(v=A + N + 16, stride=2 * N),                      # into the next sequence's keys
    dict(v=A + 4 * N - 16, stride=2 * N),                  # two sequences on
    dict(v=A - N + 16, stride=2 * N),                      # before the keys
    dict(v=A + N, stride=N + 16),
    dict(k_scale=A + 2 * N - 4, stride=4 * N, scale_stride=4 * N, v=A + N),
    dict(v_scale=A + 128 * MB + S - 4, scale_stride=2 * S),
    dict(k_scale=A + 2 * N, stride=4 * N, scale_stride=2 * S, v=A + N),  # between the keys, at another stride
])
def test_append_refuses(over):
    assert append(kv_struct(**over)) == mt.EINVAL
    assert "overlap each other" in mt.last_error(), mt.last_error()


def test_copy_refuses():
    src, L = kv_struct(stride=4 * N, v=A + N), mt.load()
    for k, v in ((A + N, A + 3 * N), (A + 2 * N, A + 4 * N), (A + 2 * N + 16, A + 3 * N + 16)):
        dst = kv_struct(stride=4 * N, k=k, v=v, k_scale=A + 256 * MB, v_scale=A + 257 * MB)
        assert L.mt_kv_copy(ref(src), ref(dst), B, 1, HKV, None, None, None) == mt.EINVAL
        assert "overlap" in mt.last_error(), mt.last_error()
