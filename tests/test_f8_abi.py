"""The 8-bit and shared-prefix entry points without a GPU: refusals before any HIP call, calls without work,
the Python classes' checks, and the tests' own oracle of the format."""
import ctypes

import numpy as np
import pytest
import torch

import mingtts as mt
import _f8_util as U

A = 1 << 20  # fake aligned device addresses, never dereferenced
MB = 1 << 20


def kv_struct(base=A, hkv=2, cache_len=64, t=mt.F8, B=4, **over):
    f = dict(k=base, v=base + 64 * MB, k_scale=base + 128 * MB, v_scale=base + 129 * MB, stride=hkv * cache_len * 64,
             scale_stride=hkv * cache_len, cache_len=cache_len, cache_t=t)
    f.update(over)
    return mt.KvStruct(*[f[n] for n, _ in mt.KvStruct._fields_])


def ref(s):
    return ctypes.byref(s) if s is not None else None


def append(kv, qkv=1024 * MB, ldq=18 * 64, B=4, T=1, hq=14, hkv=2, inv_freq=A, q=1536 * MB, ldo=14 * 64):
    return mt.load().mt_rope_append(qkv, ldq, B, T, hq, hkv, None, None, 0, ref(kv), inv_freq, q, ldo, None)


@pytest.mark.parametrize("kv,call,needle", [
    (dict(t=mt.BF16), {}, "f32, f16 or f8"),
    (dict(cache_t=9), {}, "f32, f16 or f8"),
    (dict(k=0), {}, "null k or v"),
    (dict(v=A + 8), {}, "16-byte aligned"),
    (dict(cache_len=0), {}, "cache_len"),
    (dict(cache_len=(1 << 30) + 4), {}, "cache_len"),
    (dict(cache_len=66), {}, "multiple of 4"),
    (dict(k_scale=0), {}, "null scales"),
    (dict(v_scale=A + 1), {}, "4-byte aligned"),
    (dict(stride=64), {}, "stride"),
    (dict(stride=2 * 64 * 64 + 8), {}, "stride"),
    (dict(scale_stride=64), {}, "scale_stride"),
    (dict(v=A), {}, "overlap each other"),
    (dict(), dict(qkv=0), "null pointer"),
    (dict(), dict(inv_freq=0), "null pointer"),
    (dict(), dict(ldq=17 * 64), "ldq"),
    (dict(), dict(ldo=13 * 64), "ldo"),
    (dict(), dict(qkv=1024 * MB + 4), "16-byte aligned"),
    (dict(), dict(ldo=14 * 64 + 2), "16-byte row strides"),
    (dict(), dict(q=1024 * MB), "overlaps qkv"),
    (dict(k=1024 * MB), {}, "overlap qkv"),
    (dict(), dict(hkv=0), "hkv"),
    (dict(), dict(B=1 << 16, T=1 << 16), "too many"),
])
def test_append_refuses(kv, call, needle):
    assert append(kv_struct(**kv), **call) == mt.EINVAL
    assert needle in mt.last_error(), mt.last_error()


def test_null_caches_are_refused():
    assert append(None) == mt.EINVAL and "null kv" in mt.last_error()
    L = mt.load()
    assert L.mt_kv_copy(None, ref(kv_struct()), 1, 1, 2, None, None, None) == mt.EINVAL
    assert L.mt_kv_copy(ref(kv_struct()), None, 1, 1, 2, None, None, None) == mt.EINVAL


def test_copy_refuses_overlap():
    L = mt.load()
    s = kv_struct()
    assert L.mt_kv_copy(ref(s), ref(s), 4, 1, 2, None, None, None) == mt.EINVAL and "overlap" in mt.last_error()
    d = kv_struct(base=2048 * MB, t=mt.F16, v=2048 * MB + 64)
    assert L.mt_kv_copy(ref(s), ref(d), 4, 1, 2, None, None, None) == mt.EINVAL and "each other" in mt.last_error()


def attend(kv, prefix=None, q=1024 * MB, ldq=896, B=4, T=1, hq=14, hkv=2, prefix_len=0, len_max=0, window=0, out=1536 * MB,
           ldo=896, ws=None, wsn=0):
    return mt.load().mt_attention_shared(q, ldq, B, T, hq, hkv, None, None, ref(kv), ref(prefix), prefix_len, len_max, window,
                                         out, ldo, 0.125, ws, wsn, None)


@pytest.mark.parametrize("kv,prefix,call,needle", [
    (dict(), None, dict(hq=13), "multiple of hkv"),
    (dict(), None, dict(hq=0), "multiple of hkv"),
    (dict(), None, dict(q=0), "null pointer"),
    (dict(), None, dict(ldq=64), "ldq / ldo"),
    (dict(), None, dict(out=1536 * MB + 8), "16-byte aligned"),
    (dict(), None, dict(out=1024 * MB + 896 * 4), "out overlaps q"),
    (dict(), None, dict(prefix_len=3), "null prefix"),
    (dict(), dict(t=mt.F16), dict(prefix_len=3), "one type"),
    (dict(), dict(), dict(prefix_len=65), "past the prefix"),
    (dict(t=mt.BF16), None, {}, "f32, f16 or f8"),
    (dict(), None, dict(hq=8194), "too many"),
    (dict(), None, dict(B=1 << 20, T=100, hq=16, hkv=1, ldq=1024), "too many"),
])
def test_attention_refuses(kv, prefix, call, needle):
    p = kv_struct(base=2816 * MB, **prefix) if prefix is not None else None
    assert attend(kv_struct(**kv), p, **call) == mt.EINVAL
    assert needle in mt.last_error(), mt.last_error()


def test_attention_refuses_a_small_workspace():
    L = mt.load()
    need = L.mt_attention_shared_workspace(1, 1, 14, 2, 0, 1 << 17, 0, mt.F8)
    if need == 0:
        pytest.skip("this size is not split")
    kv = kv_struct(cache_len=1 << 17)
    for ws, n in ((None, need), (A, need - 1), (A + 8, need)):
        assert attend(kv, B=1, ws=ws, wsn=n) == mt.EINVAL and "workspace" in mt.last_error()


def quant(x=A, xt=mt.F32, rows=4, K=256, ldx=256, norm=None, nt=mt.F16, eps=1e-6, codes=1024 * MB, ldq=256, scales=1536 * MB, lds=4):
    return mt.load().mt_quantize_f8(x, xt, rows, K, ldx, norm, nt, eps, codes, ldq, scales, lds, None)


@pytest.mark.parametrize("call,needle", [
    (dict(xt=mt.F8), "f32, f16 or bf16"),
    (dict(K=0), "multiple of 16"),
    (dict(K=40, ldx=40), "multiple of 16"),
    (dict(x=0), "null pointer"),
    (dict(ldx=128), "ldx"),
    (dict(ldq=128), "ldq"),
    (dict(lds=3), "lds"),
    (dict(K=1024, ldx=1024, ldq=1024), "lds"),
    (dict(x=A + 4), "16-byte aligned"),
    (dict(codes=1024 * MB + 8), "16-byte aligned"),
    (dict(scales=1536 * MB + 2), "4-byte aligned"),
    (dict(norm=A + 2), "16-byte aligned"),
    (dict(norm=A, nt=mt.F32), "norm must be"),
    (dict(norm=A, eps=-1.0), "eps"),
    (dict(norm=A, eps=float("nan")), "eps"),
    (dict(norm=A, K=1 << 20, ldx=1 << 20, ldq=1 << 20, lds=1 << 13), "a norm over K"),
    (dict(codes=A), "overlap"),
    (dict(scales=1024 * MB + 16), "overlap"),
    (dict(rows=1 << 31), "too many"),
    (dict(rows=1 << 30, lds=64), "too many"),
])
def test_quantize_refuses(call, needle):
    assert quant(**call) == mt.EINVAL
    assert needle in mt.last_error(), mt.last_error()


def lin(x=A, xt=mt.F8, xs=512 * MB, ldxs=4, norm=None, w=1024 * MB, ws=1536 * MB, w2=None, w2s=None, bias=None, bt=mt.F16,
        y=2048 * MB, M=4, N=64, K=256, ldx=256, ldy=64, flags=0, eps=0.0):
    return mt.load().mt_linear_f8(x, xt, xs, ldxs, norm, w, ws, w2, w2s, bias, bt, y, mt.GemvParams(M, N, K, ldx, ldy, flags, eps),
                                  None)


@pytest.mark.parametrize("call,code,needle", [
    (dict(xt=7), mt.EINVAL, "activation dtype"),
    (dict(flags=64), mt.EINVAL, "unknown flag"),
    (dict(flags=mt.GemvFlags.bias), mt.EINVAL, "MT_BIAS without"),
    (dict(bias=A, bt=mt.F32), mt.EINVAL, "must be f16 or bf16"),
    (dict(flags=mt.GemvFlags.siluGate), mt.EINVAL, "without w2"),
    (dict(flags=mt.GemvFlags.siluGate, w2=A), mt.EINVAL, "without w2"),
    (dict(w=0), mt.EINVAL, "null x"),
    (dict(ws=0), mt.EINVAL, "null x"),
    (dict(K=24, ldx=32), mt.EINVAL, "multiple of 16"),
    (dict(ldx=128), mt.EINVAL, "ldx"),
    (dict(ldy=32), mt.EINVAL, "ldy"),
    (dict(x=A + 8), mt.EINVAL, "16-byte aligned"),
    (dict(w=1024 * MB + 8), mt.EINVAL, "16-byte aligned"),
    (dict(ws=1536 * MB + 1), mt.EINVAL, "scales must be"),
    (dict(xs=0), mt.EINVAL, "xs must be"),
    (dict(ldxs=6), mt.EINVAL, "xs must be"),
    (dict(K=1024, ldx=1024, ldxs=4), mt.EINVAL, "xs must be"),
    (dict(norm=A), mt.EINVAL, "not quantised yet"),
    (dict(xt=mt.F32, M=17), mt.ENOTSUP, "mt_quantize_f8 first"),
    (dict(xt=mt.F32, norm=A, K=32784, ldx=32784), mt.ENOTSUP, "mt_quantize_f8 first"),
    (dict(xt=mt.F32, norm=A, eps=-1.0), mt.EINVAL, "eps"),
    (dict(x=2048 * MB), mt.EINVAL, "x overlaps y"),
    (dict(xs=2048 * MB), mt.EINVAL, "xs overlaps y"),
    (dict(M=1 << 31), mt.EINVAL, "too large"),
    (dict(N=1 << 31, ldy=1 << 31), mt.EINVAL, "too large"),
    (dict(K=1 << 23, ldx=1 << 23), mt.EINVAL, "past 2^22"),
    (dict(ldx=1 << 23), mt.EINVAL, "past 2^22"),
])
def test_linear_refuses(call, code, needle):
    assert lin(**call) == code
    assert needle in mt.last_error(), mt.last_error()


def test_the_tile_choice_is_checked():
    with pytest.raises(mt.MingTTSError, match="tile choice"):
        mt.set_tuning(mt.TUNE_F8_TILE, 99)
    assert mt.set_tuning(mt.TUNE_F8_TILE, -1) == 0


def test_calls_without_work():
    kv = kv_struct()
    assert append(kv, B=0) == append(kv, T=0) == mt.OK
    assert attend(kv, B=0) == attend(kv, T=0) == mt.OK
    assert mt.load().mt_kv_copy(ref(kv), ref(kv), 0, 5, 2, None, None, None) == mt.OK
    assert quant(rows=0) == lin(M=0) == lin(N=0) == mt.OK


def test_the_other_entry_points_refuse_8_bits():
    assert mt.linear_raw(A, mt.F8, A, None, mt.F16, None, 8 * A, 2, 64, 64, 64, 64, 0, stream=0) == mt.EINVAL
    assert mt.linear_raw(A, mt.F32, A, None, mt.F8, None, 8 * A, 2, 64, 64, 64, 64, 0, stream=0) == mt.EINVAL
    rc = mt.load().mt_attention_decode(A, 896, 2, 14, 2, A, 0, A, A, mt.F8, 512, 1 << 16, A, 896, 0.125, None)
    assert rc == mt.EINVAL


def test_python_classes_check():
    z = torch.zeros
    k8, s8 = z(2, 2, 8, 64, dtype=torch.uint8), z(2, 2, 8, dtype=torch.uint8)
    kv = mt.KV(k8, k8.clone(), s8, s8.clone())
    assert (kv.batch, kv.hkv, kv.cache_len, kv.type) == (2, 2, 8, mt.F8)
    assert mt.KV(k8[0], k8[1], s8[0], s8[1]).batch == 1
    f = k8.view(torch.float8_e4m3fn)
    assert mt.KV(f, f.clone(), s8, s8.clone()).type == mt.F8
    bad = [(k8, k8.clone(), None, None), (k8, k8[:1], s8, s8), (k8, k8.clone(), s8, s8[:, :1]), (z(2, 2, 8, 32), z(2, 2, 8, 32), None, None),
           (z(2, 2, 8, 64, dtype=torch.bfloat16),) * 2 + (None, None), (z(2, 2, 16, 64)[:, :, ::2],) * 2 + (None, None)]
    for b in bad:
        with pytest.raises(ValueError):
            mt.KV(*b)
    with pytest.raises(ValueError):
        mt.kv_copy(kv, mt.KV(z(2, 4, 8, 64), z(2, 4, 8, 64)), 2, 1)
    with pytest.raises(ValueError):
        mt.kv_copy(kv, mt.KV(z(2, 2, 8, 64), z(2, 2, 8, 64)), 3, 1)
    with pytest.raises(ValueError):
        mt.F8Matrix(z(4, 40, dtype=torch.uint8), z(4, 4, dtype=torch.uint8))
    with pytest.raises(ValueError):
        mt.F8Matrix(z(4, 48, dtype=torch.uint8), z(4, 1, dtype=torch.uint8))
    w = mt.F8Matrix(z(4, 48, dtype=torch.uint8), z(4, 4, dtype=torch.uint8))
    with pytest.raises(ValueError):
        mt.linear_f8(z(2, 64), w, z(2, 4))
    with pytest.raises(ValueError):
        mt.linear_f8(z(2, 48), w, z(2, 4), M=3)
    with pytest.raises(ValueError, match="fp32"):
        mt.linear_f8(z(2, 48), w, z(2, 4, dtype=torch.float16))
    q, o, pos = z(2, 896), z(2, 896), z(2, dtype=torch.int64)
    with pytest.raises(ValueError, match="int32"):
        mt.attention_shared(q, 2, 1, 14, 2, pos, kv, o)
    with pytest.raises(ValueError, match="fp32"):
        mt.attention_shared(q.half(), 2, 1, 14, 2, pos.int(), kv, o)
    with pytest.raises(ValueError, match="int32"):
        mt.rope_append(z(2, 1152), 2, 1, 14, 2, pos, kv, z(32))


def test_python_refuses_strided_rows():
    w = mt.F8Matrix(torch.zeros(4, 48, dtype=torch.uint8), torch.zeros(4, 4, dtype=torch.uint8))
    for x in (torch.zeros(48, 2).t(), torch.zeros(2, 96)[:, ::2]):
        with pytest.raises(ValueError, match="contiguous"):
            mt.linear_f8(x, w, torch.zeros(2, 4))


def test_python_refuses_short_vectors():
    w = mt.F8Matrix(torch.zeros(4, 48, dtype=torch.uint8), torch.zeros(4, 4, dtype=torch.uint8))
    for more in (dict(bias=torch.zeros(3, dtype=torch.float16)), dict(norm=torch.zeros(47, dtype=torch.float16))):
        with pytest.raises(ValueError, match="holds"):
            mt.linear_f8(torch.zeros(2, 48), w, torch.zeros(2, 4), **more)


def test_python_refuses_two_devices():
    c, s = torch.zeros(2, 2, 8, 64, dtype=torch.uint8), torch.ones(2, 2, 8, dtype=torch.uint8)
    for bad in ((c, c.to("meta"), s, s), (c, c, s, s.to("meta"))):
        with pytest.raises(ValueError, match="one device"):
            mt.KV(*bad)
    with pytest.raises(ValueError, match="one device"):
        mt.F8Matrix(torch.zeros(4, 48, dtype=torch.uint8), torch.zeros(4, 4, dtype=torch.uint8, device="meta"))


def test_the_oracle_of_the_format():
    """Every code is its own nearest code at scale 1, midpoints go to the even one, blocks take the least scale."""
    x = np.where(np.isnan(U.TABLE), 0, U.TABLE)
    x[0] = 448.0
    c, s = U.encode(x[None], 256)
    keep = ~np.isnan(U.TABLE)
    keep[0] = False
    assert s[0, 0] == 127 and np.array_equal(c[0][keep], np.arange(256)[keep])
    mid = (U.TABLE[:126] + U.TABLE[1:127]) / 2
    c, _ = U.encode(np.append(mid, 448.0)[None], 128)
    assert np.array_equal(c[0][:126], [i + (i & 1) for i in range(126)])
    for top, want in ((448.0, 127), (449.0, 128), (224.0, 126), (0.0, 1), (2.0 ** -140, 1), (3.4e38, 247), (448 * 2.0 ** -126, 1)):
        assert U.encode(np.array([[top] + [0.0] * 63]), 64)[1][0, 0] == want
    back = U.decode(*U.encode(np.random.default_rng(1).standard_normal((50, 64)), 64), 64)
    assert np.isfinite(back).all()
    c, s = U.encode(np.array([[1.0, np.inf, -np.inf, np.nan] + [0.0] * 60]), 64)
    assert s[0, 0] == U.encode(np.array([[1.0] + [0.0] * 63]), 64)[1][0, 0] and list(c[0][1:3]) == [127, 255]


def test_sizes_past_a_launch_are_refused():
    """Sizes whose pointers and strides are sound but whose threads do not fit one launch."""
    lib, far, big = mt.load(), 1 << 44, 1 << 28
    kv, long, dst = kv_struct(hkv=1), kv_struct(hkv=1, cache_len=4096), kv_struct(base=256 * MB, hkv=1)
    calls = [
        lambda: lib.mt_rope_append(far, 192, 1, big, 1, 1, None, None, 0, ref(kv), A, None, 0, None),
        lambda: lib.mt_kv_copy(ref(kv), ref(dst), 1, big, 1, None, None, None),
        lambda: lib.mt_attention_shared(far, 64, 1, big, 1, 1, None, None, ref(long), None, 0, 0, 0, 2 * far, 64, 0.125, None, 0, None),
        lambda: lib.mt_quantize_f8(far, mt.F16, 1 << 27, 16, 16, None, mt.F16, 1e-6, 2 * far, 16, 3 * far, 4, None),
        lambda: lib.mt_quantize_f8(far, mt.F16, 1 << 25, 16, 16, A, mt.F16, 1e-6, 2 * far, 16, 3 * far, 4, None),
        lambda: lib.mt_linear_f8(A, mt.F32, None, 0, None, far, 2 * far, None, None, None, mt.F16, 3 * far,
                                 mt.GemvParams(1, 1 << 30, 16, 16, 1 << 30, 0, 0.0), None),
        lambda: lib.mt_linear_f8(far, mt.F8, 2 * far, 4, None, 3 * far, 4 * far, None, None, None, mt.F16, 5 * far,
                                 mt.GemvParams(1 << 28, 1024, 16, 16, 1024, 0, 0.0), None),
    ]
    for c in calls:
        assert c() == mt.EINVAL
        assert "too many" in mt.last_error(), mt.last_error()
