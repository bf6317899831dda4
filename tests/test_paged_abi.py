"""The paged and windowed entry points without a GPU: refusals before any HIP call, calls without work, and what the
Python classes and calls check."""
import ctypes
import os
import subprocess
import sys

import pytest
import torch

import mingtts as mt

A = 1 << 20  # fake aligned device addresses, never dereferenced
MB = 1 << 20


def paged(base=A, hkv=2, page_len=16, t=mt.F8, **over):
    f = dict(k=base, v=base + 64 * MB, k_scale=base + 128 * MB, v_scale=base + 129 * MB, stride=hkv * page_len * 64,
             scale_stride=hkv * page_len, table=base + 130 * MB, pages=100, page_len=page_len, table_len=8, table_stride=8, cache_t=t)
    f.update(over)
    return mt.PagedKvStruct(*[f[n] for n, _ in mt.PagedKvStruct._fields_])


def contiguous(base=A, hkv=2, cache_len=64, t=mt.F8, **over):
    f = dict(k=base, v=base + 64 * MB, k_scale=base + 128 * MB, v_scale=base + 129 * MB, stride=hkv * cache_len * 64,
             scale_stride=hkv * cache_len, cache_len=cache_len, cache_t=t)
    f.update(over)
    return mt.KvStruct(*[f[n] for n, _ in mt.KvStruct._fields_])


def ref(s):
    return ctypes.byref(s) if s is not None else None


def append(kv, qkv=1024 * MB, ldq=18 * 64, B=4, T=1, hq=14, hkv=2, inv_freq=A, q=1536 * MB, ldo=14 * 64):
    return mt.load().mt_rope_append_paged(qkv, ldq, B, T, hq, hkv, None, None, 0, ref(kv), inv_freq, q, ldo, None)


def attend(kv, q=1024 * MB, ldq=896, B=4, T=1, hq=14, hkv=2, len_max=0, window=0, sinks=0, out=1536 * MB, ldo=896, ws=None, wsn=0):
    f = mt.load().mt_attention_paged if isinstance(kv, mt.PagedKvStruct) or kv is None else mt.load().mt_attention_sinks
    return f(q, ldq, B, T, hq, hkv, None, None, ref(kv), len_max, window, sinks, out, ldo, 0.125, ws, wsn, None)


CACHES = [
    (dict(t=mt.BF16), "f32, f16 or f8"),
    (dict(cache_t=9), "f32, f16 or f8"),
    (dict(k=0), "null k, v or table"),
    (dict(table=0), "null k, v or table"),
    (dict(v=A + 8), "16-byte"),
    (dict(table=A + 130 * MB + 2), "4-byte aligned"),
    (dict(pages=0), "no pages"),
    (dict(page_len=0), "page_len"),
    (dict(page_len=24), "page_len"),
    (dict(page_len=32784, stride=1 << 24), "page_len"),
    (dict(table_len=0), "entries"),
    (dict(table_len=(1 << 26) + 1, table_stride=1 << 27), "entries"),
    (dict(table_stride=7), "table_stride"),
    (dict(stride=64), "stride"),
    (dict(stride=2 * 16 * 64 + 8), "stride"),
    (dict(stride=1 << 60), "stride"),
    (dict(k_scale=0), "null scales"),
    (dict(v_scale=A + 1), "4-byte aligned"),
    (dict(scale_stride=16), "scale_stride"),
    (dict(scale_stride=34), "scale_stride"),
]


@pytest.mark.parametrize("kv,needle", CACHES)
def test_caches_are_refused(kv, needle):
    for call in (append, attend):
        assert call(paged(**kv)) == mt.EINVAL
        assert needle in mt.last_error(), mt.last_error()


@pytest.mark.parametrize("kv,call,needle", [
    (dict(v=A), {}, "overlap each other"),
    (dict(table=A + 64 * MB), {}, "overlap each other"),
    (dict(), dict(qkv=0), "null pointer"),
    (dict(), dict(inv_freq=0), "null pointer"),
    (dict(), dict(ldq=17 * 64), "ldq"),
    (dict(), dict(ldo=13 * 64), "ldo"),
    (dict(), dict(qkv=1024 * MB + 4), "16-byte aligned"),
    (dict(), dict(q=1024 * MB), "overlaps qkv"),
    (dict(k=1024 * MB), {}, "overlap qkv"),
    (dict(table=1536 * MB + 64), {}, "overlap qkv or q"),
    (dict(), dict(hkv=0), "hkv"),
    (dict(), dict(B=1 << 16, T=1 << 16), "too many"),
])
def test_append_refuses(kv, call, needle):
    assert append(paged(**kv), **call) == mt.EINVAL
    assert needle in mt.last_error(), mt.last_error()


@pytest.mark.parametrize("make", [paged, contiguous])
@pytest.mark.parametrize("kv,call,needle", [
    (dict(), dict(hq=13), "multiple of hkv"),
    (dict(), dict(hq=0), "multiple of hkv"),
    (dict(), dict(q=0), "null pointer"),
    (dict(), dict(out=0), "null pointer"),
    (dict(), dict(ldq=64), "ldq / ldo"),
    (dict(), dict(out=1536 * MB + 8), "16-byte aligned"),
    (dict(), dict(ldo=898), "16-byte row strides"),
    (dict(), dict(out=1024 * MB + 896 * 4), "out overlaps q"),
    (dict(), dict(out=A), "out overlaps the caches"),
    (dict(t=mt.BF16), {}, "f32, f16 or f8"),
    (dict(), dict(hq=8194), "too many"),
    (dict(), dict(B=1 << 20, T=100, hq=16, hkv=1, ldq=1024), "too many"),
])
def test_attention_refuses(make, kv, call, needle):
    assert attend(make(**kv), **call) == mt.EINVAL
    assert needle in mt.last_error(), mt.last_error()


def test_null_caches():
    assert append(None) == mt.EINVAL and "null kv" in mt.last_error()
    assert attend(None) == mt.EINVAL and "null kv" in mt.last_error()
    assert mt.load().mt_attention_sinks(A, 896, 1, 1, 14, 2, None, None, None, 0, 0, 0, 2 * A, 896, 0.125, None, 0, None) == mt.EINVAL


def test_no_rows_is_no_call():
    for B, T in ((0, 1), (3, 0)):
        assert append(paged(), B=B, T=T) == mt.OK and attend(paged(), B=B, T=T) == mt.OK and attend(contiguous(), B=B, T=T) == mt.OK


def test_interleaved_pools_are_taken_apart():
    """Keys and values of one pool, page by page, do not meet; half a page on they do."""
    rows = 2 * 16 * 64
    kv = paged(t=mt.F16, v=A + 2 * rows, stride=2 * rows, pages=100)
    assert append(kv, inv_freq=0) == mt.EINVAL and "null pointer" in mt.last_error()
    assert append(kv, hq=0, ldq=256, q=0, qkv=A + 2 * rows * 2 * 50) == mt.EINVAL and "overlap qkv" in mt.last_error()
    assert append(paged(t=mt.F16, v=A + rows, stride=2 * rows)) == mt.EINVAL and "overlap each other" in mt.last_error()


@pytest.mark.parametrize("make", [paged, contiguous])
def test_small_workspaces_are_refused(make):
    L = mt.load()
    kv = make(table_len=8192, table_stride=8192) if make is paged else make(cache_len=1 << 17)
    need = L.mt_attention_window_workspace(1, 1, 14, 2, 1 << 17, 0, 0, mt.F8)
    if need == 0:
        pytest.skip("this size is not split")
    for ws, n in ((None, need), (A, need - 1), (A + 8, need)):
        assert attend(kv, B=1, ws=ws, wsn=n) == mt.EINVAL and "workspace" in mt.last_error()


APPEND = """
import ctypes, sys
sys.path[:0] = %r
import mingtts as mt
import test_paged_abi as t
L, rows, heads = mt.load(), int(sys.argv[1]), int(sys.argv[2])
kv = t.paged() if sys.argv[3] == "paged" else t.contiguous()
call = L.mt_rope_append_paged if sys.argv[3] == "paged" else L.mt_rope_append
a = (1 << 50, heads * 64, 1, rows, heads - 4, 2, None, None, 0, ctypes.byref(kv), t.A, None, 0, None)
rc = call(*a)
print(rc, mt.last_error())
"""


@pytest.mark.parametrize("which", ["paged", "contiguous"])
@pytest.mark.parametrize("rows,heads", [(30_000_000, 64), (33_000_000, 18), (33_000_000, 20), (8_400_000, 255)])
def test_many_rows_are_no_refusal(which, rows, heads):
    """Appends of as many rows as 256 threads for two rows hold, by a process that sees no device: the launch fails, not the sizes."""
    here = os.path.dirname(os.path.abspath(__file__))
    code = APPEND % [here, os.path.join(os.path.dirname(here), "ming-tts_amd")]
    env = {**os.environ, "HIP_VISIBLE_DEVICES": "-1", "ROCR_VISIBLE_DEVICES": "-1"}
    out = subprocess.run([sys.executable, "-c", code, str(rows), str(heads), which], env=env, capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stderr
    rc = int(out.stdout.split()[0])
    assert rc < 0 and rc != mt.EINVAL, out.stdout


@pytest.mark.parametrize("make", [paged, contiguous])
@pytest.mark.parametrize("ws", [1024 * MB, 1536 * MB, A + 1 * MB, A + 65 * MB, A + 128 * MB, "table"])
def test_workspaces_lie_apart(make, ws):
    L = mt.load()
    kv = make(table_len=8192, table_stride=8192, pages=8192) if make is paged else make(cache_len=1 << 17)
    need = L.mt_attention_window_workspace(1, 1, 14, 2, 1 << 17, 0, 0, mt.F8)
    assert need > 0
    if ws == "table":
        if make is contiguous:
            return
        ws = A + 130 * MB + 8192 * 4 - 16
    assert attend(kv, B=1, ws=ws, wsn=need) == mt.EINVAL and "workspace overlaps" in mt.last_error()


# ------------------------------------------------------------- Python --

class Reached(Exception):
    pass


@pytest.fixture
def no_launch(monkeypatch):
    def on(device, stream):
        raise Reached

    monkeypatch.setattr(mt, "_on", on)


z = torch.zeros


def i32(*shape):
    return z(*shape, dtype=torch.int32)


def pages(**over):
    c, s = z(9, 2, 16, 64, dtype=torch.uint8), z(9, 2, 16, dtype=torch.uint8)
    return mt.PagedKV(**{**dict(k=c, v=c.clone(), table=i32(3, 4), k_scale=s, v_scale=s.clone()), **over})


@pytest.mark.parametrize("over,needle", [
    (dict(v=z(9, 2, 32, 64, dtype=torch.uint8)), "one shape"),
    (dict(v=z(9, 2, 16, 64)), "one shape"),
    (dict(v_scale=None), "one shape"),
    (dict(k=z(9, 2, 16, 32), v=z(9, 2, 16, 32)), "heads of 64"),
    (dict(k=z(9, 2, 16, 64, dtype=torch.bfloat16), v=z(9, 2, 16, 64, dtype=torch.bfloat16)), "heads of 64"),
    (dict(k=z(2, 16, 64), v=z(2, 16, 64)), "contiguous but for the pages"),
    (dict(k=z(0, 2, 16, 64), v=z(0, 2, 16, 64)), "contiguous but for the pages"),
    (dict(k=z(9, 16, 2, 64).transpose(1, 2), v=z(9, 16, 2, 64).transpose(1, 2)), "contiguous but for the pages"),
    (dict(k_scale=z(9, 2, 15, dtype=torch.uint8), v_scale=z(9, 2, 15, dtype=torch.uint8)), "one scale byte"),
    (dict(table=z(3, 4)), "table"),
    (dict(table=z(3, 4, dtype=torch.int64)), "table"),
    (dict(table=i32(12)), "table"),
    (dict(table=i32(4, 3).T), "table"),
    (dict(table=i32(3, 4).to("meta")), "one device"),
])
def test_pools_are_refused(over, needle):
    with pytest.raises(ValueError, match=needle):
        pages(**over)


def py_append(**over):
    a = dict(qkv=z(6, 512), B=3, T=2, hq=4, hkv=2, pos=i32(3), kv=pages(), inv_freq=z(32), q=z(6, 256), counts=i32(3))
    mt.rope_append_paged(**{**a, **over})


def py_paged(**over):
    a = dict(q=z(6, 256), B=3, T=2, hq=4, hkv=2, pos=i32(3), kv=pages(), out=z(6, 256), counts=i32(3))
    mt.attention_paged(**{**a, **over})


def flat():
    c, s = z(3, 2, 8, 64, dtype=torch.uint8), z(3, 2, 8, dtype=torch.uint8)
    return mt.KV(c, c.clone(), s, s.clone())


def py_sinks(**over):
    py_paged_args = dict(q=z(6, 256), B=3, T=2, hq=4, hkv=2, pos=i32(3), kv=flat(), out=z(6, 256), counts=i32(3))
    mt.attention_sinks(**{**py_paged_args, **over})


CALLS = [py_append, py_paged, py_sinks]


@pytest.mark.parametrize("call", CALLS)
def test_plain_calls_are_taken(call, no_launch):
    for over in (dict(), dict(pos=None, counts=None), dict(pos=z(3, dtype=torch.uint32))):
        with pytest.raises(Reached):
            call(**over)


@pytest.mark.parametrize("call", CALLS)
def test_operands_are_refused(call, no_launch):
    other = flat() if call is not py_sinks else pages()
    for over, needle in ((dict(pos=z(3)), "int32"), (dict(counts=i32(2)), "int32"), (dict(pos=i32(6)[::2]), "int32"),
                         (dict(B=4), "sequences"), (dict(hkv=1), "heads"), (dict(kv=other), "takes a"),
                         (dict(T=3), "rows of")):
        with pytest.raises(ValueError, match=needle):
            call(**over)


@pytest.mark.parametrize("call", [py_paged, py_sinks])
def test_workspaces_are_refused(call, no_launch):
    with pytest.raises(ValueError, match="workspace"):
        call(workspace=z(8, 8)[:, ::2])


def test_one_page_and_one_table_row():
    """Strides that torch does not keep: those of a dimension of one."""
    kv = pages(k=z(1, 2, 16, 64, dtype=torch.uint8), v=z(1, 2, 16, 64, dtype=torch.uint8), k_scale=z(1, 2, 16, dtype=torch.uint8),
               v_scale=z(1, 2, 16, dtype=torch.uint8), table=i32(1, 1))
    assert (kv.struct.stride, kv.struct.scale_stride, kv.cache_len, kv.batch) == (2048, 32, 16, 1)
