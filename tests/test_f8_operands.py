"""What the Python calls of the 8-bit and shared-prefix operators refuse before they pass an address on, and what they take,
without a GPU: a call whose operands are accepted gets as far as asking for the stream."""
import pytest
import torch

import mingtts as mt


class Reached(Exception):
    pass


@pytest.fixture(autouse=True)
def no_launch(monkeypatch):
    def on(device, stream):
        raise Reached

    monkeypatch.setattr(mt, "_on", on)


z = torch.zeros
B, T, HQ, HKV, CAP, K, N = 3, 2, 4, 2, 8, 48, 24


def i32(*shape):
    return z(*shape, dtype=torch.int32)


def caches(batch=B):
    c, s = z(batch, HKV, CAP, 64, dtype=torch.uint8), z(batch, HKV, CAP, dtype=torch.uint8)
    return mt.KV(c, c.clone(), s, s.clone())


def append(**over):
    a = dict(qkv=z(B * T, 512), B=B, T=T, hq=HQ, hkv=HKV, pos=i32(B), kv=caches(), inv_freq=z(32), q=z(B * T, 256), counts=i32(B))
    mt.rope_append(**{**a, **over})


def copy(**over):
    a = dict(src=caches(), dst=caches(), B=B, T=T, pos=i32(B), counts=i32(B))
    mt.kv_copy(**{**a, **over})


def attend(**over):
    a = dict(q=z(B * T, 256), B=B, T=T, hq=HQ, hkv=HKV, pos=i32(B), kv=caches(), out=z(B * T, 256), counts=i32(B))
    mt.attention_shared(**{**a, **over})


def matrix(rows=N):
    return mt.F8Matrix(z(rows, K, dtype=torch.uint8), z(rows, 4, dtype=torch.uint8))


def linear(**over):
    a = dict(x=z(4, K), w=matrix(), y=z(4, N))
    mt.linear_f8(**{**a, **over})


def quantize(**over):
    a = dict(x=z(N, K), out=matrix())
    mt.quantize_f8(**{**a, **over})


CALLS = [append, copy, attend, linear, quantize]


@pytest.mark.parametrize("call", CALLS)
def test_the_plain_calls_are_taken(call):
    with pytest.raises(Reached):
        call()


@pytest.mark.parametrize("call", [append, copy, attend])
@pytest.mark.parametrize("name", ["pos", "counts"])
@pytest.mark.parametrize("bad", [z(B), z(B, dtype=torch.int64), i32(B - 1), i32(2 * B)[::2], i32(B, 2)[:, 0]],
                         ids=["fp32", "int64", "short", "strided", "column"])
def test_positions_and_counts(call, name, bad):
    with pytest.raises(ValueError, match="int32"):
        call(**{name: bad})


@pytest.mark.parametrize("call", [append, copy, attend])
@pytest.mark.parametrize("good", [None, i32(B + 2), i32(B, 1), z(B, dtype=torch.uint32), i32(9)[3:]], ids=str)
def test_positions_and_counts_that_are_taken(call, good):
    with pytest.raises(Reached):
        call(pos=good, counts=good)


# A row operand: its call, its name, and the rows and columns that the call reads or writes.
ROWS = [(append, "qkv", B * T, 512), (append, "q", B * T, 256), (attend, "q", B * T, 256), (attend, "out", B * T, 256),
        (linear, "y", 4, N)]


@pytest.mark.parametrize("call,name,rows,width", ROWS)
def test_rows(call, name, rows, width):
    bad = [z(rows - 1, width), z(rows, width - 1), z(rows, 2 * width)[:, ::2], z(width, rows).t(), z(rows * width - 1),
           z(2, rows // 2, width - 1), z(2, rows, width)[:, ::2, 1:], z(rows // 2, 2, width).transpose(0, 1), z(())]
    for t in bad:
        with pytest.raises(ValueError, match="rows of"):
            call(**{name: t})
    for t in (z(rows, width, dtype=torch.float16), z(rows, width, dtype=torch.int32), z(rows, width, dtype=torch.float64)):
        with pytest.raises(ValueError, match="fp32"):
            call(**{name: t})


@pytest.mark.parametrize("call,name,rows,width", ROWS)
def test_rows_that_are_taken(call, name, rows, width):
    for t in (z(rows + 1, width + 4), z(rows, 2 * width)[:, :width], z(2 * rows, width)[::2], z(2, rows // 2, width),
              z(2, rows // 2, 2 * width)[:, :, :width], z(rows, 1, width), z(1, rows, 2 * width)[..., width:]):
        with pytest.raises(Reached):
            call(**{name: t})


@pytest.mark.parametrize("call,name,rows,width,ld", [r + (ld,) for r, ld in zip(ROWS, ("ldq", "ldo", "ldq", "ldo", "ldy"))])
def test_rows_at_a_given_stride(call, name, rows, width, ld):
    """A tensor of any shape, from its first element on."""
    most = (rows - 1) * (width + 4) + width
    for t in (z(most), z(rows, width + 4), z(most + 5)[5:], z(2, rows, width)):
        with pytest.raises(Reached):
            call(**{name: t, ld: width + 4})
    for t in (z(most - 1), z(most + 5)[6:], z(rows, width)):
        with pytest.raises(ValueError, match="rows of"):
            call(**{name: t, ld: width + 4})


@pytest.mark.parametrize("bad", [z(31), z(64)[::2], z(32, dtype=torch.float64), z(32, dtype=torch.int32)], ids=["short", "strided", "fp64", "int32"])
def test_frequencies(bad):
    with pytest.raises(ValueError, match="32 fp32"):
        append(inv_freq=bad)


def h16(*shape):
    return z(*shape, dtype=torch.float16)


@pytest.mark.parametrize("call,name,n", [(linear, "bias", N), (linear, "norm", K), (quantize, "norm", K)])
def test_vectors(call, name, n):
    for t in (h16(2 * n)[::2], h16(n, 2)[:, 0], h16(n - 1), h16(1).expand(n)):
        with pytest.raises(ValueError, match="values"):
            call(**{name: t})
    for t in (h16(n), h16(n + 8), h16(2 * n)[n:]):
        with pytest.raises(Reached):
            call(**{name: t})


@pytest.mark.parametrize("rows", [4, 20])  # quantised on the way in, and by a call before
def test_a_strided_norm_of_many_rows(rows):
    with pytest.raises(ValueError, match="values"):
        linear(x=z(rows, K), y=z(rows, N), norm=h16(2 * K)[::2])


def test_a_prefix_length_without_a_prefix():
    with pytest.raises(ValueError, match="prefix"):
        attend(prefix_len=5)
    one = mt.KV(*[t[0] for t in (caches().k, caches().v, caches().k_scale, caches().v_scale)])
    for over in (dict(prefix_len=0), dict(prefix=one), dict(prefix=one, prefix_len=5)):
        with pytest.raises(Reached):
            attend(**over)


@pytest.mark.parametrize("bad", [z(1 << 21, dtype=torch.uint8)[::2], z(1 << 10, 1 << 12, dtype=torch.uint8)[:, :1 << 11]], ids=["strided", "columns"])
def test_a_workspace_that_is_not_one_run(bad):
    with pytest.raises(ValueError, match="workspace"):
        attend(workspace=bad)


def test_a_workspace_on_another_device():
    """(a host tensor stands for the caches' device here, so this one says that it is elsewhere)"""
    class Elsewhere(torch.Tensor):
        def get_device(self):
            return 1

    with pytest.raises(ValueError, match="workspace"):
        attend(workspace=z(1 << 20, dtype=torch.uint8).as_subclass(Elsewhere))
    for good in (z(1 << 20, dtype=torch.uint8), z(1 << 18)):
        with pytest.raises(Reached):
            attend(workspace=good)


def test_scales_that_end_before_their_last_rows_stride():
    """mt_quantize_f8 clears a row's bytes up to its stride, the last row's too."""
    wide = z(N, 8, dtype=torch.uint8)
    codes = z(N, K, dtype=torch.uint8)
    with pytest.raises(ValueError, match="stride"):
        quantize(out=mt.F8Matrix(codes, wide[:, 4:]))
    with pytest.raises(ValueError, match="stride"):
        quantize(out=mt.F8Matrix(codes[1:], wide[1:, 4:]), x=z(N - 1, K))
    for out, n in ((mt.F8Matrix(codes, wide[:, :4]), N), (mt.F8Matrix(codes[1:], wide[:-1, 4:]), N - 1)):
        with pytest.raises(Reached):
            quantize(out=out, x=z(n, K))


def test_a_matrix_of_no_rows(monkeypatch):
    """Nothing to do, as in the C call."""
    monkeypatch.setattr(mt, "_on", lambda device, stream: 0)
    for k in (K, 1024):
        m = mt.F8Matrix.quantize(z(0, k))
        assert m.shape == (0, k) and tuple(m.scales.shape) == (0, 4 * ((k + 511) // 512))


@pytest.mark.parametrize("call,name,rows,width", ROWS)
def test_rows_of_several_dimensions(call, name, rows, width):
    """Heads as a dimension of their own, slices of wider rows, both with leading dimensions of their own."""
    h = width // 8
    wide = z(2, rows // 2, 12, h)
    for t in (z(rows, 8, h), z(2, rows // 2, 8, h), wide[:, :, :8], wide[:, :, 4:], z(rows, 12, h)[:, 2:10], z(rows, 1, 8, h)):
        with pytest.raises(Reached):
            call(**{name: t})
    for t in (z(rows, 7, h), z(rows, 8, 2 * h)[:, :, :h], z(rows, h, 8).transpose(1, 2), z(8, rows, h).transpose(0, 1), z(rows - 1, 8, h),
              z(rows, 0, h)):
        with pytest.raises(ValueError, match="rows of"):
            call(**{name: t})
