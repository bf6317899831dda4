"""mt_quantize_f8 and mt_linear_f8 against 64 bits."""
import numpy as np
import pytest
import torch

import mingtts as mt
import _f8_util as U
from _gpu_util import say

pytestmark = pytest.mark.gpu
F = mt.GemvFlags
XT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def matrix(w, gpu):
    """An F8Matrix of w by the definition, and its values in 64 bits."""
    n, k = w.shape
    c, s = U.encode(w, 128)
    lds = 4 * ((k + 511) // 512)
    sb = np.zeros((n, lds), np.uint8)
    sb[:, :s.shape[1]] = s
    return mt.F8Matrix(torch.from_numpy(c).to(gpu), torch.from_numpy(sb).to(gpu)), U.decode(c, s, 128)


@pytest.mark.parametrize("xt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,k", [(1, 16), (3, 128), (5, 144), (2, 896), (7, 4864), (33, 1040)])
def test_quantize(gpu, xt, rows, k):
    say(f"quantize {xt} {rows}x{k}")
    rng = np.random.default_rng(rows * k)
    x = rng.standard_normal((rows, k)) * 10.0 ** rng.uniform(-6, 6, (rows, 1))
    t = torch.from_numpy(x).to(XT[xt])
    wide = torch.zeros(rows, k + 48, dtype=XT[xt], device=gpu)
    wide[:, :k] = t.to(gpu)
    codes = torch.full((rows + 1, k + 32), 9, dtype=torch.uint8, device=gpu)
    lds = 4 * ((k + 511) // 512)
    scales = torch.full((rows + 1, lds + 4), 9, dtype=torch.uint8, device=gpu)
    out = mt.F8Matrix(codes[:rows, :k], scales[:rows, :lds])
    mt.quantize_f8(wide[:, :k], out)
    c, s = U.encode(t.double().numpy(), 128)
    assert np.array_equal(out.codes.cpu().numpy(), c)
    assert np.array_equal(out.scales.cpu().numpy()[:, :s.shape[1]], s)
    assert bool((codes[rows] == 9).all()) and bool((codes[:, k:] == 9).all()) and bool((scales[rows] == 9).all())
    # the row's remaining bytes, up to its stride, are padding
    assert bool((scales[:rows, s.shape[1]:] == 0).all())


def test_quantize_special_values(gpu):
    x = np.zeros((4, 256), np.float32)
    x[0, :4] = [np.inf, 1.0, np.nan, -np.inf]
    x[1] = 2.0 ** -140
    x[2, 5], x[2, 200] = 3.4e38, 1e-38
    m = mt.F8Matrix.quantize(torch.from_numpy(x).to(gpu))
    c, s = U.encode(x.astype(np.float64), 128)
    got, nan = m.codes.cpu().numpy(), (c & 127) == 127
    assert np.array_equal(m.scales.cpu().numpy()[:, :2], s)
    assert np.array_equal(got[~nan], c[~nan]) and ((got[nan] & 127) == 127).all()


@pytest.mark.parametrize("nt", ["f16", "bf16"])
@pytest.mark.parametrize("rows,k", [(1, 16), (9, 896), (3, 4864), (2, 20000)])
def test_quantize_norm(gpu, nt, rows, k):
    rng = np.random.default_rng(k)
    x = rng.standard_normal((rows, k)).astype(np.float32) * 3
    g = torch.from_numpy(1 + 0.1 * rng.standard_normal(k)).to(XT[nt])
    m = mt.F8Matrix.quantize(torch.from_numpy(x).to(gpu), norm=g.to(gpu), eps=1e-5)
    x64 = x.astype(np.float64)
    want = x64 / np.sqrt((x64 ** 2).mean(1, keepdims=True) + 1e-5) * g.double().numpy()
    s = m.scales.cpu().numpy()
    got = U.decode(m.codes.cpu().numpy(), s, 128)
    step = np.repeat(2.0 ** (s.astype(float) - 127), 128, -1)[:, :k] * 2.0 ** -10
    # half a step of the format, and the fp32 arithmetic before it (a row's sum of squares in pieces of 8, 16 lanes
    # and K / 2048 blocks, a square root, a division, two products: under 40 roundings)
    assert (np.abs(got - want) <= np.maximum(np.abs(want) * 2.0 ** -4, step) + 40 * U.EPS32 * np.abs(want)).all()


def epilogue64(y, u, bias, flags, old):
    if bias is not None:
        y = y + bias
    if flags & F.siluGate:
        y = y / (1 + np.exp(-y)) * u
    if flags & F.gelu:
        y = 0.5 * y * (1 + np.tanh(0.7978845608028654 * (y + 0.044715 * y ** 3)))
    if flags & F.silu:
        y = y / (1 + np.exp(-y))
    return y + old if flags & F.accumulate else y


def run_linear(gpu, M, N, K, flags=0, xt="f32", bias=None, quantized=False, norm=None, pad=0, seed=0):
    rng = np.random.default_rng(M * 7 + N * 3 + K + seed)
    x = torch.from_numpy(rng.standard_normal((M, K)).astype(np.float32)).to(XT[xt])
    w, w64 = matrix(rng.standard_normal((N, K)) * 0.05, gpu)
    w2, u64 = matrix(rng.standard_normal((N, K)) * 0.05, gpu) if flags & F.siluGate else (None, None)
    b = torch.from_numpy(rng.standard_normal(N)).to(XT[bias]) if bias else None
    y = torch.full((M + 1, N + pad), 0.5, device=gpu)
    old = rng.standard_normal((M, N)).astype(np.float32)
    y[:M, :N] = torch.from_numpy(old).to(gpu)
    xd = torch.zeros(M, K + 16 * (pad > 0), dtype=XT[xt], device=gpu)
    xd[:, :K] = x.to(gpu)
    xd = xd[:, :K]
    x64 = U.decode(*U.encode(x.double().numpy(), 128), 128)
    if quantized:
        xd = mt.F8Matrix.quantize(xd)
    mt.linear_f8(xd, w, y, M=M, flags=flags, w2=w2, bias=b.to(gpu) if bias else None, ldy=N + pad)
    got = y.cpu().numpy()
    assert (got[M] == 0.5).all() and (got[:, N:] == 0.5).all()
    got = got[:M, :N]
    acc, u = x64 @ w64.T, None
    # Exact products; the sums take K / 16 + 64 roundings in whatever order (a matrix instruction's may be towards
    # zero: whole steps).
    r = (K / 16 + 64) * 2 * U.EPS32
    tol = r * (np.abs(x64) @ np.abs(w64).T)
    if flags & F.siluGate:
        u = x64 @ u64.T
        z = acc + (b.double().numpy() if bias else 0)
        tol = 1.1 * tol * np.abs(u) + np.abs(z / (1 + np.exp(-z))) * r * (np.abs(x64) @ np.abs(u64).T)
    else:
        tol = 1.2 * tol  # the slope of GELU and SiLU is at most 1.13
    want = epilogue64(acc, u, b.double().numpy() if bias else None, flags, old)
    # bias, activation (a few hardware roundings of values around 1) and the accumulation
    tol = tol + 16 * U.EPS32 * (np.abs(want) + np.abs(acc) * (1 + (np.abs(u) if u is not None else 0)) + np.abs(old) + 1)
    assert np.isfinite(got).all()
    worst = (np.abs(got - want) / tol).max()
    assert worst <= 1, f"{worst:.3g} of the bound"
    rel = np.linalg.norm(got - want) / np.linalg.norm(want)
    assert rel <= 3e-6, rel
    return got


@pytest.mark.parametrize("xt,quantized", [("f32", False), ("f16", False), ("bf16", False), ("f32", True)])
@pytest.mark.parametrize("M,N,K", [(1, 16, 16), (1, 896, 4864), (2, 1152, 896), (3, 17, 144), (5, 40, 4096), (16, 896, 4864), (16, 7, 1008),
                                   (13, 1, 2064), (8, 130, 12800)])
def test_few_rows(gpu, M, N, K, xt, quantized):
    say(f"few rows {M}x{N}x{K} {xt} {quantized}")
    run_linear(gpu, M, N, K, xt=xt, quantized=quantized, pad=4)


@pytest.fixture(params=[0, 1, 2, 3, 4])
def tile(request):
    """The call's own choice, then each of the GEMM's tiles by force."""
    mt.set_tuning(mt.TUNE_F8_TILE, request.param)
    yield request.param
    mt.set_tuning(mt.TUNE_F8_TILE, -1)


@pytest.mark.parametrize("M,N,K", [(17, 16, 16), (17, 64, 128), (31, 1152, 896), (64, 100, 176), (65, 129, 1040), (128, 896, 4864), (200, 333, 640),
                                   (257, 255, 512), (300, 1000, 2064), (512, 640, 896), (600, 16, 1024)])
def test_many_rows(gpu, tile, M, N, K):
    say(f"many rows {M}x{N}x{K}")
    run_linear(gpu, M, N, K)
    run_linear(gpu, M, N, K, pad=4, xt="bf16", seed=1)


FLAGS = [F.gelu, F.silu, F.accumulate, F.siluGate, F.siluGate | F.accumulate, F.gelu | F.accumulate]


@pytest.mark.parametrize("bias", [None, "f16", "bf16"])
@pytest.mark.parametrize("flags", FLAGS)
@pytest.mark.parametrize("M,N,K", [(2, 100, 896), (70, 200, 272), (140, 131, 144)])
def test_epilogues(gpu, tile, M, N, K, flags, bias):
    if M <= 16 and tile:
        pytest.skip("no GEMM")
    say(f"epilogue {M}x{N}x{K} {flags} {bias}")
    run_linear(gpu, M, N, K, flags=flags, bias=bias, pad=3)


@pytest.mark.parametrize("M", [1, 4, 16])
@pytest.mark.parametrize("K", [896, 4864, 20000])
def test_the_norm_on_the_way_gives_the_quantised_rows(gpu, M, K):
    """x normalised and quantised inside the call enters as mt_quantize_f8's bytes: the same product bit for bit."""
    rng = np.random.default_rng(M + K)
    x = torch.from_numpy(rng.standard_normal((M, K)).astype(np.float32)).to(gpu)
    g = torch.from_numpy(1 + 0.2 * rng.standard_normal(K)).to(torch.bfloat16).to(gpu)
    w, _ = matrix(rng.standard_normal((80, K)) * 0.05, gpu)
    a, b = torch.zeros(M, 80, device=gpu), torch.zeros(M, 80, device=gpu)
    mt.linear_f8(x, w, a, norm=g, eps=1e-5)
    mt.linear_f8(mt.F8Matrix.quantize(x, norm=g, eps=1e-5), w, b)
    assert torch.equal(a, b)


@pytest.mark.parametrize("M", [3, 80])
def test_scales_far_apart_and_nan_rows(gpu, M):
    """Blocks whose scales differ by 2^60 and more: each output keeps its own size.  A NaN stays in its row and
    its feature."""
    rng = np.random.default_rng(5)
    K, N = 512, 48
    x = rng.standard_normal((M, K)) * np.repeat(2.0 ** np.array([-40, 0, 20, -90]), 128)
    w = rng.standard_normal((N, K)) * np.repeat(2.0 ** np.array([40, 0, -20, 90]), 128)
    wm, w64 = matrix(w, gpu)
    x32 = x.astype(np.float32)
    y = torch.zeros(M, N, device=gpu)
    mt.linear_f8(torch.from_numpy(x32).to(gpu), wm, y)
    x64 = U.decode(*U.encode(x32.astype(np.float64), 128), 128)
    assert (np.abs(y.cpu().numpy() - x64 @ w64.T) <= (K / 16 + 64) * 2 * U.EPS32 * (np.abs(x64) @ np.abs(w64).T)).all()
    x32[1, 7] = np.nan
    wm.codes[9, 300] = 127
    y2 = torch.zeros(M, N, device=gpu)
    mt.linear_f8(torch.from_numpy(x32).to(gpu), wm, y2)
    y2, nan = y2.cpu().numpy(), np.zeros((M, N), bool)
    nan[1], nan[:, 9] = True, True
    assert np.isnan(y2[nan]).all() and np.array_equal(y2[~nan], y.cpu().numpy()[~nan])


@pytest.mark.parametrize("M", [2, 100])
@pytest.mark.parametrize("K", [144, 640, 1040])
def test_padding_scale_bytes_are_not_read(gpu, tile, M, K):
    """The bytes behind a row's last block, up to the next multiple of four, may be anything."""
    rng = np.random.default_rng(4)
    w, _ = matrix(rng.standard_normal((70, K)) * 0.05, gpu)
    x = mt.F8Matrix.quantize(torch.from_numpy(rng.standard_normal((M, K)).astype(np.float32)).to(gpu))
    a, b = torch.zeros(M, 70, device=gpu), torch.zeros(M, 70, device=gpu)
    mt.linear_f8(x, w, a)
    n = (K + 127) // 128
    for m in (x, w):
        m.scales[:, n:] = 255
    mt.linear_f8(x, w, b)
    assert torch.equal(a, b)


@pytest.mark.parametrize("M", [2, 100])
def test_graph_and_streams(gpu, M):
    """Replays see new inputs; two streams at once give the bits of one after the other."""
    rng = np.random.default_rng(6)
    w, _ = matrix(rng.standard_normal((300, 896)) * 0.05, gpu)
    xs = [torch.from_numpy(rng.standard_normal((M, 896)).astype(np.float32)).to(gpu) for _ in range(5)]
    want = []
    for x in xs:
        y = torch.zeros(M, 300, device=gpu)
        mt.linear_f8(x, w, y)
        want.append(y)
    x, y = xs[0].clone(), torch.zeros(M, 300, device=gpu)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mt.linear_f8(x, w, y)
    for a, b in zip(xs, want):
        x.copy_(a)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, b)
    streams = [torch.cuda.Stream() for _ in range(2)]
    ys = [torch.zeros(M, 300, device=gpu) for _ in xs]
    torch.cuda.synchronize()
    for i, a in enumerate(xs):
        mt.linear_f8(a, w, ys[i], stream=streams[i % 2])
    torch.cuda.synchronize()
    for a, b in zip(ys, want):
        assert torch.equal(a, b)


def test_scratch_belongs_to_the_calls_stream(gpu):
    """Memory that a call takes comes from its own stream's pool (the null stream's for handle 0), so that what is freed
    is used again in that stream's order."""
    x = torch.randn(4, 4096, device=gpu)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for stream, owner in ((None, 0), (0, 0), (side, side.cuda_stream), (side.cuda_stream, side.cuda_stream)):
        m = mt.F8Matrix.quantize(x, stream=stream)
        at = m.codes.data_ptr()
        segments = [g for g in torch.cuda.memory_snapshot() if g["address"] <= at < g["address"] + g["total_size"]]
        assert len(segments) == 1 and segments[0]["stream"] == owner
        torch.cuda.synchronize()
        assert torch.equal(m.codes, mt.F8Matrix.quantize(x).codes)


@pytest.mark.parametrize("M", [2, 40])
def test_operands_on_the_host_are_refused(gpu, M):
    w, _ = matrix(np.ones((32, 256)), gpu)
    x, y, host = torch.ones(M, 256, device=gpu), torch.zeros(M, 32, device=gpu), torch.ones(256, dtype=torch.float16)
    for more in (dict(bias=host[:32]), dict(norm=host)):
        with pytest.raises(ValueError, match="one device"):
            mt.linear_f8(x, w, y, **more)
    with pytest.raises(ValueError):
        mt.linear_f8(x.cpu(), w, y)
    with pytest.raises(ValueError):
        mt.linear_f8(x, w, y.cpu())
    torch.cuda.synchronize()
    assert not y.any()
