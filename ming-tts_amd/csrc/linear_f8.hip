// Matrices in 8 bits (f8.hpp: a block is 128 consecutive values of a row): the quantiser
// (mt_quantize_f8) and the linears over such weights (mt_linear_f8): few rows here, more in f8_gemm.hpp.
//
// Quantiser: 4096 x 4096 fp32 in 17.5 us (84 MB, 4.8 TB/s: a large copy's rate), 512 x 896 in 2.
// Few rows: gate|up (2 x 4864 x 896) of two fp32 rows 5.6 us, 4.9 of rows that come quantised (8.7 MB; 1.7 us at a large
// copy's rate and 1.7 for an empty launch); down (896 x 4864) of 16 fp32 rows 9.1 us, 7.4 quantised: 56 workgroups that each
// quantise all of x.  Bound: latency at two rows, the quantising at sixteen.
#include <algorithm>

#include "f8_linear.hpp"
#include "mt_internal.hpp"

namespace mt {

namespace {

typedef short bf16x8v __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8t __attribute__((ext_vector_type(8)));
typedef float f32x4v __attribute__((ext_vector_type(4)));

// Eight values of type XT at p.
template <int XT>
__device__ __forceinline__ void load8(const void *p, float *x) {
    if constexpr (XT == DT_F32) {
        const float4 a = static_cast<const float4 *>(p)[0], b = static_cast<const float4 *>(p)[1];
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
        x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else {
        unpack8<XT>(*static_cast<const uint4 *>(p), x);
    }
}

// Eight values of a row from k on (zeros past K), the RMSNorm's gain and scale applied if there is one.
template <int XT>
__device__ __forceinline__ void load_x8(const char *xr, uint32_t k, uint32_t K, const uint16_t *norm, int nt, float rs, float *v) {
    constexpr uint32_t ES = XT == DT_F32 ? 4 : 2;
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = 0.0f;
    if (k >= K) return;
    load8<XT>(xr + static_cast<size_t>(k) * ES, v);
    if (norm) {
        float g[8];
        const uint4 w = *reinterpret_cast<const uint4 *>(norm + k);
        if (nt == DT_BF16) unpack8<DT_BF16>(w, g); else unpack8<DT_F16>(w, g);
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = v[e] * rs * g[e];
    }
}

// The sum of squares of a block of 128 by the 16 lanes that hold it.
__device__ __forceinline__ float block_square(const float *v) {
    float sq = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; e++) sq = fmaf(v[e], v[e], sq);
    return group_sum(sq, 16);
}
// The RMSNorm's factor of a row from its blocks' sums of squares, by 16 lanes (l16 of them): one order of
// the sums wherever a row is normalised, so the same rows give the same codes.
__device__ __forceinline__ float row_factor(const float *sq, uint32_t blocks, uint32_t l16, uint32_t K, float eps) {
    float t = 0.0f;
    for (uint32_t i = l16; i < blocks; i += 16) t += sq[i];
    return 1.0f / sqrtf(group_sum(t, 16) / static_cast<float>(K) + eps);
}

// The codes of a block's eight values a lane, by its 16 lanes, and the block's scale byte.
__device__ __forceinline__ u32x2v block_encode(const float *v, uint32_t &s) {
    float top = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; e++) top = fmaxf(top, f8_abs(v[e]));
    s = f8_scale(row16_max(top));
    const float inv = f8_inv_pow2(s);
    return u32x2v{f8_encode4(v[0], v[1], v[2], v[3], inv), f8_encode4(v[4], v[5], v[6], v[7], inv)};
}

// Rows normalised first: one row a workgroup, 16 lanes a block of 128, eight values each.
template <int XT>
__global__ __launch_bounds__(256) void quantize_norm_kernel(const void *x, uint32_t K, uint32_t ldx, const uint16_t *norm, int nt,
                                                            float eps, uint8_t *codes, uint32_t ldq, uint8_t *scales, uint32_t lds) {
    constexpr uint32_t ES = XT == DT_F32 ? 4 : 2;
    extern __shared__ float sq[];
    const uint32_t row = blockIdx.x, l16 = threadIdx.x & 15, grp = threadIdx.x / 16, blocks = (K + 127) / 128;
    const char *xr = static_cast<const char *>(x) + static_cast<size_t>(row) * ldx * ES;
    float v[8];
    for (uint32_t kb = grp; kb < blocks; kb += 16) {
        load_x8<XT>(xr, kb * 128 + 8 * l16, K, nullptr, 0, 1.0f, v);
        const float t = block_square(v);
        if (l16 == 0) sq[kb] = t;
    }
    __syncthreads();
    const float rs = row_factor(sq, blocks, l16, K, eps);
    for (uint32_t kb = grp; kb < lds; kb += 16) {  // the row's padding bytes included
        const uint32_t k = kb * 128 + 8 * l16;
        load_x8<XT>(xr, k, K, norm, nt, rs, v);
        uint32_t s;
        const u32x2v w = block_encode(v, s);
        if (k < K) *reinterpret_cast<u32x2v *>(codes + static_cast<size_t>(row) * ldq + k) = w;
        if (l16 == 0) scales[static_cast<size_t>(row) * lds + kb] = static_cast<uint8_t>(kb < blocks ? s : 0);
    }
}

// Rows as they are: 16 lanes a block of 128, as many blocks in flight as the rows have.  Lane l holds values 4 l .. + 3 and
// 64 + 4 l .. + 3, so a load instruction's lanes stand side by side.  Bound: the bytes.
template <int XT>
__global__ __launch_bounds__(256) void quantize_kernel(const void *x, uint64_t all, uint32_t K, uint32_t ldx, uint8_t *codes,
                                                       uint32_t ldq, uint8_t *scales, uint32_t lds) {
    constexpr uint32_t ES = XT == DT_F32 ? 4 : 2;
    // The group's block of all rows' blocks (the padding bytes' too): the workgroup's first by a division, lds is 4 or more.
    const uint64_t first = static_cast<uint64_t>(blockIdx.x) * 16;
    const uint32_t l16 = threadIdx.x & 15;
    if (first + threadIdx.x / 16 >= all) return;
    size_t row = first / lds;
    uint32_t kb = static_cast<uint32_t>(first - row * lds) + threadIdx.x / 16;
#pragma unroll
    for (int j = 0; j < 4; j++)
        if (kb >= lds) kb -= lds, row++;
    const uint32_t k = kb * 128 + 4 * l16;
    const char *xr = static_cast<const char *>(x) + row * ldx * ES + static_cast<size_t>(k) * ES;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int h = 0; h < 2; h++) {
        if (k + 64 * h >= K) continue;
        if constexpr (XT == DT_F32) {
            const float4 w = *reinterpret_cast<const float4 *>(xr + 64 * h * ES);
            v[4 * h] = w.x; v[4 * h + 1] = w.y; v[4 * h + 2] = w.z; v[4 * h + 3] = w.w;
        } else {
            const u32x2v w = *reinterpret_cast<const u32x2v *>(xr + 64 * h * ES);
            v[4 * h] = dec_lo<XT>(w[0]); v[4 * h + 1] = dec_hi<XT>(w[0]);
            v[4 * h + 2] = dec_lo<XT>(w[1]); v[4 * h + 3] = dec_hi<XT>(w[1]);
        }
    }
    uint32_t s;
    const u32x2v w = block_encode(v, s);
    uint8_t *c = codes + row * ldq + k;
    if (k < K) *reinterpret_cast<uint32_t *>(c) = w[0];
    if (k + 64 < K) *reinterpret_cast<uint32_t *>(c + 64) = w[1];
    if (l16 == 0) scales[row * lds + kb] = static_cast<uint8_t>(kb * 128 < K ? s : 0);
}

// A lane's 32 codes of a row from k on (those past K as zeros) and the block's scale byte.
struct RowCodes {
    u32x4v c[2];
    uint32_t s;
};
__device__ __forceinline__ RowCodes row_load(const uint8_t *codes, uint32_t k, uint32_t K, const uint8_t *scale) {
    RowCodes r;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        r.c[i] = u32x4v{0u, 0u, 0u, 0u};
        if (k + 16 * i < K) r.c[i] = *reinterpret_cast<const u32x4v *>(codes + k + 16 * i);
    }
    r.s = *scale;
    return r;
}
// Their bf16 values, four operands of eight.
__device__ __forceinline__ void row_values(const RowCodes &r, bf16x8t (&o)[4]) {
    const float f = f8_pow2(r.s);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t a = r.c[i / 2][2 * (i & 1)], b = r.c[i / 2][2 * (i & 1) + 1];
        o[i] = __builtin_bit_cast(bf16x8t, u32x4v{f8_bf16x2<false>(a, f), f8_bf16x2<true>(a, f), f8_bf16x2<false>(b, f),
                                                  f8_bf16x2<true>(b, f)});
    }
}

// Few rows of x: a workgroup of up to 16 waves takes 16 features and MT tiles of 16 rows, each wave every
// WAVES-th block of 128 values of K.  A lane's 32 codes of a weight row are two loads; x comes quantised, or (MT
// 1) the wave quantises its blocks itself, 16 lanes a block, and passes the codes through LDS into the operand's
// order (its own, so the loop has no barrier).  The waves' sums meet in LDS in wave order.
constexpr uint32_t FEW_LDX = 144;                      // bytes of a row of a wave's codes (128 and a skew)
constexpr uint32_t FEW_WAVE = 16 * FEW_LDX + 16 * 4;   // bytes of a wave's codes and scales

template <int XT, bool GATED>
__global__ __launch_bounds__(1024) void few_rows_kernel(F8LinearArgs a, int bt) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    constexpr uint32_t ES = XT == DT_F32 ? 4 : XT == DT_F8 ? 1 : 2;
    const uint32_t tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, g = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6), waves = blockDim.x / 64;
    const uint32_t n0 = blockIdx.x * 16, n = min(n0 + l16, a.N - 1), m0 = blockIdx.y * 16, rows = min(a.M - m0, 16u);
    const uint32_t blocks = (a.K + 127) / 128;
    uint8_t *mine = lds + wave * FEW_WAVE;
    uint32_t *scale = reinterpret_cast<uint32_t *>(mine + 16 * FEW_LDX);
    const char *x = static_cast<const char *>(a.x);

    float rs[4] = {1.f, 1.f, 1.f, 1.f};
    if constexpr (XT != DT_F8) {
        if (a.norm) {
            float *sq = reinterpret_cast<float *>(lds + waves * FEW_WAVE);  // [M][blocks]
            for (uint32_t kb = wave; kb < blocks; kb += waves)
                for (uint32_t r = g; r < a.M; r += 4) {
                    float v[8];
                    load_x8<XT>(x + static_cast<size_t>(r) * a.ldx * ES, kb * 128 + 8 * l16, a.K, nullptr, 0, 1.0f, v);
                    const float t = block_square(v);
                    if (l16 == 0) sq[r * blocks + kb] = t;
                }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (4 * i + g < a.M) rs[i] = row_factor(sq + (4 * i + g) * blocks, blocks, l16, a.K, a.eps);
        }
    }

    f32x4v acc = {0.f, 0.f, 0.f, 0.f}, acc2 = acc;
    // A block's loads are issued as soon as the registers of the block before are converted: one round trip to memory a
    // block, each begun before the products of the block ahead of it (a wave has one block up to K 2048, three at K 4864).
    RowCodes w, u, xc;
    float v[4][8];
    auto load_w = [&](uint32_t kb) {
        const uint32_t k = kb * 128 + 32 * g;
        w = row_load(a.w + static_cast<size_t>(n) * a.K, k, a.K, a.ws + static_cast<size_t>(n) * a.lds + kb);
        if constexpr (GATED) u = row_load(a.w2 + static_cast<size_t>(n) * a.K, k, a.K, a.w2s + static_cast<size_t>(n) * a.lds + kb);
    };
    auto load_x = [&](uint32_t kb) {
        if constexpr (XT == DT_F8) {
            const size_t m = m0 + min(l16, rows - 1);
            xc = row_load(static_cast<const uint8_t *>(a.x) + m * a.ldx, kb * 128 + 32 * g, a.K, a.xs + m * a.ldxs + kb);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if (4u * i >= rows) break;
                load_x8<XT>(x + static_cast<size_t>(min(4 * i + g, rows - 1)) * a.ldx * ES, kb * 128 + 8 * l16, a.K, a.norm, bt, rs[i], v[i]);
            }
        }
    };
    load_x(wave);  // first: loads return in order, and x has the longer way to go
    load_w(wave);
    for (uint32_t kb = wave; kb < blocks; kb += waves) {
        const uint32_t next = kb + waves;
        if constexpr (XT != DT_F8) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t r = 4 * i + g;
                if (4u * i >= rows) break;
                uint32_t s;
                *reinterpret_cast<u32x2v *>(mine + r * FEW_LDX + 8 * l16) = block_encode(v[i], s);
                if (l16 == 0) scale[r] = s;
            }
            wave_sync();
            const uint32_t m = min(l16, rows - 1);
            xc.c[0] = *reinterpret_cast<const u32x4v *>(mine + m * FEW_LDX + 32 * g);
            xc.c[1] = *reinterpret_cast<const u32x4v *>(mine + m * FEW_LDX + 32 * g + 16);
            xc.s = scale[m];
            wave_sync();
        }
        bf16x8t xv[4], wv[4], uv[4];
        row_values(xc, xv);
        if (next < blocks) load_x(next);
        row_values(w, wv);
        if constexpr (GATED) row_values(u, uv);
        if (next < blocks) load_w(next);
#pragma unroll
        for (int i = 0; i < 4; i++) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wv[i], xv[i], acc, 0, 0, 0);
        if constexpr (GATED) {
#pragma unroll
            for (int i = 0; i < 4; i++) acc2 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(uv[i], xv[i], acc2, 0, 0, 0);
        }
    }

    // Part [wave][gate][row][feature].
    __syncthreads();
    float *part = reinterpret_cast<float *>(lds);
    constexpr uint32_t PW = GATED ? 512 : 256;
    *reinterpret_cast<f32x4v *>(part + wave * PW + l16 * 16 + 4 * g) = acc;
    if constexpr (GATED) *reinterpret_cast<f32x4v *>(part + wave * PW + 256 + l16 * 16 + 4 * g) = acc2;
    __syncthreads();
    for (uint32_t i = tid; i < rows * 16; i += blockDim.x) {
        const uint32_t row = m0 + i / 16, nn = n0 + (i & 15);
        if (nn >= a.N) continue;
        float s = 0.0f, s2 = 0.0f;
        for (uint32_t w0 = 0; w0 < waves; w0 += 4) {  // four waves' sums read at once
            float v[4], v2[4];
#pragma unroll
            for (uint32_t j = 0; j < 4; j++) {
                const uint32_t w = min(w0 + j, waves - 1);
                v[j] = part[w * PW + i];
                if constexpr (GATED) v2[j] = part[w * PW + 256 + i];
            }
#pragma unroll
            for (uint32_t j = 0; j < 4; j++) {
                s += w0 + j < waves ? v[j] : 0.0f;
                if constexpr (GATED) s2 += w0 + j < waves ? v2[j] : 0.0f;
            }
        }
        const float b = !(a.flags & F_BIAS) ? 0.0f : bt == DT_BF16 ? dec1<DT_BF16>(a.bias[nn]) : dec1<DT_F16>(a.bias[nn]);
        float *y = a.y + static_cast<size_t>(row) * a.ldy + nn;
        const float v = epilogue(s, s2, b, a.flags);
        *y = a.flags & F_ACCUM ? v + *y : v;
    }
}

// Waves of a workgroup: the blocks of K over at most 16, evenly.
uint32_t few_waves(uint32_t K) {
    const uint32_t blocks = (K + 127) / 128, each = (blocks + 15) / 16;
    return (blocks + each - 1) / each;
}

template <int XT>
int few_rows(const F8LinearArgs &a, int bt, hipStream_t stream) {
    const uint32_t blocks = (a.K + 127) / 128, waves = few_waves(a.K);
    const bool gated = (a.flags & F_SILU_GATE) != 0;
    const uint32_t codes = XT == DT_F8 ? 0 : waves * FEW_WAVE, sums = waves * 1024 * (gated ? 2 : 1);
    const uint32_t bytes = std::max(codes + (a.norm ? a.M * blocks * 4 : 0), sums);
    const dim3 grid((a.N - 1) / 16 + 1, (a.M - 1) / 16 + 1), block(64 * waves);
    const int rc = check_grid("linear (8-bit, few rows)", grid.x, block.x);
    if (rc) return rc;
    if (gated) hipLaunchKernelGGL((few_rows_kernel<XT, true>), grid, block, bytes, stream, a, bt);
    else hipLaunchKernelGGL((few_rows_kernel<XT, false>), grid, block, bytes, stream, a, bt);
    return check_launch("linear (8-bit, few rows)");
}

}  // namespace

int launch_quantize_f8(const void *x, int xt, uint32_t rows, uint32_t K, uint32_t ldx, const uint16_t *norm, int nt, float eps,
                       uint8_t *codes, uint32_t ldq, uint8_t *scales, uint32_t lds, hipStream_t stream) {
    const uint64_t all = static_cast<uint64_t>(rows) * lds;
    const int rc = check_grid("quantize", norm ? rows : (all + 15) / 16, 256);
    if (rc) return rc;
    if (norm) {
        const uint32_t shared = (K + 127) / 128 * 4;
#define QUANTIZE(XT) \
    hipLaunchKernelGGL(quantize_norm_kernel<XT>, dim3(rows), dim3(256), shared, stream, x, K, ldx, norm, nt, eps, codes, ldq, scales, lds)
        if (xt == DT_F32) QUANTIZE(DT_F32);
        else if (xt == DT_F16) QUANTIZE(DT_F16);
        else QUANTIZE(DT_BF16);
#undef QUANTIZE
        return check_launch("quantize (norm)");
    }
    const dim3 grid(static_cast<uint32_t>((all + 15) / 16));
#define QUANTIZE(XT) hipLaunchKernelGGL(quantize_kernel<XT>, grid, dim3(256), 0, stream, x, all, K, ldx, codes, ldq, scales, lds)
    if (xt == DT_F32) QUANTIZE(DT_F32);
    else if (xt == DT_F16) QUANTIZE(DT_F16);
    else QUANTIZE(DT_BF16);
#undef QUANTIZE
    return check_launch("quantize");
}

int launch_linear_f8(const F8LinearArgs &a, int xt, int bt, hipStream_t stream) {
    if (xt == DT_F32) return few_rows<DT_F32>(a, bt, stream);
    if (xt == DT_F16) return few_rows<DT_F16>(a, bt, stream);
    if (xt == DT_BF16) return few_rows<DT_BF16>(a, bt, stream);
    // Rows that come quantised: this kernel while its waves are at most 16 a CU (a tile of 16 x 16 without LDS or
    // barriers is the quicker one until the CUs queue).  Measured, us, it against the GEMM: 64 rows of 896 x 4864
    // (2912 waves of 256 CUs) 7.6 against 11.0, 64 of 1152 x 896 (2016) 4.5 against 5.0, 96 of 896 x 4864 (4368) 12.7 against
    // 11.0, 174 of 1152 x 896 (5544) 6.4 against 5.1, 64 of 2 x 4864 x 896 (8512) 10.2 against 6.5.
    const int cus = device_cus();
    const uint64_t tiles = static_cast<uint64_t>((a.N - 1) / 16 + 1) * ((a.M - 1) / 16 + 1);
    if (tuning().f8_tile.load(std::memory_order_relaxed) == 0 && a.M <= 16 * 65535u &&
        tiles * few_waves(a.K) <= 16ull * (cus > 0 ? cus : 256))
        return few_rows<DT_F8>(a, bt, stream);
    return launch_gemm_f8(a, bt, stream);
}

}  // namespace mt
