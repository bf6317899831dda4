// Matrices in 8 bits (f8.hpp: a block is 128 consecutive values of a row): the quantiser
// (mt_quantize_f8) and the linears over such weights (mt_linear_f8).
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

// One row a workgroup: 16 lanes a block of 128, eight values each.
template <int XT>
__global__ __launch_bounds__(256) void quantize_kernel(const void *x, uint32_t K, uint32_t ldx, const uint16_t *norm, int nt,
                                                       float eps, uint8_t *codes, uint32_t ldq, uint8_t *scales, uint32_t lds) {
    constexpr uint32_t ES = XT == DT_F32 ? 4 : 2;
    extern __shared__ float sq[];
    const uint32_t row = blockIdx.x, l16 = threadIdx.x & 15, grp = threadIdx.x / 16, blocks = (K + 127) / 128;
    const char *xr = static_cast<const char *>(x) + static_cast<size_t>(row) * ldx * ES;
    float v[8], rs = 1.0f;
    if (norm) {
        for (uint32_t kb = grp; kb < blocks; kb += 16) {
            load_x8<XT>(xr, kb * 128 + 8 * l16, K, nullptr, 0, 1.0f, v);
            const float t = block_square(v);
            if (l16 == 0) sq[kb] = t;
        }
        __syncthreads();
        rs = row_factor(sq, blocks, l16, K, eps);
    }
    for (uint32_t kb = grp; kb < lds; kb += 16) {  // the row's padding bytes included
        const uint32_t k = kb * 128 + 8 * l16;
        load_x8<XT>(xr, k, K, norm, nt, rs, v);
        uint32_t s;
        const u32x2v w = block_encode(v, s);
        if (k < K) *reinterpret_cast<u32x2v *>(codes + static_cast<size_t>(row) * ldq + k) = w;
        if (l16 == 0) scales[static_cast<size_t>(row) * lds + kb] = static_cast<uint8_t>(kb < blocks ? s : 0);
    }
}

// A lane's 32 codes of a row (from k on, those past K as zeros) as bf16 values, four operands of eight.
__device__ __forceinline__ void row_operand(const uint8_t *codes, uint32_t k, uint32_t K, uint32_t s, bf16x8t (&o)[4]) {
    const float f = f8_pow2(s);
#pragma unroll
    for (int i = 0; i < 2; i++) {
        u32x4v w = {0u, 0u, 0u, 0u};
        if (k + 16 * i < K) w = *reinterpret_cast<const u32x4v *>(codes + k + 16 * i);
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const u32x4v d = {f8_bf16x2<false>(w[2 * j], f), f8_bf16x2<true>(w[2 * j], f), f8_bf16x2<false>(w[2 * j + 1], f),
                              f8_bf16x2<true>(w[2 * j + 1], f)};
            o[2 * i + j] = __builtin_bit_cast(bf16x8t, d);
        }
    }
}

// Up to 16 rows of x: a workgroup of up to 16 waves takes 16 features, each wave every WAVES-th block of
// 128 values of K.  A lane's 32 codes of a weight row are two loads; x comes quantised, or the wave
// quantises its blocks itself, 16 lanes a block, and passes the codes through LDS into the operand's order (its
// own, so the loop has no barrier).  The waves' sums meet in LDS in wave order.
constexpr uint32_t FEW_LDX = 144;                      // bytes of a row of a wave's codes (128 and a skew)
constexpr uint32_t FEW_WAVE = 16 * FEW_LDX + 16 * 4;   // bytes of a wave's codes and scales

template <int XT, bool GATED>
__global__ __launch_bounds__(1024) void few_rows_kernel(F8LinearArgs a, int bt) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    constexpr uint32_t ES = XT == DT_F32 ? 4 : XT == DT_F8 ? 1 : 2;
    const uint32_t tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, g = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6), waves = blockDim.x / 64;
    const uint32_t n0 = blockIdx.x * 16, n = min(n0 + l16, a.N - 1), m = min(l16, a.M - 1);
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
    for (uint32_t kb = wave; kb < blocks; kb += waves) {
        const uint32_t k = kb * 128 + 32 * g;
        bf16x8t wv[4], gv[4], xv[4];
        row_operand(a.w + static_cast<size_t>(n) * a.K, k, a.K, a.ws[static_cast<size_t>(n) * a.lds + kb], wv);
        if constexpr (GATED) row_operand(a.w2 + static_cast<size_t>(n) * a.K, k, a.K, a.w2s[static_cast<size_t>(n) * a.lds + kb], gv);
        if constexpr (XT == DT_F8) {
            row_operand(static_cast<const uint8_t *>(a.x) + static_cast<size_t>(m) * a.ldx, k, a.K,
                        a.xs[static_cast<size_t>(m) * a.ldxs + kb], xv);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t r = 4 * i + g;
                if (4u * i >= a.M) break;
                float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                if (r < a.M) load_x8<XT>(x + static_cast<size_t>(r) * a.ldx * ES, kb * 128 + 8 * l16, a.K, a.norm, bt, rs[i], v);
                uint32_t s;
                *reinterpret_cast<u32x2v *>(mine + r * FEW_LDX + 8 * l16) = block_encode(v, s);
                if (l16 == 0) scale[r] = s;
            }
            wave_sync();
            row_operand(mine + m * FEW_LDX, 32 * g, 128, scale[m], xv);
            wave_sync();
        }
        f32x4v t = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 4; i++) t = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wv[i], xv[i], t, 0, 0, 0);
        acc += t;
        if constexpr (GATED) {
            t = f32x4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < 4; i++) t = __builtin_amdgcn_mfma_f32_16x16x32_bf16(gv[i], xv[i], t, 0, 0, 0);
            acc2 += t;
        }
    }

    // Part [wave][gate][row][feature].
    __syncthreads();
    float *part = reinterpret_cast<float *>(lds);
    constexpr uint32_t PW = GATED ? 512 : 256;
    *reinterpret_cast<f32x4v *>(part + wave * PW + l16 * 16 + 4 * g) = acc;
    if constexpr (GATED) *reinterpret_cast<f32x4v *>(part + wave * PW + 256 + l16 * 16 + 4 * g) = acc2;
    __syncthreads();
    for (uint32_t i = tid; i < a.M * 16; i += blockDim.x) {
        const uint32_t row = i / 16, nn = n0 + (i & 15);
        if (nn >= a.N) continue;
        float s = 0.0f, s2 = 0.0f;
        for (uint32_t w = 0; w < waves; w++) {
            s += part[w * PW + i];
            if constexpr (GATED) s2 += part[w * PW + 256 + i];
        }
        const float b = !(a.flags & F_BIAS) ? 0.0f : bt == DT_BF16 ? dec1<DT_BF16>(a.bias[nn]) : dec1<DT_F16>(a.bias[nn]);
        float *y = a.y + static_cast<size_t>(row) * a.ldy + nn;
        const float v = epilogue(s, s2, b, a.flags);
        *y = a.flags & F_ACCUM ? v + *y : v;
    }
}

template <int XT>
void few_rows(const F8LinearArgs &a, int bt, hipStream_t stream) {
    const uint32_t blocks = (a.K + 127) / 128, each = (blocks + 15) / 16, waves = (blocks + each - 1) / each;
    const bool gated = (a.flags & F_SILU_GATE) != 0;
    uint32_t bytes = waves * FEW_WAVE + (a.norm ? a.M * blocks * 4 : 0);
    static_assert(FEW_WAVE >= 2048, "the waves' sums overlay their codes");
    const dim3 grid((a.N + 15) / 16), block(64 * waves);
    if (gated) hipLaunchKernelGGL((few_rows_kernel<XT, true>), grid, block, bytes, stream, a, bt);
    else hipLaunchKernelGGL((few_rows_kernel<XT, false>), grid, block, bytes, stream, a, bt);
}

}  // namespace

int launch_quantize_f8(const void *x, int xt, uint32_t rows, uint32_t K, uint32_t ldx, const uint16_t *norm, int nt, float eps,
                       uint8_t *codes, uint32_t ldq, uint8_t *scales, uint32_t lds, hipStream_t stream) {
    const uint32_t shared = norm ? (K + 127) / 128 * 4 : 0;
#define QUANTIZE(XT) \
    hipLaunchKernelGGL(quantize_kernel<XT>, dim3(rows), dim3(256), shared, stream, x, K, ldx, norm, nt, eps, codes, ldq, scales, lds)
    if (xt == DT_F32) QUANTIZE(DT_F32);
    else if (xt == DT_F16) QUANTIZE(DT_F16);
    else QUANTIZE(DT_BF16);
#undef QUANTIZE
    return check_launch("quantize");
}

int launch_linear_f8(const F8LinearArgs &a, int xt, int bt, hipStream_t stream) {
    if (a.M <= 16) {
        if (xt == DT_F32) few_rows<DT_F32>(a, bt, stream);
        else if (xt == DT_F16) few_rows<DT_F16>(a, bt, stream);
        else if (xt == DT_BF16) few_rows<DT_BF16>(a, bt, stream);
        else few_rows<DT_F8>(a, bt, stream);
        return check_launch("linear (8-bit, few rows)");
    }
    return launch_gemm_f8(a, bt, stream);
}

}  // namespace mt
