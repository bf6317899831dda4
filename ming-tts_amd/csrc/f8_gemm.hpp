// The GEMM over 8-bit matrices: y = epilogue(x w^T), x and w in e4m3 with a scale a block of 128 (f8.hpp).
//
//   - Codes travel global -> LDS directly (16 bytes a lane, half of what 16-bit operands would), a stage of 128 k at a time,
//     and become bf16 in registers, behind the LDS read, with their block's scale in the conversion: the values are exact, so
//     the bf16 MFMAs see exact operands and nothing is left to scale afterwards.
//   - Why not the 8-bit MFMAs: they lose low bits inside an instruction (v_mfma_scale_f32_16x16x128_f8f6f4 and
//     v_mfma_f32_16x16x32_fp8_fp8 alike: normwise 1.2e-5 for rounded normal data, 7e-5 for codes of all sizes, against 6e-8
//     for bf16 over the same values), too much for fp32 outputs.
//   - A chain of MFMAs over the whole of K: normwise 8e-8 at K 4096, 1.8e-7 at 16384.
//   - A buffer descriptor ends with the tile's rows and the loads of chunks past K are out of its bounds: both read as zeros,
//     no branch in the loop.
//   - Bound: the MFMAs (54 % busy at 4096^3), the conversions beside them (3 vector instructions an MFMA) and a barrier a stage.
//     4096 x 4096 x 4096: 109-117 us a launch, depending on the machine, 1.17-1.26 PFLOP/s; the library's bf16 product of that size
//     takes 98 us (1.40) here.  Without the conversions 106, without the LDS reads 96, without the global loads 96; raised
//     priority for the MFMAs, fixed orders of conversions and MFMAs, deeper pipelines of smaller stages all came out slower.
#pragma once

#include "f8_linear.hpp"

namespace mt {
namespace f8 {

typedef float f32x16v __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8v __attribute__((ext_vector_type(8)));

// A tile of BM rows of x and BN rows of the weights (gated: BN / 2 features of w and of w2), on WM x WN
// waves of MB x NB fragments of 32 x 32.
// KG groups of such waves take every KG-th block of 128 k each; their sums meet at the end.  LDS holds P stages a
// group, P - 1 of them on their way.
template <int MB_, int NB_, int WM_, int WN_, int KG_, int P_>
struct Tile {
    static constexpr int MB = MB_, NB = NB_, WM = WM_, WN = WN_, KG = KG_, P = P_, WAVES = WM * WN;
    static constexpr int BM = 32 * MB * WM, BN = 32 * NB * WN;
    static constexpr uint32_t STAGE = (BM + BN) * 128;  // bytes of a stage
    static constexpr int LOADS = (BM + BN) / 8 / WAVES;   // loads of 1 KiB a wave and stage
    static_assert(BM % (8 * WAVES) == 0 && BN % (8 * WAVES) == 0, "whole loads a wave");
};

__device__ __forceinline__ void lds16(__amdgpu_buffer_rsrc_t r, uint32_t lds, uint32_t off) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, reinterpret_cast<__attribute__((address_space(3))) void *>(lds), 16, static_cast<int>(off),
                                             0, 0, 0);
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_of(const uint8_t *p, uint32_t rows, uint32_t ld, uint32_t K) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(p), 0, static_cast<int>((rows - 1) * ld + K), 0x00020000);
}

// Workgroup ids are dealt to the eight XCDs in turn: a contiguous run of tiles for each.
__device__ __forceinline__ uint32_t xcd_order(uint32_t b, uint32_t n) {
    const uint32_t x = b & 7u, i = b >> 3, q = n >> 3, r = n & 7u;
    return (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + i;
}

template <class TL, bool GATED>
__global__ __launch_bounds__(64 * TL::WAVES * TL::KG, 2) void gemm_kernel(F8LinearArgs a, int bt, uint32_t tiles_m, uint32_t tiles_n) {
    constexpr int MB = TL::MB, NB = TL::NB, BM = TL::BM, BN = TL::BN, W = TL::WAVES, KG = TL::KG;
    constexpr uint32_t FEAT = GATED ? BN / 2 : BN;  // features of a tile
    constexpr uint32_t OUT = 0xF0000000u;           // past every buffer: the load gives zeros
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    const uint32_t tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, g = lane >> 5;
    const uint32_t id = __builtin_amdgcn_readfirstlane(tid >> 6), kg = id / W, wave = id % W;
    const uint32_t wm = wave % TL::WM, wn = wave / TL::WM;
    const uint32_t tile = xcd_order(blockIdx.x, gridDim.x), tm = tile % tiles_m, tn = tile / tiles_m;
    const uint32_t m0 = tm * BM, n0 = tn * FEAT;
    const uint32_t mrows = min(static_cast<uint32_t>(BM), a.M - m0), nrows = min(FEAT, a.N - n0);
    const uint32_t blocks = (a.K + 127) / 128, steps = (blocks + KG - 1) / KG;

    const __amdgpu_buffer_rsrc_t xr = rows_of(static_cast<const uint8_t *>(a.x) + static_cast<size_t>(m0) * a.ldx, mrows, a.ldx, a.K);
    const __amdgpu_buffer_rsrc_t wr = rows_of(a.w + static_cast<size_t>(n0) * a.K, nrows, a.K, a.K);
    const __amdgpu_buffer_rsrc_t ur = rows_of((GATED ? a.w2 : a.w) + static_cast<size_t>(n0) * a.K, nrows, a.K, a.K);

    // A wave's load of 1 KiB: eight rows, lane l's 16-byte chunk l % 8 of row l / 8, which holds the row's
    // chunk (l % 8) ^ (row / 2 % 8): 16 rows' same chunk then lies in 16 different places of the
    // 64 banks (two rows each 256 bytes).
    const uint32_t lr = lane >> 3;
    const uint32_t base = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) uint8_t *)lds));
    auto chunk = [&](uint32_t r8) { return 16 * ((lane & 7) ^ (4 * (r8 & 1) + (lr >> 1))); };
    // The group's step, its block KG step + kg (past the last one: zeros), into a buffer.
    auto stage = [&](uint32_t step, uint32_t buffer) {
        const uint32_t at = base + (buffer * KG + kg) * TL::STAGE, k0 = (step * KG + kg) * 128;
#pragma unroll
        for (int i = 0; i < BM / 8 / W; i++) {
            const uint32_t r8 = wave + W * i, k = k0 + chunk(r8);
            lds16(xr, at + r8 * 1024, k < a.K ? (8 * r8 + lr) * a.ldx + k : OUT);
        }
#pragma unroll
        for (int i = 0; i < BN / 8 / W; i++) {
            const uint32_t r8 = wave + W * i, k = k0 + chunk(r8);
            const bool second = GATED && r8 >= BN / 16;
            const uint32_t row = 8 * (second ? r8 - BN / 16 : r8) + lr;
            const uint32_t off = k < a.K ? row * a.K + k : OUT;
            if (second) lds16(ur, at + BM * 128 + r8 * 1024, off);
            else lds16(wr, at + BM * 128 + r8 * 1024, off);
        }
    };
    // Fragment rows of the lane in the tile, and their scales' rows.
    uint32_t arow[MB], brow[NB];
    const uint8_t *asc[MB], *bsc[NB];
#pragma unroll
    for (int i = 0; i < MB; i++) {
        arow[i] = (wm * MB + i) * 32 + l32;
        asc[i] = a.xs + static_cast<size_t>(min(m0 + arow[i], a.M - 1)) * a.ldxs;
    }
#pragma unroll
    for (int j = 0; j < NB; j++) {
        const bool second = GATED && j >= NB / 2;
        const uint32_t f = GATED ? (wn * (NB / 2) + j % (NB / 2 ? NB / 2 : 1)) * 32 + l32 : (wn * NB + j) * 32 + l32;
        brow[j] = second ? BN / 2 + f : f;
        bsc[j] = (second ? a.w2s : a.ws) + static_cast<size_t>(min(n0 + f, a.N - 1)) * a.lds;
    }
    // A word holds four blocks' scales, of which the group's are every KG-th.
    constexpr int SC = 4 / KG;  // steps a word
    uint32_t as[MB], bs[NB], an[MB], bn[NB];
    auto scales = [&](uint32_t kb) {
#pragma unroll
        for (int i = 0; i < MB; i++) an[i] = *reinterpret_cast<const uint32_t *>(asc[i] + kb);
#pragma unroll
        for (int j = 0; j < NB; j++) bn[j] = *reinterpret_cast<const uint32_t *>(bsc[j] + kb);
    };

    f32x16v acc[MB][NB];
#pragma unroll
    for (int i = 0; i < MB; i++)
#pragma unroll
        for (int j = 0; j < NB; j++)
#pragma unroll
            for (int r = 0; r < 16; r++) acc[i][j][r] = 0.0f;

    // 32 k of a stage: half g of the lanes holds the 16 of chunk 2 q + g, eight for each of two steps.
    struct Raw {
        u32x4v a[MB], b[NB];
    };
    const uint32_t sw = (l32 >> 1) & 7;
    auto read = [&](Raw &f, const uint8_t *at, int q) {
        const uint32_t c = 16 * ((2 * q + g) ^ sw);
#pragma unroll
        for (int i = 0; i < MB; i++) f.a[i] = *reinterpret_cast<const u32x4v *>(at + arow[i] * 128 + c);
#pragma unroll
        for (int j = 0; j < NB; j++) f.b[j] = *reinterpret_cast<const u32x4v *>(at + BM * 128 + brow[j] * 128 + c);
    };
    auto value = [](const u32x4v &w, int s, float f) {
        return __builtin_bit_cast(bf16x8v, u32x4v{f8_bf16x2<false>(w[2 * s], f), f8_bf16x2<true>(w[2 * s], f),
                                                  f8_bf16x2<false>(w[2 * s + 1], f), f8_bf16x2<true>(w[2 * s + 1], f)});
    };
    // (block past the last one: codes of zeros, whose scale bytes may be anything)
    auto compute = [&](const uint8_t *at, int c, uint32_t block) {
        const uint32_t byte = block < blocks ? 255u : 0u;
        float fa[MB], fb[NB];
#pragma unroll
        for (int i = 0; i < MB; i++) fa[i] = f8_pow2((as[i] >> (8 * (c * KG + kg))) & byte);
#pragma unroll
        for (int j = 0; j < NB; j++) fb[j] = f8_pow2((bs[j] >> (8 * (c * KG + kg))) & byte);
        Raw f[2];
        read(f[0], at, 0);
#pragma unroll
        for (int q = 0; q < 4; q++) {
            if (q < 3) read(f[(q + 1) & 1], at, q + 1);
#pragma unroll
            for (int s = 0; s < 2; s++) {
                bf16x8v av[MB], bv[NB];
#pragma unroll
                for (int i = 0; i < MB; i++) av[i] = value(f[q & 1].a[i], s, fa[i]);
#pragma unroll
                for (int j = 0; j < NB; j++) bv[j] = value(f[q & 1].b[j], s, fb[j]);
#pragma unroll
                for (int i = 0; i < MB; i++)
#pragma unroll
                    for (int j = 0; j < NB; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(av[i], bv[j], acc[i][j], 0, 0, 0);
            }
        }
    };

    // Stage kb is waited for with P - 2 younger ones still on their way (the scales' loads among them only make
    // that wait longer); behind the barrier every wave has left the buffer that stage kb + P - 1 takes.
    constexpr int P = TL::P;
    scales(0);
#pragma unroll
    for (int i = 0; i < P - 1; i++) stage(i, i);
    uint32_t buffer = 0;
    for (uint32_t i0 = 0; i0 < steps; i0 += SC) {
#pragma unroll
        for (int i = 0; i < MB; i++) as[i] = an[i];
#pragma unroll
        for (int j = 0; j < NB; j++) bs[j] = bn[j];
#pragma unroll
        for (int c = 0; c < SC; c++) {
            if (i0 + c >= steps) break;
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((P - 2) * TL::LOADS) : "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            stage(i0 + c + P - 1, buffer == 0 ? P - 1 : buffer - 1);
            if (c == 0) scales(min((i0 + SC) * KG, (blocks - 1) & ~3u));
            compute(lds + (buffer * KG + kg) * TL::STAGE, c, (i0 + c) * KG + kg);
            buffer = buffer == P - 1 ? 0 : buffer + 1;
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // nothing lands in LDS behind here

    // The groups' sums in their order, all in group 0.
    if constexpr (KG > 1) {
        constexpr int REGS = MB * NB * 16;
        static_assert((KG - 1) * W * REGS * 256 <= KG * P * TL::STAGE, "the sums overlay the stages");
        float *sum = reinterpret_cast<float *>(lds);
        __syncthreads();
        if (kg > 0) {
#pragma unroll
            for (int i = 0; i < MB; i++)
#pragma unroll
                for (int j = 0; j < NB; j++)
#pragma unroll
                    for (int r = 0; r < 16; r += 4)
                        *reinterpret_cast<float4 *>(sum + (((kg - 1) * W + wave) * REGS + (i * NB + j) * 16 + r) * 64 + 4 * lane) =
                            make_float4(acc[i][j][r], acc[i][j][r + 1], acc[i][j][r + 2], acc[i][j][r + 3]);
        }
        __syncthreads();
        if (kg > 0) return;
#pragma unroll
        for (int q = 0; q < KG - 1; q++)
#pragma unroll
            for (int i = 0; i < MB; i++)
#pragma unroll
                for (int j = 0; j < NB; j++)
#pragma unroll
                    for (int r = 0; r < 16; r += 4) {
                        const float4 v = *reinterpret_cast<const float4 *>(sum + ((q * W + wave) * REGS + (i * NB + j) * 16 + r) * 64 + 4 * lane);
                        acc[i][j][r] += v.x;
                        acc[i][j][r + 1] += v.y;
                        acc[i][j][r + 2] += v.z;
                        acc[i][j][r + 3] += v.w;
                    }
    }

    // Lane l holds feature l % 32 of rows 8 (r / 4) + 4 g + r % 4 of each fragment.
    const bool whole = mrows == BM;
    with_flag_set(a.flags, [&](auto fl) {
        constexpr uint32_t FL = decltype(fl)::value;
#pragma unroll
        for (int j = 0; j < (GATED ? NB / 2 : NB); j++) {
            const uint32_t n = n0 + brow[j];
            if (n >= a.N) continue;
            const float b = !(a.flags & F_BIAS) ? 0.0f : bt == DT_BF16 ? dec1<DT_BF16>(a.bias[n]) : dec1<DT_F16>(a.bias[n]);
#pragma unroll
            for (int i = 0; i < MB; i++)
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const uint32_t m = m0 + (wm * MB + i) * 32 + 8 * (r >> 2) + 4 * g + (r & 3);
                    if (!whole && m >= a.M) continue;
                    float *y = a.y + static_cast<size_t>(m) * a.ldy + n;
                    const float v = epilogue_set<FL>(acc[i][j][r], GATED ? acc[i][j + NB / 2][r] : 0.0f, b, a.flags);
                    *y = accumulates<FL>(a.flags) ? v + *y : v;
                }
        }
    });
}

}  // namespace f8
}  // namespace mt
