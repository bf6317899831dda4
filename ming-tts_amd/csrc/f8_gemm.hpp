// The GEMM over 8-bit matrices: y = epilogue(x w^T), tiles staged through LDS as codes.
#pragma once

#include "f8_linear.hpp"

namespace mt {
namespace f8 {

typedef float f32x16v __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8v __attribute__((ext_vector_type(8)));

// A tile of BM rows of x and BN rows of the weights (gated: BN / 2 features of w and of w2), on WM x WN
// waves of MB x NB fragments of 32 x 32.
template <int MB_, int NB_, int WM_, int WN_>
struct Tile {
    static constexpr int MB = MB_, NB = NB_, WM = WM_, WN = WN_, WAVES = WM * WN;
    static constexpr int BM = 32 * MB * WM, BN = 32 * NB * WN;
    static constexpr uint32_t STAGE = (BM + BN) * 128;  // bytes of a stage: 128 k
};

__device__ __forceinline__ void lds16(__amdgpu_buffer_rsrc_t r, uint32_t lds, uint32_t off) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, reinterpret_cast<__attribute__((address_space(3))) void *>(lds), 16, static_cast<int>(off),
                                             0, 0, 0);
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_of(const uint8_t *p, uint32_t rows, uint32_t ld, uint32_t K) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(p), 0, static_cast<int>((rows - 1) * ld + K), 0x00020000);
}

template <class TL, bool GATED>
__global__ __launch_bounds__(64 * TL::WAVES) void gemm_kernel(F8LinearArgs a, int bt, uint32_t tiles_m, uint32_t tiles_n) {
    constexpr int MB = TL::MB, NB = TL::NB, BM = TL::BM, BN = TL::BN, W = TL::WAVES;
    constexpr uint32_t FEAT = GATED ? BN / 2 : BN;  // features of a tile
    constexpr uint32_t OUT = 0xF0000000u;           // past every buffer: the load gives zeros
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    const uint32_t tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, g = lane >> 5;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave % TL::WM, wn = wave / TL::WM;
    const uint32_t tm = blockIdx.x % tiles_m, tn = blockIdx.x / tiles_m;
    const uint32_t m0 = tm * BM, n0 = tn * FEAT;
    const uint32_t mrows = min(static_cast<uint32_t>(BM), a.M - m0), nrows = min(FEAT, a.N - n0);
    const uint32_t blocks = (a.K + 127) / 128;

    const __amdgpu_buffer_rsrc_t xr = rows_of(static_cast<const uint8_t *>(a.x) + static_cast<size_t>(m0) * a.ldx, mrows, a.ldx, a.K);
    const __amdgpu_buffer_rsrc_t wr = rows_of(a.w + static_cast<size_t>(n0) * a.K, nrows, a.K, a.K);
    const __amdgpu_buffer_rsrc_t ur = rows_of((GATED ? a.w2 : a.w) + static_cast<size_t>(n0) * a.K, nrows, a.K, a.K);

    // A wave's load of 1 KiB: eight rows, lane l's 16-byte chunk l % 8 of row l / 8, which holds the row's
    // chunk (l % 8) ^ (row % 8), so eight rows' same chunk lie in eight different bank groups.
    const uint32_t lr = lane >> 3, lc = 16 * ((lane & 7) ^ lr);
    const uint32_t base = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) uint8_t *)lds));
    auto stage = [&](uint32_t kb) {
        const uint32_t at = base + (kb & 1) * TL::STAGE, k = kb * 128 + lc;
        const bool in = k < a.K;
#pragma unroll
        for (int i = 0; i < BM / 8 / W; i++) {
            const uint32_t r8 = wave + W * i;
            lds16(xr, at + r8 * 1024, in ? (8 * r8 + lr) * a.ldx + k : OUT);
        }
#pragma unroll
        for (int i = 0; i < BN / 8 / W; i++) {
            const uint32_t r8 = wave + W * i;
            const bool second = GATED && r8 >= BN / 16;
            const uint32_t row = 8 * (second ? r8 - BN / 16 : r8) + lr;
            const uint32_t off = in ? row * a.K + k : OUT;
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

    scales(0);
    stage(0);
    for (uint32_t kb = 0; kb < blocks; kb++) {
        if ((kb & 3) == 0) {
#pragma unroll
            for (int i = 0; i < MB; i++) as[i] = an[i];
#pragma unroll
            for (int j = 0; j < NB; j++) bs[j] = bn[j];
        }
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (kb + 1 < blocks) stage(kb + 1);
        if ((kb & 3) == 0 && kb + 4 < blocks) scales(kb + 4);
        const uint8_t *at = lds + (kb & 1) * TL::STAGE, *bt_ = at + BM * 128;
        float fa[MB], fb[NB];
#pragma unroll
        for (int i = 0; i < MB; i++) fa[i] = f8_pow2((as[i] >> (8 * (kb & 3))) & 255u);
#pragma unroll
        for (int j = 0; j < NB; j++) fb[j] = f8_pow2((bs[j] >> (8 * (kb & 3))) & 255u);
#pragma unroll
        for (int q = 0; q < 4; q++) {
            // 32 k: half g of the lanes holds the 16 of chunk 2 q + g, eight for each of two steps
            u32x4v ar[MB], br[NB];
#pragma unroll
            for (int i = 0; i < MB; i++) ar[i] = *reinterpret_cast<const u32x4v *>(at + arow[i] * 128 + 16 * ((2 * q + g) ^ (arow[i] & 7)));
#pragma unroll
            for (int j = 0; j < NB; j++) br[j] = *reinterpret_cast<const u32x4v *>(bt_ + brow[j] * 128 + 16 * ((2 * q + g) ^ (brow[j] & 7)));
#pragma unroll
            for (int s = 0; s < 2; s++) {
                bf16x8v av[MB], bv[NB];
#pragma unroll
                for (int i = 0; i < MB; i++)
                    av[i] = __builtin_bit_cast(bf16x8v, u32x4v{f8_bf16x2<false>(ar[i][2 * s], fa[i]), f8_bf16x2<true>(ar[i][2 * s], fa[i]),
                                                               f8_bf16x2<false>(ar[i][2 * s + 1], fa[i]), f8_bf16x2<true>(ar[i][2 * s + 1], fa[i])});
#pragma unroll
                for (int j = 0; j < NB; j++)
                    bv[j] = __builtin_bit_cast(bf16x8v, u32x4v{f8_bf16x2<false>(br[j][2 * s], fb[j]), f8_bf16x2<true>(br[j][2 * s], fb[j]),
                                                               f8_bf16x2<false>(br[j][2 * s + 1], fb[j]), f8_bf16x2<true>(br[j][2 * s + 1], fb[j])});
#pragma unroll
                for (int i = 0; i < MB; i++)
#pragma unroll
                    for (int j = 0; j < NB; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(av[i], bv[j], acc[i][j], 0, 0, 0);
            }
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
