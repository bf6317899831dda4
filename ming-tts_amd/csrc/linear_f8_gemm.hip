// The GEMM over 8-bit matrices (f8_gemm.hpp): its tiles and their choice.
#include "f8_gemm.hpp"
#include "mt_internal.hpp"

namespace mt {

namespace {

template <class TL, bool GATED>
int launch_tile(const F8LinearArgs &a, int bt, hipStream_t stream) {
    static_assert(TL::KG * TL::P * TL::STAGE <= 160 * 1024, "LDS of a CU");
    const uint32_t feat = GATED ? TL::BN / 2 : TL::BN;
    const uint32_t tm = (a.M - 1) / TL::BM + 1, tn = (a.N - 1) / feat + 1;
    const int rc = check_grid("linear (8-bit GEMM)", static_cast<uint64_t>(tm) * tn, 64 * TL::WAVES * TL::KG);
    if (rc) return rc;
    hipLaunchKernelGGL((f8::gemm_kernel<TL, GATED>), dim3(tm * tn), dim3(64 * TL::WAVES * TL::KG), TL::KG * TL::P * TL::STAGE, stream, a, bt,
                       tm, tn);
    return check_launch("linear (8-bit GEMM)");
}

}  // namespace

// The tile of a linear: 1 = 256 x 256, 2 = 64 x 128, 3 = 64 x 64 with two groups on K, 4 = 32 x 64 with four (x rows
// by weight rows, those of the gate partner counted).
//
// A tile's K loop costs about the same time whatever the tile (each step's barrier, LDS reads and conversions),
// so the small ones pay while they only fill CUs that would idle: the smallest that leaves at most one workgroup a
// CU.  Measured (us, tiles 4 / 3 / 2): 512 x 896, K 4864 (224 tiles of 32 x 64) 11.9 / 15.8 / 25.2; 512 x 1152,
// K 896 (288; 144 of 64 x 64) 8.8 / 6.1 / 7.8; 512 x 4096, K 1024 (512 of 64 x 64) 16.4 / 9.3 / 9.6; 128 x 2 x
// 4864, K 896 (304) 13.9 / 8.8 / 7.5.  The 256 x 256 tiles run at 1250 against 950 TFLOP/s where they fill the CUs
// over a long K (4096 x 4096 x 4096: 110 against 144 us), and take 49 against 42 at 2048 x 2 x 4864, K 896.
int gemm_f8_tile(uint32_t M, uint32_t cols, uint32_t K, int cus) {
    auto tiles = [&](uint64_t bm, uint64_t bn) { return (M + bm - 1) / bm * ((cols + bn - 1) / bn); };
    const uint64_t cu = cus > 0 ? cus : 256, big = tiles(256, 256), rounds = (big + cu - 1) / cu;
    if (K >= 2048 && 5 * big >= 4 * cu * rounds) return 1;
    return tiles(32, 64) <= cu ? 4 : tiles(64, 64) <= cu ? 3 : 2;
}

int launch_gemm_f8(const F8LinearArgs &a, int bt, hipStream_t stream) {
    const bool gated = (a.flags & F_SILU_GATE) != 0;
    int tile = tuning().f8_tile.load(std::memory_order_relaxed);
    if (tile == 0) tile = gemm_f8_tile(a.M, gated ? 2 * a.N : a.N, a.K, device_cus());
    // A gated wave holds fragments of both weights; the others are spread over more waves.
    switch (tile) {
        case 1: return gated ? launch_tile<f8::Tile<4, 2, 2, 4, 1, 2>, true>(a, bt, stream) : launch_tile<f8::Tile<4, 2, 2, 4, 1, 2>, false>(a, bt, stream);
        case 2: return gated ? launch_tile<f8::Tile<1, 2, 2, 2, 1, 2>, true>(a, bt, stream) : launch_tile<f8::Tile<1, 2, 2, 2, 1, 2>, false>(a, bt, stream);
        case 3: return gated ? launch_tile<f8::Tile<1, 2, 2, 1, 2, 2>, true>(a, bt, stream) : launch_tile<f8::Tile<1, 1, 2, 2, 2, 2>, false>(a, bt, stream);
        default: return gated ? launch_tile<f8::Tile<1, 2, 1, 1, 4, 2>, true>(a, bt, stream) : launch_tile<f8::Tile<1, 1, 1, 2, 4, 2>, false>(a, bt, stream);
    }
}

}  // namespace mt
