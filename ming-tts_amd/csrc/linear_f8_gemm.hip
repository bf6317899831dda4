// The GEMM over 8-bit matrices (f8_gemm.hpp): its tiles and their choice.
#include "f8_gemm.hpp"
#include "mt_internal.hpp"

namespace mt {

namespace {

template <class TL>
int launch_tile(const F8LinearArgs &a, int bt, hipStream_t stream) {
    const bool gated = (a.flags & F_SILU_GATE) != 0;
    const uint32_t feat = gated ? TL::BN / 2 : TL::BN;
    const uint32_t tm = (a.M + TL::BM - 1) / TL::BM, tn = (a.N + feat - 1) / feat;
    const uint32_t lds = 2 * TL::STAGE;
    if (gated) hipLaunchKernelGGL((f8::gemm_kernel<TL, true>), dim3(tm * tn), dim3(64 * TL::WAVES), lds, stream, a, bt, tm, tn);
    else hipLaunchKernelGGL((f8::gemm_kernel<TL, false>), dim3(tm * tn), dim3(64 * TL::WAVES), lds, stream, a, bt, tm, tn);
    return check_launch("linear (8-bit GEMM)");
}

}  // namespace

int launch_gemm_f8(const F8LinearArgs &a, int bt, hipStream_t stream) {
    int tile = tuning().f8_tile.load(std::memory_order_relaxed);
    if (tile == 0) tile = a.M <= 64 ? 3 : a.M <= 1024 ? 2 : 1;
    switch (tile) {
        case 1: return launch_tile<f8::Tile<4, 2, 2, 4>>(a, bt, stream);
        case 2: return launch_tile<f8::Tile<2, 2, 2, 2>>(a, bt, stream);
        default: return launch_tile<f8::Tile<1, 2, 2, 2>>(a, bt, stream);
    }
}

}  // namespace mt
