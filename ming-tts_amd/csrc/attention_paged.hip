// Attention of B sequences, T query rows each, over their own keys in pages (mt_attention_paged) or in contiguous caches
// (mt_attention_sinks): all of them, or a sliding window and the first `sinks` ones.
//
// out = sum_j p_j v_j / sum_j p_j with p_j = exp(s_j - max s), s_j = scale q . k_j, over the slots j <= i of a row at slot i that have
// j > i - window or j < sinks.
//
//   - One wave a row and query head: 64 keys at a time, each lane a key's score, then each lane a dim's sum, an online softmax
//     in fp32.
#include "attend_tiles.hpp"
#include "mt_internal.hpp"

namespace mt {

namespace {

// Where the head's rows of slot `slot` of sequence b stand, in rows of 64 elements and in scale bytes from the caches' start;
// false: nowhere.
__device__ __forceinline__ bool find(const PagedArgs &kv, uint32_t b, uint32_t kvh, uint32_t slot, uint64_t &row, uint64_t &scale) {
    uint64_t page = b;
    uint32_t in = slot;
    bool have = true;
    if (kv.table) {
        const uint32_t e = kv.entry(slot);
        page = kv.table[static_cast<size_t>(b) * kv.table_stride + e];
        in -= e * kv.page_len;
        have = page < kv.pages;
    }
    const uint64_t at = static_cast<uint64_t>(kvh) * kv.page_len + in;
    row = page * kv.stride + at * 64;
    scale = page * kv.sstride + at;
    return have;
}

// Element `row + e` of the caches.
template <int CT>
__device__ __forceinline__ float cached(const void *base, const uint8_t *scales, uint64_t row, uint64_t scale, uint32_t e) {
    if constexpr (CT == DT_F32) return static_cast<const float *>(base)[row + e];
    else if constexpr (CT == DT_F16) return (float)static_cast<const _Float16 *>(base)[row + e];
    else return bf16_lo(f8_bf16x2<false>(static_cast<const uint8_t *>(base)[row + e], 1.0f)) * f8_pow2(scales[scale]);
}

// The keys of a row at slot `slot`: those before `first`, and [lo, hi).
__device__ __forceinline__ void row_keys(const WindowArgs &a, uint64_t slot, uint32_t &first, uint32_t &lo, uint32_t &hi) {
    hi = static_cast<uint32_t>(min(slot, static_cast<uint64_t>(a.kv.len - 1))) + 1;
    lo = a.window > 0 && hi > a.window ? hi - a.window : 0;
    first = min(a.sinks, lo);
}

// One query head of a row by one wave, touching the row's own keys only.  (The maximum takes no notice of NaN, so a NaN score
// has to become its weight by itself where no other score of its keys is above -infinity.)
template <int CT>
__device__ __forceinline__ void attend_wave(const WindowArgs &a, uint32_t b, uint32_t row, uint32_t head, uint64_t slot) {
    const uint32_t lane = threadIdx.x & 63, kvh = head / a.group;
    const float *q = a.q + static_cast<size_t>(row) * a.ldq + head * 64;
    uint32_t first, lo, hi;
    row_keys(a, slot, first, lo, hi);
    const uint32_t n = first + (hi - lo);
    float m = -INFINITY, l = 0.0f, o = 0.0f;
    for (uint32_t k0 = 0; k0 < n; k0 += 64) {
        const uint32_t k = k0 + lane;
        uint64_t at = 0, sc = 0;
        const bool have = k < n && find(a.kv, b, kvh, k < first ? k : lo + (k - first), at, sc);
        float s = -INFINITY;
        if (have) {
            float d = 0.0f;
            for (uint32_t e = 0; e < 64; e++) d = fmaf(q[e], cached<CT>(a.kv.k, a.kv.ks, at, sc, e), d);
            s = d * a.scale;
        }
        const float mn = fmaxf(m, wave_max(s));
        const float al = m == -INFINITY ? 0.0f : exp_hw(m - mn);
        const float p = !have ? 0.0f : mn == -INFINITY ? (s != s ? s : 0.0f) : exp_hw(s - mn);
        m = mn;
        l = fmaf(l, al, group_sum(p, 64));
        o *= al;
        for (uint64_t left = __ballot(have); left; left &= left - 1) {
            const int j = __ffsll(static_cast<unsigned long long>(left)) - 1;
            const uint64_t aj = __shfl(static_cast<unsigned long long>(at), j, 64), sj = __shfl(static_cast<unsigned long long>(sc), j, 64);
            o = fmaf(__shfl(p, j, 64), cached<CT>(a.kv.v, a.kv.vs, aj, sj, lane), o);
        }
    }
    a.out[static_cast<size_t>(row) * a.ldo + head * 64 + lane] = l == 0.0f ? 0.0f : o / l;
}

constexpr uint32_t AP_THREADS = 256;

template <int CT>
__global__ __launch_bounds__(AP_THREADS) void attention_window_kernel(WindowArgs a) {
    const uint32_t i = blockIdx.x * (AP_THREADS / 64) + threadIdx.x / 64, row = i / a.hq;
    uint32_t b;
    uint64_t slot;
    if (row >= a.rows.B * a.rows.T || !a.rows.at(row, b, slot)) return;
    attend_wave<CT>(a, b, row, i - row * a.hq, slot);
}

}  // namespace

int launch_attention_window(const WindowArgs &a, int ct, hipStream_t stream) {
    const uint64_t groups = (static_cast<uint64_t>(a.rows.B) * a.rows.T * a.hq + AP_THREADS / 64 - 1) / (AP_THREADS / 64);
    const int rc = check_grid("attention window", groups, AP_THREADS);
    if (rc) return rc;
    const dim3 grid(static_cast<uint32_t>(groups));
    if (ct == DT_F32) hipLaunchKernelGGL(attention_window_kernel<DT_F32>, grid, dim3(AP_THREADS), 0, stream, a);
    else if (ct == DT_F16) hipLaunchKernelGGL(attention_window_kernel<DT_F16>, grid, dim3(AP_THREADS), 0, stream, a);
    else hipLaunchKernelGGL(attention_window_kernel<DT_F8>, grid, dim3(AP_THREADS), 0, stream, a);
    return check_launch("attention window");
}

}  // namespace mt
