// Attention of B sequences, T query rows each, over keys that all of them share and then over their
// own (mt_attention_shared), for caches of fp32, fp16 and 8 bits.
#include "f8.hpp"
#include "mt_internal.hpp"

namespace mt {

namespace {

template <int CT>
struct Cached {
    static constexpr uint32_t ES = CT == DT_F32 ? 4 : CT == DT_F16 ? 2 : 1;  // bytes of a value
    static constexpr uint32_t ROW = 64 * ES;                                 // bytes of a position's head
};

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int i = 32; i > 0; i >>= 1) v = fmaxf(v, __shfl_xor(v, i, 64));
    return v;
}

// One head's keys and values: those of the shared prefix (slots 0 .. prefix - 1) and then a
// sequence's own.
struct HeadKv {
    const char *k[2], *v[2];       // [0] prefix, [1] own: the head's first row
    const uint8_t *ks[2], *vs[2];  // 8-bit caches: the head's first scale
    uint32_t prefix;
};

template <int CT>
__device__ __forceinline__ HeadKv head_kv(const SharedArgs &a, uint32_t b, uint32_t kvh) {
    HeadKv h;
    const size_t own = b * a.kv.stride * Cached<CT>::ES + static_cast<size_t>(kvh) * a.kv.len * Cached<CT>::ROW;
    const size_t pre = static_cast<size_t>(kvh) * a.prefix.len * Cached<CT>::ROW;
    h.k[1] = static_cast<const char *>(a.kv.k) + own;
    h.v[1] = static_cast<const char *>(a.kv.v) + own;
    h.k[0] = static_cast<const char *>(a.prefix.k) + pre;
    h.v[0] = static_cast<const char *>(a.prefix.v) + pre;
    if constexpr (CT == DT_F8) {
        const size_t so = b * a.kv.sstride + static_cast<size_t>(kvh) * a.kv.len, sp = static_cast<size_t>(kvh) * a.prefix.len;
        h.ks[1] = a.kv.ks + so;
        h.vs[1] = a.kv.vs + so;
        h.ks[0] = a.prefix.ks + sp;
        h.vs[0] = a.prefix.vs + sp;
    }
    h.prefix = a.prefix_len;
    return h;
}

// Value e of a cached row.
template <int CT>
__device__ __forceinline__ float cached(const char *base, const uint8_t *scales, size_t slot, uint32_t e) {
    const char *row = base + slot * Cached<CT>::ROW;
    if constexpr (CT == DT_F32) return reinterpret_cast<const float *>(row)[e];
    else if constexpr (CT == DT_F16) return (float)reinterpret_cast<const _Float16 *>(row)[e];
    else return bf16_lo(f8_bf16x2<false>(reinterpret_cast<const uint8_t *>(row)[e], f8_pow2(scales[slot])));
}

// One query head over keys [lo, hi) (prefix first) by one wave, touching those keys only: each lane a
// key's score, then each lane a dim's sum.  An online softmax in fp32, 64 keys at a time.
template <int CT>
__device__ void attend_wave(const float *q, const HeadKv &h, uint64_t lo, uint64_t hi, float scale, float *out) {
    const uint32_t lane = threadIdx.x & 63;
    float m = -INFINITY, l = 0.0f, o = 0.0f;
    for (uint64_t k0 = lo; k0 < hi; k0 += 64) {
        const uint64_t key = k0 + lane;
        float s = -INFINITY;
        if (key < hi) {
            const int own = key >= h.prefix;
            const size_t slot = own ? key - h.prefix : key;
            float d = 0.0f;
            for (uint32_t e = 0; e < 64; e++) d = fmaf(q[e], cached<CT>(h.k[own], h.ks[own], slot, e), d);
            s = d * scale;
        }
        const float mn = fmaxf(m, wave_max(s));
        const float al = m == -INFINITY ? 0.0f : exp_hw(m - mn);
        const float p = key >= hi || mn == -INFINITY ? 0.0f : exp_hw(s - mn);
        m = mn;
        l = fmaf(l, al, group_sum(p, 64));
        o *= al;
        const uint32_t n = static_cast<uint32_t>(min(hi - k0, static_cast<uint64_t>(64)));
        for (uint32_t j = 0; j < n; j++) {
            const uint64_t kj = k0 + j;
            const int own = kj >= h.prefix;
            const size_t slot = own ? kj - h.prefix : kj;
            o = fmaf(__shfl(p, static_cast<int>(j), 64), cached<CT>(h.v[own], h.vs[own], slot, lane), o);
        }
    }
    out[lane] = o / l;
}

// The keys of a row whose own slot is `slot`: [lo, hi) of the prefix and the own keys together.
__device__ __forceinline__ void row_keys(const SharedArgs &a, uint64_t slot, uint64_t &lo, uint64_t &hi) {
    const uint64_t at = min(slot, static_cast<uint64_t>(a.kv.len - 1));
    hi = at + 1 + a.prefix_len;
    lo = a.window > 0 && hi > a.window ? hi - a.window : 0;
}

constexpr int AS_THREADS = 256;

template <int CT>
__global__ __launch_bounds__(AS_THREADS) void attention_rows_of(SharedArgs a) {
    const uint64_t i = static_cast<uint64_t>(blockIdx.x) * (AS_THREADS / 64) + threadIdx.x / 64;
    if (i >= static_cast<uint64_t>(a.rows.B) * a.rows.T * a.hq) return;
    const uint32_t row = static_cast<uint32_t>(i / a.hq), h = static_cast<uint32_t>(i - static_cast<uint64_t>(row) * a.hq);
    uint32_t b;
    uint64_t slot, lo, hi;
    if (!a.rows.at(row, b, slot)) return;
    row_keys(a, slot, lo, hi);
    attend_wave<CT>(a.q + static_cast<size_t>(row) * a.ldq + h * 64, head_kv<CT>(a, b, h / (a.hq / a.hkv)), lo, hi, a.scale,
                    a.out + static_cast<size_t>(row) * a.ldo + h * 64);
}

}  // namespace

int launch_attention_shared(const SharedArgs &a, int ct, hipStream_t stream) {
    const uint64_t waves = static_cast<uint64_t>(a.rows.B) * a.rows.T * a.hq;
    const dim3 grid(static_cast<uint32_t>((waves + AS_THREADS / 64 - 1) / (AS_THREADS / 64)));
    if (ct == DT_F32) hipLaunchKernelGGL(attention_rows_of<DT_F32>, grid, dim3(AS_THREADS), 0, stream, a);
    else if (ct == DT_F16) hipLaunchKernelGGL(attention_rows_of<DT_F16>, grid, dim3(AS_THREADS), 0, stream, a);
    else hipLaunchKernelGGL(attention_rows_of<DT_F8>, grid, dim3(AS_THREADS), 0, stream, a);
    return check_launch("attention shared");
}

}  // namespace mt
