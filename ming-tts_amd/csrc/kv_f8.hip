// The caches' writers: RoPE and append of new rows (mt_rope_append) and the copy of positions from
// one cache to another (mt_kv_copy), for caches of fp32, fp16 and 8 bits (f8.hpp: a block is the 64
// values of one head at one position).
//
// Reference kernel replaced: ropeCache (Shaders.swift:451-486), for rows of many sequences.
//
//   - Angles: position times frequency is exact in 64 bits (up to position 2^29), and its turns are taken off there, so a far position
//     costs no bits (an fp32 product is off by 2^-24 of the angle: 0.008 radians at position 131072).  Sine,
//     cosine and rotation stay in 64 bits up to the one rounding into q or the cache: an 8-bit code that an
//     fp32 rotation's error tips over is off by a whole step of 2^-3 (about one in a million values), and about one in 2^14
//     fp16 keys would be the wrong neighbour of a tie if it were rounded to fp32 first.
//   - Eight lanes a head: lane r holds dims 4 r .. + 3 and 32 + 4 r .. + 3, both halves of its four
//     pairs.  The block's largest value is three DPP steps, the codes two words a lane.
//   - Bound: launch latency for a decode step's rows (1.9 us for two), the bytes of qkv and q for prompts (16 sequences of
//     up to 330 rows, 33 MB: 8-10 us, and 2.2-4 for their copy to fp16).
#include "f8.hpp"
#include "mt_internal.hpp"

namespace mt {

namespace {

constexpr int KV_THREADS = 256;
constexpr uint32_t KV_OCTETS = KV_THREADS / 8;
// Most rows of a workgroup (5280 rows of 16 ragged prompts: one 9.4 us, two 9.0, four 9.6, eight 11.1).
constexpr uint32_t KV_ROWS = 2;

// cos and sin of the angle pos * freq.
__device__ __forceinline__ double2 turn(uint64_t pos, float freq) {
    double t = static_cast<double>(pos) * static_cast<double>(freq) * 0.15915494309189535;
    t -= rint(t);
    double s, c;
    sincospi(2.0 * t, &s, &c);
    return make_double2(c, s);
}

// d as fp32, towards zero and with the last bit set where that loses anything: a rounding of the result to fewer bits is the
// rounding of d.
__device__ __forceinline__ float to_odd(double d) {
    const float f = static_cast<float>(d);
    uint32_t u = __float_as_uint(f);
    if (static_cast<double>(f) != d) u = (u - (fabs(static_cast<double>(f)) > fabs(d) ? 1u : 0u)) | 1u;
    return __uint_as_float(u);
}

// Eight values x (dims d0 .. + 3 and d1 .. + 3 of a 64-wide row) into a cache row of type CT; every
// lane of the head's octet calls it.
template <int CT>
__device__ __forceinline__ void store_row(const float *x, void *cache, uint8_t *scales, size_t row, uint32_t d0, uint32_t d1,
                                          uint32_t r) {
    if constexpr (CT == DT_F32) {
        float *p = static_cast<float *>(cache) + row * 64;
        *reinterpret_cast<float4 *>(p + d0) = make_float4(x[0], x[1], x[2], x[3]);
        *reinterpret_cast<float4 *>(p + d1) = make_float4(x[4], x[5], x[6], x[7]);
    } else if constexpr (CT == DT_F16) {
        _Float16 *p = static_cast<_Float16 *>(cache) + row * 64;
        typedef _Float16 h4 __attribute__((ext_vector_type(4)));
        *reinterpret_cast<h4 *>(p + d0) = h4{(_Float16)x[0], (_Float16)x[1], (_Float16)x[2], (_Float16)x[3]};
        *reinterpret_cast<h4 *>(p + d1) = h4{(_Float16)x[4], (_Float16)x[5], (_Float16)x[6], (_Float16)x[7]};
    } else {
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) top = fmaxf(top, f8_abs(x[i]));
        const uint32_t s = f8_scale(octet_max(top));
        const float inv = f8_inv_pow2(s);
        uint8_t *p = static_cast<uint8_t *>(cache) + row * 64;
        *reinterpret_cast<uint32_t *>(p + d0) = f8_encode4(x[0], x[1], x[2], x[3], inv);
        *reinterpret_cast<uint32_t *>(p + d1) = f8_encode4(x[4], x[5], x[6], x[7], inv);
        if (r == 0) scales[row] = static_cast<uint8_t>(s);
    }
}

template <int CT>
__global__ __launch_bounds__(KV_THREADS) void rope_append_kernel(const float *qkv, uint32_t ldq, RowsArgs rows, uint32_t hq,
                                                                 uint32_t hkv, uint32_t offset, KvArgs kv,
                                                                 const float *inv_freq, float *q, uint32_t ldo,
                                                                 uint32_t per_group) {
    __shared__ double2 cs[KV_ROWS][32];
    const uint32_t tid = threadIdx.x, r = tid & 7, all = rows.B * rows.T;
    const uint32_t row0 = blockIdx.x * per_group, n = min(per_group, all - row0);
    if (tid < n * 32) {
        uint32_t b;
        uint64_t slot;
        rows.at(row0 + tid / 32, b, slot);
        cs[tid / 32][tid & 31] = turn(slot + offset, inv_freq[tid & 31]);
    }
    __syncthreads();
    const uint32_t heads = hq + 2 * hkv;
    for (uint32_t i = tid / 8; i < n * heads; i += KV_OCTETS) {
        const uint32_t m = i / heads, h = i - m * heads, row = row0 + m;
        uint32_t b;
        uint64_t slot;
        if (!rows.at(row, b, slot)) continue;
        const bool is_q = h < hq;
        if (is_q ? q == nullptr : slot >= kv.len) continue;
        const float *src = qkv + static_cast<size_t>(row) * ldq + h * 64 + 4 * r;
        const float4 lo = *reinterpret_cast<const float4 *>(src), hi = *reinterpret_cast<const float4 *>(src + 32);
        float x[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
        if (h < hq + hkv) {
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const double2 t = cs[m][4 * r + e];
                const double a = x[e], b2 = x[4 + e];
                const double lo2 = fma(-b2, t.y, a * t.x), hi2 = fma(a, t.y, b2 * t.x);
                // (a NaN among the odd ones stays one; infinities are exact)
                x[e] = CT != DT_F32 && !is_q ? to_odd(lo2) : static_cast<float>(lo2);
                x[4 + e] = CT != DT_F32 && !is_q ? to_odd(hi2) : static_cast<float>(hi2);
            }
        }
        if (is_q) {
            float *dst = q + static_cast<size_t>(row) * ldo + h * 64 + 4 * r;
            *reinterpret_cast<float4 *>(dst) = make_float4(x[0], x[1], x[2], x[3]);
            *reinterpret_cast<float4 *>(dst + 32) = make_float4(x[4], x[5], x[6], x[7]);
        } else {
            const bool is_k = h < hq + hkv;
            const uint32_t kh = is_k ? h - hq : h - hq - hkv;
            const size_t at = static_cast<size_t>(kh) * kv.len + slot;
            constexpr size_t ES = CT == DT_F32 ? 4 : CT == DT_F16 ? 2 : 1;
            char *cache = static_cast<char *>(is_k ? kv.k : kv.v) + b * kv.stride * ES;
            uint8_t *scales = CT == DT_F8 ? (is_k ? kv.ks : kv.vs) + b * kv.sstride : nullptr;
            store_row<CT>(x, cache, scales, at, 4 * r, 32 + 4 * r, r);
        }
    }
}

template <int ST, int CT>
__global__ __launch_bounds__(KV_THREADS) void kv_copy_kernel(KvArgs src, KvArgs dst, RowsArgs rows, uint32_t hkv) {
    const uint64_t i = static_cast<uint64_t>(blockIdx.x) * KV_OCTETS + threadIdx.x / 8;
    const uint32_t r = threadIdx.x & 7;
    const uint64_t all = static_cast<uint64_t>(rows.B) * rows.T * hkv * 2;
    if (i >= all) return;
    const uint32_t row = static_cast<uint32_t>(i / (2 * hkv)), h = static_cast<uint32_t>(i - static_cast<uint64_t>(row) * 2 * hkv);
    uint32_t b;
    uint64_t slot;
    if (!rows.at(row, b, slot) || slot >= src.len || slot >= dst.len) return;
    const bool is_k = h < hkv;
    const uint32_t kh = is_k ? h : h - hkv;
    const size_t from = static_cast<size_t>(kh) * src.len + slot, to = static_cast<size_t>(kh) * dst.len + slot;
    const void *sc = is_k ? src.k : src.v;
    void *dc = is_k ? dst.k : dst.v;
    const uint8_t *ss = ST == DT_F8 ? (is_k ? src.ks : src.vs) + b * src.sstride : nullptr;
    uint8_t *ds = CT == DT_F8 ? (is_k ? dst.ks : dst.vs) + b * dst.sstride : nullptr;
    if constexpr (ST == DT_F8 && CT == DT_F8) {
        const uint8_t *p = static_cast<const uint8_t *>(sc) + b * src.stride + from * 64 + 8 * r;
        uint8_t *o = static_cast<uint8_t *>(dc) + b * dst.stride + to * 64 + 8 * r;
        *reinterpret_cast<u32x2v *>(o) = *reinterpret_cast<const u32x2v *>(p);
        if (r == 0) ds[to] = ss[from];
        return;
    }
    float x[8];
    if constexpr (ST == DT_F32) {
        const float *p = static_cast<const float *>(sc) + b * src.stride + from * 64 + 8 * r;
        const float4 lo = *reinterpret_cast<const float4 *>(p), hi = *reinterpret_cast<const float4 *>(p + 4);
        x[0] = lo.x; x[1] = lo.y; x[2] = lo.z; x[3] = lo.w;
        x[4] = hi.x; x[5] = hi.y; x[6] = hi.z; x[7] = hi.w;
    } else if constexpr (ST == DT_F16) {
        const uint16_t *p = static_cast<const uint16_t *>(sc) + b * src.stride + from * 64 + 8 * r;
        unpack8<DT_F16>(*reinterpret_cast<const uint4 *>(p), x);
    } else {
        const uint8_t *p = static_cast<const uint8_t *>(sc) + b * src.stride + from * 64 + 8 * r;
        const u32x2v w = *reinterpret_cast<const u32x2v *>(p);
        const float s = f8_pow2(ss[from]);
        f8_decode4(w[0], s, x);
        f8_decode4(w[1], s, x + 4);
    }
    constexpr size_t ES = CT == DT_F32 ? 4 : CT == DT_F16 ? 2 : 1;
    store_row<CT>(x, static_cast<char *>(dc) + b * dst.stride * ES, ds, to, 8 * r, 8 * r + 4, r);
}

template <int ST>
void copy_from(const KvArgs &src, const KvArgs &dst, int dt, const RowsArgs &rows, uint32_t hkv, dim3 grid, hipStream_t stream) {
    if (dt == DT_F32)
        hipLaunchKernelGGL((kv_copy_kernel<ST, DT_F32>), grid, dim3(KV_THREADS), 0, stream, src, dst, rows, hkv);
    else if (dt == DT_F16)
        hipLaunchKernelGGL((kv_copy_kernel<ST, DT_F16>), grid, dim3(KV_THREADS), 0, stream, src, dst, rows, hkv);
    else
        hipLaunchKernelGGL((kv_copy_kernel<ST, DT_F8>), grid, dim3(KV_THREADS), 0, stream, src, dst, rows, hkv);
}

}  // namespace

int launch_rope_append(const float *qkv, uint32_t ldq, const RowsArgs &rows, uint32_t hq, uint32_t hkv, uint32_t offset,
                       const KvArgs &kv, int ct, const float *inv_freq, float *q, uint32_t ldo, hipStream_t stream) {
    const uint32_t all = rows.B * rows.T;
    // One row a workgroup while that leaves CUs free, else the rows that share the angles' set-up.
    const uint32_t per = all <= 512 ? 1 : KV_ROWS;
    const dim3 grid((all + per - 1) / per);
    const int rc = check_grid("rope append", grid.x, KV_THREADS);
    if (rc) return rc;
    if (ct == DT_F32)
        hipLaunchKernelGGL(rope_append_kernel<DT_F32>, grid, dim3(KV_THREADS), 0, stream, qkv, ldq, rows, hq, hkv, offset, kv,
                           inv_freq, q, ldo, per);
    else if (ct == DT_F16)
        hipLaunchKernelGGL(rope_append_kernel<DT_F16>, grid, dim3(KV_THREADS), 0, stream, qkv, ldq, rows, hq, hkv, offset, kv,
                           inv_freq, q, ldo, per);
    else
        hipLaunchKernelGGL(rope_append_kernel<DT_F8>, grid, dim3(KV_THREADS), 0, stream, qkv, ldq, rows, hq, hkv, offset, kv,
                           inv_freq, q, ldo, per);
    return check_launch("rope append");
}

int launch_kv_copy(const KvArgs &src, int st, const KvArgs &dst, int dt, const RowsArgs &rows, uint32_t hkv, hipStream_t stream) {
    const uint64_t octets = static_cast<uint64_t>(rows.B) * rows.T * hkv * 2;
    const dim3 grid(static_cast<uint32_t>((octets + KV_OCTETS - 1) / KV_OCTETS));
    const int rc = check_grid("kv copy", grid.x, KV_THREADS);
    if (rc) return rc;
    if (st == DT_F32) copy_from<DT_F32>(src, dst, dt, rows, hkv, grid, stream);
    else if (st == DT_F16) copy_from<DT_F16>(src, dst, dt, rows, hkv, grid, stream);
    else copy_from<DT_F8>(src, dst, dt, rows, hkv, grid, stream);
    return check_launch("kv copy");
}

}  // namespace mt
