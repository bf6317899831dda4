// Attention of B sequences, T query rows each, over keys that all of them share and then over their
// own (mt_attention_shared), for caches of fp32, fp16 and 8 bits.
#include <algorithm>

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
__device__ void attend_wave(const float *q, const HeadKv &h, uint32_t lo, uint32_t hi, float scale, float *out) {
    const uint32_t lane = threadIdx.x & 63;
    float m = -INFINITY, l = 0.0f, o = 0.0f;
    for (uint32_t k0 = lo; k0 < hi; k0 += 64) {
        const uint32_t key = k0 + lane;
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
        const uint32_t n = min(hi - k0, 64u);
        for (uint32_t j = 0; j < n; j++) {
            const uint32_t kj = k0 + j;
            const int own = kj >= h.prefix;
            const size_t slot = own ? kj - h.prefix : kj;
            o = fmaf(__shfl(p, static_cast<int>(j), 64), cached<CT>(h.v[own], h.vs[own], slot, lane), o);
        }
    }
    out[lane] = o / l;
}

// The keys of a row whose own slot is `slot`: [lo, hi) of the prefix and the own keys together (at most
// 2^30 of each).
__device__ __forceinline__ void row_keys(const SharedArgs &a, uint64_t slot, uint32_t &lo, uint32_t &hi) {
    hi = static_cast<uint32_t>(min(slot, static_cast<uint64_t>(a.kv.len - 1))) + 1 + a.prefix_len;
    lo = a.window > 0 && hi > a.window ? hi - a.window : 0;
}

// ---------------------------------------------------------------- matrix cores --

typedef float f32x4v __attribute__((ext_vector_type(4)));
typedef float f32x2v __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8t __attribute__((ext_vector_type(8)));

template <int CT>
struct Kind {
    static constexpr bool HALF = CT == DT_F16;          // the MFMA's type: fp16, else bf16
    static constexpr int NQ = CT == DT_F16 ? 2 : 3;     // pieces of q and of the weights
    static constexpr int NC = CT == DT_F32 ? 3 : 1;     // pieces of k and v
    static constexpr int KW = CT == DT_F8 ? 1 : CT == DT_F16 ? 2 : 4;  // 16-byte loads of a lane's 16 dims of a key
    static constexpr float PS = CT == DT_F16 ? 16384.0f : 1.0f;        // the weights' scale in their pieces
};

template <bool HALF>
__device__ __forceinline__ f32x4v mma(u32x4v a, u32x4v b, f32x4v c) {
    if constexpr (HALF)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8t, a), __builtin_bit_cast(f16x8t, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8t, a), __builtin_bit_cast(bf16x8t, b), c, 0, 0, 0);
}

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2v{a, b}, bf16x2t));
}
// A pair as three bf16 pieces (24 bits), or as two fp16 ones (22 bits).
template <int CT>
__device__ __forceinline__ void split2(float a, float b, uint32_t *p) {
    if constexpr (CT == DT_F16) {
        p[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(a, b));
        p[1] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2v{a - f16_lo(p[0]), b - f16_hi(p[0])}, f16x2t));
    } else {
        p[0] = pack_bf16(a, b);
        const float r = a - bf16_lo(p[0]), s = b - bf16_hi(p[0]);
        p[1] = pack_bf16(r, s);
        p[2] = pack_bf16(r - bf16_lo(p[1]), s - bf16_hi(p[1]));
    }
}
template <int CT>
__device__ __forceinline__ void split8(const float *x, u32x4v *p) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
        uint32_t w[3];
        split2<CT>(x[2 * e], x[2 * e + 1], w);
#pragma unroll
        for (int i = 0; i < Kind<CT>::NQ; i++) p[i][e] = w[i];
    }
}

// acc + c . q over the pieces' products that are not below 2^-24, the small ones first.
template <int CT>
__device__ __forceinline__ f32x4v dot(const u32x4v *c, const u32x4v *q, f32x4v acc) {
    constexpr bool H = Kind<CT>::HALF;
    if constexpr (CT == DT_F32) {
        acc = mma<H>(c[2], q[0], acc);
        acc = mma<H>(c[0], q[2], acc);
        acc = mma<H>(c[1], q[1], acc);
        acc = mma<H>(c[1], q[0], acc);
        acc = mma<H>(c[0], q[1], acc);
    } else {
#pragma unroll
        for (int i = Kind<CT>::NQ - 1; i > 0; i--) acc = mma<H>(c[0], q[i], acc);
    }
    return mma<H>(c[0], q[0], acc);
}

// The maximum over the four lanes 16 apart.
__device__ __forceinline__ float rows_max(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

constexpr int AS_WAVES = 8;
constexpr uint32_t AS_LD = 68;  // floats of a row in the waves' hand-over (64 and a 16-byte skew)

// A workgroup's rows (of all rows (sequence, t, head of the group) of one key head) and keys.
struct Item {
    uint32_t kvh, r0, r1;      // rows [r0, r1)
    uint32_t b;                // the sequence whose own keys are read
    uint32_t p0, p1, o0, o1;   // tiles of 32 prefix keys and of 32 own keys
    uint32_t split;            // apart: the part's place
};

template <int CT, int RT, bool APART>
__global__ __launch_bounds__(64 * AS_WAVES) void attention_shared_kernel(SharedArgs a) {
    typedef Kind<CT> KD;
    constexpr uint32_t ROW = Cached<CT>::ROW;
    extern __shared__ __attribute__((aligned(16))) float part[];  // [wave][16 RT][AS_LD], then [2][wave][16 RT]
    __shared__ uint32_t redo[AS_WAVES];
    const uint32_t tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, g = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t wk = wave % a.keys, wr = wave / a.keys, groups = AS_WAVES / a.keys;
    const uint32_t G = a.hq / a.hkv, T = a.rows.T, span = groups * 16 * RT;  // rows of a workgroup
    const uint32_t P = a.prefix_len;

    Item it;
    const uint32_t seq_tiles = (T * G + span - 1) / span;
    uint32_t x = blockIdx.x;
    bool own = true, pre = true;
    if constexpr (APART) {
        const uint32_t pre_items = a.sp * a.hkv * ((a.rows.B * T * G + span - 1) / span);
        own = x >= pre_items;
        pre = !own;
        if (own) x -= pre_items;
    }
    uint32_t parts = 1, mine = 0;
    if constexpr (APART) {
        parts = own ? a.so : a.sp;
        mine = x % parts;
        x /= parts;
    }
    it.kvh = x % a.hkv;
    x /= a.hkv;
    it.split = own ? a.sp + mine : mine;
    if (own) {
        it.b = x / seq_tiles;
        const uint32_t n = a.rows.counts ? min(a.rows.counts[it.b], T) : T;
        it.r0 = it.b * T * G + (x % seq_tiles) * span;
        it.r1 = min(it.b * T * G + n * G, it.r0 + span);
        if (it.r0 >= it.r1) return;
    } else {
        it.b = 0;
        it.r0 = x * span;
        it.r1 = min(a.rows.B * T * G, it.r0 + span);
    }

    // The wave's rows: their keys [lo, hi) of the prefix and the own keys together (none: not a row), and q.
    uint32_t lo[RT], hi[RT];
    u32x4v qf[RT][2][KD::NQ];
    float c[RT];
    const float c0 = a.scale * 1.4426950408889634f;
#pragma unroll
    for (int i = 0; i < RT; i++) {
        const uint32_t r = it.r0 + (wr * RT + i) * 16 + l16, row = r / G;
        uint32_t b = 0;
        uint64_t slot = 0;
        lo[i] = hi[i] = 0;
        float v[16];
#pragma unroll
        for (int e = 0; e < 16; e++) v[e] = 0.0f;
        if (r < it.r1 && a.rows.at(row, b, slot)) {
            row_keys(a, slot, lo[i], hi[i]);
            const float4 *p = reinterpret_cast<const float4 *>(a.q + static_cast<size_t>(row) * a.ldq + (it.kvh * G + r % G) * 64 + 16 * g);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float4 w = p[e];
                v[4 * e] = w.x; v[4 * e + 1] = w.y; v[4 * e + 2] = w.z; v[4 * e + 3] = w.w;
            }
        }
        float f = c0;
        c[i] = 1.0f;
        if constexpr (CT == DT_F16) {  // the row's largest |q| to 2^13 .. 2^14
            float mx = 0.0f;
#pragma unroll
            for (int e = 0; e < 16; e++) mx = fmaxf(mx, fabsf(v[e]));
            mx = rows_max(mx);
            const int ex = min(267 - static_cast<int>(__float_as_uint(mx) >> 23), 253);
            f = __uint_as_float(static_cast<uint32_t>(ex) << 23);
            c[i] = fabsf(c0) * __uint_as_float(static_cast<uint32_t>(254 - ex) << 23);
            if (c0 < 0.0f) f = -f;
        }
#pragma unroll
        for (int e = 0; e < 16; e++) v[e] *= f;
#pragma unroll
        for (int kk = 0; kk < 2; kk++) split8<CT>(v + 8 * kk, qf[i][kk]);
    }
    // What the rows have in common: keys from the smallest lo to the largest hi; those between inner_lo and inner_hi
    // belong to every row.
    uint32_t lo_all = ~0u, hi_all = 0, inner_lo[RT], inner_hi[RT];
#pragma unroll
    for (int i = 0; i < RT; i++) {
        uint32_t l = hi[i] ? lo[i] : ~0u, h = hi[i], il = lo[i], ih = hi[i] ? hi[i] : ~0u;
#pragma unroll
        for (int d = 1; d < 16; d *= 2) {
            l = min(l, static_cast<uint32_t>(__shfl_xor(static_cast<int>(l), d, 64)));
            h = max(h, static_cast<uint32_t>(__shfl_xor(static_cast<int>(h), d, 64)));
            il = max(il, static_cast<uint32_t>(__shfl_xor(static_cast<int>(il), d, 64)));
            ih = min(ih, static_cast<uint32_t>(__shfl_xor(static_cast<int>(ih), d, 64)));
        }
        lo_all = min(lo_all, static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(l)));
        hi_all = max(hi_all, static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(h)));
        inner_lo[i] = __builtin_amdgcn_readfirstlane(il);
        inner_hi[i] = __builtin_amdgcn_readfirstlane(ih);
    }
    // The wave's tiles: the rows' tiles, this workgroup's part of them, every `keys`-th of those.
    const bool any = hi_all > 0;
    const uint32_t pend = pre && any ? min(hi_all, P) : 0;
    const uint32_t oend = own && any && hi_all > P ? hi_all - P : 0;  // own keys end here
    it.p0 = pend ? min(lo_all, pend) / 32 : 0;
    it.p1 = (pend + 31) / 32;
    it.o0 = oend && lo_all > P ? (lo_all - P) / 32 : 0;
    it.o1 = (oend + 31) / 32;
    if constexpr (APART) {
        const uint32_t first = own ? it.o0 : it.p0, n = own ? it.o1 - it.o0 : it.p1 - it.p0;
        const uint32_t s0 = first + static_cast<uint32_t>(static_cast<uint64_t>(n) * mine / parts);
        const uint32_t s1 = first + static_cast<uint32_t>(static_cast<uint64_t>(n) * (mine + 1) / parts);
        if (own) it.o0 = s0, it.o1 = s1;
        else it.p0 = s0, it.p1 = s1;
    }
    const uint32_t np = it.p1 - it.p0, nt = np + (it.o1 - it.o0);

    const HeadKv h = head_kv<CT>(a, it.b, it.kvh);
    u32x4v kr[2 * KD::KW];
    uint32_t vr[8 * KD::KW];
    uint32_t ksc[2], vsc[2];
    // Tile t's keys: of slot s0, those past `end` re-read the last one.
    auto place = [&](uint32_t t, uint32_t &seg, uint32_t &s0, uint32_t &end) {
        seg = t >= np ? 1 : 0;
        s0 = 32 * (seg ? it.o0 + t - np : it.p0 + t);
        end = seg ? oend : pend;
    };
    auto loadk = [&](uint32_t t) {
        uint32_t seg, s0, end;
        place(t, seg, s0, end);
        const char *base = seg ? h.k[1] : h.k[0];
        const uint8_t *sc = seg ? h.ks[1] : h.ks[0];
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const uint32_t slot = min(s0 + 16 * u + l16, end - 1);
            const u32x4v *p = reinterpret_cast<const u32x4v *>(base + static_cast<size_t>(slot) * ROW + 16 * Cached<CT>::ES * g);
#pragma unroll
            for (int i = 0; i < KD::KW; i++) kr[u * KD::KW + i] = p[i];
            if constexpr (CT == DT_F8) ksc[u] = sc[slot];
        }
    };
    auto loadv = [&](uint32_t t) {
        uint32_t seg, s0, end;
        place(t, seg, s0, end);
        const char *base = (seg ? h.v[1] : h.v[0]) + 4 * Cached<CT>::ES * l16;
        const uint8_t *sc = seg ? h.vs[1] : h.vs[0];
        auto ld = [&](int j, uint32_t slot) {
            const char *p = base + static_cast<size_t>(slot) * ROW;
            if constexpr (CT == DT_F8) {
                vr[j] = *reinterpret_cast<const uint32_t *>(p);
            } else if constexpr (CT == DT_F16) {
                const u32x2v w = *reinterpret_cast<const u32x2v *>(p);
                vr[2 * j] = w[0];
                vr[2 * j + 1] = w[1];
            } else {
                const u32x4v w = *reinterpret_cast<const u32x4v *>(p);
#pragma unroll
                for (int e = 0; e < 4; e++) vr[4 * j + e] = w[e];
            }
        };
        if (s0 + 32 <= end) {
#pragma unroll
            for (int j = 0; j < 8; j++) ld(j, s0 + 16 * (j >> 2) + 4 * g + (j & 3));
            if constexpr (CT == DT_F8) {
#pragma unroll
                for (int u = 0; u < 2; u++) vsc[u] = *reinterpret_cast<const uint32_t *>(sc + s0 + 16 * u + 4 * g);
            }
        } else {
            if constexpr (CT == DT_F8) vsc[0] = vsc[1] = 0;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const uint32_t slot = min(s0 + 16 * (j >> 2) + 4 * g + (j & 3), end - 1);
                ld(j, slot);
                if constexpr (CT == DT_F8) vsc[j >> 2] |= static_cast<uint32_t>(sc[slot]) << (8 * (j & 3));
            }
        }
    };

    f32x4v o[RT][4];
    float sub[RT], ls[RT];
#pragma unroll
    for (int i = 0; i < RT; i++) {
        sub[i] = INFINITY;
        ls[i] = 0.0f;
#pragma unroll
        for (int d = 0; d < 4; d++) o[i][d] = f32x4v{0.f, 0.f, 0.f, 0.f};
    }
    uint32_t t = wk;
    if (t < nt) {
        loadk(t);
        loadv(t);
    }
    for (; t < nt; t += a.keys) {
        const uint32_t next = t + a.keys;
        uint32_t seg, s0, end;
        place(t, seg, s0, end);
        const uint32_t k0 = s0 + (seg ? P : 0), stop = end + (seg ? P : 0);
        f32x4v s[RT][2];
#pragma unroll
        for (int u = 0; u < 2; u++) {
#pragma unroll
            for (int i = 0; i < RT; i++) s[i][u] = f32x4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int kk = 0; kk < 2; kk++) {
                u32x4v kf[KD::NC];
                if constexpr (CT == DT_F8) {
                    const float f = f8_pow2(ksc[u]);
                    const uint32_t w0 = kr[u][2 * kk], w1 = kr[u][2 * kk + 1];
                    kf[0] = u32x4v{f8_bf16x2<false>(w0, f), f8_bf16x2<true>(w0, f), f8_bf16x2<false>(w1, f), f8_bf16x2<true>(w1, f)};
                } else if constexpr (CT == DT_F16) {
                    kf[0] = kr[2 * u + kk];
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const u32x4v w = kr[4 * u + 2 * kk + (e >> 1)];
                        uint32_t p[3];
                        split2<CT>(__uint_as_float(w[2 * (e & 1)]), __uint_as_float(w[2 * (e & 1) + 1]), p);
#pragma unroll
                        for (int i = 0; i < 3; i++) kf[i][e] = p[i];
                    }
                }
#pragma unroll
                for (int i = 0; i < RT; i++) s[i][u] = dot<CT>(kf, qf[i][kk], s[i][u]);
            }
        }
        if (next < nt) loadk(next);

        u32x4v pf[RT][KD::NQ];
        float al[RT];
#pragma unroll
        for (int i = 0; i < RT; i++) {
            if (!(k0 >= inner_lo[i] && k0 + 32 <= min(inner_hi[i], stop))) {
                // keys of the segment up to its end that lie in [lo, hi)
                const uint32_t top = min(hi[i], stop);
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const uint32_t key = k0 + 16 * u + 4 * g + r;
                        s[i][u][r] = key >= lo[i] && key < top ? s[i][u][r] : -INFINITY;
                    }
            }
            float mx = -INFINITY;
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int r = 0; r < 4; r++) mx = fmaxf(mx, s[i][u][r]);
            mx = rows_max(mx);
            const float sn = fminf(sub[i], -(mx * c[i]));
            al[i] = sn == sub[i] ? 1.0f : __builtin_amdgcn_exp2f(sn - sub[i]);
            sub[i] = sn;
            const float su = sn == INFINITY ? 0.0f : sn;
            float x8[8], sum = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                x8[j] = __builtin_amdgcn_exp2f(fmaf(s[i][j >> 2][j & 3], c[i], su));
                sum += x8[j];
            }
            ls[i] = fmaf(ls[i], al[i], sum);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                if constexpr (CT == DT_F8) x8[j] *= f8_pow2((vsc[j >> 2] >> (8 * (j & 3))) & 255u);
                else x8[j] *= KD::PS;
            }
            split8<CT>(x8, pf[i]);
        }

        // p . v: a tile's sum starts from zero and joins the running one in one rounding.
#pragma unroll
        for (int d = 0; d < 4; d++) {
            u32x4v vf[KD::NC];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if constexpr (CT == DT_F8) {
                    const uint32_t w = __builtin_amdgcn_perm(vr[2 * e + 1], vr[2 * e], d < 2 ? 0x05010400u : 0x07030602u);
                    vf[0][e] = d & 1 ? f8_bf16x2<true>(w, 1.0f) : f8_bf16x2<false>(w, 1.0f);
                } else if constexpr (CT == DT_F16) {
                    vf[0][e] = __builtin_amdgcn_perm(vr[2 * (2 * e + 1) + (d >> 1)], vr[2 * (2 * e) + (d >> 1)],
                                                     d & 1 ? 0x07060302u : 0x05040100u);
                } else {
                    uint32_t p[3];
                    split2<CT>(__uint_as_float(vr[4 * (2 * e) + d]), __uint_as_float(vr[4 * (2 * e + 1) + d]), p);
#pragma unroll
                    for (int i = 0; i < 3; i++) vf[i][e] = p[i];
                }
            }
#pragma unroll
            for (int i = 0; i < RT; i++) {
                const f32x4v ot = dot<CT>(vf, pf[i], f32x4v{0.f, 0.f, 0.f, 0.f});
#pragma unroll
                for (int r = 0; r < 4; r++) o[i][d][r] = fmaf(o[i][d][r], al[i], ot[r]);
            }
        }
        if (next < nt) loadv(next);
    }

    // The waves' parts of each row meet in wave order: a thread joins four dims of a row.
    float *ms = part + AS_WAVES * 16 * RT * AS_LD, *sums = ms + AS_WAVES * 16 * RT;
#pragma unroll
    for (int i = 0; i < RT; i++) {
        float *p = part + ((wave * RT + i) * 16 + l16) * AS_LD + 16 * g;
#pragma unroll
        for (int r = 0; r < 4; r++)
            *reinterpret_cast<float4 *>(p + 4 * r) = make_float4(o[i][0][r], o[i][1][r], o[i][2][r], o[i][3][r]);
        const float l = ls[i] + __shfl_xor(ls[i], 16, 64), all = l + __shfl_xor(l, 32, 64);
        if (g == 0) {
            ms[(wave * RT + i) * 16 + l16] = sub[i];
            sums[(wave * RT + i) * 16 + l16] = all;
        }
    }
    if (tid < AS_WAVES) redo[tid] = 0;
    __syncthreads();
    for (uint32_t j = tid; j < span * 16; j += 64 * AS_WAVES) {
        const uint32_t rr = j / 16, d4 = 4 * (j & 15), r = it.r0 + rr;  // row rr of the workgroup
        if (r >= it.r1) continue;
        const uint32_t row = r / G, head = it.kvh * G + r % G;
        uint32_t b;
        uint64_t slot;
        if (!a.rows.at(row, b, slot)) continue;
        // the row's place in its waves' parts: waves grp * keys + w, tile and row inside
        const uint32_t grp = rr / (16 * RT), in = rr - grp * 16 * RT;
        float m = INFINITY;
        for (uint32_t w = 0; w < a.keys; w++) m = fminf(m, ms[(grp * a.keys + w) * 16 * RT + in]);
        float l = 0.0f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        for (uint32_t w = 0; w < a.keys; w++) {
            const uint32_t at = (grp * a.keys + w) * 16 * RT + in;
            const float mw = ms[at], f = mw == INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mw);
            const float4 v = *reinterpret_cast<const float4 *>(part + at * AS_LD + d4);
            l = fmaf(sums[at], f, l);
            acc.x = fmaf(v.x, f, acc.x);
            acc.y = fmaf(v.y, f, acc.y);
            acc.z = fmaf(v.z, f, acc.z);
            acc.w = fmaf(v.w, f, acc.w);
        }
        if constexpr (APART) {
            const uint32_t S = a.sp + a.so;
            const size_t at = (static_cast<size_t>(row) * a.hq + head) * S + it.split;
            float2 *ml = reinterpret_cast<float2 *>(a.part + static_cast<size_t>(a.rows.B) * T * a.hq * S * 64);
            if (m != INFINITY) *reinterpret_cast<float4 *>(a.part + at * 64 + d4) = acc;
            if (d4 == 0) ml[at] = make_float2(m, l);
        } else {
            const float f = 1.0f / (l * KD::PS);
            acc.x *= f; acc.y *= f; acc.z *= f; acc.w *= f;
            if (fabsf(acc.x) < INFINITY && fabsf(acc.y) < INFINITY && fabsf(acc.z) < INFINITY && fabsf(acc.w) < INFINITY)
                *reinterpret_cast<float4 *>(a.out + static_cast<size_t>(row) * a.ldo + head * 64 + d4) = acc;
            else
                atomicOr(&redo[rr / 32], 1u << (rr % 32));
        }
    }
    if constexpr (!APART) {
        // Rows with an output that is not finite once more, each from its own keys alone.
        __syncthreads();
        for (uint32_t rr = wave; rr < span; rr += AS_WAVES) {
            if (!((redo[rr / 32] >> (rr % 32)) & 1)) continue;
            const uint32_t r = it.r0 + rr, row = r / G, head = it.kvh * G + r % G;
            uint32_t b;
            uint64_t slot;
            uint32_t l, e;
            a.rows.at(row, b, slot);
            row_keys(a, slot, l, e);
            attend_wave<CT>(a.q + static_cast<size_t>(row) * a.ldq + head * 64, h, l, e, a.scale,
                            a.out + static_cast<size_t>(row) * a.ldo + head * 64);
        }
    }
}

// The parts of a row and head, of which there are sp + so, joined: thread (p, d4) takes every 16th part's four dims.
template <int CT>
__global__ __launch_bounds__(256) void attention_join_kernel(SharedArgs a) {
    __shared__ float4 acc[16][16];
    __shared__ float sums[16], ms[16];
    const uint32_t tid = threadIdx.x, p = tid / 16, d4 = 4 * (tid & 15);
    const uint32_t row = blockIdx.x / a.hq, head = blockIdx.x - row * a.hq, S = a.sp + a.so;
    uint32_t b;
    uint64_t slot;
    uint32_t lo, hi;
    if (!a.rows.at(row, b, slot)) return;
    const size_t at = static_cast<size_t>(blockIdx.x) * S;
    const float2 *ml = reinterpret_cast<const float2 *>(a.part + static_cast<size_t>(a.rows.B) * a.rows.T * a.hq * S * 64) + at;
    const float *o = a.part + at * 64;
    float m = INFINITY, l = 0.0f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    for (uint32_t s = p; s < S; s += 16) {
        const float2 e = ml[s];
        if (e.x == INFINITY) continue;
        const float4 x = *reinterpret_cast<const float4 *>(o + static_cast<size_t>(s) * 64 + d4);
        const float mn = fminf(m, e.x);
        const float f = m == INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mn - m), k = __builtin_amdgcn_exp2f(mn - e.x);
        m = mn;
        l = fmaf(l, f, e.y * k);
        v.x = fmaf(v.x, f, x.x * k);
        v.y = fmaf(v.y, f, x.y * k);
        v.z = fmaf(v.z, f, x.z * k);
        v.w = fmaf(v.w, f, x.w * k);
    }
    acc[p][tid & 15] = v;
    if (d4 == 0) {
        sums[p] = l;
        ms[p] = m;
    }
    __syncthreads();
    if (tid >= 64) return;  // one wave joins the 16: lane d is dim d
    float mm = INFINITY;
#pragma unroll
    for (int i = 0; i < 16; i++) mm = fminf(mm, ms[i]);
    float total = 0.0f, x = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const float f = ms[i] == INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mm - ms[i]);
        total = fmaf(sums[i], f, total);
        x = fmaf(reinterpret_cast<const float *>(acc[i])[tid], f, x);
    }
    x *= 1.0f / (total * Kind<CT>::PS);
    float *out = a.out + static_cast<size_t>(row) * a.ldo + head * 64;
    if (__all(fabsf(x) < INFINITY)) {
        out[tid] = x;
        return;
    }
    row_keys(a, slot, lo, hi);
    attend_wave<CT>(a.q + static_cast<size_t>(row) * a.ldq + head * 64, head_kv<CT>(a, b, head / (a.hq / a.hkv)), lo, hi, a.scale, out);
}

template <int CT, int RT>
int launch_kind(const SharedArgs &a, bool apart, hipStream_t stream) {
    const uint32_t G = a.hq / a.hkv, span = AS_WAVES / a.keys * 16 * RT, B = a.rows.B, T = a.rows.T;
    const uint32_t lds = AS_WAVES * 16 * RT * (AS_LD + 2) * 4;
    const uint64_t own = static_cast<uint64_t>(B) * a.hkv * ((T * G + span - 1) / span);
    if (!apart) {
        hipLaunchKernelGGL((attention_shared_kernel<CT, RT, false>), dim3(static_cast<uint32_t>(own)), dim3(64 * AS_WAVES), lds, stream, a);
        return check_launch("attention shared");
    }
    const uint64_t pre = static_cast<uint64_t>(a.sp) * a.hkv * ((static_cast<uint64_t>(B) * T * G + span - 1) / span);
    hipLaunchKernelGGL((attention_shared_kernel<CT, RT, true>), dim3(static_cast<uint32_t>(pre + own * a.so)), dim3(64 * AS_WAVES), lds,
                       stream, a);
    int rc = check_launch("attention shared (parts)");
    if (rc) return rc;
    hipLaunchKernelGGL(attention_join_kernel<CT>, dim3(B * T * a.hq), dim3(256), 0, stream, a);
    return check_launch("attention shared (join)");
}

}  // namespace

SharedPlan shared_plan(uint32_t B, uint32_t T, uint32_t hq, uint32_t hkv, uint32_t prefix_len, uint32_t len_max, uint32_t window,
                       int ct) {
    const uint32_t G = hq / hkv;
    SharedPlan p{1, AS_WAVES, false, 0, 0};
    (void)ct;
    // keys an own row attends at most
    uint64_t own = len_max, pre = prefix_len;
    if (window) own = own < window ? own : window, pre = pre < window ? pre : window;
    const uint64_t rows = static_cast<uint64_t>(T) * G, tiles = (rows + 15) / 16;
    // waves that other rows can use
    while (p.keys > 1 && tiles * p.keys > AS_WAVES * 2) p.keys /= 2;
    const uint64_t span = AS_WAVES / p.keys * 16, groups = static_cast<uint64_t>(B) * hkv * ((rows + span - 1) / span);
    const uint64_t steps = (own + pre + 31) / 32 / p.keys;  // tiles a wave
    if (p.keys == AS_WAVES && groups < 256 && steps > 4) {
        p.apart = true;
        p.so = static_cast<uint32_t>(std::max<uint64_t>(1, std::min<uint64_t>((own + 255) / 256, 512 / groups)));
        const uint64_t pg = static_cast<uint64_t>(hkv) * ((B * rows + span - 1) / span);
        p.sp = pre ? static_cast<uint32_t>(std::max<uint64_t>(1, std::min<uint64_t>((pre + 255) / 256, 512 / pg))) : 0;
    }
    return p;
}

int launch_attention_shared(const SharedArgs &a, const SharedPlan &p, int ct, hipStream_t stream) {
    SharedArgs b = a;
    b.keys = p.keys;
    b.sp = p.sp;
    b.so = p.so;
    if (ct == DT_F32) return launch_kind<DT_F32, 1>(b, p.apart, stream);
    if (ct == DT_F16) return launch_kind<DT_F16, 1>(b, p.apart, stream);
    return launch_kind<DT_F8, 1>(b, p.apart, stream);
}

}  // namespace mt
