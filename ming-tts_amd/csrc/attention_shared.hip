// Attention of B sequences, T query rows each, over keys that all of them share and then over their
// own (mt_attention_shared), for caches of fp32, fp16 and 8 bits (f8.hpp).
//
// out = sum_j p_j v_j / sum_j p_j with p_j = 2^(s_j - max s), s_j = log2(e) scale q . k_j, over the keys of the row: one pass
// with a running maximum, on the matrix cores.
//
//   - Rows: the query heads of a key head's group are rows of their own, (sequence, t, head of the group) in order, 16 to
//     an MFMA tile, so a decode step's 7 heads read a key once and so do the rows of many sequences over the prefix.
//   - Scores: S^T = K Q^T with v_mfma_f32_16x16x32.  Lane (l16, g) reads dims 16 g .. + 15 of key l16 (one 16-byte load of an
//     8-bit row: 16 keys an instruction, whole rows); the dims' order is free as long as q follows it.  The accumulator gives
//     the lane keys 4 g .. + 3 of its own row l16, so the softmax is in-lane but for one exchange of the maximum a step.
//   - p . v: O^T = V^T P^T.  The weights stay where the scores stood; a lane reads dims 4 l16 .. + 3 of those keys' values and
//     byte permutes put two keys side by side.
//   - 8 bits: a key's codes become bf16 with its scale in the conversion (exact from scale byte 3 on); a value's scale goes
//     into its weight, whose pieces are then the weight times a power of two.  bf16 has the range for any scale, but its
//     steps end at 2^-133: what a weight's pieces lose there is below 2^-134, times a code below 2^-125 a key.
//   - Precision: q and the weights as three bf16 pieces (24 bits) against 8-bit and fp32 caches, those in three pieces too,
//     the 6 products above 2^-24; two fp16 pieces (22 bits) against fp16 caches.  All sums in fp32; a step's p . v starts from
//     zero and joins the running sum in one rounding.  Normwise error against fp64 1e-7 to 4e-7 up to 131072 keys (the plain fp32
//     form: 2e-7 to 2e-6).
//   - A step is 64 keys (32 of fp32), eight or four waves a workgroup take every keys-th one and meet in LDS in wave order.  The next
//     step's keys are requested behind the scores, its values behind p . v, through buffer descriptors that end with the keys:
//     what stands behind them is never read.  Keys inside that are not a row's (causal, window) weigh exactly zero;
//     where such a key or value is not finite, a row's outputs are not either, and it is done again from its own keys alone.
//     A NaN among a row's own scores is in the weights' sum, so the row is NaN wherever its keys are placed.
//   - Few rows over many keys, or a prefix for many sequences: parts of the keys go to workgroups of their own and a second
//     kernel joins them (shared_plan).  Sums meet in a fixed order everywhere: the same call gives the same bits.
//   - Bound: instructions.  A step of 64 8-bit keys is about 380 vector instructions and 48 MFMAs a wave whether 7 or 16 rows
//     are used (waves busy 60 %, waiting for memory 35 %), so long caches run at 2.2-3.2 TB/s where a large copy reaches
//     4.9; 128 sequences of up to 4096 keys (68 MB) take 20.4 us, 64 of them 15.6, one of 131072 15.6, the guided pair's step over
//     512 keys 6.1 (graph replay; an empty launch is 1.7), 1 prompt of 300 rows 6.8, of 2048 rows 34.
#include <algorithm>
#include <type_traits>

#include "attend_tiles.hpp"
#include "mt_internal.hpp"

namespace mt {

namespace {

// One head's keys and values: those of the shared prefix (slots 0 .. prefix - 1) and then a
// sequence's own.
struct HeadKv {
    const char *pk, *pv, *ok, *ov;          // prefix and own: the head's first row
    const uint8_t *pks, *pvs, *oks, *ovs;  // 8-bit caches: the head's first scale
    uint32_t prefix;
};

template <int CT>
__device__ __forceinline__ HeadKv head_kv(const SharedArgs &a, uint32_t b, uint32_t kvh) {
    HeadKv h{};
    const size_t own = b * a.kv.stride * Cached<CT>::ES + static_cast<size_t>(kvh) * a.kv.len * Cached<CT>::ROW;
    const size_t pre = static_cast<size_t>(kvh) * a.prefix.len * Cached<CT>::ROW;
    h.ok = static_cast<const char *>(a.kv.k) + own;
    h.ov = static_cast<const char *>(a.kv.v) + own;
    h.pk = static_cast<const char *>(a.prefix.k) + pre;
    h.pv = static_cast<const char *>(a.prefix.v) + pre;
    if constexpr (CT == DT_F8) {
        const size_t so = b * a.kv.sstride + static_cast<size_t>(kvh) * a.kv.len, sp = static_cast<size_t>(kvh) * a.prefix.len;
        h.oks = a.kv.ks + so;
        h.ovs = a.kv.vs + so;
        h.pks = a.prefix.ks + sp;
        h.pvs = a.prefix.vs + sp;
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
    else return bf16_lo(f8_bf16x2<false>(reinterpret_cast<const uint8_t *>(row)[e], 1.0f)) * f8_pow2(scales[slot]);
}

// One query head over keys [lo, hi) (prefix first) by one wave, touching those keys only: each lane a
// key's score, then each lane a dim's sum.  An online softmax in fp32, 64 keys at a time.  (The maximum takes no notice of
// NaN, so a NaN score has to become its weight by itself where no other score of its keys is above -infinity.)
template <int CT>
__device__ __forceinline__ void attend_wave(const float *q, const HeadKv &h, uint32_t lo, uint32_t hi, float scale, float *out) {
    const uint32_t lane = threadIdx.x & 63;
    float m = -INFINITY, l = 0.0f, o = 0.0f;
    for (uint32_t k0 = lo; k0 < hi; k0 += 64) {
        const uint32_t key = k0 + lane;
        float s = -INFINITY;
        if (key < hi) {
            const bool own = key >= h.prefix;
            const size_t slot = own ? key - h.prefix : key;
            float d = 0.0f;
            for (uint32_t e = 0; e < 64; e++) d = fmaf(q[e], cached<CT>(own ? h.ok : h.pk, own ? h.oks : h.pks, slot, e), d);
            s = d * scale;
        }
        const float mn = fmaxf(m, wave_max(s));
        const float al = m == -INFINITY ? 0.0f : exp_hw(m - mn);
        const float p = key >= hi ? 0.0f : mn == -INFINITY ? (s != s ? s : 0.0f) : exp_hw(s - mn);
        m = mn;
        l = fmaf(l, al, group_sum(p, 64));
        o *= al;
        const uint32_t n = min(hi - k0, 64u);
        for (uint32_t j = 0; j < n; j++) {
            const uint32_t kj = k0 + j;
            const bool own = kj >= h.prefix;
            const size_t slot = own ? kj - h.prefix : kj;
            o = fmaf(__shfl(p, static_cast<int>(j), 64), cached<CT>(own ? h.ov : h.pv, own ? h.ovs : h.pvs, slot, lane), o);
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

constexpr uint32_t AS_WAVES = 8, AS_FEW = 4;  // waves of a workgroup: all on one row tile's keys, or one of several

// The keys of n slots from `base` on (those past n: zeros, which the buffer's bound gives).
template <int CT>
__device__ __forceinline__ void load_keys(Raw<CT> &r, const char *base, const uint8_t *sc, uint32_t n, uint32_t l16, uint32_t g) {
    constexpr uint32_t ROW = Cached<CT>::ROW;
    const __amdgpu_buffer_rsrc_t b = span_of(base, n * ROW);
#pragma unroll
    for (int u = 0; u < 2 * Raw<CT>::SUB; u++)
#pragma unroll
        for (int i = 0; i < Kind<CT>::KW; i++)
            r.k[u * Kind<CT>::KW + i] = __builtin_amdgcn_raw_buffer_load_b128(b, l16 * ROW + 16 * Cached<CT>::ES * g + 16 * ROW * u + 16 * i, 0, 0);
    if constexpr (CT == DT_F8) {
        const __amdgpu_buffer_rsrc_t s = span_of(sc, n);
#pragma unroll
        for (int u = 0; u < 2 * Raw<CT>::SUB; u++) r.ks[u] = __builtin_amdgcn_raw_buffer_load_b8(s, l16 + 16 * u, 0, 0);
    }
}
template <int CT>
__device__ __forceinline__ void load_values(Raw<CT> &r, const char *base, const uint8_t *sc, uint32_t n, uint32_t l16, uint32_t g) {
    constexpr uint32_t ROW = Cached<CT>::ROW;
    const __amdgpu_buffer_rsrc_t b = span_of(base, n * ROW);
#pragma unroll
    for (int j = 0; j < 8 * Raw<CT>::SUB; j++) {
        const uint32_t at = 4 * g * ROW + 4 * Cached<CT>::ES * l16 + (16 * (j >> 2) + (j & 3)) * ROW;
        if constexpr (CT == DT_F8) {
            r.v[j] = __builtin_amdgcn_raw_buffer_load_b32(b, at, 0, 0);
        } else if constexpr (CT == DT_F16) {
            const u32x2v w = __builtin_amdgcn_raw_buffer_load_b64(b, at, 0, 0);
            r.v[2 * j] = w[0];
            r.v[2 * j + 1] = w[1];
        } else {
            const u32x4v w = __builtin_amdgcn_raw_buffer_load_b128(b, at, 0, 0);
#pragma unroll
            for (int e = 0; e < 4; e++) r.v[4 * j + e] = w[e];
        }
    }
    if constexpr (CT == DT_F8) {  // four keys' bytes a load: up to three past n, which the caches' whole words hold
        const __amdgpu_buffer_rsrc_t s = span_of(sc, (n + 3) & ~3u);
#pragma unroll
        for (int u = 0; u < 2 * Raw<CT>::SUB; u++) r.vs[u] = __builtin_amdgcn_raw_buffer_load_b32(s, 4 * g + 16 * u, 0, 0);
    }
}

// (at most 168 registers let three workgroups of four waves stand on a CU: eight prompts of 130 rows 24.1 -> 21.5 us)
template <int CT, bool APART, int WAVES>
__global__ __launch_bounds__(64 * WAVES, WAVES == 4 && CT != DT_F32 ? 3 : 2) void attention_shared_kernel(SharedArgs a) {
    typedef Kind<CT> KD;
    constexpr int SUB = Raw<CT>::SUB;
    constexpr uint32_t ROW = Cached<CT>::ROW, TK = Raw<CT>::TK;
    __shared__ __attribute__((aligned(16))) float part[WAVES * 16 * AT_LD];
    __shared__ float ms[WAVES * 16], sums[WAVES * 16];
    __shared__ uint32_t redo[WAVES / 2];
    const uint32_t tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, g = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t wk = wave % a.keys, wr = wave / a.keys;
    const uint32_t G = a.group, T = a.rows.T, span = WAVES / a.keys * 16;  // rows of a workgroup
    auto by_group = [&](uint32_t v) { return __umulhi(v, a.group_magic); };  // v / G (SharedArgs)
    const uint32_t P = a.prefix_len;

    // The workgroup's rows [r0, r1) of all rows (sequence, t, head of the group) of one key head, whose own keys are
    // sequence b's, and its part of the keys.
    const uint32_t seq_tiles = (T * G + span - 1) / span;
    uint32_t x = blockIdx.x, parts = 1, mine = 0;
    bool own = true, pre = P > 0;
    if constexpr (APART) {
        const uint32_t pre_items = a.sp * a.hkv * ((a.rows.B * T * G + span - 1) / span);
        own = x >= pre_items;
        pre = !own;
        if (own) x -= pre_items;
        parts = own ? a.so : a.sp;
        mine = x % parts;
        x /= parts;
    }
    const uint32_t kvh = x % a.hkv;
    x /= a.hkv;
    uint32_t b = 0, r0, r1;
    if (own) {
        b = x / seq_tiles;
        const uint32_t n = a.rows.counts ? min(a.rows.counts[b], T) : T;
        r0 = b * T * G + (seq_tiles - 1 - x % seq_tiles) * span;  // the longest rows first
        r1 = min(b * T * G + n * G, r0 + span);
        if (r0 >= r1) return;
    } else {
        r0 = x * span;
        r1 = min(a.rows.B * T * G, r0 + span);
    }

    // The lane's row (all four g's the same one), its query's 16 dims and its keys [lo, hi) of the prefix and the own
    // keys together (none: not a row).
    const uint32_t rw = r0 + wr * 16, r = rw + l16, row = G == 1 ? r : by_group(r), head = kvh * G + r - row * G;
    uint32_t lo = 0, hi = 0;
    float4 qv[4] = {};
    {
        uint32_t rb = b;
        uint64_t slot = 0;
        bool have = r < r1;
        if (own) slot = (a.rows.pos ? a.rows.pos[b] : 0u) + static_cast<uint64_t>(row - b * T);
        else have = have && a.rows.at(row, rb, slot);
        if (have) {
            const float4 *p = reinterpret_cast<const float4 *>(a.q + static_cast<size_t>(row) * a.ldq + head * 64 + 16 * g);
#pragma unroll
            for (int e = 0; e < 4; e++) qv[e] = p[e];
            row_keys(a, slot, lo, hi);
        }
    }
    // What the wave's rows have in common: keys from lo_all to hi_all, of which those from inner_lo to inner_hi belong to
    // every row.  A sequence's rows are in order; rows of many sequences differ by their windows.
    uint32_t lo_all = 0, hi_all = 0, inner_lo = 0, inner_hi = ~0u;
    if (own) {
        if (rw < r1) {
            const uint64_t at = a.rows.pos ? a.rows.pos[b] : 0u;
            const uint32_t top = min(rw + 16, r1) - 1;
            const uint32_t first = (G == 1 ? rw : by_group(rw)) - b * T, last = (G == 1 ? top : by_group(top)) - b * T;
            row_keys(a, at + first, lo_all, inner_hi);
            row_keys(a, at + last, inner_lo, hi_all);
        }
    } else if (a.window == 0) {
        hi_all = P;
    } else {
        uint32_t l = hi ? lo : ~0u, h = hi, il = lo;
#pragma unroll
        for (int d = 1; d < 16; d *= 2) {
            l = min(l, static_cast<uint32_t>(__shfl_xor(static_cast<int>(l), d, 64)));
            h = max(h, static_cast<uint32_t>(__shfl_xor(static_cast<int>(h), d, 64)));
            il = max(il, static_cast<uint32_t>(__shfl_xor(static_cast<int>(il), d, 64)));
        }
        lo_all = l;
        hi_all = h;
        inner_lo = il;
    }
    auto scalar = [](uint32_t &v) { v = __builtin_amdgcn_readfirstlane(v); };
    scalar(lo_all), scalar(hi_all), scalar(inner_lo), scalar(inner_hi);
    // Their tiles of TK keys, first those of the prefix, then the own ones: this workgroup's part of them, every keys-th.
    const uint32_t pend = pre ? min(hi_all, P) : 0, oend = own && hi_all > P ? hi_all - P : 0;
    uint32_t p0 = min(lo_all, pend) / TK, p1 = (pend + TK - 1) / TK;
    uint32_t o0 = oend && lo_all > P ? (lo_all - P) / TK : 0, o1 = (oend + TK - 1) / TK;
    if constexpr (APART) {
        // The prefix in equal parts; the own keys in runs of a.run tiles, the last part all that is left, so a workgroup's work
        // does not grow with its sequence.
        const uint32_t first = pick(own, p0, o0), last = pick(own, p1, o1), n = last - first;
        const uint32_t t0 = own ? min(last, first + mine * a.run) : first + n * mine / parts;  // below 2^25 tiles, 128 parts
        const uint32_t t1 = mine == parts - 1 ? last
                            : own             ? min(last, t0 + a.run)
                                              : first + n * (mine + 1) / parts;
        p0 = own ? 0 : t0;
        p1 = own ? 0 : t1;
        o0 = own ? t0 : 0;
        o1 = own ? t1 : 0;
    }
    scalar(p0), scalar(p1), scalar(o0), scalar(o1);
    const uint32_t np = p1 - p0, nt = np + (o1 - o0);
    if constexpr (APART) {
        if (nt == 0) {  // all waves alike (they share their rows): no key for any row
            if (tid < 16 && hi > 0) {
                const uint32_t S = a.sp + a.so;
                const size_t at = (static_cast<size_t>(row) * a.hq + head) * S + (own ? a.sp + mine : mine);
                reinterpret_cast<float2 *>(a.part + static_cast<size_t>(a.rows.B) * T * a.hq * S * 64)[at] = make_float2(INFINITY, 0.0f);
            }
            return;
        }
    }

    const HeadKv h = head_kv<CT>(a, b, kvh);
    Raw<CT> raw;
    auto tile = [&](uint32_t t, bool &seg, uint32_t &s0, uint32_t &end) {
        seg = t >= np;
        s0 = TK * pick(seg, p0 + t, o0 + t - np);
        end = pick(seg, pend, oend);
    };
    // Loads of a tile past the last one are issued too, of no bytes: with as many loads in flight on every path, the waits for
    // the values leave the next keys on their way.  (A branch around them made each a wait for all: 26.3 us against 25.0
    // for the eight prompts, 23.5 against 21.4 for 128 sequences of up to 4096 keys; a copy of the step without loads for
    // the last tile: 25.4 and 23.2.)
    auto keys = [&](uint32_t t) {
        bool seg;
        uint32_t s0, end;
        tile(t, seg, s0, end);
        load_keys<CT>(raw, pick(seg, h.pk, h.ok) + static_cast<size_t>(s0) * ROW, CT == DT_F8 ? pick(seg, h.pks, h.oks) + s0 : nullptr,
                      t < nt ? min(end - s0, TK) : 0, l16, g);
    };
    auto values = [&](uint32_t t) {
        bool seg;
        uint32_t s0, end;
        tile(t, seg, s0, end);
        load_values<CT>(raw, pick(seg, h.pv, h.ov) + static_cast<size_t>(s0) * ROW, CT == DT_F8 ? pick(seg, h.pvs, h.ovs) + s0 : nullptr,
                        t < nt ? min(end - s0, TK) : 0, l16, g);
    };
    uint32_t t = wk;
    __builtin_amdgcn_sched_barrier(0);  // in this order, as in the loop, or its first wait is for all of them
    keys(t);
    __builtin_amdgcn_sched_barrier(0);
    values(t);
    __builtin_amdgcn_sched_barrier(0);

    // The query as the operand's pieces, scaled so that the scores are base-2 exponents (fp16 pieces: times c).
    u32x4v qf[2][KD::NQ];
    const float c0 = a.scale * 1.4426950408889634f;
    float c = 1.0f;
    {
        float v[16];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            v[4 * e] = qv[e].x; v[4 * e + 1] = qv[e].y; v[4 * e + 2] = qv[e].z; v[4 * e + 3] = qv[e].w;
        }
        float f = c0;
        if constexpr (CT == DT_F16) {  // the row's largest |q| to 2^13 .. 2^14
            float mx = 0.0f;
#pragma unroll
            for (int e = 0; e < 16; e++) mx = fmaxf(mx, fabsf(v[e]));
            mx = rows_max(mx);
            const int ex = min(267 - static_cast<int>(__float_as_uint(mx) >> 23), 253);
            f = __uint_as_float(static_cast<uint32_t>(ex) << 23);
            c = fabsf(c0) * __uint_as_float(static_cast<uint32_t>(254 - ex) << 23);
            if (c < 0x1p-126f) c = 0x1p-126f;  // not 0, so that a key outside weighs 0 (-infinity times c); scores are below 2^37
            if (c0 < 0.0f) f = -f;
        }
#pragma unroll
        for (int e = 0; e < 16; e++) v[e] *= f;
#pragma unroll
        for (int kk = 0; kk < 2; kk++) split8<CT>(v + 8 * kk, qf[kk]);
    }

    f32x4v o[4];
    float sub = INFINITY, ls = 0.0f;  // minus the running maximum (+infinity: no key yet), the lane's share of the weights' sum
#pragma unroll
    for (int d = 0; d < 4; d++) o[d] = f32x4v{0.f, 0.f, 0.f, 0.f};
    for (; t < nt; t += a.keys) {
        const uint32_t next = t + a.keys;
        bool seg;
        uint32_t s0, end;
        tile(t, seg, s0, end);
        const uint32_t k0 = s0 + (seg ? P : 0), stop = end + (seg ? P : 0);
        f32x4v s[2 * SUB];
#pragma unroll
        for (int u = 0; u < 2 * SUB; u++) s[u] = f32x4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < 2; kk++) {
            u32x4v kf[2 * SUB][KD::NC];
#pragma unroll
            for (int u = 0; u < 2 * SUB; u++) {
                if constexpr (CT == DT_F8) {
                    const float f = f8_pow2(raw.ks[u]);
                    const uint32_t w0 = raw.k[u][2 * kk], w1 = raw.k[u][2 * kk + 1];
                    kf[u][0] = u32x4v{f8_bf16x2<false>(w0, f), f8_bf16x2<true>(w0, f), f8_bf16x2<false>(w1, f), f8_bf16x2<true>(w1, f)};
                } else if constexpr (CT == DT_F16) {
                    kf[u][0] = raw.k[2 * u + kk];
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const u32x4v w = raw.k[4 * u + 2 * kk + (e >> 1)];
                        uint32_t p[3];
                        split2<CT>(__uint_as_float(w[2 * (e & 1)]), __uint_as_float(w[2 * (e & 1) + 1]), p);
#pragma unroll
                        for (int i = 0; i < 3; i++) kf[u][i][e] = p[i];
                    }
                }
            }
            dots<CT, 2 * SUB>(kf, qf[kk], s);
        }
        keys(next);

        if (k0 < inner_lo || k0 + TK > min(inner_hi, stop)) {
            // keys of the segment up to its end that lie in [lo, hi)
            const uint32_t top = min(hi, stop);
#pragma unroll
            for (int u = 0; u < 2 * SUB; u++) {
                const uint32_t first = k0 + 16 * u + 4 * g;
#pragma unroll
                for (int e = 0; e < 4; e++) s[u][e] = first + e >= lo && first + e < top ? s[u][e] : -INFINITY;
                if constexpr (CT == DT_F8) {  // a scale byte past the segment may stand for anything
                    const uint32_t n = stop > first ? min(stop - first, 4u) : 0;
                    raw.vs[u] &= n == 4 ? ~0u : (1u << (8 * n)) - 1;
                }
            }
        }
        float mx = -INFINITY;
#pragma unroll
        for (int u = 0; u < 2 * SUB; u++)
#pragma unroll
            for (int e = 0; e < 4; e++) mx = fmaxf(mx, s[u][e]);
        mx = rows_max(mx);
        const float sn = fminf(sub, -(mx * c));
        const float al = sn == sub ? 1.0f : __builtin_amdgcn_exp2f(sn - sub);  // brings older sums to the new maximum
        sub = sn;
        const float su = sn == INFINITY ? 0.0f : sn;
        u32x4v pf[SUB][KD::NQ];
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < SUB; i++) {
            float p[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                p[j] = __builtin_amdgcn_exp2f(fmaf(s[2 * i + (j >> 2)][j & 3], c, su));
                sum += p[j];
            }
#pragma unroll
            for (int j = 0; j < 8; j++) {
                if constexpr (CT == DT_F8) p[j] *= f8_pow2((raw.vs[2 * i + (j >> 2)] >> (8 * (j & 3))) & 255u);
                else p[j] *= KD::PS;
            }
            split8<CT>(p, pf[i]);
        }
        ls = fmaf(ls, al, sum);

        // p . v: a tile's sum starts from zero and joins the running one in one rounding.
        f32x4v ot[4];
#pragma unroll
        for (int d = 0; d < 4; d++) ot[d] = f32x4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < SUB; i++) {
            u32x4v vf[4][KD::NC];
#pragma unroll
            for (int d = 0; d < 4; d++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int j = 8 * i + 2 * e;
                    if constexpr (CT == DT_F8) {
                        const uint32_t w = __builtin_amdgcn_perm(raw.v[j + 1], raw.v[j], d < 2 ? 0x05010400u : 0x07030602u);
                        vf[d][0][e] = d & 1 ? f8_bf16x2<true>(w, 1.0f) : f8_bf16x2<false>(w, 1.0f);
                    } else if constexpr (CT == DT_F16) {
                        vf[d][0][e] = __builtin_amdgcn_perm(raw.v[2 * (j + 1) + (d >> 1)], raw.v[2 * j + (d >> 1)],
                                                            d & 1 ? 0x07060302u : 0x05040100u);
                    } else {
                        uint32_t w[3];
                        split2<CT>(__uint_as_float(raw.v[4 * j + d]), __uint_as_float(raw.v[4 * (j + 1) + d]), w);
#pragma unroll
                        for (int q = 0; q < 3; q++) vf[d][q][e] = w[q];
                    }
                }
            dots<CT, 4>(vf, pf[i], ot);
        }
#pragma unroll
        for (int d = 0; d < 4; d++)
#pragma unroll
            for (int e = 0; e < 4; e++) o[d][e] = fmaf(o[d][e], al, ot[d][e]);
        values(next);
    }

    // The waves' parts of each row meet in wave order: a thread joins four dims of a row.
    {
        float *p = part + (wave * 16 + l16) * AT_LD + 16 * g;
#pragma unroll
        for (int e = 0; e < 4; e++) *reinterpret_cast<float4 *>(p + 4 * e) = make_float4(o[0][e], o[1][e], o[2][e], o[3][e]);
        const float l = ls + __shfl_xor(ls, 16, 64), all = l + __shfl_xor(l, 32, 64);
        if (g == 0) {
            ms[wave * 16 + l16] = sub;
            sums[wave * 16 + l16] = all;
        }
    }
    if (tid < WAVES / 2) redo[tid] = 0;
    __syncthreads();
    for (uint32_t j = tid; j < span * 16; j += 64 * WAVES) {
        const uint32_t rr = j / 16, d4 = 4 * (j & 15), rj = r0 + rr;  // row rr of the workgroup
        if (rj >= r1) continue;
        const uint32_t rowj = G == 1 ? rj : by_group(rj), headj = kvh * G + rj - rowj * G;
        if (!own) {
            uint32_t rb;
            uint64_t slot;
            if (!a.rows.at(rowj, rb, slot)) continue;
        }
        const uint32_t w0 = rr / 16 * a.keys, in = rr & 15;  // the row's waves, its place in each
        float m = INFINITY, l = 0.0f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        auto join = [&](auto count) {  // a count known here: all parts are read at once
            constexpr uint32_t N = decltype(count)::value;
            float mw[N], sw[N];
            float4 v[N];
#pragma unroll
            for (uint32_t w = 0; w < N; w++) {
                const uint32_t at = (w0 + w) * 16 + in;
                mw[w] = ms[at];
                sw[w] = sums[at];
                v[w] = *reinterpret_cast<const float4 *>(part + at * AT_LD + d4);
            }
#pragma unroll
            for (uint32_t w = 0; w < N; w++) m = fminf(m, mw[w]);
#pragma unroll
            for (uint32_t w = 0; w < N; w++) {
                const float f = mw[w] == INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mw[w]);
                l = fmaf(sw[w], f, l);
                acc.x = fmaf(v[w].x, f, acc.x);
                acc.y = fmaf(v[w].y, f, acc.y);
                acc.z = fmaf(v[w].z, f, acc.z);
                acc.w = fmaf(v[w].w, f, acc.w);
            }
        };
        if (a.keys == WAVES) join(std::integral_constant<uint32_t, WAVES>{});
        else if (a.keys == 2) join(std::integral_constant<uint32_t, 2>{});
        else join(std::integral_constant<uint32_t, 1>{});
        if constexpr (APART) {
            const uint32_t S = a.sp + a.so;
            const size_t at = (static_cast<size_t>(rowj) * a.hq + headj) * S + (own ? a.sp + mine : mine);
            float2 *ml = reinterpret_cast<float2 *>(a.part + static_cast<size_t>(a.rows.B) * T * a.hq * S * 64);
            *reinterpret_cast<float4 *>(a.part + at * 64 + d4) = acc;
            if (d4 == 0) ml[at] = make_float2(m, l);
        } else {
            const float f = 1.0f / (l * KD::PS);
            acc.x *= f; acc.y *= f; acc.z *= f; acc.w *= f;
            if (fabsf(acc.x) < INFINITY && fabsf(acc.y) < INFINITY && fabsf(acc.z) < INFINITY && fabsf(acc.w) < INFINITY)
                *reinterpret_cast<float4 *>(a.out + static_cast<size_t>(rowj) * a.ldo + headj * 64 + d4) = acc;
            else
                atomicOr(&redo[rr / 32], 1u << (rr % 32));
        }
    }
    if constexpr (!APART) {
        // Rows with an output that is not finite once more, each from its own keys alone.
        __syncthreads();
        for (uint32_t rr = wave; rr < span; rr += WAVES) {
            if (!((redo[rr / 32] >> (rr % 32)) & 1)) continue;
            const uint32_t rj = r0 + rr, rowj = G == 1 ? rj : by_group(rj), headj = kvh * G + rj - rowj * G;
            uint32_t rb;
            uint64_t slot;
            uint32_t l, e;
            a.rows.at(rowj, rb, slot);
            row_keys(a, slot, l, e);
            attend_wave<CT>(a.q + static_cast<size_t>(rowj) * a.ldq + headj * 64, h, l, e, a.scale,
                            a.out + static_cast<size_t>(rowj) * a.ldo + headj * 64);
        }
    }
}

// The parts of a row and head, of which there are sp + so, joined: lane d is dim d, a wave takes every waves-th part, and the
// waves' sums meet in wave order.
constexpr uint32_t AJ_WAVES = 16;  // at most

template <int CT>
__global__ __launch_bounds__(64 * AJ_WAVES) void attention_join_kernel(SharedArgs a) {
    __shared__ float acc[AJ_WAVES][64], sums[AJ_WAVES], ms[AJ_WAVES];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x / 64;
    const uint32_t row = blockIdx.x / a.hq, head = blockIdx.x - row * a.hq, S = a.sp + a.so;
    uint32_t b;
    uint64_t slot;
    if (!a.rows.at(row, b, slot)) return;
    const size_t at = static_cast<size_t>(blockIdx.x) * S;
    const float2 *ml = reinterpret_cast<const float2 *>(a.part + static_cast<size_t>(a.rows.B) * a.rows.T * a.hq * S * 64) + at;
    const float *o = a.part + at * 64 + lane;
    float m = INFINITY, l = 0.0f, v = 0.0f;
    for (uint32_t s0 = wave; s0 < S; s0 += 4 * waves) {  // four parts' loads at once
        float2 e[4];
        float x[4];
#pragma unroll
        for (uint32_t i = 0; i < 4; i++) {
            const uint32_t s = min(s0 + i * waves, S - 1);
            e[i] = ml[s];
            x[i] = o[static_cast<size_t>(s) * 64];
        }
#pragma unroll
        for (uint32_t i = 0; i < 4; i++) {
            // A part without a key of the row, or with scores of -infinity alone, has no sums; one of NaN scores alone has no
            // maximum either, but a sum that is NaN.
            if (s0 + i * waves >= S || (e[i].x == INFINITY && e[i].y == 0.0f)) continue;
            const float mn = fminf(m, e[i].x);
            const float f = m == INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mn - m), k = __builtin_amdgcn_exp2f(mn - e[i].x);
            m = mn;
            l = fmaf(l, f, e[i].y * k);
            v = fmaf(v, f, x[i] * k);
        }
    }
    if (waves > 1) {
        acc[wave][lane] = v;
        if (lane == 0) {
            sums[wave] = l;
            ms[wave] = m;
        }
        __syncthreads();
        if (wave > 0) return;
        m = INFINITY;
        for (uint32_t i = 0; i < waves; i++) m = fminf(m, ms[i]);
        l = v = 0.0f;
        for (uint32_t i = 0; i < waves; i++) {
            const float f = ms[i] == INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - ms[i]);
            l = fmaf(sums[i], f, l);
            v = fmaf(acc[i][lane], f, v);
        }
    }
    v *= 1.0f / (l * Kind<CT>::PS);
    float *out = a.out + static_cast<size_t>(row) * a.ldo + head * 64;
    if (__all(fabsf(v) < INFINITY)) {
        out[lane] = v;
        return;
    }
    uint32_t lo, hi;
    row_keys(a, slot, lo, hi);
    attend_wave<CT>(a.q + static_cast<size_t>(row) * a.ldq + head * 64, head_kv<CT>(a, b, head / a.group), lo, hi, a.scale, out);
}

template <int CT>
int launch_kind(const SharedArgs &a, const SharedPlan &p, hipStream_t stream) {
    const uint32_t span = p.waves / a.keys * 16, B = a.rows.B, T = a.rows.T;
    const uint64_t own = static_cast<uint64_t>(B) * a.hkv * ((T * a.group + span - 1) / span);
    const dim3 grid(static_cast<uint32_t>(own)), block(64 * p.waves);
    int rc;
    if (!p.apart) {
        rc = check_grid("attention shared", own, block.x);
        if (rc) return rc;
        if (p.waves == AS_WAVES) hipLaunchKernelGGL((attention_shared_kernel<CT, false, AS_WAVES>), grid, block, 0, stream, a);
        else hipLaunchKernelGGL((attention_shared_kernel<CT, false, AS_FEW>), grid, block, 0, stream, a);
        return check_launch("attention shared");
    }
    const uint64_t pre = static_cast<uint64_t>(a.sp) * a.hkv * ((static_cast<uint64_t>(B) * T * a.group + span - 1) / span);
    const uint32_t waves = std::min(AJ_WAVES, (a.sp + a.so + 1) / 2);
    rc = check_grid("attention shared (parts)", pre + own * a.so, block.x);
    if (!rc) rc = check_grid("attention shared (join)", static_cast<uint64_t>(B) * T * a.hq, 64 * waves);
    if (rc) return rc;
    hipLaunchKernelGGL((attention_shared_kernel<CT, true, AS_FEW>), dim3(static_cast<uint32_t>(pre + own * a.so)), block, 0, stream, a);
    rc = check_launch("attention shared (parts)");
    if (rc) return rc;
    hipLaunchKernelGGL(attention_join_kernel<CT>, dim3(B * T * a.hq), dim3(64 * waves), 0, stream, a);
    return check_launch("attention shared (join)");
}

}  // namespace

// Where the work goes, from the sizes alone: 256 compute units are an MI355X's, not asked for, so that a workspace sized once
// fits wherever the call runs.  A CU holds one workgroup of eight waves, or of four waves three with 8-bit and fp16 caches
// (at most 168 registers a lane) and two with fp32 ones (184); the rule is measured on 8 bits and used for all three.
// Eight waves take about 2 us for each 512 keys of their rows, and the second kernel of the split form costs about as much
// as 1200 keys.
//   - One row tile (16 rows) a workgroup of eight waves that split its keys, while that fills at most every CU once: 4
//     sequences of 40 rows over 500 + 300 keys (144 workgroups) 8.8 us, with two tiles a workgroup 13.2, four 19.4.
//   - More row tiles: four waves a tile, and two or four tiles a workgroup only where that would leave a wave less
//     than four steps.  Eight prompts of 130 rows over 1000 + 256 keys (912 tiles) 21.1 us, two tiles a workgroup 24.4,
//     eight waves 25.3; 1 of 2048 rows 37.7, 50.1; but 8 of 512 rows (1 to 8 steps) 28.3, four tiles a workgroup 25.1.
//     The longest rows go first (2048 rows 37.7 -> 35.4).
//   - apart: all keys of the prefix (once for all rows) and of the sequences spread over the CUs evenly, if the
//     longest workgroup then costs less than the longest in one pass.  Measured, one pass against apart: 64 sequences
//     of up to 4096 keys 21.0 against 16.2 us, 128 of them 20.8 against 26, 16 sequences over 8192 + 512 keys
//     36.5 against 11.5, 128 over 2048 + 512 14.9 against 14.7, 256 over 4096 + 1024 47 against 29.3.
// What the estimate does not see: parts are whole, and a key costs the same whether 7 or 16 rows of a tile use it.  So the choice
// is not steady where the two forms cost about the same: over 2048 + 512 keys up to 64 sequences share the prefix, 96 and 128 do
// not, 129 to 160 do, 192 to 256 do not.  Row tiles of many rows (the second rule) never share it; only one row a sequence and
// prompts were measured there, nothing between.
SharedPlan shared_plan(uint32_t B, uint32_t T, uint32_t hq, uint32_t hkv, uint32_t prefix_len, uint32_t len_max, uint32_t window,
                       int ct) {
    const uint64_t tk = ct == DT_F32 ? Raw<DT_F32>::TK : Raw<DT_F8>::TK, cus = 256;
    SharedPlan p{AS_WAVES, AS_WAVES, false, 0, 0, 0};
    // keys a row attends at most
    const uint64_t own = std::max<uint64_t>(1, window ? std::min<uint64_t>(len_max, static_cast<uint64_t>(window) + T - 1) : len_max);
    const uint64_t pre = window ? std::min(prefix_len, window) : prefix_len;
    const uint64_t rows = static_cast<uint64_t>(T) * (hq / hkv), heads = static_cast<uint64_t>(B) * hkv;
    auto groups = [&](uint64_t waves, uint64_t keys) { return heads * ((rows + waves / keys * 16 - 1) / (waves / keys * 16)); };
    if (rows > 16 && groups(AS_WAVES, AS_WAVES) > cus) {
        p.waves = p.keys = AS_FEW;
        while (p.keys > 1 && groups(AS_FEW, p.keys) > 4 * cus && pre + own < 4 * tk * p.keys) p.keys /= 2;
        return p;
    }
    const uint64_t own_groups = groups(AS_WAVES, AS_WAVES), pre_groups = pre ? hkv * ((B * rows + 15) / 16) : 0;
    const uint64_t share = (pre_groups * pre + own_groups * own) / (2 * cus), part = std::max<uint64_t>(share, 256);  // keys a workgroup, two a CU
    // At most 128 parts each, or the second kernel becomes the longer one.
    const uint64_t sp = pre ? std::min<uint64_t>(std::max<uint64_t>(1, pre / part), 128) : 0;
    const uint64_t so = std::min<uint64_t>(std::max<uint64_t>(1, own / part), 128);
    const uint64_t longest = std::max({share, pre ? pre / sp : 0, own / so});
    if (2 * longest + 1200 < (own_groups + cus - 1) / cus * (pre + own)) {
        p.apart = true;
        p.waves = p.keys = AS_FEW;
        p.sp = static_cast<uint32_t>(sp);
        p.so = static_cast<uint32_t>(so);
        p.run = static_cast<uint32_t>((own + so * tk - 1) / (so * tk));
    }
    return p;
}

int launch_attention_shared(const SharedArgs &a, const SharedPlan &p, int ct, hipStream_t stream) {
    SharedArgs b = a;
    b.keys = p.keys;
    b.sp = p.sp;
    b.so = p.so;
    b.run = p.run;
    b.group = a.hq / a.hkv;
    b.group_magic = static_cast<uint32_t>((1ull << 32) / b.group + 1);
    if (ct == DT_F32) return launch_kind<DT_F32>(b, p, stream);
    if (ct == DT_F16) return launch_kind<DT_F16>(b, p, stream);
    return launch_kind<DT_F8>(b, p, stream);
}

}  // namespace mt
