// Attention of B sequences, T query rows each, over their own keys in pages (mt_attention_paged) or in contiguous caches
// (mt_attention_sinks): all of them, or a sliding window and the first `sinks` ones.
//
// out = sum_j p_j v_j / sum_j p_j with p_j = exp(s_j - max s), s_j = scale q . k_j, over the slots j <= i of a row at slot i that have
// j > i - window or j < sinks.
//
//   - One wave a row and query head: 64 keys at a time, each lane a key's score, then each lane a dim's sum, an online softmax
//     in fp32.
#include <algorithm>
#include <type_traits>

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

// ---------------------------------------------------------------- matrix cores --

constexpr uint32_t AW_WAVES = 8, AW_FEW = 4;  // waves of a workgroup

// The key tiles of a row tile: those of the first keys, then those of the window (one run where they touch).
struct Tiles {
    uint32_t first, from, n;  // tiles before `first`, then tiles from `from` on; n of them
    uint32_t lo, hi;          // the keys that some row attends: [lo, hi) and those before a.sinks
    uint32_t in_lo, in_hi;    // those that all rows attend: [in_lo, in_hi) and those before min(a.sinks, in_hi)
    __device__ __forceinline__ uint32_t at(uint32_t i) const { return i < first ? i : from + (i - first); }
};

// Rows `top` .. `last` of sequence b (0 .. T - 1) together, TK keys a tile.
template <uint32_t TK>
__device__ __forceinline__ Tiles tiles_of(const WindowArgs &a, uint32_t b, uint32_t top, uint32_t last) {
    const uint64_t pos = a.rows.pos ? a.rows.pos[b] : 0u;
    Tiles t;
    uint32_t f;
    row_keys(a, pos + top, f, t.lo, t.in_hi);
    row_keys(a, pos + last, f, t.in_lo, t.hi);
    const uint32_t end = (t.hi + TK - 1) / TK;
    t.first = (min(a.sinks, t.lo) + TK - 1) / TK;
    t.from = max(t.lo / TK, t.first);
    t.n = t.first + (end - t.from);
    return t;
}

// A tile of keys in pieces of `LEN` slots, each within one page: where each stands, and how many of its slots some row may see.
template <int PIECES>
struct Pieces {
    uint64_t row[PIECES], scale[PIECES];  // as in find()
    uint32_t n[PIECES];
    uint32_t none;  // bit i: piece i has no page
};

// (the table is read through the scalar cache: nothing writes it while a kernel runs)
typedef const __attribute__((address_space(4))) uint32_t *ScalarTable;

template <bool PAGED, int PIECES, uint32_t TK>
__device__ __forceinline__ void entries_of(const WindowArgs &a, uint32_t b, uint32_t tile, uint32_t *page) {
    if constexpr (PAGED) {
        const ScalarTable table = (ScalarTable)(a.kv.table + static_cast<size_t>(b) * a.kv.table_stride);
#pragma unroll
        for (int i = 0; i < PIECES; i++) {
            const uint32_t s = min(tile * TK + i * (TK / PIECES), a.kv.len - 1);
            page[i] = table[a.kv.entry(s)];
        }
    }
}

template <bool PAGED, int PIECES, uint32_t TK>
__device__ __forceinline__ void pieces_of(const WindowArgs &a, const Tiles &t, uint32_t b, uint32_t kvh, uint32_t tile, bool have,
                                          const uint32_t *page, Pieces<PIECES> &p) {
    constexpr uint32_t LEN = TK / PIECES;
    p.none = 0;
#pragma unroll
    for (int i = 0; i < PIECES; i++) {
        const uint32_t s = tile * TK + i * LEN;
        uint64_t pg = b;
        uint32_t in = s;
        bool there = have && s < t.hi && (s < a.sinks || s + LEN > t.lo);
        if constexpr (PAGED) {
            pg = page[i];
            in -= a.kv.entry(s) * a.kv.page_len;
            if (page[i] >= a.kv.pages) {
                there = false;
                p.none |= 1u << i;
            }
        }
        if (!there) pg = in = 0;
        const uint64_t r = static_cast<uint64_t>(kvh) * a.kv.page_len + in;
        p.row[i] = pg * a.kv.stride + r * 64;
        p.scale[i] = pg * a.kv.sstride + r;
        p.n[i] = there ? min(t.hi - s, LEN) : 0;
    }
}

// The keys (values) of a tile's pieces; zeros, which the buffers' bounds give, for slots that no row sees and without a page.
template <int CT, int PIECES>
__device__ __forceinline__ void load_keys(Raw<CT> &r, const WindowArgs &a, const Pieces<PIECES> &p, uint32_t l16, uint32_t g) {
    constexpr uint32_t ROW = Cached<CT>::ROW;
    constexpr int GROUPS = 2 * Raw<CT>::SUB, EACH = GROUPS / PIECES;  // groups of 16 keys, those of a piece
#pragma unroll
    for (int i = 0; i < PIECES; i++) {
        const __amdgpu_buffer_rsrc_t b = span_of(static_cast<const char *>(a.kv.k) + p.row[i] * Cached<CT>::ES, p.n[i] * ROW);
#pragma unroll
        for (int u = 0; u < EACH; u++)
#pragma unroll
            for (int w = 0; w < Kind<CT>::KW; w++)
                r.k[(EACH * i + u) * Kind<CT>::KW + w] =
                    __builtin_amdgcn_raw_buffer_load_b128(b, l16 * ROW + 16 * Cached<CT>::ES * g + 16 * ROW * u + 16 * w, 0, 0);
        if constexpr (CT == DT_F8) {
            const __amdgpu_buffer_rsrc_t s = span_of(a.kv.ks + p.scale[i], p.n[i]);
#pragma unroll
            for (int u = 0; u < EACH; u++) r.ks[EACH * i + u] = __builtin_amdgcn_raw_buffer_load_b8(s, l16 + 16 * u, 0, 0);
        }
    }
}
template <int CT, int PIECES>
__device__ __forceinline__ void load_values(Raw<CT> &r, const WindowArgs &a, const Pieces<PIECES> &p, uint32_t l16, uint32_t g) {
    constexpr uint32_t ROW = Cached<CT>::ROW;
    constexpr int GROUPS = 2 * Raw<CT>::SUB, EACH = GROUPS / PIECES;
#pragma unroll
    for (int i = 0; i < PIECES; i++) {
        const __amdgpu_buffer_rsrc_t b = span_of(static_cast<const char *>(a.kv.v) + p.row[i] * Cached<CT>::ES, p.n[i] * ROW);
#pragma unroll
        for (int j = 0; j < 4 * EACH; j++) {
            const uint32_t at = 4 * g * ROW + 4 * Cached<CT>::ES * l16 + (16 * (j >> 2) + (j & 3)) * ROW;
            const int o = 4 * EACH * i + j;
            if constexpr (CT == DT_F8) {
                r.v[o] = __builtin_amdgcn_raw_buffer_load_b32(b, at, 0, 0);
            } else if constexpr (CT == DT_F16) {
                const u32x2v w = __builtin_amdgcn_raw_buffer_load_b64(b, at, 0, 0);
                r.v[2 * o] = w[0];
                r.v[2 * o + 1] = w[1];
            } else {
                const u32x4v w = __builtin_amdgcn_raw_buffer_load_b128(b, at, 0, 0);
#pragma unroll
                for (int e = 0; e < 4; e++) r.v[4 * o + e] = w[e];
            }
        }
        if constexpr (CT == DT_F8) {  // four keys' bytes a load: up to three past n, which the caches' whole words hold
            const __amdgpu_buffer_rsrc_t s = span_of(a.kv.vs + p.scale[i], (p.n[i] + 3) & ~3u);
#pragma unroll
            for (int u = 0; u < EACH; u++) r.vs[EACH * i + u] = __builtin_amdgcn_raw_buffer_load_b32(s, 4 * g + 16 * u, 0, 0);
        }
    }
}

// v / G (WindowArgs)
__device__ __forceinline__ uint32_t by_group(const WindowArgs &a, uint32_t v) {
    return a.group == 1 ? v : __umulhi(v, a.group_magic);
}

// Grid: x the sequences' row tiles, y the key heads, z the parts.
template <int CT, bool PAGED, int PIECES, bool APART, int WAVES>
__global__ __launch_bounds__(64 * WAVES, WAVES == 4 && CT != DT_F32 ? 3 : 2) void attention_window_kernel(WindowArgs a) {
    typedef Kind<CT> KD;
    constexpr int SUB = Raw<CT>::SUB;
    constexpr uint32_t TK = Raw<CT>::TK;
    __shared__ __attribute__((aligned(16))) float part[WAVES * 16 * AT_LD];
    __shared__ float ms[WAVES * 16], sums[WAVES * 16];
    __shared__ uint32_t redo[WAVES / 2];
    const uint32_t tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, g = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t wk = wave % a.keys, wr = wave / a.keys;
    const uint32_t G = a.group, T = a.rows.T, span = WAVES / a.keys * 16;  // rows of a workgroup

    // The workgroup's rows [r0, r1) of sequence b's rows (t, head of the group), the longest first.
    const uint32_t kvh = blockIdx.y, b = a.seq_tiles == 1 ? blockIdx.x : blockIdx.x / a.seq_tiles;
    const uint32_t n = a.rows.counts ? min(a.rows.counts[b], T) : T;
    const uint32_t r0 = (a.seq_tiles - 1 - (blockIdx.x - b * a.seq_tiles)) * span, r1 = min(n * G, r0 + span);
    if (r0 >= r1) return;

    // The lane's row (all four g's the same one), its query's 16 dims and its keys [lo, hi) and those before a.sinks.
    const uint32_t rw = r0 + wr * 16, r = rw + l16, t = by_group(a, r), head = kvh * G + r - t * G;
    const uint64_t pos = a.rows.pos ? a.rows.pos[b] : 0u;
    uint32_t lo = 0, hi = 0, first;
    float4 qv[4] = {};
    if (r < r1) {
        const float4 *p = reinterpret_cast<const float4 *>(a.q + (static_cast<size_t>(b) * T + t) * a.ldq + head * 64 + 16 * g);
#pragma unroll
        for (int e = 0; e < 4; e++) qv[e] = p[e];
        row_keys(a, pos + t, first, lo, hi);
    }
    Tiles tl{};
    uint32_t i = 0, end = 0;  // this wave's tiles: every keys-th one from i on
    if (rw < r1) {
        tl = tiles_of<TK>(a, b, by_group(a, rw), by_group(a, min(rw + 16, r1) - 1));
        end = tl.n;
        if constexpr (APART) {
            i = min(end, blockIdx.z * a.run);
            if (blockIdx.z + 1 < a.parts) end = min(end, i + a.run);
            if (i == end) return;  // (all waves alike: they share their rows)
        }
        i += wk;
    }

    Raw<CT> raw;
    uint32_t page[PIECES] = {};  // the entries of the tile after the one whose keys are on their way
    Pieces<PIECES> pc;
    auto entries = [&](uint32_t j) { entries_of<PAGED, PIECES, TK>(a, b, tl.at(min(j, end - 1)), page); };
    auto pieces = [&](uint32_t j) { pieces_of<PAGED, PIECES, TK>(a, tl, b, kvh, tl.at(min(j, end - 1)), j < end, page, pc); };
    // Loads of a tile past the last one are issued too, of no bytes: with as many loads in flight on every path, the waits for
    // the values leave the next keys on their way.
    if (end > 0) {
        entries(i);
        pieces(i);
        __builtin_amdgcn_sched_barrier(0);  // in this order, as in the loop, or its first wait is for all of them
        load_keys<CT>(raw, a, pc, l16, g);
        __builtin_amdgcn_sched_barrier(0);
        load_values<CT>(raw, a, pc, l16, g);
        __builtin_amdgcn_sched_barrier(0);
    }

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
    for (; i < end; i += a.keys) {
        const uint32_t k0 = tl.at(i) * TK, none = pc.none;
        entries(i + a.keys);
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
                        for (int x = 0; x < 3; x++) kf[u][x][e] = p[x];
                    }
                }
            }
            dots<CT, 2 * SUB>(kf, qf[kk], s);
        }
        pieces(i + a.keys);
        load_keys<CT>(raw, a, pc, l16, g);

        if (!((k0 >= tl.in_lo || k0 + TK <= a.sinks) && k0 + TK <= tl.in_hi) || none) {
#pragma unroll
            for (int u = 0; u < 2 * SUB; u++) {
                const uint32_t key = k0 + 16 * u + 4 * g;
                const uint32_t top = PAGED && (none >> (u * PIECES / (2 * SUB)) & 1) ? 0 : hi;
#pragma unroll
                for (int e = 0; e < 4; e++) s[u][e] = (key + e >= lo || key + e < a.sinks) && key + e < top ? s[u][e] : -INFINITY;
                if constexpr (CT == DT_F8) {  // a scale byte past the keys may stand for anything
                    const uint32_t k = tl.hi > key ? min(tl.hi - key, 4u) : 0;
                    raw.vs[u] &= k == 4 ? ~0u : (1u << (8 * k)) - 1;
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
        for (int x = 0; x < SUB; x++) {
            float p[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                p[j] = __builtin_amdgcn_exp2f(fmaf(s[2 * x + (j >> 2)][j & 3], c, su));
                sum += p[j];
            }
#pragma unroll
            for (int j = 0; j < 8; j++) {
                if constexpr (CT == DT_F8) p[j] *= f8_pow2((raw.vs[2 * x + (j >> 2)] >> (8 * (j & 3))) & 255u);
                else p[j] *= KD::PS;
            }
            split8<CT>(p, pf[x]);
        }
        ls = fmaf(ls, al, sum);

        // p . v: a tile's sum starts from zero and joins the running one in one rounding.
        f32x4v ot[4];
#pragma unroll
        for (int d = 0; d < 4; d++) ot[d] = f32x4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int x = 0; x < SUB; x++) {
            u32x4v vf[4][KD::NC];
#pragma unroll
            for (int d = 0; d < 4; d++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int j = 8 * x + 2 * e;
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
            dots<CT, 4>(vf, pf[x], ot);
        }
#pragma unroll
        for (int d = 0; d < 4; d++)
#pragma unroll
            for (int e = 0; e < 4; e++) o[d][e] = fmaf(o[d][e], al, ot[d][e]);
        load_values<CT>(raw, a, pc, l16, g);
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
        const uint32_t tj = by_group(a, rj), headj = kvh * G + rj - tj * G;
        const size_t row = static_cast<size_t>(b) * T + tj;
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
            const size_t at = (row * a.hq + headj) * a.parts + blockIdx.z;
            float2 *ml = reinterpret_cast<float2 *>(a.part + static_cast<size_t>(a.rows.B) * T * a.hq * a.parts * 64);
            *reinterpret_cast<float4 *>(a.part + at * 64 + d4) = acc;
            if (d4 == 0) ml[at] = make_float2(m, l);
        } else {
            const float f = 1.0f / (l * KD::PS);
            acc.x *= f; acc.y *= f; acc.z *= f; acc.w *= f;
            if (fabsf(acc.x) < INFINITY && fabsf(acc.y) < INFINITY && fabsf(acc.z) < INFINITY && fabsf(acc.w) < INFINITY)
                *reinterpret_cast<float4 *>(a.out + row * a.ldo + headj * 64 + d4) = acc;
            else
                atomicOr(&redo[rr / 32], 1u << (rr % 32));
        }
    }
    if constexpr (!APART) {
        // Rows with an output that is not finite (or without a weight) once more, each from its own keys alone.
        __syncthreads();
        for (uint32_t rr = wave; rr < span; rr += WAVES) {
            if (!((redo[rr / 32] >> (rr % 32)) & 1)) continue;
            const uint32_t rj = r0 + rr, tj = by_group(a, rj);
            attend_wave<CT>(a, b, b * T + tj, kvh * G + rj - tj * G, pos + tj);
        }
    }
}

// The parts of a row and head joined: lane d is dim d, a wave takes every waves-th part, and the waves' sums meet in wave order.
constexpr uint32_t AJ_WAVES = 16;  // at most

template <int CT>
__global__ __launch_bounds__(64 * AJ_WAVES) void window_join_kernel(WindowArgs a) {
    __shared__ float acc[AJ_WAVES][64], sums[AJ_WAVES], ms[AJ_WAVES];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x / 64;
    const uint32_t row = blockIdx.x, head = blockIdx.y;
    uint32_t b;
    uint64_t slot;
    if (!a.rows.at(row, b, slot)) return;
    // The parts that the row's tile has.
    const uint32_t t = row - b * a.rows.T, kvh = head / a.group, r = t * a.group + head - kvh * a.group;
    const uint32_t n = a.rows.counts ? min(a.rows.counts[b], a.rows.T) : a.rows.T, rw = r & ~15u;
    const Tiles tl = tiles_of<Raw<CT>::TK>(a, b, by_group(a, rw), by_group(a, min(rw + 16, n * a.group) - 1));
    const uint32_t S = min(a.parts, (tl.n + a.run - 1) / a.run);
    const size_t at = (static_cast<size_t>(row) * a.hq + head) * a.parts;
    const float2 *ml = reinterpret_cast<const float2 *>(a.part + static_cast<size_t>(a.rows.B) * a.rows.T * a.hq * a.parts * 64) + at;
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
    if (__all(fabsf(v) < INFINITY)) a.out[static_cast<size_t>(row) * a.ldo + head * 64 + lane] = v;
    else attend_wave<CT>(a, b, row, head, slot);
}

template <int CT, bool PAGED, int PIECES>
int launch_tiles(const WindowArgs &a, const WindowPlan &p, hipStream_t stream) {
    const dim3 grid(a.rows.B * a.seq_tiles, a.hkv, a.parts), block(64 * p.waves);
    if (a.parts > 1) hipLaunchKernelGGL((attention_window_kernel<CT, PAGED, PIECES, true, AW_FEW>), grid, block, 0, stream, a);
    else if (p.waves == AW_FEW) hipLaunchKernelGGL((attention_window_kernel<CT, PAGED, PIECES, false, AW_FEW>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((attention_window_kernel<CT, PAGED, PIECES, false, AW_WAVES>), grid, block, 0, stream, a);
    const int rc = check_launch("attention window");
    if (rc || a.parts == 1) return rc;
    hipLaunchKernelGGL(window_join_kernel<CT>, dim3(a.rows.B * a.rows.T, a.hq), dim3(64 * std::min(AJ_WAVES, (a.parts + 1) / 2)), 0, stream, a);
    return check_launch("attention window (join)");
}

template <int CT>
int launch_kind(const WindowArgs &a, const WindowPlan &p, hipStream_t stream) {
    constexpr int PIECES = Raw<CT>::TK / 16;
    if (!a.kv.table) return launch_tiles<CT, false, 1>(a, p, stream);
    // Pages that hold whole tiles: one page a tile.
    if (a.kv.page_len % Raw<CT>::TK == 0) return launch_tiles<CT, true, 1>(a, p, stream);
    return launch_tiles<CT, true, PIECES>(a, p, stream);
}

}  // namespace

// Where the work goes, from the sizes alone: 256 compute units are an MI355X's, not asked for, so that a workspace sized once
// fits wherever the call runs.
WindowPlan window_plan(uint32_t B, uint32_t T, uint32_t hq, uint32_t hkv, uint32_t len_max, uint32_t window, uint32_t sinks, int ct) {
    const uint64_t tk = ct == DT_F32 ? Raw<DT_F32>::TK : Raw<DT_F8>::TK, cus = 256;
    WindowPlan p{AW_WAVES, AW_WAVES, 1, 0};
    const uint64_t seen = window ? static_cast<uint64_t>(window) + sinks + T - 1 : len_max;
    const uint64_t own = std::max<uint64_t>(1, std::min<uint64_t>(len_max, seen));  // keys a row tile attends at most
    const uint64_t rows = static_cast<uint64_t>(T) * (hq / hkv), heads = static_cast<uint64_t>(B) * hkv;
    auto groups = [&](uint64_t waves, uint64_t keys) { return heads * ((rows + waves / keys * 16 - 1) / (waves / keys * 16)); };
    if (rows > 16 && groups(AW_WAVES, AW_WAVES) > cus) {
        p.waves = p.keys = AW_FEW;
        while (p.keys > 1 && groups(AW_FEW, p.keys) > 4 * cus && own < 4 * tk * p.keys) p.keys /= 2;
        return p;
    }
    const uint64_t all = groups(AW_WAVES, AW_WAVES);
    const uint64_t share = all * own / (2 * cus), part = std::max<uint64_t>(share, 256);  // keys a workgroup, two a CU
    const uint64_t so = std::min<uint64_t>(std::max<uint64_t>(1, own / part), 128);
    const uint64_t longest = std::max<uint64_t>(share, own / so);
    if (so > 1 && 2 * longest + 1200 < (all + cus - 1) / cus * own) {
        p.waves = p.keys = AW_FEW;
        p.parts = static_cast<uint32_t>(so);
        p.run = static_cast<uint32_t>((own + so * tk - 1) / (so * tk));
    }
    return p;
}

int launch_attention_window(const WindowArgs &args, const WindowPlan &p, int ct, hipStream_t stream) {
    WindowArgs a = args;
    a.keys = p.keys;
    a.parts = p.parts;
    a.run = p.run;
    const uint32_t span = p.waves / p.keys * 16;
    a.seq_tiles = (a.rows.T * a.group + span - 1) / span;
    int rc = check_grid("attention window", static_cast<uint64_t>(a.rows.B) * a.seq_tiles, 64 * p.waves);
    if (!rc && p.parts > 1) rc = check_grid("attention window (join)", static_cast<uint64_t>(a.rows.B) * a.rows.T, 64 * AJ_WAVES);
    if (rc) return rc;
    if (ct == DT_F32) return launch_kind<DT_F32>(a, p, stream);
    if (ct == DT_F16) return launch_kind<DT_F16>(a, p, stream);
    return launch_kind<DT_F8>(a, p, stream);
}

}  // namespace mt
