// Attention of B sequences, T query rows each, over their own keys in pages (mt_attention_paged) or in contiguous caches
// (mt_attention_sinks): all of them, or a sliding window and the first `sinks` ones.
//
// out = sum_j p_j v_j / sum_j p_j with p_j = exp(s_j - max s), s_j = scale q . k_j, over the slots j <= i of a row at slot i that have
// j > i - window or j < sinks.
//
// Scores and weights on the matrix cores (16 x 16 x 32), to about fp32's accuracy: q and the weights p as two fp16 pieces against fp16
// caches (K, V exact), as three bf16 pieces against 8-bit ones (K, V times a power of two exact in bf16) and against fp32 ones (three
// pieces too, the six products that matter).  A tile's p . v starts from zero and joins the running sum in one rounding: the
// matrix cores cut where they add.  The softmax is one pass over the keys with a running reference and sum in fp32.
//
//   - A tile is 16 rows (tokens times the heads that share a key head, so a decode step of 7 heads a key head fills 7 of them) by 64
//     keys (fp32: 32).  S = K q^T, with keys as the matrix's rows: a lane then has 4 consecutive keys of one row, which are
//     the weights' operand of p . v as they stand.
//   - Few rows (attention_window_kernel): bytes bound.  A wave streams its own tiles, the next tile's keys and values on their way
//     while one is worked on; the waves of a workgroup take tiles in turn and meet in LDS, and where there are few workgroups the keys
//     are split over several, which meet in the one that ends last.  In a graph 256 sequences of up to 4096 slots take 61 us in
//     fp16, 4.4 TB/s of keys and values (a large copy: 5.0); 64 of them 18.8; one of 131072 slots 20; two of 512 6.6, of
//     which 1.7 are an empty launch and the rest loads that wait for each other: position, table, keys, values.
//   - Many rows (window_rows_kernel): bound by its products and the instructions around them.  A 16 x 64 tile of fp16 keys is 32
//     matrix instructions of 16 cycles and about 400 cycles of others; they overlap by half.  One prompt of 8192 rows: 256 us, 470
//     TFLOP/s counted as one product each of q k and p v (940 as computed, a large fp16 product: 1510).
//   - Rows whose result is not finite, or without a weight, are computed once more by themselves, from their own keys alone
//     (attend_wave): tiles hold slots that a row does not attend, whose NaN would reach it through a weight of zero.
#include <algorithm>
#include <atomic>
#include <chrono>
#include <cmath>
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

// v / G (WindowArgs)
__device__ __forceinline__ uint32_t by_group(const WindowArgs &a, uint32_t v) {
    return a.group == 1 ? v : __umulhi(v, a.group_magic);
}

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

// Where a run of LEN slots within one page stands: bytes from the caches' (and scales') start, and how many of its slots some row may
// see.  A wave holds 64 of them, a lane each, made at once: what a tile needs are lane reads and additions (address arithmetic a
// tile, on scalars, was 280 scalar instructions a tile beside 210 vector ones).
struct Spans {
    uint32_t lo, hi, n, scale_lo, scale_hi;
    uint64_t holes;  // lanes whose run has no page
    static __device__ __forceinline__ uint32_t lane_of(uint32_t v, uint32_t i) {
        return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), static_cast<int>(i)));
    }
    __device__ __forceinline__ uint64_t at(uint32_t i) const { return lane_of(lo, i) | static_cast<uint64_t>(lane_of(hi, i)) << 32; }
    __device__ __forceinline__ uint64_t scale(uint32_t i) const {
        return lane_of(scale_lo, i) | static_cast<uint64_t>(lane_of(scale_hi, i)) << 32;
    }
    __device__ __forceinline__ uint32_t rows(uint32_t i) const { return lane_of(n, i); }
};

// The table's entry of slot s of sequence b.
template <bool PAGED>
__device__ __forceinline__ uint32_t entry_of(const WindowArgs &a, uint32_t b, uint32_t s) {
    if constexpr (!PAGED) return b;
    return a.kv.table[static_cast<size_t>(b) * a.kv.table_stride + a.kv.entry(min(s, a.kv.len - 1))];
}

// The lane's run: LEN slots from s on (none, unless `have`), of the given entry.
template <int CT, bool PAGED, uint32_t LEN>
__device__ __forceinline__ Spans span_run(const WindowArgs &a, const Tiles &t, uint32_t kvh, uint32_t s, bool have, uint32_t entry) {
    const bool bad = PAGED && entry >= a.kv.pages, there = have && !bad && s < t.hi && (s < a.sinks || s + LEN > t.lo);
    const uint64_t page = there ? entry : 0u, in = there ? s - (PAGED ? a.kv.entry(s) * a.kv.page_len : 0u) : 0u;
    const uint64_t at = static_cast<uint64_t>(kvh) * a.kv.page_len + in, byte = (page * a.kv.stride + at * 64) * Cached<CT>::ES;
    Spans p{};
    p.lo = static_cast<uint32_t>(byte);
    p.hi = static_cast<uint32_t>(byte >> 32);
    if constexpr (CT == DT_F8) {
        const uint64_t sc = page * a.kv.sstride + at;
        p.scale_lo = static_cast<uint32_t>(sc);
        p.scale_hi = static_cast<uint32_t>(sc >> 32);
    }
    p.n = there ? min(t.hi - s, LEN) : 0;
    p.holes = PAGED ? __ballot(bad) : 0;
    return p;
}

// A row's query as the operand's pieces, scaled so that the scores are base-2 exponents (`scaled`: times c, 1 / c = unit).  Lane
// (l16, g) holds dims 16 g .. + 15, or, in halves, 8 g .. + 7 and 32 + 8 g .. + 7.
template <int CT>
struct Query {
    u32x4v f[2][Kind<CT>::NQ];
    float c, unit;
    bool scaled;
};
struct RawQuery {
    float4 v[4];
};
template <bool HALVES>
__device__ __forceinline__ RawQuery load_query(const float *q, uint32_t g, bool have) {
    const float4 *p = reinterpret_cast<const float4 *>(q + (HALVES ? 8 : 16) * g);
    RawQuery r;
#pragma unroll
    for (int e = 0; e < 4; e++) r.v[e] = have ? p[HALVES ? 8 * (e / 2) + (e & 1) : e] : make_float4(0.f, 0.f, 0.f, 0.f);
    return r;
}
template <int CT>
__device__ __forceinline__ Query<CT> query_of(const RawQuery &r, float scale) {
    Query<CT> x;
    float v[16];
#pragma unroll
    for (int e = 0; e < 4; e++) {
        v[4 * e] = r.v[e].x; v[4 * e + 1] = r.v[e].y; v[4 * e + 2] = r.v[e].z; v[4 * e + 3] = r.v[e].w;
    }
    const float c0 = scale * 1.4426950408889634f;
    float f = c0;
    x.c = x.unit = 1.0f;
    x.scaled = false;
    if constexpr (CT == DT_F16) {
        float mx = 0.0f;
#pragma unroll
        for (int e = 0; e < 16; e++) mx = fmaxf(mx, fabsf(v[e]));
        mx = rows_max(mx);
        // Two pieces hold 22 bits of q times the scale where the row's largest is 1/8 to 2^14, or next to nothing.
        const float top = mx * fabsf(c0);
        x.scaled = __any(!(top >= 0.125f && top < 16384.0f) && top != 0.0f);
        if (x.scaled) {  // the row's largest |q| to 2^13 .. 2^14
            const int ex = min(267 - static_cast<int>(__float_as_uint(mx) >> 23), 253);
            f = __uint_as_float(static_cast<uint32_t>(ex) << 23);
            // (not 0: scores times less than 2^-100 are next to nothing all the same, being below 2^37)
            x.c = fmaxf(fabsf(c0) * __uint_as_float(static_cast<uint32_t>(254 - ex) << 23), 0x1p-100f);
            x.unit = 1.0f / x.c;
            if (c0 < 0.0f) f = -f;
        }
    }
#pragma unroll
    for (int e = 0; e < 16; e++) v[e] *= f;
#pragma unroll
    for (int kk = 0; kk < 2; kk++) split8<CT>(v + 8 * kk, x.f[kk]);
    return x;
}

// The running sums of a row.  Weights are 2^(s + ref) of its scores s (as base-2 exponents): ref brings the largest score so far to
// BASE, or, since it changes only where a score would be past BASE + AHEAD, to BASE + AHEAD at most, once the row has a score
// (begun).  Most tiles then neither rescale the sums nor subtract a maximum: `below`, ref as the products' starting sum, does that.
// Weights of fp16 pieces are up to 2^15; one of 2^-21 of the largest or less loses what is below 2^-31 of that.
constexpr float AHEAD = 8.0f;
template <int CT>
constexpr float BASE = CT == DT_F16 ? 7.0f : 0.0f;

struct Sums {
    float ref = 0.0f, ls = 0.0f;  // ls: the lane's share of the weights' sum
    bool begun = false;
    f32x4v below = {0.f, 0.f, 0.f, 0.f}, o[4] = {};  // o[d]: dims 16 d + 4 g .. + 3 (or those of load_values)
    // What the join of parts takes: minus the reference, or infinity.
    __device__ __forceinline__ float mark() const { return begun ? ref : INFINITY; }
};

// Scores s[u][e], of key 16 u + 4 g + e of a tile from slot k0 on, that the row (or, from `top` on, none) does not see.
template <int NK>
__device__ __forceinline__ void hide(f32x4v (&s)[NK], uint32_t k0, uint32_t g, uint32_t lo, uint32_t hi, uint32_t sinks, uint32_t none, int runs) {
#pragma unroll
    for (int u = 0; u < NK; u++) {
        const uint32_t key = k0 + 16 * u + 4 * g, top = (none >> (u * runs / NK)) & 1 ? 0 : hi;
#pragma unroll
        for (int e = 0; e < 4; e++) s[u][e] = (key + e >= lo || key + e < sinks) && key + e < top ? s[u][e] : -INFINITY;
    }
}

// The scores' reference, a new one where they need it.
template <int CT, int NK>
__device__ __forceinline__ void refer(f32x4v (&s)[NK], Sums &m, float unit) {
    float mx = -INFINITY;
#pragma unroll
    for (int u = 0; u < NK; u++)
#pragma unroll
        for (int e = 0; e < 4; e++) mx = fmaxf(mx, s[u][e]);
    if (!__any(mx > (m.begun ? BASE<CT> + AHEAD : -INFINITY))) return;
    mx = rows_max(mx);
    const float up = mx > (m.begun ? BASE<CT> : -INFINITY) ? mx - BASE<CT> : 0.0f, al = m.begun ? __builtin_amdgcn_exp2f(-up) : 1.0f;
    m.ref -= up;
    m.begun = m.begun || mx > -INFINITY;
    m.ls *= al;
    const float at = m.ref * unit;
    m.below = f32x4v{at, at, at, at};
#pragma unroll
    for (int u = 0; u < NK; u++)
#pragma unroll
        for (int e = 0; e < 4; e++) s[u][e] -= up;
#pragma unroll
    for (int d = 0; d < 4; d++) m.o[d] *= al;
}

// Eight weights as pieces.
template <int CT>
__device__ __forceinline__ void weights8(const float *x, u32x4v *p) {
    if constexpr (CT != DT_F16) return split8<CT>(x, p);
    // The upper piece is the weight cut to 11 bits, so the rest is exact (two cycles an instruction each; one that subtracts the packed
    // half, v_fma_mixlo_f16, takes eight).
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const float a = x[2 * e], b = x[2 * e + 1];
        const float ah = __uint_as_float(__float_as_uint(a) & 0xFFFFE000u), bh = __uint_as_float(__float_as_uint(b) & 0xFFFFE000u);
        p[0][e] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(ah, bh));
        p[1][e] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2v{a - ah, b - bh}, f16x2t));
    }
}

// The keys (values) of a tile's pieces, whose spans lanes `first` and on hold; zeros, which the buffers' bounds give, for slots that
// no row sees and without a page.
template <int CT, int PIECES>
__device__ __forceinline__ void load_keys(Raw<CT> &r, const WindowArgs &a, const Spans &p, uint32_t first, uint32_t lane) {
    constexpr uint32_t ROW = Cached<CT>::ROW;
    constexpr int GROUPS = 2 * Raw<CT>::SUB, EACH = GROUPS / PIECES, LOADS = Kind<CT>::KW;  // groups of 16 keys, those of a piece; loads of a group
#pragma unroll
    for (int i = 0; i < PIECES; i++) {
        const __amdgpu_buffer_rsrc_t b = span_of(static_cast<const char *>(a.kv.k) + p.at(first + i), p.rows(first + i) * ROW);
#pragma unroll
        for (int u = 0; u < EACH * LOADS; u++) r.k[EACH * LOADS * i + u] = __builtin_amdgcn_raw_buffer_load_b128(b, 16 * lane + 1024 * u, 0, 0);
        if constexpr (CT == DT_F8) {
            const __amdgpu_buffer_rsrc_t s = span_of(a.kv.ks + p.scale(first + i), p.rows(first + i));
#pragma unroll
            for (int u = 0; u < EACH; u++) r.ks[EACH * i + u] = __builtin_amdgcn_raw_buffer_load_b8(s, (lane & 15) + 16 * u, 0, 0);
        }
    }
}
// Loaded so, whole rows side by side (the loads of a wave whose neighbouring lanes are of different rows take the CU's address unit four
// times as long), the keys change lanes in LDS: byte of chunk c (16 bytes) of a row, which keeps the same chunk of 16 rows in
// different banks.
template <int CT>
__device__ __forceinline__ uint32_t key_at(uint32_t row, uint32_t c) {
    const uint32_t f = CT == DT_F32 ? row & 15 : CT == DT_F16 ? (row >> 1) & 7 : (row >> 2) & 3;
    return row * Cached<CT>::ROW + ((c ^ f) << 4);
}
template <int CT>
__device__ __forceinline__ void turn_keys(Raw<CT> &r, char *lds, uint32_t lane) {
    constexpr uint32_t CHUNKS = Cached<CT>::ROW / 16, ROWS = 64 / CHUNKS;
    constexpr int N = 2 * Raw<CT>::SUB * Kind<CT>::KW;
#pragma unroll
    for (int j = 0; j < N; j++) *reinterpret_cast<u32x4v *>(lds + key_at<CT>(j * ROWS + lane / CHUNKS, lane % CHUNKS)) = r.k[j];
    wave_sync();
#pragma unroll
    for (int u = 0; u < 2 * Raw<CT>::SUB; u++)
#pragma unroll
        for (int w = 0; w < Kind<CT>::KW; w++)
            r.k[u * Kind<CT>::KW + w] = *reinterpret_cast<const u32x4v *>(lds + key_at<CT>(16 * u + (lane & 15), (lane >> 4) * Kind<CT>::KW + w));
}
template <int CT, int PIECES>
__device__ __forceinline__ void load_values(Raw<CT> &r, const WindowArgs &a, const Spans &p, uint32_t first, uint32_t l16, uint32_t g) {
    constexpr uint32_t ROW = Cached<CT>::ROW;
    constexpr int GROUPS = 2 * Raw<CT>::SUB, EACH = GROUPS / PIECES;
#pragma unroll
    for (int i = 0; i < PIECES; i++) {
        const __amdgpu_buffer_rsrc_t b = span_of(static_cast<const char *>(a.kv.v) + p.at(first + i), p.rows(first + i) * ROW);
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
            const __amdgpu_buffer_rsrc_t s = span_of(a.kv.vs + p.scale(first + i), (p.rows(first + i) + 3) & ~3u);
#pragma unroll
            for (int u = 0; u < EACH; u++) r.vs[EACH * i + u] = __builtin_amdgcn_raw_buffer_load_b32(s, 4 * g + 16 * u, 0, 0);
        }
    }
}

constexpr uint32_t AW_WAVES = 8, AW_FEW = 4;  // waves of a workgroup

// Split keys: the parts of a row tile meet in the workgroup that ends last.  Their sums are written and read with device scope, past
// the XCDs' L2s, which do not see each other's: a release and an acquire of all that an L2 holds (fences) made 64 sequences of up to
// 4096 keys 56 us where this takes 20.
__device__ __forceinline__ void put(uint64_t *p, uint64_t v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ uint64_t get(const uint64_t *p) { return __hip_atomic_load(const_cast<uint64_t *>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ float low(uint64_t v) { return __uint_as_float(static_cast<uint32_t>(v)); }
__device__ __forceinline__ float high(uint64_t v) { return __uint_as_float(static_cast<uint32_t>(v >> 32)); }
__device__ __forceinline__ uint64_t two(float a, float b) { return __float_as_uint(a) | static_cast<uint64_t>(__float_as_uint(b)) << 32; }

// Part `mine` of `n` of a unit is stored: are all?  A part's flag holds the call's tag once it is; the workgroups that see all (the
// last one does, since each looks once its own flag stands) take the flags back, so that a replay of the call finds none set, and
// join, to the same bits.  Whatever else the flags' memory holds is no tag: it is a random number of 64 bits.
__device__ __forceinline__ bool all_there(uint64_t *flags, uint32_t mine, uint32_t n, uint64_t tag, uint32_t *said) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // each wave's stores stand
    __syncthreads();
    if (threadIdx.x < 64) {
        if (threadIdx.x == 0) put(flags + mine, tag);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        bool all = true;
        for (uint32_t i = threadIdx.x; i < n; i += 64) all = all && get(flags + i) == tag;
        all = __all(all);
        if (threadIdx.x == 0) *said = all;
    }
    __syncthreads();
    const bool last = *said != 0;
    if (last)
        for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) put(flags + i, 0);
    return last;
}

// The S parts of rows [r0, r1) of a tile joined.  A row's are taken by W groups of 16 lanes, every W-th part each, which meet in LDS
// in their order; a lane has four dims.
template <int CT, int WAVES>
__device__ __forceinline__ void join_parts(const WindowArgs &a, uint32_t b, uint32_t kvh, uint32_t r0, uint32_t r1, uint32_t S, uint64_t pos, char *lds) {
    constexpr uint32_t GROUPS = WAVES * 4, BATCH = 8;
    const uint32_t lane = threadIdx.x & 15, group = threadIdx.x / 16, n = r1 - r0;
    const uint32_t items = n > 8 ? 16 : n > 4 ? 8 : n > 2 ? 4 : n > 1 ? 2 : 1, W = GROUPS / items, it = group % items;
    const uint32_t r = r0 + it, t = by_group(a, r), head = kvh * a.group + r - t * a.group;
    const size_t row = static_cast<size_t>(b) * a.rows.T + t;
    const bool have = it < n;
    float m = INFINITY, l = 0.0f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    // (the sums of parts before: brought to a smaller mark; a part without a key of the row, or with scores of -infinity alone, has no sums;
    // one of NaN scores alone has no reference either, but a sum that is NaN)
    auto add = [&](float pm, float pl, float4 x) {
        if (pm == INFINITY && pl == 0.0f) return;
        const float mn = fminf(m, pm), f = m == INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mn - m), k = __builtin_amdgcn_exp2f(mn - pm);
        m = mn;
        l = fmaf(l, f, pl * k);
        v.x = fmaf(v.x, f, x.x * k);
        v.y = fmaf(v.y, f, x.y * k);
        v.z = fmaf(v.z, f, x.z * k);
        v.w = fmaf(v.w, f, x.w * k);
    };
    if (have) {
        const size_t at = (row * a.hq + head) * a.parts;
        const uint64_t *marks = reinterpret_cast<const uint64_t *>(a.part + static_cast<size_t>(a.rows.B) * a.rows.T * a.hq * a.parts * 64) + at;
        const uint64_t *sums = reinterpret_cast<const uint64_t *>(a.part + at * 64) + 2 * lane;
        for (uint32_t s0 = group / items; s0 < S; s0 += BATCH * W) {  // so many parts' loads at once
            uint64_t e[BATCH], x[BATCH][2];
#pragma unroll
            for (uint32_t i = 0; i < BATCH; i++) {
                const size_t p = s0 + i * W;
                e[i] = two(INFINITY, 0.0f);
                x[i][0] = x[i][1] = 0;
                if (p < S) {
                    e[i] = get(marks + p);
                    x[i][0] = get(sums + p * 32);
                    x[i][1] = get(sums + p * 32 + 1);
                }
            }
#pragma unroll
            for (uint32_t i = 0; i < BATCH; i++) add(low(e[i]), high(e[i]), make_float4(low(x[i][0]), high(x[i][0]), low(x[i][1]), high(x[i][1])));
        }
    }
    if (W > 1) {
        float4 *acc = reinterpret_cast<float4 *>(lds);
        float2 *mark = reinterpret_cast<float2 *>(lds + GROUPS * 256);
        acc[group * 16 + lane] = v;
        if (lane == 0) mark[group] = make_float2(m, l);
        __syncthreads();
        if (threadIdx.x / 64 * 4 >= items) return;  // (whole waves)
        m = INFINITY;
        l = 0.0f;
        v = make_float4(0.f, 0.f, 0.f, 0.f);
        for (uint32_t g = group; g < GROUPS; g += items) add(mark[g].x, mark[g].y, acc[g * 16 + lane]);
    }
    const float f = 1.0f / l;
    v.x *= f; v.y *= f; v.z *= f; v.w *= f;
    const bool good = fabsf(v.x) < INFINITY && fabsf(v.y) < INFINITY && fabsf(v.z) < INFINITY && fabsf(v.w) < INFINITY;
    const bool own = have && group < items;
    uint64_t bad = __ballot(own && !good);
    if (own && !((bad >> (threadIdx.x & 48)) & 0xFFFF)) reinterpret_cast<float4 *>(a.out + row * a.ldo + head * 64)[lane] = v;
    while (bad) {  // rows with an output that is not finite (or without a weight) once more, each from its own keys alone
        const uint32_t x = (__ffsll(static_cast<unsigned long long>(bad)) - 1) / 16, rx = r0 + threadIdx.x / 64 * 4 + x, tx = by_group(a, rx);
        bad &= ~(0xFFFFull << (16 * x));
        attend_wave<CT>(a, b, b * a.rows.T + tx, kvh * a.group + rx - tx * a.group, pos + tx);
    }
}

// Few rows.  Grid: x the sequences' row tiles, y the key heads, z the parts.  What a decode step spends beyond its bytes is loads that
// wait for each other, so the table's entries and the query are requested before the position is known, and a wave holds the
// places of its next 64 runs of slots, from loads made a round earlier.
template <int CT, bool PAGED, int PIECES, bool APART, int WAVES>
__global__ __launch_bounds__(64 * WAVES, WAVES == 4 && CT != DT_F32 ? 3 : 2) void attention_window_kernel(WindowArgs a) {
    typedef Kind<CT> KD;
    constexpr int SUB = Raw<CT>::SUB, NK = 2 * SUB;
    constexpr uint32_t TK = Raw<CT>::TK;
    constexpr uint32_t AREA = TK * Cached<CT>::ROW > 16 * AT_LD * 4 ? TK * Cached<CT>::ROW : 16 * AT_LD * 4;  // a tile's keys, or a wave's sums
    __shared__ __attribute__((aligned(16))) char lds[WAVES * AREA];
    __shared__ float ms[WAVES * 16], sums[WAVES * 16];
    const uint32_t tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, g = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    constexpr bool TWO = !APART && WAVES == AW_FEW;  // four waves may have two row tiles
    const uint32_t keys = TWO ? a.keys : WAVES, wk = wave % keys, wr = wave / keys;
    const uint32_t G = a.group, T = a.rows.T, span = WAVES / keys * 16;  // rows of a workgroup

    // The workgroup's rows [r0, r1) of sequence b's rows (t, head of the group), the longest first.
    // (A CU gets every 256th workgroup or so: each head and part begins at another sequence, or a CU would get all of a long one.)
    uint32_t x = blockIdx.x + a.shift * (blockIdx.y + a.hkv * blockIdx.z);
    if (x >= gridDim.x) x -= gridDim.x;
    const uint32_t kvh = blockIdx.y, b = a.seq_tiles == 1 ? x : x / a.seq_tiles;
    const uint32_t n = a.rows.counts ? min(a.rows.counts[b], T) : T;
    const uint32_t r0 = (a.seq_tiles - 1 - (x - b * a.seq_tiles)) * span, r1 = min(n * G, r0 + span);
    if (r0 >= r1) return;

    // The lane's row (all four g's the same one) and its keys [lo, hi) and those before a.sinks.
    const uint32_t rw = r0 + wr * 16, r = rw + l16, t = by_group(a, r), head = kvh * G + r - t * G;
    const bool have = r < r1;
    // What does not wait for the sequence's position goes first: the query, and, where no window moves the first tile, its entries.
    const RawQuery rq = load_query<false>(a.q + (static_cast<size_t>(b) * T + t) * a.ldq + head * 64, g, have);
    constexpr uint32_t EACH = 64 / PIECES, LEN = TK / PIECES;  // tiles whose spans a wave holds, slots of a piece
    uint32_t early = 0;
    if (PAGED && a.window == 0) {
        const uint32_t tile = (APART ? blockIdx.z * a.run : 0) + wk + lane / PIECES * keys;
        early = entry_of<PAGED>(a, b, tile * TK + lane % PIECES * LEN);  // (window_plan keeps it within 32 bits)
    }
    const uint64_t pos = a.rows.pos ? a.rows.pos[b] : 0u;
    uint32_t lo = 0, hi = 0, first;
    if (have) row_keys(a, pos + t, first, lo, hi);
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
    // The spans of EACH tiles of this wave, and the entries of the next ones.
    const uint32_t i0 = i;
    auto slot_of = [&](uint32_t q) { return tl.at(min(i0 + (q + lane / PIECES) * keys, end - 1)) * TK + lane % PIECES * LEN; };
    auto spans = [&](uint32_t q, uint32_t entry) {
        return span_run<CT, PAGED, LEN>(a, tl, kvh, slot_of(q), i0 + (q + lane / PIECES) * keys < end, entry);
    };
    Spans sp{};
    uint32_t q = 0, next_entry = 0;  // this wave's tiles so far
    // Loads of a tile past the last one are issued too, of no bytes: with as many loads in flight on every path, the waits for
    // the values leave the next keys on their way.
    if (i < end) {
        sp = spans(0, PAGED && a.window == 0 ? early : entry_of<PAGED>(a, b, slot_of(0)));
        __builtin_amdgcn_sched_barrier(0);  // in this order, as in the loop, or its first wait is for all of them
        load_keys<CT, PIECES>(raw, a, sp, 0, lane);
        __builtin_amdgcn_sched_barrier(0);
        load_values<CT, PIECES>(raw, a, sp, 0, l16, g);
        __builtin_amdgcn_sched_barrier(0);
        if (i + EACH * keys < end) next_entry = entry_of<PAGED>(a, b, slot_of(EACH));
    }
    const Query<CT> qu = query_of<CT>(rq, a.scale);

    Sums m;
    for (; i < end; i += keys, q++) {
        const uint32_t k0 = tl.at(i) * TK, none = PAGED ? static_cast<uint32_t>(sp.holes >> (q % EACH * PIECES)) & ((1u << PIECES) - 1) : 0;
        turn_keys<CT>(raw, lds + wave * AREA, lane);
        f32x4v s[NK];
#pragma unroll
        for (int kk = 0; kk < 2; kk++) {
            u32x4v kf[NK][KD::NC];
#pragma unroll
            for (int u = 0; u < NK; u++) {
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
                if (kk == 0) s[u] = m.below;
            }
            dots<CT, NK>(kf, qu.f[kk], s);
        }
        const uint32_t at = (q + 1) % EACH;
        if (at == 0 && i + keys < end) {
            sp = spans(q + 1, next_entry);
            if (i + (1 + EACH) * keys < end) next_entry = entry_of<PAGED>(a, b, slot_of(q + 1 + EACH));
        } else if (i + keys >= end) {
            sp.n = 0;
        }
        load_keys<CT, PIECES>(raw, a, sp, at * PIECES, lane);

        if (!((k0 >= tl.in_lo || k0 + TK <= a.sinks) && k0 + TK <= tl.in_hi) || none) {
            hide<NK>(s, k0, g, lo, hi, a.sinks, none, PIECES);
            if constexpr (CT == DT_F8) {  // a scale byte past the keys may stand for anything
#pragma unroll
                for (int u = 0; u < NK; u++) {
                    const uint32_t key = k0 + 16 * u + 4 * g, k = tl.hi > key ? min(tl.hi - key, 4u) : 0;
                    raw.vs[u] &= k == 4 ? ~0u : (1u << (8 * k)) - 1;
                }
            }
        }
        if (qu.scaled) {
#pragma unroll
            for (int u = 0; u < NK; u++) s[u] *= qu.c;
        }
        refer<CT, NK>(s, m, qu.unit);
        u32x4v pf[SUB][KD::NQ];
#pragma unroll
        for (int x = 0; x < SUB; x++) {
            float p[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                p[j] = __builtin_amdgcn_exp2f(s[2 * x + (j >> 2)][j & 3]);
                m.ls += p[j];
                if constexpr (CT == DT_F8) p[j] *= f8_pow2((raw.vs[2 * x + (j >> 2)] >> (8 * (j & 3))) & 255u);
            }
            weights8<CT>(p, pf[x]);
        }

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
        for (int d = 0; d < 4; d++) m.o[d] += ot[d];
        load_values<CT, PIECES>(raw, a, sp, at * PIECES, l16, g);
    }

    // The waves' parts of each row meet in wave order: a thread joins four dims of a row.
    {
        float *p = reinterpret_cast<float *>(lds + wave * AREA) + l16 * AT_LD + 16 * g;
#pragma unroll
        for (int e = 0; e < 4; e++) *reinterpret_cast<float4 *>(p + 4 * e) = make_float4(m.o[0][e], m.o[1][e], m.o[2][e], m.o[3][e]);
        const float l = m.ls + __shfl_xor(m.ls, 16, 64), all = l + __shfl_xor(l, 32, 64);
        if (g == 0) {
            ms[wave * 16 + l16] = m.mark();
            sums[wave * 16 + l16] = all;
        }
    }
    __syncthreads();
    for (uint32_t j = tid; j < span * 16; j += 64 * WAVES) {
        const uint32_t rr = j / 16, d4 = 4 * (j & 15), rj = r0 + rr;  // row rr of the workgroup
        if (r0 + (j & ~63u) / 16 >= r1) break;  // (whole waves)
        const uint32_t tj = by_group(a, rj), headj = kvh * G + rj - tj * G;
        const size_t row = static_cast<size_t>(b) * T + tj;
        const uint32_t w0 = rr / 16 * keys, in = rr & 15;  // the row's waves, its place in each
        float mk = INFINITY, l = 0.0f;
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
                v[w] = *reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(lds + (w0 + w) * AREA) + in * AT_LD + d4);
            }
#pragma unroll
            for (uint32_t w = 0; w < N; w++) mk = fminf(mk, mw[w]);
#pragma unroll
            for (uint32_t w = 0; w < N; w++) {
                // (sums without a reference are zeros, or NaN)
                const float f = mw[w] == INFINITY ? 1.0f : __builtin_amdgcn_exp2f(mk - mw[w]);
                l = fmaf(sw[w], f, l);
                acc.x = fmaf(v[w].x, f, acc.x);
                acc.y = fmaf(v[w].y, f, acc.y);
                acc.z = fmaf(v[w].z, f, acc.z);
                acc.w = fmaf(v[w].w, f, acc.w);
            }
        };
        if (keys == WAVES) join(std::integral_constant<uint32_t, WAVES>{});
        else if constexpr (TWO) join(std::integral_constant<uint32_t, WAVES / 2>{});
        if constexpr (APART) {
            if (rj < r1) {
                const size_t at = (row * a.hq + headj) * a.parts + blockIdx.z;
                uint64_t *to = reinterpret_cast<uint64_t *>(a.part + at * 64 + d4);
                put(to, two(acc.x, acc.y));
                put(to + 1, two(acc.z, acc.w));
                if (d4 == 0) put(reinterpret_cast<uint64_t *>(a.part + static_cast<size_t>(a.rows.B) * T * a.hq * a.parts * 64) + at, two(mk, l));
            }
        } else {
            const float f = 1.0f / l;
            acc.x *= f; acc.y *= f; acc.z *= f; acc.w *= f;
            const bool good = fabsf(acc.x) < INFINITY && fabsf(acc.y) < INFINITY && fabsf(acc.z) < INFINITY && fabsf(acc.w) < INFINITY;
            uint64_t bad = __ballot(rj < r1 && !good);
            if (rj < r1 && !((bad >> (lane & 48)) & 0xFFFF)) *reinterpret_cast<float4 *>(a.out + row * a.ldo + headj * 64 + d4) = acc;
            while (bad) {  // rows with an output that is not finite (or without a weight) once more, each from its own keys alone
                const uint32_t x = (__ffsll(static_cast<unsigned long long>(bad)) - 1) / 16, rx = r0 + (j & ~63u) / 16 + x, tx = by_group(a, rx);
                bad &= ~(0xFFFFull << (16 * x));
                attend_wave<CT>(a, b, b * T + tx, kvh * G + rx - tx * G, pos + tx);
            }
        }
    }
    if constexpr (APART) {
        __shared__ uint32_t said;
        const uint32_t S = min(a.parts, (tl.n + a.run - 1) / a.run);  // the tile's parts
        const size_t unit = static_cast<size_t>(x) * a.hkv + kvh;
        uint64_t *flags = reinterpret_cast<uint64_t *>(a.part + static_cast<size_t>(a.rows.B) * T * a.hq * a.parts * 66) + unit * a.parts;
        if (!all_there(flags, blockIdx.z, S, a.tag, &said)) return;
        join_parts<CT, WAVES>(a, b, kvh, r0, r1, S, pos, lds);
    }
}

// ------------------------------------------------------------- many rows --

// Rows of prompts.  The WR waves of a workgroup have 16 rows each and share its tiles of keys in LDS, 16 bits a value (as NC pieces),
// converted once: a tile is worked on while the next is on its way, which needs one barrier a tile.  fp16 rows go from memory to LDS
// by themselves, without passing registers: a prompt of 8192 rows took 310 us through registers (3 waves a SIMD), takes 274 us so, and
// 256 us with the 4 waves a SIMD that the registers saved allow (4 through registers spill: slower than 3).  Tiles of 64 keys share
// their two planes of 16 KB a stage; the values' operand is read transposed from LDS.
typedef short s16x4v __attribute__((ext_vector_type(4)));
constexpr uint32_t WR = 4;

template <int CT>
struct Staged {
    static constexpr uint32_t TK = CT == DT_F32 ? 32 : 64;      // keys of a tile
    static constexpr uint32_t PLANE = TK * 128;                  // bytes of a piece of its keys (or values)
    static constexpr uint32_t TILE = PLANE * Kind<CT>::NC;       // and of all pieces
    static constexpr uint32_t CHUNKS = Cached<CT>::ROW / 16;     // 16-byte chunks of a cached row
    static constexpr uint32_t ROWS = 64 / CHUNKS;                // rows of a wave's load
    static constexpr uint32_t HALF = TK / ROWS;                  // loads of a tile's keys, and of its values
    static constexpr int RUNS = TK / 16;                         // runs of 16 slots, each within one page
};
// Byte of chunk c (eight 16-bit values) of a tile's row.  LDS has 64 banks, so two rows are apart by themselves; the swizzle keeps
// the same chunk of 16 rows apart, and chunks 2 d and 2 d + 1 of eight rows.
__device__ __forceinline__ uint32_t chunk_at(uint32_t row, uint32_t c) {
    return row * 128 + ((c ^ (((row >> 1) & 3) << 1 | ((row >> 3) & 1))) << 4);
}

template <int CT, bool PAGED>
__global__ __launch_bounds__(64 * WR, CT == DT_F16 ? 4 : 3) void window_rows_kernel(WindowArgs a) {
    typedef Kind<CT> KD;
    typedef Staged<CT> SD;
    constexpr uint32_t TK = SD::TK, ROW = Cached<CT>::ROW, SPAN = WR * 16;
    constexpr int NK = TK / 16, LOADS = 2 * SD::HALF / WR;
    constexpr bool DIRECT = CT == DT_F16;
    static_assert(2 * SD::HALF % WR == 0, "whole loads a wave");
    __shared__ __attribute__((aligned(16))) char lds[2][2][SD::TILE];  // two tiles, keys and values of each
    const uint32_t tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, g = lane >> 4;
    const uint32_t wr = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t G = a.group, T = a.rows.T;

    // Workgroups go to the XCDs in turn: those of one sequence and key head go to one, whose L2 then fetches their keys once.
    const uint32_t xcds = a.by_xcd ? 8 : 1, xcd = blockIdx.x % xcds, item = blockIdx.x / xcds;
    const uint32_t lap = item / a.seq_tiles, group = lap * xcds + xcd;
    const uint32_t b = group / a.hkv, kvh = group - b * a.hkv;
    if (b >= a.rows.B) return;
    const uint32_t n = a.rows.counts ? min(a.rows.counts[b], T) : T;
    const uint32_t r0 = (a.seq_tiles - 1 - (item - lap * a.seq_tiles)) * SPAN, r1 = min(n * G, r0 + SPAN);  // the longest first
    if (r0 >= r1) return;
    // The lane's row (all four g's the same one).
    const uint32_t rw = r0 + wr * 16, r = rw + l16, t = by_group(a, r), head = kvh * G + r - t * G;
    const size_t row = static_cast<size_t>(b) * T + t;
    const bool have = r < r1;
    const RawQuery rq = load_query<true>(a.q + row * a.ldq + head * 64, g, have);  // (waits for nothing else)
    const uint64_t pos = a.rows.pos ? a.rows.pos[b] : 0u;
    uint32_t lo = 0, hi = 0, first;
    if (have) row_keys(a, pos + t, first, lo, hi);
    // The workgroup's tiles, one a step, and the wave's rows' keys.
    const Tiles tl = tiles_of<TK>(a, b, by_group(a, r0), by_group(a, r1 - 1));
    Tiles mine{};
    if (rw < r1) mine = tiles_of<TK>(a, b, by_group(a, rw), by_group(a, min(rw + 16, r1) - 1));
    const uint32_t steps = tl.n;

    // A step's tile on its way: this wave's chunks of it.  The spans of EACH steps' tiles, and the entries of the next ones.
    u32x4v raw[LOADS];
    uint32_t scales[LOADS];
    constexpr uint32_t EACH = 64 / SD::RUNS;
    auto tile_of = [&](uint32_t step) { return tl.at(min(step, steps - 1)); };
    auto slot_of = [&](uint32_t step) { return tile_of(step + lane / SD::RUNS) * TK + lane % SD::RUNS * 16; };
    auto spans = [&](uint32_t step, uint32_t entry) {
        return span_run<CT, PAGED, 16>(a, tl, kvh, slot_of(step), step + lane / SD::RUNS < steps, entry);
    };
    // DIRECT: LDS takes a load's lanes side by side, so a lane fetches the chunk that belongs where it writes.  (What is past a span's
    // bounds arrives as zeros there too.)
    const uint32_t into = chunk_at(wr % 2 * SD::ROWS + lane / SD::CHUNKS, lane % SD::CHUNKS) % 128 + lane / SD::CHUNKS * 128;
    auto request = [&](const Spans &sp, uint32_t step) {
#pragma unroll
        for (int j = 0; j < LOADS; j++) {
            const bool is_v = j * WR + wr >= SD::HALF;
            const uint32_t x = (j * WR + wr) % SD::HALF * SD::ROWS, i = step % EACH * SD::RUNS + x / 16, in = x % 16;  // the load's first row
            const uint32_t n = sp.rows(i), rows = n > in ? min(n - in, SD::ROWS) : 0;
            const __amdgpu_buffer_rsrc_t from = span_of(static_cast<const char *>(pick(is_v, a.kv.k, a.kv.v)) + sp.at(i) + in * ROW, rows * ROW);
            if constexpr (DIRECT)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (__attribute__((address_space(3))) void *)(lds[step & 1][is_v ? 1 : 0] + x * ROW), 16, into, 0, 0, 0);
            else
                raw[j] = __builtin_amdgcn_raw_buffer_load_b128(from, 16 * lane, 0, 0);
            if constexpr (CT == DT_F8)
                scales[j] = __builtin_amdgcn_raw_buffer_load_b8(span_of(pick(is_v, a.kv.ks, a.kv.vs) + sp.scale(i) + in, rows), lane / SD::CHUNKS, 0, 0);
        }
    };
    auto store = [&](uint32_t buf) {
        if constexpr (DIRECT) {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            return;
        }
#pragma unroll
        for (int j = 0; j < LOADS; j++) {
            const uint32_t id = j * WR + wr, x = id % SD::HALF * SD::ROWS + lane / SD::CHUNKS, c = lane % SD::CHUNKS;
            char *tile = lds[buf][id >= SD::HALF ? 1 : 0];
            const u32x4v w = raw[j];
            if constexpr (CT == DT_F8) {
                const float f = f8_pow2(scales[j]);
#pragma unroll
                for (int h = 0; h < 2; h++)
                    *reinterpret_cast<u32x4v *>(tile + chunk_at(x, 2 * c + h)) =
                        u32x4v{f8_bf16x2<false>(w[2 * h], f), f8_bf16x2<true>(w[2 * h], f), f8_bf16x2<false>(w[2 * h + 1], f), f8_bf16x2<true>(w[2 * h + 1], f)};
            } else {
                uint32_t p[3], q[3];
                split2<CT>(__uint_as_float(w[0]), __uint_as_float(w[1]), p);
                split2<CT>(__uint_as_float(w[2]), __uint_as_float(w[3]), q);
#pragma unroll
                for (int i = 0; i < 3; i++) *reinterpret_cast<u32x2v *>(tile + i * SD::PLANE + chunk_at(x, c / 2) + 8 * (c & 1)) = u32x2v{p[i], q[i]};
            }
        }
    };
    auto holes = [&](const Spans &sp, uint32_t step) {  // runs of 16 slots without a page
        return PAGED ? static_cast<uint32_t>(sp.holes >> (step % EACH * SD::RUNS)) & ((1u << SD::RUNS) - 1) : 0;
    };
    Spans sp = spans(0, entry_of<PAGED>(a, b, slot_of(0)));
    uint32_t next_entry = steps > EACH ? entry_of<PAGED>(a, b, slot_of(EACH)) : 0;
    request(sp, 0);
    uint32_t none = holes(sp, 0), none_next = 0;
    const Query<CT> qu = query_of<CT>(rq, a.scale);
    store(0);
    __syncthreads();

    Sums m;
    for (uint32_t step = 0; step < steps; step++) {
        const uint32_t buf = step & 1;
        if (step + 1 < steps) {
            if ((step + 1) % EACH == 0) {
                sp = spans(step + 1, next_entry);
                if (step + 1 + EACH < steps) next_entry = entry_of<PAGED>(a, b, slot_of(step + 1 + EACH));
            }
            request(sp, step + 1);
            none_next = holes(sp, step + 1);
        }
        const uint32_t k0 = tile_of(step) * TK;
        if (rw < r1 && k0 < mine.hi && (k0 < a.sinks || k0 + TK > mine.lo)) {
            const char *kt = lds[buf][0], *vt = lds[buf][1];
            f32x4v s[NK];
            {
                u32x4v kf[NK][2][KD::NC];
#pragma unroll
                for (int u = 0; u < NK; u++)
#pragma unroll
                    for (int kk = 0; kk < 2; kk++)
#pragma unroll
                        for (int x = 0; x < KD::NC; x++)
                            kf[u][kk][x] = *reinterpret_cast<const u32x4v *>(kt + x * SD::PLANE + chunk_at(16 * u + l16, 4 * kk + g));
                __builtin_amdgcn_sched_barrier(0);  // all reads on their way: one latency, not one a group of keys
#pragma unroll
                for (int kk = 0; kk < 2; kk++)
#pragma unroll
                    for (int x = 0; x < Products<CT>::N; x++)
#pragma unroll
                        for (int u = 0; u < NK; u++)
                            s[u] = mma<KD::HALF>(kf[u][kk][Products<CT>::C[x]], qu.f[kk][Products<CT>::Q[x]], kk + x == 0 ? m.below : s[u]);
            }
            u32x4v vf[4][KD::NC];
            auto values = [&](int x) {
#pragma unroll
                for (int d = 0; d < 4; d++)
#pragma unroll
                    for (int y = 0; y < KD::NC; y++) {
                        u32x2v w[2];
#pragma unroll
                        for (int z = 0; z < 2; z++) {  // lane l16 gets dim 16 d + l16 of four keys, of which it points at a quarter of one
                            const char *p = vt + y * SD::PLANE + chunk_at(32 * x + 16 * z + 4 * g + (l16 >> 2), 2 * d + ((l16 & 3) >> 1)) + 8 * (l16 & 1);
                            w[z] = __builtin_bit_cast(u32x2v, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4v *)(p)));
                        }
                        vf[d][y] = u32x4v{w[0][0], w[0][1], w[1][0], w[1][1]};
                    }
            };
            values(0);
            __builtin_amdgcn_sched_barrier(0);
            if (!((k0 >= mine.in_lo || k0 + TK <= a.sinks) && k0 + TK <= mine.in_hi) || none) hide<NK>(s, k0, g, lo, hi, a.sinks, none, NK);
            if (qu.scaled) {
#pragma unroll
                for (int u = 0; u < NK; u++) s[u] *= qu.c;
            }
            refer<CT, NK>(s, m, qu.unit);
            // p . v: a tile's sum starts from zero and joins the running one in one rounding.
            f32x4v ot[4];
#pragma unroll
            for (int d = 0; d < 4; d++) ot[d] = f32x4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int x = 0; x < NK / 2; x++) {
                u32x4v pf[KD::NQ];
                float p[8];
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    p[j] = __builtin_amdgcn_exp2f(s[2 * x + j / 4][j % 4]);
                    m.ls += p[j];
                }
                weights8<CT>(p, pf);
#pragma unroll
                for (int y = 0; y < Products<CT>::N; y++)
#pragma unroll
                    for (int d = 0; d < 4; d++) ot[d] = mma<KD::HALF>(vf[d][Products<CT>::C[y]], pf[Products<CT>::Q[y]], ot[d]);
                if (x + 1 < NK / 2) values(x + 1);
            }
#pragma unroll
            for (int d = 0; d < 4; d++) m.o[d] += ot[d];
        }
        none = none_next;
        if (step + 1 < steps) store(buf ^ 1);
        __syncthreads();
    }

    m.ls += __shfl_xor(m.ls, 16, 64);
    m.ls += __shfl_xor(m.ls, 32, 64);
    const float f = 1.0f / m.ls;
    bool good = true;
#pragma unroll
    for (int d = 0; d < 4; d++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            m.o[d][e] *= f;
            good = good && fabsf(m.o[d][e]) < INFINITY;
        }
    const uint64_t bad64 = __ballot(have && !good), bad32 = bad64 | bad64 >> 32;
    uint32_t bad = static_cast<uint32_t>(bad32 | bad32 >> 16) & 0xFFFFu;
    if (have && !((bad >> l16) & 1)) {
        uint32_t own = r;
        asm("" : "+v"(own));  // the address anew: held over the loop it would cost registers that the loop needs
        const uint32_t to = by_group(a, own);
        float *p = a.out + (static_cast<size_t>(b) * T + to) * a.ldo + (kvh * G + own - to * G) * 64 + 4 * g;
#pragma unroll
        for (int d = 0; d < 4; d++) *reinterpret_cast<f32x4v *>(p + 16 * d) = m.o[d];
    }
    // Rows with an output that is not finite (or without a weight) once more, each from its own keys alone.
    for (; bad; bad &= bad - 1) {
        const uint32_t rj = rw + __builtin_ctz(bad), tj = by_group(a, rj);
        attend_wave<CT>(a, b, b * T + tj, kvh * G + rj - tj * G, pos + tj);
    }
}

template <int CT, bool PAGED, int PIECES>
int launch_few(const WindowArgs &a, const WindowPlan &p, hipStream_t stream) {
    const dim3 grid(a.rows.B * a.seq_tiles, a.hkv, a.parts), block(64 * p.waves);
    if (a.parts > 1 && p.waves == AW_FEW) hipLaunchKernelGGL((attention_window_kernel<CT, PAGED, PIECES, true, AW_FEW>), grid, block, 0, stream, a);
    else if (a.parts > 1) hipLaunchKernelGGL((attention_window_kernel<CT, PAGED, PIECES, true, AW_WAVES>), grid, block, 0, stream, a);
    else if (p.waves == AW_FEW) hipLaunchKernelGGL((attention_window_kernel<CT, PAGED, PIECES, false, AW_FEW>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((attention_window_kernel<CT, PAGED, PIECES, false, AW_WAVES>), grid, block, 0, stream, a);
    return check_launch("attention window");
}

template <int CT, bool PAGED>
int launch_rows(const WindowArgs &a, const WindowPlan &p, hipStream_t stream) {
    const uint32_t groups = a.rows.B * a.hkv;
    const dim3 grid((a.by_xcd ? (groups + 7) / 8 * 8 : groups) * a.seq_tiles), block(64 * p.waves);
    hipLaunchKernelGGL((window_rows_kernel<CT, PAGED>), grid, block, 0, stream, a);
    return check_launch("attention window (rows)");
}

template <int CT>
int launch_kind(const WindowArgs &a, const WindowPlan &p, hipStream_t stream) {
    if (p.shared) return a.kv.table ? launch_rows<CT, true>(a, p, stream) : launch_rows<CT, false>(a, p, stream);
    constexpr int PIECES = Raw<CT>::TK / 16;
    if (!a.kv.table) return launch_few<CT, false, 1>(a, p, stream);
    // Pages that hold whole tiles: one page a tile.
    if (a.kv.page_len % Raw<CT>::TK == 0) return launch_few<CT, true, 1>(a, p, stream);
    return launch_few<CT, true, PIECES>(a, p, stream);
}

}  // namespace

// A number that no earlier call had and no memory holds but by a chance of 2^-63.
static uint64_t new_tag() {
    static std::atomic<uint64_t> state{static_cast<uint64_t>(std::chrono::system_clock::now().time_since_epoch().count()) ^ reinterpret_cast<uintptr_t>(&state)};
    uint64_t x = state.fetch_add(0x9E3779B97F4A7C15ull, std::memory_order_relaxed);
    x = (x ^ (x >> 30)) * 0xBF58476D1CE4E5B9ull;
    x = (x ^ (x >> 27)) * 0x94D049BB133111EBull;
    return (x ^ (x >> 31)) | 1;
}

// Where the work goes, from the sizes alone: 256 compute units are an MI355X's, not asked for, so that a workspace sized once
// fits wherever the call runs.  Units are row tiles of 16, `own` the keys one attends at most.  Measured in graphs, us, the rule's side
// first: 14 heads over 2 key heads, so two units a sequence of a decode step, fp16 unless it is said; one sequence fills the cache, the
// others are of any length up to that, or, in a skewed batch, up to 1000 slots.
//   - Prompts' rows share LDS where there are workgroups of 64 rows for the chip: 64 prompts of 100 rows behind up to 1180 slots
//     (1408 workgroups) 46 against 69 with waves of their own; 10 of 130 (300) 22 against 28.  In between, from 400 on, either side wins, by the
//     prompts: 14 of 130 (420) 28.1 against 26.4, 16 (480) 26.5 against 27.5, two of 1000 behind 8000 (440) 152 against 147;
//     8 bits, 18 of 130 (540) 37.5 against 35.0.  fp32 tiles are of 32 keys and cost their barriers more often, so from 512 on: four of
//     701 in a window (528) 30 against 40, two of 1000 of 16 heads (512) 50 against 54, but 18 of 130 (540) 73 against 60; one of 2000
//     of 16 heads (500) 96 against 115 shared.
//   - A workgroup's waves share one row tile and split its keys: 8 of 130 rows 19, 2 waves a tile 22, one 32.  With more than four
//     workgroups a compute unit and few keys to split, two waves a tile.
//   - Eight waves where units leave compute units idle: 64 sequences of 1024 9.4 against 10.1 with four, 8 bits 8.9 against 10.0.  Four
//     where they do not: 130 of 1024 12.6 against 14.0 (fp32 21.5 against 20.2); or where tiles are too few for eight: 20 rows
//     at 128 slots 5.9 against 6.4, though a decode step's rows at 256 5.6 against 5.4.
//   - Keys split over workgroups: one sequence of 131072 slots in 64 parts 20, in 32 23, unsplit 369.  Below some length the meeting costs
//     more than it gives.  Up to 64 units 1536: one of 1536 8.6 against 9.1, of 1280 unsplit 8.3 against 8.5; 32 of 2048 10.9 against
//     11.8, of 1536 10.5 against 10.3.  Above that 2560: 34 of 2560 12.5 against 13.1, 64 of 2560 14.2 against 14.0, of 2048
//     unsplit 12.4 against 13.2; 8 bits 2048: 64 of 2048 12.3 against 12.8, of 1536 unsplit 10.9 against 11.8.  fp32 tiles cost
//     twice as much: up to 32 units 512 (one of 512 8.5 against 9.1, of 384 unsplit 7.7 against 8.3), above that 896 (36 of 896 12.1 against
//     12.9, 64 of 896 14.1 against 13.3, of 768 unsplit 12.5 against 12.8; 32 would gain from 512 on: 9.7 unsplit against 8.7).
//   - As many parts as there are compute units for, but two at least, and four from 8192 keys on, for a batch with one long
//     sequence: skewed, 64 sequences of 16384 take 26 in four parts and 40 in two, of 65536 73 and 136, where lengths spread evenly
//     lose (64 of 16384 65 against 60, 40 54 against 42 in three).  At 129 to 160 units two parts cost such evenly spread lengths as
//     well (80 of 4096 25 against 20 unsplit; skewed of 7168 24 against 26) and four gain in both (80 of 16384 86 against 92, skewed 27 against
//     52).  Past 160 units none: evenly spread, 96 of 8192 51.2 against 52.5 in four, 128 60.1 against 62.5; but 8 bits (34.5 against
//     30.9 for 96), fp32 (97 against 85) and skewed batches (96 of 16384 52 against 27, of 65536 187 against 74) would gain.
//   - A part costs the join its loads, a longer one its waves their rounds, so both grow with the root of the keys, up to 64 parts before
//     the rounding to whole rounds of their waves, which can make them more (76): one sequence of 131072 in 8 bits in 64 19.1, in 86 19.7;
//     1600 slots in 7 parts of 4 tiles 9.0, in 5 of 5 9.8.  At least 256 keys a part, fp32 128 (1024 in 8 parts 8.6, in 4 10.0).
//   - Eight waves a part where parts leave half the compute units idle and have 512 keys or more (one of 65536 16.3 against 18.0),
//     or, not in fp16, have a compute unit each and 1024 (8 bits, 32 of 8192 16.4 against 18.0; fp16 18.2 against 18.4 with eight).
//     For up to 8 units of 16384 keys or more fp16 has half as many parts, of eight waves: two of 32768 14.0 against 15.3, of
//     98304 21.0 against 23.8, though four of 131072, more than the caches on the chip keep, 52 against 38.
//   - The workgroups of a sequence and key head go to one XCD where that spreads over all eight: four prompts of 701 rows in
//     fp32 30.2 against 34.9 (32 of 130 in fp16 40 against 38.5); one prompt over two key heads stays spread, 44 against 121.
WindowPlan window_plan(uint32_t B, uint32_t T, uint32_t hq, uint32_t hkv, uint32_t len_max, uint32_t window, uint32_t sinks, int ct) {
    const uint64_t tk = ct == DT_F32 ? Raw<DT_F32>::TK : Raw<DT_F8>::TK, cus = 256;
    WindowPlan p{AW_WAVES, AW_WAVES, 1, 0, false, false};
    len_max = std::min(len_max, 1u << 30);  // a sequence has no more slots
    const uint64_t seen = window ? static_cast<uint64_t>(window) + sinks + T - 1 : len_max;
    const uint64_t own = std::max<uint64_t>(1, std::min<uint64_t>(len_max, seen));  // keys a row tile attends at most
    const uint64_t rows = static_cast<uint64_t>(T) * (hq / hkv), heads = static_cast<uint64_t>(B) * hkv;
    auto groups = [&](uint64_t waves, uint64_t keys) { return heads * ((rows + waves / keys * 16 - 1) / (waves / keys * 16)); };
    const uint64_t wide = heads * ((rows + 16 * WR - 1) / (16 * WR)), units = groups(AW_WAVES, AW_WAVES);
    if (rows > 16 && wide >= (ct == DT_F32 ? 2 * cus : 400)) {
        p.shared = true;
        p.waves = WR;
        p.keys = 1;
        p.by_xcd = heads % 8 == 0 || heads > 32;
        return p;
    }
    if (rows > 16 && units > cus) {
        p.waves = p.keys = AW_FEW;
        // (Two are enough: rows that would be more than four workgroups a compute unit with two share LDS.)
        if (units > 4 * cus && own < 4 * tk * AW_FEW) p.keys = 2;
        return p;
    }
    if (units > cus || own <= AW_FEW * tk) p.waves = p.keys = AW_FEW;
    const uint64_t split = ct == DT_F32 ? (units > 32 ? 896 : 512) : units <= 64 ? 1536 : ct == DT_F16 ? 2560 : 2048;
    if (units <= 160 && own >= split) {
        const uint64_t tiles = (own + tk - 1) / tk;
        const uint64_t even = static_cast<uint64_t>(std::sqrt(static_cast<double>(own / (ct == DT_F32 ? 8 : 16))));
        const uint64_t places = ct == DT_F16 && units <= 8 && own >= 16384 ? cus / 2 : cus;
        const uint64_t parts = std::min<uint64_t>({64, own / (ct == DT_F32 ? 128 : 256), even, std::max<uint64_t>(places / units, own >= 8192 ? 4 : 2)});
        const uint64_t run = (tiles + parts - 1) / parts;
        const bool half = units * parts <= cus / 2;  // of the compute units have a part
        p.waves = p.keys = run * tk >= (half ? 512 : 1024) && (half || (ct != DT_F16 && units * parts <= cus)) ? AW_WAVES : AW_FEW;
        // Whole rounds of the waves: the nearer number of tiles, the smaller one only while its parts have places.
        const uint64_t less = run / p.waves * p.waves, more = less + p.waves;
        const bool down = run == less || (run - less < more - run && less > 0 && units * ((tiles + less - 1) / less) <= places);
        p.run = static_cast<uint32_t>(down ? less : more);
        p.parts = static_cast<uint32_t>((tiles + p.run - 1) / p.run);
    }
    return p;
}

int launch_attention_window(const WindowArgs &args, const WindowPlan &p, int ct, hipStream_t stream) {
    WindowArgs a = args;
    a.keys = p.keys;
    a.parts = p.parts;
    a.run = p.run;
    a.span = p.waves / p.keys * 16;
    a.by_xcd = p.by_xcd;
    const uint64_t tiles = (static_cast<uint64_t>(a.rows.T) * a.group + a.span - 1) / a.span, groups = static_cast<uint64_t>(a.rows.B) * a.hkv;
    a.seq_tiles = static_cast<uint32_t>(tiles);
    a.shift = static_cast<uint32_t>(a.rows.B * tiles / (static_cast<uint64_t>(a.hkv) * p.parts));
    int rc = p.shared ? check_grid("attention window (rows)", (groups + 7) / 8 * 8 * tiles, 64 * p.waves)
                      : check_grid("attention window", a.rows.B * tiles, 64 * p.waves);
    if (p.parts > 1) a.tag = new_tag();
    if (rc) return rc;
    if (ct == DT_F32) return launch_kind<DT_F32>(a, p, stream);
    if (ct == DT_F16) return launch_kind<DT_F16>(a, p, stream);
    return launch_kind<DT_F8>(a, p, stream);
}

}  // namespace mt
