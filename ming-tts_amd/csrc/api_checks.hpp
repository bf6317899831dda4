// Argument checks that the C entries of the caches' operators share (api_f8.cpp, api_paged.cpp).
#pragma once

#include "f8.hpp"
#include "mingtts_hip.h"
#include "mt_internal.hpp"

namespace mt {

inline bool aligned(const void *p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

// Do [a, a + an) and [b, b + bn) meet?
inline bool meet(const void *a, uint64_t an, const void *b, uint64_t bn) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return an && bn && x < y + bn && y < x + an;
}

// The keys, values or scales of B sequences: `each` bytes a sequence, `stride` bytes from one to the next.
struct Runs {
    const void *p;
    uint64_t each, stride;
    uint32_t B;
    uint64_t all() const { return each ? (B - 1) * stride + each : 0; }
};
// Do two of them meet?  Those of one stride may lie between each other (a sequence's keys and values side by side): they are
// apart if, from a run of a on, the next run of b starts behind it and ends before a's next one.
inline bool meet(const Runs &a, const Runs &b) {
    if (!meet(a.p, a.all(), b.p, b.all())) return false;
    if (a.B == 1 || a.stride != b.stride) return true;
    const uintptr_t x = reinterpret_cast<uintptr_t>(a.p), y = reinterpret_cast<uintptr_t>(b.p);
    const uint64_t s = a.stride, at = y >= x ? (y - x) % s : (s - (x - y) % s) % s;
    return at < a.each || at + b.each > s;
}

inline uint64_t elem_bytes(int t) { return t == DT_F32 ? 4 : t == DT_F8 ? 1 : 2; }

// Bytes from the first to the last element of `rows` rows of `width` elements of `size` bytes.
inline uint64_t span(uint64_t rows, uint64_t width, uint64_t ld, uint64_t size) { return rows ? ((rows - 1) * ld + width) * size : 0; }

inline int validate_rows(const char *who, uint32_t B, uint32_t T, uint32_t hq, uint32_t hkv) {
    if (hkv == 0) return set_error(MT_EINVAL, "%s: hkv must be positive", who);
    const uint64_t heads = static_cast<uint64_t>(hq) + 2ull * hkv;
    if (heads > 0xFFFF || static_cast<uint64_t>(B) * T > 0x7FFFFFFFull || static_cast<uint64_t>(B) * T * heads > 0x7FFFFFFFull)
        return set_error(MT_EINVAL, "%s: %u x %u rows of %u + 2 x %u heads are too many", who, B, T, hq, hkv);
    return MT_OK;
}

// The rows that a rotation reads (`in` bytes from qkv on) and, if q is given, writes (`outb` bytes).
inline int validate_qkv(const char *who, const float *qkv, uint32_t ldq, uint32_t B, uint32_t T, uint32_t hq, uint32_t hkv,
                        const float *inv_freq, const float *q, uint32_t ldo, uint64_t &in, uint64_t &outb) {
    if (!qkv || !inv_freq) return set_error(MT_EINVAL, "%s: null pointer", who);
    const uint64_t width = (static_cast<uint64_t>(hq) + 2 * hkv) * 64, all = static_cast<uint64_t>(B) * T;
    if (ldq < width || (q && ldo < static_cast<uint64_t>(hq) * 64))
        return set_error(MT_EINVAL, "%s: ldq %u < (hq + 2 hkv) * 64 or ldo %u < hq * 64", who, ldq, ldo);
    if (!aligned(qkv, 16) || ldq % 4 || (q && (!aligned(q, 16) || ldo % 4)))
        return set_error(MT_EINVAL, "%s: qkv and q must be 16-byte aligned with 16-byte row strides", who);
    in = span(all, width, ldq, 4);
    outb = q ? span(all, static_cast<uint64_t>(hq) * 64, ldo, 4) : 0;
    if (q && !(q == qkv && ldo == ldq) && meet(qkv, in, q, outb))
        return set_error(MT_EINVAL, "%s: q overlaps qkv (in place: q = qkv and ldo = ldq)", who);
    return MT_OK;
}

inline int validate_kv(const char *who, const char *what, const mt_kv *c, uint32_t B, uint32_t hkv, KvArgs &out) {
    if (!c) return set_error(MT_EINVAL, "%s: null %s", who, what);
    if (c->cache_t != DT_F32 && c->cache_t != DT_F16 && c->cache_t != DT_F8)
        return set_error(MT_EINVAL, "%s: %s must be f32, f16 or f8", who, what);
    if (!c->k || !c->v) return set_error(MT_EINVAL, "%s: null k or v of %s", who, what);
    if (!aligned(c->k, 16) || !aligned(c->v, 16)) return set_error(MT_EINVAL, "%s: k and v of %s must be 16-byte aligned", who, what);
    if (c->cache_len == 0 || c->cache_len > (1u << 30))
        return set_error(MT_EINVAL, "%s: cache_len %u of %s outside 1..2^30", who, c->cache_len, what);
    const uint64_t slots = static_cast<uint64_t>(hkv) * c->cache_len;
    if (B > 1 && (c->stride < slots * 64 || c->stride % 16))
        return set_error(MT_EINVAL, "%s: stride of %s smaller than one cache or no multiple of 16", who, what);
    if (c->cache_t == DT_F8) {
        if (!c->k_scale || !c->v_scale) return set_error(MT_EINVAL, "%s: null scales of %s", who, what);
        if (!aligned(c->k_scale, 4) || !aligned(c->v_scale, 4) || c->cache_len % 4)
            return set_error(MT_EINVAL, "%s: scales of %s must be 4-byte aligned and cache_len a multiple of 4", who, what);
        if (B > 1 && (c->scale_stride < slots || c->scale_stride % 4))
            return set_error(MT_EINVAL, "%s: scale_stride of %s smaller than one cache or no multiple of 4", who, what);
    }
    out = KvArgs{c->k, c->v, c->k_scale, c->v_scale, B > 1 ? c->stride : 0, B > 1 ? c->scale_stride : 0, c->cache_len};
    return MT_OK;
}

// The memory of B sequences' caches: keys, values and, in 8 bits, their scales.
struct KvRuns {
    Runs r[4];
    KvRuns(const KvArgs &c, int ct, uint32_t B, uint32_t hkv) {
        const uint64_t slots = static_cast<uint64_t>(hkv) * c.len, es = elem_bytes(ct), scales = ct == DT_F8 ? slots : 0;
        r[0] = Runs{c.k, slots * 64 * es, c.stride * es, B};
        r[1] = Runs{c.v, slots * 64 * es, c.stride * es, B};
        r[2] = Runs{c.ks, scales, c.sstride, B};
        r[3] = Runs{c.vs, scales, c.sstride, B};
    }
    bool meet_each_other() const {
        for (int i = 1; i < 4; i++)
            for (int j = 0; j < i; j++)
                if (meet(r[i], r[j])) return true;
        return false;
    }
};

}  // namespace mt
