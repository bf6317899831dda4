// The C ABI of the operators on 8-bit storage and shared prefixes (include/mingtts_hip.h): argument
// validation, before any HIP call, and the launchers' operands.
#include "api_checks.hpp"
#include "f8_linear.hpp"
#include "mingtts_hip.h"
#include "mt_internal.hpp"

using namespace mt;

extern "C" {

int mt_rope_append(const float *qkv, uint32_t ldq, uint32_t B, uint32_t T, uint32_t hq, uint32_t hkv, const uint32_t *pos,
                   const uint32_t *counts, uint32_t offset, const mt_kv *kv, const float *inv_freq, float *q, uint32_t ldo,
                   mt_stream_t stream) {
    const char *who = "mt_rope_append";
    int rc = validate_rows(who, B, T, hq, hkv);
    if (rc) return rc;
    if (B == 0 || T == 0) return MT_OK;
    RowsArgs rows{pos, counts, B, T};
    KvArgs c;
    rc = validate_kv(who, "kv", kv, B, hkv, c);
    if (rc) return rc;
    uint64_t in, outb;
    rc = validate_qkv(who, qkv, ldq, B, T, hq, hkv, inv_freq, q, ldo, in, outb);
    if (rc) return rc;
    const KvRuns caches(c, kv->cache_t, B, hkv);
    for (const Runs &r : caches.r)
        if (meet(r.p, r.all(), qkv, in) || meet(r.p, r.all(), q, outb))
            return set_error(MT_EINVAL, "%s: the caches overlap qkv or q", who);
    if (caches.meet_each_other()) return set_error(MT_EINVAL, "%s: the caches overlap each other", who);
    return launch_rope_append(qkv, ldq, rows, hq, hkv, offset, c, kv->cache_t, inv_freq, q, ldo,
                              reinterpret_cast<hipStream_t>(stream));
}

int mt_kv_copy(const mt_kv *src, const mt_kv *dst, uint32_t B, uint32_t T, uint32_t hkv, const uint32_t *pos,
               const uint32_t *counts, mt_stream_t stream) {
    const char *who = "mt_kv_copy";
    int rc = validate_rows(who, B, T, 0, hkv);
    if (rc) return rc;
    if (B == 0 || T == 0) return MT_OK;
    KvArgs s, d;
    rc = validate_kv(who, "src", src, B, hkv, s);
    if (!rc) rc = validate_kv(who, "dst", dst, B, hkv, d);
    if (rc) return rc;
    const KvRuns from(s, src->cache_t, B, hkv), to(d, dst->cache_t, B, hkv);
    for (const Runs &a : from.r)
        for (const Runs &b : to.r)
            if (meet(a, b)) return set_error(MT_EINVAL, "%s: src and dst overlap", who);
    if (to.meet_each_other()) return set_error(MT_EINVAL, "%s: dst's caches overlap each other", who);
    return launch_kv_copy(s, src->cache_t, d, dst->cache_t, RowsArgs{pos, counts, B, T}, hkv, reinterpret_cast<hipStream_t>(stream));
}

uint64_t mt_attention_shared_workspace(uint32_t B, uint32_t T, uint32_t hq, uint32_t hkv, uint32_t prefix_len, uint32_t len_max,
                                       uint32_t window, mt_dtype cache_t) {
    if (validate_rows("mt_attention_shared_workspace", B, T, hq, hkv) || hq == 0 || hq % hkv || B == 0 || T == 0) return 0;
    const SharedPlan p = shared_plan(B, T, hq, hkv, prefix_len, len_max, window, cache_t);
    return p.apart ? static_cast<uint64_t>(B) * T * hq * (p.sp + p.so) * (64 + 2) * 4 : 0;
}

int mt_attention_shared(const float *q, uint32_t ldq, uint32_t B, uint32_t T, uint32_t hq, uint32_t hkv, const uint32_t *pos,
                        const uint32_t *counts, const mt_kv *kv, const mt_kv *prefix, uint32_t prefix_len, uint32_t len_max,
                        uint32_t window, float *out, uint32_t ldo, float scale, void *workspace, uint64_t workspace_bytes,
                        mt_stream_t stream) {
    const char *who = "mt_attention_shared";
    int rc = validate_rows(who, B, T, hq, hkv);
    if (rc) return rc;
    if (hq == 0 || hq % hkv) return set_error(MT_EINVAL, "%s: hq %u must be a positive multiple of hkv %u", who, hq, hkv);
    const uint64_t G = hq / hkv;
    if (G > 4096 || static_cast<uint64_t>(B) * T * G > 0xFFFFFFFFull / G)
        return set_error(MT_EINVAL, "%s: %u x %u rows of %u query heads a key head are too many", who, B, T, hq / hkv);
    if (B == 0 || T == 0) return MT_OK;
    SharedArgs a{};
    rc = validate_kv(who, "kv", kv, B, hkv, a.kv);
    if (rc) return rc;
    if (prefix_len) {
        rc = validate_kv(who, "prefix", prefix, 1, hkv, a.prefix);
        if (rc) return rc;
        if (prefix->cache_t != kv->cache_t) return set_error(MT_EINVAL, "%s: prefix and kv must be of one type", who);
        if (prefix_len > prefix->cache_len)
            return set_error(MT_EINVAL, "%s: prefix_len %u past the prefix's cache_len %u", who, prefix_len, prefix->cache_len);
    }
    if (!q || !out) return set_error(MT_EINVAL, "%s: null pointer", who);
    if (ldq < static_cast<uint64_t>(hq) * 64 || ldo < static_cast<uint64_t>(hq) * 64)
        return set_error(MT_EINVAL, "%s: ldq / ldo < hq * 64", who);
    if (!aligned(q, 16) || ldq % 4 || !aligned(out, 16) || ldo % 4)
        return set_error(MT_EINVAL, "%s: q / out must be 16-byte aligned with 16-byte row strides", who);
    const uint64_t all = static_cast<uint64_t>(B) * T, w = static_cast<uint64_t>(hq) * 64;
    if (meet(q, span(all, w, ldq, 4), out, span(all, w, ldo, 4))) return set_error(MT_EINVAL, "%s: out overlaps q", who);
    const uint32_t most = len_max ? len_max : kv->cache_len;
    const uint64_t need = mt_attention_shared_workspace(B, T, hq, hkv, prefix_len, most, window, static_cast<mt_dtype>(kv->cache_t));
    if (need && (!workspace || !aligned(workspace, 16) || workspace_bytes < need))
        return set_error(MT_EINVAL, "%s: needs %llu bytes of 16-byte aligned workspace, got %llu", who,
                         static_cast<unsigned long long>(need), static_cast<unsigned long long>(workspace ? workspace_bytes : 0));
    a.q = q;
    a.out = out;
    a.ldq = ldq;
    a.ldo = ldo;
    a.hq = hq;
    a.hkv = hkv;
    a.window = window;
    a.rows = RowsArgs{pos, counts, B, T};
    a.prefix_len = prefix_len;
    a.scale = scale;
    a.part = static_cast<float *>(workspace);
    return launch_attention_shared(a, shared_plan(B, T, hq, hkv, prefix_len, most, window, kv->cache_t), kv->cache_t, reinterpret_cast<hipStream_t>(stream));
}

int mt_quantize_f8(const void *x, mt_dtype xt, uint32_t rows, uint32_t K, uint32_t ldx, const void *norm, mt_dtype nt, float eps,
                   uint8_t *codes, uint32_t ldq, uint8_t *scales, uint32_t lds, mt_stream_t stream) {
    const char *who = "mt_quantize_f8";
    if (xt != MT_F32 && xt != MT_F16 && xt != MT_BF16) return set_error(MT_EINVAL, "%s: x must be f32, f16 or bf16", who);
    if (norm && nt != MT_F16 && nt != MT_BF16) return set_error(MT_EINVAL, "%s: norm must be f16 or bf16", who);
    if (norm && !(eps >= 0.0f)) return set_error(MT_EINVAL, "%s: RMSNorm eps must be >= 0", who);
    if (norm && K > 16 * F8_NORM_K) return set_error(MT_EINVAL, "%s: a norm over K %u > %u", who, K, 16 * F8_NORM_K);
    if (K == 0 || K % 16) return set_error(MT_EINVAL, "%s: K must be a positive multiple of 16, got %u", who, K);
    // A block's first value is 128 times its number: 32 bits hold both.
    if (K > (1u << 31) || lds > (1u << 24)) return set_error(MT_EINVAL, "%s: K %u past 2^31 or lds %u past 2^24", who, K, lds);
    if (rows == 0) return MT_OK;
    if (rows > 0x7FFFFFFFu || static_cast<uint64_t>(rows) * lds > 0x7FFFFFFFull * 16)
        return set_error(MT_EINVAL, "%s: %u rows of %u blocks are too many", who, rows, lds);
    if (!x || !codes || !scales) return set_error(MT_EINVAL, "%s: null pointer", who);
    if (ldx < K || ldq < K) return set_error(MT_EINVAL, "%s: ldx %u or ldq %u < K %u", who, ldx, ldq, K);
    if (lds < 4 * ((K + 511) / 512) || lds % 4) return set_error(MT_EINVAL, "%s: lds %u must be a multiple of 4 of at least 4 ceil(K / 512)", who, lds);
    if (!aligned(x, 16) || ldx * elem_bytes(xt) % 16 || (norm && !aligned(norm, 16)) || !aligned(codes, 16) || ldq % 16 || !aligned(scales, 4))
        return set_error(MT_EINVAL, "%s: x, norm and codes must be 16-byte aligned with 16-byte row strides, scales 4-byte aligned", who);
    const uint64_t in = span(rows, K, ldx, elem_bytes(xt)), cb = span(rows, K, ldq, 1), sb = static_cast<uint64_t>(rows) * lds;
    if (meet(x, in, codes, cb) || meet(x, in, scales, sb) || meet(codes, cb, scales, sb))
        return set_error(MT_EINVAL, "%s: x, codes and scales must not overlap", who);
    return launch_quantize_f8(x, xt, rows, K, ldx, static_cast<const uint16_t *>(norm), nt, eps, codes, ldq, scales, lds,
                              reinterpret_cast<hipStream_t>(stream));
}

int mt_linear_f8(const void *x, mt_dtype xt, const uint8_t *xs, uint32_t ldxs, const void *norm, const uint8_t *w,
                 const uint8_t *ws, const uint8_t *w2, const uint8_t *w2s, const void *bias, mt_dtype bt, float *y,
                 mt_gemv_params p, mt_stream_t stream) {
    const char *who = "mt_linear_f8";
    if (xt != MT_F32 && xt != MT_F16 && xt != MT_BF16 && xt != MT_F8) return set_error(MT_EINVAL, "%s: unknown activation dtype %d", who, xt);
    const uint32_t known = MT_BIAS | MT_ACCUM | MT_GELU | MT_SILU_GATE | MT_SILU;
    if (p.flags & ~known) return set_error(MT_EINVAL, "%s: unknown flag bits 0x%x", who, p.flags & ~known);
    uint32_t flags = p.flags;
    if (bias) flags |= MT_BIAS;
    if ((flags & MT_BIAS) && !bias) return set_error(MT_EINVAL, "%s: MT_BIAS without a bias pointer", who);
    if ((bias || norm) && bt != MT_F16 && bt != MT_BF16) return set_error(MT_EINVAL, "%s: bias and norm must be f16 or bf16", who);
    const bool gated = (flags & MT_SILU_GATE) != 0;
    if (gated && (!w2 || !w2s)) return set_error(MT_EINVAL, "%s: MT_SILU_GATE without w2", who);
    if (p.M == 0 || p.N == 0) return MT_OK;
    if (p.M > 0x7FFFFFFFu || p.N > 0x7FFFFFFFu / (gated ? 2 : 1)) return set_error(MT_EINVAL, "%s: M %u x N %u is too large", who, p.M, p.N);
    if (!x || !w || !ws || !y) return set_error(MT_EINVAL, "%s: null x, w, ws or y", who);
    if (p.K == 0 || p.K % 16) return set_error(MT_EINVAL, "%s: K must be a positive multiple of 16, got %u", who, p.K);
    if (p.ldx < p.K || p.ldy < p.N) return set_error(MT_EINVAL, "%s: ldx %u < K %u or ldy %u < N %u", who, p.ldx, p.K, p.ldy, p.N);
    if (p.K > (1u << 22) || (xt == MT_F8 && p.ldx > (1u << 22)))
        return set_error(MT_EINVAL, "%s: K %u or ldx %u past 2^22", who, p.K, p.ldx);
    const uint64_t es = elem_bytes(xt);
    if (!aligned(x, 16) || p.ldx * es % 16 || !aligned(w, 16) || (gated && !aligned(w2, 16)))
        return set_error(MT_EINVAL, "%s: x, w and w2 must be 16-byte aligned, x with a 16-byte row stride", who);
    if (!aligned(ws, 4) || (gated && !aligned(w2s, 4))) return set_error(MT_EINVAL, "%s: scales must be 4-byte aligned", who);
    if (!aligned(y, 4) || (bias && !aligned(bias, 2)) || (norm && !aligned(norm, 16)))
        return set_error(MT_EINVAL, "%s: y must be 4-byte, bias 2-byte and norm 16-byte aligned", who);
    const uint32_t lds = 4 * ((p.K + 511) / 512);
    const uint64_t yb = span(p.M, p.N, p.ldy, 4);
    if (xt == MT_F8) {
        if (norm) return set_error(MT_EINVAL, "%s: norm applies to x that is not quantised yet", who);
        if (!xs || !aligned(xs, 4) || ldxs < lds || ldxs % 4)
            return set_error(MT_EINVAL, "%s: xs must be 4-byte aligned, its row stride a multiple of 4 of at least %u", who, lds);
        if (meet(xs, static_cast<uint64_t>(p.M) * ldxs, y, yb)) return set_error(MT_EINVAL, "%s: xs overlaps y", who);
    } else {
        if (norm && !(p.eps >= 0.0f)) return set_error(MT_EINVAL, "%s: RMSNorm eps must be >= 0", who);
        if (p.M > 16) return set_error(MT_ENOTSUP, "%s: quantises up to 16 rows itself, got %u: mt_quantize_f8 first", who, p.M);
        if (norm && p.K > F8_NORM_K) return set_error(MT_ENOTSUP, "%s: a norm over K %u > %u: mt_quantize_f8 first", who, p.K, F8_NORM_K);
    }
    if (meet(x, span(p.M, p.K, p.ldx, es), y, yb)) return set_error(MT_EINVAL, "%s: x overlaps y", who);
    F8LinearArgs a{x, xt == MT_F8 ? xs : nullptr, w, ws, gated ? w2 : w, gated ? w2s : ws,
                   static_cast<const uint16_t *>(bias), static_cast<const uint16_t *>(norm), y,
                   p.M, p.N, p.K, p.ldx, ldxs, lds, p.ldy, flags, p.eps};
    return launch_linear_f8(a, xt, bt, reinterpret_cast<hipStream_t>(stream));
}

}  // extern "C"
