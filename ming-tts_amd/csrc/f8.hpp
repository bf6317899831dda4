// The 8-bit format of the caches and matrices: OCP e4m3 codes (4 exponent bits, 3 mantissa bits,
// largest 448, one NaN a sign, no infinities) in blocks with one scale byte s each, 2^(s - 127).
//
// A block's scale is the least power of two, 2^-126 or more, that brings its largest finite |x| to
// 448 or less; the codes are x / scale to nearest, ties to even.  Both steps are exact but for that
// one rounding (half a step of 3 mantissa bits: 2^-4 of the value), so every way of computing the
// same x gives the same bytes, and a code times its scale is a bf16 number from scale byte 3 on: the conversion
// instructions that take the scale (v_cvt_scalef32_pk_bf16_fp8) give the value without a rounding.  Under bytes 1 and 2
// (blocks whose largest |x| is at most 448 2^-125) the least codes are finer than bf16, whose steps end at 2^-133.
// Infinities and NaN become NaN codes and do not count for the scale.  A finite |x| of 248 2^120 or more is rounded
// to 2^128, which fp32 and bf16 read as infinity.
#pragma once

#include "mt_device.hpp"

namespace mt {

enum : int { DT_F8 = 3 };

typedef uint32_t u32x4v __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2v __attribute__((ext_vector_type(2)));

// |x|, or 0 for what does not count.
__device__ __forceinline__ float f8_abs(float x) {
    const float a = fabsf(x);
    return a < INFINITY ? a : 0.0f;
}

// The scale byte of a block whose largest finite |x| is `top`: 448 = 1.75 2^8, so the exponent less
// 8, and one more where the mantissa is above 1.75 (the added 0x1FFFFF carries exactly then).
__device__ __forceinline__ uint32_t f8_scale(float top) {
    const int s = static_cast<int>((__float_as_uint(top) + 0x1FFFFFu) >> 23) - 8;
    return static_cast<uint32_t>(max(s, 1));
}
// 2^(s - 127) and 2^(127 - s) of a scale byte 1 .. 253.
__device__ __forceinline__ float f8_pow2(uint32_t s) { return __uint_as_float(s << 23); }
__device__ __forceinline__ float f8_inv_pow2(uint32_t s) { return __uint_as_float((254u - s) << 23); }

// Four values times inv = 2^(127 - s) as codes, the first in the lowest byte.
__device__ __forceinline__ uint32_t f8_encode4(float a, float b, float c, float d, float inv) {
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a * inv, b * inv, 0, false);
    return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(c * inv, d * inv, lo, true));
}

// Two codes (the low or the high half of a word) times the scale, as two packed bf16.
template <bool HI>
__device__ __forceinline__ uint32_t f8_bf16x2(uint32_t w, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(static_cast<int>(w), scale, HI));
}

// Four codes of a word times the scale as fp32, exactly: the least product, 2^-9 2^-126, is an fp32 number.
__device__ __forceinline__ void f8_decode4(uint32_t w, float scale, float *o) {
    const uint32_t a = f8_bf16x2<false>(w, 1.0f), b = f8_bf16x2<true>(w, 1.0f);
    o[0] = bf16_lo(a) * scale; o[1] = bf16_hi(a) * scale;
    o[2] = bf16_lo(b) * scale; o[3] = bf16_hi(b) * scale;
}

// A wave's LDS writes before it stand before its reads behind it.
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// Largest over aligned octets and groups of 16 lanes, the same in all of them.
__device__ __forceinline__ float octet_max(float v) {
    v = fmaxf(v, dpp_mov<0xB1>(v));   // quad_perm [1, 0, 3, 2]
    v = fmaxf(v, dpp_mov<0x4E>(v));   // quad_perm [2, 3, 0, 1]
    return fmaxf(v, dpp_mov<0x141>(v));  // row_half_mirror
}
__device__ __forceinline__ float row16_max(float v) {
    v = octet_max(v);
    return fmaxf(v, dpp_mov<0x140>(v));  // row_mirror
}

// The caches of one layer, as the kernels take them (mt_kv).
struct KvArgs {
    void *k, *v;
    uint8_t *ks, *vs;
    uint64_t stride, sstride;
    uint32_t len;
};

// Rows of B sequences, T each: row b T + t is sequence b's row t, which exists for t < counts[b]
// (all T without counts) and stands at slot pos[b] + t (t without pos).
struct RowsArgs {
    const uint32_t *pos, *counts;
    uint32_t B, T;
    __device__ __forceinline__ bool at(uint32_t row, uint32_t &b, uint64_t &slot) const {
        b = row / T;
        const uint32_t t = row - b * T;
        slot = static_cast<uint64_t>(pos ? pos[b] : 0u) + t;
        return !counts || t < counts[b];
    }
};

// Caches in pages (mt_paged_kv), or, without a table, contiguous ones (mt_kv) as one page a sequence.
struct PagedArgs {
    void *k, *v;
    uint8_t *ks, *vs;
    uint64_t stride, sstride;  // elements and scale bytes from page to page
    const uint32_t *table;
    uint32_t pages, page_len;  // page_len without a table: the cache's slots
    uint32_t len, table_stride;  // slots and entries of a sequence
    uint64_t page_magic;         // 2^37 / (page_len / 16) + 1

    // The entry of slot `s`: s / page_len = (s / 16) / (page_len / 16), both whole numbers, the second at most 2^11.  The product
    // of s / 16 < 2^26 with the magic number, off by at most 2^11 2^-37 of itself, stays below 2^64 and its quotient exact.
    __host__ __device__ __forceinline__ uint32_t entry(uint32_t s) const {
        return static_cast<uint32_t>(((s >> 4) * page_magic) >> 37);
    }
};

// The operands of mt_attention_paged and mt_attention_sinks.
struct WindowArgs {
    const float *q;
    float *out;
    uint32_t ldq, ldo, hq, hkv, window, sinks;
    RowsArgs rows;
    PagedArgs kv;
    float scale;
    float *part;    // split keys: [B T, hq, parts] sums of 64, as many pairs (minus the reference, the weights' sum), and the flags
                    // [row tiles, hkv, parts] that a part is there
    uint64_t tag;    // the call's, which such flags hold
    uint32_t parts, run;  // parts of a row tile's keys, and the key tiles of each (the last: all that is left)
    uint32_t keys;        // waves of a workgroup that share rows and split their keys (the rest: other rows)
    uint32_t span;        // rows of a workgroup
    uint32_t seq_tiles;   // row tiles (workgroups of `span` rows) of a sequence and key head
    uint32_t shift;       // row tiles that a key head's and part's first workgroup is ahead of the one before
    bool by_xcd;          // rows of prompts: a sequence's and key head's workgroups on one XCD
    uint32_t group, group_magic;  // as in SharedArgs
};

// How mt_attention_paged and mt_attention_sinks place their work (window_plan).
struct WindowPlan {
    uint32_t waves, keys;  // waves of a workgroup, those that share rows and split their keys
    uint32_t parts, run;   // parts of 1: one pass; more: joined by the workgroup of a row tile that ends last; tiles of a part
    bool shared;           // rows of prompts: the waves share their keys in LDS
    bool by_xcd;           // and a sequence's and key head's workgroups go to one XCD
};

// How mt_attention_shared places its work (shared_plan).
struct SharedPlan {
    uint32_t waves;     // of a workgroup
    uint32_t keys;      // waves of a workgroup that share rows and split their keys (the rest: other rows): all, 2 or 1
    bool apart;         // prefix and own keys in workgroups of their own, joined by a second kernel
    uint32_t sp, so;    // parts of the prefix's and of the own keys then
    uint32_t run;       // tiles of own keys a part
};

// The operands of mt_attention_shared.
struct SharedArgs {
    const float *q;
    float *out;
    uint32_t ldq, ldo, hq, hkv, window;
    RowsArgs rows;
    KvArgs kv, prefix;
    uint32_t prefix_len;
    float scale;
    float *part;    // apart: [B T, hq, sp + so] sums of 64 and behind them as many pairs (minus the maximum, the weights' sum)
    uint32_t sp, so, run;
    uint32_t keys;  // waves that split the keys
    uint32_t group, group_magic;  // hq / hkv, and 2^32 / group + 1: v / group is the high word of their product while
                                  // v group stays below 2^32 (rows times hq times group: validated)
};

}  // namespace mt
