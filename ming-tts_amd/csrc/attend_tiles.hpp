// What the attention kernels on 16-row MFMA tiles share (mt_attention_shared, mt_attention_paged, mt_attention_sinks): the types
// of the caches, the pieces that fp32 operands are split into, and a tile's raw keys and values.
#pragma once

#include "f8.hpp"

namespace mt {

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

// The products of pieces that are not below 2^-24, the small ones first: of piece C of k (or v) and piece Q of q (or the
// weights).
template <int CT>
struct Products {
    static constexpr int N = CT == DT_F32 ? 6 : Kind<CT>::NQ;
    static constexpr int C[6] = {CT == DT_F32 ? 2 : 0, 0, CT == DT_F32 ? 1 : 0, 1, 0, 0};
    static constexpr int Q[6] = {CT == DT_F32 ? 0 : Kind<CT>::NQ - 1, CT == DT_F32 ? 2 : Kind<CT>::NQ - 2, CT == DT_F32 ? 1 : 0, 0, 1, 0};
};
// acc[i] + c[i] . q for N sums at once: an MFMA waits for the one before it on the same sum, so the sums take turns.
template <int CT, int N>
__device__ __forceinline__ void dots(const u32x4v (*c)[Kind<CT>::NC], const u32x4v *q, f32x4v *acc) {
#pragma unroll
    for (int p = 0; p < Products<CT>::N; p++)
#pragma unroll
        for (int i = 0; i < N; i++) acc[i] = mma<Kind<CT>::HALF>(c[i][Products<CT>::C[p]], q[Products<CT>::Q[p]], acc[i]);
}

// The maximum over the four lanes 16 apart.
__device__ __forceinline__ float rows_max(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

constexpr uint32_t AT_LD = 68;  // floats of a row in the waves' hand-over (64 and a 16-byte skew)

// One wave's 16 rows and TK = 32 SUB keys at a time: the raw keys and values of a tile.  Lane (l16, g) holds dims
// 16 g .. + 15 of keys 16 u + l16 (u < 2 SUB), and dims 4 l16 .. + 3 of the values of keys 32 i + 4 g + j and 32 i
// + 16 + 4 g + j (i < SUB, j < 4), which are the weights' places in the scores' accumulators.
template <int CT>
struct Raw {
    static constexpr int SUB = CT == DT_F32 ? 1 : 2;
    static constexpr uint32_t TK = 32 * SUB;
    u32x4v k[2 * SUB * Kind<CT>::KW];
    uint32_t v[8 * SUB * Kind<CT>::KW];
    uint32_t ks[2 * SUB], vs[2 * SUB];
};

__device__ __forceinline__ __amdgpu_buffer_rsrc_t span_of(const void *p, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), 0, static_cast<int>(bytes), 0x00020000);
}

// One of two values: a conditional of two variables would name one of the variables, and keep both in memory.
template <class V>
__device__ __forceinline__ V pick(bool second, V first, V other) {
    return second ? other : first;
}

}  // namespace mt
