// The 8-bit KV format (THB_KV_E4M3) and its pages.
//
// Format.  A head vector x (one token, one KV head, K or V) is stored as one
// power-of-two scale and head_dim codes in e4m3 (sign, 4 exponent bits of
// bias 7, 3 mantissa bits; largest 448, smallest step 2^-9):
//   e = the least integer with max|x| <= 448 * 2^e, at least -126;
//   code[d] = x[d] * 2^-e rounded to the nearest e4m3 value, ties to even.
// The stored value is code * 2^e.  A power of two costs a float format no
// accuracy (every value keeps its 4 significant bits whatever e is; a divisor
// max|x| / 448 would only move the underflow border, 2^-15 of max|x|, by at
// most a factor of two) and makes scaling exact in both directions: codes do
// not depend on how a division rounds, any value comes back exactly in f32 and
// bf16, and storing what was read back gives the same values.  The scale is kept
// as the byte b = e + 127 in [1, 247], the exponent field of the f32 2^e: one
// byte per vector beside its head_dim codes.  A vector that holds an infinity
// or a NaN has no scale: it is stored as b = 255 with zero codes and reads as
// NaN in every element (its f32 "scale" 255 << 23 is an infinity, and 0 * inf
// is NaN, so readers need no test for it).  Codes in the pool are therefore
// always finite.
//
// Pages.  Rows are padded to W = head_dim rounded up to 64 codes.  A page of P
// slots (a multiple of 16) is P / 16 tiles of 16 slots; a tile of K or of V is
// W / 64 blocks of 1 KiB, each exactly what one 16-byte load per lane of a
// wavefront brings in (lane 16 a + c: bytes [256 a + 16 c, + 16)), in the
// order the matrix cores take operands:
//   K block j, lane (a, c): slot c; dims 64 j + 8 a .. + 8, then 64 j + 32 + 8 a .. + 8
//     (the A operands of two 16x16x32 products);
//   V block j, lane (a, c): dims 64 j + 4 c .. + 4, of each the slots 4 a .. 4 a + 3
//     (a quarter of the A operand of four products, whose row c is dim
//     64 j + 4 c + i for i = 0 .. 3).
// Scales lie in a third plane, 2 P bytes a page: for each 4 slots the 4 bytes
// of K, then the 4 of V (what a lane's four scores need, as one 8-byte load).
#pragma once

#include "codec.hpp"

namespace thb {

__host__ __device__ inline uint32_t q8_width(uint32_t hd) { return (hd + 63u) & ~63u; }

// Byte offset of the 8 codes of dims [d, d + 8) (d a multiple of 8) of slot s
// in a K page.
__host__ __device__ inline uint32_t q8_k_off(uint32_t s, uint32_t d, uint32_t width) {
    return (s >> 4) * (width * 16u) + ((d >> 6) << 10) + ((d >> 3) & 3u) * 256u + (s & 15u) * 16u + ((d >> 5) & 1u) * 8u;
}
// Byte offset of dim d of slot s in a V page (slots 4 k .. 4 k + 3 of one dim
// are 4 bytes, dims 4 i .. 4 i + 3 follow one another).
__host__ __device__ inline uint32_t q8_v_off(uint32_t s, uint32_t d, uint32_t width) {
    return (s >> 4) * (width * 16u) + ((d >> 6) << 10) + ((s >> 2) & 3u) * 256u + (d & 63u) * 4u + (s & 3u);
}
// Byte offset of slot s's scale in a page of scales.
__host__ __device__ inline uint32_t q8_s_off(uint32_t s, bool is_v) { return (s >> 2) * 8u + (is_v ? 4u : 0u) + (s & 3u); }

// Scale byte of a vector whose largest magnitude has the f32 bits `amax`
// (infinities and NaN compare above every finite number).
__host__ __device__ inline uint32_t q8_scale_byte(uint32_t amax) {
    if (amax >= 0x7f800000u) return 255u;
    const int32_t b = static_cast<int32_t>(amax >> 23) - 8 + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0);
    return b < 1 ? 1u : static_cast<uint32_t>(b);
}


// 2^-e of scale byte b (0 for 255: every finite element becomes code 0; the
// caller drops what is not finite).
__device__ inline float q8_inv_scale(uint32_t b) { return __uint_as_float(b == 255u ? 0u : (254u - b) << 23); }

// Codes of 4 scaled values, |x| <= 448, the first in the lowest byte
// (v_cvt_pk_fp8_f32: nearest, ties to even).
__device__ inline uint32_t q8_encode4(float x0, float x1, float x2, float x3) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(x0, x1, 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(x2, x3, w, true);
    return static_cast<uint32_t>(w);
}

// Codes of 8 elements under scale byte b.
__device__ inline uint2 q8_encode8(const float (&x)[8], uint32_t b) {
    if (b == 255u) return make_uint2(0u, 0u);
    const float r = q8_inv_scale(b);
    return make_uint2(q8_encode4(x[0] * r, x[1] * r, x[2] * r, x[3] * r),
                      q8_encode4(x[4] * r, x[5] * r, x[6] * r, x[7] * r));
}

// The largest magnitude's bits among 8 elements.
__device__ inline uint32_t q8_amax8(const float (&x)[8]) {
    uint32_t m = 0u;
#pragma unroll
    for (int e = 0; e < 8; e++) m = max(m, __float_as_uint(x[e]) & 0x7fffffffu);
    return m;
}

// The values of 8 codes.
__device__ inline void q8_decode8(const uint2& w, float scale, float (&x)[8]) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    const f32x2 v[4] = {__builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w.x), false),
                        __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w.x), true),
                        __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w.y), false),
                        __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w.y), true)};
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] = v[e >> 1][e & 1] * scale;
}

// Writes 8 values as type DT at element e (a multiple of 8), rounded to nearest
// even.
template <uint32_t DT>
__device__ inline void q8_put8(void* dst, uint64_t e, const float (&x)[8]) {
    if constexpr (DT == THB_DT_F32) {
        f32x4* p = reinterpret_cast<f32x4*>(static_cast<float*>(dst) + e);
        p[0] = f32x4{x[0], x[1], x[2], x[3]};
        p[1] = f32x4{x[4], x[5], x[6], x[7]};
    } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            uint32_t b[2];
#pragma unroll
            for (int k = 0; k < 2; k++) {
                if constexpr (DT == THB_DT_F16) {
                    b[k] = __builtin_bit_cast(uint16_t, static_cast<_Float16>(x[2 * i + k]));
                } else {
                    const uint32_t f = __float_as_uint(x[2 * i + k]);
                    b[k] = (f & 0x7fffffffu) > 0x7f800000u ? (f >> 16) | 0x40u : (f + 0x7fffu + ((f >> 16) & 1u)) >> 16;
                }
            }
            w[i] = b[0] | (b[1] << 16);
        }
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(dst) + e) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

}  // namespace thb
