// tbq_mx.hpp -- pages of the key/value cache in MXFP4 (include/tbq_kv.h,
// TBQ_KV_MXFP4): where a row's codes and scales lie, and blocks of 32 values to
// codes and back.
//
// A block is one scale byte b, 2^(b - 127), and 32 codes e2m1.  gfx950's
// v_cvt_scalef32_pk_f16_fp4 makes two halves of two codes and a scale, which it
// takes from the exponent bits of a float (b << 23), in one instruction at full
// rate; b = 255 gives NaN.  With b within [104, 140] every value is a half.
//
// The layout follows the products that read it.  K's operand has 8 dims of a
// position a lane: a row's codes lie side by side, so a lane's 16 bytes are one
// block of a position.  V's operand has positions side by side: 8 dims (4 bytes)
// of four positions lie together, so a lane's 16 bytes are those of four
// positions, and so are the four scale bytes of a block.
#pragma once

#include "tbq_paged_attn.hpp"

namespace tbq {

constexpr int MX_LEAST = -23, MX_MOST = 13;   // exponents of the scales that append writes
constexpr int MX_NAN = 255;

typedef PgVec<pg_f16>::h8 mx_h8;
typedef pg_f16 mx_h2 __attribute__((ext_vector_type(2)));

// Bytes of a row (one position of a kv head, of K or of V); of a kv head in a page.
__host__ __device__ constexpr int mx_row(int D) { return D / 2 + D / 32; }
template <int D>
__device__ __forceinline__ long long mx_head(const PgArgs &a, int page, int h) {
    return ((long long)page * a.NKV + h) * ((long long)mx_row(D) << a.shift);
}
// Bytes before 8 dims 8 g.. of the row `in` of a page, and before the scale of block b.
template <int D>
__device__ __forceinline__ int mx_k_code(int in, int g) { return in * (D / 2) + 4 * g; }
template <int D>
__device__ __forceinline__ int mx_v_code(int in, int g) { return (in >> 2) * (2 * D) + 16 * g + 4 * (in & 3); }
template <int D>
__device__ __forceinline__ int mx_k_scale(int in, int b) { return in * (D / 32) + b; }
template <int D>
__device__ __forceinline__ int mx_v_scale(int in, int b) { return (in >> 2) * (D / 8) + 4 * b + (in & 3); }

// A scale byte as the float that the conversions take (255: NaN).
__device__ __forceinline__ float mx_scale(uint32_t byte) { return __builtin_bit_cast(float, byte << 23); }

// Codes 2 i and 2 i + 1 of eight.
template <int I>
__device__ __forceinline__ mx_h2 mx_pair(uint32_t codes, float scale) {
    return __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, I);
}
__device__ __forceinline__ mx_h8 mx_eight(uint32_t codes, float scale) {
    const mx_h2 a = mx_pair<0>(codes, scale), b = mx_pair<1>(codes, scale), c = mx_pair<2>(codes, scale),
                d = mx_pair<3>(codes, scale);
    return mx_h8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Exponent of the scale of a block whose largest magnitude is a (finite): the least
// E with a <= 7 * 2^E.  7 is where the last code, 6, is no further off than codes
// between 4 and 6 can be (values N(0, 1): relative error 0.112; 0.115 with 6 or 8).
__device__ __forceinline__ int mx_exponent(float a) {
    int e;
    const float m = frexpf(a, &e);
    return a > 0.f ? min(max(e - 3 + (m > 0.875f ? 1 : 0), MX_LEAST), MX_MOST) : MX_LEAST;
}

// y as a float that stands to every float of fewer bits, and halfway between two of them, as y does: rounded
// to an odd last bit where it is not a float.  So what is rounded from it is what would be rounded from y.
__device__ __forceinline__ float mx_odd(double y) {
    const float f = (float)y;
    const double d = y - (double)f;
    const uint32_t b = __builtin_bit_cast(uint32_t, f);
    const uint32_t n = (d > 0.) == (y > 0.) ? b + 1 : b - 1;   // the float on y's other side
    return (d > 0. || d < 0.) && f != 0.f && !(b & 1) ? __builtin_bit_cast(float, n) : f;   // (infinities stay)
}

// The codes of eight values: the nearest ones to x / scale, ties to the even one, at most 6
// (v_cvt_scalef32_pk_fp4_f32; checked against the definition at every border of every scale and beside it).
__device__ __forceinline__ uint32_t mx_codes(const float (&x)[8], float scale) {
    uint32_t c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[0], x[1], scale, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[2], x[3], scale, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[4], x[5], scale, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[6], x[7], scale, 3);
}

}  // namespace tbq
