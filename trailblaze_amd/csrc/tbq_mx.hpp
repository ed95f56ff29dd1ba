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
template <typename F>
__device__ __forceinline__ int mx_exponent(F a) {
    int e;
    const F m = frexp(a, &e);
    return a > 0 ? min(max(e - 3 + (m > F(0.875) ? 1 : 0), MX_LEAST), MX_MOST) : MX_LEAST;
}

// The nearest code of y (in units of the scale), ties to the even one.
template <typename F>
__device__ __forceinline__ uint32_t mx_code(F y) {
    const F m = y < 0 ? -y : y;
    const int c = (m > F(0.25)) + (m >= F(0.75)) + (m > F(1.25)) + (m >= F(1.75)) + (m > F(2.5)) + (m >= F(3.5)) +
                  (m > F(5));
    return (uint32_t)c | (y < 0 ? 8u : 0u);
}

}  // namespace tbq
