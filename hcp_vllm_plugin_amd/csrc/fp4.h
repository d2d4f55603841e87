// The 4-bit KV cache: where its bytes lie and how 16-bit values get into it.
//
// The bytes of one (block, KV head) are, for block size B and head_dim d (a
// multiple of 32), B * (d + d / 16) of them:
//   K codes   [B][d / 2]             a key's row, two columns to a byte
//   V codes   [B / 4][d / 8][4][4]   four keys side by side: 4 bytes (8 columns) each
//   K scales  [B / 4][d / 32][4]     a byte for 32 columns of a key
//   V scales  [B / 4][d / 32][4]
// so that the decode kernel's lanes load what the matrix instructions take:
// 32 columns of one key of K, 8 columns of four keys of V, 16 bytes each, a
// wave 1 KB in a row.  A code is sign, two bits of exponent, one of mantissa
// (0, 0.5, 1, 1.5, 2, 3, 4, 6); a scale byte b stands for 2^(b - 127), 255 for
// NaN: the format that v_cvt_scalef32_* reads and writes.
#pragma once

#include "common.h"

namespace hcp {

struct Fp4Region {
  int32_t d, bs;
  __host__ __device__ int64_t bytes() const { return static_cast<int64_t>(bs) * (d + d / 16); }
  __device__ __forceinline__ int k_code(int off, int oct) const { return off * (d / 2) + oct * 4; }
  __device__ __forceinline__ int v_code(int off, int oct) const {
    return bs * (d / 2) + ((off >> 2) * (d / 8) + oct) * 16 + (off & 3) * 4;
  }
  __device__ __forceinline__ int k_scale(int off, int grp) const {
    return bs * d + ((off >> 2) * (d / 32) + grp) * 4 + (off & 3);
  }
  __device__ __forceinline__ int v_scale(int off, int grp) const {
    return bs * (d / 32) + k_scale(off, grp);
  }
};

typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

// Largest magnitude of 8 packed 16-bit floats, as their bits without the sign:
// these order like the values, infinities and NaN last.
__device__ __forceinline__ uint32_t mag_max8(u32x4 x) {
  u16x2 m = __builtin_bit_cast(u16x2, x[0] & 0x7fff7fffu);
#pragma unroll
  for (int i = 1; i < 4; ++i)
    m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, x[i] & 0x7fff7fffu));
  return m[0] > m[1] ? m[0] : m[1];
}

// Scale byte of 32 values whose largest magnitude has these bits: the least
// power of two of which the magnitude is at most 7 times (what lies between 6
// and 7 is off by no more than half the codes' last step; over normally
// distributed values the error is 0.112 of their deviation, 0.1155 with the
// limit at 6, 0.115 at 8, 0.1116 with the better of the two tried out).  Kept
// so that every code's value is a finite normal number of the model's type, or
// fp16's subnormal 2^-24.  With an infinity or a NaN among them: NaN.
template <typename T>
__device__ __forceinline__ uint32_t fp4_scale(uint32_t mag) {
  constexpr bool kBf = sizeof(T) == 2 && __is_same(T, __bf16);
  constexpr uint32_t lo = kBf ? 2 : 104, hi = kBf ? 252 : 140;
  constexpr uint32_t kInf = kBf ? 0x7f80u : 0x7c00u;
  if (mag >= kInf) return 255;
  // 7 = 1.75 * 2^2: two below the magnitude's own exponent, one where its
  // mantissa is past 1.75
  const uint32_t bits = __float_as_uint(Elem<T>::to_float(static_cast<uint16_t>(mag)));
  const uint32_t e = (bits + 0x1fffffu) >> 23;
  return e < lo + 2 ? lo : e - 2 < hi ? e - 2 : hi;
}

// Codes of 8 packed values at a scale byte (rounded to nearest, ties to the
// even code, past 6 to 6), the first in the low bits.  (The dwords by value: a
// bit cast of a vector's element reads element 0.)
template <typename T>
__device__ __forceinline__ uint32_t fp4_codes(u32x4 x, uint32_t scale);
#define HCP_FP4_CODES(T, V2, CVT)                                                 \
  template <>                                                                     \
  __device__ __forceinline__ uint32_t fp4_codes<T>(u32x4 x, uint32_t scale) {     \
    const float s = __uint_as_float(scale << 23);                                 \
    const uint32_t w0 = x[0], w1 = x[1], w2 = x[2], w3 = x[3];                    \
    uint32_t c = CVT(0u, __builtin_bit_cast(V2, w0), s, 0);                       \
    c = CVT(c, __builtin_bit_cast(V2, w1), s, 1);                                 \
    c = CVT(c, __builtin_bit_cast(V2, w2), s, 2);                                 \
    c = CVT(c, __builtin_bit_cast(V2, w3), s, 3);                                 \
    return scale == 255 ? 0u : c;                                                 \
  }
HCP_FP4_CODES(__bf16, bf16x2, __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16)
HCP_FP4_CODES(_Float16, f16x2, __builtin_amdgcn_cvt_scalef32_pk_fp4_f16)
#undef HCP_FP4_CODES

// Two packed values of the codes in byte SEL of a dword; exact (the scale is a
// power of two whose products are in range), NaN for scale byte 255.
template <typename T, int SEL>
__device__ __forceinline__ uint32_t fp4_pair(uint32_t codes, float scale) {
  if constexpr (__is_same(T, __bf16))
    return __builtin_bit_cast(uint32_t,
                              __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, SEL));
  else
    return __builtin_bit_cast(uint32_t,
                              __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, SEL));
}
template <typename T>
__device__ __forceinline__ u32x4 fp4_values(uint32_t codes, float scale) {
  return u32x4{fp4_pair<T, 0>(codes, scale), fp4_pair<T, 1>(codes, scale),
               fp4_pair<T, 2>(codes, scale), fp4_pair<T, 3>(codes, scale)};
}

// The larger of x over the four lanes of a quad (one scale's 32 columns, eight
// to a lane).
__device__ __forceinline__ uint32_t quad_max(uint32_t x) {
  uint32_t y = __builtin_amdgcn_update_dpp(0, x, 0xb1, 0xf, 0xf, true);  // quad_perm 1,0,3,2
  x = x > y ? x : y;
  y = __builtin_amdgcn_update_dpp(0, x, 0x4e, 0xf, 0xf, true);  // quad_perm 2,3,0,1
  return x > y ? x : y;
}

// Eight columns (octet oct) of one key's K or V row into a region: the lanes of
// a quad hold the four octets of a scale.
template <typename T>
__device__ __forceinline__ void fp4_store(char* region, Fp4Region r, bool is_v, int off, int oct,
                                          u32x4 x) {
  const uint32_t scale = fp4_scale<T>(quad_max(mag_max8(x)));
  *reinterpret_cast<uint32_t*>(region + (is_v ? r.v_code(off, oct) : r.k_code(off, oct))) =
      fp4_codes<T>(x, scale);
  if ((oct & 3) == 0)
    region[is_v ? r.v_scale(off, oct >> 2) : r.k_scale(off, oct >> 2)] = static_cast<char>(scale);
}

}  // namespace hcp
