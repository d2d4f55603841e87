// What the split-KV decode kernels over the 4-bit cache share.
#pragma once

#include <type_traits>

#include "decode_share.h"

namespace hcp {

// A wave's tile (16 keys) in LDS: its codes, each lane's 16 bytes of a load next to
// the other lanes', then its scales.
template <int D>
struct Fp4Tile {
  static constexpr int NC = D / 64;             // loads of codes, 1 KB each
  static constexpr int SC = 1024 * NC;          // where the scales begin
  static constexpr int SW = D == 256 ? 32 : 16; // dwords of K (or V) scales
  static constexpr int BYTES = SC + 256;
  static constexpr int NI = NC + 1;             // loads
  static constexpr int P = D == 256 ? 2 : 1;    // 16-byte pieces of K (or V) per lane
};

#define HCP_LDS_PTR(T) __attribute__((address_space(3))) T*

template <typename T>
__device__ __forceinline__ T lds_at(const HCP_LDS_PTR(char) p) {
  return *reinterpret_cast<const HCP_LDS_PTR(T)>(p);
}

// How far (in powers of two) a score may pass the running maximum, and what the
// maximum's own weight is: fp16's terms have 2^-24 for their last place, so that
// weights begin 2^7 higher, the largest at 2^15 of its 65504.
constexpr float kRaise = 8.f;
template <typename T>
constexpr float kLift = __is_same(T, __bf16) ? 0.f : 7.f;

// Two weights (or NaN) in two 16-bit terms: hi the weight rounded, lo what is left of
// it, rounded: 2^-17 of it (fp16 2^-22, and 2^-25 at least).  Both to the nearest:
// cut off, many small weights next to a large one would add up to less than they are.
// (two_terms of common.h keeps both terms positive for products with an infinity; the
// 4-bit cache holds none.)
template <typename T>
__device__ __forceinline__ void split_weights(float a, float b, uint32_t& hi, uint32_t& lo) {
  hi = pack2<T>(a, b);
  lo = pack2<T>(a - Elem<T>::to_float(static_cast<uint16_t>(hi & 0xffffu)),
                b - Elem<T>::to_float(static_cast<uint16_t>(hi >> 16)));
}

// Byte J of a dword of scales as a float, in one instruction.
template <int J>
__device__ __forceinline__ float fp4_scale_of(uint32_t w) {
  uint32_t r;
  asm("v_lshlrev_b32_sdwa %0, %1, %2 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:DWORD "
      "src1_sel:BYTE_%3"
      : "=v"(r)
      : "v"(23), "v"(w), "n"(J));
  return __uint_as_float(r);
}

}  // namespace hcp
