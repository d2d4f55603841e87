// Cosines and sines by position, the table that qk_rope.hip reads:
//   row t = [cos(t f_i) a, i < rot / 2 | sin(t f_i) a, i < rot / 2].
//
// At position 10^6 a 32-bit angle would be off by 0.06.  Here an angle is a 64-bit
// fraction of a turn, t (f_i / 2 pi) modulo 1: exact but for the frequency's own
// rounding, and the next row's is one addition away.  From there, by the table's type:
//
// float32: the angle within an eighth of a turn of a quarter's end, as a float and what is
// left of it (2^-47); sine and cosine are minimax polynomials in x^2 (of degrees 7 and 8 in x, by
// exchange, the leading terms x and 1 - x^2 / 2), off by 2^-29 and 2^-33, and the last addition
// is the only rounding of a whole value: off by 2^-23.7 at most, and by 1.1 times what
// rounding alone is on average.  The factor comes in two terms for the same reason.
//
// 16 bits: the upper 32 bits say which half of the turn, which turns both signs, and an
// angle within a quarter turn of that, whose polynomials (degrees 9 and 10) are off by
// 2^-25.8 and 2^-27.6: in all by 2^-22 (2^-22.05 and 2^-22.8 over 20 million angles), a
// 2^-14th of bf16's step below 1 and a 2^-11th of fp16's.  (Small sines are off by 10^-9 as the
// others are, those below 2^-21 by more than their own half step.)  Two thirds of the
// instructions, and those bound these tables.
//
// Bound by the writes: nothing is read but the frequencies, which are kernel arguments.  A
// pair takes 24 instructions in 16 bits (40 with angles and polynomials in 64: a 1000003 x
// 128 bf16 table, 256 MB, 59 us for 39 into one buffer, 43 a call into others; a fill takes
// 36.6 and 38.5) and 37 in float32 (131072 x 128, 67 MB, with a factor 12.3 us, 11.8 with what 16
// bits take, 13.7 with 64, a fill 11.3).  4096 x 64 float32 2.6.
#include "params.h"

namespace hcp {

constexpr int kTableThreads = 256;
// A workgroup makes four passes over rows in a row, fewer where that leaves less than eight
// workgroups to a CU.  (1000003 x 128 bf16 into another buffer each time 43 us; with three, five
// and eight passes 45, 49 and 50, with 2048 workgroups that take rows far apart 48.  131072 x
// 128 float32 12.4; with two passes, 4096 workgroups, 13.2, with eight 12.6.)
constexpr int kTableBlocks = 2048, kTablePasses = 4;

// Cosine and sine of a turn's fraction, times the factor (FACTOR) in its two terms.
template <bool FACTOR>
__device__ __forceinline__ void cos_sin32(uint64_t phase, float f, float f_lo, float& c, float& s) {
#pragma clang fp contract(off)
  constexpr float kUnit = 0x1.921fb6p-32f, kUnitLo = -0x1.777a5cp-57f;  // 2 pi / 2^34
  const uint32_t q = static_cast<uint32_t>(phase >> 32);
  // from the nearest quarter's end: 24 bits (of q times 4), and the 32 behind them
  const float h = static_cast<float>(static_cast<int32_t>(((q << 2) + 128u) & ~255u));
  const float lo = static_cast<float>(
      static_cast<int32_t>(__builtin_amdgcn_alignbit(q, static_cast<uint32_t>(phase), 6)));
  const float p = h * kUnit;
  const float rest = __builtin_fmaf(
      lo, kUnit * 0x1p-24f, __builtin_fmaf(h, kUnitLo, __builtin_fmaf(h, kUnit, -p)));
  const float z = p * p;
  float u = __builtin_fmaf(z, -1.94955661e-04f, 8.33197776e-03f);
  u = __builtin_fmaf(z, u, -1.66666508e-01f);
  float v = __builtin_fmaf(z, 2.44383773e-05f, -1.38873665e-03f);
  v = __builtin_fmaf(z, v, 4.16666456e-02f);
  const float x = __builtin_fmaf(p * z, u, rest);  // sine less p, cosine less 1
  const float y = __builtin_fmaf(z, __builtin_fmaf(z, v, -0.5f), -(p * rest));
  float cr, sr;
  if constexpr (FACTOR) {
    const float m = f * p;
    sr = m + __builtin_fmaf(f, x, __builtin_fmaf(f_lo, p, __builtin_fmaf(f, p, -m)));
    cr = f + __builtin_fmaf(f, y, __builtin_fmaf(f_lo, y, f_lo));
  } else {
    sr = p + x;
    cr = 1.f + y;
  }
  // quarters of a turn, rounded as h is (an eighth, and half of its step): 1 and 3 swap the
  // two, 2 and 3 turn the sine, 1 and 2 the cosine
  const uint32_t k = q + 0x20000020u, odd = k << 1;
  const bool swap = static_cast<int32_t>(odd) < 0;
  c = __uint_as_float(__float_as_uint(swap ? sr : cr) ^ ((k ^ odd) & 0x80000000u));
  s = __uint_as_float(__float_as_uint(swap ? cr : sr) ^ (k & 0x80000000u));
}

// To 2^-22, for values that are rounded to 16 bits.
__device__ __forceinline__ void cos_sin16(uint64_t phase, float f, float& c, float& s) {
  const uint32_t q = static_cast<uint32_t>(phase >> 32) + 0x40000000u;
  const float x = static_cast<float>(static_cast<int32_t>(q & 0x7fffffffu) - 0x40000000) *
                  1.4629180792671596e-09f;  // 2 pi / 2^32
  const float z = x * x;
  float u = __builtin_fmaf(z, 2.6000548e-06f, -1.9806615e-04f);
  u = __builtin_fmaf(z, u, 8.3330171e-03f);
  u = __builtin_fmaf(z, u, -1.6666657e-01f);
  float v = __builtin_fmaf(z, -2.6077106e-07f, 2.4761886e-05f);
  v = __builtin_fmaf(z, v, -1.3888404e-03f);
  v = __builtin_fmaf(z, v, 4.1666642e-02f);
  v = __builtin_fmaf(z, v, -0.5f);
  const float a = __uint_as_float(__float_as_uint(f) ^ (q & 0x80000000u));
  c = __builtin_fmaf(z, v, 1.f) * a;
  s = __builtin_fmaf(x * z, u, x) * a;
}

// A workgroup writes `rows` rows in a row, a thread 16 bytes of cosines and 16 of sines of
// every step-th of them.
template <typename T, bool FACTOR>
__global__ __launch_bounds__(kTableThreads) void rope_table_kernel(RopeTableParams p, int rows) {
  constexpr int N = 16 / sizeof(T);
  const int half = p.rot / 2, per = half / N, step = kTableThreads / per;
  const int first = threadIdx.x / per, col = (threadIdx.x - first * per) * N;
  int64_t row = static_cast<int64_t>(blockIdx.x) * rows + first;
  const int64_t all = static_cast<int64_t>(blockIdx.x + 1) * rows;
  const int64_t end = first >= step ? 0 : all < p.num_positions ? all : p.num_positions;
  uint64_t phase[N], next[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const uint64_t f = p.turns[col + j];
    phase[j] = f * static_cast<uint64_t>(row);
    next[j] = f * static_cast<uint64_t>(step);
  }
  T* to = reinterpret_cast<T*>(p.out) + row * p.stride + col;
  for (; row < end; row += step, to += step * p.stride) {
    T c[N], s[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      float cj, sj;
      if constexpr (sizeof(T) == 4)
        cos_sin32<FACTOR>(phase[j], p.factor, p.factor_lo, cj, sj);
      else
        cos_sin16(phase[j], p.factor, cj, sj);
      phase[j] += next[j];
      c[j] = static_cast<T>(cj);
      s[j] = static_cast<T>(sj);
    }
    u32x4 cw, sw;
    __builtin_memcpy(&cw, c, 16);
    __builtin_memcpy(&sw, s, 16);
    *reinterpret_cast<u32x4*>(to) = cw;
    *reinterpret_cast<u32x4*>(to + half) = sw;
  }
}

hipError_t launch_rope_table(const RopeTableParams& p, int dtype, hipStream_t st) {
  const int64_t per = p.rot / 2 / (dtype == HCP_DTYPE_F32 ? 4 : 8);
  const int64_t step = kTableThreads / per;  // rows of a workgroup's pass
  const int64_t some = (p.num_positions + step * kTableBlocks - 1) / (step * kTableBlocks);
  const int64_t passes = some < kTablePasses ? some : kTablePasses;
  const int rows = static_cast<int>(step * passes);
  const dim3 g(static_cast<unsigned>((p.num_positions + rows - 1) / rows)), b(kTableThreads);
  if (dtype == HCP_DTYPE_F32 && p.factor == 1.f && p.factor_lo == 0.f)
    hipLaunchKernelGGL((rope_table_kernel<float, false>), g, b, 0, st, p, rows);
  else if (dtype == HCP_DTYPE_F32)
    hipLaunchKernelGGL((rope_table_kernel<float, true>), g, b, 0, st, p, rows);
  else if (dtype == HCP_DTYPE_BF16)
    hipLaunchKernelGGL((rope_table_kernel<__bf16, true>), g, b, 0, st, p, rows);
  else
    hipLaunchKernelGGL((rope_table_kernel<_Float16, true>), g, b, 0, st, p, rows);
  return hipGetLastError();
}

}  // namespace hcp
