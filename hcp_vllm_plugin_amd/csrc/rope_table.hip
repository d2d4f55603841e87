// Cosines and sines by position, the table that qk_rope.hip reads:
//   row t = [cos(t f_i) a, i < rot / 2 | sin(t f_i) a, i < rot / 2].
//
// At position 10^6 a 32-bit angle would be off by 0.06, so the angle is formed and
// reduced in 64 bits: in turns, t (f_i / 2 pi), whose fraction is exact, then in
// quarters of a turn, of which the nearest whole one says which of the two functions
// and which sign.  What is left is within 1/8 turn and exact to 2^-24 of itself in 32
// bits, where the Taylor polynomials to x^9 and x^10 are off by less than 2^-28.
//
// Bound by the writes: nothing is read but the frequencies, which are kernel arguments.
#include "params.h"

namespace hcp {

__device__ __forceinline__ void cos_sin(double turns, float& c, float& s) {
  const double quarters = 4.0 * (turns - __builtin_rint(turns));
  const double whole = __builtin_rint(quarters);
  const int k = static_cast<int>(whole);
  const float x = static_cast<float>((quarters - whole) * 1.5707963267948966), z = x * x;
  float p = __builtin_fmaf(z, 1.f / 362880, -1.f / 5040);
  p = __builtin_fmaf(z, p, 1.f / 120);
  p = __builtin_fmaf(z, p, -1.f / 6);
  const float sx = __builtin_fmaf(x * z, p, x);
  float q = __builtin_fmaf(z, -1.f / 3628800, 1.f / 40320);
  q = __builtin_fmaf(z, q, -1.f / 720);
  q = __builtin_fmaf(z, q, 1.f / 24);
  q = __builtin_fmaf(z, q, -0.5f);
  const float cx = __builtin_fmaf(z, q, 1.f);
  const float a = k & 1 ? sx : cx, b = k & 1 ? cx : sx;
  c = (k + 1) & 2 ? -a : a;  // quarters 1 and 2
  s = k & 2 ? -b : b;        // quarters 2 and 3 (or -2 and -1)
}

constexpr int kTableThreads = 256;

// A thread writes 16 bytes of cosines and 16 of sines.
template <typename T>
__global__ __launch_bounds__(kTableThreads) void rope_table_kernel(RopeTableParams p) {
  constexpr int N = 16 / sizeof(T);
  const int half = p.rot / 2, per = half / N;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kTableThreads + threadIdx.x;
  const int64_t row = i / per;
  if (row >= p.num_positions) return;
  const int col = static_cast<int>(i - row * per) * N;
  T c[N], s[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    float cj, sj;
    cos_sin(static_cast<double>(row) * p.turns[col + j], cj, sj);
    c[j] = static_cast<T>(cj * p.factor);
    s[j] = static_cast<T>(sj * p.factor);
  }
  T* const to = reinterpret_cast<T*>(p.out) + row * p.stride + col;
  u32x4 cw, sw;
  __builtin_memcpy(&cw, c, 16);
  __builtin_memcpy(&sw, s, 16);
  *reinterpret_cast<u32x4*>(to) = cw;
  *reinterpret_cast<u32x4*>(to + half) = sw;
}

hipError_t launch_rope_table(const RopeTableParams& p, int dtype, hipStream_t st) {
  const int64_t per = p.rot / 2 / (dtype == HCP_DTYPE_F32 ? 4 : 8);
  const int64_t blocks = (p.num_positions * per + kTableThreads - 1) / kTableThreads;
  const dim3 g(static_cast<unsigned>(blocks)), b(kTableThreads);
  if (dtype == HCP_DTYPE_F32)
    hipLaunchKernelGGL(rope_table_kernel<float>, g, b, 0, st, p);
  else if (dtype == HCP_DTYPE_BF16)
    hipLaunchKernelGGL(rope_table_kernel<__bf16>, g, b, 0, st, p);
  else
    hipLaunchKernelGGL(rope_table_kernel<_Float16>, g, b, 0, st, p);
  return hipGetLastError();
}

}  // namespace hcp
