// Cosines and sines by position, the table that qk_rope.hip reads:
//   row t = [cos(t f_i) a, i < rot / 2 | sin(t f_i) a, i < rot / 2].
//
// At position 10^6 a 32-bit angle would be off by 0.06.  Here an angle is a 64-bit
// fraction of a turn, t (f_i / 2 pi) modulo 1: exact but for the frequency's own
// rounding, and the next row's is one addition away.  Its upper 32 bits say which half of
// the turn, which turns both signs, and an angle within a quarter turn of that; there sine
// and cosine are minimax polynomials in x^2 (of degrees 9 and 10 in x, by exchange, the
// leading terms x and 1 - x^2 / 2), off by 2^-28 and 2^-31, so that 32-bit rounding is
// what counts: 2^-22.9 and 2^-23.4 measured over 2 million angles, 4.9e-8 on average where a
// float32's rounding alone is 2.1e-8.  (With angle and polynomials in 64 bits a float32 table of
// 131072 x 128 took 13.7 us for 12.3; what is rotated with it is rounded to 16 bits or fewer.)
//
// Bound by the writes: nothing is read but the frequencies, which are kernel arguments.  A
// pair takes 24 instructions; reduced in 64-bit floating point to quarters of a turn it
// took 40, and a 1000003 x 128 bf16 table (256 MB) 59 us; so 39 into one buffer, 43 a call into
// others (a fill takes 36.6 and 38.5).  131072 x 128 in float32 (67 MB) 12, a fill 11.3; 4096 x 64
// 2.6.
#include "params.h"

namespace hcp {

constexpr int kTableThreads = 256;
// A workgroup makes four passes over rows in a row, fewer where that leaves less than eight
// workgroups to a CU.  (1000003 x 128 bf16 into another buffer each time 43 us; with three, five
// and eight passes 45, 49 and 50, with 2048 workgroups that take rows far apart 48.  131072 x
// 128 float32 11.8 for 12.)
constexpr int kTableBlocks = 2048, kTablePasses = 4;

// A workgroup writes `rows` rows in a row, a thread 16 bytes of cosines and 16 of sines of
// every step-th of them.
template <typename T>
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
      const uint32_t q = static_cast<uint32_t>(phase[j] >> 32) + 0x40000000u;
      phase[j] += next[j];
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
      const float a = __uint_as_float(__float_as_uint(p.factor) ^ (q & 0x80000000u));
      c[j] = static_cast<T>(__builtin_fmaf(z, v, 1.f) * a);
      s[j] = static_cast<T>(__builtin_fmaf(x * z, u, x) * a);
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
  if (dtype == HCP_DTYPE_F32)
    hipLaunchKernelGGL(rope_table_kernel<float>, g, b, 0, st, p, rows);
  else if (dtype == HCP_DTYPE_BF16)
    hipLaunchKernelGGL(rope_table_kernel<__bf16>, g, b, 0, st, p, rows);
  else
    hipLaunchKernelGGL(rope_table_kernel<_Float16>, g, b, 0, st, p, rows);
  return hipGetLastError();
}

}  // namespace hcp
