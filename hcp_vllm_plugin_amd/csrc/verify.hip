// Verification of drafted tokens against the target's logits (or probabilities).
//
// Row i of a sequence has weights w = exp((x - max x) / temperature) with sum Z (or w =
// x).  Draft i, drawn from q, is accepted while u_i q(d) Z < w(d); the token after the
// accepted ones is drawn from r = max(w - q Z, 0) of the row that refused (w without d
// where there is no q), or from the last row's w: the first index at which the running
// sum of r passes u times the whole.  With temperature 0 a draft is accepted where it is
// the row's largest entry, and the token is that.
//
// Which side of a border a sum lies on decides a token, so what is compared with u is
// in 64 bits; 32 would give another token once in some hundred rows where the
// probabilities are flat.  But only one row of a sequence is drawn from.  So
//  1 verify_stats: every row once, in 32 bits: maximum, its index, the sum of the
//    weights, for slices of 8192 (the weights of a thread added in 32 bits, the rest
//    in 64).  Bound by HBM: this is what has to be read.
//  2 verify_decide, a workgroup to a sequence: accepts by those sums; where a draft
//    is so near the border that their error may matter, the row is summed again in 64
//    bits.
//  3 verify_sums: Z (or the sum of r, without q) of the drawn row in 64 bits, slices of
//    2048.
//  4 verify_residual (with q): the sum of r.
//  5 verify_pick: the slice, and in it the token.
// Sums are added in an order that the sizes alone decide, so that a call gives the same
// tokens every time.
#include "params.h"

namespace hcp {

constexpr int kVerThreads = 256;
constexpr int kVerWaves = kVerThreads / 64;
constexpr int kStatSlice = kVerStatSlice;  // 32 values to a thread
static_assert(kStatSlice == 32 * kVerThreads && kVerSumSlice == 8 * kVerThreads, "slices");

// (rows begin where their type may)
typedef uint32_t u32x4_u __attribute__((ext_vector_type(4), aligned(2)));
typedef const __attribute__((address_space(1))) u32x4_u gu32x4_u;
__device__ __forceinline__ u32x4 ldg16_u(const void* p) {
  return *reinterpret_cast<gu32x4_u*>(reinterpret_cast<uintptr_t>(p));
}

// Elements 8 g .. 8 g + 7 of a row of v, `fill` past its end.
template <typename T>
__device__ __forceinline__ void load8(const void* row, int g, int v, float fill, float (&x)[8]) {
  const T* const at = reinterpret_cast<const T*>(row) + 8 * static_cast<int64_t>(g);
  if (8 * g + 8 <= v) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const u32x4 w = ldg16_u(at + 4 * h);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[4 * h + j] = __uint_as_float(w[j]);
      }
    } else {
      const u32x4 w = ldg16_u(at);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[2 * j] = Elem<T>::to_float(static_cast<uint16_t>(w[j] & 0xffffu));
        x[2 * j + 1] = Elem<T>::to_float(static_cast<uint16_t>(w[j] >> 16));
      }
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    x[j] = fill;
    if (8 * g + j < v) x[j] = static_cast<float>(global_ptr(at)[j]);
  }
}

// The weight of an entry x of a row with maximum `top`: of logits in 64 bits.  -inf and
// NaN have none (and the target's probabilities below 0, or infinite).
template <bool PROBS>
__device__ __forceinline__ double weight(float x, float top, double inverse) {
  if constexpr (PROBS) return x > 0.f && x < INFINITY ? static_cast<double>(x) : 0.0;
  if (!(x > -INFINITY)) return 0.0;
  if (x == top) return 1.0;  // (an infinity too, and then nothing else)
  if (top == INFINITY) return 0.0;
  return exp((static_cast<double>(x) - static_cast<double>(top)) * inverse);
}

struct VerifySeq {  // of one sequence, in LDS or registers
  int64_t row0;
  int n;       // its rows
  bool greedy;
  double inverse;  // 1 / temperature
};
__device__ __forceinline__ VerifySeq verify_seq(const VerifyParams& p, int b) {
  VerifySeq s;
  int64_t a, z;
  if (p.starts_wide) {
    a = global_ptr(reinterpret_cast<const int64_t*>(p.row_starts))[b];
    z = global_ptr(reinterpret_cast<const int64_t*>(p.row_starts))[b + 1];
  } else {
    a = global_ptr(reinterpret_cast<const int32_t*>(p.row_starts))[b];
    z = global_ptr(reinterpret_cast<const int32_t*>(p.row_starts))[b + 1];
  }
  z = z < p.num_rows ? z : p.num_rows;
  s.row0 = a;
  s.n = a < 0 || z <= a ? 0 : z - a < p.max_tokens ? static_cast<int>(z - a) : p.max_tokens;
  const float t = p.temperature != nullptr ? global_ptr(p.temperature)[b] : 1.f;
  s.greedy = !(t > 0.f);
  s.inverse = s.greedy ? 1.0 : 1.0 / static_cast<double>(t);
  return s;
}
__device__ __forceinline__ const char* target_row(const VerifyParams& p, int64_t row) {
  return reinterpret_cast<const char*>(p.target) + row * p.row_bytes;
}
__device__ __forceinline__ int64_t draft_token(const VerifyParams& p, int64_t row) {
  return p.tokens_wide ? global_ptr(reinterpret_cast<const int64_t*>(p.tokens))[row]
                       : global_ptr(reinterpret_cast<const int32_t*>(p.tokens))[row];
}

// Larger value, or the lower index of equal ones.
__device__ __forceinline__ void best_of(float& m, int& i, float om, int oi) {
  if (om > m || (om == m && oi < i)) {
    m = om;
    i = oi;
  }
}

template <typename T, bool PROBS>
__global__ __launch_bounds__(kVerThreads) void verify_stats_kernel(VerifyParams p) {
  __shared__ float sm_m[kVerWaves];
  __shared__ int sm_i[kVerWaves];
  __shared__ double sm_s[kVerWaves];
  const int slice = blockIdx.x % p.stat_slices, unit = blockIdx.x / p.stat_slices;
  const int b = unit / p.max_tokens, j = unit - b * p.max_tokens;
  const VerifySeq s = verify_seq(p, b);
  if (j >= s.n) return;
  const char* const row = target_row(p, s.row0 + j);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  float x[4][8];
  float m = -INFINITY;
  int at = 0x7fffffff;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    load8<T>(row, (slice * kStatSlice / 8) + k * kVerThreads + tid, p.vocab, -INFINITY, x[k]);
#pragma unroll
  for (int k = 0; k < 4; ++k)
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (x[k][e] > m) {  // (the first of equal ones; no NaN)
        m = x[k][e];
        at = slice * kStatSlice + (k * kVerThreads + tid) * 8 + e;
      }
#pragma unroll
  for (int w = 32; w > 0; w >>= 1) best_of(m, at, __shfl_xor(m, w), __shfl_xor(at, w));
  if (lane == 0) {
    sm_m[wave] = m;
    sm_i[wave] = at;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kVerWaves; ++w) best_of(m, at, sm_m[w], sm_i[w]);
  const float c = static_cast<float>(s.inverse * 1.4426950408889634);
  float sum = 0.f;
#pragma unroll
  for (int k = 0; k < 4; ++k)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if constexpr (PROBS)
        sum += x[k][e] > 0.f && x[k][e] < INFINITY ? x[k][e] : 0.f;
      else
        sum += !(x[k][e] > -INFINITY) ? 0.f
               : x[k][e] == m         ? 1.f
               : m == INFINITY        ? 0.f
                                      : fast_exp2((x[k][e] - m) * c);
    }
  double d = sum;
#pragma unroll
  for (int w = 32; w > 0; w >>= 1) d += __shfl_xor(d, w);
  if (lane == 0) sm_s[wave] = d;
  __syncthreads();
  if (tid == 0) {
    d = 0.0;
#pragma unroll
    for (int w = 0; w < kVerWaves; ++w) d += sm_s[w];
    VerifyStat& o = p.stats[static_cast<int64_t>(unit) * p.stat_slices + slice];
    o.top = m;
    o.index = at;
    o.sum = d;
  }
}

// Sum over the workgroup of every thread's x, in a fixed order.
__device__ __forceinline__ double block_sum(double x, double* sm) {
#pragma unroll
  for (int w = 32; w > 0; w >>= 1) x += __shfl_xor(x, w);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = x;
  __syncthreads();
  double r = 0.0;
#pragma unroll
  for (int w = 0; w < kVerWaves; ++w) r += sm[w];
  return r;
}

// How far the 32-bit sums may be off, relative: a weight by 2^-22 and its argument's
// share, 2^-23 of |log2 w|, which over a row averages to its entropy (17.2 bits at
// 150000 tokens, 24 at most here); the additions in a thread by 32 steps of 2^-24.
constexpr double kSumError = 1e-5;

template <typename T, bool PROBS>
__global__ __launch_bounds__(kVerThreads) void verify_decide_kernel(VerifyParams p) {
  __shared__ float sm_top[kVerMaxTokens];
  __shared__ int sm_at[kVerMaxTokens];
  __shared__ double sm_z[kVerMaxTokens];
  __shared__ double sm_s[kVerWaves];
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const VerifySeq s = verify_seq(p, b);
  // the rows' maxima and sums from those of their slices
  for (int j = wave; j < s.n; j += kVerWaves) {
    const VerifyStat* const st =
        p.stats + (static_cast<int64_t>(b) * p.max_tokens + j) * p.stat_slices;
    float m = -INFINITY;
    int at = 0x7fffffff;
    for (int i = lane; i < p.stat_slices; i += 64) best_of(m, at, st[i].top, st[i].index);
#pragma unroll
    for (int w = 32; w > 0; w >>= 1) best_of(m, at, __shfl_xor(m, w), __shfl_xor(at, w));
    double z = 0.0;
    for (int i = lane; i < p.stat_slices; i += 64) {
      if constexpr (PROBS)
        z += st[i].sum;
      else if (st[i].sum > 0.0)
        z += st[i].sum * weight<false>(st[i].top, m, s.inverse);
    }
#pragma unroll
    for (int w = 32; w > 0; w >>= 1) z += __shfl_xor(z, w);
    if (lane == 0) {
      sm_top[j] = m;
      sm_at[j] = at;
      sm_z[j] = z;
    }
  }
  __syncthreads();
  int taken = 0;
  for (; taken + 1 < s.n; ++taken) {  // (the same in every thread)
    const int j = taken;
    const int64_t d = draft_token(p, s.row0 + j + 1);
    if (d < 0 || d >= p.vocab) break;
    if (s.greedy) {
      if (sm_at[j] != d) break;
      continue;
    }
    const char* const row = target_row(p, s.row0 + j);
    const double w =
        weight<PROBS>(static_cast<float>(global_ptr(reinterpret_cast<const T*>(row))[d]), sm_top[j],
                      s.inverse);
    double uq = global_ptr(p.uniform)[b * p.uniform_stride + j];
    if (p.draft_probs != nullptr)
      uq *= static_cast<double>(
          global_ptr(p.draft_probs)[b * p.q_stride_seq + j * p.q_stride_row + d]);
    double z = sm_z[j];
    if (fabs(uq * z - w) <= kSumError * w) {  // too near to tell: the row in 64 bits
      double x = 0.0;
      for (int g = tid; g < (p.vocab + 7) / 8; g += kVerThreads) {
        float e[8];
        load8<T>(row, g, p.vocab, -INFINITY, e);
#pragma unroll
        for (int k = 0; k < 8; ++k) x += weight<PROBS>(e[k], sm_top[j], s.inverse);
      }
      z = block_sum(x, sm_s);
    }
    if (!(uq * z < w)) break;
  }
  // tokens, and what the row that is drawn from is
  const float top = s.n > 0 ? sm_top[taken] : -INFINITY;
  const bool none = s.n == 0 || (PROBS ? !(sm_z[taken] > 0.0) && !(s.greedy && top > -INFINITY)
                                       : top == -INFINITY);
  const int64_t own = none ? -1 : s.greedy ? sm_at[taken] : -1;
  for (int j = tid; j < p.max_tokens; j += kVerThreads) {
    const int64_t t = j < taken ? draft_token(p, s.row0 + j + 1) : j == taken ? own : -1;
    const int64_t to = static_cast<int64_t>(b) * p.max_tokens + j;
    if (p.tokens_wide)
      reinterpret_cast<int64_t*>(p.out)[to] = t;
    else
      reinterpret_cast<int32_t*>(p.out)[to] = static_cast<int32_t>(t);
  }
  if (tid == 0) {
    p.num_out[b] = s.n == 0 ? 0 : taken + !none;
    VerifyRow& o = p.rows[b];
    o.row = none || s.greedy ? -1 : s.row0 + taken;
    o.taken = taken;
    o.refused = taken + 1 < s.n;
    o.top = top;
    o.inverse = s.inverse;
    const int64_t d = taken + 1 < s.n ? draft_token(p, s.row0 + taken + 1) : -1;
    o.draft = d >= 0 && d < p.vocab ? static_cast<int32_t>(d) : -1;
  }
}

// Entries 8 g .. of what a sequence is drawn from: with WEIGHTS the weights, else the
// residual r (w where nothing was refused).
template <typename T, bool PROBS, bool WEIGHTS>
__device__ __forceinline__ void drawn8(const VerifyParams& p, const VerifyRow& o, int b, int g,
                                       double z, double (&r)[8]) {
  float x[8];
  load8<T>(target_row(p, o.row), g, p.vocab, PROBS ? 0.f : -INFINITY, x);
#pragma unroll
  for (int k = 0; k < 8; ++k) r[k] = weight<PROBS>(x[k], o.top, o.inverse);
  if (WEIGHTS || !o.refused) return;
  if (p.draft_probs != nullptr) {
    float q[8];
    load8<float>(p.draft_probs + b * p.q_stride_seq + o.taken * p.q_stride_row, g, p.vocab, 0.f, q);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const double y = r[k] - static_cast<double>(q[k]) * z;
      r[k] = y > 0.0 ? y : 0.0;
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (8 * g + k == o.draft) r[k] = 0.0;
  }
}

// Sum of the slices' sums, in a fixed order, in every thread.
__device__ __forceinline__ double slices_sum(const double* part, int n, double* sm) {
  double x = 0.0;
  for (int i = threadIdx.x; i < n; i += kVerThreads) x += global_ptr(part)[i];
  return block_sum(x, sm);
}

// RESIDUAL false: Z of the drawn row, or without draft probabilities the sum of r;
// true: the sum of r, of a sequence that refused.
template <typename T, bool PROBS, bool RESIDUAL>
__global__ __launch_bounds__(kVerThreads) void verify_sums_kernel(VerifyParams p) {
  __shared__ double sm_s[kVerWaves];
  const int slice = blockIdx.x % p.sum_slices, b = blockIdx.x / p.sum_slices;
  const VerifyRow o = p.rows[b];
  if (o.row < 0 || (RESIDUAL && !o.refused)) return;
  const double z =
      RESIDUAL ? slices_sum(p.sums + static_cast<int64_t>(b) * p.sum_slices, p.sum_slices, sm_s) : 0.0;
  double r[8], x = 0.0;
  const int g = slice * kVerThreads + threadIdx.x;
  if (RESIDUAL || p.draft_probs == nullptr)
    drawn8<T, PROBS, false>(p, o, b, g, z, r);
  else
    drawn8<T, PROBS, true>(p, o, b, g, z, r);
#pragma unroll
  for (int k = 0; k < 8; ++k) x += r[k];
  x = block_sum(x, sm_s);
  if (threadIdx.x == 0)
    (RESIDUAL ? p.residuals : p.sums)[static_cast<int64_t>(b) * p.sum_slices + slice] = x;
}

// Prefix sums (inclusive) over the workgroup's threads.
__device__ __forceinline__ double block_prefix(double x, double* sm) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int w = 1; w < 64; w <<= 1) {
    const double y = __shfl_up(x, w);
    if (lane >= w) x += y;
  }
  __syncthreads();
  if (lane == 63) sm[wave] = x;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kVerWaves; ++w)
    if (w < wave) x += sm[w];
  return x;
}

// The first thread whose running sum passes `want`; where rounding leaves none, the
// last with a sum above 0 (-1: no such either).  own: the thread's sum, upto: with those
// before it.
__device__ __forceinline__ int first_past(double own, double upto, double want, int* sm) {
  __syncthreads();
  if (threadIdx.x == 0) {
    sm[0] = kVerThreads;
    sm[1] = -1;
  }
  __syncthreads();
  if (own > 0.0) {
    if (upto > want) atomicMin(&sm[0], static_cast<int>(threadIdx.x));
    atomicMax(&sm[1], static_cast<int>(threadIdx.x));
  }
  __syncthreads();
  return sm[0] < kVerThreads ? sm[0] : sm[1];
}
// The same of n values, one after the other; `before` becomes the sum before it.
template <typename F>
__device__ __forceinline__ int first_past_of(int n, double want, double& before, F value) {
  int at = -1;
  double run = before;
  for (int i = 0; i < n; ++i) {
    const double x = value(i);
    if (x > 0.0) {
      at = i;
      before = run;
      if (run + x > want) break;
    }
    run += x;
  }
  return at;
}

template <typename T, bool PROBS>
__global__ __launch_bounds__(kVerThreads) void verify_pick_kernel(VerifyParams p) {
  __shared__ double sm_s[kVerWaves], sm_c[kVerThreads + 1];
  __shared__ int sm_f[2], sm_slice;
  const int b = blockIdx.x, tid = threadIdx.x, n = p.sum_slices;
  const VerifyRow o = p.rows[b];
  if (o.row < 0) return;
  const int64_t to = static_cast<int64_t>(b) * p.max_tokens + o.taken;
  auto put = [&](int token) __attribute__((always_inline)) {
    if (p.tokens_wide)
      reinterpret_cast<int64_t*>(p.out)[to] = token;
    else
      reinterpret_cast<int32_t*>(p.out)[to] = token;
  };
  const double* const sums = p.sums + static_cast<int64_t>(b) * n;
  const double* part = sums;
  bool weights = !o.refused;
  double z = 0.0;
  if (o.refused && p.draft_probs != nullptr) {
    z = slices_sum(sums, n, sm_s);
    part = p.residuals + static_cast<int64_t>(b) * n;
  }
  double total = slices_sum(part, n, sm_s);
  if (o.refused && !(total > 0.0)) {  // w is nowhere above q Z: drawn from w
    if (p.draft_probs == nullptr) {   // (which is the draft alone)
      if (tid == 0) put(o.draft);
      return;
    }
    weights = true;
    part = sums;
    total = z;
  }
  const double want =
      static_cast<double>(global_ptr(p.uniform)[b * p.uniform_stride + p.max_tokens - 1]) * total;
  // the slice: every thread adds up some in a row
  const int per = (n + kVerThreads - 1) / kVerThreads, i0 = tid * per;
  double own = 0.0;
  for (int i = i0; i < i0 + per && i < n; ++i) own += global_ptr(part)[i];
  double upto = block_prefix(own, sm_s);
  if (tid == 0) sm_c[0] = 0.0;
  sm_c[tid + 1] = upto;
  int who = first_past(own, upto, want, sm_f);
  if (who < 0) return;  // (no thread has a sum: not where `total` is above 0)
  if (tid == who) {
    double before = sm_c[who];
    sm_slice = i0 + first_past_of(n - i0 < per ? n - i0 : per, want, before,
                                  [&](int i) { return global_ptr(part)[i0 + i]; });
    sm_c[kVerThreads] = before;
  }
  __syncthreads();
  const int slice = sm_slice;
  double before = sm_c[kVerThreads];
  // the token in it
  double r[8];
  const int g = slice * kVerThreads + tid;
  if (weights)
    drawn8<T, PROBS, true>(p, o, b, g, z, r);
  else
    drawn8<T, PROBS, false>(p, o, b, g, z, r);
  own = 0.0;
#pragma unroll
  for (int k = 0; k < 8; ++k) own += r[k];
  upto = before + block_prefix(own, sm_s);
  sm_c[tid] = upto;
  who = first_past(own, upto, want, sm_f);
  if (tid == who) {
    before = tid > 0 ? sm_c[tid - 1] : before;
    const int k = first_past_of(8, want, before, [&](int i) { return r[i]; });
    put(8 * g + k);
  }
}

template <typename T, bool PROBS>
static hipError_t launch_verify_t(const VerifyParams& p, hipStream_t st) {
  const dim3 t(kVerThreads), seqs(static_cast<unsigned>(p.num_seqs));
  const dim3 slices(static_cast<unsigned>(p.num_seqs * p.sum_slices));
  hipLaunchKernelGGL((verify_stats_kernel<T, PROBS>),
                     dim3(static_cast<unsigned>(p.num_seqs * p.max_tokens * p.stat_slices)), t, 0,
                     st, p);
  hipLaunchKernelGGL((verify_decide_kernel<T, PROBS>), seqs, t, 0, st, p);
  hipLaunchKernelGGL((verify_sums_kernel<T, PROBS, false>), slices, t, 0, st, p);
  if (p.draft_probs != nullptr)
    hipLaunchKernelGGL((verify_sums_kernel<T, PROBS, true>), slices, t, 0, st, p);
  hipLaunchKernelGGL((verify_pick_kernel<T, PROBS>), seqs, t, 0, st, p);
  return hipGetLastError();
}

hipError_t launch_verify(const VerifyParams& p, int dtype, bool probs, hipStream_t st) {
  switch (dtype) {
    case HCP_DTYPE_F32:
      return probs ? launch_verify_t<float, true>(p, st) : launch_verify_t<float, false>(p, st);
    case HCP_DTYPE_BF16:
      return probs ? launch_verify_t<__bf16, true>(p, st) : launch_verify_t<__bf16, false>(p, st);
    default:
      return probs ? launch_verify_t<_Float16, true>(p, st)
                   : launch_verify_t<_Float16, false>(p, st);
  }
}

}  // namespace hcp
