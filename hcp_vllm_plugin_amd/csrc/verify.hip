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
// Few slices are decided by every workgroup of verify_sums for itself (1 x 4 rows of 32000:
// 18 us a call for 20); in small vocabularies a workgroup does 2 to 5 for its sequence
// (verify_finish: 200 x 1-8 rows of 50257 float32 probabilities 56 us a call for 74).
// Sums are added in an order that the sizes alone decide, so that a call gives the same
// tokens every time.
//
// 64 x 5 rows of 152064 bf16 logits with q (97 MB of logits read, 39 MB of the drawn
// rows' q): 18 us, 5, 11, 10 and 5; the two sums in 64 bits are bound by their
// exponentials and by starting behind one another.  200 x 1-8 rows of 50257
// probabilities: 29 us (177 MB) and 20.
#include "params.h"

namespace hcp {

constexpr int kVerWaves = kVerThreads / 64;
constexpr int kVerSmall = 65536;  // a vocabulary that one workgroup goes over
constexpr int kStatSlice = kVerStatSlice;  // 32 values to a thread
static_assert(kStatSlice == 32 * kVerThreads && kVerSumSlice == 8 * kVerThreads, "slices");

// (rows begin where their type may)
typedef uint32_t u32x4_u __attribute__((ext_vector_type(4), aligned(2)));
typedef const __attribute__((address_space(1))) u32x4_u gu32x4_u;
__device__ __forceinline__ u32x4 ldg16_u(const void* p) {
  return *reinterpret_cast<gu32x4_u*>(reinterpret_cast<uintptr_t>(p));
}

// Elements 8 g .. 8 g + 7 of a row, all of them there.
template <typename T>
__device__ __forceinline__ void load8_full(const void* row, int g, float (&x)[8]) {
  const T* const at = reinterpret_cast<const T*>(row) + 8 * static_cast<int64_t>(g);
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
}
// The same of a row of v, `fill` past its end.
template <typename T>
__device__ __forceinline__ void load8(const void* row, int g, int v, float fill, float (&x)[8]) {
  if (8 * g + 8 <= v) return load8_full<T>(row, g, x);
  const T* const at = reinterpret_cast<const T*>(row) + 8 * static_cast<int64_t>(g);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    x[j] = fill;
    if (8 * g + j < v) x[j] = static_cast<float>(global_ptr(at)[j]);
  }
}
// N of them, groups g, g + STEP, ..; `end`: past the workgroup's last element.  (A
// branch around every load would have each waited for by itself: 64 x 5 rows of 152064
// bf16 took 21 us.)
template <typename T, int N, int STEP = kVerThreads>
__device__ __forceinline__ void load8s(const void* row, int g, int end, int v, float fill,
                                       float (&x)[N][8]) {
  if (end <= v) {
#pragma unroll
    for (int k = 0; k < N; ++k) load8_full<T>(row, g + k * STEP, x[k]);
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) load8<T>(row, g + k * STEP, v, fill, x[k]);
  }
}

// 2^y for y <= 0 in 64 bits: the fraction's polynomial (Chebyshev interpolation on +-1/2,
// off by 3.2e-16 of it), scaled.  Below -1100, and for a NaN: 0.  (As fast as a 32-bit
// one would be: additions and products of 64 bits take no longer here.)
__device__ __forceinline__ double exp2_64(double y) {
  y = __builtin_fmax(y, -1100.0);
  const double n = __builtin_rint(y), r = y - n;
  double p = 7.072585949269224e-09;
  p = __builtin_fma(p, r, 1.0208690299958306e-07);
  p = __builtin_fma(p, r, 1.321544258792169e-06);
  p = __builtin_fma(p, r, 1.5252657260200837e-05);
  p = __builtin_fma(p, r, 0.0001540353044173605);
  p = __builtin_fma(p, r, 0.0013333558230164974);
  p = __builtin_fma(p, r, 0.009618129107606888);
  p = __builtin_fma(p, r, 0.05550410866444772);
  p = __builtin_fma(p, r, 0.24022650695910097);
  p = __builtin_fma(p, r, 0.69314718055995);
  p = __builtin_fma(p, r, 1.0);
  return __builtin_amdgcn_ldexp(p, static_cast<int>(n));
}

// The weight of an entry x of a row with maximum `top`: of logits 2^((x - top) rate), rate =
// log2 e / temperature.  -inf and NaN have none (they come out of the maximum above as
// -1100), and next to an infinity nothing else has; probabilities below 0, or infinite,
// have none.
template <bool PROBS>
__device__ __forceinline__ double weight(float x, float top, double rate) {
  if constexpr (PROBS) return x > 0.f && x < INFINITY ? static_cast<double>(x) : 0.0;
  if (top == INFINITY) return x == INFINITY ? 1.0 : 0.0;
  return exp2_64((static_cast<double>(x) - static_cast<double>(top)) * rate);
}

struct VerifySeq {  // of one sequence, in LDS or registers
  int64_t row0;
  int n;       // its rows
  bool greedy;
  double rate;  // log2 e / temperature
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
  s.rate = 1.4426950408889634 / (s.greedy ? 1.0 : static_cast<double>(t));
  return s;
}
__device__ __forceinline__ const char* target_row(const VerifyParams& p, int64_t row) {
  return reinterpret_cast<const char*>(p.target) + row * p.row_bytes;
}
__device__ __forceinline__ int64_t draft_token(const VerifyParams& p, int64_t row) {
  return p.tokens_wide ? global_ptr(reinterpret_cast<const int64_t*>(p.tokens))[row]
                       : global_ptr(reinterpret_cast<const int32_t*>(p.tokens))[row];
}

// Prefix sums over the wave's lanes (and their whole, by the last lane) by DPP moves: two
// and an addition a step, where a shuffle through LDS takes as long as ten of them.
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_add(double x) {
  const uint64_t w = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(w), CTRL, ROWS, 0xf, false);
  const uint32_t hi =
      __builtin_amdgcn_update_dpp(0, static_cast<int>(w >> 32), CTRL, ROWS, 0xf, false);
  return x + __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
__device__ __forceinline__ double wave_prefix64(double x) {
  x = dpp_add<0x111, 0xf>(x);  // row_shr:1
  x = dpp_add<0x112, 0xf>(x);
  x = dpp_add<0x114, 0xf>(x);
  x = dpp_add<0x118, 0xf>(x);
  x = dpp_add<0x142, 0xa>(x);  // row_bcast:15
  return dpp_add<0x143, 0xc>(x);  // row_bcast:31
}
__device__ __forceinline__ double last_lane(double x) {
  const uint64_t w = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(w), 63);
  const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(w >> 32), 63);
  return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
__device__ __forceinline__ double wave_sum(double x) { return last_lane(wave_prefix64(x)); }
// Maximum over the wave's lanes; no NaN among them.
template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp_max(float x) {
  return fmaxf(x, __int_as_float(__builtin_amdgcn_update_dpp(
                      __float_as_int(-INFINITY), __float_as_int(x), CTRL, ROWS, 0xf, false)));
}
__device__ __forceinline__ float wave_max(float x) {
  x = dpp_max<0x111, 0xf>(x);
  x = dpp_max<0x112, 0xf>(x);
  x = dpp_max<0x114, 0xf>(x);
  x = dpp_max<0x118, 0xf>(x);
  x = dpp_max<0x142, 0xa>(x);
  x = dpp_max<0x143, 0xc>(x);
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 63));
}

// Larger value, or the lower index of equal ones.
__device__ __forceinline__ void best_of(float& m, int& i, float om, int oi) {
  if (om > m || (om == m && oi < i)) {
    m = om;
    i = oi;
  }
}

// The largest of three, in one instruction; anything where one is a NaN.  (fmaxf would have
// every value of a row made quiet first.)
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

// A thread's 32 values stay in registers between the maximum and the weights.  A greedy
// row needs the index of its maximum and no weights, another one no index.
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
  load8s<T, 4>(row, slice * kStatSlice / 8 + tid, (slice + 1) * kStatSlice, p.vocab, -INFINITY, x);
  if (!PROBS || s.greedy) {
    float t = m;
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int e = 0; e < 8; e += 2) t = max3(t, x[k][e], x[k][e + 1]);
    m = t;
    // a NaN may have taken the place of the maximum
    bool nan = false;
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int e = 0; e < 8; e += 2) nan |= __builtin_isunordered(x[k][e], x[k][e + 1]);
    if (__builtin_amdgcn_ballot_w64(nan) != 0) {
      m = -INFINITY;
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (!(x[k][e] > -INFINITY)) x[k][e] = -INFINITY;
          m = x[k][e] > m ? x[k][e] : m;
        }
    }
    m = wave_max(m);
    if (lane == 0) sm_m[wave] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kVerWaves; ++w) m = fmaxf(m, sm_m[w]);
  }
  int at = 0x7fffffff;
  double d = 0.0;
  if (s.greedy) {
#pragma unroll
    for (int k = 3; k >= 0; --k)
#pragma unroll
      for (int e = 7; e >= 0; --e)
        if (x[k][e] == m) at = slice * kStatSlice + (k * kVerThreads + tid) * 8 + e;
#pragma unroll
    for (int w = 32; w > 0; w >>= 1) {
      const int o = __shfl_xor(at, w);
      at = o < at ? o : at;
    }
    if (lane == 0) sm_i[wave] = at;
  } else {
    // (six additions deep: what their rounding may come to is in kSumError)
    float sums[8] = {};
    auto add = [&](auto f) __attribute__((always_inline)) {
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int e = 0; e < 8; ++e) sums[e] += f(x[k][e]);
    };
    float scale = 1.f;
    if constexpr (PROBS) {
      add([](float v) __attribute__((always_inline)) { return v > 0.f && v < INFINITY ? v : 0.f; });
    } else if (m == INFINITY) {
      add([](float v) __attribute__((always_inline)) { return v == INFINITY ? 1.f : 0.f; });
    } else if (m > -INFINITY) {
      // (x - m) c in one fma: what m c loses to rounding, 1/8 at most, is the same power for
      // all.  (Without that bound it would pass the exponent's range: m = 30 at a temperature
      // of 10^-8 has lost = 200.)
      const float c = fminf(static_cast<float>(s.rate), 0x1p126f);
      const float mc = m * c, lost = __builtin_fmaf(m, c, -mc);
      if (c > 0.f && fabsf(mc) < 0x1p22f) {
        add([&](float v) __attribute__((always_inline)) {
          return fast_exp2(__builtin_fmaf(v, c, -mc));
        });
        scale = fast_exp2(-lost);
      } else {  // (halves where v - m may pass 32 bits' range; a NaN, of -inf times 0, to 0)
        const float h = fabsf(m) < 0x1p100f ? 1.f : 0.5f, ch = c / h, mh = m * h;
        add([&](float v) __attribute__((always_inline)) {
          return fast_exp2(fmaxf(__builtin_fmaf(v, h, -mh) * ch, -INFINITY));
        });
      }
    }
    const float sum = scale * (((sums[0] + sums[1]) + (sums[2] + sums[3])) +
                               ((sums[4] + sums[5]) + (sums[6] + sums[7])));
    d = wave_sum(sum);
    if (lane == 0) sm_s[wave] = d;
  }
  __syncthreads();
  if (tid == 0) {
    VerifyStat o{m, 0x7fffffff, 0.0};
#pragma unroll
    for (int w = 0; w < kVerWaves; ++w) {
      if (s.greedy)
        o.index = sm_i[w] < o.index ? sm_i[w] : o.index;
      else
        o.sum += sm_s[w];
    }
    p.stats[static_cast<int64_t>(unit) * p.stat_slices + slice] = o;
  }
}

// Sum over a workgroup of W waves of every thread's x, in a fixed order.
template <int W = kVerWaves>
__device__ __forceinline__ double block_sum(double x, double* sm) {
  x = wave_sum(x);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = x;
  __syncthreads();
  double r = 0.0;
#pragma unroll
  for (int w = 0; w < W; ++w) r += sm[w];
  return r;
}

// How far the 32-bit sums may be off, relative.  A weight's argument, log2 w, by 2^-23 of
// itself (its factor's rounding and its own, and 2^-27 for what m c lost; 3 2^-24 where the
// products are large): the weight by ln 2 times that, which over the weights of a slice, the
// largest of them 1, averages to no more than its entropy, 13 bits; 1.6e-6.  The exponential
// and the factor of the whole by 2^-23 and 2^-22, six additions and a product by 2^-24 each:
// 0.8e-6.  For rates of kLeastRate to kMostRate, which the kernel's 32-bit factor holds to
// 2^-24.
constexpr double kSumError = 2.5e-6, kLeastRate = 0x1p-126, kMostRate = 0x1p126;

template <int W>
struct DecideShared {
  float top[kVerMaxTokens];
  int at[kVerMaxTokens];
  double z[kVerMaxTokens], uq[kVerMaxTokens], w[kVerMaxTokens];
  double sums[W];
  uint64_t ok, near;
  VerifyRow row;
};

// Which drafts of sequence b are accepted, by a workgroup of W waves: gives what the one
// token more is drawn from, and with `write` writes the tokens and their number.
template <typename T, bool PROBS, int W>
__device__ __forceinline__ VerifyRow decide(const VerifyParams& p, int b, DecideShared<W>& sm,
                                            bool write = true) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const VerifySeq s = verify_seq(p, b);
  // lane i of every wave looks at draft i.  Its token is fetched with the slices' sums of
  // the wave's first row, its numbers while those are added up
  const bool mine = lane + 1 < s.n;
  auto stats_of = [&](int j) __attribute__((always_inline)) {
    return p.stats + (static_cast<int64_t>(b) * p.max_tokens + j) * p.stat_slices;
  };
  auto first_of = [&](int j) __attribute__((always_inline)) {  // of this lane's first slice
    VerifyStat o{-INFINITY, 0x7fffffff, 0.0};
    if (j < s.n && lane < p.stat_slices) o = global_ptr(stats_of(j))[lane];
    return o;
  };
  VerifyStat slice = first_of(wave);
  const int64_t d = mine ? draft_token(p, s.row0 + lane + 1) : -1;
  const bool token = d >= 0 && d < p.vocab;
  float xd = -INFINITY, ud = 0.f, qd = 1.f;
  if (token && !s.greedy) {
    xd = static_cast<float>(
        global_ptr(reinterpret_cast<const T*>(target_row(p, s.row0 + lane)))[d]);
    ud = global_ptr(p.uniform)[b * p.uniform_stride + lane];
    if (p.draft_probs != nullptr)
      qd = global_ptr(p.draft_probs)[b * p.q_stride_seq + lane * p.q_stride_row + d];
  }
  // the rows' maxima and sums from those of their slices
  for (int j = wave; j < s.n; j += W) {
    const VerifyStat* const st = stats_of(j);
    if (j > wave) slice = first_of(j);
    float m = slice.top;
    int at = slice.index;
    for (int i = lane + 64; i < p.stat_slices; i += 64)
      best_of(m, at, global_ptr(st)[i].top, global_ptr(st)[i].index);
#pragma unroll
    for (int w = 32; w > 0; w >>= 1) best_of(m, at, __shfl_xor(m, w), __shfl_xor(at, w));
    auto part = [&](const VerifyStat& o) __attribute__((always_inline)) {
      return PROBS ? o.sum : o.sum > 0.0 ? o.sum * weight<false>(o.top, m, s.rate) : 0.0;
    };
    double z = part(slice);
    for (int i = lane + 64; i < p.stat_slices; i += 64) z += part(global_ptr(st)[i]);
    z = wave_sum(z);
    if (lane == 0) {
      sm.top[j] = m;
      sm.at[j] = at;
      sm.z[j] = z;
    }
  }
  __syncthreads();
  if (wave == 0) {
    const double uq = static_cast<double>(ud) * static_cast<double>(qd);
    bool ok = false, near = false;
    if (token) {
      if (s.greedy) {
        ok = sm.at[lane] == d && sm.top[lane] > -INFINITY;  // (a row without entries has 0 there)
      } else {
        const double w = weight<PROBS>(xd, sm.top[lane], s.rate), v = uq * sm.z[lane];
        ok = v < w;
        // (probabilities may pass 32 bits' range in a thread's sum; the largest weight of
        // logits is 1, so that a sum below that would be none)
        near = w > 0.0 && (fabs(v - w) <= kSumError * w || !(sm.z[lane] < INFINITY) ||
                           (!PROBS && !(sm.z[lane] >= 0.5 && s.rate >= kLeastRate &&
                                        s.rate <= kMostRate)));
        sm.uq[lane] = uq;
        sm.w[lane] = w;
      }
    }
    const uint64_t oks = __builtin_amdgcn_ballot_w64(ok), nears = __builtin_amdgcn_ballot_w64(near);
    if (lane == 0) {
      sm.ok = oks;
      sm.near = nears;
    }
  }
  __syncthreads();
  int taken = 0;
  for (; taken + 1 < s.n; ++taken) {  // (the same in every thread)
    if (sm.near >> taken & 1) {  // too near to tell: the row in 64 bits
      const char* const row = target_row(p, s.row0 + taken);
      double x[4] = {};
      for (int g = tid; g < (p.vocab + 7) / 8; g += 4 * 64 * W) {  // four on their way
        float e[4][8];
        load8s<T, 4, 64 * W>(row, g, 8 * (g + 3 * 64 * W + 1), p.vocab, -INFINITY, e);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int k = 0; k < 8; ++k) x[i] += weight<PROBS>(e[i][k], sm.top[taken], s.rate);
      }
      if (!(sm.uq[taken] * block_sum<W>((x[0] + x[1]) + (x[2] + x[3]), sm.sums) < sm.w[taken])) break;
    } else if (!(sm.ok >> taken & 1)) {
      break;
    }
  }
  // tokens, and what the row that is drawn from is
  const float top = s.n > 0 ? sm.top[taken] : -INFINITY;
  const bool none = s.n == 0 || (PROBS && !s.greedy ? !(sm.z[taken] > 0.0) : top == -INFINITY);
  const int64_t own = none || !s.greedy ? -1 : sm.at[taken];
  if (wave == 0) {  // (lane i holds the draft that would be token i)
    if (write && lane < p.max_tokens) {
      const int64_t t = lane < taken ? d : lane == taken ? own : -1;
      const int64_t to = static_cast<int64_t>(b) * p.max_tokens + lane;
      if (p.tokens_wide)
        reinterpret_cast<int64_t*>(p.out)[to] = t;
      else
        reinterpret_cast<int32_t*>(p.out)[to] = static_cast<int32_t>(t);
    }
    if (lane == taken) {
      VerifyRow o;
      o.row = none || s.greedy ? -1 : s.row0 + taken;
      o.taken = taken;
      o.refused = mine;
      o.top = top;
      o.rate = s.rate;
      o.draft = token ? static_cast<int32_t>(d) : -1;
      sm.row = o;
      if (write) p.num_out[b] = s.n == 0 ? 0 : taken + !none;
    }
  }
  __syncthreads();
  return sm.row;
}

// (16 waves to a sequence for the drafts that are too near: a row of 152064 logits in 35 us, 49
// with four; one in 10^5 is)
template <typename T, bool PROBS>
__global__ __launch_bounds__(1024) void verify_decide_kernel(VerifyParams p) {
  __shared__ DecideShared<16> sm;
  const VerifyRow o = decide<T, PROBS, 16>(p, blockIdx.x, sm);
  if (threadIdx.x == 0) p.rows[blockIdx.x] = o;
}

// What 8 entries of a sequence's drawn row come to, x from the target and q from the draft
// (where `have`), the first of them entry 8 g: with `weights` the weights, else the residual
// r (w where nothing was refused).
template <bool PROBS>
__device__ __forceinline__ void drawn8(const VerifyRow& o, bool weights, bool have, int g, double z,
                                       const float (&x)[8], const float (&q)[8], double (&r)[8]) {
#pragma unroll
  for (int k = 0; k < 8; ++k) r[k] = weight<PROBS>(x[k], o.top, o.rate);
  if (weights || !o.refused) return;
  if (have) {
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
// The same from memory; `end`: past the workgroup's last entry.
template <typename T, bool PROBS>
__device__ __forceinline__ void drawn8(const VerifyParams& p, const VerifyRow& o, int b,
                                       bool weights, int g, int end, double z, double (&r)[8]) {
  float x[1][8], q[1][8];
  const bool have = p.draft_probs != nullptr && o.refused && !weights;
  load8s<T, 1>(target_row(p, o.row), g, end, p.vocab, PROBS ? 0.f : -INFINITY, x);
  if (have)
    load8s<float, 1>(p.draft_probs + b * p.q_stride_seq + o.taken * p.q_stride_row, g, end, p.vocab,
                     0.f, q);
  drawn8<PROBS>(o, weights, have, g, z, x[0], q[0], r);
}

// Sum of the slices' sums, in a fixed order, in every thread.
__device__ __forceinline__ double slices_sum(const double* part, int n, double* sm) {
  double x = 0.0;
  for (int i = threadIdx.x; i < n; i += kVerThreads) x += global_ptr(part)[i];
  return block_sum(x, sm);
}

// RESIDUAL false: Z of the drawn row, or without draft probabilities the sum of r;
// true: the sum of r, of a sequence that refused.  (One slice to a workgroup: with two or
// four, 64 x 152064 took as long or longer.)
// DECIDE: with step 2 before it, in every workgroup.
template <typename T, bool PROBS, bool RESIDUAL, bool DECIDE>
__global__ __launch_bounds__(kVerThreads) void verify_sums_kernel(VerifyParams p) {
  __shared__ double sm_s[kVerWaves];
  const int slice = blockIdx.x % p.sum_slices, b = blockIdx.x / p.sum_slices;
  VerifyRow o;
  if constexpr (DECIDE) {
    __shared__ DecideShared<kVerWaves> sm;
    o = decide<T, PROBS, kVerWaves>(p, b, sm, slice == 0);
    if (slice == 0 && threadIdx.x == 0) p.rows[b] = o;
  } else {
    o = p.rows[b];
  }
  if (o.row < 0 || (RESIDUAL && !o.refused)) return;
  const double z =
      RESIDUAL ? slices_sum(p.sums + static_cast<int64_t>(b) * p.sum_slices, p.sum_slices, sm_s) : 0.0;
  double r[8], x = 0.0;
  const int g = slice * kVerThreads + threadIdx.x, end = (slice + 1) * kVerSumSlice;
  drawn8<T, PROBS>(p, o, b, !RESIDUAL && p.draft_probs != nullptr, g, end, z, r);
#pragma unroll
  for (int k = 0; k < 8; ++k) x += r[k];
  x = block_sum(x, sm_s);
  if (threadIdx.x == 0)
    (RESIDUAL ? p.residuals : p.sums)[static_cast<int64_t>(b) * p.sum_slices + slice] = x;
}

// Prefix sums (inclusive) over the workgroup's threads.
__device__ __forceinline__ double block_prefix(double x, double* sm) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  x = wave_prefix64(x);
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
__device__ __forceinline__ int first_past(double own, double upto, double want, int (*sm)[2]) {
  const uint64_t some = __builtin_amdgcn_ballot_w64(own > 0.0);
  const uint64_t past = __builtin_amdgcn_ballot_w64(own > 0.0 && upto > want);
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) {
    sm[wave][0] = past ? 64 * wave + __builtin_ctzll(past) : -1;
    sm[wave][1] = some ? 64 * wave + 63 - __builtin_clzll(some) : -1;
  }
  __syncthreads();
  int first = -1, last = -1;
#pragma unroll
  for (int w = kVerWaves - 1; w >= 0; --w) {
    first = sm[w][0] >= 0 ? sm[w][0] : first;
    last = last < 0 ? sm[w][1] : last;
  }
  return first >= 0 ? first : last;
}

// The first of 8 entries at which the running sum passes `want`, else the last above 0.
__device__ __forceinline__ int first_of8(const double (&r)[8], double run, double want) {
  int at = 0;
  bool past = false;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    if (!past && r[k] > 0.0) at = k;
    run += r[k];
    past |= r[k] > 0.0 && run > want;
  }
  return at;
}
__device__ __forceinline__ void put_token(const VerifyParams& p, const VerifyRow& o, int b, int token) {
  const int64_t to = static_cast<int64_t>(b) * p.max_tokens + o.taken;
  if (p.tokens_wide)
    reinterpret_cast<int64_t*>(p.out)[to] = token;
  else
    reinterpret_cast<int32_t*>(p.out)[to] = token;
}

// Steps 2 to 5 in one workgroup of 16 waves to a sequence, for vocabularies up to
// kVerSmall: 8192 entries at a time, the sums of every wave's 512 kept, of which the one
// with the token is gone over again by its wave.
template <typename T, bool PROBS>
__global__ __launch_bounds__(1024) void verify_finish_kernel(VerifyParams p) {
  constexpr int W = 16, kAt = 64 * W * 8, kIts = kVerSmall / kAt;
  __shared__ DecideShared<W> sm;
  __shared__ double sm_seg[kIts * W];
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const double u = global_ptr(p.uniform)[b * p.uniform_stride + p.max_tokens - 1];
  const VerifyRow o = decide<T, PROBS, W>(p, b, sm);
  if (o.row < 0) return;
  const int its = (p.vocab + kAt - 1) / kAt;
  const bool residual = o.refused && p.draft_probs != nullptr;
  auto added = [&](const double (&r)[8]) __attribute__((always_inline)) {
    return ((r[0] + r[1]) + (r[2] + r[3])) + ((r[4] + r[5]) + (r[6] + r[7]));
  };
  // f(it, sum of this thread's entries) over the row
  auto over = [&](bool weights, double z, auto f) __attribute__((always_inline)) {
#pragma unroll 1
    for (int it = 0; it < its; ++it) {
      double r[8];
      drawn8<T, PROBS>(p, o, b, weights, it * 64 * W + tid, (it + 1) * kAt, z, r);
      f(it, added(r));
    }
  };
  double z = 0.0;
  if (residual) {
    over(true, 0.0, [&](int, double x) __attribute__((always_inline)) { z += x; });
    z = block_sum<W>(z, sm.sums);
  }
  bool weights = !o.refused;
  double total = 0.0;
  for (int again = 0; again < 2; ++again) {
    over(weights, z, [&](int it, double x) __attribute__((always_inline)) {
      x = wave_sum(x);
      if (lane == 0) sm_seg[it * W + wave] = x;
    });
    __syncthreads();
    total = 0.0;
    for (int i = lane; i < its * W; i += 64) total += sm_seg[i];
    total = wave_sum(total);
    if (total > 0.0 || !o.refused || again) break;
    // nothing is left of w where q is not below it: drawn from w (and without draft
    // probabilities there is the draft alone)
    if (!residual) {
      if (tid == 0) put_token(p, o, b, o.draft);
      return;
    }
    weights = true;
    __syncthreads();  // (every wave has read the sums)
  }
  // the wave's 512 entries in which the running sum passes `want`, in every wave alike;
  // where rounding leaves none, the last with a sum
  const double want = u * total;
  int seg = -1, last = -1;
  double before = 0.0, before_last = 0.0, run = 0.0;
  for (int i0 = 0; i0 < its * W && seg < 0; i0 += 64) {
    const double own = i0 + lane < its * W ? sm_seg[i0 + lane] : 0.0;
    const double upto = run + wave_prefix64(own);
    double ahead = __shfl_up(upto, 1);  // (by all lanes: one that is off gives nothing)
    ahead = lane > 0 ? ahead : run;
    const uint64_t some = __builtin_amdgcn_ballot_w64(own > 0.0);
    const uint64_t past = __builtin_amdgcn_ballot_w64(own > 0.0 && upto > want);
    if (past) {
      const int l = __builtin_ctzll(past);
      seg = i0 + l;
      before = __shfl(ahead, l);
    } else if (some) {
      const int l = 63 - __builtin_clzll(some);
      last = i0 + l;
      before_last = __shfl(ahead, l);
    }
    run = last_lane(upto);
  }
  if (seg < 0) {
    seg = last;
    before = before_last;
  }
  if (seg < 0 || wave != seg % W) return;
  double r[8];
  drawn8<T, PROBS>(p, o, b, weights, seg / W * 64 * W + tid, (seg / W + 1) * kAt, z, r);
  const double own = added(r), upto = before + wave_prefix64(own);
  const double ahead = __shfl_up(upto, 1);
  const uint64_t some = __builtin_amdgcn_ballot_w64(own > 0.0);
  const uint64_t past = __builtin_amdgcn_ballot_w64(own > 0.0 && upto > want);
  const int who = past ? __builtin_ctzll(past) : 63 - __builtin_clzll(some);
  if (lane == who)
    put_token(p, o, b, seg / W * kAt + 8 * tid + first_of8(r, lane > 0 ? ahead : before, want));
}

template <typename T, bool PROBS>
__global__ __launch_bounds__(kVerThreads) void verify_pick_kernel(VerifyParams p) {
  __shared__ double sm_s[kVerWaves], sm_c[kVerThreads + 1];
  __shared__ int sm_f[kVerWaves][2], sm_g[kVerWaves][2];
  const int b = blockIdx.x, tid = threadIdx.x, n = p.sum_slices;
  const double u = global_ptr(p.uniform)[b * p.uniform_stride + p.max_tokens - 1];
  const VerifyRow o = p.rows[b];
  if (o.row < 0) return;
  const double* const sums = p.sums + static_cast<int64_t>(b) * n;
  const bool residual = o.refused && p.draft_probs != nullptr;
  const double* part = residual ? p.residuals + static_cast<int64_t>(b) * n : sums;
  bool weights = !o.refused;
  // every thread adds up some slices in a row
  const int per = (n + kVerThreads - 1) / kVerThreads, i0 = tid * per;
  auto owns = [&](const double* of) __attribute__((always_inline)) {
    double x = 0.0;
    for (int i = i0; i < i0 + per && i < n; ++i) x += global_ptr(of)[i];
    return x;
  };
  double own = owns(part);
  const double z = residual ? slices_sum(sums, n, sm_s) : 0.0;
  double upto = block_prefix(own, sm_s);
  sm_c[tid + 1] = upto;
  if (tid == 0) sm_c[0] = 0.0;
  __syncthreads();
  double total = sm_c[kVerThreads];
  if (o.refused && !(total > 0.0)) {  // w is nowhere above q Z: drawn from w
    if (!residual) {                  // (which is the draft alone)
      if (tid == 0) put_token(p, o, b, o.draft);
      return;
    }
    weights = true;
    part = sums;
    own = owns(part);
    upto = block_prefix(own, sm_s);
    __syncthreads();
    sm_c[tid + 1] = upto;
    __syncthreads();
    total = sm_c[kVerThreads];
  }
  const double want = u * total;
  int who = first_past(own, upto, want, sm_f);
  if (who < 0) return;  // (no thread has a sum: not where `total` is above 0)
  int slice = who;
  double before = sm_c[who];
  if (per > 1) {  // which of its slices
    double run = before;
    for (int i = who * per; i < (who + 1) * per && i < n; ++i) {
      const double x = global_ptr(part)[i];
      if (x > 0.0) {
        slice = i;
        before = run;
        if (run + x > want) break;
      }
      run += x;
    }
  }
  // the token in it
  double r[8];
  const int g = slice * kVerThreads + tid, end = (slice + 1) * kVerSumSlice;
  drawn8<T, PROBS>(p, o, b, weights, g, end, z, r);
  own = 0.0;
#pragma unroll
  for (int k = 0; k < 8; ++k) own += r[k];
  upto = before + block_prefix(own, sm_s);
  __syncthreads();
  sm_c[tid + 1] = upto;
  if (tid == 0) sm_c[0] = before;
  who = first_past(own, upto, want, sm_g);
  if (tid == who)
    put_token(p, o, b, kVerSumSlice * slice + 8 * tid + first_of8(r, sm_c[who], want));
}

template <typename T, bool PROBS>
static hipError_t launch_verify_t(const VerifyParams& p, hipStream_t st) {
  const dim3 t(kVerThreads), seqs(static_cast<unsigned>(p.num_seqs));
  hipLaunchKernelGGL((verify_stats_kernel<T, PROBS>),
                     dim3(static_cast<unsigned>(p.num_seqs * p.max_tokens * p.stat_slices)), t, 0,
                     st, p);
  // Steps 2 to 5 at once where one workgroup goes over the vocabulary as soon as four launches
  // do: one round of 8192 logits (1 x 4000 16 us for 19, 128 x 8192 16 for 20; but 1 x
  // 12000 20 for 18, 64 x 50257 48 for 34, their exponentials), four of probabilities (1 x
  // 32000 15.0 for 15.3, 64 x 24000 19 for 23), eight of them for many sequences (64 x 65000
  // 34.4 for 34.5, 128 x 50257 40 for 46, but 16 x 50257 21 for 18).
  if (p.vocab <= (PROBS ? p.num_seqs >= 64 ? kVerSmall : kVerSmall / 2 : kVerSmall / 8)) {
    hipLaunchKernelGGL((verify_finish_kernel<T, PROBS>), seqs, dim3(1024), 0, st, p);
    return hipGetLastError();
  }
  const int64_t n = static_cast<int64_t>(p.num_seqs) * p.sum_slices;
  const dim3 slices(static_cast<unsigned>(n));
  // Few slices: step 2 in every workgroup of step 3, a launch less, of which all are on
  // the chip at once (1200 slices of logits 27 us for 28, 2048 39.7 for 37.6; 2048 of
  // probabilities 32 for 35, 3200 47 for 46).
  if (n <= (PROBS ? 2048 : 1536)) {
    hipLaunchKernelGGL((verify_sums_kernel<T, PROBS, false, true>), slices, t, 0, st, p);
  } else {
    hipLaunchKernelGGL((verify_decide_kernel<T, PROBS>), seqs, dim3(1024), 0, st, p);
    hipLaunchKernelGGL((verify_sums_kernel<T, PROBS, false, false>), slices, t, 0, st, p);
  }
  if (p.draft_probs != nullptr)
    hipLaunchKernelGGL((verify_sums_kernel<T, PROBS, true, false>), slices, t, 0, st, p);
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
