// Norm of every query and key head, rotation by position and the write into the
// paged cache in one pass over q, k and v.
//
//   y = x / sqrt(mean(x^2) + eps) * w        (a head's row of d columns; w optional)
//   (y_i, y_j) -> (y_i c - y_j s, y_j c + y_i s)   for the pairs (i, i + rot / 2), or
//                                            (2 i, 2 i + 1), of the first rot columns,
//                                            c, s = table[pos][i], table[pos][rot / 2 + i]
//
// rounded from 32 bits to 16.  A key on its way into the 4-bit cache is computed in
// 64 bits up to there: next to a border between two codes a difference in the last place is a
// whole step of the code, and so the cache does not depend on the order in which
// something is summed.
//
// HBM-bound: 4 d bytes for a query row, 4 d (16-bit cache) or 2 d + 17 d / 32 for a
// key or value row; 8192 tokens of 28 / 4 x 128 (155 MB) 32.2 us, 4.8 TB/s, where a
// large copy runs at 4.9; 4096 of 64 / 8 x 128 into the 4-bit cache (157 MB) 34.3 us;
// one token 3.6 us.  Few KV heads leave their job's rows empty: 5003 tokens of 14 / 2 x
// 64 without a cache, a wave's 16 rows taken by 14 query heads and then by 2 of keys, 7.8
// us where their 21 MB would copy in 4.3.  A lane holds 16 columns of a row, the
// eight of a pair's first sides and the eight of their second sides, so that nothing
// is exchanged but the sum of squares, over the 8 lanes of a row at d = 128; it keeps
// its 8 cosines and sines for all heads of its token (read again for every head they
// would be twice the row's own bytes).
#include "params.h"

namespace hcp {

// Eight values of a 16-bit or 32-bit array.
template <typename T>
__device__ __forceinline__ void load8(const void* p, int64_t at, bool wide, float (&x)[8]) {
  if (wide) {
    const char* a = reinterpret_cast<const char*>(p) + at * 4;
    const u32x4 lo = ldg16(a), hi = ldg16(a + 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = __uint_as_float(lo[i]);
      x[4 + i] = __uint_as_float(hi[i]);
    }
  } else {
    const u32x4 v = ldg16(reinterpret_cast<const char*>(p) + at * 2);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = Elem<T>::to_float(static_cast<uint16_t>(v[i]));
      x[2 * i + 1] = Elem<T>::to_float(static_cast<uint16_t>(v[i] >> 16));
    }
  }
}

__device__ __forceinline__ float inv_sqrt(float x) { return 1.f / __builtin_sqrtf(x); }
__device__ __forceinline__ double inv_sqrt(double x) { return 1.0 / __builtin_sqrt(x); }

// What a lane knows of its part of a row and of its token.
struct RopeLane {
  int ca, cb;        // its two chunks of eight columns
  bool has_a, has_b; // chunks inside the row
  bool turned;       // rotated columns
  float cs[8], sn[8];
};

// One row's part (chunks a and b, packed) normed with weight w and rotated.
template <typename T>
__device__ __forceinline__ void rope_row(const RopeParams& p, const RopeLane& l, bool norm,
                                         const float (&wa)[8], const float (&wb)[8], int lanes,
                                         u32x4& a, u32x4& b) {
  float x[8], y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] = Elem<T>::to_float(static_cast<uint16_t>(a[i >> 1] >> (16 * (i & 1))));
    y[i] = Elem<T>::to_float(static_cast<uint16_t>(b[i >> 1] >> (16 * (i & 1))));
  }
  if (norm) {
    float sq = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) sq += x[i] * x[i] + y[i] * y[i];
    for (int m = 1; m < lanes; m *= 2) sq += __shfl_xor(sq, m);
    const float inv = inv_sqrt(sq / p.d + static_cast<float>(p.eps));
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[i] *= inv * wa[i];
      y[i] *= inv * wb[i];
    }
  }
  if (l.turned) {
    if (p.interleaved) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float u = x[2 * i], v = x[2 * i + 1], c0 = l.cs[i], s0 = l.sn[i];
        x[2 * i] = u * c0 - v * s0;
        x[2 * i + 1] = v * c0 + u * s0;
        const float q = y[2 * i], r = y[2 * i + 1], c1 = l.cs[4 + i], s1 = l.sn[4 + i];
        y[2 * i] = q * c1 - r * s1;
        y[2 * i + 1] = r * c1 + q * s1;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float u = x[i], v = y[i], c0 = l.cs[i], s0 = l.sn[i];
        x[i] = u * c0 - v * s0;
        y[i] = v * c0 + u * s0;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    a[i] = pack2<T>(x[2 * i], x[2 * i + 1]);
    b[i] = pack2<T>(y[2 * i], y[2 * i + 1]);
  }
}

// The same in 64 bits, four columns at a time, each widened where it is used: all
// sixteen at once, with weights and angles held widened across the wave's rows,
// take 167 registers where these take 126, and leave three waves on a SIMD (4096
// tokens at 64 / 8 heads x 128: 52 us with the read back, then 42).
template <typename T>
__device__ __forceinline__ void rope_row_wide(const RopeParams& p, const RopeLane& l, bool norm,
                                              const float (&wa)[8], const float (&wb)[8],
                                              int lanes, u32x4& a, u32x4& b) {
  auto wide = [](float x) __attribute__((always_inline)) {
    asm volatile("" : "+v"(x));
    return static_cast<double>(x);
  };
  auto lo = [](uint32_t x) __attribute__((always_inline)) {
    return static_cast<double>(Elem<T>::to_float(static_cast<uint16_t>(x)));
  };
  auto hi = [](uint32_t x) __attribute__((always_inline)) {
    return static_cast<double>(Elem<T>::to_float(static_cast<uint16_t>(x >> 16)));
  };
  auto turn = [](double& u, double& v, double c, double s) __attribute__((always_inline)) {
    const double w = u * c - v * s;
    v = v * c + u * s;
    u = w;
  };
  double inv = 1;
  if (norm) {
    double sq = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      sq += lo(a[i]) * lo(a[i]) + hi(a[i]) * hi(a[i]);
      sq += lo(b[i]) * lo(b[i]) + hi(b[i]) * hi(b[i]);
    }
    for (int m = 1; m < lanes; m *= 2) sq += __shfl_xor(sq, m);
    inv = inv_sqrt(sq / p.d + p.eps);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    double x0 = lo(a[i]), x1 = hi(a[i]), y0 = lo(b[i]), y1 = hi(b[i]);
    if (norm) {
      x0 *= inv * wide(wa[2 * i]);
      x1 *= inv * wide(wa[2 * i + 1]);
      y0 *= inv * wide(wb[2 * i]);
      y1 *= inv * wide(wb[2 * i + 1]);
    }
    if (l.turned) {
      if (p.interleaved) {
        turn(x0, x1, wide(l.cs[i]), wide(l.sn[i]));
        turn(y0, y1, wide(l.cs[4 + i]), wide(l.sn[4 + i]));
      } else {
        turn(x0, y0, wide(l.cs[2 * i]), wide(l.sn[2 * i]));
        turn(x1, y1, wide(l.cs[2 * i + 1]), wide(l.sn[2 * i + 1]));
      }
    }
    a[i] = pack2<T>(static_cast<float>(x0), static_cast<float>(x1));
    b[i] = pack2<T>(static_cast<float>(y0), static_cast<float>(y1));
    __builtin_amdgcn_sched_barrier(0);
  }
}

// A wave takes every wpt-th job of a token; a job is as many query heads as the
// wave has rows, or as many key and value rows.
template <typename T, int CACHE>
__global__ __launch_bounds__(256) void qk_rope_kernel(RopeParams p) {
  __shared__ u32x4 sm_rows[CACHE == kRopeCacheFp4 ? 4 : 1][CACHE == kRopeCacheFp4 ? 128 : 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t w = static_cast<int64_t>(blockIdx.x) * 4 + wave;
  const int64_t t = w / p.wpt;
  if (t >= p.num_tokens) return;
  const int lpr = 1 << p.lpr_shift, rows = 64 >> p.lpr_shift;
  const int u = lane & (lpr - 1), row = lane >> p.lpr_shift;
  const int chunks = p.d / 8;
  RopeLane l;
  {
    const int half = p.rot / 16;  // chunks of a pair's first sides
    const bool pairs = !p.interleaved && u < half;
    l.ca = pairs ? u : 2 * u;
    l.cb = pairs ? u + half : 2 * u + 1;
    l.has_a = l.ca < chunks;
    l.has_b = l.cb < chunks;
    l.turned = u < half;
    if (l.turned) {
      int64_t pos = p.pos_wide ? reinterpret_cast<const int64_t*>(p.pos)[t]
                               : reinterpret_cast<const int32_t*>(p.pos)[t];
      pos = pos < 0 ? 0 : pos < p.max_pos ? pos : p.max_pos - 1;
      const int64_t at = pos * p.table_stride + 8 * u;
      load8<T>(p.table, at, p.table_wide, l.cs);
      load8<T>(p.table, at + p.rot / 2, p.table_wide, l.sn);
    }
  }
  const u32x4 zero = {0, 0, 0, 0};
  float wa[8], wb[8];
  auto weights = [&](const void* wt) __attribute__((always_inline)) {
    if (wt == nullptr) return;
    if (l.has_a) load8<T>(wt, 8 * l.ca, p.w_wide, wa);
    if (l.has_b) load8<T>(wt, 8 * l.cb, p.w_wide, wb);
  };
  auto fetch = [&](const char* src, u32x4& a, u32x4& b) __attribute__((always_inline)) {
    a = l.has_a ? ldg16(src + 16 * l.ca) : zero;
    b = l.has_b ? ldg16(src + 16 * l.cb) : zero;
  };
  auto put = [&](char* dst, const u32x4& a, const u32x4& b) __attribute__((always_inline)) {
    if (l.has_a) *reinterpret_cast<u32x4*>(dst + 16 * l.ca) = a;
    if (l.has_b) *reinterpret_cast<u32x4*>(dst + 16 * l.cb) = b;
  };

  int j = static_cast<int>(w - t * p.wpt);
  const int qjobs = (p.num_heads + rows - 1) / rows;
  if (j < qjobs) {
    weights(p.q_weight);
    for (; j < qjobs; j += p.wpt) {
      const int h = j * rows + row;
      const bool in = h < p.num_heads;
      u32x4 a = zero, b = zero;
      if (in)
        fetch(reinterpret_cast<const char*>(p.q) +
                  (t * p.q_stride_tok + h * p.q_stride_head) * 2, a, b);
      rope_row<T>(p, l, p.q_weight != nullptr, wa, wb, lpr, a, b);
      if (in)
        put(reinterpret_cast<char*>(p.q_out) +
                (t * p.qo_stride_tok + h * p.qo_stride_head) * 2, a, b);
    }
  }
  j -= qjobs;
  int64_t slot = -1;
  if (CACHE != kRopeNoCache && t < p.num_cached)
    slot = p.slots_wide ? reinterpret_cast<const int64_t*>(p.slots)[t]
                        : reinterpret_cast<const int32_t*>(p.slots)[t];
  const bool write = slot >= 0 && slot < p.num_slots;
  const int kvrows = CACHE == kRopeNoCache ? p.num_kv_heads : 2 * p.num_kv_heads;
  const int kvjobs = (kvrows + rows - 1) / rows;
  if (j >= kvjobs) return;
  weights(p.k_weight);
  for (; j < kvjobs; j += p.wpt) {
    const int i = j * rows + row;
    const bool is_v = i >= p.num_kv_heads;
    const int h = is_v ? i - p.num_kv_heads : i;
    const bool in = i < kvrows;
    u32x4 a = zero, b = zero;
    if (in)
      fetch(is_v ? reinterpret_cast<const char*>(p.v) +
                       (t * p.v_stride_tok + h * p.v_stride_head) * 2
                 : reinterpret_cast<const char*>(p.k) +
                       (t * p.k_stride_tok + h * p.k_stride_head) * 2, a, b);
    // (the 64-bit arithmetic not for a job of values alone: 42.6 -> 40.7 us there)
    if (CACHE != kRopeCacheFp4 || j * rows < p.num_kv_heads) {
      u32x4 ka = a, kb = b;
      if constexpr (CACHE == kRopeCacheFp4)
        rope_row_wide<T>(p, l, p.k_weight != nullptr, wa, wb, lpr, ka, kb);
      else
        rope_row<T>(p, l, p.k_weight != nullptr, wa, wb, lpr, ka, kb);
      if (!is_v) {
        a = ka;
        b = kb;
        if (in && p.k_out != nullptr)
          put(reinterpret_cast<char*>(p.k_out) +
                  (t * p.ko_stride_tok + h * p.ko_stride_head) * 2, a, b);
      }
    }
    if constexpr (CACHE == kRopeCache16) {
      if (in && write)
        put(reinterpret_cast<char*>(is_v ? p.v_cache : p.k_cache) +
                ((slot >> p.bs_shift) * p.stride_block + h * p.stride_head +
                 (slot & p.bs_mask) * p.stride_tok) * 2, a, b);
    } else if constexpr (CACHE == kRopeCacheFp4) {
      // through LDS into the order of the cache: four lanes the 32 columns of a
      // scale (the wave's own rows: its LDS accesses stay in order)
      u32x4* const sm = sm_rows[wave];
      if (l.has_a) sm[row * chunks + l.ca] = a;
      if (l.has_b) sm[row * chunks + l.cb] = b;
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      if (write) {
        for (int c = lane; c < rows * chunks; c += 64) {
          const int rr = c / chunks, ii = j * rows + rr;
          if (ii >= kvrows) break;
          const bool v = ii >= p.num_kv_heads;
          char* region = reinterpret_cast<char*>(p.k_cache) +
                         (slot >> p.bs_shift) * p.stride_block +
                         (v ? ii - p.num_kv_heads : ii) * p.stride_head;
          fp4_store<T>(region, Fp4Region{p.d, p.bs_mask + 1}, v,
                       static_cast<int>(slot & p.bs_mask), c - rr * chunks, sm[c]);
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
  }
}

template <typename T>
static hipError_t launch_rope_t(const RopeParams& p, int cache, hipStream_t st) {
  const dim3 g(static_cast<unsigned>((p.num_tokens * p.wpt + 3) / 4)), b(256);
  if (cache == kRopeCacheFp4)
    hipLaunchKernelGGL((qk_rope_kernel<T, kRopeCacheFp4>), g, b, 0, st, p);
  else if (cache == kRopeCache16)
    hipLaunchKernelGGL((qk_rope_kernel<T, kRopeCache16>), g, b, 0, st, p);
  else
    hipLaunchKernelGGL((qk_rope_kernel<T, kRopeNoCache>), g, b, 0, st, p);
  return hipGetLastError();
}

hipError_t launch_qk_rope(RopeParams p, int dtype, int cache, hipStream_t st) {
  p.lpr_shift = 0;
  while ((16 << p.lpr_shift) < p.d) ++p.lpr_shift;
  const int rows = 64 >> p.lpr_shift;
  const int kvrows = cache == kRopeNoCache ? p.num_kv_heads : 2 * p.num_kv_heads;
  const int jobs = (p.num_heads + rows - 1) / rows + (kvrows + rows - 1) / rows;
  // one wave for a token where tokens fill the machine, else its jobs side by side
  const int64_t want = (2048 + p.num_tokens - 1) / p.num_tokens;
  p.wpt = static_cast<int32_t>(want < jobs ? want : jobs);
  return dtype == HCP_DTYPE_BF16 ? launch_rope_t<__bf16>(p, cache, st)
                                 : launch_rope_t<_Float16>(p, cache, st);
}

}  // namespace hcp
