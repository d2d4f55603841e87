// Block tables, slots and positions of a step, from the requests' lengths.
//
//   held_r = ceil(ctx_r / B), need_r = ceil((ctx_r + new_r) / B)
//   table[r][held_r .. need_r) = free[f_r ..), f_r the sum of need - held before r
//   start_r = the sum of new before r; token t of request r: pos = ctx_r + t - start_r,
//   slot = table[r][pos / B] * B + pos % B
//
// Bound by latency: a few kilobytes, one launch.  Every workgroup sums the
// requests' lengths by itself (up to 4096 of them, 1, 4 or 16 to a thread, all
// loaded at once; sums and cached lengths in LDS) and takes its share of the tokens
// and of the new table entries, each of which finds its request by bisection; a
// token in a new block takes its id from the free list, not from the table that
// another workgroup may still be writing.  64 / 1000 / 4000 requests 3.3 / 5.6 / 11.7
// us (with the lengths loaded one after the other 0.4, 1.3 and 4.8 us more).
#include "decode_share.h"
#include "params.h"

namespace hcp {

// Sums stop at 2^32 - 1 (added in any order they then still agree): no token or
// block that far out is listed.
__device__ __forceinline__ uint32_t add_sat(uint32_t a, uint32_t b) {
  return __builtin_elementwise_add_sat(a, b);
}
__device__ __forceinline__ uint32_t wave_prefix_sat(uint32_t x) {
  x = add_sat(x, __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false));  // row_shr:1
  x = add_sat(x, __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false));
  x = add_sat(x, __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false));
  x = add_sat(x, __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false));
  x = add_sat(x, __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false));  // row_bcast:15
  x = add_sat(x, __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false));  // row_bcast:31
  return x;
}

// Lengths r, r + 1, .., 0 .. 2^30 each whatever stands there, those past n 0: all
// loads on their way at once.
template <int N>
__device__ __forceinline__ void lengths(const void* a, bool wide, int64_t stride, int r, int n,
                                        uint32_t (&x)[N]) {
  int64_t y[N];
  if (wide) {
#pragma unroll
    for (int j = 0; j < N; ++j)
      y[j] = reinterpret_cast<const int64_t*>(a)[(r + j < n ? r + j : 0) * stride];
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j)
      y[j] = reinterpret_cast<const int32_t*>(a)[(r + j < n ? r + j : 0) * stride];
  }
  constexpr int64_t kMost = int64_t{1} << 30;
#pragma unroll
  for (int j = 0; j < N; ++j)
    x[j] = r + j >= n || y[j] < 0 ? 0 : static_cast<uint32_t>(y[j] < kMost ? y[j] : kMost);
}

// Largest r with sum[r] <= x (sum[0] = 0, not decreasing; x < sum[n]).
__device__ __forceinline__ int find(const uint32_t* sum, int n, uint32_t x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (sum[mid] <= x)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

constexpr int kTabThreads = 256;
constexpr uint32_t kMax32 = 0x7fffffff;

// EPT: requests of a thread, at most.
template <int EPT>
__global__ __launch_bounds__(kTabThreads) void step_tables_kernel(StepTablesParams p) {
  constexpr int W = kTabThreads / 64, N = EPT * kTabThreads;
  __shared__ uint32_t sm_tok[N + 1], sm_blk[N + 1], sm_ctx[N];
  __shared__ uint32_t sm_w[2][W];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int n = p.num_seqs;
  auto blocks = [&](uint32_t tokens) __attribute__((always_inline)) {
    const uint32_t b = (tokens + (1u << p.bs_shift) - 1) >> p.bs_shift;
    return b < static_cast<uint32_t>(p.width) ? b : static_cast<uint32_t>(p.width);
  };
  uint32_t ts = 0, bsum = 0, tok[EPT], blk[EPT];  // sums within the thread, so far
  const int r0 = tid * EPT;
  if (n > 0) {
    uint32_t c[EPT], m[EPT];
    lengths(p.ctx, p.ctx_wide, p.ctx_stride, r0, n, c);
    lengths(p.fresh, p.fresh_wide, p.fresh_stride, r0, n, m);
#pragma unroll
    for (int j = 0; j < EPT; ++j) {
      tok[j] = ts = add_sat(ts, m[j]);
      blk[j] = bsum = add_sat(bsum, blocks(c[j] + m[j]) - blocks(c[j]));
      sm_ctx[r0 + j] = c[j];
      if (blockIdx.x == 0 && r0 + j < n)
        p.seq_lens[r0 + j] = static_cast<int32_t>(c[j] + m[j] < kMax32 ? c[j] + m[j] : kMax32);
    }
  }
  const uint32_t ti = wave_prefix_sat(ts), bi = wave_prefix_sat(bsum);
  if (lane == 63) {
    sm_w[0][wave] = ti;
    sm_w[1][wave] = bi;
  }
  __syncthreads();
  // what comes before this thread's requests: the lane before it has the rest
  const uint32_t tl = __shfl_up(ti, 1), bl = __shfl_up(bi, 1);
  uint32_t tb = lane > 0 ? tl : 0, bb = lane > 0 ? bl : 0;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    if (w < wave) {
      tb = add_sat(tb, sm_w[0][w]);
      bb = add_sat(bb, sm_w[1][w]);
    }
  }
  if (tid == 0) sm_tok[0] = sm_blk[0] = 0;
  if (n > 0) {
#pragma unroll
    for (int j = 0; j < EPT; ++j) {
      sm_tok[r0 + j + 1] = add_sat(tok[j], tb);
      sm_blk[r0 + j + 1] = add_sat(blk[j], bb);
    }
  }
  __syncthreads();
  const uint32_t tokens = sm_tok[n], fresh = sm_blk[n];
  if (blockIdx.x == 0) {
    for (int r = tid; r <= n; r += kTabThreads)
      p.starts[r] = static_cast<int32_t>(sm_tok[r] < kMax32 ? sm_tok[r] : kMax32);
    if (tid == 0) *p.used = static_cast<int32_t>(fresh < kMax32 ? fresh : kMax32);
  }
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kTabThreads + tid;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kTabThreads;
  for (int64_t i = first; i < fresh; i += step) {
    const int r = find(sm_blk, n, static_cast<uint32_t>(i));
    p.table[r * p.table_stride + blocks(sm_ctx[r]) + (i - sm_blk[r])] =
        i < p.num_free ? p.free[i] : -1;
  }
  for (int64_t t = first; t < p.num_tokens; t += step) {
    int64_t pos = 0, slot = -1;
    if (t < tokens) {
      const int r = find(sm_tok, n, static_cast<uint32_t>(t));
      const uint32_t c = sm_ctx[r];
      pos = c + (t - sm_tok[r]);
      const int64_t b = pos >> p.bs_shift;
      if (b < p.width) {
        const int64_t f = sm_blk[r] + (b - blocks(c));
        // (one load, from the table or from the free list)
        const int32_t* at = b < blocks(c) ? p.table + r * p.table_stride + b
                            : f < p.num_free ? p.free + f : nullptr;
        const int64_t id = at != nullptr ? *at : -1;
        if (id >= 0) slot = (id << p.bs_shift) + (pos & ((1 << p.bs_shift) - 1));
      }
    }
    p.positions[t] = pos;
    p.slots[t] = slot;
  }
}

hipError_t launch_step_tables(const StepTablesParams& p, hipStream_t st) {
  // a token a thread; new table entries go over the same threads
  int64_t grid = (p.num_tokens + kTabThreads - 1) / kTabThreads;
  grid = grid < 1 ? 1 : grid < 1024 ? grid : 1024;
  const dim3 g(static_cast<unsigned>(grid)), b(kTabThreads);
  if (p.num_seqs <= kTabThreads)
    hipLaunchKernelGGL(step_tables_kernel<1>, g, b, 0, st, p);
  else if (p.num_seqs <= 4 * kTabThreads)
    hipLaunchKernelGGL(step_tables_kernel<4>, g, b, 0, st, p);
  else
    hipLaunchKernelGGL(step_tables_kernel<kStepMaxSeqs / kTabThreads>, g, b, 0, st, p);
  return hipGetLastError();
}

}  // namespace hcp
