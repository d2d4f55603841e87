// Block tables, slots and positions of a step, from the requests' lengths.
//
//   held_r = ceil(ctx_r / B), need_r = ceil((ctx_r + new_r) / B)
//   table[r][held_r .. need_r) = free[f_r ..), f_r the sum of need - held before r
//   start_r = the sum of new before r; token t of request r: pos = ctx_r + t - start_r,
//   slot = table[r][pos / B] * B + pos % B
//
// Bound by latency: a few kilobytes, one launch.  Every workgroup sums the
// requests' lengths by itself (up to 4096 of them, 16 to a thread, the sums in
// LDS) and takes its share of the tokens and of the new table entries, each of
// which finds its request by bisection; a token in a new block takes its id from
// the free list, not from the table that another workgroup may still be writing.
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

// The lengths of request r: 0 .. 2^30 each, whatever stands there.
__device__ __forceinline__ uint32_t length_at(const void* a, bool wide, int64_t stride, int r) {
  const int64_t x = wide ? reinterpret_cast<const int64_t*>(a)[r * stride]
                         : reinterpret_cast<const int32_t*>(a)[r * stride];
  constexpr int64_t kMost = int64_t{1} << 30;
  return static_cast<uint32_t>(x < 0 ? 0 : x < kMost ? x : kMost);
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

__global__ __launch_bounds__(kTabThreads) void step_tables_kernel(StepTablesParams p) {
  constexpr int EPT = kStepMaxSeqs / kTabThreads, W = kTabThreads / 64;
  __shared__ uint32_t sm_tok[kStepMaxSeqs + 1], sm_blk[kStepMaxSeqs + 1];
  __shared__ uint32_t sm_w[2][W];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int n = p.num_seqs;
  const int each = (n + kTabThreads - 1) / kTabThreads;  // requests of a thread, at most EPT
  auto blocks = [&](uint32_t tokens) __attribute__((always_inline)) {
    const uint32_t b = (tokens + (1u << p.bs_shift) - 1) >> p.bs_shift;
    return b < static_cast<uint32_t>(p.width) ? b : static_cast<uint32_t>(p.width);
  };
  uint32_t ts = 0, bsum = 0;
  for (int j = 0; j < each; ++j) {
    const int r = tid * each + j;
    if (r >= n) break;
    const uint32_t c = length_at(p.ctx, p.ctx_wide, p.ctx_stride, r);
    const uint32_t m = length_at(p.fresh, p.fresh_wide, p.fresh_stride, r);
    ts = add_sat(ts, m);
    bsum = add_sat(bsum, blocks(c + m) - blocks(c));
    sm_tok[r + 1] = ts;  // sums within the thread, so far
    sm_blk[r + 1] = bsum;
    if (blockIdx.x == 0) p.seq_lens[r] = static_cast<int32_t>(c + m < 0x7fffffffu ? c + m : 0x7fffffffu);
  }
  const uint32_t ti = wave_prefix_sat(ts), bi = wave_prefix_sat(bsum);
  if (lane == 63) {
    sm_w[0][wave] = ti;
    sm_w[1][wave] = bi;
  }
  __syncthreads();
  uint32_t tb = 0, bb = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    if (w < wave) {
      tb = add_sat(tb, sm_w[0][w]);
      bb = add_sat(bb, sm_w[1][w]);
    }
  }
  // what comes before this thread's requests: the lane before it has the rest
  const uint32_t tl = __shfl_up(ti, 1), bl = __shfl_up(bi, 1);
  if (lane > 0) {
    tb = add_sat(tb, tl);
    bb = add_sat(bb, bl);
  }
  if (tid == 0) sm_tok[0] = sm_blk[0] = 0;
  for (int j = 0; j < each; ++j) {
    const int r = tid * each + j;
    if (r >= n) break;
    sm_tok[r + 1] = add_sat(sm_tok[r + 1], tb);
    sm_blk[r + 1] = add_sat(sm_blk[r + 1], bb);
  }
  __syncthreads();
  const uint32_t tokens = sm_tok[n], fresh = sm_blk[n];
  if (blockIdx.x == 0) {
    for (int r = tid; r <= n; r += kTabThreads)
      p.starts[r] = static_cast<int32_t>(sm_tok[r] < 0x7fffffffu ? sm_tok[r] : 0x7fffffffu);
    if (tid == 0) *p.used = static_cast<int32_t>(fresh < 0x7fffffffu ? fresh : 0x7fffffffu);
  }
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kTabThreads + tid;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kTabThreads;
  for (int64_t i = first; i < fresh; i += step) {
    const int r = find(sm_blk, n, static_cast<uint32_t>(i));
    const uint32_t held = blocks(length_at(p.ctx, p.ctx_wide, p.ctx_stride, r));
    p.table[r * p.table_stride + held + (i - sm_blk[r])] = i < p.num_free ? p.free[i] : -1;
  }
  for (int64_t t = first; t < p.num_tokens; t += step) {
    int64_t pos = 0, slot = -1;
    if (t < tokens) {
      const int r = find(sm_tok, n, static_cast<uint32_t>(t));
      const uint32_t c = length_at(p.ctx, p.ctx_wide, p.ctx_stride, r);
      pos = c + (t - sm_tok[r]);
      const int64_t b = pos >> p.bs_shift;
      if (b < p.width) {
        const uint32_t held = blocks(c);
        int64_t id;
        if (b < held) {
          id = p.table[r * p.table_stride + b];
        } else {
          const int64_t f = sm_blk[r] + (b - held);
          id = f < p.num_free ? p.free[f] : -1;
        }
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
  hipLaunchKernelGGL(step_tables_kernel, dim3(static_cast<unsigned>(grid)), dim3(kTabThreads), 0,
                     st, p);
  return hipGetLastError();
}

}  // namespace hcp
