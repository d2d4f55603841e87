// The equal shares of a decode batch whose lengths are read on the device: shared
// by the split-KV decode kernels that run without a plan.
#pragma once

#include "params.h"

namespace hcp {

// The kernel's one argument, by a pointer the compiler cannot see through:
// its loads stay where they are used.
template <typename P>
__device__ __forceinline__ const P& fresh_params() {
  auto k = __builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(k));
  return *(const P*)k;
}

// Inclusive prefix sum over the wave's lanes, by DPP moves (inside rows of 16
// lanes, then row 0 -> 1 and 2 -> 3, then the lower half into the upper):
// an add each, where six shuffles through LDS take about 100 cycles each.
__device__ __forceinline__ int wave_prefix(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr:1
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);  // row_shr:2
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);  // row_shr:4
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);  // row_shr:8
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast:15
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast:31
  return x;
}

// Lengths (or first keys) r, r + 1, .. as the caller gives them, those past n the
// last one's: all loads on their way at once, not one after the other.
template <int N>
__device__ __forceinline__ void paged_lens(const void* lens, bool wide, int r, int n,
                                           int64_t (&x)[N]) {
  if (wide) {
#pragma unroll
    for (int j = 0; j < N; ++j)
      x[j] = global_ptr(reinterpret_cast<const int64_t*>(lens))[r + j < n ? r + j : n - 1];
  } else {
    int32_t y[N];
#pragma unroll
    for (int j = 0; j < N; ++j)
      y[j] = global_ptr(reinterpret_cast<const int32_t*>(lens))[r + j < n ? r + j : n - 1];
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = y[j];
  }
}

// Cuts the keys of all sequences, laid end to end in chunks of 32, into equal
// shares, one for each of at most p.d.num_wgs workgroups, each of at least LEAST
// chunks (twice that past a LATE-th of the workgroups); every sequence counts for
// START chunks more, what its split costs to start.  count(all, len): the chunks of
// a sequence with `all` keys in the cache, the last `len` of them seen.  A
// workgroup of NT threads gets its share in sm_cut: first sequence (-1: none) and
// first chunk of it, last sequence and the end in its chunks; sm_len / sm_all
// [kDecMaxSeqs] get the keys of every sequence (sm_all -1: HCP_LEN_NOT_RUN).
// STARTS: p.starts counts.  last(p, j, all, seen): how many of its `seen` keys the
// thread's j-th sequence looks at, the last ones; may make `all` less.  Ends with a
// barrier.
struct LastWindow {
  __device__ __forceinline__ int operator()(const PagedDecParams& p, int, int, int seen) const {
    return p.window > 0 && seen > p.window ? p.window : seen;
  }
};
template <int NT, int START, int LEAST, int LATE, bool STARTS, typename Count,
          typename Last = LastWindow>
__device__ __forceinline__ void paged_shares(const PagedDecParams& p_, int wg, int* sm_len,
                                             int* sm_all, int (*sm_w)[NT / 64], int* sm_cut,
                                             Count count, Last last = {}) {
  constexpr int EPT = kDecMaxSeqs / NT;  // sequences per thread of the prefix sum
  constexpr int W = NT / 64;
  const int n = p_.num_seqs;
  // ---- prefix sums over the sequences: chunks, sequences with keys ----
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int c[EPT], cs = 0, zs = 0;
  int64_t lens[EPT], from[EPT];
  paged_lens(p_.lens, p_.lens_wide, tid * EPT, n, lens);
  if constexpr (STARTS) {
    if (p_.starts != nullptr) paged_lens(p_.starts, p_.lens_wide, tid * EPT, n, from);
  }
#pragma unroll
  for (int j = 0; j < EPT; ++j) {
    const int r = tid * EPT + j;
    const int64_t given = r < n ? lens[j] : 0;
    int all =  // keys that the sequence's query sees; max_len < 2^31
        static_cast<int>(given < 0 ? 0 : given < p_.max_len ? given : p_.max_len);
    int seen = all;
    if constexpr (STARTS) {
      if (p_.starts != nullptr && r < n) {
        const int64_t s = from[j];
        seen = s <= 0 ? all : s < all ? all - static_cast<int>(s) : 0;
      }
    }
    const int len = last(p_, j, all, seen);
    if (r < n) {
      sm_all[r] = given == HCP_LEN_NOT_RUN ? -1 : all;
      sm_len[r] = len;
    }
    c[j] = count(all, len);
    cs += c[j];
    zs += c[j] > 0;
  }
  const int ci = wave_prefix(cs), zi = wave_prefix(zs);
  if (lane == 63) {
    sm_w[0][wave] = ci;
    sm_w[1][wave] = zi;
  }
  if (tid == 0) sm_cut[0] = -1;
  __syncthreads();
  int cb = ci - cs, zb = zi - zs;
  unsigned total = 0, some = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    if (w < wave) {
      cb += sm_w[0][w];
      zb += sm_w[1][w];
    }
    total += sm_w[0][w];
    some += sm_w[1][w];
  }
  // ---- this workgroup's share ----
  unsigned wgs = static_cast<unsigned>(p_.d.num_wgs);
  {
    const unsigned least = (total + LEAST - 1) / LEAST, twice = total / (2 * LEAST);
    const unsigned early = (wgs + LATE - 1) / LATE;
    const unsigned few = early < least ? early : least, many = few > twice ? few : twice;
    wgs = wgs < many ? wgs : many;
  }
  if (static_cast<unsigned>(wg) < wgs) {
    const unsigned share = total / wgs;
    const unsigned start = share < START ? share : START;
    const unsigned span = total + start * some, q = span / wgs, rem = span - q * wgs;
    // cuts at span * w / wgs; the thread whose sequence holds one says which
    // of its chunks come before it (in steps of 4, one for each wave, where
    // the shares are long)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const unsigned w = wg + i, x = q * w + rem * w / wgs;
      unsigned base = cb + start * zb;
#pragma unroll
      for (int j = 0; j < EPT; ++j) {
        const unsigned next = base + (c[j] > 0 ? c[j] + start : 0u);
        if (x >= base && (x < next || (w == wgs && x == next && c[j] > 0))) {
          unsigned in = x - base > start ? x - base - start : 0u;
          if (share >= 16) in = (in + 2) & ~3u;
          if (w == wgs || in > static_cast<unsigned>(c[j])) in = c[j];
          sm_cut[2 * i] = tid * EPT + j;
          sm_cut[2 * i + 1] = in;
        }
        base = next;
      }
    }
  }
  __syncthreads();
}

}  // namespace hcp
