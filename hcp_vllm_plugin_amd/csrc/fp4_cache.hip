// Writes into the 4-bit KV cache and reads of what it stands for.
#include "params.h"

namespace hcp {

__device__ __forceinline__ int64_t slot_at(const void* slots, bool wide, int64_t t) {
  return wide ? reinterpret_cast<const int64_t*>(slots)[t]
              : static_cast<int64_t>(reinterpret_cast<const int32_t*>(slots)[t]);
}

// A thread's (token, head) row and its eight columns of it: threads are counted in
// 32 bits, so that the divisions are too.
struct RowPart {
  uint32_t t;
  int h, oct;
};
__device__ __forceinline__ RowPart row_part(uint32_t gid, Fp4Region r, int opr_shift, int heads) {
  const uint32_t opr = r.d / 8;  // octets of a row: a multiple of 4, so quads share one
  const uint32_t row = opr_shift >= 0 ? gid >> opr_shift : gid / opr;
  const uint32_t t = row / static_cast<uint32_t>(heads);
  return {t, static_cast<int>(row - t * heads), static_cast<int>(gid - row * opr)};
}

// One thread per eight columns of a (token, head) row, of K and of V (a thread for
// either: 65536 x 8 x 128 at consecutive slots 84 us, with both loads of one on their
// way 70, 4.8 TB/s; 16 tokens 2.4 and 2.5).  HBM-bound: 2 d bytes read and 17 d / 32
// written per row.  A negative slot or one past the cache is skipped.
template <typename T>
__global__ __launch_bounds__(256) void fp4_write_kernel(Fp4Params p) {
  const auto [part, h, oct] = row_part(blockIdx.x * 256u + threadIdx.x, p.r, p.opr_shift,
                                       p.num_kv_heads);
  const int64_t t = part;
  if (t >= p.num_tokens) return;
  const int64_t slot = slot_at(p.slots, p.slots_wide, t);
  if (slot < 0 || slot >= p.num_slots) return;
  const u32x4 k = ldg16(reinterpret_cast<const char*>(p.key) +
                        (t * p.k_stride_tok + h * p.k_stride_head + oct * 8) * 2);
  const u32x4 v = ldg16(reinterpret_cast<const char*>(p.value) +
                        (t * p.v_stride_tok + h * p.v_stride_head + oct * 8) * 2);
  char* region = p.cache + (slot >> p.bs_shift) * p.stride_block + h * p.stride_head;
  const int off = static_cast<int>(slot & (p.r.bs - 1));
  fp4_store<T>(region, p.r, false, off, oct, k);
  fp4_store<T>(region, p.r, true, off, oct, v);
}

// Eight columns of K and of V of one key, out of its region.
template <typename T>
__device__ __forceinline__ void fp4_fetch(const char* region, Fp4Region r, int off, int oct,
                                          u32x4& k, u32x4& v) {
  const auto* u8 = reinterpret_cast<const uint8_t*>(region);
  const uint32_t ck = *reinterpret_cast<const uint32_t*>(region + r.k_code(off, oct));
  const uint32_t cv = *reinterpret_cast<const uint32_t*>(region + r.v_code(off, oct));
  const uint32_t sk = u8[r.k_scale(off, oct >> 2)], sv = u8[r.v_scale(off, oct >> 2)];
  k = fp4_values<T>(ck, __uint_as_float(sk << 23));
  v = fp4_values<T>(cv, __uint_as_float(sv << 23));
}

// The rows at `slots` as 16-bit values [n, Hkv, d]; a slot outside the cache
// reads as zeros.
template <typename T>
__global__ __launch_bounds__(256) void fp4_read_kernel(Fp4Params p) {
  const uint32_t gid = blockIdx.x * 256u + threadIdx.x;
  const auto [part, h, oct] = row_part(gid, p.r, p.opr_shift, p.num_kv_heads);
  const int64_t t = part;
  if (t >= p.num_tokens) return;
  const int64_t slot = slot_at(p.slots, p.slots_wide, t);
  u32x4 k = {0, 0, 0, 0}, v = k;
  if (slot >= 0 && slot < p.num_slots)
    fp4_fetch<T>(p.cache + (slot >> p.bs_shift) * p.stride_block + h * p.stride_head, p.r,
                 static_cast<int>(slot & (p.r.bs - 1)), oct, k, v);
  reinterpret_cast<u32x4*>(p.k_out)[gid] = k;
  reinterpret_cast<u32x4*>(p.v_out)[gid] = v;
}

constexpr uint32_t kGatherParts = 4;  // of a thread of fp4_gather_kernel

// Entry e's keys [start, start + len) of its request's blocks to rows
// out_start[e] .. of [num_rows, Hkv, d], for the prefill kernel.  The threads are
// laid over the rows that there are, and find their entry: 200 entries of 100 keys
// and one of 128k at 4 x 128 88 us (1570 with a workgroup for every entry and part
// of the longest), 64 of 512 15.8 (15.3), one of 32k 15.1.  Four parts a thread pay
// for the search (with one 152, 24.0 and 17.1; with eight 93, 16.2 and 15.7).
template <typename T>
__global__ __launch_bounds__(256) void fp4_gather_kernel(Fp4GatherParams p) {
  const uint32_t base = blockIdx.x * 256u * kGatherParts;
  {
    const uint32_t i = blockIdx.x * 256u + threadIdx.x;
    if (p.entries_out != nullptr && i < static_cast<uint32_t>(p.num_entries)) {
      hcp_varlen_entry e = p.entries[i];
      e.kv.k_addr = reinterpret_cast<uint64_t>(p.k_out);
      e.kv.v_addr = reinterpret_cast<uint64_t>(p.v_out);
      e.kv.block_table = 0;
      e.kv.stride_tok = static_cast<int64_t>(p.num_kv_heads) * p.r.d;
      e.kv.stride_head = p.r.d;
      e.kv.stride_block = 0;
      e.kv.start = p.out_start[i];
      e.kv.block_size = e.kv.num_blocks = 0;
      p.entries_out[i] = e;
    }
  }
  // the last entry that begins at or before the workgroup's first row: 64 candidates
  // a step
  const int64_t first = row_part(base, p.r, p.opr_shift, p.num_kv_heads).t;
  if (first >= p.num_rows) return;
  int e = 0;
  for (int span = p.num_entries; span > 1;) {
    const int step = (span + 63) / 64, at = (threadIdx.x & 63) * step;
    const bool before = at < span && p.out_start[e + at] <= first;
    const int k = __builtin_popcountll(__builtin_amdgcn_ballot_w64(before)) - 1;
    if (k < 0) return;  // (rows before the first entry's)
    e += k * step;
    span = step < span - k * step ? step : span - k * step;
  }
  e = __builtin_amdgcn_readfirstlane(e);
  int64_t begin = p.out_start[e];
  hcp_kv_segment s = p.entries[e].kv;
  int64_t next = e + 1 < p.num_entries ? p.out_start[e + 1] : INT64_MAX;
#pragma unroll
  for (uint32_t i = 0; i < kGatherParts; ++i) {
    const uint32_t gid = base + 256u * i + threadIdx.x;
    const auto [part, h, oct] = row_part(gid, p.r, p.opr_shift, p.num_kv_heads);
    const int64_t row = part;
    if (row >= p.num_rows) return;
    if (row >= next) {
      do {
        ++e;
        next = e + 1 < p.num_entries ? p.out_start[e + 1] : INT64_MAX;
      } while (row >= next);
      begin = p.out_start[e];
      s = p.entries[e].kv;
    }
    const int64_t t = row - begin;
    if (t < 0 || t >= s.len || s.block_table == 0) continue;
    const int64_t pos = s.start + t;
    uint32_t blk = static_cast<uint32_t>(
        reinterpret_cast<const int32_t*>(s.block_table)[pos >> p.bs_shift]);
    blk = blk < p.num_blocks ? blk : p.num_blocks - 1;  // past the cache: its last block
    u32x4 k, v;
    fp4_fetch<T>(p.cache + blk * p.stride_block + h * p.stride_head, p.r,
                 static_cast<int>(pos & (p.r.bs - 1)), oct, k, v);
    reinterpret_cast<u32x4*>(p.k_out)[gid] = k;
    reinterpret_cast<u32x4*>(p.v_out)[gid] = v;
  }
}

hipError_t launch_fp4_write(const Fp4Params& p, int dtype, hipStream_t st) {
  const int64_t grid = (p.num_tokens * p.num_kv_heads * (p.r.d / 8) + 255) / 256;
  const dim3 g(static_cast<unsigned>(grid));
  if (dtype == HCP_DTYPE_BF16)
    hipLaunchKernelGGL(fp4_write_kernel<__bf16>, g, dim3(256), 0, st, p);
  else
    hipLaunchKernelGGL(fp4_write_kernel<_Float16>, g, dim3(256), 0, st, p);
  return hipGetLastError();
}

hipError_t launch_fp4_read(const Fp4Params& p, int dtype, hipStream_t st) {
  const int64_t grid = (p.num_tokens * p.num_kv_heads * (p.r.d / 8) + 255) / 256;
  const dim3 g(static_cast<unsigned>(grid));
  if (dtype == HCP_DTYPE_BF16)
    hipLaunchKernelGGL(fp4_read_kernel<__bf16>, g, dim3(256), 0, st, p);
  else
    hipLaunchKernelGGL(fp4_read_kernel<_Float16>, g, dim3(256), 0, st, p);
  return hipGetLastError();
}

hipError_t launch_fp4_gather(const Fp4GatherParams& p, int dtype, hipStream_t st) {
  const int64_t parts = p.num_rows * p.num_kv_heads * (p.r.d / 8);
  const int64_t work = (parts + kGatherParts - 1) / kGatherParts;
  // (a thread at least for every entry)
  const dim3 g(static_cast<unsigned>(((work > p.num_entries ? work : p.num_entries) + 255) / 256));
  if (dtype == HCP_DTYPE_BF16)
    hipLaunchKernelGGL(fp4_gather_kernel<__bf16>, g, dim3(256), 0, st, p);
  else
    hipLaunchKernelGGL(fp4_gather_kernel<_Float16>, g, dim3(256), 0, st, p);
  return hipGetLastError();
}

}  // namespace hcp
