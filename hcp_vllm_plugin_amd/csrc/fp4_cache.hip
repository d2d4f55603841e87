// Writes into the 4-bit KV cache and reads of what it stands for.
#include "params.h"

namespace hcp {

__device__ __forceinline__ int64_t slot_at(const void* slots, bool wide, int64_t t) {
  return wide ? reinterpret_cast<const int64_t*>(slots)[t]
              : static_cast<int64_t>(reinterpret_cast<const int32_t*>(slots)[t]);
}

// One thread per eight columns of a (token, head) row, of K (grid.y 0) or V.
// HBM-bound: 2 d bytes read and 17 d / 32 written per row.  A negative slot or
// one past the cache is skipped.
template <typename T>
__global__ __launch_bounds__(256) void fp4_write_kernel(Fp4Params p) {
  const int64_t gid = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int opr = p.r.d / 8;  // octets of a row: a multiple of 4, so quads share one
  const int64_t row = p.opr_shift >= 0 ? gid >> p.opr_shift : gid / opr;
  if (row >= p.num_tokens * p.num_kv_heads) return;
  const int oct = static_cast<int>(gid - row * opr);
  const int64_t t = row / p.num_kv_heads;
  const int h = static_cast<int>(row - t * p.num_kv_heads);
  const int64_t slot = slot_at(p.slots, p.slots_wide, t);
  if (slot < 0 || slot >= p.num_slots) return;
  const bool is_v = blockIdx.y != 0;
  const char* src = is_v ? reinterpret_cast<const char*>(p.value) +
                               (t * p.v_stride_tok + h * p.v_stride_head + oct * 8) * 2
                         : reinterpret_cast<const char*>(p.key) +
                               (t * p.k_stride_tok + h * p.k_stride_head + oct * 8) * 2;
  char* region = p.cache + (slot >> p.bs_shift) * p.stride_block + h * p.stride_head;
  fp4_store<T>(region, p.r, is_v, static_cast<int>(slot & (p.r.bs - 1)), oct, ldg16(src));
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
  const int64_t gid = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int opr = p.r.d / 8;
  const int64_t row = p.opr_shift >= 0 ? gid >> p.opr_shift : gid / opr;
  if (row >= p.num_tokens * p.num_kv_heads) return;
  const int oct = static_cast<int>(gid - row * opr);
  const int64_t t = row / p.num_kv_heads;
  const int h = static_cast<int>(row - t * p.num_kv_heads);
  const int64_t slot = slot_at(p.slots, p.slots_wide, t);
  u32x4 k = {0, 0, 0, 0}, v = k;
  if (slot >= 0 && slot < p.num_slots)
    fp4_fetch<T>(p.cache + (slot >> p.bs_shift) * p.stride_block + h * p.stride_head, p.r,
                 static_cast<int>(slot & (p.r.bs - 1)), oct, k, v);
  reinterpret_cast<u32x4*>(p.k_out)[gid] = k;
  reinterpret_cast<u32x4*>(p.v_out)[gid] = v;
}

// Entry e's keys [start, start + len) of its request's blocks to rows
// out_start[e] .. of [total, Hkv, d], for the prefill kernel: grid.y the entry.
template <typename T>
__global__ __launch_bounds__(256) void fp4_gather_kernel(Fp4GatherParams p) {
  const hcp_kv_segment s = p.entries[blockIdx.y].kv;
  if (p.entries_out != nullptr && blockIdx.x == 0 && threadIdx.x == 0) {
    hcp_varlen_entry e = p.entries[blockIdx.y];
    e.kv.k_addr = reinterpret_cast<uint64_t>(p.k_out);
    e.kv.v_addr = reinterpret_cast<uint64_t>(p.v_out);
    e.kv.block_table = 0;
    e.kv.stride_tok = static_cast<int64_t>(p.num_kv_heads) * p.r.d;
    e.kv.stride_head = p.r.d;
    e.kv.stride_block = 0;
    e.kv.start = p.out_start[blockIdx.y];
    e.kv.block_size = e.kv.num_blocks = 0;
    p.entries_out[blockIdx.y] = e;
  }
  const int64_t gid = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int opr = p.r.d / 8;
  const int64_t row = p.opr_shift >= 0 ? gid >> p.opr_shift : gid / opr;
  if (row >= s.len * p.num_kv_heads || s.block_table == 0) return;
  const int oct = static_cast<int>(gid - row * opr);
  const int64_t t = row / p.num_kv_heads;
  const int h = static_cast<int>(row - t * p.num_kv_heads);
  const int64_t pos = s.start + t;
  uint32_t blk = static_cast<uint32_t>(
      reinterpret_cast<const int32_t*>(s.block_table)[pos >> p.bs_shift]);
  blk = blk < p.num_blocks ? blk : p.num_blocks - 1;  // past the cache: its last block
  u32x4 k, v;
  fp4_fetch<T>(p.cache + blk * p.stride_block + h * p.stride_head, p.r,
               static_cast<int>(pos & (p.r.bs - 1)), oct, k, v);
  const int64_t dst = (((p.out_start[blockIdx.y] + t) * p.num_kv_heads + h) * opr + oct);
  reinterpret_cast<u32x4*>(p.k_out)[dst] = k;
  reinterpret_cast<u32x4*>(p.v_out)[dst] = v;
}

hipError_t launch_fp4_write(const Fp4Params& p, int dtype, hipStream_t st) {
  const int64_t grid = (p.num_tokens * p.num_kv_heads * (p.r.d / 8) + 255) / 256;
  const dim3 g(static_cast<unsigned>(grid), 2);
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
  const int64_t grid = (p.max_len * p.num_kv_heads * (p.r.d / 8) + 255) / 256;
  // (a workgroup at least, for the entries)
  const dim3 g(static_cast<unsigned>(grid > 0 ? grid : 1), static_cast<unsigned>(p.num_entries));
  if (dtype == HCP_DTYPE_BF16)
    hipLaunchKernelGGL(fp4_gather_kernel<__bf16>, g, dim3(256), 0, st, p);
  else
    hipLaunchKernelGGL(fp4_gather_kernel<_Float16>, g, dim3(256), 0, st, p);
  return hipGetLastError();
}

}  // namespace hcp
