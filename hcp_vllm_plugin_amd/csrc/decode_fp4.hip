// Split-KV decode over the 4-bit cache: one query token per sequence, lengths
// and block tables read on the device (no plan), as decode_paged_kernel.
//
// For query head h of KV head h / G: out = sum_j softmax_j(q . k_j * scale) v_j over
// k_j[d] = code * 2^(b - 127), one scale byte b for 32 columns.  A key of a head is
// d + d / 16 bytes where 16-bit values take 4 d, so the same HBM rate would ask for
// 3.8 times the keys per second, and what a key costs in instructions counts:
//  * the cache lies as the matrix operands do (fp4.h): a lane loads 32 columns of
//    one key of K, or 8 columns of four keys of V, in 16 bytes, a wave 1 KB in a
//    row; one v_cvt_scalef32_pk makes two 16-bit operand values of a byte, exactly,
//    its scale applied;
//  * S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_16x16x32 as in decode_split_body:
//    16 query heads are the columns, the contraction order of either product is
//    free, so K's is the order of a lane's bytes and P stays in the registers S
//    came in; V's keys are paired by one v_perm for two values;
//  * the running maximum is raised, and O rescaled, only when a weight is past 2^8
//    (fp32 sums and two 16-bit terms of P have room for that), so that a chunk
//    needs the maximum of its weights alone; their sum is a matrix product with
//    ones.
// The 4 waves of a workgroup take the 32-key chunks of its share in turn (chunks
// lie on multiples of 32 positions, so that 16 keys never cross a block), each
// through LDS of its own, where the next chunk lands while one is computed (held
// in registers instead, two chunks take 212 of them at 128 columns and spill at
// 256: 364 us for 32 x 4k-16k keys of 16 / 8 x 256, then 137; 14 / 2 x 64, 64 x
// 16k-32k 64 -> 51 us).  The waves are combined through LDS; decode_reduce_kernel
// merges a sequence's partials.
//
// Bound by HBM, us of a pass with the merge: 64 x 16k-32k keys of 28 / 4 x 128 (851 MB)
// 144-148, 5.9 TB/s (146 against 144 on one card with the scores' maximum, the sum and
// the scales in more instructions); 256 x 16k of these heads (2.29 GB) 369, 6.2 TB/s; 64 x
// 16k of 16 / 8 x 256 (2.28 GB) 355, 6.4 TB/s; the 16-bit kernel reads its blocks at 6.6.
// On the same card the same launches with compute() left out 142, 358 and 344.  At
// 64 columns a chunk has as many instructions for half the bytes, and a head's 1088
// bytes of a 16-token block are eight and a half lines of which nine are fetched (1.22
// GB of HBM for 1.14 GB): 256 x 32k keys of 14 / 2 x 64 take 210 us, 196 without
// compute().  One sequence of 2000 keys: 8.3 us and 4.2 for the merge, the chain of
// latencies (lengths, block ids, keys, combine, merge).
#include "decode_share.h"

namespace hcp {

// A wave's tile (16 keys) in LDS: its codes, each lane's 16 bytes of a load next to
// the other lanes', then its scales.
template <int D>
struct Fp4Tile {
  static constexpr int NC = D / 64;             // loads of codes, 1 KB each
  static constexpr int SC = 1024 * NC;          // where the scales begin
  static constexpr int SW = D == 256 ? 32 : 16; // dwords of K (or V) scales
  static constexpr int BYTES = SC + 256;
  static constexpr int NI = NC + 1;             // loads
  static constexpr int P = D == 256 ? 2 : 1;    // 16-byte pieces of K (or V) per lane
};

#define HCP_LDS_PTR(T) __attribute__((address_space(3))) T*

template <typename T>
__device__ __forceinline__ T lds_at(const HCP_LDS_PTR(char) p) {
  return *reinterpret_cast<const HCP_LDS_PTR(T)>(p);
}

// How far (in powers of two) a score may pass the running maximum, and what the
// maximum's own weight is: fp16's terms have 2^-24 for their last place, so that
// weights begin 2^7 higher, the largest at 2^15 of its 65504.
constexpr float kRaise = 8.f;
template <typename T>
constexpr float kLift = __is_same(T, __bf16) ? 0.f : 7.f;

// Two weights (or NaN) in two 16-bit terms: hi the weight rounded, lo what is left of
// it, rounded: 2^-17 of it (fp16 2^-22, and 2^-25 at least).  Both to the nearest:
// cut off, many small weights next to a large one would add up to less than they are.
// (two_terms of common.h keeps both terms positive for products with an infinity; the
// 4-bit cache holds none.)
template <typename T>
__device__ __forceinline__ void split_weights(float a, float b, uint32_t& hi, uint32_t& lo) {
  hi = pack2<T>(a, b);
  lo = pack2<T>(a - Elem<T>::to_float(static_cast<uint16_t>(hi & 0xffffu)),
                b - Elem<T>::to_float(static_cast<uint16_t>(hi >> 16)));
}

// Byte J of a dword of scales as a float, in one instruction.
template <int J>
__device__ __forceinline__ float fp4_scale_of(uint32_t w) {
  uint32_t r;
  asm("v_lshlrev_b32_sdwa %0, %1, %2 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:DWORD "
      "src1_sel:BYTE_%3"
      : "=v"(r)
      : "v"(23), "v"(w), "n"(J));
  return __uint_as_float(r);
}

template <int D, typename T, bool KEEP_NAN>
__device__ __forceinline__ void fp4_split_body(const PagedDecParams& p, int kvh_in, int chunk_in,
                                               int slot_out, int r, int first, int all,
                                               int kb, int ke, char (*bufE)[2 * Fp4Tile<D>::BYTES],
                                               char (*bufO)[2 * Fp4Tile<D>::BYTES],
                                               float (*sm_m)[16], float (*sm_l)[16]) {
  using E = Elem<T>;
  using V8 = typename E::vec8;
  using Tile = Fp4Tile<D>;
  constexpr int QSTEPS = D / 32;
  constexpr int NU = D / 16;
  constexpr int W = 4;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c16 = lane & 15, g4 = lane >> 4;
  const int kvh = __builtin_amdgcn_readfirstlane(kvh_in);
  const int chunk = __builtin_amdgcn_readfirstlane(chunk_in);
  const int G = p.d.group - 16 * chunk < 16 ? p.d.group - 16 * chunk : 16;
  const int h0 = kvh * p.d.group + 16 * chunk;
  const int dv = p.d.head_dim;

  // Q^T: column c16 = query head h0 + c16; the lane's columns of k-step s are
  // (D / 4) g4 + 8 s .. + 7, the order of its K bytes
  V8 qf[QSTEPS];
  {
    const bool hv = c16 < G;
    const char* qrow = reinterpret_cast<const char*>(p.d.q) +
                       (r * p.d.q_stride_tok +
                        static_cast<int64_t>(h0 + (hv ? c16 : 0)) * p.d.q_stride_head) * 2;
#pragma unroll
    for (int s = 0; s < QSTEPS; ++s) {
      const int d0 = D / 4 * g4 + 8 * s;
      qf[s] = as_vec8<V8>(hv && d0 < dv ? ldg16(qrow + d0 * 2) : u32x4{0, 0, 0, 0});
    }
  }

  const int bs = p.kv.block_size, bs_shift = 31 - __builtin_clz(bs);
  const auto* bt = global_ptr(reinterpret_cast<const char*>(
      p.kv.block_table + static_cast<uint64_t>(r) * p.bt_stride * 4));
  const uint32_t id_max = static_cast<uint32_t>(p.kv.num_blocks) - 1;
  const char* head = reinterpret_cast<const char*>(p.kv.k_addr) + kvh * p.kv.stride_head;

  // Lane offsets in a region.  A piece past the row's dv columns is fetched from
  // the row's first instead: it meets zeros of Q, or lands in columns of O that
  // are not stored.
  const int vb = bs * (dv / 2), ng = dv / 32;
  int koff[Tile::P], voff[Tile::P];  // (D 64: one load, K in the lower lanes, V in the upper)
  // where in a tile a lane finds its K codes, K scale (a byte), V codes and V scales
  // (a dword: four keys)
  int kc_at[Tile::P], vc_at[Tile::P];
#pragma unroll
  for (int i = 0; i < Tile::P; ++i) {
    int key = c16, d0 = D / 4 * g4, quad = g4, oct = NU * c16 / 8;
    kc_at[i] = lane * 16;
    vc_at[i] = Tile::P * 1024 + lane * 16;
    if constexpr (D == 64) {
      const int l = lane & 31;
      key = l >> 1;
      d0 = 32 * (l & 1);
      quad = l >> 3;
      oct = l & 7;
      kc_at[i] = c16 * 32 + g4 * 8;
      vc_at[i] = 512 + g4 * 128 + (c16 >> 1) * 16;
    } else if constexpr (D == 256) {
      // A lane takes two pieces in a row of either, but what a load fetches lies in a
      // row too: keys 8 i .. of K, quads 2 i and 2 i + 1 of V, four lanes the 64 bytes
      // of four pieces (with every other piece of 2 KB in a load, 64 x 16k keys of
      // 16 / 8 heads took 418 us on a card where these take 368).  The order of the four in LDS spreads the
      // reads of 16 lanes over all banks for V, over half of them for K (over all of
      // them, K's 64 bytes in another order: 369).
      const int q = lane >> 2, r = lane & 3, e = c16 >> 1;
      key = 8 * i + (q >> 1);
      d0 = 128 * (q & 1) + 32 * (r ^ (key >> 1 & 3));
      quad = 2 * i + (q >> 3);
      oct = 4 * (q & 7) + (r ^ (q >> 2 & 1));
      kc_at[i] = (c16 >> 3) * 1024 + ((c16 & 7) * 2 + (g4 >> 1)) * 64 +
                 ((2 * (g4 & 1) + i) ^ (c16 >> 1 & 3)) * 16;
      vc_at[i] = 2048 + (g4 >> 1) * 1024 + ((g4 & 1) * 8 + e) * 64 +
                 ((2 * (c16 & 1) + i) ^ (e >> 2)) * 16;
    }
    koff[i] = key * (dv / 2) + (d0 < dv ? d0 / 2 : 0);
    voff[i] = vb + (quad * (dv / 8) + (oct < dv / 8 ? oct : 0)) * 16;
    if (D == 64 && lane >= 32) koff[i] = voff[i];
  }
  const int si = lane & (Tile::SW - 1), sv = lane / Tile::SW & 1;
  const int soff = bs * dv + sv * bs * ng + (si < 4 * ng ? si : 0) * 4;
  const int region = static_cast<int>(Fp4Region{dv, bs}.bytes());

  // Block ids of a chunk's tiles, in the two halves of the wave.
  auto fetch_ids = [&](int x0) __attribute__((always_inline)) {
    const int x = x0 + (lane & 32) / 2;
    const uint32_t at = static_cast<uint32_t>(x < all ? x : all - 1) >> bs_shift << 2;
    return *global_ptr(reinterpret_cast<const uint32_t*>(reinterpret_cast<uintptr_t>(bt) + at));
  };
  // (buffer loads: behind global loads into LDS the compiler waits for every load
  // before it uses one's result)
  auto issue = [&](int x0, uint32_t ids, HCP_LDS_PTR(char) dst) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      uint32_t id = __builtin_amdgcn_readlane(ids, 32 * t);
      id = id < id_max ? id : id_max;  // past the cache: its last block
      const int off = (x0 + 16 * t) & (bs - 1);
      const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
          const_cast<char*>(head + id * p.kv.stride_block), 0, region, 0x00020000);
      auto load = [&](int at, int o, int so) __attribute__((always_inline)) {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            rs, reinterpret_cast<HCP_LDS_PTR(void)>(dst + t * Tile::BYTES + at), 16, o, so, 0, 2);
      };
      const int row = off * (dv / 2);
#pragma unroll
      for (int i = 0; i < Tile::P; ++i) {
        load(i * 1024, koff[i], row);
        if constexpr (D > 64) load((Tile::P + i) * 1024, voff[i], row);
      }
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rs, reinterpret_cast<HCP_LDS_PTR(void)>(dst + t * Tile::BYTES + Tile::SC), 4, soff,
          off * ng, 0, 2);
    }
  };
  int ks_at[Tile::P];
#pragma unroll
  for (int i = 0; i < Tile::P; ++i) {
    const int g = D / 4 * g4 / 32 + i;
    ks_at[i] = Tile::SC + ((c16 >> 2) * ng + (g < ng ? g : 0)) * 4 + (c16 & 3);
  }
  const int vgrp = NU * c16 / 32;
  const int vs_at = Tile::SC + Tile::SW * 4 + (g4 * ng + (vgrp < ng ? vgrp : 0)) * 4;

  const float c = p.d.scale_log2;
  // -(running maximum, kLift below), 0 before the first; the weight past which it is raised; the
  // sum of the weights as rounded (a matrix product with ones, in every row)
  float neg_m = 0.f, limit = -1.f;
  const float most = __builtin_exp2f(kRaise + kLift<T>);
  f32x4 lacc = f32x4{};
  const V8 ones = as_vec8<V8>(__is_same(T, __bf16)
                                  ? u32x4{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u}
                                  : u32x4{0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u});
  const uint32_t half = c16 & 1 ? 0x07060302u : 0x05040100u;
  f32x4 oacc[NU];
#pragma unroll
  for (int u = 0; u < NU; ++u) oacc[u] = f32x4{};

  auto compute = [&](int x0, const HCP_LDS_PTR(char) src) __attribute__((always_inline)) {
    f32x4 s[2] = {f32x4{}, f32x4{}};
    uint32_t vsw[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const HCP_LDS_PTR(char) const tile = src + t * Tile::BYTES;
#pragma unroll
      for (int i = 0; i < Tile::P; ++i) {
        const float ks =
            __uint_as_float(static_cast<uint32_t>(lds_at<uint8_t>(tile + ks_at[i])) << 23);
        if constexpr (D == 64) {
          const u32x2 w = lds_at<u32x2>(tile + kc_at[0]);
#pragma unroll
          for (int q = 0; q < 2; ++q)
            s[t] = E::mfma16(as_vec8<V8>(fp4_values<T>(w[q], ks)), qf[q], s[t]);
        } else {
          const u32x4 w = lds_at<u32x4>(tile + kc_at[i]);
#pragma unroll
          for (int q = 0; q < 4; ++q)
            s[t] = E::mfma16(as_vec8<V8>(fp4_values<T>(w[q], ks)), qf[4 * i + q], s[t]);
        }
      }
      vsw[t] = lds_at<uint32_t>(tile + vs_at);
    }
    if (x0 < first || x0 + 32 > ke) {
      // keys outside the split: no weight, and a finite value whatever their
      // bytes say (0 times a NaN would stay one)
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = x0 + 16 * t + 4 * g4 + i;
          if (key < first || key >= ke) {
            s[t][i] = -INFINITY;
            vsw[t] &= ~(0xffu << (8 * i));
          }
        }
    }
    float w[2][4];
    auto weights = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) w[t][i] = fast_exp2(__builtin_fmaf(s[t][i], c, neg_m));
    };
    weights();
    const float top = fmaxf(fmaxf(fmaxf(w[0][0], w[0][1]), fmaxf(w[0][2], w[0][3])),
                            fmaxf(fmaxf(w[1][0], w[1][1]), fmaxf(w[1][2], w[1][3])));
    if (__builtin_amdgcn_ballot_w64(top > limit) != 0) {
      float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                       fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3]))) * c;
      mx = fmaxf(mx, __shfl_xor(mx, 16));
      mx = fmaxf(mx, __shfl_xor(mx, 32));
      const float m_old = limit < 0.f ? -INFINITY : -neg_m;
      const float m_new = fmaxf(m_old, mx - kLift<T>);
      neg_m = m_new == -INFINITY ? 0.f : -m_new;
      limit = m_new == -INFINITY ? -1.f : most;
      const float alpha = fast_exp2(m_old + neg_m);
      lacc *= alpha;
#pragma unroll
      for (int u = 0; u < NU; ++u) oacc[u] *= alpha;
      weights();
    }
    u32x4 pw, rw;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t hi, lo;
        split_weights<T>(w[t][2 * i], w[t][2 * i + 1], hi, lo);
        pw[2 * t + i] = hi;
        rw[2 * t + i] = lo;
      }
    const V8 pf = as_vec8<V8>(pw), rf = as_vec8<V8>(rw);
    lacc = E::mfma16(ones, pf, lacc);
    lacc = E::mfma16(ones, rf, lacc);
    float vs[8];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      vs[4 * t] = fp4_scale_of<0>(vsw[t]);
      vs[4 * t + 1] = fp4_scale_of<1>(vsw[t]);
      vs[4 * t + 2] = fp4_scale_of<2>(vsw[t]);
      vs[4 * t + 3] = fp4_scale_of<3>(vsw[t]);
    }
    u32x4 vw[2][Tile::P];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < Tile::P; ++i)
        vw[t][i] = lds_at<u32x4>(src + t * Tile::BYTES + vc_at[i]);
    if constexpr (D == 64) {
      // a lane's two of the four bytes, of two keys in one dword
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          vw[t][0][j] = __builtin_amdgcn_perm(vw[t][0][2 * j + 1], vw[t][0][2 * j], half);
    }
    // columns 2 u and 2 u + 1 of 8 keys -> two operands
    auto pv = [&](auto sel, auto piece, int u) __attribute__((always_inline)) {
      uint32_t x[8];
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        constexpr int S = decltype(sel)::value;
        const u32x4 v = vw[j >> 2][decltype(piece)::value];
        const int at = D == 64 ? (j & 3) >> 1 : j & 3;
        x[j] = fp4_pair<T, S>(v[at], vs[j]);
        x[j + 1] = fp4_pair<T, D == 64 ? S + 2 : S>(v[D == 64 ? at : at + 1], vs[j + 1]);
      }
      u32x4 a, b;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        a[j] = __builtin_amdgcn_perm(x[2 * j + 1], x[2 * j], 0x05040100u);
        b[j] = __builtin_amdgcn_perm(x[2 * j + 1], x[2 * j], 0x07060302u);
      }
      oacc[2 * u] = E::mfma16(as_vec8<V8>(a), pf, oacc[2 * u]);
      oacc[2 * u] = E::mfma16(as_vec8<V8>(a), rf, oacc[2 * u]);
      oacc[2 * u + 1] = E::mfma16(as_vec8<V8>(b), pf, oacc[2 * u + 1]);
      oacc[2 * u + 1] = E::mfma16(as_vec8<V8>(b), rf, oacc[2 * u + 1]);
    };
    using I0 = std::integral_constant<int, 0>;
    using I1 = std::integral_constant<int, 1>;
    using I2 = std::integral_constant<int, 2>;
    using I3 = std::integral_constant<int, 3>;
    pv(I0{}, I0{}, 0);
    pv(I1{}, I0{}, 1);
    if constexpr (D > 64) {
      pv(I2{}, I0{}, 2);
      pv(I3{}, I0{}, 3);
    }
    if constexpr (D > 128) {
      pv(I0{}, I1{}, 4);
      pv(I1{}, I1{}, 5);
      pv(I2{}, I1{}, 6);
      pv(I3{}, I1{}, 7);
    }
  };

  // The wave's chunks, kb + 32 (wave, wave + W, ..): the block ids of the one after
  // the next are fetched, the next one's bytes loaded, and when only those are
  // outstanding the current one has landed.  (Loads without a branch around
  // them, so that the compiler's waits are exact too: past the last chunk they
  // repeat it.)
  constexpr int ST = 32 * W;
  int x = kb + 32 * wave;
  if (x < ke) {
    HCP_LDS_PTR(char) const be = (HCP_LDS_PTR(char))(bufE[wave]);
    HCP_LDS_PTR(char) const bo = (HCP_LDS_PTR(char))(bufO[wave]);
    const int last = x + (ke - 1 - x) / ST * ST;
    auto upto = [&](int y) __attribute__((always_inline)) { return y < last ? y : last; };
    uint32_t ia = fetch_ids(x), ib = fetch_ids(upto(x + ST));
    __builtin_amdgcn_sched_barrier(0);
    issue(x, ia, be);
    while (true) {
      ia = fetch_ids(upto(x + 2 * ST));
      // (ids before the loads: waiting for them must not wait for these)
      __builtin_amdgcn_sched_barrier(0);
      issue(upto(x + ST), ib, bo);
      wait_vmcnt<2 * Tile::NI + 1>();
      compute(x, be);
      x += ST;
      if (x > last) break;
      ib = fetch_ids(upto(x + 2 * ST));
      __builtin_amdgcn_sched_barrier(0);
      issue(upto(x + ST), ia, be);
      wait_vmcnt<2 * Tile::NI + 1>();
      compute(x, bo);
      x += ST;
      if (x > last) break;
    }
  }

  // ---- combine the W waves, in the chunk buffers (two waves to each) ----
  wait_vmcnt<0>();  // the last loads still write there
  __syncthreads();
  float (*const so_e)[16][D + 4] = reinterpret_cast<float (*)[16][D + 4]>(&bufE[0][0]);
  float (*const so_o)[16][D + 4] = reinterpret_cast<float (*)[16][D + 4]>(&bufO[0][0]);
  static_assert(sizeof(float) * 2 * 16 * (D + 4) <= W * 2 * Tile::BYTES, "combine staging");
  float (*const mine)[D + 4] = wave < 2 ? so_e[wave] : so_o[wave - 2];
  if (g4 == 0) {
    sm_m[wave][c16] = limit < 0.f ? -INFINITY : -neg_m;
    sm_l[wave][c16] = lacc[0];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int u = 0; u < NU; u += 4)
      *reinterpret_cast<f32x4*>(&mine[c16][NU * (4 * g4 + i) + u]) =
          f32x4{oacc[u][i], oacc[u + 1][i], oacc[u + 2][i], oacc[u + 3][i]};
  __syncthreads();
  for (int idx = tid; idx < G * D; idx += 64 * W) {
    const int h = idx / D, d = idx % D;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < W; ++w) M = fmaxf(M, sm_m[w][h]);
    const float Mu = M == -INFINITY ? 0.f : M;
    float L = 0.f, O = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float sc = fast_exp2(sm_m[w][h] - Mu);
      L += sm_l[w][h] * sc;
      O += (w < 2 ? so_e[w] : so_o[w - 2])[h][d] * sc;
    }
    const int64_t slot = static_cast<int64_t>(slot_out) * p.d.num_heads + h0 + h;
    const bool some = KEEP_NAN ? L != 0.f : L > 0.f;
    global_ptr(p.d.ws_o)[slot * D + d] = some ? O / L : 0.f;
    if (d == 0) global_ptr(p.d.ws_lse)[slot] = some ? M * kLn2 + __logf(L) : -INFINITY;
  }
}

// The batch is cut as for decode_paged_kernel, a share at least one chunk for each
// wave.  At 64 columns four workgroups fit a CU (64 x 16k-32k keys of 14 / 2 x 64:
// 55 -> 51 us), but the second two pay only from two chunks for each wave on (16 x
// 1k-8k: 12.3 us, 15.0 with all of them).
template <int D, typename T, bool KEEP_NAN>
__global__ __launch_bounds__(256, D == 64 ? 4 : 2) void decode_fp4_kernel(PagedDecParams p) {
  constexpr int W = 4;
  __shared__ __attribute__((aligned(1024))) char bufE[W][2 * Fp4Tile<D>::BYTES];
  __shared__ __attribute__((aligned(1024))) char bufO[W][2 * Fp4Tile<D>::BYTES];
  __shared__ float sm_m[W][16], sm_l[W][16];
  __shared__ int sm_len[kDecMaxSeqs], sm_all[kDecMaxSeqs];  // keys seen, in the cache (-1: not run)
  __shared__ int sm_w[2][W];
  __shared__ int sm_cut[4];
  int kvh;
  int64_t item;
  if (!xcd_remap(blockIdx.x, static_cast<int64_t>(p.d.num_wgs) * p.d.head_chunks,
                 p.d.num_kv_heads, &kvh, &item))
    return;
  const int chunk = static_cast<int>(item % p.d.head_chunks);
  const int wg = static_cast<int>(item / p.d.head_chunks);
  auto first_chunk = [](int all, int len) { return (all - len) & ~31; };
  paged_shares<64 * W, 8, 4, D == 64 ? 2 : 1, true>(
      p, wg, sm_len, sm_all, sm_w, sm_cut, [&](int all, int len) {
        return len > 0 ? (all - first_chunk(all, len) + 31) >> 5 : 0;
      });
  const int r0 = __builtin_amdgcn_readfirstlane(sm_cut[0]);
  const int o0 = __builtin_amdgcn_readfirstlane(sm_cut[1]);
  const int r1 = r0 < 0 ? -2 : __builtin_amdgcn_readfirstlane(sm_cut[2]);  // -1, -2: no share
  const int o1 = __builtin_amdgcn_readfirstlane(sm_cut[3]);
  for (int r = r0; r <= r1; ++r) {
    const int len = __builtin_amdgcn_readfirstlane(sm_len[r]);
    if (len <= 0) continue;
    const int all = __builtin_amdgcn_readfirstlane(sm_all[r]);
    const int base = first_chunk(all, len), c = (all - base + 31) >> 5;
    const int b = r == r0 ? o0 : 0, e = r == r1 ? o1 : c;
    if (b >= e) continue;
    if (kvh == 0 && chunk == 0 && threadIdx.x == 0) {
      if (b == 0) global_ptr(p.seq_slots)[2 * r] = wg + r;
      if (e == c) global_ptr(p.seq_slots)[2 * r + 1] = wg + r;
    }
    const int end = base + 32 * e;
    fp4_split_body<D, T, KEEP_NAN>(p, kvh, chunk, wg + r, r, all - len, all, base + 32 * b,
                                   end < all ? end : all, bufE, bufO, sm_m, sm_l);
    __syncthreads();  // this split has been combined out of the buffers
  }
  // the reduce goes by the slots alone: a sequence without keys says so
  if (wg == 0 && kvh == 0 && chunk == 0) {
    for (int r = threadIdx.x; r < p.num_seqs; r += 64 * W) {
      if (sm_len[r] > 0) continue;
      global_ptr(p.seq_slots)[2 * r] = 0;
      global_ptr(p.seq_slots)[2 * r + 1] = sm_all[r] < 0 ? -2 : -1;
    }
  }
}

template <int D, typename T>
static hipError_t launch_fp4_t(const PagedDecParams& p, const RedParams& rp, int dtype,
                               hipStream_t st) {
  const int64_t grid = xcd_grid_size(static_cast<int64_t>(p.d.num_wgs) * p.d.head_chunks,
                                     p.d.num_kv_heads);
  const dim3 g(static_cast<unsigned>(grid)), b(256);
  if (p.d.keep_nan)
    hipLaunchKernelGGL((decode_fp4_kernel<D, T, true>), g, b, 0, st, p);
  else
    hipLaunchKernelGGL((decode_fp4_kernel<D, T, false>), g, b, 0, st, p);
  const hipError_t err = hipGetLastError();
  return err != hipSuccess ? err : launch_decode_reduce(rp, p.d.num_wgs, p.d.head_dim, dtype, st);
}

hipError_t launch_decode_fp4(const PagedDecParams& p, const RedParams& rp, int dtype,
                             hipStream_t st) {
  const bool bf = dtype == HCP_DTYPE_BF16;
  switch (padded_head_dim(p.d.head_dim)) {
    case 256:
      return bf ? launch_fp4_t<256, __bf16>(p, rp, dtype, st)
                : launch_fp4_t<256, _Float16>(p, rp, dtype, st);
    case 128:
      return bf ? launch_fp4_t<128, __bf16>(p, rp, dtype, st)
                : launch_fp4_t<128, _Float16>(p, rp, dtype, st);
    default:
      return bf ? launch_fp4_t<64, __bf16>(p, rp, dtype, st)
                : launch_fp4_t<64, _Float16>(p, rp, dtype, st);
  }
}

}  // namespace hcp
