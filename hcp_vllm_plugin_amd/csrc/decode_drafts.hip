// Split-KV decode of sequences with a few query tokens each (the newest one and
// those drafted behind it) over a paged cache of 16-bit or 4-bit values; lengths,
// row starts and block tables are read on the device.
//
// Token t of a sequence's n, all keys in the cache: hi = all - n + 1 + t, and
//   out = sum_j softmax_j(q . k_j * scale) v_j over hi - window <= j < hi.
//
// The n G rows of a KV head (token by token, G query heads each) are the columns
// of v_mfma_f32_16x16x32, RT tiles of 16 of them, so that a key is read from HBM
// once for all of them:
//   S^T = K Q^T, O^T = V^T P^T, the operands of K and V made once for all tiles.
// A workgroup takes an equal share of the batch's keys (paged_shares); its waves
// take the 32-key chunks of the share in turn, each through LDS of its own, where
// the next chunk lands while one is computed.  Chunks lie on multiples of 32
// positions, so that 16 keys lie in one block and are loaded with one descriptor
// of it: the cache's size does not matter, and rows past the sequence read as
// zeros.  The weights are held against a maximum that is raised only when a weight
// passes 2^8 (a row's sums and two 16-bit terms of P have room for that).  Q of more
// than 32 rows lies in LDS: in registers it would take half as many as O does.
//
// A value that a row does not see must not reach it, not even as 0 times a NaN.
// Only the chunks around the tokens' own positions (and a window's start) hold
// keys that some rows see and others do not: there infinities and NaN of V become
// zeros in LDS, and are added to the rows that see them when the waves are combined.
//
// Bound by HBM at long contexts: 64 x 5 tokens over 16k-32k keys, 28 / 4 heads of 128
// columns in bf16 (3.27 GB), 506 us and 7 to join, 6.4 TB/s; with the arithmetic left out
// it takes 513 in all.  After many launches in a row the clock falls, and with
// it the products' rate: 538.  A window of 4096 at 16 / 8 x 256 (502 MB) 86 us, 5.9
// TB/s.  Over the 4-bit cache the products and conversions bound it: 48 x 4 tokens over
// 8k-32k keys, 64 / 8 x 128 (907 MB), 200 us, 253 at the low clock, 167 without
// arithmetic.  24 x 1-6 tokens over 512-8192 keys (211 MB) 45 us, where the bytes take 32:
// what a split begins and ends with.  One sequence of 900 keys 10 us, waits all of them.
// Loading K one and a half chunks ahead, through LDS freed by the scores, was no faster
// (560 us for 550 of the first, on one card).
#include "decode_fp4.h"

namespace hcp {

#ifndef HCP_DRAFTS_FP4
#define HCP_DRAFTS_FP4 0  // 0: 16-bit caches, and the merge; 1: the 4-bit cache
#endif

constexpr int kDraftBufWord3 = 0x00020000;
constexpr int kDraftStreamAux = 2;  // non-temporal: read once per launch

// Keys lo .. lo + n - 1.
struct KeyRange {
  int lo;
  uint32_t n;
  __device__ __forceinline__ bool has(int key) const { return static_cast<uint32_t>(key - lo) < n; }
};

// ---- K and V of a chunk of a 16-bit cache ----
template <int D, typename T>
struct Keys16 {
  using E = Elem<T>;
  using V8 = typename E::vec8;
  static constexpr int NU = D / 16, QSTEPS = D / 32;
  static constexpr int ROWB = 2 * D, CPR = ROWB / 16;
  static constexpr int M = CPR < 16 ? CPR - 1 : 15;  // rows' 16-byte slots are XORed with row & M
  static constexpr int KPI = 1024 / ROWB;            // rows of a load
  static constexpr int OPT = 16 / KPI;               // loads of a tile's K (or V)
  static constexpr int CHB = 32 * ROWB;
  static constexpr int BYTES = 2 * CHB, LOADS = 4 * OPT;
  static constexpr int W = D == 256 ? 2 : 4;
  static constexpr int START = 8, LEAST = 2, LATE = 1;  // paged_shares; START of a tile

  const char *k, *v;
  const int32_t* bt;
  int64_t stride_block;
  int rowb, bs, bs_shift, all, dv;
  uint32_t id_max;
  int off[OPT];
  int lane, c16, g4;

  __device__ __forceinline__ void init(const DraftParams& p, int kvh, int r, int all_, int lane_) {
    const hcp_kv_segment& kv = p.p.kv;
    lane = lane_;
    c16 = lane & 15;
    g4 = lane >> 4;
    all = all_;
    dv = p.p.d.head_dim;
    k = reinterpret_cast<const char*>(kv.k_addr) + 2 * kvh * kv.stride_head;
    v = reinterpret_cast<const char*>(kv.v_addr) + 2 * kvh * kv.stride_head;
    stride_block = 2 * kv.stride_block;
    rowb = static_cast<int>(2 * kv.stride_tok);
    bs = kv.block_size;
    bs_shift = 31 - __builtin_clz(bs);
    id_max = static_cast<uint32_t>(kv.num_blocks) - 1;
    bt = global_ptr(reinterpret_cast<const int32_t*>(kv.block_table) +
                    static_cast<int64_t>(r) * p.p.bt_stride);
#pragma unroll
    for (int i = 0; i < OPT; ++i) off[i] = piece(i * KPI + lane / CPR);
  }
  // The 16-byte slot of a row that this lane fetches; past the row's dv columns it has to
  // read as zeros, as Q does there (the first slot's infinities would be NaN next to those):
  // a place past any descriptor's range.
  static constexpr int kPast = 0x7fffff00;
  __device__ __forceinline__ int slot(int row) const { return (lane % CPR) ^ (row & M); }
  __device__ __forceinline__ int piece(int row) const {
    return slot(row) < dv / 8 ? row * rowb + 16 * slot(row) : kPast;
  }

  __device__ __forceinline__ uint32_t fetch_ids(int x0) const {
    const int x = x0 + (lane & 32) / 2;
    return static_cast<uint32_t>(global_ptr(bt)[(x < all ? x : all - 1) >> bs_shift]);
  }
  __device__ __forceinline__ void issue(int x0, uint32_t ids, HCP_LDS_PTR(char) dst) const {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      uint32_t id = __builtin_amdgcn_readlane(ids, 32 * t);
      id = id < id_max ? id : id_max;  // past the cache: its last block
      const int x = x0 + 16 * t, rows = all - x;
      const int64_t o = id * stride_block + static_cast<int64_t>(x & (bs - 1)) * rowb;
      const int nrec = rows <= 0 ? 0 : ((rows < 16 ? rows : 16) - 1) * rowb + 2 * dv;
      const __amdgpu_buffer_rsrc_t rk =
          __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(k + o), 0, nrec, kDraftBufWord3);
      const __amdgpu_buffer_rsrc_t rv =
          __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(v + o), 0, nrec, kDraftBufWord3);
#pragma unroll
      for (int i = 0; i < OPT; ++i) {
        const int at = (t * OPT + i) * 1024;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, reinterpret_cast<HCP_LDS_PTR(void)>(dst + at),
                                                 16, off[i], 0, 0, kDraftStreamAux);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            rv, reinterpret_cast<HCP_LDS_PTR(void)>(dst + CHB + at), 16, off[i], 0, 0,
            kDraftStreamAux);
      }
    }
  }
  // The same from blocks of fewer than 16 keys: an id and an address for each row.
  __device__ __forceinline__ void issue_small(int x0, HCP_LDS_PTR(char) dst) const {
    const char *ka[2 * OPT], *va[2 * OPT];
#pragma unroll
    for (int j = 0; j < 2 * OPT; ++j) {
      const int row = j * KPI + lane / CPR;
      int x = x0 + row;
      x = x < all ? x : all - 1;  // past the sequence: its last key, which has no weight here
      uint32_t id = static_cast<uint32_t>(global_ptr(bt)[x >> bs_shift]);
      id = id < id_max ? id : id_max;
      const int c = slot(row & 15);
      const int64_t o = id * stride_block + static_cast<int64_t>(x & (bs - 1)) * rowb +
                        (c < dv / 8 ? 16 * c : 0);  // (clear_past)
      ka[j] = k + o;
      va[j] = v + o;
    }
#pragma unroll
    for (int j = 0; j < 2 * OPT; ++j) {
      __builtin_amdgcn_global_load_lds(
          reinterpret_cast<const __attribute__((address_space(1))) void*>(
              reinterpret_cast<uintptr_t>(ka[j])),
          reinterpret_cast<HCP_LDS_PTR(void)>(dst + j * 1024), 16, 0, kDraftStreamAux);
      __builtin_amdgcn_global_load_lds(
          reinterpret_cast<const __attribute__((address_space(1))) void*>(
              reinterpret_cast<uintptr_t>(va[j])),
          reinterpret_cast<HCP_LDS_PTR(void)>(dst + CHB + j * 1024), 16, 0, kDraftStreamAux);
    }
  }
  // Zeros in K past the rows' dv columns, once what issue_small loaded has landed.
  __device__ __forceinline__ void clear_past(HCP_LDS_PTR(char) dst) const {
    if (dv == D) return;
    asm volatile("" ::: "memory");  // (not ahead of the wait for them)
#pragma unroll
    for (int j = 0; j < 2 * OPT; ++j)
      if (slot((j * KPI + lane / CPR) & 15) >= dv / 8)
        *reinterpret_cast<HCP_LDS_PTR(u32x4)>(dst + j * 1024 + 16 * lane) = u32x4{0, 0, 0, 0};
  }
  // Q's 16-byte slot of k-step s
  __device__ __forceinline__ int q_slot(int s) const { return 4 * s + g4; }

  // f(s, operand) over the k-steps of tile t: row 16 t + c16, columns 32 s + 8 g4 ..
  template <typename F>
  __device__ __forceinline__ void k_operands(const HCP_LDS_PTR(char) src, int t, F f) const {
#pragma unroll
    for (int s = 0; s < QSTEPS; ++s)
      f(s, as_vec8<V8>(lds_at<u32x4>(src + (16 * t + c16) * ROWB +
                                     16 * ((4 * s + g4) ^ (c16 & M)))));
  }

  static constexpr int HALVES = NU == 16 ? 2 : 1, VW = NU == 4 ? 2 : 4;
  // Key j of 8 of this lane, relative to the chunk.
  __device__ __forceinline__ int v_key(int j) const { return 16 * (j >> 2) + 4 * g4 + (j & 3); }
  // Its words 4 h .. of columns NU c16 .. + NU - 1.
  __device__ __forceinline__ u32x4 v_words(const HCP_LDS_PTR(char) src, int j, int h) const {
    const int row = v_key(j);
    const HCP_LDS_PTR(char) const vrow = src + CHB + row * ROWB;
    if constexpr (NU == 16) return lds_at<u32x4>(vrow + 16 * ((2 * c16 + h) ^ (row & M)));
    if constexpr (NU == 8) return lds_at<u32x4>(vrow + 16 * (c16 ^ (row & M)));
    const u32x2 x = lds_at<u32x2>(vrow + 16 * ((c16 >> 1) ^ (row & M)) + 8 * (c16 & 1));
    return u32x4{x[0], x[1], 0, 0};
  }
  // Zeros in place of the infinities and NaN of a chunk's V; whether a key of the
  // range had one.
  __device__ __forceinline__ bool clean_v(HCP_LDS_PTR(char) src, int x0, KeyRange any) const {
    constexpr uint32_t kExp = __is_same(T, __bf16) ? 0x7f80u : 0x7c00u;
    bool odd = false;
#pragma unroll 1
    for (int at = 16 * lane; at < CHB; at += 1024) {
      u32x4 x = lds_at<u32x4>(src + CHB + at);
      bool bad = false;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        uint32_t keep = 0xffffffffu;
        if ((x[w] & kExp) == kExp) keep &= 0xffff0000u;
        if ((x[w] >> 16 & kExp) == kExp) keep &= 0xffffu;
        bad |= keep != 0xffffffffu;
        x[w] &= keep;
      }
      if (bad) *reinterpret_cast<HCP_LDS_PTR(u32x4)>(src + CHB + at) = x;
      odd |= bad && any.has(x0 + at / ROWB);
    }
    return odd;
  }
  // V of a key and column where it is an infinity or a NaN, else 0.
  __device__ __forceinline__ float odd_value(int key, int d) const {
    if (d >= dv) return 0.f;
    uint32_t id = static_cast<uint32_t>(global_ptr(bt)[key >> bs_shift]);
    id = id < id_max ? id : id_max;
    const float x = Elem<T>::to_float(*global_ptr(reinterpret_cast<const uint16_t*>(
        v + id * stride_block + static_cast<int64_t>(key & (bs - 1)) * rowb + 2 * d)));
    return fabsf(x) < INFINITY ? 0.f : x;
  }
  // f(u, operand) over columns NU row + u of V^T
  template <typename F>
  __device__ __forceinline__ void v_operands(const HCP_LDS_PTR(char) src, F f) const {
#pragma unroll
    for (int h = 0; h < HALVES; ++h) {
      u32x4 vc[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) vc[j] = v_words(src, j, h);
#pragma unroll
      for (int i = 0; i < 2 * VW; ++i) {
        u32x4 a;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          a[j] = __builtin_amdgcn_perm(vc[2 * j + 1][i >> 1], vc[2 * j][i >> 1],
                                       i & 1 ? 0x07060302u : 0x05040100u);
        f(2 * VW * h + i, as_vec8<V8>(a));
      }
    }
  }
  // Two 16-bit terms of a weight, positive both: products with an infinity stay it.
  static __device__ __forceinline__ void terms(float a, float b, uint32_t& hi, uint32_t& lo) {
    two_terms<T>(a, b, hi, lo);
  }
};

// ---- K and V of a chunk of the 4-bit cache: bytes, loads and operands as in
// decode_fp4_kernel ----
template <int D, typename T>
struct Keys4 {
  using E = Elem<T>;
  using V8 = typename E::vec8;
  using Tile = Fp4Tile<D>;
  static constexpr int NU = D / 16, QSTEPS = D / 32;
  static constexpr int BYTES = 2 * Tile::BYTES, LOADS = 2 * Tile::NI;
  static constexpr int W = 4;
  static constexpr int START = 8, LEAST = 4, LATE = D == 64 ? 2 : 1;

  const char* head;
  const int32_t* bt;
  int64_t stride_block;
  int bs, bs_shift, all, dv, ng, region, soff;
  uint32_t id_max, half;
  int koff[Tile::P], voff[Tile::P], kc_at[Tile::P], vc_at[Tile::P], ks_at[Tile::P], vs_at;
  int lane, c16, g4;

  __device__ __forceinline__ void init(const DraftParams& p, int kvh, int r, int all_, int lane_) {
    const hcp_kv_segment& kv = p.p.kv;
    lane = lane_;
    c16 = lane & 15;
    g4 = lane >> 4;
    all = all_;
    dv = p.p.d.head_dim;
    bs = kv.block_size;
    bs_shift = 31 - __builtin_clz(bs);
    id_max = static_cast<uint32_t>(kv.num_blocks) - 1;
    head = reinterpret_cast<const char*>(kv.k_addr) + kvh * kv.stride_head;
    stride_block = kv.stride_block;
    bt = global_ptr(reinterpret_cast<const int32_t*>(kv.block_table) +
                    static_cast<int64_t>(r) * p.p.bt_stride);
    half = c16 & 1 ? 0x07060302u : 0x05040100u;
    ng = dv / 32;
    const int vb = bs * (dv / 2);
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
        const int q = lane >> 2, e4 = lane & 3, e = c16 >> 1;
        key = 8 * i + (q >> 1);
        d0 = 128 * (q & 1) + 32 * (e4 ^ (key >> 1 & 3));
        quad = 2 * i + (q >> 3);
        oct = 4 * (q & 7) + (e4 ^ (q >> 2 & 1));
        kc_at[i] = (c16 >> 3) * 1024 + ((c16 & 7) * 2 + (g4 >> 1)) * 64 +
                   ((2 * (g4 & 1) + i) ^ (c16 >> 1 & 3)) * 16;
        vc_at[i] = 2048 + (g4 >> 1) * 1024 + ((g4 & 1) * 8 + e) * 64 +
                   ((2 * (c16 & 1) + i) ^ (e >> 2)) * 16;
      }
      koff[i] = key * (dv / 2) + (d0 < dv ? d0 / 2 : 0);
      voff[i] = vb + (quad * (dv / 8) + (oct < dv / 8 ? oct : 0)) * 16;
      if (D == 64 && lane >= 32) koff[i] = voff[i];
      const int g = D / 4 * g4 / 32 + i;
      ks_at[i] = Tile::SC + ((c16 >> 2) * ng + (g < ng ? g : 0)) * 4 + (c16 & 3);
    }
    const int si = lane & (Tile::SW - 1), sv = lane / Tile::SW & 1;
    soff = bs * dv + sv * bs * ng + (si < 4 * ng ? si : 0) * 4;
    region = static_cast<int>(Fp4Region{dv, bs}.bytes());
    const int vgrp = NU * c16 / 32;
    vs_at = Tile::SC + Tile::SW * 4 + (g4 * ng + (vgrp < ng ? vgrp : 0)) * 4;
  }

  __device__ __forceinline__ uint32_t fetch_ids(int x0) const {
    const int x = x0 + (lane & 32) / 2;
    return static_cast<uint32_t>(global_ptr(bt)[(x < all ? x : all - 1) >> bs_shift]);
  }
  __device__ __forceinline__ void issue_small(int, HCP_LDS_PTR(char)) const {}
  __device__ __forceinline__ void clear_past(HCP_LDS_PTR(char)) const {}
  __device__ __forceinline__ void issue(int x0, uint32_t ids, HCP_LDS_PTR(char) dst) const {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      uint32_t id = __builtin_amdgcn_readlane(ids, 32 * t);
      id = id < id_max ? id : id_max;
      const int at = (x0 + 16 * t) & (bs - 1);
      const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
          const_cast<char*>(head + id * stride_block), 0, x0 < all ? region : 0, kDraftBufWord3);
      auto load = [&](int to, int o, int so) __attribute__((always_inline)) {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            rs, reinterpret_cast<HCP_LDS_PTR(void)>(dst + t * Tile::BYTES + to), 16, o, so, 0,
            kDraftStreamAux);
      };
      const int row = at * (dv / 2);
#pragma unroll
      for (int i = 0; i < Tile::P; ++i) {
        load(i * 1024, koff[i], row);
        if constexpr (D > 64) load((Tile::P + i) * 1024, voff[i], row);
      }
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rs, reinterpret_cast<HCP_LDS_PTR(void)>(dst + t * Tile::BYTES + Tile::SC), 4, soff,
          at * ng, 0, kDraftStreamAux);
    }
  }
  __device__ __forceinline__ int q_slot(int s) const { return D / 32 * g4 + s; }

  template <typename F>
  __device__ __forceinline__ void k_operands(const HCP_LDS_PTR(char) src, int t, F f) const {
    const HCP_LDS_PTR(char) const tile = src + t * Tile::BYTES;
#pragma unroll
    for (int i = 0; i < Tile::P; ++i) {
      const float ks = __uint_as_float(static_cast<uint32_t>(lds_at<uint8_t>(tile + ks_at[i])) << 23);
      if constexpr (D == 64) {
        const u32x2 w = lds_at<u32x2>(tile + kc_at[0]);
#pragma unroll
        for (int q = 0; q < 2; ++q) f(q, as_vec8<V8>(fp4_values<T>(w[q], ks)));
      } else {
        const u32x4 w = lds_at<u32x4>(tile + kc_at[i]);
#pragma unroll
        for (int q = 0; q < 4; ++q) f(4 * i + q, as_vec8<V8>(fp4_values<T>(w[q], ks)));
      }
    }
  }

  // A scale of 0 (2^-127) in place of those of a chunk's V that are NaN, or of keys out of
  // the range; whether a key of the range had a NaN.
  __device__ __forceinline__ bool clean_v(HCP_LDS_PTR(char) src, int x0, KeyRange any) const {
    bool odd = false;
    if (lane < 8 * ng) {  // a dword: four keys of a tile, 32 columns
      const int t = lane >= 4 * ng, i = lane - 4 * ng * t, key = x0 + 16 * t + i / ng * 4;
      const HCP_LDS_PTR(char) const at = src + t * Tile::BYTES + Tile::SC + Tile::SW * 4 + 4 * i;
      const uint32_t w = lds_at<uint32_t>(at);
      uint32_t keep = w;
#pragma unroll 1
      for (int j = 0; j < 4; ++j) {
        const bool nan = (w >> (8 * j) & 255) == 255, in = any.has(key + j);
        if (nan || !in) keep &= ~(0xffu << (8 * j));
        odd |= nan && in;
      }
      if (keep != w) *reinterpret_cast<HCP_LDS_PTR(uint32_t)>((HCP_LDS_PTR(char))at) = keep;
    }
    return odd;
  }
  __device__ __forceinline__ float odd_value(int key, int d) const {
    if (d >= dv) return 0.f;
    uint32_t id = static_cast<uint32_t>(global_ptr(bt)[key >> bs_shift]);
    id = id < id_max ? id : id_max;
    const uint8_t scale = *global_ptr(reinterpret_cast<const uint8_t*>(
        head + id * stride_block + Fp4Region{dv, bs}.v_scale(key & (bs - 1), d >> 5)));
    return scale == 255 ? __builtin_nanf("") : 0.f;
  }
  template <typename F>
  __device__ __forceinline__ void v_operands(const HCP_LDS_PTR(char) src, F f) const {
    float vs[8];
    u32x4 vw[2][Tile::P];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint32_t w = lds_at<uint32_t>(src + t * Tile::BYTES + vs_at);
      vs[4 * t] = fp4_scale_of<0>(w);
      vs[4 * t + 1] = fp4_scale_of<1>(w);
      vs[4 * t + 2] = fp4_scale_of<2>(w);
      vs[4 * t + 3] = fp4_scale_of<3>(w);
#pragma unroll
      for (int i = 0; i < Tile::P; ++i)
        vw[t][i] = lds_at<u32x4>(src + t * Tile::BYTES + vc_at[i]);
      if constexpr (D == 64) {
        // a lane's two of the four bytes, of two keys in one dword
#pragma unroll
        for (int j = 0; j < 2; ++j)
          vw[t][0][j] = __builtin_amdgcn_perm(vw[t][0][2 * j + 1], vw[t][0][2 * j], half);
      }
    }
    // columns 2 u and 2 u + 1 of 8 keys -> two operands
    auto two = [&](auto sel, auto piece, int u) __attribute__((always_inline)) {
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
      f(2 * u, as_vec8<V8>(a));
      f(2 * u + 1, as_vec8<V8>(b));
    };
    using I0 = std::integral_constant<int, 0>;
    using I1 = std::integral_constant<int, 1>;
    using I2 = std::integral_constant<int, 2>;
    using I3 = std::integral_constant<int, 3>;
    two(I0{}, I0{}, 0);
    two(I1{}, I0{}, 1);
    if constexpr (D > 64) {
      two(I2{}, I0{}, 2);
      two(I3{}, I0{}, 3);
    }
    if constexpr (D > 128) {
      two(I0{}, I1{}, 4);
      two(I1{}, I1{}, 5);
      two(I2{}, I1{}, 6);
      two(I3{}, I1{}, 7);
    }
  }
  static __device__ __forceinline__ void terms(float a, float b, uint32_t& hi, uint32_t& lo) {
    split_weights<T>(a, b, hi, lo);
  }
};

// One split: keys [kb, ke) of sequence r for rows [16 RT chunk, ..) of a KV head.
template <template <int, typename> class Keys, int D, typename T, int RT>
__device__ __forceinline__ void drafts_split_body(
    const DraftParams& p, int kvh, int chunk, int slot, int r, int row0, int n, int first, int all,
    int kb, int ke, char (*bufE)[Keys<D, T>::BYTES], char (*bufO)[Keys<D, T>::BYTES], char* sm_q_,
    float (*sm_m)[16 * RT], float (*sm_l)[16 * RT], int* sm_odd) {
  using E = Elem<T>;
  using V8 = typename E::vec8;
  using K = Keys<D, T>;
  constexpr int W = K::W, NU = K::NU, QSTEPS = K::QSTEPS;
  constexpr int CPR = D / 8, QM = CPR < 16 ? CPR - 1 : 15;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c16 = lane & 15, g4 = lane >> 4;
  const int G = p.p.d.group, rows = n * G, rho0 = 16 * RT * chunk;
  const int window = p.window;

  K keys;
  keys.init(p, kvh, r, all, lane);
  HCP_LDS_PTR(char) const be = (HCP_LDS_PTR(char))(bufE[wave]);
  HCP_LDS_PTR(char) const bo = (HCP_LDS_PTR(char))(bufO[wave]);

  // The wave's chunks, kb + 32 (wave, wave + W, ..).  The first one's bytes are on their
  // way while Q is fetched.
  constexpr int ST = 32 * W;
  int x = kb + 32 * wave;
  const bool some = x < ke;
  const int last = x + (ke - 1 - x) / ST * ST;
  auto upto = [&](int y) __attribute__((always_inline)) { return y < last ? y : last; };
  auto next = [&]() __attribute__((always_inline)) { return x + ST <= last ? x + ST : all; };
#if HCP_DRAFTS_FP4
  constexpr bool small = false;
#else
  const bool small = p.p.kv.block_size < 16;
#endif
  uint32_t ia = 0, ib = 0;
  if (some) {
    if (small) {
      keys.issue_small(x, be);
    } else {
      ia = keys.fetch_ids(x);
      ib = keys.fetch_ids(upto(x + ST));
      keys.issue(x, ia, be);
    }
  }

  // Q of up to 32 rows goes to registers (through bufO, not loaded into yet)
  constexpr bool kHold = RT * QSTEPS <= 8;
  static_assert(!kHold || 16 * RT * 2 * D <= W * K::BYTES, "staging of Q");
  char* const sm_q = kHold ? &bufO[0][0] : sm_q_;
  HCP_LDS_PTR(char) const qs = (HCP_LDS_PTR(char))sm_q;
  // a row's 16-byte slots XORed with it
  for (int i = tid; i < 16 * RT * CPR; i += 64 * W) {
    const int row = i / CPR, c = i % CPR, rho = rho0 + row;
    const int t = rho / G, g = rho - t * G;
    u32x4 x{0, 0, 0, 0};
    if (rho < rows && 8 * c < p.p.d.head_dim)
      x = ldg16(reinterpret_cast<const char*>(p.p.d.q) +
                ((static_cast<int64_t>(row0) + t) * p.p.d.q_stride_tok +
                 static_cast<int64_t>(kvh * G + g) * p.p.d.q_stride_head) * 2 + 16 * c);
    *reinterpret_cast<u32x4*>(sm_q + row * 2 * D + 16 * (c ^ (row & QM))) = x;
  }
  // keys that this lane's row of each tile sees; none for rows past the last
  KeyRange see[RT];
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    const int rho = rho0 + 16 * i + c16;
    const int hi = rho < rows ? all - n + 1 + rho / G : 0;
    see[i].lo = window > 0 && hi > window ? hi - window : 0;
    see[i].n = hi > 0 ? hi - see[i].lo : 0;
  }
  // chunks that reach past `edge_hi`, or begin before `edge_lo`, hold keys that not
  // every token sees
  const int edge_hi = all - n + 1, edge_lo = window > 0 ? all - window : 0;
  const KeyRange any{first, static_cast<uint32_t>(all - first)};
  if (tid == 0) *sm_odd = 0;
  __syncthreads();

  V8 qf[kHold ? RT : 1][kHold ? QSTEPS : 1];
  auto q_at = [&](int i, int s) __attribute__((always_inline)) {
    return as_vec8<V8>(lds_at<u32x4>(qs + (16 * i + c16) * 2 * D +
                                     16 * (keys.q_slot(s) ^ (c16 & QM))));
  };
  if constexpr (kHold) {
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int s = 0; s < QSTEPS; ++s) qf[i][s] = q_at(i, s);
    __syncthreads();
  }

  const float c = p.p.d.scale_log2;
  const float most = __builtin_exp2f(kRaise + kLift<T>);
  // of each tile: -(running maximum, kLift below), 0 before the first; the weight past
  // which it is raised; the sum of this lane's weights
  float neg_m[RT], limit[RT], lsum[RT];
  f32x4 oacc[RT][NU];
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    neg_m[i] = 0.f;
    limit[i] = -1.f;
    lsum[i] = 0.f;
#pragma unroll
    for (int u = 0; u < NU; ++u) oacc[i][u] = f32x4{};
  }

  auto compute = [&](int x0, HCP_LDS_PTR(char) src) __attribute__((always_inline)) {
    const bool edge = x0 + 32 > edge_hi || x0 < edge_lo;
    f32x4 s[RT][2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int i = 0; i < RT; ++i) s[i][t] = f32x4{};
      keys.k_operands(src, t, [&](int st, V8 a) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < RT; ++i) {
          if constexpr (kHold)
            s[i][t] = E::mfma16(a, qf[i][st], s[i][t]);
          else
            s[i][t] = E::mfma16(a, q_at(i, st), s[i][t]);
        }
      });
    }
    if (edge) {
      // (opaque: the comparisons are made here, not ahead of the branch for every chunk)
      int at = x0 + 4 * g4;
      asm volatile("" : "+v"(at));
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (!see[i].has(at + 16 * t + j)) s[i][t][j] = -INFINITY;
          // (a few masks at a time: many would push the loop's scalars out of their registers)
          __builtin_amdgcn_sched_barrier(0);
        }
      if (keys.clean_v(src, x0, any)) *sm_odd = 1;
    }
    V8 pf[RT], rf[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      float w[2][4];
      auto weights = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int j = 0; j < 4; ++j) w[t][j] = fast_exp2(__builtin_fmaf(s[i][t][j], c, neg_m[i]));
      };
      weights();
      const float top = fmaxf(fmaxf(fmaxf(w[0][0], w[0][1]), fmaxf(w[0][2], w[0][3])),
                              fmaxf(fmaxf(w[1][0], w[1][1]), fmaxf(w[1][2], w[1][3])));
      if (__builtin_amdgcn_ballot_w64(top > limit[i]) != 0) {
        float mx = fmaxf(fmaxf(fmaxf(s[i][0][0], s[i][0][1]), fmaxf(s[i][0][2], s[i][0][3])),
                         fmaxf(fmaxf(s[i][1][0], s[i][1][1]), fmaxf(s[i][1][2], s[i][1][3]))) * c;
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        const float m_old = limit[i] < 0.f ? -INFINITY : -neg_m[i];
        const float m_new = fmaxf(m_old, mx - kLift<T>);
        neg_m[i] = m_new == -INFINITY ? 0.f : -m_new;
        limit[i] = m_new == -INFINITY ? -1.f : most;
        const float alpha = fast_exp2(m_old + neg_m[i]);
        lsum[i] *= alpha;
#pragma unroll
        for (int u = 0; u < NU; ++u) oacc[i][u] *= alpha;
        weights();
      }
      u32x4 pw, rw;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          uint32_t hi, lo;
          K::terms(w[t][2 * j], w[t][2 * j + 1], hi, lo);
          pw[2 * t + j] = hi;
          rw[2 * t + j] = lo;
        }
      pf[i] = as_vec8<V8>(pw);
      rf[i] = as_vec8<V8>(rw);
      lsum[i] += ((w[0][0] + w[0][1]) + (w[0][2] + w[0][3])) +
                 ((w[1][0] + w[1][1]) + (w[1][2] + w[1][3]));
    }
    auto pv = [&](int u, V8 a) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        oacc[i][u] = E::mfma16(a, pf[i], oacc[i][u]);
        oacc[i][u] = E::mfma16(a, rf[i], oacc[i][u]);
      }
    };
    keys.v_operands(src, pv);
  };

  // The block ids of the chunk after the next are fetched, the next one's bytes
  // loaded, and when only those are outstanding the current one has landed.  (Loads
  // without a branch around them, or the compiler's own waits for the ids would be for
  // everything: past the last chunk they are out of their descriptor's range and fetch
  // nothing.  Repeating the last chunk, as a single-token split does, cost 24 sequences of
  // 0.5k-8k keys 2 us.)  With K's buffer filled again as soon as the scores are made, half
  // a chunk more on its way, 64 x 16k-32k keys took no less (560 us for 550).
  if (some && !small) {
    while (true) {
      ia = keys.fetch_ids(upto(x + 2 * ST));
      __builtin_amdgcn_sched_barrier(0);
      keys.issue(next(), ib, bo);
      wait_vmcnt<K::LOADS + 1>();
      compute(x, be);
      x += ST;
      if (x > last) break;
      ib = keys.fetch_ids(upto(x + 2 * ST));
      __builtin_amdgcn_sched_barrier(0);
      keys.issue(next(), ia, be);
      wait_vmcnt<K::LOADS + 1>();
      compute(x, bo);
      x += ST;
      if (x > last) break;
    }
  } else if (some) {
    for (; x <= last; x += ST) {
      wait_vmcnt<0>();
      keys.clear_past(be);
      compute(x, be);
      keys.issue_small(upto(x + ST), be);
    }
  }

  // ---- combine the W waves, a tile at a time in the chunk buffers ----
  wait_vmcnt<0>();  // the last loads still write there
  const DraftParams& po = fresh_params<DraftParams>();  // (not held across the loop)
  // (all of them in bufO where there is room)
  constexpr int HW = sizeof(float) * W * 16 * (D + 4) <= W * K::BYTES ? 0 : W / 2;
  static_assert(sizeof(float) * (W - HW) * 16 * (D + 4) <= W * K::BYTES, "combine staging");
  float (*const so_e)[16][D + 4] = reinterpret_cast<float (*)[16][D + 4]>(&bufE[0][0]);
  float (*const so_o)[16][D + 4] = reinterpret_cast<float (*)[16][D + 4]>(&bufO[0][0]);
  float (*const mine)[D + 4] = wave < HW ? so_e[wave] : so_o[wave - HW];
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    float l = lsum[i] + __shfl_xor(lsum[i], 16);
    l += __shfl_xor(l, 32);
    __syncthreads();
    if (g4 == 0) {
      sm_m[wave][16 * i + c16] = limit[i] < 0.f ? -INFINITY : -neg_m[i];
      sm_l[wave][16 * i + c16] = l;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int u = 0; u < NU; u += 4)
        *reinterpret_cast<f32x4*>(&mine[c16][NU * (4 * g4 + j) + u]) =
            f32x4{oacc[i][u][j], oacc[i][u + 1][j], oacc[i][u + 2][j], oacc[i][u + 3][j]};
    __syncthreads();
    for (int idx = tid; idx < 16 * (D / 4); idx += 64 * W) {
      const int h = idx / (D / 4), d = idx % (D / 4) * 4, rho = rho0 + 16 * i + h;
      if (rho >= rows) break;
      float mw[W], M = -INFINITY;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        mw[w] = sm_m[w][16 * i + h];
        M = fmaxf(M, mw[w]);
      }
      const float Mu = M == -INFINITY ? 0.f : M;
      float L = 0.f;
      f32x4 O{};
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float sc = fast_exp2(mw[w] - Mu);
        L += sm_l[w][16 * i + h] * sc;
        O += *reinterpret_cast<const f32x4*>(&(w < HW ? so_e[w] : so_o[w - HW])[h][d]) * sc;
      }
      const int t = rho / G, hq = kvh * G + rho - t * G;
      if (*sm_odd) {  // what clean_v took out, for the rows that see it
        const int hi = all - n + 1 + t, lo = window > 0 ? hi - window : 0;
        for (int x0 = kb; x0 < ke; x0 += 32) {
          if (!(x0 + 32 > edge_hi || x0 < edge_lo)) continue;
          for (int key = x0 > lo ? x0 : lo; key < x0 + 32 && key < hi; ++key)
            for (int j = 0; j < 4; ++j) O[j] += keys.odd_value(key, d + j);
        }
      }
      const int64_t at = (static_cast<int64_t>(slot) * po.max_tokens + t) * po.p.d.num_heads + hq;
      const bool some = L != 0.f;  // a NaN too: it is the row's result
      const float inv = some ? 1.f / L : 0.f;
      *global_ptr(reinterpret_cast<f32x4*>(po.p.d.ws_o + at * D + d)) = some ? O * inv : f32x4{};
      if (d == 0) global_ptr(po.p.d.ws_lse)[at] = some ? M * kLn2 + __logf(L) : -INFINITY;
    }
  }
}

// Rows of sequence r that are run, and the first: none past q's or max_tokens.
__device__ __forceinline__ int draft_rows(const DraftParams& p, int64_t a, int64_t b, int& row0) {
  if (a < 0 || a >= p.q_rows || b <= a) return 0;
  row0 = static_cast<int>(a);
  int64_t n = b - a;
  n = n < p.max_tokens ? n : p.max_tokens;
  return static_cast<int>(n < p.q_rows - a ? n : p.q_rows - a);
}
__device__ __forceinline__ int64_t draft_start(const DraftParams& p, int r) {
  return p.p.lens_wide ? global_ptr(reinterpret_cast<const int64_t*>(p.row_starts))[r]
                       : global_ptr(reinterpret_cast<const int32_t*>(p.row_starts))[r];
}

template <template <int, typename> class Keys, int D, typename T, int RT>
__global__ __attribute__((amdgpu_flat_work_group_size(64 * Keys<D, T>::W, 64 * Keys<D, T>::W),
                          amdgpu_waves_per_eu(drafts_per_cu(HCP_DRAFTS_FP4, D, RT)))) void
decode_drafts_kernel(DraftParams p) {
  using K = Keys<D, T>;
  constexpr int W = K::W, NT = 64 * W, EPT = kDecMaxSeqs / NT;
  __shared__ __attribute__((aligned(1024))) char bufE[W][K::BYTES];
  __shared__ __attribute__((aligned(1024))) char bufO[W][K::BYTES];
  __shared__ __attribute__((aligned(16))) char sm_q[RT * K::QSTEPS <= 8 ? 16 : 16 * RT * 2 * D];
  __shared__ float sm_m[W][16 * RT], sm_l[W][16 * RT];
  __shared__ int sm_len[kDecMaxSeqs], sm_all[kDecMaxSeqs];  // keys seen, in the cache (-1: not run)
  __shared__ int sm_row0[kDecMaxSeqs];    // rows that are run: the first, their number
  __shared__ uint8_t sm_n[kDecMaxSeqs];
  __shared__ int sm_w[2][W];
  __shared__ int sm_cut[4], sm_odd;
  int kvh_;
  int64_t item;
  if (!xcd_remap(blockIdx.x, static_cast<int64_t>(p.p.d.num_wgs) * p.p.d.head_chunks,
                 p.p.d.num_kv_heads, &kvh_, &item))
    return;
  const int kvh = __builtin_amdgcn_readfirstlane(kvh_);
  const int chunk = __builtin_amdgcn_readfirstlane(static_cast<int>(item % p.p.d.head_chunks));
  const int wg = __builtin_amdgcn_readfirstlane(static_cast<int>(item / p.p.d.head_chunks));
  // the row starts of this thread's sequences, on their way with the lengths
  int64_t starts[EPT + 1];
  paged_lens(p.row_starts, p.p.lens_wide, threadIdx.x * EPT, p.p.num_seqs + 1, starts);
  auto first_chunk = [](int all, int len) { return (all - len) & ~31; };
  paged_shares<NT, K::START * RT, K::LEAST, K::LATE, false>(
      p.p, wg, sm_len, sm_all, sm_w, sm_cut,
      [&](int all, int len) { return len > 0 ? (all - first_chunk(all, len) + 31) >> 5 : 0; },
      [&](const PagedDecParams&, int j, int& all, int) __attribute__((always_inline)) {
        int row0;
        const int n = draft_rows(p, starts[j], starts[j + 1], row0);
        if (n == 0) return 0;
        sm_row0[threadIdx.x * EPT + j] = row0;
        sm_n[threadIdx.x * EPT + j] = static_cast<uint8_t>(n);
        // (keys of tokens that are not run are behind those that are)
        const int64_t rest = starts[j + 1] - starts[j] - n;
        all = rest < all ? all - static_cast<int>(rest) : 0;
        const uint32_t reach = static_cast<uint32_t>(p.window) + n - 1;  // of the first token's window
        return p.window > 0 && static_cast<uint32_t>(all) > reach ? static_cast<int>(reach) : all;
      });
  const int r0 = __builtin_amdgcn_readfirstlane(sm_cut[0]);
  const int o0 = __builtin_amdgcn_readfirstlane(sm_cut[1]);
  const int r1 = r0 < 0 ? -2 : __builtin_amdgcn_readfirstlane(sm_cut[2]);  // -1, -2: no share
  const int o1 = __builtin_amdgcn_readfirstlane(sm_cut[3]);
  for (int r = r0; r <= r1; ++r) {
    const DraftParams& p = fresh_params<DraftParams>();
    const int len = __builtin_amdgcn_readfirstlane(sm_len[r]);
    if (len <= 0) continue;
    const int all = __builtin_amdgcn_readfirstlane(sm_all[r]);
    const int base = first_chunk(all, len), c = (all - base + 31) >> 5;
    const int b = r == r0 ? o0 : 0, e = r == r1 ? o1 : c;
    if (b >= e) continue;
    if (kvh == 0 && chunk == 0 && threadIdx.x == 0) {
      if (b == 0) global_ptr(p.p.seq_slots)[2 * r] = wg + r;
      if (e == c) global_ptr(p.p.seq_slots)[2 * r + 1] = wg + r;
    }
    const int n = __builtin_amdgcn_readfirstlane(sm_n[r]);
    if (16 * RT * chunk >= n * p.p.d.group) continue;  // this chunk of rows is empty
    const int row0 = __builtin_amdgcn_readfirstlane(sm_row0[r]);
    const int end = base + 32 * e;
    drafts_split_body<Keys, D, T, RT>(p, kvh, chunk, wg + r, r, row0, n, all - len, all,
                                      base + 32 * b, end < all ? end : all, bufE, bufO, sm_q, sm_m,
                                      sm_l, &sm_odd);
    __syncthreads();  // this split has been combined out of the buffers
  }
  // the merge goes by the slots: a sequence without keys says so
  if (wg == 0 && kvh == 0 && chunk == 0) {
    for (int r = threadIdx.x; r < p.p.num_seqs; r += NT) {
      if (sm_len[r] > 0) continue;
      global_ptr(p.p.seq_slots)[2 * r] = 0;
      global_ptr(p.p.seq_slots)[2 * r + 1] = sm_all[r] < 0 ? -2 : -1;
    }
  }
}

template <template <int, typename> class Keys, int D, typename T>
static hipError_t launch_drafts_t(const DraftParams& p, int tiles, hipStream_t st) {
  const dim3 g(static_cast<unsigned>(xcd_grid_size(
      static_cast<int64_t>(p.p.d.num_wgs) * p.p.d.head_chunks, p.p.d.num_kv_heads)));
  const dim3 b(64 * Keys<D, T>::W);
  if (tiles == 1)
    hipLaunchKernelGGL((decode_drafts_kernel<Keys, D, T, 1>), g, b, 0, st, p);
  else if (tiles == 2)
    hipLaunchKernelGGL((decode_drafts_kernel<Keys, D, T, 2>), g, b, 0, st, p);
  else if constexpr (D < 256) {
    if (tiles == 3)
      hipLaunchKernelGGL((decode_drafts_kernel<Keys, D, T, 3>), g, b, 0, st, p);
    else
      hipLaunchKernelGGL((decode_drafts_kernel<Keys, D, T, 4>), g, b, 0, st, p);
  }
  return hipGetLastError();
}

template <template <int, typename> class Keys>
static hipError_t launch_drafts_d(const DraftParams& p, int tiles, int dtype, hipStream_t st) {
  const bool bf = dtype == HCP_DTYPE_BF16;
  switch (padded_head_dim(p.p.d.head_dim)) {
    case 256:
      return bf ? launch_drafts_t<Keys, 256, __bf16>(p, tiles, st)
                : launch_drafts_t<Keys, 256, _Float16>(p, tiles, st);
    case 128:
      return bf ? launch_drafts_t<Keys, 128, __bf16>(p, tiles, st)
                : launch_drafts_t<Keys, 128, _Float16>(p, tiles, st);
    default:
      return bf ? launch_drafts_t<Keys, 64, __bf16>(p, tiles, st)
                : launch_drafts_t<Keys, 64, _Float16>(p, tiles, st);
  }
}

#if HCP_DRAFTS_FP4
hipError_t launch_drafts_fp4(const DraftParams& p, int tiles, int dtype, hipStream_t st) {
  return launch_drafts_d<Keys4>(p, tiles, dtype, st);
}
#else
hipError_t launch_drafts16(const DraftParams& p, int tiles, int dtype, hipStream_t st) {
  return launch_drafts_d<Keys16>(p, tiles, dtype, st);
}

// Merge of a row's partials, a wave to HW heads of a (sequence, token): out = sum_i w_i
// O_i / sum_i w_i, w_i = exp(lse_i - max).  Lane B h + i holds weight i of head h, and
// every lane D / 64 columns of each head.  Bound by latency: the row's place and slots are
// fetched at once, then the LSEs with the first partials' columns, before any weight is
// known.  Four heads to a wave where there are more rows than the machine holds waves at
// once (48 x 4 rows of 64 heads 6.5 us, 12 with one), one where there are few with many
// partials (9 x 8 rows of 14 heads 4.3 us, 6.7 with four).
template <int D, typename T, int HW>
__global__ __launch_bounds__(256) void drafts_reduce_kernel(DraftParams p, DraftOut o) {
  constexpr int N = D / 64, B = 64 / HW, U = 16 / HW;  // partials of a batch, fetched at once
  typedef float vf __attribute__((ext_vector_type(N == 1 ? 2 : N)));  // (of one: its first)
  const int lane = threadIdx.x & 63, sub = lane / B, mine = lane % B;
  const int heads = p.p.d.num_heads, hgs = (heads + HW - 1) / HW;
  const int unit = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
  const int st = unit / hgs, head = (unit - st * hgs) * HW;
  const int seq = st / p.max_tokens, t = st - seq * p.max_tokens;
  if (seq >= p.p.num_seqs) return;
  const int64_t from = draft_start(p, seq), to = draft_start(p, seq + 1);
  // kept inside the workspace whatever stands there: a caller that changes the lengths
  // while the split kernel reads them leaves pairs unwritten
  const int a = p.p.seq_slots[2 * seq], z = p.p.seq_slots[2 * seq + 1];
  int row0 = 0;
  if (t >= draft_rows(p, from, to, row0)) return;
  const int p0 = a < 0 ? 0 : a < p.num_slots ? a : p.num_slots;
  const int n = (z < -2 ? -2 : z < p.num_slots ? z : p.num_slots - 1) - p0 + 1;
  if (n < 0) return;  // not run
  const int64_t step = static_cast<int64_t>(p.max_tokens) * heads;
  const int64_t at = (static_cast<int64_t>(p0) * p.max_tokens + t) * heads + head;
  const float* lcol = p.p.d.ws_lse + at;
  const float* ocol = p.p.d.ws_o + at * D + N * lane;
  const int have = heads - head < HW ? heads - head : HW;
  auto column = [&](int64_t i, int h) __attribute__((always_inline)) {
    const float* c = ocol + (i * step + (h < have ? h : 0)) * D;
    vf x;
    if constexpr (N == 1)
      x = vf{*global_ptr(c), 0.f};
    else
      x = *global_ptr(reinterpret_cast<const vf*>(c));
    return x;
  };
  auto lane_of = [&](float x, int l) __attribute__((always_inline)) {
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), l));
  };
  float m = -INFINITY, S = 0.f;  // of this lane's head
  vf O[HW] = {};
  for (int i0 = 0; i0 < n; i0 += B) {
    const int some = n - i0 < B ? n - i0 : B;
    const float l =
        mine < some && sub < have ? global_ptr(lcol)[(i0 + mine) * step + sub] : -INFINITY;
    vf v[U][HW];
    auto fetch = [&](int i) __attribute__((always_inline)) {
#pragma unroll
      for (int k = 0; k < U; ++k)
#pragma unroll
        for (int h = 0; h < HW; ++h) v[k][h] = column(i0 + (i + k < some ? i + k : some - 1), h);
    };
    fetch(0);
    // (the maximum leaves a NaN out: its weight is NaN whatever that is)
    float mn = l;
#pragma unroll
    for (int x = B / 2; x > 0; x >>= 1) mn = fmaxf(mn, __shfl_xor(mn, x));
    mn = fmaxf(m, mn);
    const float ref = mn == -INFINITY ? 0.f : mn;
    // (what came before, where a NaN may stand with m still -inf, is kept)
    const float sc = m == -INFINITY ? 1.f : __expf(m - ref);
    const float w = __expf(l - ref);
    float ws = w;
#pragma unroll
    for (int x = B / 2; x > 0; x >>= 1) ws += __shfl_xor(ws, x);
    S = S * sc + ws;
    m = mn;
#pragma unroll
    for (int h = 0; h < HW; ++h) O[h] *= lane_of(sc, B * h);
    for (int i = 0; i < some; i += U) {
      if (i > 0) fetch(i);
#pragma unroll
      for (int k = 0; k < U; ++k)
#pragma unroll
        for (int h = 0; h < HW; ++h) {
          const float wk = lane_of(w, (B * h + i + k) & 63);
          // (past the last: not summed, whatever its columns hold)
          O[h] = i + k < some ? O[h] + v[k][h] * wk : O[h];
        }
    }
  }
  const int64_t row = static_cast<int64_t>(row0) + t;
#pragma unroll
  for (int h = 0; h < HW; ++h) {
    if (h >= have) break;
    const float sum = lane_of(S, B * h);
    uint16_t* orow =
        reinterpret_cast<uint16_t*>(o.out) + row * o.stride_tok + (head + h) * o.stride_head;
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (N * lane + j < p.p.d.head_dim)
        orow[N * lane + j] = Elem<T>::from_float(sum != 0.f ? O[h][j] / sum : 0.f);
  }
  if (o.lse != nullptr && mine == 0 && sub < have)
    o.lse[(head + sub) * o.lse_stride_head + row] = S != 0.f ? m + __logf(S) : -INFINITY;
}

template <int D, typename T>
static void launch_drafts_reduce_t(const DraftParams& p, const DraftOut& o, hipStream_t st) {
  const int64_t rows = static_cast<int64_t>(p.p.num_seqs) * p.max_tokens, heads = p.p.d.num_heads;
  // (64 x 5 rows of 28 heads, 2048 keys: 63 us for the two launches with four heads to a wave, 66
  // with one; 16 x 5 31.3 and 31.8, 16 x 2 22.7 and 22.2, 1 x 5 24 and 20)
  const bool many = rows * heads > 2048;
  const int64_t units = rows * (many ? (heads + 3) / 4 : heads);
  const dim3 g(static_cast<unsigned>((units + 3) / 4)), b(256);
  if (many)
    hipLaunchKernelGGL((drafts_reduce_kernel<D, T, 4>), g, b, 0, st, p, o);
  else
    hipLaunchKernelGGL((drafts_reduce_kernel<D, T, 1>), g, b, 0, st, p, o);
}

hipError_t launch_drafts_reduce(const DraftParams& p, const DraftOut& o, int dtype, hipStream_t st) {
  const bool bf = dtype == HCP_DTYPE_BF16;
  switch (padded_head_dim(p.p.d.head_dim)) {
    case 256:
      bf ? launch_drafts_reduce_t<256, __bf16>(p, o, st)
         : launch_drafts_reduce_t<256, _Float16>(p, o, st);
      break;
    case 128:
      bf ? launch_drafts_reduce_t<128, __bf16>(p, o, st)
         : launch_drafts_reduce_t<128, _Float16>(p, o, st);
      break;
    default:
      bf ? launch_drafts_reduce_t<64, __bf16>(p, o, st)
         : launch_drafts_reduce_t<64, _Float16>(p, o, st);
      break;
  }
  return hipGetLastError();
}
#endif

}  // namespace hcp
