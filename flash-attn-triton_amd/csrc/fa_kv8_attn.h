// Attention of query rows against the paged KV cache held in 8 bits
// (fa_fwd_kvcache8): one token per sequence, a few, or chunks, batched or packed.
// The cache's layout and scales are described in fa_kv8.h.
//
// kv8_stream_kernel: launches of at most 32 query rows per sequence and K/V head
// (row r is query r / group of query head r % group, so that the heads sharing
// K/V share its bytes).  The launch is as many workgroups as fit the GPU at once,
// and each takes an equal stretch of the sequences' 32-key tiles in a row: the
// lengths are on the device, so every workgroup adds them up itself.  Its four
// waves take the tiles of a sequence in turn, without a barrier, and merge; a
// sequence within one stretch is written there, the pieces of the others are
// merged by kv8_combine_kernel.  S^T = K Q^T and O^T += V^T P^T run on 32x32
// matrix products, one query row per lane, with fp32 maximum, sum and output.
// What the 8 bits change:
//  * K and V tiles go global -> LDS as they are, by LDS-DMA into a ring of the
//    wave's own.  The block's power-of-two scale enters with the operand, in the
//    scaled 8-bit product (K, bf16 queries) or in v_cvt_scalef32_pk, which makes
//    16-bit operands (V, and K for fp16): a key's number times its scale is exact
//    in bf16 (and in fp16 within its range), and no score or probability is
//    rescaled.  LDS holds and moves half of what 16-bit tiles would.
//  * V^T comes from ds_read_b64_tr_b8: within 16 lanes, lanes 2r and 2r + 1 name
//    the 16 bytes of row r and lane i receives column i of the 8 rows, here the
//    8 keys whose probabilities the lane holds.
//  * Page numbers and scales of a wave's next 32 tiles are loaded together, one
//    lane per 16-key group, and handed to the scalar side by v_readlane: in the
//    loop nothing but the tile loads counts on the vector-memory counter, so
//    each wait names the tile it needs.
// Bound: HBM.  64 sequences of 512 to 8192 keys, Hq 32 Hk 8 D 128, bf16, e4m3:
// 119 us for 630 MB, 5.3 TB/s (126 us the call with its merge; 196 us for the
// 16-bit cache of these sizes); 131001 keys of one sequence, fp16: 50 us for 268 MB.
// Without the non-temporal hint on the tile loads 142 us for the first; a split of
// 2048 keys per workgroup instead of equal stretches 137 us.
// Keys past the sequence's end are never read: their bytes and scales may be
// anything.  Where the mask differs between the rows of a tile, a V number that
// is not finite would reach rows that do not see its key (0 * NaN); such tiles
// are looked through, and one that holds any adds those per row and column
// with a product of indicators.
#pragma once

#include <type_traits>

#include "fa_common.h"
#include "fa_kv8.h"

namespace fa {

constexpr int kKv8Waves = 4;
constexpr int kKv8BN = 32;            // keys of a tile of kv8_stream_kernel
constexpr int kKv8Own = 32;            // tiles of the longest stretch that holds one sequence only
constexpr float kKv8Slack = 8.f;      // a maximum is raised by more than this (log2 units) or not at all

// The 8-bit types.  bad(): the high bit of each byte of a word whose number is
// not finite.
struct E4M3 {
  static constexpr int kFormat = 0;   // of the scaled MFMA
  template <class T>
  __device__ static inline uint32_t cvt(uint32_t w, float scale, bool hi);
  __device__ static inline uint32_t bad(uint32_t w) {
    return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
  }
};
struct E5M2 {
  static constexpr int kFormat = 1;
  template <class T>
  __device__ static inline uint32_t cvt(uint32_t w, float scale, bool hi);
  __device__ static inline uint32_t bad(uint32_t w) {
    return ((w & 0x7c7c7c7cu) + 0x04040404u) & 0x80808080u;
  }
};
template <>
__device__ inline uint32_t E4M3::cvt<F16>(uint32_t w, float s, bool hi) {
  return hi ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, s, true))
            : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, s, false));
}
template <>
__device__ inline uint32_t E4M3::cvt<BF16>(uint32_t w, float s, bool hi) {
  return hi ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, true))
            : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, false));
}
template <>
__device__ inline uint32_t E5M2::cvt<F16>(uint32_t w, float s, bool hi) {
  return hi ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_bf8(w, s, true))
            : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_bf8(w, s, false));
}
template <>
__device__ inline uint32_t E5M2::cvt<BF16>(uint32_t w, float s, bool hi) {
  return hi ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(w, s, true))
            : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(w, s, false));
}

// Eight 8-bit numbers as a 16-bit MFMA operand.
template <class T, class F8>
__device__ inline u32x4 kv8_operand(uint32_t w0, uint32_t w1, float scale) {
  return u32x4{F8::template cvt<T>(w0, scale, false), F8::template cvt<T>(w0, scale, true),
               F8::template cvt<T>(w1, scale, false), F8::template cvt<T>(w1, scale, true)};
}

typedef int i32x2v __attribute__((__vector_size__(2 * sizeof(int))));
__device__ inline u32x2 lds_read_tr8(const uint8_t* p) {
  typedef __attribute__((address_space(3))) i32x2v lds_i32x2;
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2*)p));
}

// Where the 16-byte chunk c of row r of a tile sits in its LDS row: such that
// the 16 rows of a K read (one chunk each) and the 8 rows of a transposed V
// read (keys 0..3 and 8..11 of a 16-key step, two chunks each) touch distinct
// banks (256 bytes).
template <int D>
__device__ inline int kv8_k_chunk(int r, int c) {
  constexpr int kRowsPer = 256 / D;
  return c ^ ((r / kRowsPer) & (D / 16 - 1));
}
template <int D>
__device__ inline int kv8_v_chunk(int r, int c) {
  if constexpr (D == 256) return c ^ (((r & 3) | ((r >> 1) & 4)) << 1);
  else if constexpr (D == 128) return c ^ ((((r >> 1) & 1) | ((r >> 2) & 2)) << 1);
  else return c ^ (((r >> 3) & 1) << 1);
}

// The rows of a workgroup and the keys its sequence shows them.
struct Kv8Rows {
  int b, n;            // sequence, its queries
  int64_t q0;          // its first row of q (packed), 0 otherwise
  int L;               // its cached keys, clamped to [0, max_keys]
};
__device__ inline Kv8Rows kv8_rows(const Kv8AttnParams& p, int b) {
  Kv8Rows s;
  s.b = b;
  s.q0 = 0;
  s.n = p.seqlen_q;
  if (p.cu_q != nullptr) {
    // Offsets outside q would be read and written: an empty sequence instead.
    const int64_t a = p.cu_q[b], e = p.cu_q[b + 1];
    const bool ok = a >= 0 && e >= a && e <= p.total_q;
    s.q0 = ok ? a : 0;
    s.n = ok ? (int)min(e - a, (int64_t)p.seqlen_q) : 0;
  }
  const int L = p.seqlens != nullptr ? p.seqlens[b] : p.max_keys;
  s.L = L < 0 ? 0 : L > p.max_keys ? p.max_keys : L;
  return s;
}
// Row of the partials (and of the packed output) of query i.
__device__ inline int64_t kv8_out_row(const Kv8AttnParams& p, const Kv8Rows& s, int i) {
  return p.cu_q != nullptr ? s.q0 + i : (int64_t)s.b * p.seqlen_q + i;
}
__device__ inline int64_t kv8_base(const Kv8AttnParams& p, const Kv8Rows& s, int64_t sb, int64_t ss) {
  return p.cu_q != nullptr ? s.q0 * ss : (int64_t)s.b * sb;
}

// Keys [lo, hi) that rows q_first .. q_last (queries) of a sequence see between
// them.
__device__ inline void kv8_key_range(const Kv8AttnParams& p, const Kv8Rows& s, int q_first, int q_last,
                                     int& lo, int& hi) {
  const int off = p.causal ? s.L - s.n : 0;
  lo = 0;
  hi = s.L;
  if (p.causal) hi = min(hi, off + q_last + 1);
  if (p.window_right >= 0) hi = min(hi, off + q_last + p.window_right + 1);
  if (p.window_left >= 0) lo = max(lo, off + q_first - p.window_left);
  hi = max(hi, 0);
}

// buf_load16_lds with the non-temporal hint: for data that one workgroup reads.
__device__ inline void kv8_load_lds(const u32x4& r, uint32_t lds, uint32_t voff) {
  asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, 0 offen nt lds"
               :
               : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(voff), "s"(r)
               : "memory", "m0");
}

// What a query row of a lane sees and how its scores are scaled.
struct Kv8Row {
  int key_lo;
  uint32_t keys;   // sees key_lo .. key_lo + keys
  int qpos;
  float slope;
};

template <bool GENERIC>
__device__ inline Kv8Row kv8_row(const Kv8AttnParams& p, const Kv8Rows& s, int qi, int head, int k_end) {
  Kv8Row r;
  r.qpos = qi + (p.causal ? s.L - s.n : 0);
  int lo = 0, hi = k_end - 1;   // (the workgroup's keys end there)
  if (p.causal) hi = min(hi, r.qpos);
  if (p.window_right >= 0) hi = min(hi, r.qpos + p.window_right);
  if (p.window_left >= 0) lo = max(0, r.qpos - p.window_left);
  r.key_lo = hi >= lo ? lo : 1 << 30;   // none: past every key
  r.keys = hi >= lo ? (uint32_t)(hi - lo) : 0;
  r.slope = GENERIC && p.alibi != nullptr ? p.alibi[(int64_t)s.b * p.alibi_sb + head] : 0.f;
  return r;
}

// Byte offsets of a lane's operand reads in a tile of 32 keys (the swizzles
// repeat every 16 rows, so the other steps and halves are constants away).  K:
// row lane % 32, the chunks of Kv8Query.  V: the lane's 8 keys of 16-key step cc
// are 16 cc + 4 g + {0..3, 8..11}; lane i of 16 names 8 bytes of row i / 2.
template <int D, class Q>
struct Kv8Lane {
  uint32_t k[D / 32], v[D / 32];
  __device__ inline Kv8Lane() {
    const int lane = threadIdx.x & 63, c32 = lane & 31, g = lane >> 5;
    const int vr = (lane & 15) >> 1, vkey = 4 * g + (vr & 3) + 8 * (vr >> 2);
#pragma unroll
    for (int j = 0; j < D / 32; ++j) {
      k[j] = (uint32_t)(c32 * D + kv8_k_chunk<D>(c32, Q::chunk(j, g)) * 16);
      v[j] = (uint32_t)(vkey * D + kv8_v_chunk<D>(vkey, 2 * j + ((lane >> 4) & 1)) * 16 + 8 * (lane & 1));
    }
  }
};

// The queries of a wave as the B operand of S^T = K Q^T, and the product.
//
// fp16: 16-bit products.  K rows become 16-bit operands: 4 conversions per
// product.  A lane's chunk j of a row is dims 32 j + 16 g .., its low 8 for
// product 2 j and the high 8 for product 2 j + 1.
template <class T, int D>
struct Kv8Query {
  u32x4 q[D / 16];
  __device__ static inline int chunk(int j, int g) { return 2 * j + g; }
  __device__ inline void load(const uint16_t* row) {
    const int g = (threadIdx.x >> 5) & 1;
#pragma unroll
    for (int j = 0; j < D / 32; ++j) {
      q[2 * j] = load16(row + 32 * j + 16 * g);
      q[2 * j + 1] = load16(row + 32 * j + 16 * g + 8);
    }
  }
  // Waits for the loads (see the call).
  __device__ inline void pin() {
#pragma unroll
    for (int j = 0; j < D / 16; ++j) asm volatile("" : "+v"(q[j]));
  }
  // S^T of NH x 32 keys: the rows of a K tile in LDS, each scaled by its key's
  // scale byte.  The products of the halves take turns, so that the chain of one
  // accumulator is not waited for.
  template <class F8, int NH, class Lane>
  __device__ inline void scores(const uint8_t* kt, const Lane& at, const uint32_t* byte, f32x16* sc) const {
    u32x4 raw[NH][D / 32];
#pragma unroll
    for (int j = 0; j < D / 32; ++j)
#pragma unroll
      for (int h = 0; h < NH; ++h) raw[h][j] = load16(kt + at.k[j] + 32 * h * D);
#pragma unroll
    for (int h = 0; h < NH; ++h) sc[h] = f32x16{};
#pragma unroll
    for (int j = 0; j < D / 32; ++j)
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int h = 0; h < NH; ++h)
          sc[h] = T::mfma32(kv8_operand<T, F8>(raw[h][j][2 * u], raw[h][j][2 * u + 1],
                                               __uint_as_float(byte[h] << 23)),
                            q[2 * j + u], sc[h]);
  }
};

// bf16: 8-bit products (v_mfma_scale_f32_32x32x64), which take K as it is and
// its scale with it.  A bf16 number has 8 significant bits and e4m3 holds 4, so
// the query is the sum of two 8-bit ones, q = 2^e (q1 + q2 / 16), exactly as
// far as the type's range goes: to 2^-23 of the row's largest number, below
// what the fp32 sums of the products are off by.  Two products at twice the
// rate take the time of one in 16 bits, and the 4 conversions per product go.
// (fp16 has 11 bits: three products.)  chunk(j): the 16-byte halves of dims
// 64 (j / 2) + 32 g ...
typedef int i32x8 __attribute__((ext_vector_type(8)));
template <int D>
struct Kv8Query<BF16, D> {
  i32x8 q[2][D / 64];
  int byte;   // e + 127
  __device__ static inline int chunk(int j, int g) { return 4 * (j / 2) + 2 * g + (j & 1); }
  u32x4 raw_[D / 16];
  __device__ inline void load(const uint16_t* row) {
    const int g = (threadIdx.x >> 5) & 1;
#pragma unroll
    for (int j = 0; j < D / 16; ++j) raw_[j] = load16(row + 64 * (j / 4) + 32 * g + 8 * (j % 4));
  }
  __device__ inline void pin() {
#pragma unroll
    for (int j = 0; j < D / 16; ++j) asm volatile("" : "+v"(raw_[j]));
    uint32_t top = 0;   // largest magnitude, as the bits of a bf16
#pragma unroll
    for (int j = 0; j < D / 16; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) top = max(top, max(raw_[j][e] & 0x7fffu, (raw_[j][e] >> 16) & 0x7fffu));
    auto r = __builtin_amdgcn_permlane32_swap(top, top, false, false);
    top = max((uint32_t)r[0], (uint32_t)r[1]);
    // The least e with top <= 1.75 * 2^(8 + e); NaN and infinities: a NaN scale.
    byte = (int)(top >> 7) - 8 + ((top & 0x7fu) > 0x60u ? 1 : 0);
    byte = top >= 0x7f80u ? 255 : max(byte, 5);   // (the second part's is 4 less)
    const float by = __uint_as_float((uint32_t)(254 - min(byte, 253)) << 23);
#pragma unroll
    for (int j = 0; j < D / 8; ++j) {   // four numbers
      float x[4], y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        x[e] = BF16::to_float((uint16_t)(raw_[j / 2][2 * (j & 1) + e / 2] >> (16 * (e & 1)))) * by;
      int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
      w = __builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], w, true);
      const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
      y[0] = (x[0] - lo[0]) * 16.f, y[1] = (x[1] - lo[1]) * 16.f;
      y[2] = (x[2] - hi[0]) * 16.f, y[3] = (x[3] - hi[1]) * 16.f;
      int w2 = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
      w2 = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w2, true);
      q[0][j / 8][j % 8] = w;
      q[1][j / 8][j % 8] = w2;
    }
  }
  template <class F8, int NH, class Lane>
  __device__ inline void scores(const uint8_t* kt, const Lane& at, const uint32_t* kbyte, f32x16* sc) const {
    u32x4 raw[NH][D / 32];
#pragma unroll
    for (int j = 0; j < D / 32; ++j)
#pragma unroll
      for (int h = 0; h < NH; ++h) raw[h][j] = load16(kt + at.k[j] + 32 * h * D);
#pragma unroll
    for (int h = 0; h < NH; ++h) sc[h] = f32x16{};
    const int byte2 = byte == 255 ? 255 : byte - 4;
#pragma unroll
    for (int j = 0; j < D / 64; ++j)
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int h = 0; h < NH; ++h) {
          i32x8 a;
#pragma unroll
          for (int e = 0; e < 8; ++e) a[e] = (int)raw[h][2 * j + e / 4][e % 4];
          sc[h] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, q[u][j], sc[h], F8::kFormat, 0, 0,
                                                                  (int)kbyte[h], 0, u ? byte2 : byte);
        }
  }
};

// Scale, ALiBi and softcap of the scores of keys n0 .. n0 + 31.
__device__ inline void kv8_score_options(const Kv8AttnParams& p, const Kv8Row& row, int n0, f32x16& sc) {
  const int g = (threadIdx.x >> 5) & 1;
#pragma unroll
  for (int v = 0; v < 16; ++v) {
    const int key = n0 + 8 * (v >> 2) + 4 * g + (v & 3);
    float x = sc[v] * p.scale;
    x = fmaf(-row.slope, fabsf((float)(row.qpos - key)), x);
    if (p.softcap > 0.f) {
      // softcap tanh(x / softcap) = softcap (1 - 2 / (exp(2 x / softcap) + 1))
      const float ex = __builtin_amdgcn_exp2f(x * (2.f * kLog2e / p.softcap));
      x = p.softcap * (1.f - 2.f / (ex + 1.f));
    }
    sc[v] = x;
  }
}

__device__ inline void kv8_mask(const Kv8Row& row, int n0, f32x16& sc) {
  const int g = (threadIdx.x >> 5) & 1;
#pragma unroll
  for (int v = 0; v < 16; ++v) {
    const int key = n0 + 8 * (v >> 2) + 4 * g + (v & 3);
    sc[v] = (uint32_t)(key - row.key_lo) > row.keys ? -INFINITY : sc[v];
  }
}

// P of 32 keys, packed to 16 bits as the B operand of two 16-key steps, its
// fp32 sum added to l.
template <class T>
__device__ inline void kv8_exp(const f32x16& sc, float sl, float m, u32x4* pb, float& l) {
#pragma unroll
  for (int cc = 0; cc < 2; ++cc)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float e0 = __builtin_amdgcn_exp2f(fmaf(sc[cc * 8 + 2 * j], sl, -m));
      const float e1 = __builtin_amdgcn_exp2f(fmaf(sc[cc * 8 + 2 * j + 1], sl, -m));
      pb[cc][j] = T::pack2(e0, e1);
      l += e0 + e1;
    }
}

// The V^T operand of 32 keys of a tile in LDS, from row0 on: 8 bytes per 16-key
// step and 32 dims.  Read before the scores are turned into probabilities.
template <int D, class Lane>
__device__ inline void kv8_read_v(const uint8_t* vt, const Lane& at, int row0, u32x2 (*raw)[D / 32]) {
#pragma unroll
  for (int cc = 0; cc < 2; ++cc)
#pragma unroll
    for (int db = 0; db < D / 32; ++db) raw[cc][db] = lds_read_tr8(vt + at.v[db] + (row0 + 16 * cc) * D);
}

// O^T += V^T P^T over 32 keys, V scaled by vsc (16 keys each).  mixed: the rows of the wave do not all see all of these keys, and
// a V number that is not finite must not meet a P of 0.
template <class T, class F8, int D>
__device__ inline void kv8_pv(u32x2 (*raw)[D / 32], const float* vsc, const u32x4* pb, const f32x16& sc,
                              bool mixed, f32x16* acc) {
  constexpr int NDB = D / 32;
  if (mixed) {
    uint32_t flags = 0;
#pragma unroll
    for (int cc = 0; cc < 2; ++cc)
#pragma unroll
      for (int db = 0; db < NDB; ++db) flags |= F8::bad(raw[cc][db][0]) | F8::bad(raw[cc][db][1]);
    if (__builtin_amdgcn_ballot_w64(flags != 0) != 0) {
      // Visible (key, row) pairs and numbers that are not finite, as 1 and 0: a
      // row gets NaN (all bits set) in the columns where their product is not
      // zero.  In integer operations: comparisons would take a pair of scalar
      // registers each, which the loop around this has no room for.
      const uint32_t one = std::is_same<T, F16>::value ? 0x3c00u : 0x3f80u;
      auto seen1 = [&](float x) { return min(__float_as_uint(x) ^ 0xff800000u, 1u) * one; };   // not -inf
      u32x4 seen[2];
#pragma unroll
      for (int cc = 0; cc < 2; ++cc)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          seen[cc][j] = seen1(sc[cc * 8 + 2 * j]) | seen1(sc[cc * 8 + 2 * j + 1]) << 16;
#pragma unroll
      for (int db = 0; db < NDB; ++db) {
        f32x16 hit = f32x16{};
#pragma unroll
        for (int cc = 0; cc < 2; ++cc) {
          u32x4 ind;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t f = F8::bad(raw[cc][db][e]) >> 7;   // a bit per byte
            ind[2 * e] = (f & 1u) * one | ((f >> 8) & 1u) * one << 16;
            ind[2 * e + 1] = ((f >> 16) & 1u) * one | (f >> 24) * one << 16;
            raw[cc][db][e] &= ~(f * 0xffu);
          }
          hit = T::mfma32(ind, seen[cc], hit);
        }
#pragma unroll
        for (int v = 0; v < 16; ++v)
          acc[db][v] = __uint_as_float(__float_as_uint(acc[db][v]) |
                                       (uint32_t)(-(int)__float_as_uint(hit[v]) >> 31));
      }
    }
  }
#pragma unroll
  for (int cc = 0; cc < 2; ++cc)
#pragma unroll
    for (int db = 0; db < NDB; ++db)
      acc[db] = T::mfma32(kv8_operand<T, F8>(raw[cc][db][0], raw[cc][db][1], vsc[cc]), pb[cc], acc[db]);
}

// Steps 0 .. n - 1 in order, those in [b, e) by step(i, false_type), the others
// by step(i, true_type).  Loops of their own: one loop with both forms would
// copy the accumulators where they join, and a mask between the products and
// the maximum, in a block of its own, costs an instruction per score there.
template <class F>
__device__ inline void kv8_three_runs(int n, int b, int e, F step) {
  int i = 0, upto = b < e ? b : n;
  while (true) {
    for (; i < upto; ++i) step(i, std::true_type{});
    if (i >= n) break;
    for (; i < e; ++i) step(i, std::false_type{});
    upto = n;
    if (i >= n) break;
  }
}
__device__ inline int kv8_clamp(int x, int n) { return x < 0 ? 0 : x > n ? n : x; }
// The first i >= 0 with i * per >= x.
__device__ inline int ceil_steps(int x, int per) { return x <= 0 ? 0 : (x + per - 1) / per; }

// Largest of a lane's NH x 16 scores, in four chains of v_max3.
template <int NH>
__device__ inline float kv8_max(const f32x16* sc) {
  float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int h = 0; h < NH; ++h)
#pragma unroll
    for (int v = 0; v < 16; v += 8)
#pragma unroll
      for (int q = 0; q < 4; ++q) m[q] = fmaxf(fmaxf(m[q], sc[h][v + 2 * q]), sc[h][v + 2 * q + 1]);
  return fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
}

// Raises the running maximum m (log2 units) of rows whose new one passes it by
// more than kKv8Slack, and rescales their sums: P then stays below 2^8, and
// most tiles leave the output alone.
template <int NDB>
__device__ inline void kv8_raise(float mx, float& m, float& l, f32x16* acc) {
  const bool raise = mx > m + kKv8Slack;
  if (__builtin_amdgcn_ballot_w64(raise)) {
    const float m_new = raise ? mx : m;
    const float alpha = m_new == m ? 1.f : __builtin_amdgcn_exp2f(m - m_new);
    l *= alpha;
#pragma unroll
    for (int db = 0; db < NDB; ++db) acc[db] *= alpha;
    m = m_new;
  }
}

template <int D, int NST>
struct Kv8Stream {
  static constexpr int kTile = kKv8BN * D;             // bytes of a K or V tile
  static constexpr int kRing = NST * 2 * kTile;        // per wave
  static constexpr int kMerge = 32 * (D + 2) * 4;      // per wave: O rows and (m, l)
  static constexpr int kArea = kKv8Waves * (kRing > kMerge ? kRing : kMerge);
  static constexpr int kStarts = (kKv8Scan + 1) * 4;
  static constexpr int kLds = kArea + kStarts;
};

// Tiles of sequence b (those that its rows see any key of).
__device__ inline int kv8_tiles(const Kv8AttnParams& p, const Kv8Rows& s, int* first_key, int* hi) {
  int lo;
  kv8_key_range(p, s, 0, s.n - 1, lo, *hi);
  *first_key = lo & ~(kKv8BN - 1);
  return s.n > 0 && *hi > lo ? (*hi - *first_key + kKv8BN - 1) / kKv8BN : 0;
}

// How the tiles of the launch's sequences are dealt out: starts[i] for i <= n is
// where sequence i starts on a common axis, which stretches of the returned
// length cut into workgroups.  Where the stretches are long, the sequences
// follow one another, and a workgroup goes from one to the next.  Where that
// takes longer than the tiles (a sequence costs its workgroup some 5 us before
// and after them), each starts a stretch of its own, if there are enough.
__device__ inline int kv8_starts(const Kv8AttnParams& p, int* starts, int* sums) {
  constexpr int kPer = kKv8Scan / (kKv8Waves * 64);
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  int t[kPer], sum = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int b = tid * kPer + i;
    int first, hi;
    t[i] = b < p.batch ? kv8_tiles(p, kv8_rows(p, b), &first, &hi) : 0;
    sum += t[i];
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d, 64);
  if (lane == 0) sums[w] = sum;
  __syncthreads();
  int total = 0;
#pragma unroll
  for (int u = 0; u < kKv8Waves; ++u) total += sums[u];
  int per = max((total + p.positions - 1) / p.positions, kKv8Waves);
  const int own = p.batch < p.positions
      ? max((total + p.positions - p.batch - 1) / (p.positions - p.batch), kKv8Waves) : INT_MAX;
  const int unit = own <= kKv8Own ? own : 1;   // sequences start at multiples of it
  if (unit > 1) per = own;
  sum = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    t[i] = (t[i] + unit - 1) / unit * unit;
    sum += t[i];
  }
  int s = sum;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int x = __shfl_up(s, d, 64);
    if (lane >= d) s += x;
  }
  if (lane == 63) sums[kKv8Waves + w] = s;
  __syncthreads();
  int before = s - sum;
#pragma unroll
  for (int u = 0; u < kKv8Waves; ++u)
    if (u < w) before += sums[kKv8Waves + u];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int b = tid * kPer + i;
    if (b <= p.batch) starts[b] = before;
    before += t[i];
  }
  if (tid == kKv8Waves * 64 - 1) starts[kKv8Scan] = before;
  __syncthreads();
  return __builtin_amdgcn_readfirstlane(per);
}

template <class T, class F8, int D, int NST, bool GENERIC>
__global__ __launch_bounds__(kKv8Waves * 64) __attribute__((amdgpu_waves_per_eu(D == 256 ? 1 : 2)))
void kv8_stream_kernel(const Kv8AttnParams p) {
  using C = Kv8Stream<D, NST>;
  constexpr int BN = kKv8BN;
  constexpr int CPR = D / 16;              // 16-byte chunks of a row
  constexpr int RPI = 64 / CPR;            // rows of one DMA instruction
  constexpr int NI = BN / RPI;             // DMA instructions of a tile
  constexpr int IPG = 16 / RPI;            // of a 16-key group
  constexpr int NDB = D / 32;
  constexpr int kSuper = 32 * kKv8Waves;   // tiles whose pages and scales the lanes hold
  static_assert(RPI <= 16 && 16 % RPI == 0, "an instruction stays within a 16-key group");

  extern __shared__ __attribute__((aligned(16))) uint8_t smem8[];
  int* starts = reinterpret_cast<int*>(smem8 + C::kArea);

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c32 = lane & 31;
  const int g = lane >> 5;
  const int G = (int)p.group.d;

  // K/V heads vary fastest: the heads of a stretch of tokens run together.
  const int kvh = blockIdx.x % p.heads_k;
  const int pos = blockIdx.x / p.heads_k;

  // This workgroup's stretch [at, stop) of the sequences' tiles in a row.
  int b = pos, at = 0, stop = 1, per = 0;
  if (p.positions > 0) {
    per = kv8_starts(p, starts, reinterpret_cast<int*>(smem8));
    const int total = __builtin_amdgcn_readfirstlane(starts[p.batch]);
    if (blockIdx.x == 0) {   // for the merge
      for (int i = tid; i <= p.batch; i += kKv8Waves * 64) p.starts[i] = starts[i];
      if (tid == 0) p.starts[p.batch + 1] = per;
    }
    at = min(pos, total / per + 1) * per;
    stop = min(at + per, total);
    if (at >= stop) return;
    b = 0;   // the last sequence that starts at or before `at`
    for (int step = kKv8Scan / 2; step > 0; step /= 2)
      if (b + step < p.batch && starts[b + step] <= at) b += step;
    b = __builtin_amdgcn_readfirstlane(b);
  }

  const Kv8Lane<D, Kv8Query<T, D>> lane_at;
  const float sl = GENERIC ? kLog2e : p.scale * kLog2e;
  uint8_t* ring = smem8 + w * C::kRing;
  const uint32_t ring_lds = lds_address(ring);

  // One sequence after the other.
  for (; at < stop; ++b) {
    const Kv8Rows s = kv8_rows(p, b);
    const int rows = s.n * G;
    int first, hi;
    const int all_tiles = kv8_tiles(p, s, &first, &hi);
    int k_begin = first, k_end = hi, here = all_tiles;
    if (p.positions > 0) {
      if (all_tiles == 0) continue;
      const int start = __builtin_amdgcn_readfirstlane(starts[b]);
      here = min(start + all_tiles, stop) - at;
      if (here <= 0) {   // (the rest of its last stretch)
        at = min(__builtin_amdgcn_readfirstlane(starts[b + 1]), stop);
        continue;
      }
      k_begin = first + (at - start) * BN;
      k_end = min(hi, k_begin + here * BN);
      at = min(__builtin_amdgcn_readfirstlane(starts[b + 1]), stop);
    } else {
      if (rows <= 0) return;
      at = stop;
      if (all_tiles == 0) k_end = k_begin;
    }

    const int r = min(c32, rows - 1);   // (lanes past the last row repeat it)
    const bool row_valid = c32 < rows;
    const int qi = (int)fdiv(r, p.group);
    const int head = kvh * G + (r - qi * G);
    const int off = p.causal ? s.L - s.n : 0;
    Kv8Row row = kv8_row<GENERIC>(p, s, qi, head, k_end);
    // Keys that every row sees: tiles within need no mask.
    int all_lo = 0, all_hi = s.L - 1;
    if (p.causal) all_hi = min(all_hi, off);
    if (p.window_right >= 0) all_hi = min(all_hi, off + p.window_right);
    if (p.window_left >= 0) all_lo = max(0, s.n - 1 + off - p.window_left);

    Kv8Query<T, D> query;
    query.load(static_cast<const uint16_t*>(p.q) + kv8_base(p, s, p.q_sb, p.q_ss) + (int64_t)qi * p.q_ss +
               (int64_t)head * p.q_sh);

    f32x16 acc[NDB];
#pragma unroll
    for (int db = 0; db < NDB; ++db) acc[db] = f32x16{};
    float m_run = -INFINITY, l_run = 0.f;

    // Lane i holds page, slot and scale bytes of 16-key group i % 2 of this
    // wave's tile i / 2 of the kSuper tiles from s0 on.  A group without keys names
    // no page; its scale is 1.
    int s0, my_tiles, page_l, slot_l;
    uint32_t ks_l, vs_l;
    // LDS-DMA of tile t (of this wave) into its stage.  Lane l of instruction
    // m fills chunk position l % CPR of row m * RPI + l / CPR.
    auto issue = [&](int t) {
      const int key0 = s0 + (w + t * kKv8Waves) * BN;
      const uint32_t st = ring_lds + (uint32_t)((t % NST) * 2 * C::kTile);
      const int row_l = lane / CPR, chunk_pos = lane % CPR;
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        const int64_t sp = kv ? p.v_sp : p.k_sp, ss = kv ? p.v_ss : p.k_ss, sh = kv ? p.v_sh : p.k_sh;
        const uint8_t* base = kv ? p.v : p.k;
#pragma unroll
        for (int gr = 0; gr < 2; ++gr) {
          // (tiles past the last get an empty resource, so that the count of
          // loads in flight is the same on every path)
          const int i = min(2 * t + gr, 63);
          const int page = t < my_tiles ? __builtin_amdgcn_readlane(page_l, i) : -1;
          const int slot = __builtin_amdgcn_readlane(slot_l, i);
          const int left = min(s.L - (key0 + 16 * gr), 16);
          const bool live = page >= 0 && left > 0;
          const u32x4 rs = make_rsrc_words(live ? base + page * sp + slot * ss + kvh * sh : base,
                                           live ? (uint32_t)((left - 1) * ss + D) : 0u);
#pragma unroll
          for (int m = gr * IPG; m < (gr + 1) * IPG; ++m) {
            const int tr = m * RPI + row_l;
            const int chunk = kv ? kv8_v_chunk<D>(tr, chunk_pos) : kv8_k_chunk<D>(tr, chunk_pos);
            kv8_load_lds(rs, st + (uint32_t)(kv * C::kTile + m * 1024),
                         (uint32_t)((tr - 16 * gr) * (int)ss + chunk * 16));
          }
        }
      }
    };
    auto open = [&](int from) {
      s0 = from;
      my_tiles = (min((k_end - s0 + BN - 1) / BN, kSuper) - w + kKv8Waves - 1) / kKv8Waves;
      page_l = -1;
      slot_l = 0;
      ks_l = vs_l = 127;
      const int key = s0 + (w + (lane >> 1) * kKv8Waves) * BN + (lane & 1) * 16;
      if (key < k_end) {
        const int col = (int)fdiv(key, p.page);
        slot_l = key - col * (int)p.page.d;
        page_l = p.table != nullptr ? p.table[(int64_t)b * p.table_stride + col] : p.first_page + b;
        if (page_l < 0 || page_l >= p.num_pages) {
          page_l = -1;
        } else {
          const int blk = slot_l >> p.log2_block;
          ks_l = p.ks[page_l * p.ks_sp + blk * p.ks_sb + kvh * p.ks_sh];
          vs_l = p.vs[page_l * p.vs_sp + blk * p.vs_sb + kvh * p.vs_sh];
        }
      }
      for (int t = 0; t < NST - 1; ++t) issue(t);
    };

    if (k_begin < k_end) {
      open(k_begin);
      query.pin();
    }
    while (k_begin < k_end) {
      // The compiler does not count the LDS-DMA loads: a use of a loaded
      // register inside the loop would wait there for everything in flight, so
      // all of them are waited for here, once.
      asm volatile("" : "+v"(ks_l), "+v"(vs_l));
      if (GENERIC) asm volatile("" : "+v"(row.slope));

      auto step = [&](int t, auto masked) {
        const int n0 = s0 + (w + t * kKv8Waves) * BN;
        // (this wave's LDS reads of the stage that is filled now ended with the
        // previous tile's products)
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        issue(t + NST - 1);
        __builtin_amdgcn_s_waitcnt(vmcnt_imm((NST - 1) * 2 * NI + NI));   // K of tile t
        asm volatile("" ::: "memory");
        const uint8_t* kt = ring + (t % NST) * 2 * C::kTile;
        const uint32_t ks0 = __builtin_amdgcn_readlane(ks_l, 2 * t), ks1 = __builtin_amdgcn_readlane(ks_l, 2 * t + 1);
        const uint32_t ksc = c32 < 16 ? ks0 : ks1;
        f32x16 sc;
        query.template scores<F8, 1>(kt, lane_at, &ksc, &sc);
        if (GENERIC) kv8_score_options(p, row, n0, sc);
        if (masked.value) kv8_mask(row, n0, sc);
        kv8_raise<NDB>(halves_max(kv8_max<1>(&sc)) * sl, m_run, l_run, acc);
        u32x4 pb[2];
        kv8_exp<T>(sc, sl, m_run == -INFINITY ? 0.f : m_run, pb, l_run);
        __builtin_amdgcn_s_waitcnt(vmcnt_imm((NST - 1) * 2 * NI));   // V of tile t
        asm volatile("" ::: "memory");
        const float vsc[2] = {__uint_as_float((uint32_t)__builtin_amdgcn_readlane(vs_l, 2 * t) << 23),
                              __uint_as_float((uint32_t)__builtin_amdgcn_readlane(vs_l, 2 * t + 1) << 23)};
        u32x2 raw[2][NDB];
        kv8_read_v<D>(kt + C::kTile, lane_at, 0, raw);
        // (keys past the sequence's end are zeros in V)
        const bool mixed = masked.value && (n0 < all_lo || (n0 + BN - 1 > all_hi && all_hi < s.L - 1));
        kv8_pv<T, F8, D>(raw, vsc, pb, sc, mixed, acc);
      };
      const int first_key = s0 + w * BN;
      kv8_three_runs(my_tiles, kv8_clamp(ceil_steps(all_lo - first_key, kKv8Waves * BN), my_tiles),
                     kv8_clamp(ceil_steps(min(all_hi + 1, k_end) - BN + 1 - first_key, kKv8Waves * BN), my_tiles),
                     step);
      __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));   // (empty loads past the last tile)
      asm volatile("" ::: "memory");
      if (s0 + kSuper * BN >= k_end) break;
      open(s0 + kSuper * BN);
    }

    // ------------------------------------------------------------ merge waves
    // The rings become the rows' merge area once every wave is done with them.
    __syncthreads();
    float* mo = reinterpret_cast<float*>(smem8);
    float* ml = mo + kKv8Waves * 32 * D;
    const float l_w = halves_sum(l_run);
    if (row_valid) {
      float* orow = mo + (w * 32 + c32) * D;
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4)
          *reinterpret_cast<f32x4*>(orow + db * 32 + 8 * q4 + 4 * g) =
              f32x4{acc[db][4 * q4], acc[db][4 * q4 + 1], acc[db][4 * q4 + 2], acc[db][4 * q4 + 3]};
      if (g == 0) {
        ml[(w * 32 + c32) * 2] = m_run;
        ml[(w * 32 + c32) * 2 + 1] = l_w;
      }
    }
    __syncthreads();
    // Thread t: row t / 8, D / 8 dims from D / 8 * (t % 8).
    constexpr int DPT = D / 8;
    const int rr = tid >> 3;
    if (rr < rows) {
      const int d0 = (tid & 7) * DPT;
      float M = -INFINITY;
#pragma unroll
      for (int u = 0; u < kKv8Waves; ++u) M = fmaxf(M, ml[(u * 32 + rr) * 2]);
      float sum = 0.f, wt[kKv8Waves];
#pragma unroll
      for (int u = 0; u < kKv8Waves; ++u) {
        // (a wave without keys has l = 0; a NaN sum stays one)
        const float l = ml[(u * 32 + rr) * 2 + 1];
        wt[u] = l != 0.f ? __builtin_amdgcn_exp2f(ml[(u * 32 + rr) * 2] - M) : 0.f;
        sum += l * wt[u];
      }
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      float o[DPT];
#pragma unroll
      for (int e = 0; e < DPT; ++e) o[e] = 0.f;
#pragma unroll
      for (int u = 0; u < kKv8Waves; ++u) {
        const float* src = mo + (u * 32 + rr) * D + d0;
#pragma unroll
        for (int e = 0; e < DPT; e += 4) {
          const f32x4 x = *reinterpret_cast<const f32x4*>(src + e);
#pragma unroll
          for (int k = 0; k < 4; ++k) o[e + k] = fmaf(x[k], wt[u], o[e + k]);
        }
      }
      if (here == all_tiles) {   // the sequence's only workgroup
        const int oi = (int)fdiv(rr, p.group);
        uint16_t* dst = static_cast<uint16_t*>(p.o) + kv8_base(p, s, p.o_sb, p.o_ss) + (int64_t)oi * p.o_ss +
                        (int64_t)(kvh * G + (rr - oi * G)) * p.o_sh + d0;
#pragma unroll
        for (int e = 0; e < DPT; e += 8) {
          u32x4 val;
#pragma unroll
          for (int k = 0; k < 4; ++k) val[k] = T::pack2(o[e + 2 * k] * inv, o[e + 2 * k + 1] * inv);
          store16(dst + e, val);
        }
      } else {
        const int64_t prow = ((int64_t)(b + pos) * p.heads_k + kvh) * p.part_rows + rr;
        float* dst = p.o_part + prow * D + d0;
#pragma unroll
        for (int e = 0; e < DPT; e += 4)
          *reinterpret_cast<f32x4*>(dst + e) =
              f32x4{o[e] * inv, o[e + 1] * inv, o[e + 2] * inv, o[e + 3] * inv};
        if ((tid & 7) == 0) p.lse_part[prow] = sum == 0.f ? -INFINITY : M + __log2f(sum);
      }
    }
    __syncthreads();   // the next sequence's tiles come into the same LDS
  }
}

// kv8_chunk_kernel: launches with sequences of more than 32 query rows per K/V
// head, and the shorter ones beside them.  A workgroup of RW x
// KG waves owns 32 RW rows, 32 per wave; its KG groups of RW waves take the
// 64-key tiles in turn (each group with a ring of its own, whose tiles its waves
// load together) and are merged at the end, so that a workgroup's chain of
// tiles is KG times shorter: rows of long sequences beside those of short ones
// would otherwise set the launch's time (4 x 512 queries over 1580 to 5366 keys,
// Hq 32 Hk 8 D 128, bf16: 129 us = 870 TFLOP/s; one group and two workgroups per
// CU: 190 us).  Bound: the two waves of a SIMD, 64 conversions, 32 exponentials and
// about 120 other vector instructions per 1024 cycles of products.  Tile operands, masks and scales as in
// kv8_stream_kernel; pages and scales of up to NT 16-key groups are in LDS at a time
// (NT threads).
template <int D, int RW, int KG, int NST>
struct Kv8Chunk {
  static constexpr int kBN = 64;
  static constexpr int kThreads = RW * KG * 64;
  static constexpr int kTile = kBN * D;                     // bytes of a K or V tile
  static constexpr int kRings = KG * NST * 2 * kTile;
  static constexpr int kWave = 32 * (D + 2) * 4;            // a wave's rows, maxima and sums in fp32
  static constexpr int kMerge = (KG > 1 ? KG - 1 : 1) * RW * kWave;
  static constexpr int kInfo = kThreads * 12;
  static constexpr int kLds = (kRings > kMerge ? kRings : kMerge) + kInfo;
  static constexpr int kSuper = kThreads * 16 / kBN;        // tiles whose pages and scales LDS holds
};

// Row blocks of bm rows of all sequences, those of the longest chains of keys
// first (within blocks of 64 sequences), so that a launch does not end with
// one: the sequence of row block i and, in *rb, which of its blocks it is.
// False past the last one.  Every lane of the wave takes part; sequences
// without queries have none, so the host's count of them (from the rows of q)
// bounds i without knowing the lengths.
__device__ inline bool kv8_row_block(const Kv8AttnParams& p, int i, int bm, Kv8Rows* s, int* rb) {
  const int l = threadIdx.x & 63, G = (int)p.group.d;
  for (int base = 0; base < p.batch; base += 64) {
    const int m = min(64, p.batch - base);
    int nb = 0;
    uint32_t key = 0;
    Kv8Rows mine = {};
    if (l < m) {
      mine = kv8_rows(p, base + l);
      nb = (mine.n * G + bm - 1) / bm;
      // (unique: the chain in 25 bits of its float, then the earlier sequence)
      const float chain = (float)mine.L * (float)(32 + min(mine.n * G, bm));
      key = ((__float_as_uint(chain) >> 6) & ~63u) + 64u + (uint32_t)(63 - l);
    }
    int before = 0, total = 0;
    for (int j = 0; j < m; ++j) {
      const int nj = __builtin_amdgcn_readlane(nb, j);
      total += nj;
      before += (uint32_t)__builtin_amdgcn_readlane(key, j) > key ? nj : 0;
    }
    if (i >= total) {
      i -= total;
      continue;
    }
    const uint64_t hit = __builtin_amdgcn_ballot_w64(i >= before && i < before + nb);
    const int j = hit != 0 ? (int)__builtin_ctzll(hit) : 0;   // (there is one)
    s->b = base + j;
    s->n = __builtin_amdgcn_readlane(mine.n, j);
    s->L = __builtin_amdgcn_readlane(mine.L, j);
    s->q0 = (int64_t)__builtin_amdgcn_readlane((int)mine.q0, j);
    *rb = __builtin_amdgcn_readlane(nb, j) - 1 - (i - __builtin_amdgcn_readlane(before, j));
    return true;
  }
  return false;
}

template <class T, class F8, int D, int RW, int KG, int NST, bool GENERIC>
__global__ __launch_bounds__(RW * KG * 64) __attribute__((amdgpu_waves_per_eu(RW * KG / 4)))
void kv8_chunk_kernel(const Kv8AttnParams p) {
  using C = Kv8Chunk<D, RW, KG, NST>;
  constexpr int BN = C::kBN, BM = 32 * RW;
  constexpr int CPR = D / 16, RPI = 64 / CPR, IPG = 16 / RPI, NDB = D / 32;
  constexpr int GPW = 4 / RW;                  // 16-key groups of a tile that a wave loads
  constexpr int PER = 2 * GPW * IPG;           // its DMA instructions per tile
  static_assert(RW == 2 || RW == 4, "a wave loads whole 16-key groups");

  extern __shared__ __attribute__((aligned(16))) uint8_t smem8c[];

  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rw = w % RW, kg = w / RW;
  const int c32 = lane & 31, g = lane >> 5;

  // K/V heads vary fastest: with 8 of them, or a multiple, each XCD streams its
  // own heads' keys, and all XCDs get the same work.
  int item = blockIdx.x;
  const int kvh = item % p.heads_k;
  item /= p.heads_k;
  const int split = item % p.chunk_splits;
  Kv8Rows s;
  int rb;
  if (!kv8_row_block(p, item / p.chunk_splits, BM, &s, &rb)) return;
  const int b = s.b, G = (int)p.group.d;
  const int rows = min(s.n * G - rb * BM, BM);
  int lo, hi;
  kv8_key_range(p, s, (int)fdiv(rb * BM, p.group), (int)fdiv(rb * BM + rows - 1, p.group), lo, hi);
  const int k_begin = max(split * p.chunk_keys, lo & ~(BN - 1));
  const int k_end = min(hi, (split + 1) * p.chunk_keys);
  if (k_begin >= k_end && split > 0) return;

  // This wave's rows (it helps to load when it has none) and the keys that all
  // of them see.
  const int r0 = rb * BM + rw * 32;
  const int wrows = max(min(rows - rw * 32, 32), 0);
  const bool row_valid = c32 < wrows;
  const int r = r0 + max(min(c32, wrows - 1), 0) - (wrows > 0 ? 0 : rw * 32);
  const int qi = (int)fdiv(r, p.group);
  const int head = kvh * G + (r - qi * G);
  const int q_first = (int)fdiv(wrows > 0 ? r0 : rb * BM, p.group);
  const int q_last = wrows > 0 ? (int)fdiv(r0 + wrows - 1, p.group) : q_first;
  const int off = p.causal ? s.L - s.n : 0;
  Kv8Row row = kv8_row<GENERIC>(p, s, qi, head, k_end);
  int all_lo = 0, all_hi = s.L - 1;
  if (p.causal) all_hi = min(all_hi, q_first + off);
  if (p.window_right >= 0) all_hi = min(all_hi, q_first + off + p.window_right);
  if (p.window_left >= 0) all_lo = max(0, q_last + off - p.window_left);
  int wlo, whi;   // keys that any of the wave's rows sees
  kv8_key_range(p, s, q_first, q_last, wlo, whi);
  if (wrows == 0) whi = 0;

  Kv8Query<T, D> query;
  query.load(static_cast<const uint16_t*>(p.q) + kv8_base(p, s, p.q_sb, p.q_ss) + (int64_t)qi * p.q_ss +
             (int64_t)head * p.q_sh);

  query.pin();
  uint8_t* ring = smem8c + kg * NST * 2 * C::kTile;
  const uint32_t ring_lds = lds_address(ring);
  int* info_page = reinterpret_cast<int*>(smem8c + C::kLds - C::kInfo);
  int* info_slot = info_page + C::kThreads;
  uint32_t* info_scale = reinterpret_cast<uint32_t*>(info_slot + C::kThreads);   // K | V << 16

  const Kv8Lane<D, Kv8Query<T, D>> at;
  f32x16 acc[NDB];
#pragma unroll
  for (int db = 0; db < NDB; ++db) acc[db] = f32x16{};
  float m_run = -INFINITY, l_run = 0.f;
  const float sl = GENERIC ? kLog2e : p.scale * kLog2e;

  for (int s0 = k_begin; s0 < k_end; s0 += C::kSuper * BN) {
    const int n_tiles = min((k_end - s0 + BN - 1) / BN, C::kSuper);
    const int steps = (n_tiles + KG - 1) / KG;
    // Pages and scales: thread i's 16-key group.
    __syncthreads();   // the previous tiles' are done with (and the rings empty)
    {
      const int key = s0 + tid * 16;
      int page = -1, slot = 0;
      uint32_t sc = 127u | 127u << 16;
      if (key < k_end) {
        const int col = (int)fdiv(key, p.page);
        slot = key - col * (int)p.page.d;
        page = p.table != nullptr ? p.table[(int64_t)b * p.table_stride + col] : p.first_page + b;
        if (page < 0 || page >= p.num_pages) {
          page = -1;
        } else {
          const int blk = slot >> p.log2_block;
          sc = (uint32_t)p.ks[page * p.ks_sp + blk * p.ks_sb + kvh * p.ks_sh] |
               (uint32_t)p.vs[page * p.vs_sp + blk * p.vs_sb + kvh * p.vs_sh] << 16;
        }
      }
      info_page[tid] = page;
      info_slot[tid] = slot;
      info_scale[tid] = sc;
    }
    __syncthreads();

    // This wave's share of tile kg + KG * step into its stage.
    auto issue = [&](int step, uint32_t stage) {
      const int t = kg + KG * step;
      const uint32_t st = ring_lds + stage;
      const int row_l = lane / CPR, pos = lane % CPR;
#pragma unroll
      for (int u = 0; u < GPW; ++u) {
        const int gr = rw * GPW + u;
        const int at = min(4 * t + gr, C::kThreads - 1);
        const int page = t < n_tiles ? __builtin_amdgcn_readfirstlane(info_page[at]) : -1;
        const int slot = __builtin_amdgcn_readfirstlane(info_slot[at]);
        const int left = min(s.L - (s0 + t * BN + 16 * gr), 16);
        const bool live = page >= 0 && left > 0;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          const int64_t sp = kv ? p.v_sp : p.k_sp, ss = kv ? p.v_ss : p.k_ss, sh = kv ? p.v_sh : p.k_sh;
          const uint8_t* base = kv ? p.v : p.k;
          const u32x4 rs = make_rsrc_words(live ? base + page * sp + slot * ss + kvh * sh : base,
                                           live ? (uint32_t)((left - 1) * ss + D) : 0u);
#pragma unroll
          for (int m = 0; m < IPG; ++m) {
            const int in_group = m * RPI + row_l;   // (the swizzles repeat every 16 rows)
            const int chunk = kv ? kv8_v_chunk<D>(in_group, pos) : kv8_k_chunk<D>(in_group, pos);
            buf_load16_lds(rs, st + (uint32_t)(kv * C::kTile + (gr * IPG + m) * 1024),
                           (uint32_t)(in_group * (int)ss + chunk * 16));
          }
        }
      }
    };

    for (int i0 = 0; i0 < NST - 1; ++i0) issue(i0, (uint32_t)(i0 * 2 * C::kTile));
    if (GENERIC) asm volatile("" : "+v"(row.slope));
    uint32_t stage = 0, next_stage = (uint32_t)((NST - 1) * 2 * C::kTile);   // of tiles i0 and i0 + NST - 1
    auto advance = [](uint32_t st) { return st + 2 * C::kTile == NST * 2 * C::kTile ? 0u : st + 2 * C::kTile; };
    // Step i: every wave passes its barrier, whatever it does with the tile.
    auto step = [&](int i, auto masked) {
      // Tile i has landed, for every wave, and the stage that is filled next
      // has been read.
      __builtin_amdgcn_sched_barrier(0);
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((NST - 2) * PER) : "memory");
      __builtin_amdgcn_sched_barrier(0);
      issue(i + NST - 1, next_stage);
      const int t = kg + KG * i, n0 = s0 + t * BN;
      const uint8_t* kt = ring + stage;
      const uint8_t* vt = kt + C::kTile;
      stage = advance(stage);
      next_stage = advance(next_stage);
      if (masked.value && (t >= n_tiles || n0 >= whi || n0 + BN <= wlo)) return;
      const uint32_t ksc[2] = {info_scale[4 * t + (c32 >> 4)] & 0xffffu, info_scale[4 * t + 2 + (c32 >> 4)] & 0xffffu};
      float vsc[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) vsc[u] = __uint_as_float(info_scale[4 * t + u] >> 16 << 23);
      f32x16 sc[2];
      u32x2 raw[2][2][NDB];
      if constexpr (D == 256) {   // (registers for the operands of 32 keys at a time)
        query.template scores<F8, 1>(kt, at, ksc, sc);
        query.template scores<F8, 1>(kt + 32 * D, at, ksc + 1, sc + 1);
      } else {
        query.template scores<F8, 2>(kt, at, ksc, sc);
        kv8_read_v<D>(vt, at, 0, raw[0]);
        kv8_read_v<D>(vt, at, 32, raw[1]);
      }
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        if (GENERIC) kv8_score_options(p, row, n0 + 32 * hf, sc[hf]);
        if (masked.value) kv8_mask(row, n0 + 32 * hf, sc[hf]);
      }
      kv8_raise<NDB>(halves_max(kv8_max<2>(sc)) * sl, m_run, l_run, acc);
      const float m_use = m_run == -INFINITY ? 0.f : m_run;
      const bool mixed = masked.value && (n0 < all_lo || (n0 + BN - 1 > all_hi && all_hi < s.L - 1));
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        u32x4 pb[2];
        kv8_exp<T>(sc[hf], sl, m_use, pb, l_run);
        if constexpr (D == 256) kv8_read_v<D>(vt, at, 32 * hf, raw[hf]);
        kv8_pv<T, F8, D>(raw[hf], vsc + 2 * hf, pb, sc[hf], mixed, acc);
      }
    };
    // Steps [i_b, i_e) of this wave need no mask.
    const int first = s0 + kg * BN;
    const int i_b = kv8_clamp(ceil_steps(all_lo - first, KG * BN), steps);
    const int i_e = wrows > 0 ? kv8_clamp(ceil_steps(min(all_hi + 1, k_end) - BN + 1 - first, KG * BN), steps) : 0;
    kv8_three_runs(steps, i_b, i_e, step);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  }

  // Merge the key groups: groups 1 .. KG - 1 leave their rows in LDS in the
  // register order of the wave that takes them.
  float l_w = halves_sum(l_run);
  if constexpr (KG > 1) {
    __syncthreads();
    float* area = reinterpret_cast<float*>(smem8c);
    if (kg > 0) {
      float* to = area + ((kg - 1) * RW + rw) * (C::kWave / 4);
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4)
          *reinterpret_cast<f32x4*>(to + ((db * 4 + q4) * 64 + lane) * 4) =
              f32x4{acc[db][4 * q4], acc[db][4 * q4 + 1], acc[db][4 * q4 + 2], acc[db][4 * q4 + 3]};
      if (g == 0) {
        to[32 * D + 2 * c32] = m_run;
        to[32 * D + 2 * c32 + 1] = l_w;
      }
    }
    __syncthreads();
    if (kg > 0) return;
#pragma unroll
    for (int u = 1; u < KG; ++u) {
      const float* from = area + ((u - 1) * RW + rw) * (C::kWave / 4);
      const float mu = from[32 * D + 2 * c32], lu = from[32 * D + 2 * c32 + 1];
      const float m_new = fmaxf(m_run, mu);
      // (a group without keys has l = 0; a NaN sum stays one)
      const float a0 = l_w != 0.f ? __builtin_amdgcn_exp2f(m_run - m_new) : 0.f;
      const float a1 = lu != 0.f ? __builtin_amdgcn_exp2f(mu - m_new) : 0.f;
      l_w = l_w * a0 + lu * a1;
      m_run = m_new;
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
          const f32x4 x = *reinterpret_cast<const f32x4*>(from + ((db * 4 + q4) * 64 + lane) * 4);
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[db][4 * q4 + e] = acc[db][4 * q4 + e] * a0 + x[e] * a1;
        }
    }
  }
  if (!row_valid) return;
  const float inv = l_w == 0.f ? 0.f : 1.f / l_w;
  if (p.chunk_splits == 1) {
    uint16_t* dst = static_cast<uint16_t*>(p.o) + kv8_base(p, s, p.o_sb, p.o_ss) + (int64_t)qi * p.o_ss +
                    (int64_t)head * p.o_sh;
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4)
        *reinterpret_cast<u32x2*>(dst + 32 * db + 8 * q4 + 4 * g) =
            u32x2{T::pack2(acc[db][4 * q4] * inv, acc[db][4 * q4 + 1] * inv),
                  T::pack2(acc[db][4 * q4 + 2] * inv, acc[db][4 * q4 + 3] * inv)};
  } else {
    const int64_t prow = ((int64_t)split * p.total_q + kv8_out_row(p, s, qi)) * p.heads_q + head;
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4)
        *reinterpret_cast<f32x4*>(p.o_part + prow * D + 32 * db + 8 * q4 + 4 * g) =
            f32x4{acc[db][4 * q4] * inv, acc[db][4 * q4 + 1] * inv, acc[db][4 * q4 + 2] * inv,
                  acc[db][4 * q4 + 3] * inv};
    if (g == 0) p.lse_part[prow] = l_w == 0.f ? -INFINITY : m_run + __log2f(l_w);
  }
}

// Four dims of a row, merged from some of its pieces.
struct Kv8Sum {
  float m, tot;   // largest log sum (log2 units; -inf: no keys), and the weights' sum relative to it
  f32x4 acc;
  bool bad;       // a log sum was NaN
};

// Merges pieces i0, i0 + SL, ... < n of four dims of a row, `step` rows of the
// partials apart, fetched in batches of independent loads.
template <int D, int SL>
__device__ inline Kv8Sum kv8_merge(const Kv8AttnParams& p, int64_t prow, int64_t step, int i0, int n, int qd) {
  constexpr int kBatch = SL > 1 ? 8 : 16;
  Kv8Sum s = {-INFINITY, 0.f, {0.f, 0.f, 0.f, 0.f}, false};
  for (; i0 < n; i0 += kBatch * SL) {
    float ls[kBatch];
    f32x4 o[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int64_t at = prow + (i0 + u * SL) * step;
      const bool on = i0 + u * SL < n;
      ls[u] = on ? p.lse_part[at] : -INFINITY;
      o[u] = on ? *reinterpret_cast<const f32x4*>(p.o_part + at * D + qd * 4) : f32x4{0.f, 0.f, 0.f, 0.f};
    }
    float mb = s.m;
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      mb = fmaxf(mb, ls[u]);
      s.bad |= ls[u] != ls[u];
    }
    if (mb == -INFINITY) continue;
    const float again = __builtin_amdgcn_exp2f(s.m - mb);   // m == -inf -> 0
    s.tot *= again;
    s.acc *= again;
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const float wgt = ls[u] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ls[u] - mb);
      s.tot += wgt;
      s.acc += wgt * o[u];
    }
    s.m = mb;
  }
  return s;
}

// The rows whose keys more than one workgroup took, and those without keys:
// out = sum_i 2^(lse_i - lse) o_i, a workgroup within one sequence.  A thread per
// row and 4 dims, or, where rows have many pieces, a workgroup per row whose
// SL slices take every SL-th piece and merge through LDS, in an order that is
// always the same.
template <class T, int D, int SL>
__global__ __launch_bounds__(256) void kv8_combine_kernel(const Kv8AttnParams p) {
  constexpr int kQuads = D / 4;
  static_assert(SL == 1 || SL * kQuads == 256, "a workgroup per row");
  __shared__ Kv8Sum slices[SL > 1 ? 256 : 1];
  const int b = blockIdx.y, G = (int)p.group.d;
  const Kv8Rows s = kv8_rows(p, b);
  int p0 = 0, pieces = 0;
  if (p.chunk_splits == 0) {   // kv8_stream_kernel: the stretches that the sequence's tiles lie in
    const int start = p.starts[b], end = p.starts[b + 1], per = p.starts[p.batch + 1];
    p0 = start / per;
    pieces = end > start ? (end - 1) / per - p0 + 1 : 0;
    if (pieces == 1) return;
  }
  const int slice = threadIdx.x / kQuads;
  const int64_t per_wg = 256 / SL, all = (int64_t)s.n * p.heads_q * kQuads;
  for (int64_t idx = (int64_t)blockIdx.x * per_wg + threadIdx.x % per_wg; idx < all; idx += (int64_t)gridDim.x * per_wg) {
    const int64_t item = idx / kQuads;
    const int qd = (int)(idx % kQuads), h = (int)(item % p.heads_q), i = (int)(item / p.heads_q);
    uint16_t* dst = static_cast<uint16_t*>(p.o) + kv8_base(p, s, p.o_sb, p.o_ss) + (int64_t)i * p.o_ss +
                    (int64_t)h * p.o_sh;
    int64_t prow, step;
    int n = pieces;
    if (p.chunk_splits == 0) {
      step = (int64_t)p.heads_k * p.part_rows;
      prow = (int64_t)(b + p0) * step + (int64_t)(h / G) * p.part_rows + i * G + h % G;
    } else {   // kv8_chunk_kernel: the splits that meet the keys of the row's block
      const int rb = (i * G + h % G) / kKv8ChunkRows, last = min(rb * kKv8ChunkRows + kKv8ChunkRows, s.n * G) - 1;
      int lo, hi;
      kv8_key_range(p, s, (int)fdiv(rb * kKv8ChunkRows, p.group), (int)fdiv(last, p.group), lo, hi);
      const int first = lo / p.chunk_keys;
      n = hi > lo ? min(p.chunk_splits, (hi + p.chunk_keys - 1) / p.chunk_keys) - first : 0;
      step = p.total_q * p.heads_q;
      prow = first * step + kv8_out_row(p, s, i) * p.heads_q + h;
    }
    Kv8Sum sum = kv8_merge<D, SL>(p, prow, step, SL > 1 ? slice : 0, n, qd);
    if constexpr (SL > 1) {   // (one row per workgroup: every thread is here)
      __syncthreads();        // the slices of the row before may still be read
      slices[threadIdx.x] = sum;
      __syncthreads();
      if (slice > 0) continue;
      float m = sum.m;
#pragma unroll
      for (int u = 1; u < SL; ++u) m = fmaxf(m, slices[u * kQuads + qd].m);
      const float own = sum.m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(sum.m - m);
      sum.tot *= own;
      sum.acc *= own;
#pragma unroll
      for (int u = 1; u < SL; ++u) {
        const Kv8Sum& t = slices[u * kQuads + qd];
        const float wgt = t.m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(t.m - m);
        sum.tot += wgt * t.tot;
        sum.acc += wgt * t.acc;
        sum.bad |= t.bad;
      }
    }
    const float inv = sum.bad ? __uint_as_float(0x7fc00000u) : sum.tot > 0.f ? 1.f / sum.tot : 0.f;
    *reinterpret_cast<u32x2*>(dst + qd * 4) =
        u32x2{T::pack2(sum.acc[0] * inv, sum.acc[1] * inv), T::pack2(sum.acc[2] * inv, sum.acc[3] * inv)};
  }
}

// A workgroup merges each row where rows may have 8 pieces or more, and are few:
// two workgroups per CU.  Decode calls with a thread per 4 dims / a workgroup per
// row, bf16, MI355X: 32768 keys, Hq 16 Hk 1 D 128 (512 pieces) 35.7 / 18.0 us, 16
// sequences of them (256 rows) 31.5 / 30.2; 131001 keys, Hq 32 Hk 8 D 128 (64 pieces)
// 50.0 / 45.8; 8 sequences of 16384 (256 rows, 8 pieces) 45.9 / 45.5.  With more
// rows a thread per 4 dims fills the GPU too: the merge alone of 1280 rows, D 64,
// 3.8 / 6.5; calls of 2560 rows (4 chunks of 40 queries, Hq 16 Hk 4 D 128) 56.0 / 59.4.
template <class T, int D>
hipError_t launch_kv8_combine(const Kv8AttnParams& p, int64_t pieces, int64_t most_wgs, hipStream_t st) {
  const int64_t rows = (int64_t)p.seqlen_q * p.heads_q, few = (rows * (D / 4) + 255) / 256;
  const bool many = pieces >= 8 && rows * p.batch <= 512;
  const int64_t n = many ? rows : few;
  const dim3 grid((unsigned)(n < most_wgs ? n : most_wgs), (unsigned)p.batch);
  if (many) hipLaunchKernelGGL((kv8_combine_kernel<T, D, 1024 / D>), grid, dim3(256), 0, st, p);
  else hipLaunchKernelGGL((kv8_combine_kernel<T, D, 1>), grid, dim3(256), 0, st, p);
  return hipGetLastError();
}

template <class T, class F8, int D, bool GENERIC>
hipError_t launch_kv8_stream(Kv8AttnParams p, hipStream_t st) {
  constexpr int NST = D == 64 ? 3 : 2;
  using C = Kv8Stream<D, NST>;
  auto kern = kv8_stream_kernel<T, F8, D, NST, GENERIC>;
  static std::atomic<uint64_t> lds_devices{0};
  if (hipError_t e = set_lds_limit(lds_devices, kern, C::kLds); e != hipSuccess) return e;
  const int64_t wgs = (int64_t)(p.positions > 0 ? p.positions : p.batch) * p.heads_k;
  if (wgs * kKv8Waves * 64 > 0xffffffffll) return hipErrorInvalidConfiguration;
  hipLaunchKernelGGL(kern, dim3((unsigned)wgs), dim3(kKv8Waves * 64), C::kLds, st, p);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.positions == 0) return e;
  return launch_kv8_combine<T, D>(p, p.positions / p.batch, INT_MAX, st);
}

template <class T, class F8, int D, bool GENERIC>
hipError_t launch_kv8_chunk(const Kv8AttnParams& p, hipStream_t st) {
  // D = 256: one wave per SIMD has the registers for a row's sums.
  constexpr int RW = kKv8ChunkRows / 32, KG = D == 256 ? 1 : 2, NST = 3;
  using C = Kv8Chunk<D, RW, KG, NST>;
  auto kern = kv8_chunk_kernel<T, F8, D, RW, KG, NST, GENERIC>;
  static std::atomic<uint64_t> lds_devices{0};
  if (hipError_t e = set_lds_limit(lds_devices, kern, C::kLds); e != hipSuccess) return e;
  const int64_t wgs = (int64_t)p.chunk_splits * p.chunk_blocks * p.heads_k;
  if (wgs * C::kThreads > 0xffffffffll) return hipErrorInvalidConfiguration;
  hipLaunchKernelGGL(kern, dim3((unsigned)wgs), dim3(C::kThreads), C::kLds, st, p);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.chunk_splits == 1) return e;
  // (few workgroups per sequence: most sequences of a packed batch are far
  // shorter than its longest)
  return launch_kv8_combine<T, D>(p, p.chunk_splits, 8192 / p.batch + 1, st);
}

template <class T>
hipError_t launch_kv8_attn(int store, const Kv8AttnParams& p, int head_dim, hipStream_t st) {
  const bool generic = p.alibi != nullptr || p.softcap > 0.f || !(p.scale > 0.f);
#define FA_KV8(FF, DD)                                                                             \
  if (p.chunk_splits > 0)                                                                          \
    return generic ? launch_kv8_chunk<T, FF, DD, true>(p, st) : launch_kv8_chunk<T, FF, DD, false>(p, st); \
  return generic ? launch_kv8_stream<T, FF, DD, true>(p, st) : launch_kv8_stream<T, FF, DD, false>(p, st);
#define FA_KV8_D(FF)                      \
  if (head_dim == 64) { FA_KV8(FF, 64) }   \
  if (head_dim == 128) { FA_KV8(FF, 128) } \
  if (head_dim == 256) { FA_KV8(FF, 256) }
  if (store == 0) { FA_KV8_D(E4M3) } else { FA_KV8_D(E5M2) }
#undef FA_KV8_D
#undef FA_KV8
  return hipErrorInvalidValue;
}

}  // namespace fa
