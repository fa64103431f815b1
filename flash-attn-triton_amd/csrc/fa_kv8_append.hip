// New K / V rows quantized into the 8-bit paged cache (fa_kvcache8_append).
//
// A run is a stretch of consecutive rows that go to consecutive slots of one
// scale block.  With M the largest number of the 8-bit type (1.75 * 2^8 or
// 1.75 * 2^15), the run needs the least scale 2^E with amax <= M * 2^E over its
// finite numbers: read off the exponent and the mantissa of amax, nothing is
// divided.  A run that begins its block sets the scale to that; another raises
// it where needed, and then the rows that the block holds already (those below
// the run) are rounded to the new scale, x * 2^(e_old - e_new).  Scaling by a
// power of two is exact, so each number is rounded once, to nearest even; a
// number that is not finite is stored as NaN.  Slots of -1 (or outside the
// cache) are skipped.
//
// One workgroup owns a run of one head of K or V: the scale needs all of it.
// Which rows begin a run is found from the slots alone, in a window of rows
// per workgroup: one row where there are few (a decode step, whose rows are
// all runs of their own: as many workgroups as there are rows, heads and
// tensors), a block's worth where there are many (a prompt: a window per row
// would launch 64 empty workgroups for each that works).
//
// Bound: for prompts the latency of slots, then rows, then stores, covered by 16
// waves per CU: 18800 tokens, Hk 8 D 128, bf16: 27.6 us for 115 MB (with rows kept
// in fp32 between the two sweeps, 12 waves, and the slots of a run compared one by
// one: 38 us); for single tokens latency too: 64 tokens 4.4 us.
#include <type_traits>

#include "fa_common.h"
#include "fa_kv8.h"

namespace fa {

namespace {

struct E4M3Store {
  static constexpr int kTop = 8;    // largest number 1.75 * 2^kTop
  __device__ static inline uint32_t pack4(const float* x) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], w, true);
  }
  __device__ static inline void unpack4(uint32_t w, float* x) {
    const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
    const auto b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    x[0] = a[0], x[1] = a[1], x[2] = b[0], x[3] = b[1];
  }
};
struct E5M2Store {
  static constexpr int kTop = 15;
  __device__ static inline uint32_t pack4(const float* x) {
    int w = __builtin_amdgcn_cvt_pk_bf8_f32(x[0], x[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_bf8_f32(x[2], x[3], w, true);
  }
  __device__ static inline void unpack4(uint32_t w, float* x) {
    const auto a = __builtin_amdgcn_cvt_pk_f32_bf8((int)w, false);
    const auto b = __builtin_amdgcn_cvt_pk_f32_bf8((int)w, true);
    x[0] = a[0], x[1] = a[1], x[2] = b[0], x[3] = b[1];
  }
};

// 2^(byte - 127) as fp32 (byte 0: a subnormal).
__device__ inline float scale_value(int byte) {
  return __uint_as_float(byte > 0 ? (uint32_t)byte << 23 : 0x00400000u);
}

// Eight numbers of a row, as they are loaded, and in fp32.
template <class T>
struct Eight {
  u32x4 w;
  __device__ inline void load(const void* row, int d) { w = load16(static_cast<const uint16_t*>(row) + d); }
  __device__ inline float operator[](int i) const { return T::to_float((uint16_t)(w[i / 2] >> (16 * (i & 1)))); }
  __device__ inline void again() { asm volatile("" : "+v"(w)); }
};
template <>
struct Eight<float> {
  f32x4 w[2];
  __device__ inline void load(const void* row, int d) {
    const f32x4* s = reinterpret_cast<const f32x4*>(static_cast<const float*>(row) + d);
    w[0] = s[0];
    w[1] = s[1];
  }
  __device__ inline float operator[](int i) const { return w[i / 4][i % 4]; }
  __device__ inline void again() {}
};

}  // namespace

// NW waves per workgroup.
template <class T, class S, int D, int NW>
__global__ __launch_bounds__(NW * 64) void kv8_append_kernel(const Kv8AppendParams p) {
  constexpr int kLanes = D / 8;                 // lanes of a row
  constexpr int kRows = NW * 64 / kLanes;       // rows of one pass of the workgroup
  constexpr int kKeep = 8;                      // passes whose rows stay in registers between the two sweeps
  constexpr int kBytes = std::is_same<T, float>::value ? 4 : 2;
  __shared__ float wave_max[NW];
  const int tid = threadIdx.x, lane = tid & 63;
  const int h = blockIdx.y, t = blockIdx.z;
  const int my_row = tid / kLanes, d0 = (tid % kLanes) * 8;
  const uint8_t* x = static_cast<const uint8_t*>(p.x[t]) + (int64_t)h * p.x_sh[t] * kBytes;
  const int64_t x_sr = p.x_sr[t] * kBytes;
  const int block = 1 << p.log2_block;

  // What 64 rows from `row` on hold: lane i's slot, which rows begin a run and
  // which go on with the one before (from slot to slot of a block).
  const int64_t slots_end = (p.num_pages * (int64_t)p.blocks_per_page.d) << p.log2_block;
  auto look = [&](int row0, int64_t* slot, uint64_t* begins, uint64_t* goes_on) {
    const int row = row0 + lane;
    const int64_t s = row < p.rows ? p.slots[row] : -1;
    const int64_t before = row > 0 && row < p.rows ? p.slots[row - 1] : -1;
    const bool usable = s >= 0 && s < slots_end;
    const bool on = usable && before + 1 == s && (s & (block - 1)) != 0;
    *slot = s;
    *begins = __builtin_amdgcn_ballot_w64(usable && !on);
    *goes_on = __builtin_amdgcn_ballot_w64(on);
  };
  const int w0 = blockIdx.x * p.window, w1 = min(w0 + p.window, p.rows);
  for (int c0 = w0; c0 < w1; c0 += 64) {
    int64_t slot_l, unused_slot;
    uint64_t todo, goes_on, next_goes_on, unused;
    look(c0, &slot_l, &todo, &goes_on);
    look(c0 + 64, &unused_slot, &unused, &next_goes_on);
    if (w1 - c0 < 64) todo &= ((uint64_t)1 << (w1 - c0)) - 1;
    for (; todo != 0; todo &= todo - 1) {
      const int i0 = (int)__builtin_ctzll(todo), r0 = c0 + i0;
      const int64_t slot =
          (int64_t)(((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(slot_l >> 32), i0) << 32) |
                    (uint32_t)__builtin_amdgcn_readlane((int)slot_l, i0));
      const int first = (int)(slot & (block - 1));
      // Rows of the run.  (The two masks hold the 64 rows behind any of the
      // first; a larger block is looked through row group by row group.)
      uint64_t on = goes_on >> i0 >> 1 | next_goes_on << (63 - i0);
      int n = 1 + (on == ~(uint64_t)0 ? 64 : (int)__builtin_ctzll(~on));
      while (n > 64 && (n - 1) % 64 == 0 && n < block - first) {
        look(r0 + n, &unused_slot, &unused, &on);
        n += on == ~(uint64_t)0 ? 64 : (int)__builtin_ctzll(~on);
        if (on != ~(uint64_t)0) break;
      }
      const uint32_t gblock = (uint32_t)(slot >> p.log2_block);
      const int64_t page = fdiv(gblock, p.blocks_per_page);
      const int blk = (int)(gblock - (uint32_t)page * p.blocks_per_page.d);
      uint8_t* c = p.cache[t] + page * p.c_sp[t] + (int64_t)(blk << p.log2_block) * p.c_ss[t] + h * p.c_sh[t];
      uint8_t* sp = p.scale[t] + page * p.s_sp[t] + blk * p.s_sb[t] + h * p.s_sh[t];
      const int old = first > 0 ? min((int)*sp, 254) : 0;

      // Largest finite magnitude.
      const uint8_t* xr = x + (int64_t)r0 * x_sr;
      Eight<T> keep[kKeep];
      float top = 0.f;
      auto largest = [&](const Eight<T>& v) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float m = fabsf(v[e]);
          top = m < INFINITY ? fmaxf(top, m) : top;   // (false for NaN)
        }
      };
#pragma unroll
      for (int i = 0; i < kKeep; ++i) {
        if (i * kRows + my_row < n) keep[i].load(xr + (int64_t)(i * kRows + my_row) * x_sr, d0);
      }
#pragma unroll
      for (int i = 0; i < kKeep; ++i)
        if (i * kRows + my_row < n) largest(keep[i]);
      for (int i = kKeep * kRows + my_row; i < n; i += kRows) {
        Eight<T> v;
        v.load(xr + (int64_t)i * x_sr, d0);
        largest(v);
      }
      // (as they were loaded: the compiler would keep all of them in fp32 too)
#pragma unroll
      for (int i = 0; i < kKeep; ++i) keep[i].again();
#pragma unroll
      for (int d = 1; d < 64; d *= 2) top = fmaxf(top, __shfl_xor(top, d, 64));
      if constexpr (NW > 1) {
        __syncthreads();   // wave_max and the scale byte may still be read for the previous run
        if (lane == 0) wave_max[tid >> 6] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < NW; ++w) top = fmaxf(top, wave_max[w]);
      }
      const uint32_t bits = __float_as_uint(top);
      const int need = (int)(bits >> 23) - S::kTop + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
      const int e = max(old, min(max(need, 0), 254));

      auto put = [&](uint8_t* to, const auto& v, float by, bool check) {
        float y[8];
#pragma unroll
        for (int k = 0; k < 8; ++k)
          y[k] = !check || fabsf(v[k]) < INFINITY ? v[k] * by : __uint_as_float(0x7fc00000u);
        *reinterpret_cast<u32x2*>(to + d0) = u32x2{S::pack4(y), S::pack4(y + 4)};
      };
      // Rows that the block holds, where its scale grows.
      if (first > 0 && e > old) {
        const float by = e - old < 127 ? scale_value(127 + old - e) : 0.f;
        for (int i = my_row; i < first; i += kRows) {
          uint8_t* to = c + (int64_t)i * p.c_ss[t];
          const u32x2 w = *reinterpret_cast<const u32x2*>(to + d0);
          float v[8];
          S::unpack4(w[0], v);
          S::unpack4(w[1], v + 4);
          put(to, v, by, false);
        }
      }
      const float by = scale_value(254 - e);
      uint8_t* cn = c + (int64_t)first * p.c_ss[t];
#pragma unroll
      for (int i = 0; i < kKeep; ++i)
        if (i * kRows + my_row < n) put(cn + (int64_t)(i * kRows + my_row) * p.c_ss[t], keep[i], by, true);
      for (int i = kKeep * kRows + my_row; i < n; i += kRows) {
        Eight<T> v;
        v.load(xr + (int64_t)i * x_sr, d0);
        put(cn + (int64_t)i * p.c_ss[t], v, by, true);
      }
      if (tid == 0) *sp = (uint8_t)e;
    }
  }
}

template <class T, class S, int D>
hipError_t launch_append(Kv8AppendParams p, hipStream_t st) {
  // One row per workgroup while that makes at most 16384 of them.
  const int64_t pairs = 2 * (int64_t)p.heads;
  const bool few = p.rows * pairs <= 16384;
  p.window = few ? 1 : 1 << p.log2_block;
  const dim3 grid((unsigned)(((int64_t)p.rows + p.window - 1) / p.window), (unsigned)p.heads, 2);
  if (few) hipLaunchKernelGGL((kv8_append_kernel<T, S, D, 1>), grid, dim3(64), 0, st, p);
  else hipLaunchKernelGGL((kv8_append_kernel<T, S, D, 4>), grid, dim3(256), 0, st, p);
  return hipGetLastError();
}

template <class T, class S>
hipError_t launch_append_d(const Kv8AppendParams& p, int head_dim, hipStream_t st) {
  if (head_dim == 64) return launch_append<T, S, 64>(p, st);
  if (head_dim == 128) return launch_append<T, S, 128>(p, st);
  if (head_dim == 256) return launch_append<T, S, 256>(p, st);
  return hipErrorInvalidValue;
}

template <class T>
hipError_t launch_append_s(int store, const Kv8AppendParams& p, int head_dim, hipStream_t st) {
  return store == 0 ? launch_append_d<T, E4M3Store>(p, head_dim, st)
                    : launch_append_d<T, E5M2Store>(p, head_dim, st);
}

}  // namespace fa

hipError_t fa_launch_kv8_append(int dtype, int store, const fa::Kv8AppendParams& p, int head_dim,
                                hipStream_t st) {
  if (dtype == 0) return fa::launch_append_s<fa::F16>(store, p, head_dim, st);
  if (dtype == 1) return fa::launch_append_s<fa::BF16>(store, p, head_dim, st);
  return fa::launch_append_s<float>(store, p, head_dim, st);
}
