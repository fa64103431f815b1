// Parameter blocks and launchers of the operators around the paged KV cache
// held in 8 bits (fa_kv8_slots.hip, fa_kv8_append.hip, fa_kv8_attn.h), shared
// with their C ABI (fa_kv8_api.hip).  Strides are in elements (bytes, for the
// caches and scales).
//
// The cache: K and V are [pages, page_size, heads_k, head_dim] of an 8-bit
// floating-point type, with a scale byte per block of `block` slots and head,
// [pages, page_size / block, heads_k]: a cached value is its 8-bit number times
// 2^(byte - 127).  Powers of two make everything but the first rounding exact:
// the dequantization to 16 bits, the rescaling of a block whose scale grows
// (subnormals aside), and the quantized numbers themselves, which then depend
// neither on the order of the appends nor on how a division rounds.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "fa_fastdiv.h"

namespace fa {

struct SlotsParams {
  int32_t* table; int64_t table_stride; int cols;
  const int32_t* cached; const int32_t* added;
  const int32_t* free_pages; int64_t n_free; const int32_t* free_start;
  int64_t* slots; int32_t* positions; int32_t* cu; int32_t* seqlens; int32_t* free_end;
  int batch, rows;
  FastDiv page;
};

struct Kv8AppendParams {
  const void* x[2];              // new K and V rows, [rows, heads, D]
  int64_t x_sr[2], x_sh[2];
  uint8_t* cache[2];
  int64_t c_sp[2], c_ss[2], c_sh[2];   // {page, slot, head}
  uint8_t* scale[2];
  int64_t s_sp[2], s_sb[2], s_sh[2];   // {page, block, head}
  const int64_t* slots;
  int rows, heads, window;       // window: rows per workgroup
  int log2_block;
  int64_t num_pages;
  FastDiv blocks_per_page;
};

struct Kv8AttnParams {
  const void* q; void* o;
  int64_t q_sb, q_ss, q_sh, o_sb, o_ss, o_sh;   // {batch, query, head}; packed: no batch
  const uint8_t* k; const uint8_t* v;
  int64_t k_sp, k_ss, k_sh, v_sp, v_ss, v_sh;   // {page, slot, head}
  const uint8_t* ks; const uint8_t* vs;
  int64_t ks_sp, ks_sb, ks_sh, vs_sp, vs_sb, vs_sh;   // {page, block, head}
  int log2_block;
  const int* seqlens; const int* table; int64_t table_stride;
  const int* cu_q;               // packed queries: row offsets; null: [batch, seqlen_q]
  int64_t total_q;               // rows of q
  FastDiv page;
  int first_page;                // without a table: the page of sequence 0
  int num_pages, batch, seqlen_q, heads_q, heads_k, max_keys;
  FastDiv group;
  float scale, softcap;
  const float* alibi; int64_t alibi_sb;
  int causal, window_left, window_right;
  // Launches whose sequences have at most 32 rows (queries times the group) per
  // K/V head: kv8_stream_kernel, `positions` equal stretches of all tiles per
  // head (0: a workgroup per sequence).  The others (chunk_splits > 0):
  // kv8_chunk_kernel, chunk_blocks blocks of rows in all (at least), the keys in
  // chunk_splits splits of chunk_keys.
  int positions, part_rows;
  int chunk_blocks, chunk_keys, chunk_splits;
  // Partial rows and their LSEs (log2 units): of sequence b in stretch i at
  // [b + i][K/V head][part_rows], which no other pair of the staircase of
  // sequences and stretches has; of splits at [split][row of q][head].
  float* o_part; float* lse_part;
  int* starts;   // tiles before each sequence (batch + 1), and a stretch's
};

constexpr int kKv8StreamRows = 32;
constexpr int kKv8ChunkRows = 128;
constexpr int kKv8Scan = 256;   // sequences of a kv8_stream_kernel launch, at most

}  // namespace fa

hipError_t fa_launch_kvcache_slots(const fa::SlotsParams& p, hipStream_t st);
// dtype: FA_DTYPE_* of the new rows; store: FA_STORE_*.
hipError_t fa_launch_kv8_append(int dtype, int store, const fa::Kv8AppendParams& p, int head_dim,
                                hipStream_t st);
hipError_t fa_launch_kv8_attn_f16(int store, const fa::Kv8AttnParams& p, int head_dim, hipStream_t st);
hipError_t fa_launch_kv8_attn_bf16(int store, const fa::Kv8AttnParams& p, int head_dim, hipStream_t st);
