// C ABI of the operators around the 8-bit paged KV cache (declarations and
// contracts: include/fa_gfx950.h).  As in fa_api.hip: each entry point checks
// its arguments, fills a parameter block and launches on the caller's stream;
// nothing allocates device memory or synchronizes.
#include <stdarg.h>
#include <stdio.h>

#include "fa_api_internal.h"
#include "fa_common.h"
#include "fa_gfx950.h"
#include "fa_kv8.h"

namespace {

int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return fa_set_error(code, buf);
}

int hip_status(hipError_t e, const char* what) {
  if (e == hipSuccess) return fa_set_error(FA_OK, "");
  return fail(FA_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
}

// Positions are 32-bit in the kernels; windows are clamped below that.
constexpr int64_t kMaxLen = int64_t(1) << 29;
constexpr int64_t kIntMax = 0x7fffffff;
constexpr int64_t kMaxSlotStride = int64_t(1) << 26;   // 16 rows within 32-bit offsets

int clamp_window(int64_t w) {
  const int64_t cap = (int64_t(1) << 30) - 1;
  return w < 0 ? -1 : (int)(w > cap ? cap : w);
}

bool aligned(const void* ptr, const int64_t* strides, int n, int64_t elem, int64_t to) {
  if (reinterpret_cast<uintptr_t>(ptr) % to != 0) return false;
  for (int i = 0; i < n; ++i)
    if (strides[i] * elem % to != 0) return false;
  return true;
}

bool head_dim_ok(int64_t d) { return d == 64 || d == 128 || d == 256; }

// log2 of a scale block of `block` slots, or -1.
int log2_block(int64_t block) {
  for (int i = 4; i < 30; ++i)
    if (block == int64_t(1) << i) return i;
  return -1;
}

// What append and attention ask of the cache's shape.
int check_cache(const char* name, int64_t num_pages, int64_t page_size, int64_t block, int store) {
  if (store != FA_STORE_E4M3 && store != FA_STORE_E5M2)
    return fail(FA_ERR_UNSUPPORTED, "%s: unknown 8-bit type %d", name, store);
  if (log2_block(block) < 0)
    return fail(FA_ERR_UNSUPPORTED, "%s: a scale block must be a power of two of at least 16 slots, not %lld", name,
                (long long)block);
  if (num_pages < 0 || page_size < 1 || page_size > kMaxLen || page_size % block != 0)
    return fail(FA_ERR_INVALID, "%s: page_size must be a positive multiple of the scale block", name);
  if (num_pages > kIntMax || num_pages * (page_size / block) > kIntMax)
    return fail(FA_ERR_UNSUPPORTED, "%s: too many scale blocks", name);
  return FA_OK;
}

struct Plan {
  int positions, part_rows, chunk_blocks, chunk_keys, chunk_splits;
  int64_t each;        // sequences per launch
  int64_t rows;        // partial rows
  int64_t workspace;   // bytes
};

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Which kernel takes the launch and how the keys are split.  No more is known
// of the lengths than max_keys.
Plan make_plan(int64_t batch, int64_t seqlen_q, int64_t total_q, int64_t heads_q, int64_t heads_k,
               int64_t head_dim, int64_t max_keys) {
  Plan pl = {};
  const int64_t group = heads_q / heads_k, rows = seqlen_q * group;
  max_keys = max_keys > 0 ? max_keys : 1;
  pl.each = batch > 0 ? batch : 1;
  if (rows <= fa::kKv8StreamRows) {
    // As many workgroups as are resident at once.  A workgroup per sequence, and
    // no merge, where there are enough of them and none is long, or all are short
    // (Hk 8 D 128, bf16, in stretches / whole, MI355X: 64 sequences of 500 to 1000
    // keys 41 / 26 us, of 1000 to 2000 56 / 46, of 512 to 8192 129 / 145; 16 of 500
    // to 1000 20.2 / 14.9; 200 of 500 to 1000 83 / 70; 32 of 512 to 8192 74.6 / 77.6).
    const int64_t slots = head_dim == 256 ? 256 : 512;
    const bool whole = max_keys <= 512 || (batch * heads_k >= 128 && max_keys <= 4096);
    pl.positions = whole ? 0 : (int)ceil_div(slots, heads_k);
    if (!whole) {   // a launch adds up the tiles of its sequences, in 32 bits
      const int64_t most = (int64_t(1) << 30) / (max_keys / 32 + 2);
      pl.each = pl.each < most ? pl.each : most;
      pl.each = pl.each < fa::kKv8Scan ? pl.each : fa::kKv8Scan;
    }
    pl.part_rows = (int)rows;
    pl.rows = pl.positions > 0 ? (pl.each + pl.positions) * heads_k * rows : 0;
    pl.workspace = pl.positions > 0 ? pl.rows * (head_dim + 1) * 4 + (pl.each + 2) * 4 : 0;
  } else {
    const int64_t most = batch * ceil_div(rows, fa::kKv8ChunkRows);
    const int64_t by_rows = total_q * group / fa::kKv8ChunkRows + batch;
    pl.chunk_blocks = (int)(most < by_rows ? most : by_rows);
    // A workgroup per row block and K/V head; the keys are split only where these
    // do not fill the GPU (a split writes and reads its rows in fp32).
    const int64_t wgs = heads_k * pl.chunk_blocks;
    int64_t n = wgs >= 256 ? 1 : ceil_div(512, wgs);
    const int64_t cap = ceil_div(max_keys, 512);
    n = n < cap ? n : cap;
    pl.chunk_keys = (int)(ceil_div(ceil_div(max_keys, n), 64) * 64);
    pl.chunk_splits = (int)ceil_div(max_keys, pl.chunk_keys);
    pl.rows = pl.chunk_splits > 1 ? pl.chunk_splits * total_q * heads_q : 0;
    pl.workspace = pl.rows * (head_dim + 1) * 4;
  }
  return pl;
}

int check_plan(const char* name, int64_t batch, int64_t seqlen_q, int64_t total_q, int64_t heads_q,
               int64_t heads_k, int64_t head_dim, int64_t max_keys) {
  if (batch < 0 || seqlen_q < 0 || total_q < 0 || heads_q < 1 || heads_k < 1 || max_keys < 0)
    return fail(FA_ERR_INVALID, "%s: negative or zero size", name);
  if (heads_q % heads_k != 0)
    return fail(FA_ERR_INVALID, "%s: heads_q (%lld) must be a multiple of heads_k (%lld)", name,
                (long long)heads_q, (long long)heads_k);
  if (!head_dim_ok(head_dim))
    return fail(FA_ERR_UNSUPPORTED, "%s: head dimension must be 64, 128 or 256, not %lld", name,
                (long long)head_dim);
  if (batch > 65535 || heads_q > 65535 || seqlen_q > kMaxLen || max_keys > kMaxLen ||
      seqlen_q * (heads_q / heads_k) > kMaxLen || total_q > kIntMax)
    return fail(FA_ERR_UNSUPPORTED, "%s: sizes beyond 2^29 rows or keys, or 65535 sequences or heads", name);
  return FA_OK;
}

}  // namespace

extern "C" int fa_kvcache_slots(int32_t* block_table, int64_t block_table_stride, int64_t cols,
                                const int32_t* cache_seqlens, const int32_t* new_seqlens, int64_t batch,
                                const int32_t* free_pages, int64_t n_free, const int32_t* free_start,
                                int64_t page_size, int64_t max_tokens, int64_t* slot_mapping,
                                int32_t* positions, int32_t* cu_seqlens, int32_t* seqlens_out,
                                int32_t* free_end, fa_stream_t stream) {
  const char* name = "fa_kvcache_slots";
  if (batch < 0 || cols < 0 || n_free < 0 || max_tokens < 0 || page_size < 1)
    return fail(FA_ERR_INVALID, "%s: negative size", name);
  if (batch > kIntMax || n_free > kIntMax || max_tokens > kIntMax || cols * page_size > kIntMax ||
      cols > kIntMax || page_size > kMaxLen)
    return fail(FA_ERR_UNSUPPORTED, "%s: more than 2^31 - 1 requests, pages, rows or table positions", name);
  if (cu_seqlens == nullptr || free_end == nullptr ||
      (batch > 0 && (cache_seqlens == nullptr || new_seqlens == nullptr || seqlens_out == nullptr)) ||
      (batch > 0 && cols > 0 && block_table == nullptr) || (n_free > 0 && free_pages == nullptr) ||
      (max_tokens > 0 && (slot_mapping == nullptr || positions == nullptr)))
    return fail(FA_ERR_INVALID, "%s: null pointer", name);
  if (block_table_stride < cols && batch > 1)
    return fail(FA_ERR_INVALID, "%s: the rows of block_table overlap", name);
  fa::SlotsParams p;
  p.table = block_table;
  p.table_stride = block_table_stride;
  p.cols = (int)cols;
  p.cached = cache_seqlens;
  p.added = new_seqlens;
  p.free_pages = free_pages;
  p.n_free = n_free;
  p.free_start = free_start;
  p.slots = slot_mapping;
  p.positions = positions;
  p.cu = cu_seqlens;
  p.seqlens = seqlens_out;
  p.free_end = free_end;
  p.batch = (int)batch;
  p.rows = (int)max_tokens;
  p.page = fa::make_fastdiv((uint32_t)page_size);
  return hip_status(fa_launch_kvcache_slots(p, static_cast<hipStream_t>(stream)), name);
}

extern "C" int fa_kvcache8_append(const void* k, const void* v, const int64_t* k_stride,
                                  const int64_t* v_stride, int dtype, void* k_cache, void* v_cache,
                                  const int64_t* k_cache_stride, const int64_t* v_cache_stride, int store,
                                  uint8_t* k_scale, uint8_t* v_scale, const int64_t* k_scale_stride,
                                  const int64_t* v_scale_stride, const int64_t* slot_mapping, int64_t tokens,
                                  int64_t num_pages, int64_t page_size, int64_t block, int64_t heads_k,
                                  int64_t head_dim, fa_stream_t stream) {
  const char* name = "fa_kvcache8_append";
  if (int st = check_cache(name, num_pages, page_size, block, store); st != FA_OK) return st;
  if (dtype != FA_DTYPE_F16 && dtype != FA_DTYPE_BF16 && dtype != FA_DTYPE_F32)
    return fail(FA_ERR_UNSUPPORTED, "%s: unknown dtype %d", name, dtype);
  if (tokens < 0 || heads_k < 1) return fail(FA_ERR_INVALID, "%s: negative or zero size", name);
  if (!head_dim_ok(head_dim))
    return fail(FA_ERR_UNSUPPORTED, "%s: head dimension must be 64, 128 or 256, not %lld", name,
                (long long)head_dim);
  if (tokens > int64_t(1) << 27 || heads_k > 65535)
    return fail(FA_ERR_UNSUPPORTED, "%s: too many tokens or heads", name);
  if (tokens == 0 || num_pages == 0) return fa_set_error(FA_OK, "");
  if (k == nullptr || v == nullptr || k_cache == nullptr || v_cache == nullptr || k_scale == nullptr ||
      v_scale == nullptr || slot_mapping == nullptr || k_stride == nullptr || v_stride == nullptr ||
      k_cache_stride == nullptr || v_cache_stride == nullptr || k_scale_stride == nullptr ||
      v_scale_stride == nullptr)
    return fail(FA_ERR_INVALID, "%s: null pointer", name);
  const int64_t elem = dtype == FA_DTYPE_F32 ? 4 : 2;
  if (!aligned(k, k_stride, 2, elem, 16) || !aligned(v, v_stride, 2, elem, 16) ||
      !aligned(k_cache, k_cache_stride, 3, 1, 16) || !aligned(v_cache, v_cache_stride, 3, 1, 16))
    return fail(FA_ERR_INVALID, "%s: rows must be 16-byte aligned", name);
  fa::Kv8AppendParams p;
  const void* x[2] = {k, v};
  void* c[2] = {k_cache, v_cache};
  uint8_t* s[2] = {k_scale, v_scale};
  const int64_t* xs[2] = {k_stride, v_stride};
  const int64_t* cs[2] = {k_cache_stride, v_cache_stride};
  const int64_t* ss[2] = {k_scale_stride, v_scale_stride};
  for (int i = 0; i < 2; ++i) {
    p.x[i] = x[i];
    p.x_sr[i] = xs[i][0], p.x_sh[i] = xs[i][1];
    p.cache[i] = static_cast<uint8_t*>(c[i]);
    p.c_sp[i] = cs[i][0], p.c_ss[i] = cs[i][1], p.c_sh[i] = cs[i][2];
    p.scale[i] = s[i];
    p.s_sp[i] = ss[i][0], p.s_sb[i] = ss[i][1], p.s_sh[i] = ss[i][2];
  }
  p.slots = slot_mapping;
  p.rows = (int)tokens;
  p.heads = (int)heads_k;
  p.log2_block = log2_block(block);
  p.num_pages = num_pages;
  p.blocks_per_page = fa::make_fastdiv((uint32_t)(page_size / block));
  return hip_status(fa_launch_kv8_append(dtype, store, p, (int)head_dim, static_cast<hipStream_t>(stream)), name);
}

extern "C" int fa_fwd_kvcache8_plan(int64_t batch, int64_t max_seqlen_q, int64_t total_q,
                                    int64_t heads_q, int64_t heads_k, int64_t head_dim, int64_t max_keys,
                                    int64_t* workspace_bytes) {
  const char* name = "fa_fwd_kvcache8_plan";
  if (workspace_bytes == nullptr) return fail(FA_ERR_INVALID, "%s: null pointer", name);
  if (int st = check_plan(name, batch, max_seqlen_q, total_q, heads_q, heads_k, head_dim, max_keys); st != FA_OK)
    return st;
  *workspace_bytes =
      make_plan(batch, max_seqlen_q, total_q, heads_q, heads_k, head_dim, max_keys).workspace;
  return fa_set_error(FA_OK, "");
}

extern "C" int fa_fwd_kvcache8(const void* q, void* out, const int64_t* q_stride, const int64_t* o_stride, int dtype,
                               const void* k_cache, const void* v_cache, const int64_t* k_cache_stride,
                               const int64_t* v_cache_stride, int store, const uint8_t* k_scale,
                               const uint8_t* v_scale, const int64_t* k_scale_stride,
                               const int64_t* v_scale_stride, const int32_t* cache_seqlens,
                               const int32_t* block_table, int64_t block_table_stride, int64_t block_table_cols,
                               int64_t num_pages, int64_t page_size, int64_t block, const int32_t* cu_seqlens_q, int64_t batch,
                               int64_t max_seqlen_q, int64_t total_q, int64_t max_keys, int64_t heads_q,
                               int64_t heads_k, int64_t head_dim, float softmax_scale, int causal,
                               int64_t window_left, int64_t window_right, float softcap,
                               const float* alibi_slopes, int64_t alibi_batch_stride, void* workspace,
                               int64_t workspace_bytes, fa_stream_t stream) {
  const char* name = "fa_fwd_kvcache8";
  if (int st = check_plan(name, batch, max_seqlen_q, total_q, heads_q, heads_k, head_dim, max_keys); st != FA_OK)
    return st;
  if (int st = check_cache(name, num_pages, page_size, block, store); st != FA_OK) return st;
  if (dtype != FA_DTYPE_F16 && dtype != FA_DTYPE_BF16)
    return fail(FA_ERR_UNSUPPORTED, "%s: queries must be fp16 or bf16", name);
  if (!(softcap >= 0.f)) return fail(FA_ERR_INVALID, "%s: softcap must be non-negative", name);
  if (cu_seqlens_q == nullptr && total_q != batch * max_seqlen_q)
    return fail(FA_ERR_INVALID, "%s: total_q must be batch * max_seqlen_q without cu_seqlens_q", name);
  if (max_keys > (block_table != nullptr ? (block_table_cols < 0 ? 0 : block_table_cols) : 1) * page_size)
    return fail(FA_ERR_INVALID, "%s: max_keys exceeds the block table or the cache rows", name);
  if (batch == 0 || max_seqlen_q == 0 || total_q == 0) return fa_set_error(FA_OK, "");
  if (q == nullptr || out == nullptr || q_stride == nullptr || o_stride == nullptr ||
      (max_keys > 0 && num_pages > 0 &&
       (k_cache == nullptr || v_cache == nullptr || k_scale == nullptr || v_scale == nullptr)) ||
      k_cache_stride == nullptr || v_cache_stride == nullptr || k_scale_stride == nullptr ||
      v_scale_stride == nullptr)
    return fail(FA_ERR_INVALID, "%s: null pointer", name);
  if (!aligned(q, q_stride, 3, 2, 16) || !aligned(out, o_stride, 3, 2, 16) ||
      !aligned(k_cache, k_cache_stride, 3, 1, 16) || !aligned(v_cache, v_cache_stride, 3, 1, 16))
    return fail(FA_ERR_INVALID, "%s: rows must be 16-byte aligned", name);
  // (a slot past the sequence's end reads as zeros by lying past the extent of
  // those before it)
  if (k_cache_stride[1] < head_dim || v_cache_stride[1] < head_dim || k_cache_stride[1] > kMaxSlotStride ||
      v_cache_stride[1] > kMaxSlotStride)
    return fail(FA_ERR_UNSUPPORTED, "%s: slots that overlap or lie more than 2^26 bytes apart", name);
  const Plan pl = make_plan(batch, max_seqlen_q, total_q, heads_q, heads_k, head_dim, max_keys);
  if (workspace_bytes < pl.workspace || (pl.workspace > 0 && workspace == nullptr) ||
      reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
    return fail(FA_ERR_INVALID, "%s: the workspace must be as large as fa_fwd_kvcache8_plan says, and 16-byte aligned",
                name);
  fa::Kv8AttnParams p;
  p.q = q;
  p.o = out;
  p.q_sb = q_stride[0], p.q_ss = q_stride[1], p.q_sh = q_stride[2];
  p.o_sb = o_stride[0], p.o_ss = o_stride[1], p.o_sh = o_stride[2];
  p.k = static_cast<const uint8_t*>(k_cache);
  p.v = static_cast<const uint8_t*>(v_cache);
  p.k_sp = k_cache_stride[0], p.k_ss = k_cache_stride[1], p.k_sh = k_cache_stride[2];
  p.v_sp = v_cache_stride[0], p.v_ss = v_cache_stride[1], p.v_sh = v_cache_stride[2];
  p.ks = k_scale;
  p.vs = v_scale;
  p.ks_sp = k_scale_stride[0], p.ks_sb = k_scale_stride[1], p.ks_sh = k_scale_stride[2];
  p.vs_sp = v_scale_stride[0], p.vs_sb = v_scale_stride[1], p.vs_sh = v_scale_stride[2];
  p.log2_block = log2_block(block);
  p.seqlens = cache_seqlens;
  p.table = block_table;
  p.table_stride = block_table_stride;
  p.cu_q = cu_seqlens_q;
  p.total_q = total_q;
  p.page = fa::make_fastdiv((uint32_t)page_size);
  p.num_pages = (int)num_pages;
  p.first_page = 0;
  p.batch = (int)batch;
  p.seqlen_q = (int)max_seqlen_q;
  p.heads_q = (int)heads_q;
  p.heads_k = (int)heads_k;
  p.max_keys = num_pages > 0 ? (int)max_keys : 0;
  p.group = fa::make_fastdiv((uint32_t)(heads_q / heads_k));
  p.scale = softmax_scale;
  p.softcap = softcap;
  p.alibi = alibi_slopes;
  p.alibi_sb = alibi_batch_stride;
  p.causal = causal != 0;
  p.window_left = clamp_window(window_left);
  p.window_right = clamp_window(window_right);
  p.positions = pl.positions;
  p.part_rows = pl.part_rows;
  p.chunk_blocks = pl.chunk_blocks;
  p.chunk_keys = pl.chunk_keys;
  p.chunk_splits = pl.chunk_splits;
  p.o_part = static_cast<float*>(workspace);
  p.lse_part = p.o_part + pl.rows * head_dim;
  p.starts = reinterpret_cast<int*>(p.lse_part + pl.rows);
  hipStream_t st = static_cast<hipStream_t>(stream);
  // (launches of a large batch follow one another in the same workspace)
  for (int64_t b = 0; b < batch; b += pl.each) {
    fa::Kv8AttnParams c = p;
    c.batch = (int)(batch - b < pl.each ? batch - b : pl.each);
    if (p.seqlens != nullptr) c.seqlens = p.seqlens + b;
    if (p.table != nullptr) c.table = p.table + b * p.table_stride;
    if (p.cu_q != nullptr) c.cu_q = p.cu_q + b;
    if (p.alibi != nullptr) c.alibi = p.alibi + b * p.alibi_sb;
    if (p.table == nullptr) c.first_page = (int)b;
    if (p.cu_q == nullptr) {
      c.q = static_cast<const uint16_t*>(p.q) + b * p.q_sb;
      c.o = static_cast<uint16_t*>(p.o) + b * p.o_sb;
    }
    const hipError_t e = dtype == FA_DTYPE_F16 ? fa_launch_kv8_attn_f16(store, c, (int)head_dim, st)
                                               : fa_launch_kv8_attn_bf16(store, c, (int)head_dim, st);
    if (e != hipSuccess) return hip_status(e, name);
  }
  return fa_set_error(FA_OK, "");
}
