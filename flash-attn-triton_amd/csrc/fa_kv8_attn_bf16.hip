// Attention over the 8-bit KV cache, BF16 queries.
#include "fa_kv8_attn.h"

hipError_t fa_launch_kv8_attn_bf16(int store, const fa::Kv8AttnParams& p, int head_dim, hipStream_t st) {
  return fa::launch_kv8_attn<fa::BF16>(store, p, head_dim, st);
}
