// sa_paged_f32.h -- launches of the fp32 attention of many query rows over a
// paged cache (sa_paged_f32.cu); as sa_paged_tc.h, with one part per split.
#pragma once
#include "sa_internal.h"

namespace sa {
namespace pg {

int f32_prefill_launch(sa_ctx* ctx, const sa_paged_kv* kv, const float* q, long long q_tok, int n_tok, int hq,
                       const int* cu_q, int window, int sinks, float scale, float* out, long long o_tok);
int f32_prefix_splits(const sa_ctx* ctx, const sa_paged_kv* kv, int hq, int prefix_len);
int f32_prefix_launch(sa_ctx* ctx, const sa_paged_kv* kv, const float* q, long long q_tok, int hq,
                      const int* prefix_table, int prefix_len, float scale, int n_split, float* part_o, float* part_ml);

}  // namespace pg
}  // namespace sa
