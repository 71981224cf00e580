// sa_paged_tc.h -- launches of the tensor-core attention over a paged bf16
// cache (sa_paged_tc.cu).
#pragma once
#include "sa_internal.h"

namespace sa {
namespace pg {

int tc_prefill_launch(sa_ctx* ctx, const sa_paged_kv* kv, const void* q, long long q_tok, int n_tok, int hq,
                      const int* cu_q, int window, int sinks, float scale, void* out, long long o_tok);
// Key splits of a shared prefix, and the parts that they leave: unnormalised O
// [parts][n_seqs * hq][d] and (m, l) [parts][n_seqs * hq][2].
int tc_prefix_splits(const sa_ctx* ctx, const sa_paged_kv* kv, int hq, int prefix_len, int* parts);
int tc_prefix_launch(sa_ctx* ctx, const sa_paged_kv* kv, const void* q, long long q_tok, int hq, const int* prefix_table,
                     int prefix_len, float scale, int n_split, float* part_o, float* part_ml);

}  // namespace pg
}  // namespace sa
