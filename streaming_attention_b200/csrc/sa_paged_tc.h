// sa_paged_tc.h -- launches of the tensor-core attention over a paged bf16
// cache (sa_paged_tc.cu).
#pragma once
#include "sa_internal.h"

namespace sa {
namespace pg {

int tc_prefill_launch(sa_ctx* ctx, const sa_paged_kv* kv, const void* q, long long q_tok, int n_tok, int hq,
                      const int* cu_q, int window, int sinks, float scale, void* out, long long o_tok);
// Key splits of a shared prefix, and the parts that a row may have at most.
int tc_prefix_splits(const sa_ctx* ctx, const sa_paged_kv* kv, int hq, int prefix_len, int* parts);
// The first sequence whose rows have two parts per split (a last row tile that
// has no neighbour takes both slots of its CTA).
inline int tc_prefix_alt_from(int n_seqs, int G) {
    const int tpt = 128 / G, tiles = (n_seqs + tpt - 1) / tpt;
    return tiles % 2 ? (tiles - 1) * tpt : n_seqs;
}
// Leaves unnormalised O [parts][n_seqs * hq][d] and (m, l) [parts][n_seqs * hq][2];
// rows from tc_prefix_alt_from on have parts 2 s and 2 s + 1 of split s, the
// others part s.
int tc_prefix_launch(sa_ctx* ctx, const sa_paged_kv* kv, const void* q, long long q_tok, int hq, const int* prefix_table,
                     int prefix_len, float scale, int n_split, float* part_o, float* part_ml);

}  // namespace pg
}  // namespace sa
