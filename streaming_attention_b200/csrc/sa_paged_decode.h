// sa_paged_decode.h -- the paged decode's launch and workspace, for the
// shared-prefix decode that runs it on the sequences' own rows.
#pragma once
#include "sa_internal.h"

namespace sa {
namespace pg {

// Shares of (sequence, KV head) pairs that several CTAs hold: unnormalised O
// rows of d floats and (m in the log2 domain, l).
struct DecodeWs {
    float* slot_o;    // [grid][2][G][d]: the first and the last pair of a CTA
    float2* slot_ml;  // [grid][2][G]
    unsigned* count;  // [grid]: shares handed in of the pair whose first one the CTA holds; zero between calls
    int4* pair;       // [n_seqs * hkv]: first CTA (-1: the state is whole), last CTA, first CTA's slot; with `state`
    float* state_o;   // [n_seqs][hq][d]
    float2* state_ml; // [n_seqs][hq]
    int d, out_elt;
};

int decode_grid(const sa_ctx* ctx, const sa_paged_kv* kv, int hq);
// Lays the workspace out at `base` (may be null) and returns its size.
size_t decode_ws_layout(const sa_ctx* ctx, const sa_paged_kv* kv, int hq, bool to_state, void* base, DecodeWs* ws);
// to_state: every pair's state goes to ws (pair, state, slots) and `out` is not
// written.  overlap: the stream's last kernel is a shared prefix's, which started
// after everything that this launch reads was written; the launch may start while
// it runs.
int decode_launch(sa_ctx* ctx, const sa_paged_kv* kv, const void* q, long long q_stride, int hq, int window, int sinks,
                  float scale, void* out, long long o_stride, bool to_state, bool overlap, const DecodeWs& ws);

}  // namespace pg
}  // namespace sa
