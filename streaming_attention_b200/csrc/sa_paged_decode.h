// sa_paged_decode.h -- the paged decode's launch and workspace, for the
// shared-prefix decode that runs it on the sequences' own rows.
#pragma once
#include "sa_internal.h"

namespace sa {
namespace pg {

// States of (sequence, KV head) pairs: unnormalised O rows of d floats, and
// (m in the log2 domain, l).
struct DecodeWs {
    unsigned* count;  // [SA_PAGED_ZERO_BYTES / 4]: shares handed in of the pair whose first one CTA i holds; zero
                      // between calls
    float* slot_o;    // [grid][2][G][d]: shares of pairs that several CTAs hold, each CTA's first and last pair
    float2* slot_ml;  // [grid][2][G]
    float* state_o;   // [n_seqs][hq][d]: whole pairs, where a prefix's parts are to be joined with them
    float2* state_ml; // [n_seqs][hq]
    int4* pair;       // [n_seqs * hkv]: where a pair's state is: its first CTA (-1: whole), last CTA, first one's slot
    int d, out_elt;
};
// What a shared prefix left: states of every query row, [parts][n_seqs * hq].
struct PrefixParts {
    const float* o;
    const float2* ml;
    int parts;
    bool join;        // false: the launch leaves the pairs' states for a kernel that joins them with the parts
};

int decode_grid(const sa_ctx* ctx, const sa_paged_kv* kv, int hq);
// Lays the workspace out at `base` (may be null) and returns its size; prefix:
// with room for whole pairs' states.
size_t decode_ws_layout(const sa_ctx* ctx, const sa_paged_kv* kv, int hq, bool prefix, void* base, DecodeWs* ws);
// prefix (may be null): the rows of a shared prefix come before each sequence's
// own.  Where it has parts, the kernel that computes them is before this launch on
// the stream, and started after everything else that the launch reads was written:
// the launch may start while it runs, and waits for it before it joins.  Kernels
// that other threads enqueued may lie between the two: each ends after the one
// before it, so the wait (for the last of them) covers the parts, and they have
// workspaces of their own.
int decode_launch(sa_ctx* ctx, const sa_paged_kv* kv, const void* q, long long q_stride, int hq, int window, int sinks,
                  float scale, void* out, long long o_stride, const PrefixParts* prefix, const DecodeWs& ws);

}  // namespace pg
}  // namespace sa
