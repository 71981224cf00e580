// sa_paged_prefix.cu -- the C entries of the paged prefill and of the decode
// behind a shared prefix.
//
// The latter's softmax over [prefix rows, own rows] comes from states (m, l, O) of
// parts of them:
//   m = max m_i,  l = sum 2^(m_i - m) l_i,  O = sum 2^(m_i - m) O_i,  out = O / l.
// The prefix is read once for all sequences: its query rows are the B x G
// (sequence, head) pairs of a KV head, a matrix product with B G rows where a
// decode per sequence would read the prefix B times.  The decode over the
// sequences' own rows starts while that product's last CTAs run, and joins its
// parts with its own states.
#include "sa_paged.cuh"
#include "sa_paged_decode.h"
#include "sa_paged_f32.h"
#include "sa_paged_tc.h"

namespace sa {
namespace pg {

constexpr int JT = 128;

struct JoinArgs {
    Cache c;
    DecodeWs ws;
    void* out;
    long long o_stride;
    int hq, G;
    int parts;
    const float* part_o;
    const float* part_ml;
};

// W warps per (sequence, query head): a share of the prefix's parts each, the last
// one the sequence's own rows too.
template <typename OT, int D, int W>
__global__ void __launch_bounds__(JT) prefix_join_kernel(const __grid_constant__ JoinArgs a) {
    constexpr int V = D / 32, R = JT / 32 / W;             // rows of a CTA
    __shared__ float s_o[R][W][D];
    __shared__ float2 s_ml[R][W];
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) % W, r = (threadIdx.x >> 5) / W;
    const long long row = (long long)blockIdx.x * R + r, rows = (long long)a.c.n_seqs * a.hq;
    if (W == 1 && row >= rows) return;                     // R = 1 otherwise: no such row
    const int b = (int)(row / a.hq), h = (int)(row - (long long)b * a.hq), kvh = h / a.G, g = h - kvh * a.G;
    const int p0 = warp * a.parts / W, p1 = (warp + 1) * a.parts / W;
    Joined<D> s;
    s.add(p1 - p0, lane, [&](int p) { return __ldcg(reinterpret_cast<const float2*>(a.part_ml) + (p0 + p) * rows + row); },
          [&](int p) { return a.part_o + ((p0 + p) * rows + row) * D; });
    if (warp == W - 1 && seq_len(a.c, b) > 0) {
        const int4 rec = a.ws.pair[b * a.c.hkv + kvh];
        if (rec.x < 0) {
            s.add(1, lane, [&](int) { return __ldcg(a.ws.state_ml + row); }, [&](int) { return a.ws.state_o + row * D; });
        } else {
            auto at = [&](int p) { return (2LL * (rec.x + p) + (p == 0 ? rec.z : 0)) * a.G + g; };
            s.add(rec.y - rec.x + 1, lane, [&](int p) { return __ldcg(a.ws.slot_ml + at(p)); },
                  [&](int p) { return a.ws.slot_o + at(p) * D; });
        }
    }
    if constexpr (W > 1) {
        if (warp > 0) {
            const float l = s.total();
            if (lane == 0) s_ml[r][warp] = make_float2(s.m, l);
#pragma unroll
            for (int e = 0; e < V; ++e) s_o[r][warp][lane * V + e] = s.o[e];
        }
        __syncthreads();
        if (warp > 0) return;
#pragma unroll
        for (int w = 1; w < W; ++w) s.add_one(lane, s_ml[r][w].x, s_ml[r][w].y, s_o[r][w]);
    }
    s.store(static_cast<OT*>(a.out) + (long long)b * a.o_stride + (long long)h * D, lane);
}

template <typename OT, int D>
static int join_launch(const sa_ctx* ctx, const JoinArgs& j) {
    const long long rows = (long long)j.c.n_seqs * j.hq;
    if (rows < 8LL * ctx->num_sms)
        SA_CUDA_TRY(launch_pdl(prefix_join_kernel<OT, D, 4>, dim3((unsigned)rows), dim3(JT), 0, ctx->stream, j));
    else
        SA_CUDA_TRY(launch_pdl(prefix_join_kernel<OT, D, 1>, dim3((unsigned)((rows + 3) / 4)), dim3(JT), 0, ctx->stream, j));
    return SA_OK;
}

struct PrefixWs {
    DecodeWs own;
    float *part_o, *part_ml;
    int n_split, parts;
};
static size_t prefix_ws_layout(const sa_ctx* ctx, const sa_paged_kv* kv, int hq, int prefix_len, void* base,
                               PrefixWs* ws) {
    PrefixWs w = {};
    size_t at = align_up(decode_ws_layout(ctx, kv, hq, true, base, &w.own), 256);
    unsigned char* p = static_cast<unsigned char*>(base);
    if (prefix_len > 0) {
        if (kv->dtype == SA_F32) w.parts = w.n_split = f32_prefix_splits(ctx, kv, hq, prefix_len);
        else w.n_split = tc_prefix_splits(ctx, kv, hq, prefix_len, &w.parts);
        const size_t rows = (size_t)w.parts * kv->n_seqs * hq;
        w.part_o = reinterpret_cast<float*>(p ? p + at : nullptr);
        at += align_up(rows * kv->d * 4, 256);
        w.part_ml = reinterpret_cast<float*>(p ? p + at : nullptr);
        at += align_up(rows * 8, 256);
    }
    if (ws) *ws = w;
    return at;
}

static int check_tiled(const char* fn, const sa_paged_kv* kv) {
    SA_CHECK_ARG(kv->d == 64 || kv->d == 128, "%s: d = %d (supported: 64, 128)", fn, kv->d);
    return SA_OK;
}

}  // namespace pg
}  // namespace sa

SA_API int sa_attn_paged_prefill(sa_ctx* ctx, const sa_paged_kv* kv, const void* q, long long q_tok_stride, int n_tokens,
                                 int hq, const int* cu_q, int window, int sinks, float scale, void* out,
                                 long long o_tok_stride) {
    using namespace sa;
    const char* fn = "sa_attn_paged_prefill";
    clear_error();
    SA_RC_TRY(pg::check_cache(fn, kv));
    SA_RC_TRY(pg::check_tiled(fn, kv));
    SA_RC_TRY(pg::check_heads(fn, kv, hq));
    SA_RC_TRY(pg::check_scale(fn, scale));
    SA_CHECK_ARG(window >= 0 && sinks >= 0, "%s: window %d, sinks %d", fn, window, sinks);
    SA_CHECK_ARG(n_tokens >= 0, "%s: n_tokens %d", fn, n_tokens);
    if (n_tokens == 0 || kv->n_seqs == 0) return SA_OK;
    const int e = kv->dtype == SA_F32 ? 4 : 2;
    SA_CHECK_ARG(cu_q != nullptr, "%s: cu_q is NULL", fn);
    SA_RC_TRY(pg::check_rows(fn, "q", q, q_tok_stride, (long long)hq * kv->d, e));
    SA_RC_TRY(pg::check_rows(fn, "out", out, o_tok_stride, (long long)hq * kv->d, e));
    SA_CHECK_ARG(ctx != nullptr, "%s: ctx is NULL", fn);
    DeviceGuard guard(ctx->device);
    if (kv->dtype == SA_F32)
        return pg::f32_prefill_launch(ctx, kv, static_cast<const float*>(q), q_tok_stride, n_tokens, hq, cu_q, window,
                                      sinks, scale, static_cast<float*>(out), o_tok_stride);
    return pg::tc_prefill_launch(ctx, kv, q, q_tok_stride, n_tokens, hq, cu_q, window, sinks, scale, out, o_tok_stride);
}

static int check_prefix(const char* fn, const sa_paged_kv* kv, int hq, const int* prefix_table, int prefix_len) {
    using namespace sa;
    SA_RC_TRY(pg::check_cache(fn, kv));
    SA_RC_TRY(pg::check_tiled(fn, kv));
    SA_RC_TRY(pg::check_heads(fn, kv, hq));
    SA_CHECK_ARG(prefix_len >= 0 && prefix_len <= 0x7ffffe00, "%s: prefix_len %d", fn, prefix_len);
    SA_CHECK_ARG(prefix_len == 0 || prefix_table, "%s: prefix_table is NULL", fn);
    return SA_OK;
}

SA_API int sa_attn_paged_decode_prefix_workspace(sa_ctx* ctx, const sa_paged_kv* kv, int hq, int prefix_len,
                                                 size_t* bytes) {
    using namespace sa;
    const char* fn = "sa_attn_paged_decode_prefix_workspace";
    clear_error();
    static const int any = 0;
    SA_RC_TRY(check_prefix(fn, kv, hq, &any, prefix_len));
    SA_CHECK_ARG(ctx && bytes, "%s: NULL argument", fn);
    *bytes = pg::prefix_ws_layout(ctx, kv, hq, prefix_len, nullptr, nullptr);
    return SA_OK;
}

SA_API int sa_attn_paged_decode_prefix(sa_ctx* ctx, const sa_paged_kv* kv, const int* prefix_table, int prefix_len,
                                       const void* q, long long q_stride, int hq, float scale, void* out,
                                       long long o_stride, void* workspace, size_t workspace_bytes) {
    using namespace sa;
    const char* fn = "sa_attn_paged_decode_prefix";
    clear_error();
    SA_RC_TRY(check_prefix(fn, kv, hq, prefix_table, prefix_len));
    SA_RC_TRY(pg::check_scale(fn, scale));
    if (kv->n_seqs == 0) return SA_OK;
    const int e = kv->dtype == SA_F32 ? 4 : 2;
    SA_RC_TRY(pg::check_rows(fn, "q", q, q_stride, (long long)hq * kv->d, e));
    SA_RC_TRY(pg::check_rows(fn, "out", out, o_stride, (long long)hq * kv->d, e));
    SA_CHECK_ARG(ctx != nullptr, "%s: ctx is NULL", fn);
    DeviceGuard guard(ctx->device);
    pg::PrefixWs ws;
    const size_t need = pg::prefix_ws_layout(ctx, kv, hq, prefix_len, workspace, &ws);
    SA_CHECK_ARG(workspace && ((uintptr_t)workspace & 255) == 0 && workspace_bytes >= need,
                 "%s: workspace of %zu bytes (want %zu, 256-byte aligned)", fn, workspace_bytes, need);
    if (prefix_len > 0) {
        if (kv->dtype == SA_F32)
            SA_RC_TRY(pg::f32_prefix_launch(ctx, kv, static_cast<const float*>(q), q_stride, hq, prefix_table,
                                            prefix_len, scale, ws.n_split, ws.part_o, ws.part_ml));
        else
            SA_RC_TRY(pg::tc_prefix_launch(ctx, kv, q, q_stride, hq, prefix_table, prefix_len, scale, ws.n_split,
                                           ws.part_o, ws.part_ml));
    }
    // Few pairs and parts: the decode's CTAs join the parts themselves.  Else a kernel
    // of its own does (16/8 heads, 8 sequences behind 1000 rows: 13.1 us here, 14.9
    // there; 16 behind 4000: 24.8 and 22.5), with four warps per row where the rows
    // would not fill the GPU (256 rows of 37 parts: 10.0 us, with one warp each 13.0;
    // 2048 rows of 18 parts: 16.0 and 10.6).
    const bool join = kv->n_seqs * kv->hkv <= 64 && ws.parts <= 16;
    const pg::PrefixParts parts = {ws.part_o, reinterpret_cast<const float2*>(ws.part_ml), ws.parts, join};
    SA_RC_TRY(pg::decode_launch(ctx, kv, q, q_stride, hq, 0, 0, scale, out, o_stride, &parts, ws.own));
    if (join) return SA_OK;
    pg::JoinArgs j;
    j.c = pg::make_cache(ctx, kv);
    j.ws = ws.own;
    j.out = out;
    j.o_stride = o_stride;
    j.hq = hq;
    j.G = hq / kv->hkv;
    j.parts = ws.parts;
    j.part_o = ws.part_o;
    j.part_ml = ws.part_ml;
    return kv->dtype == SA_F32 ? (kv->d == 64 ? pg::join_launch<float, 64>(ctx, j) : pg::join_launch<float, 128>(ctx, j))
                               : (kv->d == 64 ? pg::join_launch<__nv_bfloat16, 64>(ctx, j)
                                              : pg::join_launch<__nv_bfloat16, 128>(ctx, j));
}
