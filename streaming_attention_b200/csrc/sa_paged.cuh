// sa_paged.cuh -- what the operators over a paged KV cache share: the view of
// the cache that kernels take, the visible rows of a query under a sliding
// window with first tokens that stay visible, and the host-side checks.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cmath>
#include <cstdint>

#include "sa_internal.h"
#include "sa_paged_plan.h"
#include "sa_ptx.cuh"
#include "sa_tc.cuh"

namespace sa {
namespace pg {

constexpr int MAX_GROUP = 16;      // largest hq / hkv
constexpr float LOG2E = 1.4426950408889634f;      // scores are taken times scale * log2(e)

// The cache as kernels see it: pages of [hkv][page][d] elements.
struct Cache {
    unsigned char* k;
    unsigned char* v;
    const int* table;          // [n_seqs] rows of table_stride entries
    const int* kv_lens;        // [n_seqs]
    long long page_stride;     // elements between pages
    long long table_stride;
    int n_pages, page_log2, hkv, n_seqs, max_pages;
    int* status;               // expired waits
    int* bad;                  // rows and pages outside the cache
};

// Rows of sequence b, within [0, max_pages * page]; a length past what the
// block table can hold is reported and cut.
__device__ __forceinline__ int seq_len(const Cache& c, int b) {
    const int n = c.kv_lens[b], cut = cut_len(n, c.max_pages, c.page_log2);
    if (cut < n) atomicExch(c.bad, SA_STATUS_BAD_INDEX);
    return cut;
}

// The page that a block-table entry names, or -1 (reported) if it is none of
// the pool's.
__device__ __forceinline__ int checked_page(const Cache& c, int entry) {
    if (page_ok(entry, c.n_pages)) return entry;
    atomicExch(c.bad, SA_STATUS_BAD_INDEX);
    return -1;
}

// One warp joins partial softmax states of one query row, lane by lane D / 32
// columns: m = max m_i, l = sum 2^(m_i - m) l_i, O = sum 2^(m_i - m) O_i.
// 32 parts at a time: the lanes fetch their (m, l), then the O rows are read
// eight at once, with nothing between the loads that waits for one of them.
template <int D>
struct Joined {
    static constexpr int V = D / 32;
    float m, l, o[V];                  // l: this lane's share, see total()
    __device__ __forceinline__ Joined() : m(-INFINITY), l(0.f) {
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = 0.f;
    }
    // ml(p) -> (m, l) of part p, read past the L1 cache;  row(p) -> its O row
    template <typename ML, typename ROW>
    __device__ __forceinline__ void add(int parts, int lane, ML ml, ROW row) {
        for (int base = 0; base < parts; base += 32) {
            float2 x = make_float2(-INFINITY, 0.f);
            if (base + lane < parts) x = ml(base + lane);
            float mx = x.x;
#pragma unroll
            for (int off = 16; off; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
            const float M = fmaxf(m, mx);
            if (M == -INFINITY) continue;
            const float corr = ex2(m - M), w = ex2(x.x - M);        // 0 for an empty state
            m = M;
            l = l * corr + w * x.y;
#pragma unroll
            for (int e = 0; e < V; ++e) o[e] *= corr;
            const int n = min(32, parts - base);
            for (int i0 = 0; i0 < n; i0 += 8) {
                float v[8][V], wi[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    wi[i] = __shfl_sync(0xffffffffu, w, (i0 + i) & 31);
                    const bool on = i0 + i < n && wi[i] != 0.f;     // the O of an empty part is not written
                    const float* r = on ? row(base + i0 + i) + lane * V : nullptr;
                    if (!on) wi[i] = 0.f;
                    if constexpr (V == 2) {
                        const float2 y = on ? __ldcg(reinterpret_cast<const float2*>(r)) : make_float2(0.f, 0.f);
                        v[i][0] = y.x; v[i][1] = y.y;
                    } else {
#pragma unroll
                        for (int c = 0; c < V; c += 4) {
                            const float4 y = on ? __ldcg(reinterpret_cast<const float4*>(r + c)) : make_float4(0.f, 0.f, 0.f, 0.f);
                            v[i][c] = y.x; v[i][c + 1] = y.y; v[i][c + 2] = y.z; v[i][c + 3] = y.w;
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < 8; ++i)
#pragma unroll
                    for (int e = 0; e < V; ++e) o[e] = fmaf(wi[i], v[i][e], o[e]);
            }
        }
    }
    // Another warp's state (its o in memory, l summed).
    __device__ __forceinline__ void add_one(int lane, float m2, float l2, const float* row) {
        const float M = fmaxf(m, m2);
        if (M == -INFINITY) return;
        const float wa = ex2(m - M), wb = ex2(m2 - M);
        m = M;
        l = l * wa + (lane == 0 ? l2 * wb : 0.f);
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = o[e] * wa + (wb > 0.f ? row[lane * V + e] * wb : 0.f);
    }
    __device__ __forceinline__ float total() const {
        float t = l;
#pragma unroll
        for (int off = 16; off; off >>= 1) t += __shfl_xor_sync(0xffffffffu, t, off);
        return t;
    }
    // The lane's columns of the normalised row, in OT.
    template <typename OT>
    __device__ __forceinline__ void store(OT* dst, int lane) const {
        const float f = row_factor(total());
        dst += lane * V;
        if constexpr (sizeof(OT) == 4) {
#pragma unroll
            for (int e = 0; e < V; e += 2) *reinterpret_cast<float2*>(dst + e) = make_float2(o[e] * f, o[e + 1] * f);
        } else {
#pragma unroll
            for (int e = 0; e < V; e += 2)
                *reinterpret_cast<__nv_bfloat162*>(dst + e) = __floats2bfloat162_rn(o[e] * f, o[e + 1] * f);
        }
    }
};

// The tokens of a ragged batch cut into units of up to `per` tokens of one
// sequence, numbered over the batch.
struct SeqUnit {
    int b, unit;            // sequence, unit of it
    int first, tokens;      // the sequence's first row in the token tensors, its tokens
    int len;                // its rows
};
// Tokens of a sequence; a range outside the token tensors is reported and counts
// as none.
__device__ __forceinline__ int seq_tokens(const Cache& c, int c0, int c1, int n_tok) {
    const int n = token_count(c0, c1, n_tok);
    if (n >= 0) return n;
    atomicExch(c.bad, SA_STATUS_BAD_INDEX);
    return 0;
}
// Unit total - 1 - back of the batch, by the whole block (scan: THREADS / 32
// numbers); false when there is none.
template <int THREADS>
__device__ bool find_seq_unit(const Cache& c, const int* cu_q, int n_tok, int per, int back, SeqUnit* s, unsigned* scan) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int run = (c.n_seqs + THREADS - 1) / THREADS;
    const int b0 = min(c.n_seqs, tid * run), b1 = min(c.n_seqs, b0 + run);
    unsigned mine = 0;
    const int len0 = b0 < b1 ? seq_len(c, b0) : 0;       // in flight with cu_q: most runs are one sequence
    for (int b = b0; b < b1; b += 8) {                   // eight loads in flight where runs are long
        int cu[9];
#pragma unroll
        for (int u = 0; u < 9; ++u) cu[u] = cu_q[min(b + u, b1)];
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (b + u < b1) mine = add_units(mine, unit_count(seq_tokens(c, cu[u], cu[u + 1], n_tok), per), THREADS);
    }
    unsigned inc = mine;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const unsigned up = __shfl_up_sync(0xffffffffu, inc, off);
        if (lane >= off) inc += up;
    }
    if (lane == 31) scan[warp] = inc;
    __syncthreads();
    unsigned before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
        if (w < warp) before += scan[w];
        total += scan[w];
    }
    if ((unsigned)back >= total) return false;
    const unsigned want = total - 1u - (unsigned)back;
    unsigned at = before + inc - mine;
    if (want >= at && want - at < mine) {
        const int b = unit_sequence(cu_q, b0, b1, n_tok, per, want, &at);
        s->b = b;
        s->unit = (int)(want - at);
        s->first = cu_q[b];
        s->tokens = cu_q[b + 1] - cu_q[b];
        s->len = b == b0 ? len0 : seq_len(c, b);
    }
    __syncthreads();
    return true;
}

// ---- host ------------------------------------------------------------------
inline int log2_exact(int x) {
    int l = 0;
    while ((1 << l) < x) ++l;
    return (1 << l) == x ? l : -1;
}

// Checks of a cache description that every entry point makes.
inline int check_cache(const char* fn, const sa_paged_kv* kv) {
    SA_CHECK_ARG(kv != nullptr, "%s: kv is NULL", fn);
    SA_CHECK_ARG(kv->dtype == SA_F32 || kv->dtype == SA_BF16, "%s: dtype %d (want SA_F32 or SA_BF16)", fn, kv->dtype);
    SA_CHECK_ARG(kv->k_pages && kv->v_pages, "%s: null k_pages/v_pages", fn);
    SA_CHECK_ARG(kv->d == 64 || kv->d == 128 || kv->d == 256, "%s: d = %d (supported: 64, 128, 256)", fn, kv->d);
    SA_CHECK_ARG(kv->page_size == 16 || kv->page_size == 32 || kv->page_size == 64 || kv->page_size == 128,
                 "%s: page_size = %d (supported: 16, 32, 64, 128)", fn, kv->page_size);
    SA_CHECK_ARG(kv->hkv >= 1 && kv->hkv <= SA_MAX_KV_HEADS, "%s: hkv = %d (1..%d)", fn, kv->hkv, SA_MAX_KV_HEADS);
    SA_CHECK_ARG(kv->n_pages >= 1, "%s: n_pages = %d", fn, kv->n_pages);
    SA_CHECK_ARG(kv->n_seqs >= 0 && kv->n_seqs <= SA_PAGED_MAX_SEQS, "%s: n_seqs = %d (0..%d)", fn, kv->n_seqs,
                 SA_PAGED_MAX_SEQS);
    SA_CHECK_ARG(kv->max_pages >= 0 && kv->table_stride >= kv->max_pages, "%s: max_pages %d, table_stride %lld", fn,
                 kv->max_pages, kv->table_stride);
    SA_CHECK_ARG((long long)kv->max_pages * kv->page_size <= 0x7ffffe00LL,
                 "%s: %d pages of %d rows per sequence exceed the 2^31 positions of a sequence", fn, kv->max_pages,
                 kv->page_size);
    SA_CHECK_ARG(kv->n_seqs == 0 || (kv->kv_lens && (kv->max_pages == 0 || kv->block_table)),
                 "%s: null block_table/kv_lens", fn);
    const int e = kv->dtype == SA_F32 ? 4 : 2;
    SA_CHECK_ARG(kv->page_stride >= (long long)kv->hkv * kv->page_size * kv->d && kv->page_stride * e % 16 == 0,
                 "%s: page_stride %lld (at least hkv * page_size * d = %lld elements, a multiple of 16 bytes)", fn,
                 kv->page_stride, (long long)kv->hkv * kv->page_size * kv->d);
    SA_CHECK_ARG((((uintptr_t)kv->k_pages | (uintptr_t)kv->v_pages) & 15) == 0,
                 "%s: k_pages/v_pages not 16-byte aligned", fn);
    return SA_OK;
}

inline int check_heads(const char* fn, const sa_paged_kv* kv, int hq) {
    SA_CHECK_ARG(hq >= 1 && hq % kv->hkv == 0 && hq / kv->hkv <= MAX_GROUP, "%s: hq = %d, hkv = %d (hq/hkv 1..%d)", fn,
                 hq, kv->hkv, MAX_GROUP);
    SA_CHECK_ARG(kv->d < 256 || hq / kv->hkv <= 8, "%s: hq/hkv = %d at d = 256 (at most 8)", fn, hq / kv->hkv);
    return SA_OK;
}

inline int check_scale(const char* fn, float scale) {
    SA_CHECK_ARG(scale > 0.f && std::isfinite(scale * LOG2E),
                 "%s: scale = %g (want a positive number that log2(e) = 1.4427 times is finite in fp32)", fn, (double)scale);
    return SA_OK;
}

// A row tensor's token stride and address.
inline int check_rows(const char* fn, const char* what, const void* p, long long stride, long long width, int e) {
    SA_CHECK_ARG(p != nullptr && ((uintptr_t)p & 15) == 0, "%s: %s is NULL or not 16-byte aligned", fn, what);
    SA_CHECK_ARG(stride >= width && stride * e % 16 == 0,
                 "%s: %s token stride %lld (at least %lld elements, a multiple of 16 bytes)", fn, what, stride, width);
    return SA_OK;
}

inline Cache make_cache(const sa_ctx* ctx, const sa_paged_kv* kv) {
    Cache c;
    c.k = static_cast<unsigned char*>(kv->k_pages);
    c.v = static_cast<unsigned char*>(kv->v_pages);
    c.table = kv->block_table;
    c.kv_lens = kv->kv_lens;
    c.page_stride = kv->page_stride;
    c.table_stride = kv->table_stride;
    c.n_pages = kv->n_pages;
    c.page_log2 = log2_exact(kv->page_size);
    c.hkv = kv->hkv;
    c.n_seqs = kv->n_seqs;
    c.max_pages = kv->max_pages;
    c.status = ctx->status;
    c.bad = ctx->status + 1;
    return c;
}

// 3-D bf16 tensor map (d, rows of a page, pages) over a pool, box 64 columns x
// box_rows rows x 1 page, 128-byte swizzle.  A page coordinate outside the
// pool reads zeros.
inline int make_page_tmap(CUtensorMap* map, const void* pages, const sa_paged_kv* kv, int box_rows) {
    const uint64_t n[3] = {(uint64_t)kv->d, (uint64_t)kv->hkv * kv->page_size, (uint64_t)kv->n_pages};
    const uint64_t stride[2] = {(uint64_t)kv->d, (uint64_t)kv->page_stride};
    const uint32_t box[3] = {64, (uint32_t)box_rows, 1};
    return make_tmap_3d_bf16(map, pages, n, stride, box);
}
// 3-D bf16 tensor map (d, heads, tokens) over query rows, box 64 columns x
// `group` heads x `toks` tokens, 128-byte swizzle: rows land token after token.
inline int make_query_tmap(CUtensorMap* map, const void* q, int d, int hq, int n_tokens, long long tok_stride, int group,
                           int toks) {
    const uint64_t n[3] = {(uint64_t)d, (uint64_t)hq, (uint64_t)n_tokens};
    const uint64_t stride[2] = {(uint64_t)d, (uint64_t)tok_stride};
    const uint32_t box[3] = {64, (uint32_t)group, (uint32_t)toks};
    return make_tmap_3d_bf16(map, q, n, stride, box);
}

}  // namespace pg
}  // namespace sa
