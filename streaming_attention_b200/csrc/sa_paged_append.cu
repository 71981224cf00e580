// sa_paged_append.cu -- new tokens' keys and values written into the pages of
// their sequences, with the rotary embedding of keys and queries applied on
// the way, and the table of rotation angles.
//
// Rotation of a head x at position p with R rotated elements, i < R/2:
//   a' = a cos(p w_i) - b sin(p w_i),   b' = b cos(p w_i) + a sin(p w_i)
// on the pairs (a, b) = (x[i], x[i + R/2]) or, interleaved, (x[2i], x[2i+1]);
// elements R.. pass through.  All in fp32 from the table's fp32 cosines and
// sines; each result is rounded once, to the cache's type.
//
// Bound: HBM.  A token's rows are read once and written once; the table row
// (R/2 cosines and sines) is shared by all of its heads.  Measured: 8418 tokens
// of 16/8 heads of 128 bf16 (140 MB in and out) 28.5 us, 4.9 TB/s; 8 tokens 2.6 us.
#include <cuda_bf16.h>
#include <algorithm>
#include <cmath>

#include "sa_paged.cuh"

namespace sa {
namespace pg {

constexpr int AT = 256;        // threads per CTA

struct AppendArgs {
    Cache c;
    const void *q, *k, *v;               // q may be null
    void* q_out;
    long long q_stride, k_stride, v_stride, qo_stride;   // elements between tokens
    const int* cu_q;                     // null: one token per sequence
    const float *cos_t, *sin_t;          // [n_pos][R/2], null: no rotation
    int n_pos, rot, interleaved;
    int n_tokens, hq, d, pos0, head_log2;
};

// Eight elements as they lie in memory.
template <typename T> struct Raw8 {
    static constexpr int N = sizeof(T) / 2;
    uint4 w[N];
    __device__ __forceinline__ void load(const T* p) {       // read once
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
    }
    __device__ __forceinline__ void floats(float* f) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t v[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (N == 2) {
                    f[4 * i + j] = __uint_as_float(v[j]);
                } else {
                    f[2 * j] = __uint_as_float(v[j] << 16);
                    f[2 * j + 1] = __uint_as_float(v[j] & 0xffff0000u);
                }
            }
        }
    }
};
// table rows are shared by a token's heads: kept in the cache
__device__ __forceinline__ void load4t(const float* p, float* f) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(p));
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
}
template <typename T> __device__ __forceinline__ void store8(T* p, const float* f);
template <> __device__ __forceinline__ void store8<float>(float* p, const float* f) {
    *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
    *(reinterpret_cast<float4*>(p) + 1) = make_float4(f[4], f[5], f[6], f[7]);
}
template <> __device__ __forceinline__ void store8<__nv_bfloat16>(__nv_bfloat16* p, const float* f) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

// Where token `tok` goes: its position, and its page and row there (page -1:
// nowhere -- behind the last sequence, or a bad index, which is reported).
struct Place {
    int pos, page, row;
};

// One warp finds a token's sequence: the number of starts cu_q[1..] at or
// before it, 32 sequences at a time; the lane of the sequence has its length
// and first token in hand.
__device__ __forceinline__ Place find_place(const AppendArgs& a, int tok, int lane) {
    Place p;
    p.pos = 0;
    p.page = -1;
    p.row = 0;
    int b = tok, t = 0, n = 1, len = 0;
    if (a.cu_q) {
        b = 0;
        for (int base = 0; base < a.c.n_seqs; base += 32) {
            const int i = base + lane;
            int c0 = 0, c1 = 0x7fffffff, l = 0;
            if (i < a.c.n_seqs) {
                c0 = a.cu_q[i];
                c1 = a.cu_q[i + 1];
                l = a.c.kv_lens[i];
            }
            const int got = __popc(__ballot_sync(0xffffffffu, c1 <= tok));
            b += got;
            if (got == 32) continue;
            c0 = __shfl_sync(0xffffffffu, c0, got);
            n = __shfl_sync(0xffffffffu, c1, got) - c0;
            len = __shfl_sync(0xffffffffu, l, got);
            t = tok - c0;
            break;
        }
    }
    if (b >= a.c.n_seqs || t < 0) return p;              // a row of no sequence
    if (!a.cu_q) {
        len = a.c.kv_lens[b];
        if (len <= 0) return p;                          // an empty slot of a padded batch
    }
    const long long at = append_row(len, n, t, a.c.max_pages, a.c.page_log2, a.pos0, a.cos_t ? a.n_pos : 1LL << 40);
    if (at < 0) {
        if (lane == 0) atomicExch(a.c.bad, SA_STATUS_BAD_INDEX);
        return p;
    }
    p.pos = (int)(a.pos0 + at);
    p.row = (int)(at & ((1 << a.c.page_log2) - 1));
    p.page = checked_page(a.c, a.c.table[(long long)b * a.c.table_stride + (at >> a.c.page_log2)]);
    return p;
}

// WPT warps per token, each by itself: it looks up the token's place while its
// first rows are on their way.  A lane moves items of two groups of eight
// elements of one head, half the rotated part (or half the rest) apart: the two
// halves of eight rotated pairs.  A head has d / 16 items, so a lane's item is
// the same one of every head it meets and its angles are fetched once.
template <typename T, typename KT, int WPT, int U>
__global__ void __launch_bounds__(AT, 2) append_kernel(const AppendArgs a) {
    const int lane = threadIdx.x & 31;
    const long long w = (long long)blockIdx.x * (AT / 32) + (threadIdx.x >> 5);
    const long long tok = w / WPT;
    if (tok >= a.n_tokens) return;
    const int head_log2 = a.head_log2;
    const int nq = a.q ? a.hq : 0, nk = nq + a.c.hkv;
    const int items = (nk + a.c.hkv) << head_log2;
    const int g = lane & ((1 << head_log2) - 1);
    const bool turns = g < a.rot / 16;
    // where the item lies in a head that is rotated, and in one that is not
    const int r0 = turns ? g * 8 : a.rot + (g - a.rot / 16) * 8, r1 = r0 + (turns ? a.rot : a.d - a.rot) / 2;
    const int v0 = g * 8, v1 = v0 + a.d / 2;
    float c[8], s[8];
    bool found = false;
    Place pl;
    for (int base = (int)(w % WPT) * 32; base < items; base += U * WPT * 32) {
        Raw8<T> x[U], y[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int it = base + u * WPT * 32 + lane, h = it >> head_log2;
            if (it < items) {
                const T* src = h < nq   ? static_cast<const T*>(a.q) + tok * a.q_stride + (long long)h * a.d
                               : h < nk ? static_cast<const T*>(a.k) + tok * a.k_stride + (long long)(h - nq) * a.d
                                        : static_cast<const T*>(a.v) + tok * a.v_stride + (long long)(h - nk) * a.d;
                x[u].load(src + (h < nk ? r0 : v0));
                y[u].load(src + (h < nk ? r1 : v1));
            }
        }
        if (!found) {
            pl = find_place(a, (int)tok, lane);
            if (pl.page < 0) return;
            found = true;
            if (turns) {
                const long long r = (long long)pl.pos * (a.rot / 2);
                if (a.interleaved) {                      // four pairs in each group
                    load4t(a.cos_t + r + g * 4, c);
                    load4t(a.sin_t + r + g * 4, s);
                    load4t(a.cos_t + r + a.rot / 4 + g * 4, c + 4);
                    load4t(a.sin_t + r + a.rot / 4 + g * 4, s + 4);
                } else {
                    load4t(a.cos_t + r + g * 8, c);
                    load4t(a.sin_t + r + g * 8, s);
                    load4t(a.cos_t + r + g * 8 + 4, c + 4);
                    load4t(a.sin_t + r + g * 8 + 4, s + 4);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int it = base + i * WPT * 32 + lane, h = it >> head_log2;
            if (it >= items) continue;
            float u[8], v[8];
            x[i].floats(u);
            y[i].floats(v);
            if (h < nk && turns) {
                if (a.interleaved) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float ua = u[2 * e], ub = u[2 * e + 1], va = v[2 * e], vb = v[2 * e + 1];
                        u[2 * e] = ua * c[e] - ub * s[e];
                        u[2 * e + 1] = ub * c[e] + ua * s[e];
                        v[2 * e] = va * c[4 + e] - vb * s[4 + e];
                        v[2 * e + 1] = vb * c[4 + e] + va * s[4 + e];
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float p = u[e], q = v[e];
                        u[e] = p * c[e] - q * s[e];
                        v[e] = q * c[e] + p * s[e];
                    }
                }
            }
            KT* dst = h < nq ? static_cast<KT*>(a.q_out) + tok * a.qo_stride + (long long)h * a.d
                             : reinterpret_cast<KT*>(h < nk ? a.c.k : a.c.v) + (long long)pl.page * a.c.page_stride +
                                   (((long long)(h < nk ? h - nq : h - nk) << a.c.page_log2) + pl.row) * a.d;
            store8<KT>(dst + (h < nk ? r0 : v0), u);
            store8<KT>(dst + (h < nk ? r1 : v1), v);
        }
    }
}

template <typename T, typename KT>
static int append_launch(cudaStream_t st, int num_sms, const AppendArgs& a) {
    // A warp per token with four items in flight where that fills the GPU (8418
    // tokens of 16/8 heads of 128 bf16: 28.2 us against 35-44 of a CTA per token,
    // which looks every token's place up eight times); below, a CTA per token
    // spreads the rows over more SMs (8 tokens: 2.5 us against 5.6).
    if (a.n_tokens >= 16 * num_sms)
        append_kernel<T, KT, 1, 4><<<(a.n_tokens + AT / 32 - 1) / (AT / 32), AT, 0, st>>>(a);
    else
        append_kernel<T, KT, AT / 32, 1><<<a.n_tokens, AT, 0, st>>>(a);
    SA_CUDA_TRY(cudaGetLastError());
    return SA_OK;
}

// cos / sin [n_pos][R/2] of p * theta^(-2i/R): angles in 64 bits (a far
// position times a frequency loses its fraction of a turn in 32), reduced to
// a fraction of a turn before they are rounded.
__global__ void rope_angles_kernel(int n_pos, int half, double log2_theta, float* cos_t, float* sin_t) {
    const long long n = (long long)n_pos * half;
    for (long long idx = blockIdx.x * (long long)blockDim.x + threadIdx.x; idx < n;
         idx += (long long)gridDim.x * blockDim.x) {
        const long long p = idx / half;
        const int i = (int)(idx - p * half);
        const double turns = (double)p * (exp2(-log2_theta * i / half) * 0.15915494309189533577);
        const double frac = turns - rint(turns);
        double s, c;
        sincospi(2.0 * frac, &s, &c);
        cos_t[idx] = (float)c;
        sin_t[idx] = (float)s;
    }
}

}  // namespace pg
}  // namespace sa

SA_API int sa_rope_table(sa_ctx* ctx, int n_pos, int rotary_dim, double theta, float* cos_t, float* sin_t) {
    using namespace sa;
    clear_error();
    SA_CHECK_ARG(n_pos >= 1 && rotary_dim >= 2 && rotary_dim % 2 == 0, "sa_rope_table: n_pos %d, rotary_dim %d", n_pos,
                 rotary_dim);
    SA_CHECK_ARG(theta > 1.0 && theta < 1e18, "sa_rope_table: theta = %g", theta);
    SA_CHECK_ARG(cos_t && sin_t, "sa_rope_table: null table");
    SA_CHECK_ARG(ctx != nullptr, "sa_rope_table: ctx is NULL");
    DeviceGuard guard(ctx->device);
    const long long n = (long long)n_pos * (rotary_dim / 2);
    const int grid = (int)std::min<long long>((n + 255) / 256, 8LL * ctx->num_sms);
    pg::rope_angles_kernel<<<grid, 256, 0, ctx->stream>>>(n_pos, rotary_dim / 2, std::log2(theta), cos_t, sin_t);
    SA_CUDA_TRY(cudaGetLastError());
    return SA_OK;
}

SA_API int sa_paged_append(sa_ctx* ctx, const sa_paged_kv* kv, int x_dtype, const void* q, long long q_tok_stride,
                           const void* k, long long k_tok_stride, const void* v, long long v_tok_stride, int n_tokens,
                           int hq, const int* cu_q, int pos0, const float* cos_t, const float* sin_t, int n_pos,
                           int rotary_dim, int interleaved, void* q_out, long long qo_tok_stride) {
    using namespace sa;
    const char* fn = "sa_paged_append";
    clear_error();
    SA_RC_TRY(pg::check_cache(fn, kv));
    SA_CHECK_ARG(x_dtype == SA_F32 || x_dtype == SA_BF16, "%s: x_dtype %d (want SA_F32 or SA_BF16)", fn, x_dtype);
    SA_CHECK_ARG(n_tokens >= 0 && pos0 >= 0, "%s: n_tokens %d, pos0 %d", fn, n_tokens, pos0);
    SA_CHECK_ARG(!!cos_t == !!sin_t, "%s: one of cos and sin is NULL", fn);
    SA_CHECK_ARG(!q || q_out, "%s: q without q_out", fn);
    const int d = kv->d, e = x_dtype == SA_F32 ? 4 : 2, eo = kv->dtype == SA_F32 ? 4 : 2;
    if (cos_t) {
        SA_CHECK_ARG(rotary_dim >= 16 && rotary_dim <= d && rotary_dim % 16 == 0,
                     "%s: rotary_dim = %d (a multiple of 16, at most d = %d)", fn, rotary_dim, d);
        SA_CHECK_ARG(n_pos >= 1, "%s: n_pos = %d", fn, n_pos);
        SA_CHECK_ARG((((uintptr_t)cos_t | (uintptr_t)sin_t) & 15) == 0, "%s: cos/sin not 16-byte aligned", fn);
    }
    if (n_tokens == 0 || kv->n_seqs == 0) return SA_OK;
    SA_RC_TRY(pg::check_rows(fn, "k", k, k_tok_stride, (long long)kv->hkv * d, e));
    SA_RC_TRY(pg::check_rows(fn, "v", v, v_tok_stride, (long long)kv->hkv * d, e));
    if (q) {
        SA_CHECK_ARG(hq >= 1, "%s: hq = %d", fn, hq);
        SA_RC_TRY(pg::check_rows(fn, "q", q, q_tok_stride, (long long)hq * d, e));
        SA_RC_TRY(pg::check_rows(fn, "q_out", q_out, qo_tok_stride, (long long)hq * d, eo));
    }
    SA_CHECK_ARG(ctx != nullptr, "%s: ctx is NULL", fn);
    DeviceGuard guard(ctx->device);
    pg::AppendArgs a;
    a.c = pg::make_cache(ctx, kv);
    a.q = q; a.k = k; a.v = v; a.q_out = q_out;
    a.q_stride = q_tok_stride; a.k_stride = k_tok_stride; a.v_stride = v_tok_stride; a.qo_stride = qo_tok_stride;
    a.cu_q = cu_q;
    a.cos_t = cos_t; a.sin_t = sin_t;
    a.n_pos = n_pos; a.rot = cos_t ? rotary_dim : 0; a.interleaved = interleaved ? 1 : 0;
    a.n_tokens = n_tokens; a.hq = hq; a.d = d; a.pos0 = pos0;
    a.head_log2 = pg::log2_exact(d / 16);
    const bool xf = x_dtype == SA_F32, cf = kv->dtype == SA_F32;
    using bf = __nv_bfloat16;
    if (xf) return cf ? pg::append_launch<float, float>(ctx->stream, ctx->num_sms, a)
                      : pg::append_launch<float, bf>(ctx->stream, ctx->num_sms, a);
    return cf ? pg::append_launch<bf, float>(ctx->stream, ctx->num_sms, a)
              : pg::append_launch<bf, bf>(ctx->stream, ctx->num_sms, a);
}
