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
// (R/2 cosines and sines) is shared by all of its heads.
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
    int n_tokens, hq, d, pos0;
};

template <typename T> __device__ __forceinline__ void load8(const T* p, float* f);
template <> __device__ __forceinline__ void load8<float>(const float* p, float* f) {
    const float4 a = __ldcs(reinterpret_cast<const float4*>(p)), b = __ldcs(reinterpret_cast<const float4*>(p) + 1);
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}
template <> __device__ __forceinline__ void load8<__nv_bfloat16>(const __nv_bfloat16* p, float* f) {
    const uint4 r = __ldcs(reinterpret_cast<const uint4*>(p));
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = __uint_as_float(w[i] << 16);
        f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
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
// before it, 32 at a time.
__device__ __forceinline__ Place find_place(const AppendArgs& a, int tok, int lane) {
    Place p;
    p.pos = 0;
    p.page = -1;
    p.row = 0;
    int b = tok, t = 0, n = 1;
    if (a.cu_q) {
        b = 0;
        for (int base = 0; base < a.c.n_seqs; base += 32) {
            const int i = base + lane;
            const bool at = i < a.c.n_seqs && a.cu_q[i + 1] <= tok;
            const int got = __popc(__ballot_sync(0xffffffffu, at));
            b += got;
            if (got < 32) break;
        }
        if (b < a.c.n_seqs) {
            const int c0 = a.cu_q[b];
            t = tok - c0;
            n = a.cu_q[b + 1] - c0;
        }
    }
    if (b >= a.c.n_seqs || t < 0) return p;              // a row of no sequence
    const int len = a.c.kv_lens[b];
    if (len <= 0 && !a.cu_q) return p;                   // an empty slot of a padded batch
    const long long at = append_row(len, n, t, a.c.max_pages, a.c.page_log2, a.pos0, a.cos_t ? a.n_pos : 1LL << 40);
    if (at < 0) {
        if (lane == 0) atomicExch(a.c.status, SA_STATUS_BAD_INDEX);
        return p;
    }
    p.pos = (int)(a.pos0 + at);
    p.row = (int)(at & ((1 << a.c.page_log2) - 1));
    p.page = checked_page(a.c, a.c.table[(long long)b * a.c.table_stride + (at >> a.c.page_log2)]);
    return p;
}

// One CTA per token.  A thread moves two groups of eight elements of one head
// at a time: the two halves of eight rotated pairs, or two neighbouring groups.
template <typename T, typename KT>
__global__ void __launch_bounds__(AT) append_kernel(const AppendArgs a) {
    __shared__ Place s_place;
    const int tok = blockIdx.x, tid = threadIdx.x;
    const int per_head = a.d / 16;                       // thread items per head
    const int heads = (a.q ? a.hq : 0) + 2 * a.c.hkv;
    const int nq = a.q ? a.hq : 0;
    const int rot_items = a.rot / 16;
    const int items = heads * per_head;
    bool ready = false;
    Place pl;
    for (int it = tid; it < items || !ready; it += AT) {
        float x[8], y[8];
        int h = 0, g = 0, o0 = 0, o1 = 0;
        const bool on = it < items;
        if (on) {
            h = it / per_head;
            g = it - h * per_head;
            const bool turn = h < nq + a.c.hkv;
            const bool split = turn && !a.interleaved && g < rot_items;
            o0 = split ? g * 8 : g * 16;
            o1 = split ? o0 + a.rot / 2 : o0 + 8;
            const T* src = h < nq ? static_cast<const T*>(a.q) + (long long)tok * a.q_stride + (long long)h * a.d
                           : h < nq + a.c.hkv
                               ? static_cast<const T*>(a.k) + (long long)tok * a.k_stride + (long long)(h - nq) * a.d
                               : static_cast<const T*>(a.v) + (long long)tok * a.v_stride +
                                     (long long)(h - nq - a.c.hkv) * a.d;
            load8<T>(src + o0, x);
            load8<T>(src + o1, y);
        }
        if (!ready) {                                     // the rows are on their way while the place is looked up
            if (tid < 32) {
                const Place p = find_place(a, tok, tid);
                if (tid == 0) s_place = p;
            }
            __syncthreads();
            pl = s_place;
            ready = true;
        }
        if (!on || pl.page < 0) break;
        if (h < nq + a.c.hkv && g < rot_items) {
            const long long r = (long long)pl.pos * (a.rot / 2);
            if (a.interleaved) {                          // eight pairs lie in x then y
                float c[8], s[8];
                load8<float>(a.cos_t + r + g * 8, c);
                load8<float>(a.sin_t + r + g * 8, s);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float xa = x[2 * i], xb = x[2 * i + 1], ya = y[2 * i], yb = y[2 * i + 1];
                    x[2 * i] = xa * c[i] - xb * s[i];
                    x[2 * i + 1] = xb * c[i] + xa * s[i];
                    y[2 * i] = ya * c[4 + i] - yb * s[4 + i];
                    y[2 * i + 1] = yb * c[4 + i] + ya * s[4 + i];
                }
            } else {
                float c[8], s[8];
                load8<float>(a.cos_t + r + o0, c);
                load8<float>(a.sin_t + r + o0, s);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float u = x[i], w = y[i];
                    x[i] = u * c[i] - w * s[i];
                    y[i] = w * c[i] + u * s[i];
                }
            }
        }
        KT* dst;
        if (h < nq) {
            dst = static_cast<KT*>(a.q_out) + (long long)tok * a.qo_stride + (long long)h * a.d;
        } else {
            const bool key = h < nq + a.c.hkv;
            const int kh = key ? h - nq : h - nq - a.c.hkv;
            dst = reinterpret_cast<KT*>(key ? a.c.k : a.c.v) + (long long)pl.page * a.c.page_stride +
                  (((long long)kh << a.c.page_log2) + pl.row) * a.d;
        }
        store8<KT>(dst + o0, x);
        store8<KT>(dst + o1, y);
    }
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
    const bool xf = x_dtype == SA_F32, cf = kv->dtype == SA_F32;
    auto kern = xf ? (cf ? pg::append_kernel<float, float> : pg::append_kernel<float, __nv_bfloat16>)
                   : (cf ? pg::append_kernel<__nv_bfloat16, float> : pg::append_kernel<__nv_bfloat16, __nv_bfloat16>);
    kern<<<n_tokens, pg::AT, 0, ctx->stream>>>(a);
    SA_CUDA_TRY(cudaGetLastError());
    return SA_OK;
}
