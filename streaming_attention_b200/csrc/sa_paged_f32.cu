// sa_paged_f32.cu -- attention of many query rows over a paged fp32 KV cache:
// the prefill and the shared prefix's part of a decode, as sa_paged_tc.cu does
// them for bf16.
//
// fp32 throughout, on FMAs: the tensor cores take no fp32 operands, and tf32 or
// bf16 ones would lose what an fp32 cache is kept for.  Bound: FMA issue
// (4 rows d FLOP per key and head).
//
// A CTA holds 64 query rows (64 / G tokens times the G heads of a KV head)
// and walks over tiles of 64 keys: S = Q K^T with a 4 x 4 piece of S per
// thread, the online softmax on it (a row lies in 16 lanes), P through shared
// memory, O += P V with 4 rows x D / 16 columns per thread.  K and V of the next
// tile are copied (cp.async) as soon as their buffers are free: K under the
// softmax and P V, V under the next S.  Rows that no query of the CTA sees are
// not read but zero-filled.
#include <algorithm>
#include <cmath>

#include "sa_paged.cuh"
#include "sa_paged_f32.h"

namespace sa {
namespace pg {

constexpr int FM = 64, FN = 64, FT = 256;
constexpr float F_LOG2E = 1.4426950408889634f;

struct F32Args {
    Cache c;
    const float* q;
    const int* cu_q;
    long long q_tok, o_tok;
    int n_tok, hq, G, tpt, window, sinks;
    float qscale;
    float* out;
    int prefix_len, n_split, units;
    const int* prefix_table;
    float *part_o, *part_ml;
};

template <int D>
struct FLay {
    static constexpr int QS = D + 4, PS = FN + 4;      // padded rows: float4 reads of 8 rows hit all banks
    static constexpr int Q = 0, K = FM * QS, V = K + FN * QS, P = V + FN * D;
    static constexpr int SMEM = (P + FM * PS) * 4;
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool on) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <int D, bool PREFIX>
__global__ void __launch_bounds__(FT, D == 64 ? 2 : 1) paged_f32_kernel(const __grid_constant__ F32Args a) {
    using L = FLay<D>;
    constexpr int CC = D / 64;                           // float4 columns per thread
    extern __shared__ __align__(16) float smf[];
    __shared__ SeqUnit s_seq;
    __shared__ int s_scan[FT / 32];
    float *sQ = smf + L::Q, *sK = smf + L::K, *sV = smf + L::V, *sP = smf + L::P;
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    if (PREFIX) pdl_trigger();

    int kvh, tok0, ntok, p0, len, j0, n_kv, split = 0;
    Tiles t;
    const int* row_table;
    if constexpr (PREFIX) {
        const int unit = blockIdx.x % a.units, r = blockIdx.x / a.units;
        kvh = r % a.c.hkv;
        split = r / a.c.hkv;
        tok0 = unit * a.tpt;
        ntok = min(a.tpt, a.n_tok - tok0);
        len = a.prefix_len;
        p0 = len - 1;
        const int tiles = (int)(((long long)len + FN - 1) / FN);
        j0 = (int)share_first(split, tiles, a.n_split);
        n_kv = (int)share_first(split + 1, tiles, a.n_split) - j0;
        t = make_unit(0, len - 1, -1, 0, 0, FN).t;
        row_table = a.prefix_table;
    } else {
        if (!find_seq_unit<FT>(a.c, a.cu_q, a.n_tok, a.tpt, blockIdx.x / a.c.hkv, &s_seq, s_scan)) return;
        kvh = blockIdx.x % a.c.hkv;
        const int off = s_seq.unit * a.tpt;
        tok0 = s_seq.first + off;
        ntok = min(a.tpt, s_seq.tokens - off);
        len = s_seq.len;
        p0 = len - s_seq.tokens + off;
        t = make_unit(p0, max(-1, p0 + ntok - 1), -1, a.window, a.sinks, FN).t;
        j0 = 0;
        n_kv = t.n;
        row_table = a.c.table + (long long)s_seq.b * a.c.table_stride;
    }

    // ---- Q, scaled (into exponents of two) on the way
    for (int i = tid; i < FM * (D / 4); i += FT) {
        const int r = i / (D / 4), c4 = i - r * (D / 4), tk = r / a.G, g = r - tk * a.G;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        if (tk < ntok)
            x = *reinterpret_cast<const float4*>(a.q + (long long)(tok0 + tk) * a.q_tok + (long long)(kvh * a.G + g) * D +
                                                 c4 * 4);
        x.x *= a.qscale; x.y *= a.qscale; x.z *= a.qscale; x.w *= a.qscale;
        *reinterpret_cast<float4*>(sQ + r * L::QS + c4 * 4) = x;
    }
    // ---- copies: four threads per key row
    const int cr = tid >> 2, cq = tid & 3;
    const uint32_t kdst = smem_u32(sK + cr * L::QS + cq * 4), vdst = smem_u32(sV + cr * D + cq * 4);
    auto place = [&](int j) -> long long {               // this thread's row of tile j in the pools, -1: zeros
        const int row = t.row0(j0 + j, FN) + cr;
        if (j >= n_kv || !t.sees(row)) return -1;
        const int page = checked_page(a.c, row_table[row >> a.c.page_log2]);
        if (page < 0) return -1;
        return (long long)page * a.c.page_stride +
               (((long long)kvh << a.c.page_log2) + (row & ((1 << a.c.page_log2) - 1))) * D + cq * 4;
    };
    auto copy = [&](uint32_t dst, const unsigned char* pool, long long at) {
        const float* src = reinterpret_cast<const float*>(pool) + (at < 0 ? 0 : at);
#pragma unroll
        for (int c = 0; c < D / 16; ++c) cp16(dst + c * 64, at < 0 ? src : src + c * 16, at >= 0);
        cp_commit();
    };
    long long at = place(0);
    if (n_kv > 0) {
        copy(kdst, a.c.k, at);
        copy(vdst, a.c.v, at);
    }

    // what this thread's rows see
    int lo[4], first[4];
    unsigned span[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int limit = PREFIX ? len - 1 : p0 + (ty * 4 + i) / a.G;
        lo[i] = PREFIX ? 0 : window_lo(limit, a.window);
        span[i] = limit < 0 ? 0u : (unsigned)(limit - lo[i] + 1);
        first[i] = PREFIX ? 0 : min(a.sinks, limit + 1);
    }
    const int all_lo = PREFIX ? 0 : window_lo(p0 + ntok - 1, a.window);
    float m[4], l[4], o[4][CC][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        m[i] = -INFINITY;
        l[i] = 0.f;
#pragma unroll
        for (int c = 0; c < CC; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i][c][e] = 0.f;
    }

    for (int j = 0; j < n_kv; ++j) {
        const long long next = place(j + 1);
        cp_wait<1>();                                    // K of this tile (V is the group after it)
        __syncthreads();
        float s[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) s[i][k] = 0.f;
#pragma unroll 4
        for (int c = 0; c < D; c += 4) {
            float4 qv[4], kv[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) qv[i] = *reinterpret_cast<const float4*>(sQ + (ty * 4 + i) * L::QS + c);
#pragma unroll
            for (int k = 0; k < 4; ++k) kv[k] = *reinterpret_cast<const float4*>(sK + (tx + 16 * k) * L::QS + c);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    s[i][k] = fmaf(qv[i].x, kv[k].x, s[i][k]);
                    s[i][k] = fmaf(qv[i].y, kv[k].y, s[i][k]);
                    s[i][k] = fmaf(qv[i].z, kv[k].z, s[i][k]);
                    s[i][k] = fmaf(qv[i].w, kv[k].w, s[i][k]);
                }
        }
        const int k0 = t.row0(j0 + j, FN);
        if (k0 + FN - 1 > p0 || !(k0 >= all_lo || k0 + FN <= a.sinks)) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int key = k0 + tx + 16 * k;
                    if ((unsigned)(key - lo[i]) >= span[i] && key >= first[i]) s[i][k] = -INFINITY;
                }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float mx = fmaxf(fmaxf(s[i][0], s[i][1]), fmaxf(s[i][2], s[i][3]));
#pragma unroll
            for (int off = 1; off < 16; off <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
            const float M = fmaxf(m[i], mx), z = M == -INFINITY ? 0.f : M;
            const float corr = ex2(m[i] - z);            // m = -inf: 0
            float ps = 0.f;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float p = ex2(s[i][k] - z);
                ps += p;
                sP[(ty * 4 + i) * L::PS + tx + 16 * k] = p;
            }
            l[i] = l[i] * corr + ps;                     // this lane's keys; the 16 lanes are added at the end
            m[i] = M;
#pragma unroll
            for (int c = 0; c < CC; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[i][c][e] *= corr;
        }
        cp_wait<0>();                                    // V of this tile
        __syncthreads();                                 // and everyone is done with K, and P is there
        if (j + 1 < n_kv) copy(kdst, a.c.k, next);
#pragma unroll 4
        for (int k = 0; k < FN; k += 4) {
            float4 pv[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) pv[i] = *reinterpret_cast<const float4*>(sP + (ty * 4 + i) * L::PS + k);
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int c = 0; c < CC; ++c) {
                    const float4 v = *reinterpret_cast<const float4*>(sV + (k + e) * D + c * 64 + tx * 4);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float p = e == 0 ? pv[i].x : e == 1 ? pv[i].y : e == 2 ? pv[i].z : pv[i].w;
                        o[i][c][0] = fmaf(p, v.x, o[i][c][0]);
                        o[i][c][1] = fmaf(p, v.y, o[i][c][1]);
                        o[i][c][2] = fmaf(p, v.z, o[i][c][2]);
                        o[i][c][3] = fmaf(p, v.w, o[i][c][3]);
                    }
                }
        }
        __syncthreads();                                 // V and P are free
        if (j + 1 < n_kv) copy(vdst, a.c.v, next);
    }

#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int off = 1; off < 16; off <<= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], off);
        const int r = ty * 4 + i, tk = r / a.G, g = r - tk * a.G;
        if (tk >= ntok) continue;
        const int h = kvh * a.G + g;
        float* dst;
        float f = 1.f;
        if constexpr (PREFIX) {
            const long long row = ((long long)split * a.n_tok + tok0 + tk) * a.hq + h;
            if (tx == 0) *reinterpret_cast<float2*>(a.part_ml + row * 2) = make_float2(m[i], l[i]);
            dst = a.part_o + row * D;
        } else {
            dst = a.out + (long long)(tok0 + tk) * a.o_tok + (long long)h * D;
            f = l[i] > 0.f ? 1.f / l[i] : 0.f;
        }
#pragma unroll
        for (int c = 0; c < CC; ++c)
            *reinterpret_cast<float4*>(dst + c * 64 + tx * 4) =
                make_float4(o[i][c][0] * f, o[i][c][1] * f, o[i][c][2] * f, o[i][c][3] * f);
    }
}

template <int D, bool PREFIX>
static int f32_launch_d(cudaStream_t st, long long grid, const F32Args& a) {
    SA_CHECK_ARG(grid < (1LL << 31), "fp32 attention: %lld CTAs", grid);
    auto k = paged_f32_kernel<D, PREFIX>;
    SA_RC_TRY(set_smem_attr_once((const void*)k, FLay<D>::SMEM));
    k<<<(unsigned)grid, FT, FLay<D>::SMEM, st>>>(a);
    SA_CUDA_TRY(cudaGetLastError());
    return SA_OK;
}

int f32_prefill_launch(sa_ctx* ctx, const sa_paged_kv* kv, const float* q, long long q_tok, int n_tok, int hq,
                       const int* cu_q, int window, int sinks, float scale, float* out, long long o_tok) {
    F32Args a = {};
    a.c = make_cache(ctx, kv);
    a.q = q; a.cu_q = cu_q; a.q_tok = q_tok; a.o_tok = o_tok;
    a.n_tok = n_tok; a.hq = hq; a.G = hq / kv->hkv; a.tpt = FM / a.G;
    a.window = window; a.sinks = sinks;
    a.qscale = scale * F_LOG2E;
    a.out = out;
    const long long units = (long long)n_tok / a.tpt + std::min(kv->n_seqs, n_tok);
    return kv->d == 64 ? f32_launch_d<64, false>(ctx->stream, units * kv->hkv, a)
                       : f32_launch_d<128, false>(ctx->stream, units * kv->hkv, a);
}

int f32_prefix_splits(const sa_ctx* ctx, const sa_paged_kv* kv, int hq, int prefix_len) {
    const int tpt = FM / (hq / kv->hkv), units = (kv->n_seqs + tpt - 1) / tpt;
    const int tiles = (int)(((long long)prefix_len + FN - 1) / FN);
    const int slots = ctx->num_sms * (kv->d == 64 ? 2 : 1);
    return std::max(1, std::min(tiles, slots / std::max(1, units * kv->hkv)));
}

int f32_prefix_launch(sa_ctx* ctx, const sa_paged_kv* kv, const float* q, long long q_tok, int hq,
                      const int* prefix_table, int prefix_len, float scale, int n_split, float* part_o, float* part_ml) {
    F32Args a = {};
    a.c = make_cache(ctx, kv);
    a.q = q; a.q_tok = q_tok;
    a.n_tok = kv->n_seqs; a.hq = hq; a.G = hq / kv->hkv; a.tpt = FM / a.G;
    a.qscale = scale * F_LOG2E;
    a.prefix_table = prefix_table; a.prefix_len = prefix_len;
    a.n_split = n_split;
    a.units = (kv->n_seqs + a.tpt - 1) / a.tpt;
    a.part_o = part_o; a.part_ml = part_ml;
    const long long grid = (long long)a.units * kv->hkv * n_split;
    return kv->d == 64 ? f32_launch_d<64, true>(ctx->stream, grid, a) : f32_launch_d<128, true>(ctx->stream, grid, a);
}

}  // namespace pg
}  // namespace sa
