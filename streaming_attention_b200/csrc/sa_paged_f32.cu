// sa_paged_f32.cu -- attention of many query rows over a paged fp32 KV cache:
// the prefill and the shared prefix's part of a decode, as sa_paged_tc.cu does
// them for bf16.
//
// fp32 results from the tensor cores, three tf32 products each (sa_tf32.cuh).
//
// A CTA of eight warps holds FM query rows (FM / G tokens times the G heads of a
// KV head) and walks over tiles of 64 keys: S = Q K^T with 16 rows per warp (32 at
// FM = 128: an operand is split once for twice the products), the warps of a row
// group sharing the keys; the row maximum and P through shared memory; O += P V with
// the row group's warps sharing O's columns.  K and V of the next tile are copied
// (cp.async) as soon as their buffers are free: K under the softmax and P V, V under
// the next S; the page of the tile after it is looked up meanwhile.  Rows that no
// query of the CTA sees are not read but zero-filled.
//
// Bound: the tensor pipe (0.63 busy over 4096 causal tokens) with the splits and the
// softmax between its products; small calls by the latency of few dependent tiles.
// Measured: 16 sequences behind 4001 rows, 16/8 heads of 128: 22.9 us for the
// prefix (42 on FMAs); three chunks of up to 300 tokens, 8/4 heads of 64, window
// 129: 21.8 us (29); 4096 tokens, 16/8 heads of 128: 1260 us, 55 TFLOP/s (45 with 64
// rows) of the 97 that three products of mma.sync give -- tcgen05's kind::tf32, half
// of bf16's rate, would give 282; errors against 64 bits 2e-7.  A CTA walks over all
// keys of its rows, so few tokens after a long cache leave SMs idle: 16 tokens, 32768
// rows: 2.2 ms.
#include <algorithm>
#include <cmath>

#include "sa_paged.cuh"
#include "sa_paged_f32.h"
#include "sa_tf32.cuh"

namespace sa {
namespace pg {

constexpr int FN = 64, FT = 256;

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

template <int D, int FM>
struct FLay {
    // Row strides of 4 mod 32 words: the eight rows of an ldmatrix, and the V
    // elements of a fragment (rows two apart, eight columns), hit all banks.
    static constexpr int RS = D + 4, PS = FN + 4;
    static constexpr int MR = FM == 128 ? 2 : 1;       // 16-row blocks per warp
    static constexpr int WM = FM / 16 / MR, WN = 8 / WM;    // warps over rows; over keys, then over columns
    static constexpr int Q = 0, K = FM * RS, V = K + FN * RS, P = V + FN * RS, X = P + FM * PS;
    static constexpr int SMEM = (X + WN * FM) * 4;
};

// c[n] += A B[n] of sixteen products.
template <int N>
__device__ __forceinline__ void add_product(float (*c)[4], const FragA<2>& a, const FragB<2> (&b)[N]) {
    float d[N][4];
    mma_exact(d, [&](int) -> const FragA<2>& { return a; }, b);
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) c[n][e] += d[n][e];
}
// 8x4 blocks of 32-bit words: lane's word is (lane / 4, lane % 4) of each block,
// lane l gives the address of row l % 8 of block l / 8.
__device__ __forceinline__ void ldsm4w(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
    uint32_t r;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(r) : "r"(addr) : "memory");
    return r;
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool on) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <int D, int FM, bool PREFIX>
__global__ void __launch_bounds__(FT, (FM == 32 || (FM == 64 && D == 64)) ? 2 : 1) paged_f32_kernel(const __grid_constant__ F32Args a) {
    using L = FLay<D, FM>;
    constexpr int MR = L::MR;
    constexpr int NT = FN / L::WN / 8;                   // 8-key blocks of S per warp
    constexpr int CT = D / L::WN / 8;                    // 8-column blocks of O per warp
    constexpr int NG = NT < 4 ? NT : 4, CG = CT < 4 ? CT : 4;    // blocks whose products interleave
    extern __shared__ __align__(16) float smf[];
    __shared__ SeqUnit s_seq;
    __shared__ unsigned s_scan[FT / 32];
    float *sQ = smf + L::Q, *sK = smf + L::K, *sV = smf + L::V, *sP = smf + L::P, *sX = smf + L::X;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int wm = warp % L::WM, wn = warp / L::WM;      // the warp's 16 MR rows; its keys and columns
    const int fr = lane >> 2, fc = lane & 3;             // row and word of a fragment
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

    // ---- copies: four threads per key row
    const int cr = tid >> 2, cq = tid & 3;
    const uint32_t kdst = smem_u32(sK + cr * L::RS + cq * 4), vdst = smem_u32(sV + cr * L::RS + cq * 4);
    // this thread's row of tile j: its page, looked up a tile before it is needed;
    // its place in the pools, -1: zeros
    auto seen = [&](int j, int row) { return j < n_kv && t.sees(row); };
    auto look = [&](int j) {
        const int row = t.row0(j0 + j, FN) + cr;
        return seen(j, row) ? row_table[row >> a.c.page_log2] : 0;
    };
    auto place = [&](int j, int entry) -> long long {
        const int row = t.row0(j0 + j, FN) + cr;
        if (!seen(j, row)) return -1;
        const int page = checked_page(a.c, entry);
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
    int entry = look(0);
    const long long at = place(0, entry);
    entry = look(1);
    if (n_kv > 0) {
        copy(kdst, a.c.k, at);
        copy(vdst, a.c.v, at);
    }

    // ---- Q, scaled (into exponents of two) on the way
    constexpr int QL = FM * (D / 4) / FT;                // float4 per thread
    float4 qv[QL];
#pragma unroll
    for (int u = 0; u < QL; ++u) {
        const int i = tid + u * FT, r = i / (D / 4), c4 = i - r * (D / 4), tk = r / a.G, g = r - tk * a.G;
        qv[u] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (tk < ntok)
            qv[u] = *reinterpret_cast<const float4*>(a.q + (long long)(tok0 + tk) * a.q_tok +
                                                     (long long)(kvh * a.G + g) * D + c4 * 4);
    }
#pragma unroll
    for (int u = 0; u < QL; ++u) {
        const int i = tid + u * FT, r = i / (D / 4), c4 = i - r * (D / 4);
        *reinterpret_cast<float4*>(sQ + r * L::RS + c4 * 4) =
            make_float4(qv[u].x * a.qscale, qv[u].y * a.qscale, qv[u].z * a.qscale, qv[u].w * a.qscale);
    }

    // what this lane's rows (fr and fr + 8 of each block) see
    const int wr = wm * MR * 16 + fr;
    int lo[2 * MR], first[2 * MR];
    unsigned span[2 * MR];
#pragma unroll
    for (int i = 0; i < 2 * MR; ++i) {
        const int limit = PREFIX ? len - 1 : p0 + (wr + 8 * i) / a.G;
        lo[i] = PREFIX ? 0 : window_lo(limit, a.window);
        span[i] = limit < 0 ? 0u : (unsigned)(limit - lo[i] + 1);
        first[i] = PREFIX ? 0 : min(a.sinks, limit + 1);
    }
    const int all_lo = PREFIX ? 0 : window_lo(p0 + ntok - 1, a.window);
    float m[2 * MR], l[2 * MR], o[MR][CT][4];
#pragma unroll
    for (int i = 0; i < 2 * MR; ++i) m[i] = -INFINITY, l[i] = 0.f;
#pragma unroll
    for (int r = 0; r < MR; ++r)
#pragma unroll
        for (int c = 0; c < CT; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[r][c][e] = 0.f;
    // ldmatrix addresses: A (16 rows x 8 words): blocks by rows, then words; B (two
    // 8-key blocks x 8 words): blocks by words, then keys
    const int ar = wm * MR * 16 + (lane & 15), aw = (lane >> 4) * 4;
    const uint32_t qa = smem_u32(sQ + ar * L::RS + aw), pa = smem_u32(sP + ar * L::PS + aw);
    const uint32_t kb = smem_u32(sK + (wn * NT * 8 + (lane >> 4) * 8 + (lane & 7)) * L::RS + ((lane >> 3) & 1) * 4);
    // V: the eight keys of a step enter in the order that P's accumulator has them
    const uint32_t vb = smem_u32(sV + 2 * fc * L::RS + wn * CT * 8 + fr);
    auto load_a = [&](FragA<2> (&x)[MR], uint32_t at_, int stride) {
#pragma unroll
        for (int r = 0; r < MR; ++r)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                uint32_t w[4];
                ldsm4w(w, at_ + (r * 16 * stride + 8 * u) * 4);
#pragma unroll
                for (int e = 0; e < 4; ++e) split_tf32(w[e], x[r].h[u][e], x[r].l[u][e]);
            }
    };

    for (int j = 0; j < n_kv; ++j) {
        const long long next = place(j + 1, entry);
        entry = look(j + 2);
        cp_wait<1>();                                    // K of this tile (V is the group after it)
        __syncthreads();
        float s[MR][NT][4];
#pragma unroll
        for (int r = 0; r < MR; ++r)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[r][n][e] = 0.f;
#pragma unroll 2
        for (int k = 0; k < D; k += 16) {
            FragA<2> x[MR];
            load_a(x, qa + k * 4, L::RS);
#pragma unroll
            for (int n = 0; n < NT; n += NG) {
                FragB<2> y[NG];
#pragma unroll
                for (int i = 0; i < NG; i += 2)
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        uint32_t w[4];
                        ldsm4w(w, kb + ((n + i) * 8 * L::RS + k + 8 * u) * 4);
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            split_tf32(w[e], y[i + (e >> 1)].h[u][e & 1], y[i + (e >> 1)].l[u][e & 1]);
                    }
#pragma unroll
                for (int r = 0; r < MR; ++r) add_product(s[r] + n, x[r], y);
            }
        }
        // accumulator: rows fr, fr + 8; keys 2 fc, 2 fc + 1 of each block
        const int k0 = t.row0(j0 + j, FN);
        if (k0 + FN - 1 > p0 || !(k0 >= all_lo || k0 + FN <= a.sinks)) {
#pragma unroll
            for (int r = 0; r < MR; ++r)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int key = k0 + (wn * NT + n) * 8 + 2 * fc + (e & 1), i = 2 * r + (e >> 1);
                        if ((unsigned)(key - lo[i]) >= span[i] && key >= first[i]) s[r][n][e] = -INFINITY;
                    }
        }
        float mx[2 * MR];
#pragma unroll
        for (int i = 0; i < 2 * MR; ++i) {
            const int r = i >> 1, e = 2 * (i & 1);
            mx[i] = fmaxf(s[r][0][e], s[r][0][e + 1]);
#pragma unroll
            for (int n = 1; n < NT; ++n) mx[i] = fmaxf(mx[i], fmaxf(s[r][n][e], s[r][n][e + 1]));
            mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
            mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
            if (fc == 0) sX[wn * FM + wr + 8 * i] = mx[i];
        }
        __syncthreads();                                 // the other warps' maxima; everyone is done with K
        if (j + 1 < n_kv) copy(kdst, a.c.k, next);
#pragma unroll
        for (int i = 0; i < 2 * MR; ++i) {
            const int r = i >> 1, e = 2 * (i & 1);
#pragma unroll
            for (int w = 0; w < L::WN; ++w) mx[i] = fmaxf(mx[i], sX[w * FM + wr + 8 * i]);
            const float M = fmaxf(m[i], mx[i]), z = M == -INFINITY ? 0.f : M;
            const float corr = ex2(m[i] - z);            // m = -inf: 0
            m[i] = M;
            float ps = 0.f;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const float p0_ = ex2(s[r][n][e] - z), p1_ = ex2(s[r][n][e + 1] - z);
                ps += p0_ + p1_;
                // key 2 fc goes to word fc of the step, key 2 fc + 1 to word fc + 4
                float* dst = sP + (wr + 8 * i) * L::PS + (wn * NT + n) * 8 + fc;
                dst[0] = p0_;
                dst[4] = p1_;
            }
            l[i] = l[i] * corr + ps;                     // this lane's keys; added up at the end
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                o[r][c][e] *= corr;
                o[r][c][e + 1] *= corr;
            }
        }
        if (j + 1 < n_kv) cp_wait<1>();                  // V of this tile (K of the next came after it)
        else cp_wait<0>();
        __syncthreads();                                 // P and V are there
#pragma unroll 2
        for (int k = 0; k < FN; k += 16) {
            FragA<2> x[MR];
            load_a(x, pa + k * 4, L::PS);
#pragma unroll
            for (int c = 0; c < CT; c += CG) {
                FragB<2> y[CG];
#pragma unroll
                for (int i = 0; i < CG; ++i)
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            split_tf32(lds32(vb + ((k + 8 * u + e) * L::RS + (c + i) * 8) * 4), y[i].h[u][e],
                                       y[i].l[u][e]);
#pragma unroll
                for (int r = 0; r < MR; ++r) add_product(o[r] + c, x[r], y);
            }
        }
        __syncthreads();                                 // V and P are free
        if (j + 1 < n_kv) copy(vdst, a.c.v, next);
    }

    // a row's sum: over its four lanes, then over the row group's warps
#pragma unroll
    for (int i = 0; i < 2 * MR; ++i) {
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
        if (fc == 0) sX[wn * FM + wr + 8 * i] = l[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2 * MR; ++i) {
        const int r = wr + 8 * i, tk = r / a.G, g = r - tk * a.G;
        if (tk >= ntok) continue;
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < L::WN; ++w) sum += sX[w * FM + r];
        const int h = kvh * a.G + g;
        float* dst;
        float f = 1.f;
        if constexpr (PREFIX) {
            const long long row = ((long long)split * a.n_tok + tok0 + tk) * a.hq + h;
            if (wn == 0 && fc == 0) *reinterpret_cast<float2*>(a.part_ml + row * 2) = make_float2(m[i], sum);
            dst = a.part_o + row * D;
        } else {
            dst = a.out + (long long)(tok0 + tk) * a.o_tok + (long long)h * D;
            f = row_factor(sum);
        }
#pragma unroll
        for (int c = 0; c < CT; ++c)
            *reinterpret_cast<float2*>(dst + (wn * CT + c) * 8 + 2 * fc) = 
                make_float2(o[i >> 1][c][2 * (i & 1)] * f, o[i >> 1][c][2 * (i & 1) + 1] * f);
    }
}

template <int D, int FM, bool PREFIX>
static int f32_launch_k(cudaStream_t st, long long grid, const F32Args& a) {
    SA_CHECK_ARG(grid < (1LL << 31), "fp32 attention: %lld CTAs", grid);
    auto k = paged_f32_kernel<D, FM, PREFIX>;
    SA_RC_TRY(set_smem_attr_once((const void*)k, FLay<D, FM>::SMEM));
    k<<<(unsigned)grid, FT, FLay<D, FM>::SMEM, st>>>(a);
    SA_CUDA_TRY(cudaGetLastError());
    return SA_OK;
}
template <bool PREFIX>
static int f32_launch(int d, int fm, cudaStream_t st, long long grid, const F32Args& a) {
    if (d == 64)
        return fm == 32 ? f32_launch_k<64, 32, PREFIX>(st, grid, a) : f32_launch_k<64, 64, PREFIX>(st, grid, a);
    return fm == 32   ? f32_launch_k<128, 32, PREFIX>(st, grid, a)
           : fm == 64 ? f32_launch_k<128, 64, PREFIX>(st, grid, a)
                      : f32_launch_k<128, 128, PREFIX>(st, grid, a);
}

int f32_prefill_launch(sa_ctx* ctx, const sa_paged_kv* kv, const float* q, long long q_tok, int n_tok, int hq,
                       const int* cu_q, int window, int sinks, float scale, float* out, long long o_tok) {
    F32Args a = {};
    a.c = make_cache(ctx, kv);
    a.q = q; a.cu_q = cu_q; a.q_tok = q_tok; a.o_tok = o_tok;
    a.n_tok = n_tok; a.hq = hq; a.G = hq / kv->hkv;
    a.window = window; a.sinks = sinks;
    a.qscale = scale * LOG2E;
    a.out = out;
    // 64 rows read K and V half as often as 32; 32 where 64 would leave SMs idle
    const int seqs = std::min(kv->n_seqs, n_tok);
    auto units = [&](int fm) { return ((long long)n_tok / (fm / a.G) + seqs) * kv->hkv; };
    int fm = units(64) < 2 * ctx->num_sms ? 32 : 64;
    // 128 for d = 128 where the average sequence has 16 units of them (the last is
    // partly empty) and they go round the SMs: 4096 tokens, 16/8 heads: 1260 us (64
    // rows: 1520), 2048: 474 (598); not yet for 4 x 512 (eight units): 175 (147), nor
    // for 8 x 130, 64/8 heads: 202 (182).  At d = 64 the halved splits do not pay for
    // the halved occupancy: 701 (687)
    if (kv->d == 128 && n_tok / seqs >= 16 * (128 / a.G) && 2 * units(128) >= 3 * ctx->num_sms) fm = 128;
    a.tpt = fm / a.G;
    return f32_launch<false>(kv->d, fm, ctx->stream, units(fm), a);
}

// Rows of a CTA behind a shared prefix: 32 where they hold all rows of a KV head; 128
// for d = 128 where that leaves no more rows empty than 64: 4000 rows, 200 query rows
// per head: 98 us (64 rows: 125), 128: 64.6 (66.7); 144 would take two CTAs for three:
// 95.6 (92.7).
static int f32_prefix_rows(const sa_paged_kv* kv, int G) {
    if (kv->n_seqs <= 32 / G) return 32;
    auto units = [&](int fm) { return (kv->n_seqs + fm / G - 1) / (fm / G); };
    return kv->d == 128 && 2 * units(128) <= units(64) + units(64) / 8 ? 128 : 64;
}

int f32_prefix_splits(const sa_ctx* ctx, const sa_paged_kv* kv, int hq, int prefix_len) {
    const int G = hq / kv->hkv, fm = f32_prefix_rows(kv, G), tpt = fm / G, units = (kv->n_seqs + tpt - 1) / tpt;
    const int tiles = (int)(((long long)prefix_len + FN - 1) / FN);
    const int slots = ctx->num_sms * ((fm == 32 || (fm == 64 && kv->d == 64)) ? 2 : 1);
    return std::max(1, std::min(tiles, slots / std::max(1, units * kv->hkv)));
}

int f32_prefix_launch(sa_ctx* ctx, const sa_paged_kv* kv, const float* q, long long q_tok, int hq,
                      const int* prefix_table, int prefix_len, float scale, int n_split, float* part_o, float* part_ml) {
    F32Args a = {};
    a.c = make_cache(ctx, kv);
    a.q = q; a.q_tok = q_tok;
    a.n_tok = kv->n_seqs; a.hq = hq; a.G = hq / kv->hkv;
    const int fm = f32_prefix_rows(kv, a.G);
    a.tpt = fm / a.G;
    a.qscale = scale * LOG2E;
    a.prefix_table = prefix_table; a.prefix_len = prefix_len;
    a.n_split = n_split;
    a.units = (kv->n_seqs + a.tpt - 1) / a.tpt;
    a.part_o = part_o; a.part_ml = part_ml;
    return f32_launch<true>(kv->d, fm, ctx->stream, (long long)a.units * kv->hkv * n_split, a);
}

}  // namespace pg
}  // namespace sa
