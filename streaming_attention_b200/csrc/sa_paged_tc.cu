// sa_paged_tc.cu -- attention of many query rows over a paged bf16 KV cache on
// the 5th-generation tensor cores: causal prefill of a ragged batch of prompt
// chunks with a sliding window and first tokens that stay visible, and the part
// of a shared-prefix decode that all sequences have in common.
//
//   out[i] = sum_j w_ij v_j / sum_j w_ij,  w_ij = 2^(scale log2(e) q_i . k_j - m_i)
// over the rows j that query i sees; m_i is a running maximum.
// P = 2^(..) is rounded to bf16 for the product with V, its sum is not: the tensor
// core takes one type for both operands, and P as the sum of two bf16 numbers would
// be half as much tensor work again where that binds (below).  The error against 64
// bits is 2.0-2.3e-3 of the outputs' size, 1.65e-3 of it the outputs' own rounding.
//
// Rows of a tile: the G = hq / hkv query heads of one KV head for 128 / G
// consecutive tokens, so that every K/V tile serves all heads that read it and
// a window's edges cost the tiles of few tokens.  A CTA holds two such slots of
// 128 rows over the same K/V tiles (neighbouring tokens); the tensor core works
// for one while the other's softmax runs.
//
// The prefix of a shared-prefix decode has no mask: query rows are (sequence,
// head) pairs, the keys are split over CTAs, each leaving (m, l, O) for a join.
// A row tile without a neighbour, there and in a prefill of few tokens, is held
// by both slots, which take alternate key tiles: that keeps the overlap that
// two slots give.
//
// Warp roles, TMEM and the softmax are those of the causal prefill kernel
// (sa_prefill.cu): warp 0 issues the TMA loads of Q and K, warp 2 those of V, one
// lane of warp 1 the MMAs; warps 4-7 and 8-11 are the softmax warpgroups of the
// slots (a thread per row).
// What pages change:
//  * a tile of 128 keys arrives as one box per page and 64-column half, issued
//    by the producer's lanes in parallel, with the block-table entries of the
//    next tile fetched while the ring is full;
//  * a page that none of the CTA's queries sees is not looked up: its box is
//    asked for at a page past the pool, which TMA fills with zeros;
//  * rows behind the sequence's last one share a page with it and may hold
//    anything: K's are masked, V's are overwritten with zeros in shared memory
//    by the softmax threads before the tile's P is handed over.
//
// Bound: the tensor pipe and the exponentials, each busy 56% of the time.
// Measured (16/8 heads of 128, short bursts): 8192 tokens under a window of 4096
// 182-186 us, 1120 TFLOP/s of visible work, 0.66 of the measured bf16 peak; 512 tokens
// over 1100 visible rows 19 us, 1 to 64 after 32700 rows 266 us (a CTA walks over all
// keys of its tokens: 8 CTAs); the prefix part of 64 sequences (32/8 heads) behind
// 32768 rows 40 us, 0.86 PFLOP/s.  A tile of two slots takes some 3150 clocks, of
// which the tensor core works 2048 and a slot's exponentials 1400: with S, P and O
// of two slots TMEM is full, and a slot's S waits for its P.V.
#include <algorithm>
#include <cmath>

#include "sa_fa.cuh"
#include "sa_paged.cuh"
#include "sa_paged_tc.h"

namespace sa {
namespace pg {

using pf::BM;
using pf::BN;
using pf::col_o;
using pf::col_p;
using pf::col_s;
using pf::wait_ab;
using pf::wait_ab_warp;

constexpr int TC_THREADS = 384;
constexpr int TC_REG_CTRL = 72, TC_REG_SOFTMAX = 216;      // 128 * 72 + 256 * 216 = 384 * 168
constexpr int BOX = 128 * 128;                             // 128 rows of 64 bf16

template <int D>
struct Lay {
    static constexpr int HALVES = D / 64;
    static constexpr int TILE = HALVES * BOX;
    static constexpr int ST = D == 64 ? 4 : 2;             // ring depth, K and V each
    static constexpr int Q = 0, K = 2 * TILE, V = K + ST * TILE, BAR = V + ST * TILE;
    static constexpr int SMEM = BAR + 512 + 1024;
};

struct TcArgs {
    Cache c;
    const int* cu_q;           // prefill
    int n_tok;                 // query rows of the q tensor: tokens, or sequences
    int G, tpt;                // heads per KV head; tokens per tile, 128 / G
    int window, sinks;
    float sl2;                 // scale * log2(e)
    void* out;                 // prefill: bf16
    long long o_tok;
    // shared prefix
    int prefix_len, n_split, units;
    const int* prefix_table;
    float* part_o;             // [parts][n_tok * hq][D], unnormalised
    float* part_ml;            // [parts][n_tok * hq][2]
    int hq;
};

template <int ST>
struct TcBars {
    uint64_t q_full;
    uint64_t k_full[ST], k_empty[ST], v_full[ST], v_empty[ST];
    uint64_t s_full[2], p_full[2][2], o_full[2];      // p_full: by slot and half of the keys
    uint64_t drain;
    uint32_t tmem_base;
    int abort;
};

// What this CTA computes.
struct Unit {
    int b, kvh;
    int tok0[2], ntok[2];      // rows of the q tensor
    int p0[2];                 // position of the slot's first query (prefill)
    int len;                   // rows of the sequence / the prefix
    UnitTiles u;
    int j0;                    // first tile (prefix: of the split)
};

// Prefill: CTA u takes unit total - 1 - u of the batch's (the last tokens of a
// sequence see the most rows: they start first).  A unit is the tokens of two
// slots, or of one tile that both slots hold (ALT).
template <bool ALT>
__device__ bool find_prefill_unit(const TcArgs& a, Unit* s, SeqUnit* su, unsigned* scan) {
    const int per = ALT ? a.tpt : 2 * a.tpt;
    if (!find_seq_unit<TC_THREADS>(a.c, a.cu_q, a.n_tok, per, blockIdx.x / a.c.hkv, su, scan)) return false;
    if (threadIdx.x == 0) {
        s->b = su->b;
        s->kvh = blockIdx.x % a.c.hkv;
        s->len = su->len;
        int last[2];
        for (int x = 0; x < 2; ++x) {
            const int t = su->unit * per + (ALT ? 0 : x * a.tpt);
            s->tok0[x] = su->first + t;
            s->ntok[x] = max(0, min(a.tpt, su->tokens - t));
            s->p0[x] = s->len - su->tokens + t;
            last[x] = s->ntok[x] ? max(-1, s->p0[x] + s->ntok[x] - 1) : -1;
        }
        s->u = make_unit(s->p0[0], last[0], last[1], a.window, a.sinks, BN);
        s->j0 = 0;
        if (ALT) {
            const int n = s->u.t.n;
            s->u.n[0] = (n + 1) / 2;
            s->u.n[1] = n / 2;
        }
    }
    __syncthreads();
    return true;
}
// Prefix: CTA = (split, KV head, pair of row tiles), the pair fastest, so that
// CTAs that read the same keys run side by side.
template <bool ALT>
__device__ void find_prefix_unit(const TcArgs& a, Unit* s) {
    if (threadIdx.x == 0) {
        const int unit = blockIdx.x % a.units, r = blockIdx.x / a.units;
        const int split = r / a.c.hkv;
        const int tiles = (int)(((long long)a.prefix_len + BN - 1) / BN);
        s->b = 0;
        s->kvh = r % a.c.hkv;
        s->len = a.prefix_len;
        for (int x = 0; x < 2; ++x) {
            s->tok0[x] = (2 * unit + x) * a.tpt;
            s->ntok[x] = max(0, min(a.tpt, a.n_tok - s->tok0[x]));
            s->p0[x] = a.prefix_len;
        }
        s->j0 = (int)share_first(split, tiles, a.n_split);
        const int n = (int)share_first(split + 1, tiles, a.n_split) - s->j0;
        if (ALT) {
            s->tok0[1] = s->tok0[0];
            s->ntok[1] = s->ntok[0];
        }
        s->u = make_unit(0, a.prefix_len - 1, a.prefix_len - 1, 0, 0, BN);
        s->u.t.n = n;
        s->u.n[0] = ALT ? (n + 1) / 2 : n;
        s->u.n[1] = ALT ? n / 2 : s->ntok[1] ? n : 0;
    }
    __syncthreads();
}

// ALT: both slots hold the same rows and take alternate key tiles.
template <int D, bool PREFIX, bool ALT>
__global__ void __launch_bounds__(TC_THREADS, 1)
paged_tc_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                const __grid_constant__ CUtensorMap tv, const __grid_constant__ TcArgs a) {
    using L = Lay<D>;
    constexpr int ST = L::ST;
    extern __shared__ unsigned char smem_raw[];
    __shared__ Unit s_unit;
    __shared__ SeqUnit s_seq;
    __shared__ unsigned s_scan[TC_THREADS / 32];
    __shared__ float2 s_ml[2][BM];
    const uint32_t raw = smem_u32(smem_raw);
    unsigned char* sm = smem_raw + (((raw + 1023u) & ~1023u) - raw);
    TcBars<ST>* B = reinterpret_cast<TcBars<ST>*>(sm + L::BAR);
    volatile int* abort = &B->abort;
    int* status = a.c.status;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (PREFIX) pdl_trigger();

    if (tid == 0) {
        tc::prefetch_tmap(&tq);
        tc::prefetch_tmap(&tk);
        tc::prefetch_tmap(&tv);
        mbar_init(&B->q_full, 1);
        for (int s = 0; s < ST; ++s) {
            mbar_init(&B->k_full[s], 1);
            mbar_init(&B->k_empty[s], 1);
            mbar_init(&B->v_full[s], 1);
            mbar_init(&B->v_empty[s], 1);
        }
        for (int x = 0; x < 2; ++x) {
            mbar_init(&B->s_full[x], 1);
            mbar_init(&B->p_full[x][0], 4);                // one arrival per softmax warp
            mbar_init(&B->p_full[x][1], 4);
            mbar_init(&B->o_full[x], 1);
        }
        mbar_init(&B->drain, 1);
        B->abort = 0;
        fence_barrier_init();
    }
    if (warp == 1) tc::tmem_alloc(&B->tmem_base, 512);
    bool any = true;
    if constexpr (PREFIX) find_prefix_unit<ALT>(a, &s_unit);
    else any = find_prefill_unit<ALT>(a, &s_unit, &s_seq, s_scan);     // the same for every thread
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t tbase = B->tmem_base;
    if (!any) {
        if (warp == 1) tc::tmem_dealloc(tbase, 512);
        return;
    }
    const Tiles t = s_unit.u.t;
    const int n_kv = t.n, kvh = s_unit.kvh;
    const int n0 = s_unit.u.n[0], n1 = s_unit.u.n[1];
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(TC_REG_CTRL));
        if ((warp == 0 || warp == 2) && n_kv > 0) {
            // ---------------------------------------------- TMA producers: Q and K, V
            const bool is_v = warp == 2;
            if (!is_v && lane == 0) {
                const int slots = (ALT || s_unit.ntok[1] == 0) ? 1 : 2;
                mbar_arrive_expect_tx(&B->q_full, (uint32_t)(slots * L::HALVES * a.tpt * a.G * 128));
                for (int x = 0; x < slots; ++x)
                    for (int f = 0; f < L::HALVES; ++f)
                        tc::tma_load_3d(sm + L::Q + x * L::TILE + f * BOX, &tq, f * 64, kvh * a.G, s_unit.tok0[x],
                                        &B->q_full);
            }
            const CUtensorMap* map = is_v ? &tv : &tk;
            uint64_t *full = is_v ? B->v_full : B->k_full, *empty = is_v ? B->v_empty : B->k_empty;
            unsigned char* ring = sm + (is_v ? L::V : L::K);
            const int pl = a.c.page_log2, page = 1 << pl, copies = BN >> pl;
            const int* row = PREFIX ? a.prefix_table : a.c.table + (long long)s_unit.b * a.c.table_stride;
            const int j0 = s_unit.j0;
            auto wanted = [&](int j) { return lane < copies && t.any(t.row0(j0 + j, BN) + lane * page, page); };
            auto entry = [&](int j) { return wanted(j) ? row[(t.row0(j0 + j, BN) + lane * page) >> pl] : -1; };
            int next = entry(0);
            int issued = 0;
            for (int j = 0; j < n_kv; ++j) {
                const int s = j % ST;
                int pg_id = a.c.n_pages;                         // past the pool: zeros
                if (wanted(j)) {
                    pg_id = checked_page(a.c, next);
                    if (pg_id < 0) pg_id = a.c.n_pages;
                }
                if (j + 1 < n_kv) next = entry(j + 1);
                if (j >= ST && !wait_ab_warp(&empty[s], ((j / ST) & 1) ^ 1, abort, status)) break;
                if (lane == 0) mbar_arrive_expect_tx(&full[s], L::TILE);
                __syncwarp();
                if (lane < copies)
                    for (int f = 0; f < L::HALVES; ++f)
                        tc::tma_load_3d(ring + s * L::TILE + f * BOX + lane * page * 128, map, f * 64, kvh << pl, pg_id,
                                        &full[s]);
                issued = j + 1;
            }
            if (*abort) {                                       // let the loads in flight land
                if (!is_v) mbar_wait(&B->q_full, 0, nullptr);
                for (int j = max(0, issued - ST); j < issued; ++j) mbar_wait(&full[j % ST], (j / ST) & 1, nullptr);
            }
        } else if (warp == 1 && n_kv > 0 && tc::elect_one()) {
            // ---------------------------------------------- MMA issuer
            constexpr uint32_t idS = tc::idesc_bf16_f32(BM, BN, false, false);
            constexpr uint32_t idO = tc::idesc_bf16_f32(BM, D, false, true);
            // descriptors of the first k-step; further ones add to the address field
            const uint64_t dQ = tc::sdesc_sw128(smem_u32(sm + L::Q), 16, 1024);
            const uint64_t dK = tc::sdesc_sw128(smem_u32(sm + L::K), 16, 1024);
            const uint64_t dV = tc::sdesc_sw128(smem_u32(sm + L::V), BOX, 1024);
            auto issue_S = [&](int x, int j) {
                const uint64_t q = dQ + (uint32_t)((ALT ? 0 : x) * (L::TILE >> 4)), k = dK + (uint32_t)((j % ST) * (L::TILE >> 4));
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk) {
                    const uint32_t off = ((kk >> 2) * BOX + (kk & 3) * 32) >> 4;
                    tc::mma_bf16(tbase + col_s(x), q + off, k + off, idS, kk > 0);
                }
            };
            // P.V of slot x's c-th tile, in two halves of 64 keys as P arrives
            auto issue_PV = [&](int x, int j, int c) {
                const uint64_t v = dV + (uint32_t)((j % ST) * (L::TILE >> 4));
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    if (!wait_ab(&B->p_full[x][half], c & 1, abort, status)) return false;
                    tc::fence_after_sync();
#pragma unroll
                    for (int k = 0; k < BN / 32; ++k) {
                        const int kk = half * (BN / 32) + k;
                        tc::mma_bf16_ts(tbase + col_o(x), tbase + col_p(x) + kk * 8, v + (uint32_t)(kk * 2048 >> 4), idO,
                                        kk > 0 ? 1u : (uint32_t)(c > 0));
                    }
                }
                return true;
            };
            auto k_ready = [&](int j) { return wait_ab(&B->k_full[j % ST], (j / ST) & 1, abort, status); };
            auto v_ready = [&](int j) { return wait_ab(&B->v_full[j % ST], (j / ST) & 1, abort, status); };
            bool ok = wait_ab(&B->q_full, 0, abort, status);
            if constexpr (ALT) {
                for (int x = 0; ok && x < 2 && x < n_kv; ++x) {
                    if (!(ok = k_ready(x))) break;
                    tc::fence_after_sync();
                    issue_S(x, x);
                    tc::mma_commit(&B->s_full[x]);
                    tc::mma_commit(&B->k_empty[x % ST]);
                }
                for (int j = 0; ok && j < n_kv; ++j) {
                    const int x = j & 1, c = j >> 1;
                    if (!(ok = v_ready(j) && issue_PV(x, j, c))) break;
                    tc::mma_commit(&B->v_empty[j % ST]);
                    if (j + 2 >= n_kv) {
                        tc::mma_commit(&B->o_full[x]);
                        continue;
                    }
                    if (!(ok = k_ready(j + 2))) break;
                    tc::fence_after_sync();
                    issue_S(x, j + 2);
                    tc::mma_commit(&B->s_full[x]);
                    tc::mma_commit(&B->k_empty[(j + 2) % ST]);
                }
            } else {
                ok = ok && k_ready(0);
                tc::fence_after_sync();
                if (ok) {
                    for (int x = 0; x < 2; ++x)
                        if (0 < (x ? n1 : n0)) {
                            issue_S(x, 0);
                            tc::mma_commit(&B->s_full[x]);
                        }
                    tc::mma_commit(&B->k_empty[0]);
                }
                for (int j = 0; ok && j < n_kv; ++j) {
                    if (!(ok = v_ready(j))) break;
                    bool k_next = false;
                    for (int x = 0; ok && x < 2; ++x) {
                        const int nx = x ? n1 : n0;
                        if (j >= nx) continue;
                        if (!(ok = issue_PV(x, j, j))) break;
                        if (j + 1 == nx) {
                            tc::mma_commit(&B->o_full[x]);
                            continue;
                        }
                        if (!k_next) {
                            if (!(ok = k_ready(j + 1))) break;
                            tc::fence_after_sync();
                            k_next = true;
                        }
                        issue_S(x, j + 1);
                        tc::mma_commit(&B->s_full[x]);
                    }
                    if (!ok) break;
                    tc::mma_commit(&B->v_empty[j % ST]);
                    if (k_next) tc::mma_commit(&B->k_empty[(j + 1) % ST]);
                }
            }
            tc::mma_commit(&B->drain);                          // issued MMAs complete before TMEM is released
            mbar_wait(&B->drain, 0, nullptr);
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(TC_REG_SOFTMAX));
        // ---------------------------------------------- softmax warpgroups
        const int x = (warp - 4) >> 2;
        const int ntok = s_unit.ntok[x];
        if (ntok > 0) {
            const int quad = warp & 3, row = quad * 32 + lane;
            const uint32_t lane_addr = tbase + ((uint32_t)(quad * 32) << 16);
            const uint32_t p_addr = lane_addr + col_p(x);
            const int tok = row / a.G, g = row - tok * a.G;
            const int nx = x ? n1 : n0, p0 = s_unit.p0[x];
            const int len = s_unit.len;
            // this row sees [lo, limit] and the first rows; every row of the slot sees
            // [all_lo, all_hi]
            const int limit = PREFIX ? len - 1 : p0 + tok;
            const int lo = PREFIX ? 0 : window_lo(limit, a.window);
            const int all_hi = PREFIX ? len - 1 : p0;
            const int all_lo = PREFIX ? 0 : window_lo(p0 + ntok - 1, a.window);
            const float sl2 = a.sl2;
            const int j0 = s_unit.j0;
            float m = -INFINITY, l = 0.f;
            // A lane whose wait expired goes on, without further waits, over whatever S and V
            // hold: the warp stays together at every vote and TMEM access (and needs no vote
            // of its own per wait: with one, 1.5% more time).  The row is given up at the end.
            bool ok = true;
            for (int c = 0; c < nx; ++c) {
                // what needs no score is settled before the wait for them
                const int j = ALT ? 2 * c + x : c;
                const int k0 = t.row0(j0 + j, BN);
                const bool masked = k0 + BN - 1 > all_hi || !(k0 >= all_lo || k0 + BN <= a.sinks);
                // the first slot that uses a tile with rows behind the last one clears
                // them in V: they enter P.V as zeros (the other's P.V is issued later)
                const bool clear = k0 + BN > len && (ALT || x == 0 || j >= n0);
                ok = ok && wait_ab(&B->s_full[x], c & 1, abort, status);
                tc::fence_after_sync();
                uint32_t u32[BN];
#pragma unroll
                for (int cb = 0; cb < BN / 32; ++cb) tc::tmem_ld32p(lane_addr + col_s(x) + cb * 32, u32 + cb * 32);
                tc::tmem_wait_ld();
                float* sc = reinterpret_cast<float*>(u32);
                if (masked) {
                    const int hi = limit + 1 - k0, from = lo - k0, first = PREFIX ? 0 : min(a.sinks, limit + 1) - k0;
#pragma unroll
                    for (int w = 0; w < 4; ++w)
                        pf::keep_bits(sc + w * 32, (pf::bits_below(hi - w * 32) & ~pf::bits_below(from - w * 32)) |
                                                       pf::bits_below(first - w * 32));
                }
                // the running maximum moves, and O is rescaled, only when a row's
                // scores outgrow it by 2^8 (the last P.V completed before S came):
                // weights reach 2^8, 2^9 where the maximum itself is rounded (scores of 2^24)
                const float mxs = pf::row_max3(sc) * sl2;
                const bool need = mxs > m + pf::RESCALE_THRESHOLD;
                if (__any_sync(0xffffffffu, need)) {
                    const float alpha = need ? ex2(m - mxs) : 1.f;
                    if (need) m = mxs;
                    l *= alpha;
                    if (c > 0) {
#pragma unroll 1
                        for (int cb = 0; cb < D / 32; ++cb) {
                            uint32_t o[32];
                            tc::tmem_ld32(lane_addr + col_o(x) + cb * 32, o);
                            tc::tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                            tc::tmem_st32(lane_addr + col_o(x) + cb * 32, o);
                        }
                    }
                }
                if (clear) {
                    const int s = j % ST, r0 = max(0, len - k0), n = (BN - r0) * 8 * L::HALVES;
                    ok = ok && wait_ab(&B->v_full[s], (j / ST) & 1, abort, status);
                    for (int i = row; i < n; i += BM) {
                        const int f = i / ((BN - r0) * 8), e = i - f * (BN - r0) * 8;
                        *reinterpret_cast<uint4*>(sm + L::V + s * L::TILE + f * BOX + r0 * 128 + e * 16) =
                            make_uint4(0, 0, 0, 0);
                    }
                    fence_proxy_async_smem();
                }
                const float nm = m == -INFINITY ? 0.f : -m;
                const unsigned long long s2 = pf::f2(sl2, sl2), n2 = pf::f2(nm, nm);
                unsigned long long ps[4] = {0ull, 0ull, 0ull, 0ull};
                // the first half of P is handed over a quarter of the tile later, when
                // its stores have long landed; the tensor core needs the time of the
                // second half for it anyway
                uint32_t pk[32];
                pf::exp_pairs<64>(sc, s2, n2, pk, ps);
                tc::tmem_st32(p_addr, pk);
                pf::exp_pairs<32>(sc + 64, s2, n2, pk, ps);
                tc::tmem_wait_st();
                tc::fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(&B->p_full[x][0]);
                pf::exp_pairs<32>(sc + 96, s2, n2, pk + 16, ps);
                tc::tmem_st32(p_addr + 32, pk);
                tc::tmem_wait_st();
                tc::fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(&B->p_full[x][1]);
                float s0, s1;
                pf::un2(pf::add2(pf::add2(ps[0], ps[1]), pf::add2(ps[2], ps[3])), s0, s1);
                l += s0 + s1;
            }
            // A slot without a tile beside one with tiles has its Q on the way all the same: the
            // rows' zeros are staged where it lands.
            if (nx > 0) ok = ok && wait_ab(&B->o_full[x], 0, abort, status);
            else if (!ALT && n_kv > 0) ok = ok && wait_ab(&B->q_full, 0, abort, status);
            constexpr bool JOIN = ALT && !PREFIX;
            if constexpr (JOIN) {                                // before the ring is written, below
                if ((x ? n0 : n1) > 0) ok = ok && wait_ab(&B->o_full[x ^ 1], 0, abort, status);
            }
            tc::fence_after_sync();
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) {
                m = given_up().m;
                l = given_up().l;
            }
            // Slots that hold the same rows join their states (those of a prefix are
            // joined with the other splits'): each hands the other's half of O's columns
            // over through the (now idle) K/V ring.  All eight warps come here, after an
            // expired wait too.
            constexpr int cols = JOIN ? D / 2 : D;
            const int col0 = JOIN ? x * (D / 2) : 0;
            float w_mine = 1.f, w_other = 0.f;
            constexpr int XS = D / 2 + 4;                        // row stride: float4 of eight rows hit all banks
            float* xo = reinterpret_cast<float*>(sm + L::K);     // [2][BM][XS]
            if constexpr (JOIN) {
                // the ring is idle: the other slot's last P.V is done too
                if (nx > 0 && ok) {
#pragma unroll 1
                    for (int cb = 0; cb < D / 64; ++cb) {
                        uint32_t o[32];
                        tc::tmem_ld32(lane_addr + col_o(x) + (x ^ 1) * (D / 2) + cb * 32, o);
                        tc::tmem_wait_ld();
                        float* dst = xo + (x * BM + row) * XS + cb * 32;
#pragma unroll
                        for (int i = 0; i < 32; i += 4)
                            *reinterpret_cast<uint4*>(dst + i) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                    }
                }
                s_ml[x][row] = make_float2(m, l);
                asm volatile("bar.sync 1, 256;" ::: "memory");
                const float2 other = s_ml[x ^ 1][row];
                const float M = fmaxf(m, other.x);
                w_mine = m == -INFINITY ? 0.f : ex2(m - M);
                w_other = other.x == -INFINITY ? 0.f : ex2(other.x - M);
                l = l * w_mine + other.y * w_other;
                m = M;
            }
            const bool mine = tok < ntok && row < a.tpt * a.G;
            const float inv = PREFIX ? 1.f : row_factor(l);
            const float fm = w_mine * inv, fo = w_other * inv;
            const long long qrow = s_unit.tok0[x] + tok;
            const int h = kvh * a.G + g;
            constexpr int ELT = PREFIX ? 4 : 2;
            unsigned char* dst;                                  // this lane's row, its first column here
            if constexpr (PREFIX) {
                const int split = (int)(blockIdx.x / a.units) / a.c.hkv;
                const long long part = ALT ? 2 * split + x : split;
                const long long at = (part * a.n_tok + qrow) * a.hq + h;
                if (mine) *reinterpret_cast<float2*>(a.part_ml + at * 2) = make_float2(m, l);
                dst = reinterpret_cast<unsigned char*>(a.part_o + at * D + col0);
            } else {
                dst = static_cast<unsigned char*>(a.out) + (qrow * a.o_tok + (long long)h * D + col0) * 2;
            }
            // Out through shared memory (this slot's Q, or the unused one, is idle by now): a
            // lane has a row in hand, but rows lie apart in memory, so lanes that store
            // side by side should store one row.  A given-up row is NaN, straight to memory.
            if (!ok) {
                if (mine)
                    for (int i = 0; i < cols * ELT / 16; ++i)
                        reinterpret_cast<uint4*>(dst)[i] = make_uint4(~0u, ~0u, ~0u, ~0u);
            } else {
                const uint32_t rows_mine = __ballot_sync(0xffffffffu, mine);
                constexpr int group = cols < 2 * D / ELT ? cols : 2 * D / ELT;   // columns staged at once: 2 D bytes a row
                constexpr int lpr = group * ELT / 16;            // 16-byte chunks, and lanes, of a row
                unsigned char* stage = sm + L::Q + x * L::TILE + quad * (32 * 2 * D);
                for (int c0 = 0; c0 < cols && rows_mine; c0 += group) {
#pragma unroll 1
                    for (int cb = c0; cb < c0 + group; cb += 32) {
                        uint32_t o[32];
                        if (nx > 0) {
                            tc::tmem_ld32(lane_addr + col_o(x) + col0 + cb, o);
                            tc::tmem_wait_ld();
                        } else {
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] = 0u;
                        }
                        float f[32];
#pragma unroll
                        for (int i = 0; i < 32; ++i) f[i] = __uint_as_float(o[i]) * fm;
                        if (JOIN && fo > 0.f) {                  // the other's O is there only if it has weight
                            const float* src = xo + ((x ^ 1) * BM + row) * XS + cb;
#pragma unroll
                            for (int i = 0; i < 32; i += 4) {
                                const float4 v = *reinterpret_cast<const float4*>(src + i);
                                f[i] = fmaf(v.x, fo, f[i]);
                                f[i + 1] = fmaf(v.y, fo, f[i + 1]);
                                f[i + 2] = fmaf(v.z, fo, f[i + 2]);
                                f[i + 3] = fmaf(v.w, fo, f[i + 3]);
                            }
                        }
                        const int ch0 = (cb - c0) * ELT / 16;
#pragma unroll
                        for (int i = 0; i < 2 * ELT; ++i) {
                            uint4 v;
                            if constexpr (PREFIX) {
                                v = make_uint4(__float_as_uint(f[4 * i]), __float_as_uint(f[4 * i + 1]),
                                               __float_as_uint(f[4 * i + 2]), __float_as_uint(f[4 * i + 3]));
                            } else {
                                v = make_uint4(pf::pack_bf16(f[8 * i], f[8 * i + 1]), pf::pack_bf16(f[8 * i + 2], f[8 * i + 3]),
                                               pf::pack_bf16(f[8 * i + 4], f[8 * i + 5]),
                                               pf::pack_bf16(f[8 * i + 6], f[8 * i + 7]));
                            }
                            *reinterpret_cast<uint4*>(stage + lane * (lpr * 16) + (((ch0 + i) ^ (lane & (lpr - 1))) << 4)) = v;
                        }
                    }
                    __syncwarp();
#pragma unroll 4
                    for (int r0 = 0; r0 < 32; r0 += 32 / lpr) {
                        const int r = r0 + lane / lpr, ch = lane & (lpr - 1);
                        unsigned char* to = reinterpret_cast<unsigned char*>(
                            __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(dst), r));
                        if ((rows_mine >> r) & 1u)
                            *reinterpret_cast<uint4*>(to + c0 * ELT + ch * 16) =
                                *reinterpret_cast<const uint4*>(stage + r * (lpr * 16) + ((ch ^ (r & (lpr - 1))) << 4));
                    }
                    __syncwarp();
                }
            }
        }
    }
    tc::fence_before_sync();
    __syncthreads();
    if (warp == 1) {
        tc::fence_after_sync();
        tc::tmem_dealloc(tbase, 512);
    }
}

template <int D, bool PREFIX, bool ALT>
static int tc_launch_k(cudaStream_t st, int grid, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv,
                       const TcArgs& a) {
    auto k = paged_tc_kernel<D, PREFIX, ALT>;
    SA_RC_TRY(set_smem_attr_once((const void*)k, Lay<D>::SMEM));
    k<<<grid, TC_THREADS, Lay<D>::SMEM, st>>>(mq, mk, mv, a);
    SA_CUDA_TRY(cudaGetLastError());
    return SA_OK;
}
template <bool PREFIX>
static int tc_launch(int d, bool alt, cudaStream_t st, int grid, const CUtensorMap& mq, const CUtensorMap& mk,
                     const CUtensorMap& mv, const TcArgs& a) {
    if (d == 64)
        return alt ? tc_launch_k<64, PREFIX, true>(st, grid, mq, mk, mv, a)
                   : tc_launch_k<64, PREFIX, false>(st, grid, mq, mk, mv, a);
    return alt ? tc_launch_k<128, PREFIX, true>(st, grid, mq, mk, mv, a)
               : tc_launch_k<128, PREFIX, false>(st, grid, mq, mk, mv, a);
}

static int tc_maps(const sa_paged_kv* kv, const void* q, long long q_tok, int n_tok, int hq, TcArgs* a, CUtensorMap* mq,
                   CUtensorMap* mk, CUtensorMap* mv) {
    a->G = hq / kv->hkv;
    a->tpt = BM / a->G;
    a->hq = hq;
    a->n_tok = n_tok;
    SA_RC_TRY(make_query_tmap(mq, q, kv->d, hq, n_tok, q_tok, a->G, a->tpt));
    SA_RC_TRY(make_page_tmap(mk, kv->k_pages, kv, kv->page_size));
    return make_page_tmap(mv, kv->v_pages, kv, kv->page_size);
}

int tc_prefill_launch(sa_ctx* ctx, const sa_paged_kv* kv, const void* q, long long q_tok, int n_tok, int hq,
                      const int* cu_q, int window, int sinks, float scale, void* out, long long o_tok) {
    TcArgs a = {};
    CUtensorMap mq, mk, mv;
    SA_RC_TRY(tc_maps(kv, q, q_tok, n_tok, hq, &a, &mq, &mk, &mv));
    a.c = make_cache(ctx, kv);
    a.cu_q = cu_q;
    a.window = window;
    a.sinks = sinks;
    a.sl2 = scale * LOG2E;
    a.out = out;
    a.o_tok = o_tok;
    // Every sequence's last unit may be partly filled.  Few units leave SMs idle:
    // where units of one tile still fit the GPU at once, a unit's key tiles are
    // shared between the slots instead of its rows (512 tokens of 16/8 heads over
    // 1100 rows: 26.4 us in 32 CTAs, 19.0 in 64).
    const int seqs = std::min(kv->n_seqs, n_tok);
    const long long singles = ((long long)n_tok / a.tpt + seqs) * kv->hkv;
    const bool alt = singles <= ctx->num_sms;
    const long long grid = alt ? singles : ((long long)n_tok / (2 * a.tpt) + seqs) * kv->hkv;
    SA_CHECK_ARG(grid < (1LL << 31), "prefill: %lld CTAs", grid);
    return tc_launch<false>(kv->d, alt, ctx->stream, (int)grid, mq, mk, mv, a);
}

// Whether the rows of a KV head fill one tile at most: both slots hold it.
static bool tc_prefix_alt(int n_seqs, int G) { return n_seqs <= BM / G; }

// One CTA per SM: as many key splits as fill the GPU, no split without a tile.
int tc_prefix_splits(const sa_ctx* ctx, const sa_paged_kv* kv, int hq, int prefix_len, int* parts) {
    const int G = hq / kv->hkv, tpt = BM / G, units = ((kv->n_seqs + tpt - 1) / tpt + 1) / 2;
    const int tiles = (int)(((long long)prefix_len + BN - 1) / BN);
    const int n = std::max(1, std::min(tiles, ctx->num_sms / std::max(1, units * kv->hkv)));
    *parts = tc_prefix_alt(kv->n_seqs, G) ? 2 * n : n;
    return n;
}

int tc_prefix_launch(sa_ctx* ctx, const sa_paged_kv* kv, const void* q, long long q_tok, int hq, const int* prefix_table,
                     int prefix_len, float scale, int n_split, float* part_o, float* part_ml) {
    TcArgs a = {};
    CUtensorMap mq, mk, mv;
    SA_RC_TRY(tc_maps(kv, q, q_tok, kv->n_seqs, hq, &a, &mq, &mk, &mv));
    a.c = make_cache(ctx, kv);
    a.sl2 = scale * LOG2E;
    a.prefix_table = prefix_table;
    a.prefix_len = prefix_len;
    a.n_split = n_split;
    a.units = ((kv->n_seqs + a.tpt - 1) / a.tpt + 1) / 2;
    a.part_o = part_o;
    a.part_ml = part_ml;
    const long long grid = (long long)a.units * kv->hkv * n_split;
    SA_CHECK_ARG(grid < (1LL << 31), "prefix: %lld CTAs", grid);
    return tc_launch<true>(kv->d, tc_prefix_alt(kv->n_seqs, a.G), ctx->stream, (int)grid, mq, mk, mv, a);
}

}  // namespace pg
}  // namespace sa
