// sa_paged_decode.cu -- one query token per sequence over a paged KV cache,
// with a sliding window and first tokens that stay visible.
//
//   out[b, h] = sum_j w_j v_j / sum_j w_j,   w_j = 2^(s_j - m),
//   s_j = scale log2(e) q[b, h] . k_j,  m the running maximum of the s_j,
// over the rows j that the query at position len - 1 sees.
//
// Bound: HBM.  Every visible K and V row is read once, for all G = hq / hkv
// query heads of its KV head.
//
// Work: the visible rows of every (sequence, KV head) are cut into tiles; the
// tiles of the whole batch form one list, and CTA c takes an equal share of
// consecutive ones, whatever the lengths.  The list follows from kv_lens on
// the device, so the host neither knows the lengths nor plans again when they
// grow (a captured launch stays right).  Only the first and the last (sequence,
// head) of a CTA can be shared with other CTAs; such shares leave their
// (m, l, O) in the workspace, and the CTA that hands in a pair's last one joins
// them (in the order of the rows, so the result does not depend on who is last).
//
// A producer warp copies tiles of 32 KB (64 KB at d = 256) into a ring of three;
// its lanes fetch the block-table entries of the next tile while the ring is
// full.  Consumers:
//  * bf16: four warps, 16 rows of a tile each, on mma.m16n8k16 with the
//    ROWS as the matrix's M and the query heads as its N, S^T = K q^T and
//    O^T += V^T P^T: one key row's G scores then cost one eighth of an N = 8
//    tile, where a layout with queries as M would fill 16 rows with G of them.
//    P^T turns from accumulator to operand layout by movmatrix, without shared
//    memory.  (tcgen05 wants M = 128 rows of A from shared memory and its
//    result in TMEM; at 4 G FLOP per 4 bytes the tensor rate is not what binds.)
//    P enters the product as the sum of two bf16 numbers: HBM binds, so the second
//    product costs nothing over long rows (64 sequences, below: 172.8 us, 173.0 with
//    one), and 0.1-0.8 us where short ones leave it in the chain of latencies (1024
//    sequences of 30 rows: 61.9, 61.1).  Against 64 bits 1.65e-3, the output's
//    rounding alone; with one 1.95e-3.
//  * fp32, up to four heads per KV head: four warps per group of at most HG heads, on
//    FMAs, an 8-lane group per row; scores, weights and sums in fp32.
//  * fp32, more heads: on the tensor cores, three tf32 products for one of fp32.
//
// Measured: 64 sequences of up to 16384 rows under a window of 4096, 32/8 heads of
// 128 bf16 (1.08 GB): 174 us, 6.2 TB/s, 0.96 of the measured copy; 13 fp32 ones of
// up to 8191 rows, 16/8 heads (0.68 GB): 108-114 us.  One sequence of 32768 rows
// (134 MB): 34 us -- some 10 us go to the plan, the first table entry and copy, and
// the join, which follow one another.  fp32, 16 sequences of up to 4000 rows, 8 KV
// heads of 128 (0.41 GB): 69 / 72 / 85 us for 1 / 2 / 4 heads each on FMAs, 91 for
// eight and 119 for sixteen on tensor cores (127 and 411 on FMAs, whose q and O did
// not fit the registers); 64/8 heads of 64: 87 (133), of 256: 157 (286).  There the
// chains of dependent products of 4 to 8 warps per SM bind (tensor pipe 0.4 busy,
// half of the issue slots).
#include <cuda_bf16.h>
#include <algorithm>
#include <cmath>

#include "sa_paged.cuh"
#include "sa_paged_decode.h"
#include "sa_tc.cuh"
#include "sa_tf32.cuh"

namespace sa {
namespace pg {

constexpr int STAGES = 3;

enum { JOIN_HERE = 1, JOIN_LATER = 2 };
struct DecodeArgs {
    Cache c;
    const void* q;
    void* out;
    long long q_stride, o_stride;      // elements between sequences
    int hq, G, window, sinks;
    float qscale;                      // scale * log2(e)
    int prefixed;                      // every query sees a shared prefix too; JOIN_HERE or JOIN_LATER
    PrefixParts prefix;
    DecodeWs ws;
};

template <typename KT, int D>
struct Geo {
    static constexpr int ELT = sizeof(KT);
    static constexpr int STAGE_BYTES = (ELT == 2 && D == 256) ? 65536 : 32768;     // K and V
    static constexpr int TK = STAGE_BYTES / (2 * D * ELT);                          // rows of a tile
    static constexpr int CTAS = STAGE_BYTES == 32768 ? 2 : 1;                       // per SM
};

// The tiles of a sequence's own rows.  Where a prefix's parts are joined here, a
// sequence without own rows has an empty one, so that somebody does it.
__device__ __forceinline__ Tiles tiles_of(const DecodeArgs& a, int len, int tk) {
    Tiles t = make_tiles(len, a.window, a.sinks, tk);
    if (a.prefixed == JOIN_HERE && t.n == 0) t.n = 1;
    return t;
}

// This CTA's share of the tile list, and the walk through it.
struct Walk {
    int b, h, i;            // sequence, KV head, tile of that pair
    int left;               // tiles of the share still ahead, this one included
    Tiles t;                // of sequence b
    __device__ __forceinline__ void next(const DecodeArgs& a, int tk) {
        --left;
        if (++i < t.n) return;
        i = 0;
        if (++h < a.c.hkv) return;
        h = 0;
        if (!left) return;
        do {
            ++b;
            t = tiles_of(a, seq_len(a.c, b), tk);
        } while (t.n == 0);
    }
};

struct Share {
    int b, h, i;            // first pair and tile
    long long first, total; // first tile of the share, tiles of the list
    int count, n_ctas;
};

// Every thread sums the tiles of a run of sequences; the block's scan gives the
// list's length and each run's start; the thread whose run holds the CTA's
// first tile finds the sequence in it.
template <int THREADS>
__device__ void plan_share(const DecodeArgs& a, int tk, Share* s, long long* scan) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr int W = THREADS / 32;
    const int per = (a.c.n_seqs + THREADS - 1) / THREADS;
    const int b0 = tid * per, b1 = min(a.c.n_seqs, b0 + per);
    long long mine = 0;
    for (int b = b0; b < b1; b += 8) {                   // eight loads in flight where runs are long
        int len[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) len[u] = b + u < b1 ? a.c.kv_lens[b + u] : 0;
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (b + u < b1) mine += tiles_of(a, cut_len(len[u], a.c.max_pages, a.c.page_log2), tk).n;
    }
    mine *= a.c.hkv;
    long long inc = mine;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const long long up = __shfl_up_sync(0xffffffffu, inc, off);
        if (lane >= off) inc += up;
    }
    if (lane == 31) scan[warp] = inc;
    if (tid == 0) s->count = 0;
    __syncthreads();
    long long before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) {
        if (w < warp) before += scan[w];
        total += scan[w];
    }
    const long long start = before + inc - mine;
    if (total > 0) {
        const long long n = min((long long)gridDim.x, total);
        const long long c = blockIdx.x;
        if (c < n) {
            const long long f = share_first(c, total, n), e = share_first(c + 1, total, n);
            if (f >= start && f < start + mine) {
                long long at = start;
                for (int b = b0; b < b1; ++b) {
                    const int nt = tiles_of(a, seq_len(a.c, b), tk).n;
                    const long long all = (long long)nt * a.c.hkv;
                    if (f < at + all) {
                        s->b = b;
                        s->h = (int)((f - at) / nt);
                        s->i = (int)((f - at) - (long long)s->h * nt);
                        break;
                    }
                    at += all;
                }
                s->first = f;
                s->count = (int)(e - f);
                s->total = total;
                s->n_ctas = (int)n;
            }
        }
    }
    // sequences without a visible row: their output is zero
    if (!a.prefixed)
        for (int b = b0; b < b1; ++b) {
            if (b % gridDim.x != blockIdx.x || seq_len(a.c, b) > 0) continue;
            const int e = a.ws.out_elt;
            uint4* o = reinterpret_cast<uint4*>(static_cast<unsigned char*>(a.out) + (long long)b * a.o_stride * e);
            const int n16 = a.hq * a.ws.d * e / 16;
            for (int i = 0; i < n16; ++i) o[i] = make_uint4(0, 0, 0, 0);
        }
    __syncthreads();
}

// Where a pair's state goes: straight to the output, to the pair's own state (to
// be joined with a prefix's parts), or to a slot of this CTA.
enum { TO_OUT = 0, TO_STATE = 1, TO_SLOT = 2 };
struct Dest {
    int kind, slot;
};

__device__ __forceinline__ Dest segment_dest(const DecodeArgs& a, const Share& s, long long seg_first, bool whole,
                                             int b, int h) {
    Dest d;
    d.kind = !whole ? TO_SLOT : a.prefixed ? TO_STATE : TO_OUT;
    d.slot = whole ? b * a.c.hkv + h : 2 * (int)blockIdx.x + (seg_first == s.first ? 0 : 1);
    return d;
}
// The shares of a pair whose tiles begin at t0 in the list: CTAs first .. last,
// the first one's in slot `slot`, the others' in slot 0.
struct Shares {
    int first, last, slot;
};
__device__ __forceinline__ Shares pair_shares(const Share& s, long long t0, int n) {
    Shares x;
    x.first = share_of(t0, s.total, s.n_ctas);
    x.last = share_of(t0 + n - 1, s.total, s.n_ctas);
    x.slot = share_first(x.first, s.total, s.n_ctas) == t0 ? 0 : 1;
    return x;
}
__device__ __forceinline__ long long share_slot(const Shares& x, int p) { return 2LL * (x.first + p) + (p == 0 ? x.slot : 0); }

__device__ __forceinline__ uint32_t pack2(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// What the pair h = pack2(a, b) leaves of a and b.
__device__ __forceinline__ uint32_t rest2(uint32_t h, float a, float b) {
    return pack2(a - __uint_as_float(h << 16), b - __uint_as_float(h & 0xffff0000u));
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t movm(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
template <int N>
__device__ __forceinline__ void bar_consumers() {
    asm volatile("bar.sync 1, %0;" ::"n"(N) : "memory");
}
struct Ring {
    uint64_t full[STAGES], empty[STAGES];
    long long scan[40];
    Share share;
    int issued;
    int failed;              // a consumer's wait expired: what follows is NaN
    int last;                // this CTA handed in a pair's last share
};

// A consumer lane's wait for tile `it` of its share; one that expires is noted, and the
// lane goes on without further waits over whatever the ring holds: the warp stays
// together at its shuffles and products without a vote per tile (1024 sequences of 30
// rows: 61.9 us, 62.7 with one), meets every barrier, and hands every share in as NaN.
__device__ __forceinline__ void consume_wait(Ring* r, int it, bool& ok, int* status) {
    if (ok && !mbar_wait(r->full + it % STAGES, (it / STAGES) & 1, status)) {
        ok = false;
        r->failed = 1;
    }
}
// The stage is free again; after an expired wait it is not: its copy may be on its way.
__device__ __forceinline__ void consumed(Ring* r, int s, bool ok, int lane) {
    __syncwarp();
    if (lane == 0 && ok) mbar_arrive(r->empty + s);
}

// For a kernel that joins the states later: where it finds a pair's.
__device__ __forceinline__ void record_pair(const DecodeArgs& a, const Share& s, long long t0, int n, int i0, bool whole,
                                            int b, int h) {
    const int pair = b * a.c.hkv + h;
    if (whole) {
        a.ws.pair[pair] = make_int4(-1, 0, 0, 0);
    } else if (i0 == 0) {
        const Shares x = pair_shares(s, t0, n);
        a.ws.pair[pair] = make_int4(x.first, x.last, x.slot, 0);
    }
}

// The consumer threads have written the state of a pair, or of a share of one
// (thread 0's warp did).  Count a share; then join what there is to join -- the
// prefix's parts, the pair's shares where this was the last one handed in -- with
// a warp per query head.
template <typename OT, int D, int NT>
__device__ __forceinline__ void hand_in(const DecodeArgs& a, Ring* r, const Share& sh, long long t0, int n, bool whole,
                                        int b, int h) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    Shares x = {};
    int shares = 1;
    __threadfence();
    bar_consumers<NT>();
    if (!whole) {
        x = pair_shares(sh, t0, n);
        shares = x.last - x.first + 1;
        if (threadIdx.x == 0) r->last = atomicAdd(a.ws.count + x.first, 1u) == (unsigned)(shares - 1);
        bar_consumers<NT>();
        if (!r->last) return;
        __threadfence();
        if (threadIdx.x == 0) a.ws.count[x.first] = 0u;
    }
    if (a.prefixed) pdl_wait();
    const long long rows = (long long)a.c.n_seqs * a.hq;
    for (int g = warp; g < a.G; g += NT / 32) {
        const long long row = (long long)b * a.hq + h * a.G + g;
        Joined<D> s;
        if (a.prefixed)
            s.add(a.prefix.parts, lane, [&](int p) { return __ldcg(a.prefix.ml + p * rows + row); },
                  [&](int p) { return a.prefix.o + (p * rows + row) * D; });
        if (whole)
            s.add(1, lane, [&](int) { return __ldcg(a.ws.state_ml + row); }, [&](int) { return a.ws.state_o + row * D; });
        else
            s.add(shares, lane, [&](int p) { return __ldcg(a.ws.slot_ml + share_slot(x, p) * a.G + g); },
                  [&](int p) { return a.ws.slot_o + (share_slot(x, p) * a.G + g) * D; });
        s.store(static_cast<OT*>(a.out) + (long long)b * a.o_stride + (long long)(h * a.G + g) * D, lane);
    }
}

// The producer warp: copies this share's tiles, pages that hold no visible row
// left out.  bf16 tiles through the tensor maps (swizzled for ldmatrix), fp32
// ones row after row.
template <typename KT, int D>
__device__ __forceinline__ void produce(const CUtensorMap* tk, const CUtensorMap* tv, const DecodeArgs& a, Ring* r,
                                        unsigned char* buf, Walk w, int lane) {
    using Z = Geo<KT, D>;
    constexpr int TK = Z::TK;
    const int pl = a.c.page_log2, page = 1 << pl;
    const int rows = min(page, TK);                      // rows of one copy
    const int copies = TK / rows;
    auto lookup = [&](const Walk& x) -> int {             // this lane's page of tile x, -1: not copied
        if (lane >= copies) return -1;
        const int r0 = x.t.row0(x.i, TK) + lane * rows;
        if (!x.t.any(r0, rows)) return -1;
        return a.c.table[(long long)x.b * a.c.table_stride + (r0 >> pl)];
    };
    auto known = [&](const Walk& x) -> bool {
        return lane < copies && x.t.any(x.t.row0(x.i, TK) + lane * rows, rows);
    };
    const int n = w.left;
    int entry = n ? lookup(w) : -1;
    int it = 0;
    for (; it < n; ++it) {
        const Walk cur = w;
        const bool use = known(cur);
        const int page_id = use ? checked_page(a.c, entry) : -1;
        w.next(a, TK);
        if (it + 1 < n) entry = lookup(w);
        const int s = it % STAGES;
        const bool free = it < STAGES || mbar_wait(r->empty + s, ((it / STAGES) & 1) ^ 1, a.c.status);
        if (!__all_sync(0xffffffffu, free)) break;       // the lanes give up together
        const unsigned got = __ballot_sync(0xffffffffu, page_id >= 0);
        const uint32_t bytes = (uint32_t)(rows * D * Z::ELT);
        if (lane == 0) mbar_arrive_expect_tx(r->full + s, 2 * __popc(got) * bytes);
        __syncwarp();
        if (page_id >= 0) {
            unsigned char* kd = buf + s * Z::STAGE_BYTES;
            unsigned char* vd = kd + Z::STAGE_BYTES / 2;
            const int in_page = cur.t.row0(cur.i, TK) & (page - 1);     // 0 unless the page is longer than a tile
            if constexpr (Z::ELT == 2) {
                const int y = (cur.h << pl) + in_page;
#pragma unroll
                for (int f = 0; f < D / 64; ++f) {
                    const int off = f * TK * 128 + lane * rows * 128;
                    tc::tma_load_3d(kd + off, tk, f * 64, y, page_id, r->full + s);
                    tc::tma_load_3d(vd + off, tv, f * 64, y, page_id, r->full + s);
                }
            } else {
                const long long at = ((long long)page_id * a.c.page_stride +
                                      (((long long)cur.h << pl) + in_page) * D) * Z::ELT;
                const int off = lane * (int)bytes;
                const uint64_t pol = policy_evict_first();
                bulk_g2s_hint(kd + off, a.c.k + at, bytes, r->full + s, pol);
                bulk_g2s_hint(vd + off, a.c.v + at, bytes, r->full + s, pol);
            }
        }
        __syncwarp();
    }
    if (lane == 0) r->issued = it;
}

// A CTA whose pipeline gave up lets its copies in flight land (bounded) before
// it leaves.
__device__ __forceinline__ void drain(Ring* r) {
    __syncthreads();
    if (threadIdx.x == 0 && r->failed)
        for (int it = max(0, r->issued - STAGES); it < r->issued; ++it)
            mbar_wait(r->full + it % STAGES, (it / STAGES) & 1, nullptr);
    __syncthreads();
}

// Behind a shared prefix the launch starts while the prefix's kernel still runs;
// it ends only after that kernel, so that the stream's next one has both.
__device__ __forceinline__ void leave(const DecodeArgs& a) {
    if (a.prefixed) pdl_wait();                          // (nothing to wait for in an ordinary launch)
}

// ---- bf16 -------------------------------------------------------------------
constexpr int BW = 4;                        // consumer warps
constexpr int BTHREADS = (BW + 1) * 32;
template <int D>
constexpr int red_floats() { return (D / 16) * 4 * 32 + 4 * 32; }     // O^T of 8 heads, then m and l, lane by lane
template <int D>
constexpr int bf16_smem() {
    return STAGES * Geo<__nv_bfloat16, D>::STAGE_BYTES + 3 * red_floats<D>() * 4 + 1024;
}

// Fold another warp's state of 8 heads (two columns a lane) into this one's.
template <int D>
__device__ __forceinline__ void fold(float (&o)[D / 16][4], float* m, float* l, const float* red, int lane) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const float m2 = red[(D / 16) * 128 + j * 32 + lane], l2 = red[(D / 16) * 128 + (2 + j) * 32 + lane];
        const float M = fmaxf(m[j], m2);
        const float wa = m[j] == -INFINITY ? 0.f : ex2(m[j] - M), wb = m2 == -INFINITY ? 0.f : ex2(m2 - M);
        m[j] = M;
        l[j] = l[j] * wa + l2 * wb;
#pragma unroll
        for (int t = 0; t < D / 16; ++t) {
            o[t][j] = o[t][j] * wa + red[(t * 4 + j) * 32 + lane] * wb;
            o[t][2 + j] = o[t][2 + j] * wa + red[(t * 4 + 2 + j) * 32 + lane] * wb;
        }
    }
}
template <int D>
__device__ __forceinline__ void put(const float (&o)[D / 16][4], const float* m, const float* l, float* red, int lane) {
#pragma unroll
    for (int t = 0; t < D / 16; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) red[(t * 4 + e) * 32 + lane] = o[t][e];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        red[(D / 16) * 128 + j * 32 + lane] = m[j];
        red[(D / 16) * 128 + (2 + j) * 32 + lane] = l[j];
    }
}

template <int D, int NT>
__global__ void __launch_bounds__(BTHREADS, Geo<__nv_bfloat16, D>::CTAS)
decode_bf16_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                   const __grid_constant__ DecodeArgs a) {
    using Z = Geo<__nv_bfloat16, D>;
    constexpr int TK = Z::TK, KB = TK / 16 / BW;       // blocks of 16 rows per warp and tile
    extern __shared__ unsigned char smem_raw[];
    __shared__ Ring r;
    const uint32_t raw = smem_u32(smem_raw);
    unsigned char* buf = smem_raw + (((raw + 1023u) & ~1023u) - raw);
    float* red = reinterpret_cast<float*>(buf + STAGES * Z::STAGE_BYTES);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    pdl_trigger();
    if (tid == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(r.full + s, 1);
            mbar_init(r.empty + s, BW);
        }
        fence_barrier_init();
        r.issued = 0;
        r.failed = 0;
    }
    plan_share<BTHREADS>(a, TK, &r.share, r.scan);
    const Share sh = r.share;
    if (sh.count == 0) {
        leave(a);
        return;
    }
    Walk w;
    w.b = sh.b; w.h = sh.h; w.i = sh.i; w.left = sh.count;
    w.t = tiles_of(a, seq_len(a.c, w.b), TK);
    __syncthreads();

    if (warp == BW) {
        produce<__nv_bfloat16, D>(&tk, &tv, a, &r, buf, w, lane);
        drain(&r);
        leave(a);
        return;
    }
    const int qc = lane >> 2, qp = (lane & 3) * 2;      // column as operand; first of two columns as accumulator
    const uint32_t sbuf = smem_u32(buf);
    // q of the next pair is on its way while the last one's states are joined
    uint32_t qf[NT][D / 16][2];
    auto load_q = [&](int b, int h) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const bool on = n * 8 + qc < a.G;
            const __nv_bfloat16* qr = static_cast<const __nv_bfloat16*>(a.q) + (long long)b * a.q_stride +
                                      (long long)(h * a.G + (on ? n * 8 + qc : 0)) * D + qp;
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
                qf[n][kk][0] = on ? __ldg(reinterpret_cast<const uint32_t*>(qr + kk * 16)) : 0u;
                qf[n][kk][1] = on ? __ldg(reinterpret_cast<const uint32_t*>(qr + kk * 16 + 8)) : 0u;
            }
        }
    };
    load_q(w.b, w.h);
    int it = 0;
    bool ok = true;
    while (w.left > 0) {
        // ---- one pair's tiles
        const int b = w.b, h = w.h, i0 = w.i;
        const Tiles t = w.t;
        const int i1 = min(t.n, i0 + w.left);
        const long long seg_first = sh.first + (sh.count - w.left);
        float o[NT][D / 16][4], m[NT][2], l[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            m[n][0] = m[n][1] = -INFINITY;
            l[n][0] = l[n][1] = 0.f;
#pragma unroll
            for (int d = 0; d < D / 16; ++d)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[n][d][e] = 0.f;
        }
        for (int i = i0; i < i1; ++i, ++it) {
            const int s = it % STAGES;
            consume_wait(&r, it, ok, a.c.status);
            const uint32_t ks = sbuf + s * Z::STAGE_BYTES, vs = ks + Z::STAGE_BYTES / 2;
            const int row0 = t.row0(i, TK);
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
                const int r0 = (warp * KB + kb) * 16;    // first of the warp's 16 rows in the tile
                const int j0 = row0 + r0;
                if (!t.any(j0, 16)) continue;
                const bool all = t.all(j0, 16);
                float sc[NT][4];
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) sc[n][e] = 0.f;
                const int krow = r0 + (lane & 15);
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk) {
                    uint32_t kf[4];
                    const int ch = (kk & 3) * 2 + (lane >> 4);
                    ldsm4(kf, ks + (kk >> 2) * (TK * 128) + krow * 128 + ((ch ^ (krow & 7)) << 4));
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma16816(sc[n], kf, qf[n][kk][0], qf[n][kk][1]);
                }
                // accumulator rows: lane/4 and lane/4 + 8; columns qp, qp + 1
                uint32_t vmask[2] = {0xffffffffu, 0xffffffffu};
                if (!all) {
                    const bool see0 = t.sees(j0 + qc), see1 = t.sees(j0 + qc + 8);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        if (!see0) sc[n][0] = sc[n][1] = -INFINITY;
                        if (!see1) sc[n][2] = sc[n][3] = -INFINITY;
                    }
                    // rows that nobody sees may hold anything: they enter the product as zeros
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        vmask[e] = (t.sees(j0 + qp + 8 * e) ? 0x0000ffffu : 0u) |
                                   (t.sees(j0 + qp + 1 + 8 * e) ? 0xffff0000u : 0u);
                }
                uint32_t ph[NT][2], pl[NT][2];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float mx0 = fmaxf(sc[n][0], sc[n][2]), mx1 = fmaxf(sc[n][1], sc[n][3]);
#pragma unroll
                    for (int off = 4; off < 32; off <<= 1) {
                        mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, off));
                        mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, off));
                    }
                    const float M0 = fmaxf(m[n][0], mx0 * a.qscale), M1 = fmaxf(m[n][1], mx1 * a.qscale);
                    if (__any_sync(0xffffffffu, M0 > m[n][0] || M1 > m[n][1])) {
                        const float c0 = m[n][0] == -INFINITY ? 0.f : ex2(m[n][0] - M0);
                        const float c1 = m[n][1] == -INFINITY ? 0.f : ex2(m[n][1] - M1);
                        l[n][0] *= c0;
                        l[n][1] *= c1;
#pragma unroll
                        for (int d = 0; d < D / 16; ++d) {
                            o[n][d][0] *= c0;
                            o[n][d][1] *= c1;
                            o[n][d][2] *= c0;
                            o[n][d][3] *= c1;
                        }
                        m[n][0] = M0;
                        m[n][1] = M1;
                    }
                    const float z0 = m[n][0] == -INFINITY ? 0.f : -m[n][0], z1 = m[n][1] == -INFINITY ? 0.f : -m[n][1];
                    const float p0 = ex2(fmaf(sc[n][0], a.qscale, z0)), p1 = ex2(fmaf(sc[n][1], a.qscale, z1));
                    const float p2 = ex2(fmaf(sc[n][2], a.qscale, z0)), p3 = ex2(fmaf(sc[n][3], a.qscale, z1));
                    l[n][0] += p0 + p2;
                    l[n][1] += p1 + p3;
                    const uint32_t h0 = pack2(p0, p1), h1 = pack2(p2, p3);
                    ph[n][0] = movm(h0);
                    ph[n][1] = movm(h1);
                    pl[n][0] = movm(rest2(h0, p0, p1));
                    pl[n][1] = movm(rest2(h1, p2, p3));
                }
                const int vrow = r0 + ((lane >> 4) << 3) + (lane & 7);
#pragma unroll
                for (int d = 0; d < D / 16; ++d) {
                    uint32_t vf[4];
                    const int ch = (d & 3) * 2 + ((lane >> 3) & 1);
                    ldsm4t(vf, vs + (d >> 2) * (TK * 128) + vrow * 128 + ((ch ^ (vrow & 7)) << 4));
                    if (!all) {
                        vf[0] &= vmask[0];
                        vf[1] &= vmask[0];
                        vf[2] &= vmask[1];
                        vf[3] &= vmask[1];
                    }
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        mma16816(o[n][d], vf, ph[n][0], ph[n][1]);
                        mma16816(o[n][d], vf, pl[n][0], pl[n][1]);
                    }
                }
            }
            consumed(&r, s, ok, lane);
            w.next(a, TK);
        }
        if (w.left > 0) load_q(w.b, w.h);
        // ---- join the four warps' states and hand the pair's over.  The next pair's
        // join writes slot 2 after a barrier that warp 0 meets once it is done here.
        const bool whole = i0 == 0 && i1 == t.n;
        const Dest ds = segment_dest(a, sh, seg_first, whole, b, h);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) l[n][j] += __shfl_xor_sync(0xffffffffu, l[n][j], off);
            if (warp >= 2) put<D>(o[n], m[n], l[n], red + (warp - 2) * red_floats<D>(), lane);
            bar_consumers<BW * 32>();
            if (warp < 2) fold<D>(o[n], m[n], l[n], red + warp * red_floats<D>(), lane);
            if (warp == 1) put<D>(o[n], m[n], l[n], red + 2 * red_floats<D>(), lane);
            bar_consumers<BW * 32>();
            if (warp != 0) continue;
            fold<D>(o[n], m[n], l[n], red + 2 * red_floats<D>(), lane);
            const bool failed = *reinterpret_cast<volatile int*>(&r.failed) != 0;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int g = n * 8 + qp + j;
                if (g >= a.G) continue;
                if (failed) {
                    m[n][j] = given_up().m;
                    l[n][j] = given_up().l;
                }
                if (ds.kind == TO_OUT) {
                    const float inv = 1.f / l[n][j];     // the pair's query sees its own row at least
                    __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(a.out) + (long long)b * a.o_stride +
                                         (long long)(h * a.G + g) * D + qc;
#pragma unroll
                    for (int d = 0; d < D / 16; ++d) {
                        dst[d * 16] = __float2bfloat16_rn(o[n][d][j] * inv);
                        dst[d * 16 + 8] = __float2bfloat16_rn(o[n][d][2 + j] * inv);
                    }
                } else {
                    const long long at = (long long)ds.slot * a.G + g;
                    float* dst = (ds.kind == TO_STATE ? a.ws.state_o : a.ws.slot_o) + at * D;
#pragma unroll
                    for (int d = 0; d < D / 16; ++d) {
                        dst[d * 16 + qc] = o[n][d][j];
                        dst[d * 16 + 8 + qc] = o[n][d][2 + j];
                    }
                    if (qc == 0)
                        (ds.kind == TO_STATE ? a.ws.state_ml : a.ws.slot_ml)[at] = make_float2(m[n][j], l[n][j]);
                }
            }
        }
        if (a.prefixed == JOIN_LATER) {
            if (tid == 0) record_pair(a, sh, seg_first - i0, t.n, i0, whole, b, h);
        } else if (a.prefixed || !whole) {
            hand_in<__nv_bfloat16, D, BW * 32>(a, &r, sh, seg_first - i0, t.n, whole, b, h);
        }
    }
    drain(&r);
    leave(a);
}

// ---- fp32 -------------------------------------------------------------------
template <int D>
struct FGeo {
    using Z = Geo<float, D>;
    static constexpr int RW = Z::TK / 4, NR = RW / 4;      // rows per warp; per 8-lane group
    static constexpr int CPL = D / 8, CH = CPL / 4;        // columns per lane, as CH float4
};
// CTAs per SM: two where their registers (q and O: 2 HG D / 8 a thread) fit.
template <int NG>
constexpr int f32_ctas() { return NG == 1 ? 2 : 1; }
template <int D, int HG, int NG>
constexpr int f32_smem() {
    return STAGES * Geo<float, D>::STAGE_BYTES + NG * 4 * HG * (D + 2) * 4 + 128;
}

// The consumers' states of a pair are in `red`, by group of HG heads, P parts each
// (one after the other, HG rows of D floats, m and l): join the parts, hand over.
template <int D, int HG, int P, int NW>
__device__ __forceinline__ void finish_f32(const DecodeArgs& a, Ring* r, const Share& sh, const Tiles& t, const float* red,
                                           const Dest& ds, long long seg_first, int i0, bool whole, int b, int h) {
    const int tid = threadIdx.x;
    const bool failed = *reinterpret_cast<volatile int*>(&r->failed) != 0;
    for (int idx = tid; idx < a.G * D; idx += NW * 32) {
        const int g = idx / D, col = idx - g * D;
        const float* src = red + ((g / HG) * P * HG + g % HG) * (D + 2);       // + HG rows per part
        float M = -INFINITY;
#pragma unroll
        for (int x = 0; x < P; ++x) M = fmaxf(M, src[x * HG * (D + 2) + D]);
        float L = 0.f, O = 0.f;
#pragma unroll
        for (int x = 0; x < P; ++x) {
            const float* y = src + x * HG * (D + 2);
            const float wt = y[D] == -INFINITY ? 0.f : ex2(y[D] - M);
            L += y[D + 1] * wt;
            O += y[col] * wt;
        }
        if (failed) {
            M = given_up().m;
            L = given_up().l;
        }
        if (ds.kind == TO_OUT) {
            static_cast<float*>(a.out)[(long long)b * a.o_stride + (long long)(h * a.G + g) * D + col] = O / L;
        } else {
            const long long at = (long long)ds.slot * a.G + g;
            (ds.kind == TO_STATE ? a.ws.state_o : a.ws.slot_o)[at * D + col] = O;
            if (col == 0) (ds.kind == TO_STATE ? a.ws.state_ml : a.ws.slot_ml)[at] = make_float2(M, L);
        }
    }
    if (a.prefixed == JOIN_LATER) {
        if (tid == 0) record_pair(a, sh, seg_first - i0, t.n, i0, whole, b, h);
    } else if (a.prefixed || !whole) {
        hand_in<float, D, NW * 32>(a, r, sh, seg_first - i0, t.n, whole, b, h);
    }
    bar_consumers<NW * 32>();                            // the buffers are free again
}

template <int D, int HG, int NG>
__global__ void __launch_bounds__((NG * 4 + 1) * 32, f32_ctas<NG>())
decode_f32_kernel(const __grid_constant__ DecodeArgs a) {
    using Z = Geo<float, D>;
    using F = FGeo<D>;
    constexpr int TK = Z::TK, NW = NG * 4, THREADS = (NW + 1) * 32;
    extern __shared__ unsigned char smem_raw[];
    __shared__ Ring r;
    unsigned char* buf = smem_raw + ((128u - (smem_u32(smem_raw) & 127u)) & 127u);
    float* red = reinterpret_cast<float*>(buf + STAGES * Z::STAGE_BYTES);   // [warp][HG][D + 2]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    pdl_trigger();
    if (tid == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(r.full + s, 1);
            mbar_init(r.empty + s, NW);
        }
        fence_barrier_init();
        r.issued = 0;
        r.failed = 0;
    }
    plan_share<THREADS>(a, TK, &r.share, r.scan);
    const Share sh = r.share;
    if (sh.count == 0) {
        leave(a);
        return;
    }
    Walk w;
    w.b = sh.b; w.h = sh.h; w.i = sh.i; w.left = sh.count;
    w.t = tiles_of(a, seq_len(a.c, w.b), TK);
    __syncthreads();

    if (warp == NW) {
        produce<float, D>(nullptr, nullptr, a, &r, buf, w, lane);
        drain(&r);
        leave(a);
        return;
    }
    const int grp = lane >> 3, sub = lane & 7, part = warp & 3, g0 = (warp >> 2) * HG;
    float qr[HG][F::CPL];
    auto load_q = [&](int b, int h) {
#pragma unroll
        for (int g = 0; g < HG; ++g) {
            const bool on = g0 + g < a.G;
            const float* qh = static_cast<const float*>(a.q) + (long long)b * a.q_stride +
                              (long long)(h * a.G + (on ? g0 + g : 0)) * D;
#pragma unroll
            for (int c = 0; c < F::CH; ++c) {
                const float4 x = *reinterpret_cast<const float4*>(qh + (sub + 8 * c) * 4);
                const float f = on ? a.qscale : 0.f;
                qr[g][c * 4] = x.x * f;
                qr[g][c * 4 + 1] = x.y * f;
                qr[g][c * 4 + 2] = x.z * f;
                qr[g][c * 4 + 3] = x.w * f;
            }
        }
    };
    load_q(w.b, w.h);
    int it = 0;
    bool ok = true;
    while (w.left > 0) {
        const int b = w.b, h = w.h, i0 = w.i;
        const Tiles t = w.t;
        const int i1 = min(t.n, i0 + w.left);
        const long long seg_first = sh.first + (sh.count - w.left);
        float o[HG][F::CPL], m[HG], l[HG];
#pragma unroll
        for (int g = 0; g < HG; ++g) {
            m[g] = -INFINITY;
            l[g] = 0.f;
#pragma unroll
            for (int c = 0; c < F::CPL; ++c) o[g][c] = 0.f;
        }
        for (int i = i0; i < i1; ++i, ++it) {
            const int s = it % STAGES;
            consume_wait(&r, it, ok, a.c.status);
            const unsigned char* ks = buf + s * Z::STAGE_BYTES;
            const unsigned char* vs = ks + Z::STAGE_BYTES / 2;
            const int row0 = t.row0(i, TK);
            float p[HG][F::NR];
            bool see[F::NR];
#pragma unroll
            for (int j = 0; j < F::NR; ++j) {
                const int rr = part * F::RW + grp + 4 * j;
                see[j] = t.sees(row0 + rr);
                float kf[F::CPL];
#pragma unroll
                for (int c = 0; c < F::CH; ++c) {
                    const float4 x = *reinterpret_cast<const float4*>(ks + rr * (D * 4) + (sub + 8 * c) * 16);
                    kf[c * 4] = x.x; kf[c * 4 + 1] = x.y; kf[c * 4 + 2] = x.z; kf[c * 4 + 3] = x.w;
                }
#pragma unroll
                for (int g = 0; g < HG; ++g) {
                    float acc = 0.f;
#pragma unroll
                    for (int c = 0; c < F::CPL; ++c) acc = fmaf(qr[g][c], kf[c], acc);
                    p[g][j] = acc;
                }
            }
#pragma unroll
            for (int g = 0; g < HG; ++g) {
                float mx = m[g];
#pragma unroll
                for (int j = 0; j < F::NR; ++j) {
                    float x = p[g][j];
                    x += __shfl_xor_sync(0xffffffffu, x, 1);
                    x += __shfl_xor_sync(0xffffffffu, x, 2);
                    x += __shfl_xor_sync(0xffffffffu, x, 4);
                    p[g][j] = x;
                    if (see[j]) mx = fmaxf(mx, x);
                }
                const float corr = m[g] == -INFINITY ? 0.f : ex2(m[g] - mx);
                float ps = 0.f;
#pragma unroll
                for (int j = 0; j < F::NR; ++j) {
                    p[g][j] = see[j] ? ex2(p[g][j] - mx) : 0.f;
                    ps += p[g][j];
                }
                l[g] = l[g] * corr + ps;
                m[g] = mx;
#pragma unroll
                for (int c = 0; c < F::CPL; ++c) o[g][c] *= corr;
            }
#pragma unroll
            for (int j = 0; j < F::NR; ++j) {
                if (!see[j]) continue;                    // the row may hold anything
                const int rr = part * F::RW + grp + 4 * j;
#pragma unroll
                for (int c = 0; c < F::CH; ++c) {
                    const float4 x = *reinterpret_cast<const float4*>(vs + rr * (D * 4) + (sub + 8 * c) * 16);
#pragma unroll
                    for (int g = 0; g < HG; ++g) {
                        o[g][c * 4] = fmaf(p[g][j], x.x, o[g][c * 4]);
                        o[g][c * 4 + 1] = fmaf(p[g][j], x.y, o[g][c * 4 + 1]);
                        o[g][c * 4 + 2] = fmaf(p[g][j], x.z, o[g][c * 4 + 2]);
                        o[g][c * 4 + 3] = fmaf(p[g][j], x.w, o[g][c * 4 + 3]);
                    }
                }
            }
            consumed(&r, s, ok, lane);
            w.next(a, TK);
        }
        const bool whole = i0 == 0 && i1 == t.n;
        const Dest ds = segment_dest(a, sh, seg_first, whole, b, h);
        if (w.left > 0) load_q(w.b, w.h);
        // the warp's four row groups, then the four warps of a head group
#pragma unroll
        for (int off = 8; off <= 16; off <<= 1)
#pragma unroll
            for (int g = 0; g < HG; ++g) {
                const float m2 = __shfl_xor_sync(0xffffffffu, m[g], off), l2 = __shfl_xor_sync(0xffffffffu, l[g], off);
                const float M = fmaxf(m[g], m2);
                const float wa = m[g] == -INFINITY ? 0.f : ex2(m[g] - M), wb = m2 == -INFINITY ? 0.f : ex2(m2 - M);
                m[g] = M;
                l[g] = l[g] * wa + l2 * wb;
#pragma unroll
                for (int c = 0; c < F::CPL; ++c) {
                    const float o2 = __shfl_xor_sync(0xffffffffu, o[g][c], off);
                    o[g][c] = o[g][c] * wa + o2 * wb;
                }
            }
        if (grp == 0) {
#pragma unroll
            for (int g = 0; g < HG; ++g) {
                float* dst = red + (warp * HG + g) * (D + 2);
#pragma unroll
                for (int c = 0; c < F::CH; ++c)
#pragma unroll
                    for (int e = 0; e < 4; ++e) dst[(sub + 8 * c) * 4 + e] = o[g][c * 4 + e];
                if (sub == 0) {
                    dst[D] = m[g];
                    dst[D + 1] = l[g];
                }
            }
        }
        bar_consumers<NW * 32>();
        finish_f32<D, HG, 4, NW>(a, &r, sh, t, red, ds, seg_first, i0, whole, b, h);
    }
    drain(&r);
    leave(a);
}

// ---- fp32, many heads per KV head -----------------------------------------------
// MH blocks of eight heads on the tensor cores, three tf32 products each: S = q K^T
// with the heads as the matrix's M (so P is an operand as it stands) and eight rows as
// its N; O += P V with eight columns as N and the rows as K.
template <int D, int MH>
struct TGeo {
    using Z = Geo<float, D>;
    static constexpr int NW = Z::TK >= 32 ? 4 : 2, RW = Z::TK / NW, NB = RW / 8;   // warps, their rows, in eights
    static constexpr int CTAS = MH * D <= 128 || (MH == 1 && NW == 2) ? 2 : 1;     // O: MH D / 4 a thread
    static constexpr int SMEM = STAGES * Z::STAGE_BYTES + NW * 8 * MH * (D + 2) * 4 + 128;
};

template <int D, int MH>
__global__ void __launch_bounds__((TGeo<D, MH>::NW + 1) * 32, (TGeo<D, MH>::CTAS))
decode_f32_heads_kernel(const __grid_constant__ DecodeArgs a) {
    using Z = Geo<float, D>;
    using F = TGeo<D, MH>;
    constexpr int TK = Z::TK, NW = F::NW, NB = F::NB, HG = 8 * MH, THREADS = (NW + 1) * 32;
    extern __shared__ unsigned char smem_raw[];
    __shared__ Ring r;
    unsigned char* buf = smem_raw + ((128u - (smem_u32(smem_raw) & 127u)) & 127u);
    float* red = reinterpret_cast<float*>(buf + STAGES * Z::STAGE_BYTES);   // [warp][HG][D + 2]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    pdl_trigger();
    if (tid == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(r.full + s, 1);
            mbar_init(r.empty + s, NW);
        }
        fence_barrier_init();
        r.issued = 0;
        r.failed = 0;
    }
    plan_share<THREADS>(a, TK, &r.share, r.scan);
    const Share sh = r.share;
    if (sh.count == 0) {
        leave(a);
        return;
    }
    Walk w;
    w.b = sh.b; w.h = sh.h; w.i = sh.i; w.left = sh.count;
    w.t = tiles_of(a, seq_len(a.c, w.b), TK);
    __syncthreads();

    if (warp == NW) {
        produce<float, D>(nullptr, nullptr, a, &r, buf, w, lane);
        drain(&r);
        leave(a);
        return;
    }
    // A fragment's lane (fr, fc) has heads fr, fr + 8 at words fc, fc + 4 of a step.
    // The sum's order is free, so those words are four neighbouring columns of a
    // sixteen for two steps, one 16-byte load of q and of K.
    const int fr = lane >> 2, fc = lane & 3;
    // Both halves of q, as the lanes take them, lie where the pair's states go in the
    // end (they are the same for all warps, and split once a pair).
    constexpr int QN = MH * D / 16 / NW;
    uint4* qs = reinterpret_cast<uint4*>(red);               // [MH][D / 16][hi, lo][lane]
    float4 nq[QN];                                           // this warp's part of the next pair's
    auto fetch_q = [&](int b, int h) {
#pragma unroll
        for (int u = 0; u < QN; ++u) {
            const int i = warp * QN + u, n = i / (D / 16), c = i % (D / 16), g = n * 8 + fr;
            nq[u] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (g < a.G)
                nq[u] = *reinterpret_cast<const float4*>(static_cast<const float*>(a.q) + (long long)b * a.q_stride +
                                                         (long long)(h * a.G + g) * D + c * 16 + fc * 4);
        }
    };
    fetch_q(w.b, w.h);
    int it = 0;
    bool ok = true;
    while (w.left > 0) {
        const int b = w.b, h = w.h, i0 = w.i;
        const Tiles t = w.t;
        const int i1 = min(t.n, i0 + w.left);
        const long long seg_first = sh.first + (sh.count - w.left);
#pragma unroll
        for (int u = 0; u < QN; ++u) {
            uint4 hi, lo;
            split_tf32(__float_as_uint(nq[u].x * a.qscale), hi.x, lo.x);
            split_tf32(__float_as_uint(nq[u].y * a.qscale), hi.y, lo.y);
            split_tf32(__float_as_uint(nq[u].z * a.qscale), hi.z, lo.z);
            split_tf32(__float_as_uint(nq[u].w * a.qscale), hi.w, lo.w);
            qs[(warp * QN + u) * 64 + lane] = hi;
            qs[(warp * QN + u) * 64 + 32 + lane] = lo;
        }
        bar_consumers<NW * 32>();
        // O: heads fr + 8 n, columns 8 c + 2 fc, + 1
        float o[D / 8][2 * MH], m[MH], l[MH];
#pragma unroll
        for (int n = 0; n < MH; ++n) {
            m[n] = -INFINITY;
            l[n] = 0.f;
        }
#pragma unroll
        for (int c = 0; c < D / 8; ++c)
#pragma unroll
            for (int e = 0; e < 2 * MH; ++e) o[c][e] = 0.f;
        for (int i = i0; i < i1; ++i, ++it) {
            const int s = it % STAGES;
            consume_wait(&r, it, ok, a.c.status);
            const unsigned char* ks = buf + s * Z::STAGE_BYTES + warp * F::RW * (D * 4);
            const unsigned char* vs = ks + Z::STAGE_BYTES / 2;
            const int row0 = t.row0(i, TK) + warp * F::RW;
            // scores: heads fr + 8 n, rows 8 x + 2 fc, + 1.  Odd rows read the second
            // sixteen of a pair first: eight lanes then meet all banks.
            float p[NB][2 * MH];
            bool see[NB][2];
#pragma unroll
            for (int x = 0; x < NB; ++x) {
#pragma unroll
                for (int e = 0; e < 2 * MH; ++e) p[x][e] = 0.f;
                const unsigned char* kr = ks + (x * 8 + fr) * (D * 4) + fc * 16 + (fr & 1) * 64;
#pragma unroll
                for (int c = 0; c < D / 16; c += 4) {
                    FragA<2> qf[4];
                    FragB<2> kf[4];
#pragma unroll
                    for (int u = 0; u < 4; u += 2) {
                        const uint4 y = *reinterpret_cast<const uint4*>(kr + (c + u) * 64);
                        const uint4 z = *reinterpret_cast<const uint4*>(kr + (c + u) * 64 + ((fr & 1) ? -64 : 64));
                        const uint4 k0 = (fr & 1) ? z : y, k1 = (fr & 1) ? y : z;
                        split_tf32(k0.x, kf[u].h[0][0], kf[u].l[0][0]);
                        split_tf32(k0.y, kf[u].h[0][1], kf[u].l[0][1]);
                        split_tf32(k0.z, kf[u].h[1][0], kf[u].l[1][0]);
                        split_tf32(k0.w, kf[u].h[1][1], kf[u].l[1][1]);
                        split_tf32(k1.x, kf[u + 1].h[0][0], kf[u + 1].l[0][0]);
                        split_tf32(k1.y, kf[u + 1].h[0][1], kf[u + 1].l[0][1]);
                        split_tf32(k1.z, kf[u + 1].h[1][0], kf[u + 1].l[1][0]);
                        split_tf32(k1.w, kf[u + 1].h[1][1], kf[u + 1].l[1][1]);
                    }
#pragma unroll
                    for (int u = 0; u < 4; ++u)
#pragma unroll
                        for (int n = 0; n < 2; ++n) {
                            uint4 hi = make_uint4(0, 0, 0, 0), lo = hi;
                            if (n < MH) {
                                hi = qs[(n * (D / 16) + c + u) * 64 + lane];
                                lo = qs[(n * (D / 16) + c + u) * 64 + 32 + lane];
                            }
                            qf[u].h[0][n] = hi.x; qf[u].h[0][2 + n] = hi.y;
                            qf[u].h[1][n] = hi.z; qf[u].h[1][2 + n] = hi.w;
                            qf[u].l[0][n] = lo.x; qf[u].l[0][2 + n] = lo.y;
                            qf[u].l[1][n] = lo.z; qf[u].l[1][2 + n] = lo.w;
                        }
                    float d[4][4];
                    mma_exact(d, [&](int n) -> const FragA<2>& { return qf[n]; }, kf);
#pragma unroll
                    for (int e = 0; e < 2 * MH; ++e) p[x][e] += (d[0][e] + d[1][e]) + (d[2][e] + d[3][e]);
                }
            }
            float mx[MH];
            bool moved = false;
#pragma unroll
            for (int n = 0; n < MH; ++n) mx[n] = m[n];
#pragma unroll
            for (int x = 0; x < NB; ++x)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    see[x][e] = t.sees(row0 + x * 8 + 2 * fc + e);
#pragma unroll
                    for (int n = 0; n < MH; ++n)
                        if (see[x][e]) mx[n] = fmaxf(mx[n], p[x][2 * n + e]);
                }
#pragma unroll
            for (int n = 0; n < MH; ++n) {
                mx[n] = fmaxf(mx[n], __shfl_xor_sync(0xffffffffu, mx[n], 1));
                mx[n] = fmaxf(mx[n], __shfl_xor_sync(0xffffffffu, mx[n], 2));
                moved |= mx[n] != m[n];
            }
            if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                for (int n = 0; n < MH; ++n) {
                    const float corr = m[n] == -INFINITY ? 0.f : ex2(m[n] - mx[n]);
                    l[n] *= corr;
                    m[n] = mx[n];
#pragma unroll
                    for (int c = 0; c < D / 8; ++c) {
                        o[c][2 * n] *= corr;
                        o[c][2 * n + 1] *= corr;
                    }
                }
            }
            // P's words fc, fc + 4 are rows 2 fc, 2 fc + 1
            FragA<NB> pf;
            bool all = true;
#pragma unroll
            for (int x = 0; x < NB; ++x)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    all &= see[x][e];
#pragma unroll
                    for (int n = 0; n < 2; ++n) {
                        uint32_t &hi = pf.h[x][2 * e + n], &lo = pf.l[x][2 * e + n];
                        if (n < MH) {
                            const float y = see[x][e] ? ex2(p[x][2 * n + e] - m[n]) : 0.f;
                            l[n] += y;
                            split_tf32(__float_as_uint(y), hi, lo);
                        } else {
                            hi = lo = 0;
                        }
                    }
                }
            all = __all_sync(0xffffffffu, all);
            // V: lane (fr, fc) has column fr of each block in rows 2 fc, 2 fc + 1, which
            // share their banks over fc: it reads four blocks from block fc on, and turns
            // them back.
#pragma unroll
            for (int c = 0; c < D / 8; c += 4) {
                FragB<NB> vf[4];
#pragma unroll
                for (int x = 0; x < NB; ++x)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const unsigned char* vr = vs + (x * 8 + 2 * fc + e) * (D * 4) + c * 32 + fr * 4;
                        uint32_t y[4], z[4];
#pragma unroll
                        for (int u = 0; u < 4; ++u) y[u] = *reinterpret_cast<const uint32_t*>(vr + ((u + fc) & 3) * 32);
                        if (!all && !see[x][e]) y[0] = y[1] = y[2] = y[3] = 0;      // the row may hold anything
#pragma unroll
                        for (int u = 0; u < 4; ++u) z[u] = (fc & 1) ? y[(u + 3) & 3] : y[u];
#pragma unroll
                        for (int u = 0; u < 4; ++u)
                            split_tf32((fc & 2) ? z[(u + 2) & 3] : z[u], vf[u].h[x][e], vf[u].l[x][e]);
                    }
                float d[4][4];
                mma_exact(d, [&](int) -> const FragA<NB>& { return pf; }, vf);
#pragma unroll
                for (int u = 0; u < 4; ++u)
#pragma unroll
                    for (int e = 0; e < 2 * MH; ++e) o[c + u][e] += d[u][e];
            }
            consumed(&r, s, ok, lane);
            w.next(a, TK);
        }
        const bool whole = i0 == 0 && i1 == t.n;
        const Dest ds = segment_dest(a, sh, seg_first, whole, b, h);
        if (w.left > 0) fetch_q(w.b, w.h);
        bar_consumers<NW * 32>();                            // everyone is done with q
#pragma unroll
        for (int n = 0; n < MH; ++n) {
            l[n] += __shfl_xor_sync(0xffffffffu, l[n], 1);
            l[n] += __shfl_xor_sync(0xffffffffu, l[n], 2);
            float* dst = red + (warp * HG + n * 8 + fr) * (D + 2);
#pragma unroll
            for (int c = 0; c < D / 8; ++c)
                *reinterpret_cast<float2*>(dst + c * 8 + 2 * fc) = make_float2(o[c][2 * n], o[c][2 * n + 1]);
            if (fc == 0) *reinterpret_cast<float2*>(dst + D) = make_float2(m[n], l[n]);
        }
        bar_consumers<NW * 32>();
        finish_f32<D, HG, NW, NW>(a, &r, sh, t, red, ds, seg_first, i0, whole, b, h);
    }
    drain(&r);
    leave(a);
}

using F32Fn = void (*)(const DecodeArgs);
struct F32Pick {
    F32Fn fn;
    int threads, smem, ctas;
};
template <int D, int HG, int NG>
static F32Pick f32_pick() {
    return {decode_f32_kernel<D, HG, NG>, (NG * 4 + 1) * 32, f32_smem<D, HG, NG>(), f32_ctas<NG>()};
}
template <int D, int MH>
static F32Pick f32_heads_pick() {
    using F = TGeo<D, MH>;
    return {decode_f32_heads_kernel<D, MH>, (F::NW + 1) * 32, F::SMEM, F::CTAS};
}
template <int D>
static F32Pick f32_pick_g(int G) {
    // the tensor cores take as long for one head as for eight: 16 sequences of up to 4000
    // rows, 8 KV heads of 128: 90 us, FMAs 72 / 85 / 126 us at 2 / 4 / 8 heads each
    if (G > 8) return f32_heads_pick<D, (D <= 128 ? 2 : 1)>();       // d = 256 has at most 8
    if (G > 4) return f32_heads_pick<D, 1>();
    if (G == 1) return f32_pick<D, 1, 1>();
    if (G == 2) return f32_pick<D, 2, 1>();
    return f32_pick<D, (D <= 128 ? 4 : 2), (D <= 128 ? 1 : 2)>();
}
static F32Pick f32_pick_d(int d, int G) {
    return d == 64 ? f32_pick_g<64>(G) : d == 128 ? f32_pick_g<128>(G) : f32_pick_g<256>(G);
}

// CTAs of a decode launch: as many as fit the GPU at once.
int decode_grid(const sa_ctx* ctx, const sa_paged_kv* kv, int hq) {
    const int ctas = kv->dtype == SA_F32 ? f32_pick_d(kv->d, hq / kv->hkv).ctas : (kv->d == 256 ? 1 : 2);
    return std::min(ctx->num_sms * ctas, SA_PAGED_ZERO_BYTES / 4);
}

template <int D>
static int launch_bf16(cudaStream_t st, int grid, bool overlap, const CUtensorMap& tk, const CUtensorMap& tv, const DecodeArgs& a) {
    auto one = decode_bf16_kernel<D, 1>;
    auto two = decode_bf16_kernel<D, (D < 256 ? 2 : 1)>;
    auto k = a.G <= 8 ? one : two;
    SA_RC_TRY(set_smem_attr_once((const void*)k, bf16_smem<D>()));
    if (overlap) {
        SA_CUDA_TRY(launch_pdl(k, dim3(grid), dim3(BTHREADS), bf16_smem<D>(), st, tk, tv, a));
    } else {
        k<<<grid, BTHREADS, bf16_smem<D>(), st>>>(tk, tv, a);
        SA_CUDA_TRY(cudaGetLastError());
    }
    return SA_OK;
}

int decode_launch(sa_ctx* ctx, const sa_paged_kv* kv, const void* q, long long q_stride, int hq, int window, int sinks,
                  float scale, void* out, long long o_stride, const PrefixParts* prefix, const DecodeWs& ws) {
    DecodeArgs a = {};
    a.c = make_cache(ctx, kv);
    a.q = q;
    a.out = out;
    a.q_stride = q_stride;
    a.o_stride = o_stride;
    a.hq = hq;
    a.G = hq / kv->hkv;
    a.window = window;
    a.sinks = sinks;
    a.qscale = scale * LOG2E;
    a.prefixed = !prefix ? 0 : prefix->join ? JOIN_HERE : JOIN_LATER;
    if (prefix) a.prefix = *prefix;
    a.ws = ws;
    const bool overlap = prefix && prefix->parts > 0;
    const int grid = decode_grid(ctx, kv, hq);
    cudaStream_t st = ctx->stream;
    if (kv->dtype == SA_F32) {
        const F32Pick p = f32_pick_d(kv->d, a.G);
        SA_RC_TRY(set_smem_attr_once((const void*)p.fn, p.smem));
        if (overlap) {
            SA_CUDA_TRY(launch_pdl(p.fn, dim3(grid), dim3(p.threads), p.smem, st, a));
        } else {
            p.fn<<<grid, p.threads, p.smem, st>>>(a);
            SA_CUDA_TRY(cudaGetLastError());
        }
        return SA_OK;
    }
    CUtensorMap tk, tv;
    const int tile = kv->d == 64 ? Geo<__nv_bfloat16, 64>::TK : Geo<__nv_bfloat16, 128>::TK;
    const int box = std::min(kv->page_size, tile);
    SA_RC_TRY(make_page_tmap(&tk, kv->k_pages, kv, box));
    SA_RC_TRY(make_page_tmap(&tv, kv->v_pages, kv, box));
    return kv->d == 64    ? launch_bf16<64>(st, grid, overlap, tk, tv, a)
           : kv->d == 128 ? launch_bf16<128>(st, grid, overlap, tk, tv, a)
                          : launch_bf16<256>(st, grid, overlap, tk, tv, a);
}

size_t decode_ws_layout(const sa_ctx* ctx, const sa_paged_kv* kv, int hq, bool prefix, void* base, DecodeWs* ws) {
    const int grid = decode_grid(ctx, kv, hq), G = hq / kv->hkv;
    const size_t slots = (size_t)grid * 2 * G, rows = (size_t)kv->n_seqs * hq, d4 = (size_t)kv->d * 4;
    size_t at = 0;
    unsigned char* p = static_cast<unsigned char*>(base);
    auto take = [&](size_t bytes) {
        const size_t o = at;
        at += align_up(bytes, 256);
        return p ? p + o : nullptr;
    };
    DecodeWs w = {};
    // first, and as long for every shape: calls of other shapes leave it zero too
    w.count = reinterpret_cast<unsigned*>(take(SA_PAGED_ZERO_BYTES));
    w.slot_o = reinterpret_cast<float*>(take(slots * d4));
    w.slot_ml = reinterpret_cast<float2*>(take(slots * 8));
    if (prefix) {
        w.state_o = reinterpret_cast<float*>(take(rows * d4));
        w.state_ml = reinterpret_cast<float2*>(take(rows * 8));
        w.pair = reinterpret_cast<int4*>(take((size_t)kv->n_seqs * kv->hkv * sizeof(int4)));
    }
    w.d = kv->d;
    w.out_elt = kv->dtype == SA_F32 ? 4 : 2;
    if (ws) *ws = w;
    return at;
}

}  // namespace pg
}  // namespace sa

SA_API int sa_attn_paged_decode_workspace(sa_ctx* ctx, const sa_paged_kv* kv, int hq, size_t* bytes) {
    using namespace sa;
    const char* fn = "sa_attn_paged_decode_workspace";
    clear_error();
    SA_CHECK_ARG(ctx && bytes, "%s: NULL argument", fn);
    SA_RC_TRY(pg::check_cache(fn, kv));
    SA_RC_TRY(pg::check_heads(fn, kv, hq));
    *bytes = pg::decode_ws_layout(ctx, kv, hq, false, nullptr, nullptr);
    return SA_OK;
}

SA_API int sa_attn_paged_decode(sa_ctx* ctx, const sa_paged_kv* kv, const void* q, long long q_stride, int hq, int window,
                                int sinks, float scale, void* out, long long o_stride, void* workspace,
                                size_t workspace_bytes) {
    using namespace sa;
    const char* fn = "sa_attn_paged_decode";
    clear_error();
    SA_RC_TRY(pg::check_cache(fn, kv));
    SA_RC_TRY(pg::check_heads(fn, kv, hq));
    SA_RC_TRY(pg::check_scale(fn, scale));
    SA_CHECK_ARG(window >= 0 && sinks >= 0, "%s: window %d, sinks %d", fn, window, sinks);
    if (kv->n_seqs == 0) return SA_OK;
    const int e = kv->dtype == SA_F32 ? 4 : 2;
    SA_RC_TRY(pg::check_rows(fn, "q", q, q_stride, (long long)hq * kv->d, e));
    SA_RC_TRY(pg::check_rows(fn, "out", out, o_stride, (long long)hq * kv->d, e));
    SA_CHECK_ARG(ctx != nullptr, "%s: ctx is NULL", fn);
    DeviceGuard guard(ctx->device);
    pg::DecodeWs ws;
    const size_t need = pg::decode_ws_layout(ctx, kv, hq, false, workspace, &ws);
    SA_CHECK_ARG(workspace && ((uintptr_t)workspace & 255) == 0 && workspace_bytes >= need,
                 "%s: workspace of %zu bytes (want %zu, 256-byte aligned)", fn, workspace_bytes, need);
    return pg::decode_launch(ctx, kv, q, q_stride, hq, window, sinks, scale, out, o_stride, nullptr, ws);
}
