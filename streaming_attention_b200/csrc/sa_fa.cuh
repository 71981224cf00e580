// sa_fa.cuh -- the pieces of the tcgen05 attention kernels (sa_prefill.cu,
// sa_paged_tc.cu): waits that give up, TMEM columns of two query slots, and a
// row's softmax step.
#pragma once
#include <cuda_bf16.h>

#include "sa_tc.cuh"

namespace sa {
namespace pf {

constexpr int BM = 128, BN = 128;              // query rows and keys of a tile
// TMEM columns of slot x: S (128 fp32 columns), P (bf16 pairs over the upper
// half of S), O
__device__ __forceinline__ uint32_t col_s(int x) { return (uint32_t)x * 128u; }
__device__ __forceinline__ uint32_t col_p(int x) { return (uint32_t)x * 128u + 64u; }
__device__ __forceinline__ uint32_t col_o(int x) { return 256u + (uint32_t)x * 128u; }
constexpr float LOG2E = 1.4426950408889634f;
constexpr float RESCALE_THRESHOLD = 8.0f;      // log2 units

__device__ __forceinline__ bool wait_ab(uint64_t* bar, uint32_t parity, volatile int* abort, int* status) {
    if (mbar_try_wait(bar, parity)) return true;
    const unsigned long long t0 = globaltimer();
    while (!mbar_try_wait(bar, parity)) {
        if (*abort) return false;
        if (globaltimer() - t0 > kWaitLimitNs) {
            *abort = 1;
            atomicExch(status, SA_STATUS_TIMEOUT);
            return false;
        }
    }
    return true;
}

// The same for a whole (converged) warp: its lanes look at the barrier and the clock
// one by one, and go on together or give up together.
__device__ __forceinline__ bool wait_ab_warp(uint64_t* bar, uint32_t parity, volatile int* abort, int* status) {
    return __all_sync(0xffffffffu, wait_ab(bar, parity, abort, status));
}

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
}

// 2^x on the FMA pipe, for x <= 8 (clamped below at -126): x = n + f with n
// the nearest integer (taken from the low mantissa bits of x + 1.5*2^23) and
// f in [-0.5, 0.5]; 2^f by a degree-3 polynomial fitted here to 2^f on that
// interval (max relative error 7.5e-5, far below the bf16 rounding of P);
// 2^n added to the exponent field with an integer add.  No transcendental-
// unit instruction is used.
__device__ __forceinline__ float exp2_poly(float x) {
    x = fmaxf(x, -126.f);
    const float t = x + 12582912.f;
    const float f = x - (t - 12582912.f);
    float p = fmaf(0.0551716685295105f, f, 0.2426111251115799f);
    p = fmaf(p, f, 0.6932609677314758f);
    p = fmaf(p, f, 0.9999280571937561f);
    return __int_as_float(__float_as_int(p) + (__float_as_int(t) << 23));
}

// Every POLY-th exponential (by column) on the FMA pipe; 0: all on the SFU.
template <int POLY>
__device__ __forceinline__ float exp2_mix(float x, int c) {
    if constexpr (POLY > 0) {
        if ((c % POLY) == POLY - 1) return exp2_poly(x);
    }
    return ex2(x);
}

// Max of a row's 128 raw scores (eight independent chains).
__device__ __forceinline__ float row_max(const float* sc) {
    float mx[8];
#pragma unroll
    for (int c = 0; c < 8; ++c) mx[c] = sc[c];
#pragma unroll
    for (int c = 8; c < BN; c += 8)
#pragma unroll
        for (int i = 0; i < 8; ++i) mx[i] = fmaxf(mx[i], sc[c + i]);
    return fmaxf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), fmaxf(fmaxf(mx[4], mx[5]), fmaxf(mx[6], mx[7])));
}

// P = 2^(sc*sl2 + nm) for one row's 128 scores, written to TMEM at p_addr as
// 64 columns of bf16 pairs (two tcgen05.st of 32 columns, not waited for);
// returns the fp32 row sum.  With TRACK_MAX the max of the raw scores is
// found in the same pass and written to *mx_out.
template <int POLY, bool TRACK_MAX>
__device__ __forceinline__ float emit_p(const float* sc, float sl2, float nm, uint32_t p_addr, float* mx_out) {
    float ps[4] = {0.f, 0.f, 0.f, 0.f};
    float mx[8];
    if constexpr (TRACK_MAX) {
#pragma unroll
        for (int i = 0; i < 8; ++i) mx[i] = sc[i];
    }
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
        uint32_t pk[32];
#pragma unroll
        for (int c = hf * 64; c < hf * 64 + 64; c += 2) {
            if constexpr (TRACK_MAX) {
                mx[c & 7] = fmaxf(mx[c & 7], sc[c]);
                mx[(c + 1) & 7] = fmaxf(mx[(c + 1) & 7], sc[c + 1]);
            }
            const float e0 = exp2_mix<POLY>(fmaf(sc[c], sl2, nm), c);
            const float e1 = exp2_mix<POLY>(fmaf(sc[c + 1], sl2, nm), c + 1);
            ps[(c >> 1) & 3] += e0 + e1;
            pk[(c >> 1) & 31] = pack_bf16(e0, e1);
        }
        tc::tmem_st32(p_addr + hf * 32, pk);
    }
    if constexpr (TRACK_MAX)
        *mx_out = fmaxf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), fmaxf(fmaxf(mx[4], mx[5]), fmaxf(mx[6], mx[7])));
    return (ps[0] + ps[1]) + (ps[2] + ps[3]);
}

// emit_p with the scale and the row sum on packed fp32 pairs (fma/add.f32x2:
// half the FMA-pipe instructions; each element rounds as in emit_p, the sum's
// order differs).
__device__ __forceinline__ unsigned long long f2(float a, float b) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void un2(unsigned long long r, float& a, float& b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(r));
}
__device__ __forceinline__ unsigned long long fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
    unsigned long long d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ unsigned long long add2(unsigned long long a, unsigned long long b) {
    unsigned long long d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
// Max of a row's 128 scores, three operands at a time.
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float row_max3(const float* sc) {
    float mx[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) mx[i] = max3(sc[3 * i], sc[3 * i + 1], sc[3 * i + 2]);
#pragma unroll
    for (int i = 0; i < 52; ++i) mx[i & 7] = max3(mx[i & 7], sc[24 + 2 * i], sc[25 + 2 * i]);
    return max3(max3(mx[0], mx[1], mx[2]), max3(mx[3], mx[4], mx[5]), fmaxf(mx[6], mx[7]));
}

// Bits [0, n) of a word.
__device__ __forceinline__ uint32_t bits_below(int n) { return n <= 0 ? 0u : (n >= 32 ? 0xffffffffu : (1u << n) - 1u); }
// -infinity where the bit of a row's 32 scores is clear.
__device__ __forceinline__ void keep_bits(float* sc, uint32_t bits) {
    if (__all_sync(0xffffffffu, bits == 0xffffffffu)) return;
#pragma unroll
    for (int i = 0; i < 32; ++i) sc[i] = (bits & (1u << i)) ? sc[i] : -INFINITY;
}

// 2^(sc * s2 + n2) of N of a row's scores as N / 2 bf16 pairs in pk, added to
// the row's sums ps.
template <int N>
__device__ __forceinline__ void exp_pairs(const float* sc, unsigned long long s2, unsigned long long n2, uint32_t* pk,
                                          unsigned long long (&ps)[4]) {
#pragma unroll
    for (int c = 0; c < N; c += 2) {
        float e0, e1;
        un2(fma2(f2(sc[c], sc[c + 1]), s2, n2), e0, e1);
        e0 = ex2(e0);
        e1 = ex2(e1);
        ps[(c >> 1) & 3] = add2(ps[(c >> 1) & 3], f2(e0, e1));
        pk[c >> 1] = pack_bf16(e0, e1);
    }
}

}  // namespace pf
}  // namespace sa
