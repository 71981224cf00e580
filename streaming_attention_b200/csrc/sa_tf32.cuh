// sa_tf32.cuh -- fp32 products on the tensor cores.
//
// An operand x is the sum of two tf32 numbers, hi = x rounded to 11 significant
// bits and lo = x - hi (exact), and
//   x y = hi hi' + hi lo' + lo hi'  (+ lo lo', at most 2^-22 of x y, left out),
// each product exact in the fp32 accumulator; the tensor core drops lo's bits past
// its eleventh, another 2^-22.  So three mma.m16n8k8 give what an fp32 FMA loop
// gives to within its own rounding, at 512 / 3 FMA a clock and SM (measured)
// where FMAs have 128 and spend half of their slots on feeding them.  (bf16
// pairs would run twice as fast, at 2^-17.)
#pragma once
#include <cstdint>

namespace sa {
namespace pg {

__device__ __forceinline__ void split_tf32(uint32_t x, uint32_t& hi, uint32_t& lo) {
    hi = (x + 0x1000u) & 0xffffe000u;
    lo = __float_as_uint(__uint_as_float(x) - __uint_as_float(hi));
}
__device__ __forceinline__ void mma1688(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The product's first step: d = A B.
__device__ __forceinline__ void mma1688_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
// The hi and lo fragments of S steps of eight.
template <int S>
struct FragA {
    uint32_t h[S][4], l[S][4];
};
template <int S>
struct FragB {
    uint32_t h[S][2], l[S][2];
};
// d[n] = A[n] B[n], the small terms first: the tensor core cuts its sums off where
// fp32 rounds, so it sums 8 S products from zero, and the caller adds them to a long
// sum in fp32.  Term by term over the N blocks: a block's products wait for one
// another, the blocks' do not.  a(n) -> A[n].
template <int N, int S, typename A>
__device__ __forceinline__ void mma_exact(float (&d)[N][4], A a, const FragB<S> (&b)[N]) {
#pragma unroll
    for (int n = 0; n < N; ++n) mma1688_first(d[n], a(n).l[0], b[n].h[0][0], b[n].h[0][1]);
#pragma unroll
    for (int n = 0; n < N; ++n) mma1688(d[n], a(n).h[0], b[n].l[0][0], b[n].l[0][1]);
#pragma unroll
    for (int s = 1; s < S; ++s) {
#pragma unroll
        for (int n = 0; n < N; ++n) mma1688(d[n], a(n).l[s], b[n].h[s][0], b[n].h[s][1]);
#pragma unroll
        for (int n = 0; n < N; ++n) mma1688(d[n], a(n).h[s], b[n].l[s][0], b[n].l[s][1]);
    }
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
        for (int n = 0; n < N; ++n) mma1688(d[n], a(n).h[s], b[n].h[s][0], b[n].h[s][1]);
}

}  // namespace pg
}  // namespace sa
