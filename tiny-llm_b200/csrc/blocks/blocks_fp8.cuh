// Numbers of 8 bits (e4m3) with one fp32 scale for each block of 128 x 128 of a matrix and each run of 128 of a row.
#pragma once

#include <cuda_fp8.h>

#include "blocks_common.cuh"

namespace tlb {

constexpr int kF8Block = 128;
constexpr float kF8Top = 448.f;                       // the largest e4m3 number
constexpr float kF8Smallest = 7.888609052210118e-31f;  // 2^-100: a run of smaller numbers is scaled as if this were its largest

// What a run's largest magnitude makes of it: number * times is rounded to e4m3, which times `scale` it stands for.  Both are quotients
// rounded once: with products by rounded reciprocals, rows of bf16 numbers (whose quotients often lie in the middle between two e4m3
// numbers) would round another way.  A run that holds an infinity or a NaN stands for NaN.
struct F8Scale {
    float times, scale;
};
__device__ __forceinline__ F8Scale f8_scale(float most) {
    const float m = most < kF8Smallest ? kF8Smallest : most;  // keeps NaN
    const bool fine = m < INFINITY;
    return {fine ? __fdiv_rn(kF8Top, m) : 0.f, fine ? __fdiv_rn(m, kF8Top) : __int_as_float(0x7fffffff)};
}
// The larger one, NaN if either is.
__device__ __forceinline__ float f8_most(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// Four numbers in the order of memory, nearest even, nothing beyond 448.
__device__ __forceinline__ uint32_t f8_pack4(float a, float b, float c, float d) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | hi << 16;
}

// blocks_fp8_rows.cu
struct F8Rows {
    const void *x;  // [rows, cols], ldx apart; gated: fp32, 128 gate columns, then 128 up columns, for each run of the inner row
    long long ldx;
    int rows, cols, dtype;
    bool gated;
    int act;
    float limit, slope;
    uint8_t *q;  // [rows, ldq], ldq a multiple of 16; zero behind the last column
    int ldq;
    float *scales;  // [ceil(cols / 128)][ld_scales]
    int ld_scales;
};
int f8_rows(const F8Rows &a, cudaStream_t st);

// blocks_fp8_product.cu: out [rows, n] = (rows of q) . w^T (+ bias)
struct F8Product {
    const uint8_t *q;
    const float *sx;
    int ldq, ld_sx, rows;
    const uint8_t *w;
    const float *sw;  // [ceil(n / 128), ceil(k / 128)]
    int ldw, n, k;
    const void *bias;
    void *out;
    int dtype;  // of bias and out
};
int f8_product(const F8Product &a, cudaStream_t st);
// the same from rows that are not rounded yet, where f8_own says so (p.q, p.sx and p.ldq are not read)
bool f8_own(const F8Product &p);
int f8_product_own(const F8Product &a, const F8Rows &x, cudaStream_t st);
// blocks_fp8_pairs.cu: the same for many rows, and, of 128 rows of a gate and 128 of an up projection in turn, the gated rows rounded to e4m3 (to.q, to.scales)
struct F8PairsWidth {
    int outputs;  // of a tile
    float block;  // us of a block of a tile; of the widths' best: of a block of all tiles of a pair
};
F8PairsWidth f8_pairs_width(int rows, int n);
int f8_pairs(const F8Product &a, cudaStream_t st);
int f8_pairs_gated(const F8Product &a, const F8Rows &to, cudaStream_t st);
long long f8_gave_up();
long long f8_pairs_gave_up();

static inline int f8_up(int n, int to) { return (n + to - 1) / to * to; }

}  // namespace tlb
