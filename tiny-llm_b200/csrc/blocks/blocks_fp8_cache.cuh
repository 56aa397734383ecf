// Pages of keys and values in 8 bits (e4m3), one scale for each 16 tokens of a head.
#pragma once

#include "blocks_fp8.cuh"

namespace tlb {

constexpr int kF8Tokens = 16;   // that share a scale
constexpr int kF8Least = -100;  // the smallest scale is 2^-100

// 2^e for -126 <= e <= 127.
__device__ __forceinline__ float f8_power(int e) { return __int_as_float((e + 127) << 23); }

// The smallest e, at least kF8Least, with most <= 448 * 2^e (448 = 1.75 * 2^8), for a finite most >= 0.
__device__ __forceinline__ int f8_exponent(float most) {
    const uint32_t bits = __float_as_uint(most);
    const int e = static_cast<int>(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u);
    return max(e, kF8Least);  // numbers below 2^-126 have the exponent field 0, far below the least
}

// A head's rows of a page lie side by side: the first byte of slot `slot`, and the scale of the 16 that it is one of.
__host__ __device__ __forceinline__ size_t f8_row(const tlb_fp8_pages &p, int page, int head, int slot) {
    return ((static_cast<size_t>(page) * p.heads + head) * p.page_size + slot) * p.dim;
}
__host__ __device__ __forceinline__ size_t f8_scale_at(const tlb_fp8_pages &p, int page, int head, int slot) {
    return (static_cast<size_t>(page) * p.heads + head) * (p.page_size / kF8Tokens) + slot / kF8Tokens;
}

// 2^32 / d, rounded up: n / d is the upper half of n times it while n * d < 2^32; 0 where `most`, the largest n, is too large for that.
static inline unsigned f8_magic(unsigned long long most, unsigned d) { return d > 1 && most < (1ull << 32) / d ? static_cast<unsigned>((1ull << 32) / d) + 1 : 0; }
__device__ __forceinline__ int f8_div(int n, int d, unsigned magic) { return magic ? static_cast<int>(__umulhi(n, magic)) : n / d; }

// What every entry asks of the pages.
int f8_check_pages(const char *op, const tlb_fp8_pages *p);
// The host's copies of a step's lengths and block table, where they are given: see tlb_fp8_append.
int f8_check_step(const char *op, const tlb_fp8_pages &p, const int32_t *lens, const int32_t *table, int batch, int max_pages, int tokens);

}  // namespace tlb
