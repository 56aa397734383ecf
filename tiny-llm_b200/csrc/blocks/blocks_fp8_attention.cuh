// What the kernels of attention over pages of 8 bits are given.
#pragma once

#include "blocks_fp8_cache.cuh"

namespace tlb {

struct F8Attend {
    tlb_fp8_pages pages;
    const void *q;  // strides in entries
    long long q_b, q_h, q_l;
    void *out;  // [batch, tokens, heads, dim]
    const int32_t *table, *lens;
    int batch, heads, group, tokens, max_pages, causal, col_blocks;
    float scale_log2, scale_rest;  // scale * log2(e), and what its rounding to fp32 left
};

}  // namespace tlb
