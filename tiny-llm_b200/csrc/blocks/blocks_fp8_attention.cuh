// What the kernels of attention over pages of 8 bits are given.
#pragma once

#include "blocks_fp8_cache.cuh"

namespace tlb {

struct F8Attend : tlb_fp8_attention_call {
    tlb_fp8_pages pages;
    int group, col_blocks;
    float scale_log2, scale_rest;  // scale * log2(e), and what its rounding to fp32 left
    F8Attend(const tlb_fp8_pages &p, const tlb_fp8_attention_call &c) : tlb_fp8_attention_call(c), pages(p), group(c.heads / p.heads), col_blocks(0) {
        const double log2 = c.scale * 1.4426950408889634;
        scale_log2 = static_cast<float>(log2), scale_rest = static_cast<float>(log2 - scale_log2);
    }
};

}  // namespace tlb
