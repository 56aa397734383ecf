// What the kernels of attention over pages of 8 bits are given.
#pragma once

#include "blocks_fp8_cache.cuh"

namespace tlb {

struct F8Attend : tlb_fp8_attention_call {
    tlb_fp8_pages pages;
    void *workspace;
    int group, col_blocks;  // query heads of a key/value head; items of a head: its columns by eights or sixteens
    int slots;              // CTAs that the GPU holds at a time
    int page_blocks;        // blocks of 16 tokens in a page
    unsigned page_magic, group_magic, heads_magic, each_magic;  // for divisions by page_blocks, group, heads and the items of a request (at_div)
    bool wide_rows;         // query rows may be read 16 bytes at a time
    float scale_log2, scale_rest;  // scale * log2(e), and what its rounding to fp32 left
    F8Attend(const tlb_fp8_pages &p, const tlb_fp8_attention_call &c, void *ws)
        : tlb_fp8_attention_call(c), pages(p), workspace(ws), group(c.heads / p.heads), col_blocks(0), slots(0), page_blocks(1), page_magic(0), group_magic(0), heads_magic(0), each_magic(0), wide_rows(false) {
        const double log2 = c.scale * 1.4426950408889634;
        scale_log2 = static_cast<float>(log2), scale_rest = static_cast<float>(log2 - scale_log2);
    }
};

}  // namespace tlb
