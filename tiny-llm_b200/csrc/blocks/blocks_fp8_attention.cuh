// What the kernels of attention over pages of 8 bits are given.
#pragma once

#include "blocks_fp8_cache.cuh"

namespace tlb {

constexpr int kAtLeast = 32;  // blocks of a piece at the least

struct F8Attend : tlb_fp8_attention_call {
    tlb_fp8_pages pages;
    void *workspace;
    int group, col_blocks;  // query heads of a key/value head; items of a head: its columns by eights or sixteens
    int slots;              // CTAs that the GPU holds at a time
    int most_pieces;        // of an item
    int ranks;              // CTAs of an item, a cluster; 1: no clusters
    int granule;            // pieces are a multiple of so many blocks
    int whole, least;       // blocks of a request that is not cut; of a piece at the least
    int page_blocks;        // blocks of 16 tokens in a page
    unsigned page_magic, group_magic, heads_magic, each_magic;  // for divisions by page_blocks, group, heads and the items of a request (f8_div)
    bool wide_rows;         // query rows may be read 16 bytes at a time
    bool long_first;        // requests (at most 32) are taken by their length, where no item is divided
    float scale_log2, scale_rest;  // scale * log2(e), and what its rounding to fp32 left
    F8Attend(const tlb_fp8_pages &p, const tlb_fp8_attention_call &c, void *ws)
        : tlb_fp8_attention_call(c), pages(p), workspace(ws), group(c.heads / p.heads), col_blocks(0), slots(0), most_pieces(1), ranks(1), granule(1), whole(0), least(kAtLeast), page_blocks(1), page_magic(0), group_magic(0), heads_magic(0), each_magic(0), wide_rows(false), long_first(false) {
        const double log2 = c.scale * 1.4426950408889634;
        scale_log2 = static_cast<float>(log2), scale_rest = static_cast<float>(log2 - scale_log2);
    }
};

constexpr float kAtLag = 15.f;  // log2: how far a running maximum may lag behind: weights up to 2^15 are f16 numbers

__device__ __forceinline__ float at_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void at_halves(uint32_t four, uint32_t &lo, uint32_t &hi) {  // four e4m3 numbers as f16
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}" : "=r"(lo), "=r"(hi) : "r"(four));
}
// Everything that the launches in front may have written - queries, pages and their scales, table, lengths, pieces - is read through L2 (tl::ld_cg, asynchronous copies): this
// launch becomes resident while they still run, and a line that its SM read meanwhile may be older than they are (eight blocks' scales share 32 bytes).
// 8 entries of a query
template <typename T>
__device__ __forceinline__ void at_query(const T *q, bool wide, float (&x)[8]) {
    if (!wide) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = to_f(tl::ld_cg(q + e));
    } else if constexpr (sizeof(T) == 2) {
        const uint4 v = tl::ld_cg(reinterpret_cast<const uint4 *>(q));
        const float2 y[4] = {tl::unpack2<bf16>(v.x), tl::unpack2<bf16>(v.y), tl::unpack2<bf16>(v.z), tl::unpack2<bf16>(v.w)};
#pragma unroll
        for (int e = 0; e < 4; ++e) x[2 * e] = y[e].x, x[2 * e + 1] = y[e].y;
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint4 v = tl::ld_cg(reinterpret_cast<const uint4 *>(q + 4 * i));
            x[4 * i] = __uint_as_float(v.x), x[4 * i + 1] = __uint_as_float(v.y), x[4 * i + 2] = __uint_as_float(v.z), x[4 * i + 3] = __uint_as_float(v.w);
        }
    }
}

__device__ __forceinline__ int at_context(const F8Attend &a, int b) {
    return static_cast<int>(max(0LL, min(static_cast<long long>(tl::ld_cg(a.lens + b)), static_cast<long long>(a.max_pages) * a.pages.page_size)));
}
__device__ __forceinline__ int at_blocks(int context) { return (context + kF8Tokens - 1) / kF8Tokens; }

// How long a piece of an item may be, in blocks: such that the pieces are about as many as the CTAs that the GPU holds at a time, or the items and half of those.  A piece
// costs its CTA some microseconds beside its blocks, so it has a.least of them.  Nothing here depends on how many idle slots there are: a step over more of
// them is cut the same way, to the bit.  Whole warps; `mine`: the blocks of request number lane; 0: nothing is cut.
typedef int AtCut;
__device__ __forceinline__ AtCut at_cut(const F8Attend &a, int mine) {
    int live = mine > 0, longest = mine;  // at most 2^26 blocks a request
    long long all = mine;
    for (int r = (threadIdx.x & 31) + 32; r < a.batch; r += 32) {
        const int n = at_blocks(at_context(a, r));
        all += n, live += n > 0, longest = max(longest, n);
    }
    live = __reduce_add_sync(0xffffffffu, live), longest = __reduce_max_sync(0xffffffffu, longest);
    all = (static_cast<long long>(__reduce_add_sync(0xffffffffu, static_cast<unsigned>(all >> 16))) << 16) + __reduce_add_sync(0xffffffffu, static_cast<unsigned>(all & 0xffff));
    const int each = a.pages.heads * a.col_blocks, room = max(a.slots - live * each, a.slots / 2);
    if (longest <= a.whole) return 0;
    const long long shares = all * each + room - 1;
    const int mean = shares <= 0x7fffffff ? static_cast<int>(shares) / room : static_cast<int>(min(shares / room, 0x3fffffffLL));  // (a division of 64 bits is long)
    return max(max(mean, (longest + a.most_pieces - 1) / a.most_pieces), a.least);
}
__device__ __forceinline__ int at_pieces(AtCut cut, int n) { return cut == 0 || n <= cut + cut / 4 ? 1 : (n + cut - 1) / cut; }  // a quarter more is no reason to cut

// The index-th piece: a request's items one after another, an item's pieces side by side.
struct AtPiece {
    int b, ctx, item, piece, pieces, size;  // size: blocks of a piece; b < 0: there are not so many
};
__device__ __forceinline__ AtPiece at_piece(const F8Attend &a, int index) {
    const int each = a.pages.heads * a.col_blocks, lane = threadIdx.x & 31;
    const int want = f8_div(index, each, a.each_magic);  // rounded down: an item's pieces over all items of a request are a multiple of them
    AtPiece x{-1, 0, 0, 0, 1, 0x3fffffff};
    if (a.long_first && !a.workspace) {
        const int ctx = lane < a.batch ? at_context(a, lane) : -1;
        int rank = 0;
#pragma unroll
        for (int r = 0; r < 32; ++r) {
            const int other = __shfl_sync(0xffffffffu, ctx, r);
            rank += other > ctx || (other == ctx && r < lane);
        }
        const unsigned mine = __ballot_sync(0xffffffffu, lane < a.batch && rank == want);
        if (mine) x.b = __ffs(mine) - 1, x.ctx = __shfl_sync(0xffffffffu, ctx, x.b);
        x.item = index - want * each;
        return x;
    }
    if (!a.workspace) {
        if (want < a.batch) x.b = want, x.ctx = at_context(a, want);
        x.item = index - want * each;
        return x;
    }
    int ctx = lane < a.batch ? at_context(a, lane) : 0, run = 0;  // lengths are read once where there are no more than lanes
    const AtCut cut = at_cut(a, at_blocks(ctx));
    for (int r0 = 0; r0 < a.batch; r0 += 32) {
        if (r0) ctx = r0 + lane < a.batch ? at_context(a, r0 + lane) : 0;
        const int mine = r0 + lane < a.batch ? at_pieces(cut, at_blocks(ctx)) : 0;
        int upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int below = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += below;
        }
        const unsigned past = __ballot_sync(0xffffffffu, want < run + upto);
        if (past) {
            const int src = __ffs(past) - 1;
            x.b = r0 + src, x.ctx = __shfl_sync(0xffffffffu, ctx, src), x.pieces = __shfl_sync(0xffffffffu, mine, src);
            x.item = index - (run + __shfl_sync(0xffffffffu, upto - mine, src)) * each;
            if (x.pieces > 1) {
                x.piece = x.item % x.pieces, x.item /= x.pieces;
                x.size = ((at_blocks(x.ctx) + x.pieces - 1) / x.pieces + a.granule - 1) / a.granule * a.granule;  // the last may come out empty
            }
            return x;
        }
        run += __shfl_sync(0xffffffffu, upto, 31);
    }
    return x;
}
// The pieces of a request's items, and those of the requests before it, of one item each.
__device__ __forceinline__ int at_pieces_of(const F8Attend &a, int request, int &before) {
    const int lane = threadIdx.x & 31;
    int ctx = lane < a.batch ? at_context(a, lane) : 0, n = 0, of = 0;
    const AtCut cut = at_cut(a, at_blocks(ctx));
    for (int r0 = 0; r0 <= request; r0 += 32) {
        if (r0) ctx = r0 + lane < a.batch ? at_context(a, r0 + lane) : 0;
        const int mine = at_pieces(cut, at_blocks(ctx));
        if (r0 + lane < request) n += mine;
        if (r0 + lane == request) of = mine;
    }
    before = __reduce_add_sync(0xffffffffu, n);
    return __shfl_sync(0xffffffffu, of, request & 31);
}

// How a call's work is divided: an item a CTA, an item a cluster (`ranks` CTAs), or pieces, which a second launch joins.
struct AtPlan {
    int ranks;
    size_t workspace;  // for pieces; 0: none
    double time;       // about how many microseconds it takes
    bool portion;      // by the kernel of blocks_fp8_portion.cu
    bool long_first = false;
};
struct AtLengths {
    long long longest, blocks, live;  // blocks of the longest request, of all; requests that are not idle
};
// blocks_fp8_attention.cu: adds up the pieces of the launch in front, items of `cols` columns each.
int f8_attend_join(const F8Attend &a, int cols, cudaStream_t st);
__host__ __device__ static inline size_t at_piece_floats(int cols, int dim) { return static_cast<size_t>(cols) * (dim + 2); }
// blocks_fp8_portion.cu: bf16 queries of many columns
constexpr int kPoRows = 256;  // columns of a CTA
bool f8_portion_takes(const tlb_fp8_pages &p, const tlb_fp8_attention_call &c);  // more than 32 columns: fewer are never sooner through there
constexpr int kPoWhole = 40, kPoLeast = 24;  // blocks of a request that is not cut, of a piece at the least
int f8_portion(F8Attend a, cudaStream_t st);
AtPlan f8_portion_plan(const tlb_fp8_pages &p, const tlb_fp8_attention_call &c, const AtLengths &n);

}  // namespace tlb
