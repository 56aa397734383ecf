// The lists of (token, choice) pairs grouped by expert, and the grouped products that read them.
#pragma once

#include <algorithm>

#include "blocks_common.cuh"

namespace tlb {

// The experts' launches follow one another closely: sort, gate|up, down and sum may each become resident while the one before is ending, and wait
// (griddep_wait, in every CTA, before anything of it is read or overwritten).  Only gate|up lets its successor in early, behind its own wait for the sort: a
// down product that says that it follows one (tlb_moe_down_next) reads the lists ahead of its wait and fills its ring with weights on every SM whose gate|up
// CTA is done, and waits for the rows alone.  Any other waits before it reads the lists, which may be the launch before's.  16 tokens, 6 of 64 experts of 1408 x 2048: 189 -> 178 us the call; 2048 tokens 472 -> 469.
template <typename... P, typename... A>
static inline cudaError_t moe_launch(void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t st, A &&...a) {
    return tl::launch_chained(kernel, grid, dim3(threads), smem, st, static_cast<P>(a)...);
}

// Which rows of its operand a tile's rows read: the sorted rows themselves (the second product), the token of the pair, or the pair.
constexpr int kGatherSorted = 0, kGatherToken = 1, kGatherPair = 2;
__device__ __forceinline__ int moe_src_row(int pair, int sorted_row, int top, int gather) {
    if (pair < 0) return -1;
    return gather == kGatherSorted ? sorted_row : gather == kGatherToken ? pair / top : pair;
}

// A warp makes one token's choice from its logits z [experts] (written over): idx and gate [top], lower index first where values are equal.  p_all [experts]:
// scoring 2, the softmax over all outputs; best [group_count]: the largest choice score of every group.
// Scores as whole numbers in registers and reductions of a warp at once, in place of exchanges of numbers and indexes out of shared memory (router's launch, bf16 rows of 2048: 64 outputs and 6 choices
// 7.2 -> 5.6 us, 128 and 33 20.6 -> 14.2; above 128 outputs, where the scores stay in shared memory, as before).
template <typename T>
__device__ __forceinline__ void moe_choose(float *z, float *p_all, float *best, int lane, int experts, int top, int scoring, const T *choice_bias, float weight_scale,
                                           int group_count, int group_keep, int32_t *idx, float *gate) {
    if (scoring == 2) {  // scores = softmax over ALL outputs; the choice adds a bias to them, the weights do not
        float m = -INFINITY, sum = 0.f;
        for (int e = lane; e < experts; e += 32) m = fmaxf(m, z[e]);
        m = warp_max(m);
        for (int e = lane; e < experts; e += 32) sum += expf(z[e] - m);
        sum = warp_sum(sum);
        for (int e = lane; e < experts; e += 32) {
            float p = expf(z[e] - m) / sum;
            p_all[e] = p;
            z[e] = p + (choice_bias ? to_f(choice_bias[e]) : 0.f);
        }
        __syncwarp();
    }
    if (group_keep > 0 && group_keep < group_count) {  // only the outputs of the best groups of neighbours can be chosen
        const int size = experts / group_count;
        for (int j = lane; j < group_count; j += 32) {
            float m = -INFINITY;
            for (int e = j * size; e < (j + 1) * size; ++e) m = fmaxf(m, z[e]);
            best[j] = m;
        }
        __syncwarp();
        for (int e = lane; e < experts; e += 32) {
            const int j = e / size;
            int ahead = 0;  // groups in front of this one (lower index wins a tie)
            for (int i = 0; i < group_count; ++i) ahead += best[i] > best[j] || (best[i] == best[j] && i < j);
            if (ahead >= group_keep) z[e] = -INFINITY;
        }
        __syncwarp();
    }
    // top-k by repeated arg-max over the warp (lower index wins a tie); weights = softmax over the chosen logits
    float first_v = 0.f, denom = 0.f;
    // A number's bits in an order that whole numbers have too; 0 for NaN, which is never chosen.  Minus zero counts as zero.
    auto ordered = [](float v) {
        const uint32_t u = __float_as_uint(v + 0.f);
        return v != v ? 0u : u & 0x80000000u ? ~u : u | 0x80000000u;
    };
    constexpr int KEPT = 4;  // outputs of a lane that stay in registers: up to 128 of them
    uint32_t kept[KEPT];
    const bool keep = experts <= 32 * KEPT;
#pragma unroll
    for (int i = 0; i < KEPT; ++i) kept[i] = keep && lane + 32 * i < experts ? ordered(z[lane + 32 * i]) : 0;
    auto number = [](uint32_t v) { return v ? __uint_as_float(v & 0x80000000u ? v & 0x7fffffffu : ~v) : -INFINITY; };
    if (keep && top <= 32) {  // lane k keeps choice k; the weights are made side by side, added in the choices' order
        uint32_t my_v = 0, first = 0;
        int my_i = 0x7fffffff;
        for (int k = 0; k < top; ++k) {
            uint32_t best_v = 0;
            int bi = 0x7fffffff;
#pragma unroll
            for (int i = 0; i < KEPT; ++i)
                if (kept[i] > best_v) best_v = kept[i], bi = lane + 32 * i;
            const uint32_t most = __reduce_max_sync(0xffffffffu, best_v);
            bi = __reduce_min_sync(0xffffffffu, best_v == most && most ? bi : 0x7fffffff);
#pragma unroll
            for (int i = 0; i < KEPT; ++i)
                if (bi == lane + 32 * i) kept[i] = ordered(-INFINITY);
            if (k == 0) first = most;
            if (lane == k) my_v = most, my_i = bi;
        }
        const float bv = number(my_v);
        const float p = scoring == 1 ? 1.0f / (1.0f + expf(-bv)) : scoring == 2 ? p_all[min(my_i, experts - 1)] : expf(bv - number(first));
        if (scoring != 1)
            for (int k = 0; k < top; ++k) denom += __shfl_sync(0xffffffffu, p, k);
        if (lane < top) idx[lane] = my_i, gate[lane] = scoring == 1 ? p : scoring == 2 ? p / (denom + 1e-20f) * weight_scale : p / denom;
        return;
    }
    for (int k = 0; k < top; ++k) {
        uint32_t best_v = 0;
        int bi = 0x7fffffff;
        if (keep) {
#pragma unroll
            for (int i = 0; i < KEPT; ++i)
                if (kept[i] > best_v) best_v = kept[i], bi = lane + 32 * i;
        } else {
            for (int e = lane; e < experts; e += 32) {
                const uint32_t v = ordered(z[e]);
                if (v > best_v) best_v = v, bi = e;
            }
        }
        const uint32_t most = __reduce_max_sync(0xffffffffu, best_v);
        bi = __reduce_min_sync(0xffffffffu, best_v == most && most ? bi : 0x7fffffff);
        const float bv = number(most);
#pragma unroll
        for (int i = 0; i < KEPT; ++i)
            if (bi == lane + 32 * i) kept[i] = ordered(-INFINITY);
        if (k == 0) first_v = bv;
        // scoring 0: softmax over the chosen logits (the first choice is the largest); 1: each choice's own sigmoid, as it is
        float p = scoring == 1 ? 1.0f / (1.0f + expf(-bv)) : scoring == 2 ? p_all[min(bi, experts - 1)] : expf(bv - first_v);
        denom += p;
        if (lane == 0) {
            idx[k] = bi;
            gate[k] = p;
            if (bi != 0x7fffffff) z[bi] = -INFINITY;
        }
        __syncwarp();
    }
    if (scoring == 1) return;
    // scoring 2: the chosen scores renormalised (a guard against an all-zero choice) and scaled
    for (int k = lane; k < top; k += 32)
        gate[k] = scoring == 2 ? gate[k] / (denom + 1e-20f) * weight_scale : gate[k] / denom;
}

// One int32 block of memory: counters [4] = {32-row tiles in use, rows in use, chunks in use, -}; chunks (expert, first row, rows,
// -), the tensor cores' work list; tile_expert, the expert of every 32-row tile; sorted_pair, the pair of every row or -1.
struct MoeLists {
    int32_t *counters;
    int4 *chunks;
    int32_t *tile_expert, *sorted_pair;
};

// The most rows of a chunk: one tensor-core tile's columns, fewer where no expert can get that many (a token names an expert once).  192: four
// stages of two weight blocks and the rows fit in shared memory (blocks_moe_tc.cu).
static inline int moe_chunk_rows(int tokens) { return std::min(192, (tokens + 15) / 16 * 16); }
// An expert's rows make one chunk, and one more for every moe_chunk_rows of them.
static inline long long moe_max_chunks(int tokens, int top, int experts) {
    const long long pairs = (long long)tokens * top;
    return pairs / moe_chunk_rows(tokens) + std::min<long long>(pairs, experts);
}
static inline MoeLists moe_lists(int32_t *p, int tokens, int top, int experts) {
    MoeLists l;
    l.counters = p;
    l.chunks = reinterpret_cast<int4 *>(p + 4);
    l.tile_expert = p + 4 + 4 * moe_max_chunks(tokens, top, experts);
    l.sorted_pair = l.tile_expert + tlb_moe_max_rows(tokens, top, experts) / 32;
    return l;
}

// One grouped product: w0 (and, gated, w1) [experts, N, K] times rows of x.  inter: activation applied, sorted rows; else pair_out.
struct MoeProduct {
    const void *x, *w0, *w1;
    MoeLists lists;
    int tokens, top, experts, K, N, act, gather;
    float limit, slope;
    void *inter;
    float *pair_out;
    bool second = false;  // the launch before is the first product of these lists, which let this one in only once they were whole
};

bool moe_tc_ok(int dtype, int K, const void *x, const void *w0, const void *w1);
int moe_tc_product(const MoeProduct &p, cudaStream_t st);

}  // namespace tlb
