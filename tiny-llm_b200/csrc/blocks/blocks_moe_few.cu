// A whole mixture-of-experts layer for the few tokens of a decoding step, in two launches, over experts of bf16 numbers or of e4m3 numbers
// with one scale for each block of 128 x 128.
//
//   first launch:  logits = router . x, the choice, inner[pair] = act(gate_e x) * (up_e x)        pair = (token, choice)
//   second launch: y[t] = sum over choices  weight * (down_e inner[pair])  (+ identity experts, + shared expert)
//
// Bound by HBM where many experts are chosen: every matrix of a chosen expert is read once.  The products are tcgen05.mma with 128 matrix rows as the M side, fed by
// TMA in boxes of 128 bytes a row, and the tokens as 16 to 64 columns: a matrix costs no thread more than its copies and the sums' additions (mma.sync on
// fragments that threads unpack took 380 instructions for 2 KB).  What the columns hold:
//
//   bf16 experts:  x as it is; an inner row as three bf16 terms
//   e4m3 experts:  both operands of a product have 8 bits, so a number is several e4m3 terms, a column each, added when the sums are taken out: x, whose 8 bits
//                  two terms of 4 hold exactly (times a power of two for each token; of bits below 2^-21 of the token's largest magnitude, which its sums of fp32 hardly
//                  hold beside it, the second term has none), an inner row three or six (times a power of two for each block of 128; few_terms).  A block of 128 is added in the
//                  tensor cores, then times its scales in fp32.
//
// First launch: the CTAs of a cluster share the router's rows and exchange the logits through shared memory, and every CTA makes the same choices and the columns
// for itself, in the place the tokens were copied to.  A tile is 64 features of an expert, gate rows and up rows in one accumulator.  Second launch: an item is 128 output
// columns of an expert for up to five of its tokens, over a part of the reduction; its partial sums go to memory, and whoever writes a token's last one adds
// them all, in order (a counter tells; no CTA waits for another outside its cluster).
//
// 64 experts of 1408 x 2048, 6 a token: 1 token 29 us in e4m3 and 37 in bf16, of which some 8 and 16 are the weights' and the rest one latency behind another (tokens and
// router rows, choice, first tile, sums, inner rows, sums, outputs); 32 tokens 134 us in e4m3, 528 MB of weights: 3.9 TB/s over the whole call, about 6 within the
// two launches' tiles, some 17 us of prologue (all CTAs: 128 KB of tokens, their columns, 32 choices).  With tokens in fp16 on mma.sync and weights through a queue of
// cp.async it took 184.  Asking the second launch's first matrices into L2 behind the first's last cost a microsecond: the two are close enough.
#include <atomic>

#include "../per_device.h"
#include "blocks_fp8.cuh"
#include "blocks_moe.cuh"
#include "blocks_tc.cuh"

namespace tlb {

constexpr int kFewThreads = 512, kFewWarps = 16;
constexpr int kFewTokens = 32, kFewPairs = 512, kFewOutputs = 1024;
constexpr int kFewWidth = 1 << 16;     // far wider than what fits: bytes of wider rows would not be ints
constexpr int kFewStage = 128 * 128;  // a stage of the ring: 128 matrix rows of 128 bytes
constexpr int kFewMostStages = 8;
constexpr int kFewItemCols = 48 * 1024, kFewItemBlocks = kFewItemCols / 1024;  // second launch: bytes of an item's columns, the most blocks of its reduction

struct FewArgs {
    const bf16 *x, *router, *router_bias, *choice_bias, *side_w;
    int tokens, dim, outputs /* of the router */, experts, top, scoring, group_count, group_keep;
    float weight_scale;
    const float *s0, *s1, *s2;  // block scales: gate (up where there is no gate), up, down
    int ff, act;
    float limit, slope;
    const bf16 *shared;
    void *out;
    // between the launches
    int32_t *idx;        // [tokens, top]
    float *gate;         // [tokens, top]
    float *side;         // [tokens]
    uint32_t *finished;  // [blocks of 128 output columns][32 tokens]: partial sums that are written
    float *inner;        // [tokens * top, ld_inner], zero behind ff
    float *part;         // [splits][tokens * top, dim]
    int32_t *lost;       // [first_ctas]: whether a CTA of the first launch gave up a wait
    int ld_inner, splits, first_ctas, room /* bytes of shared memory that a launch may use */;
};

#ifdef TLB_FEW_STARVED  // a test's build: for one CTA of the first launch the tokens never come in whole
static __device__ int g_few_starved = -1;
__device__ __forceinline__ bool few_starved() { return static_cast<int>(blockIdx.x) == g_few_starved; }
#else
__device__ __forceinline__ constexpr bool few_starved() { return false; }
#endif

// ---- small things ----------------------------------------------------------------------------------------------------

__device__ __forceinline__ uint4 few_ldg(const uint8_t *p) {
    uint4 r;
    asm volatile("ld.global.nc.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
    return r;
}
// 16 rows of 32 entries, a lane 8 of row lane / 4 (a) and of the row 8 further on (b), times 8 columns: x, the lane's 8 entries of column lane / 4.  All operands
// in the order in which the lanes hold them, which is that of the reduction index for both.
__device__ __forceinline__ void few_mma(float (&d)[4], const uint4 &a, const uint4 &b, const uint4 &x) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a.x), "r"(b.x), "r"(a.y), "r"(b.y), "r"(x.x), "r"(x.y));
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a.z), "r"(b.z), "r"(a.w), "r"(b.w), "r"(x.z), "r"(x.w));
}
// 2^e with |v| 2^-e in [0.5, 1) for a normal v, within what fp32 holds both ways
__device__ __forceinline__ int few_exponent(float most) { return max(-100, static_cast<int>(__float_as_uint(most) >> 23) - 126); }
__device__ __forceinline__ float few_exp2(int e) { return __int_as_float((e + 127) << 23); }
// Four numbers v (at most 256) as e4m3, and what is left of them, times 16.
__device__ __forceinline__ uint32_t few_term(float (&v)[4]) {
    const uint32_t q = f8_pack4(v[0], v[1], v[2], v[3]);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(q >> 16 * i), __NV_E4M3);
        const float2 f = __half22float2(__half2(h));
        v[2 * i] = (v[2 * i] - f.x) * 16.f, v[2 * i + 1] = (v[2 * i + 1] - f.y) * 16.f;
    }
    return q;
}
__device__ __forceinline__ uint32_t few_most4(const float (&v)[4]) {  // magnitudes are in the order of their bits, an infinity above all numbers, a NaN above that
    return max(max(__float_as_uint(v[0]) & 0x7fffffffu, __float_as_uint(v[1]) & 0x7fffffffu), max(__float_as_uint(v[2]) & 0x7fffffffu, __float_as_uint(v[3]) & 0x7fffffffu));
}
// Where byte `at` of row r of an operand lies: rows of 128 bytes in groups of 8, 16-byte pieces exchanged by row (128-byte swizzle).
__device__ __forceinline__ uint32_t few_swizzled(int r, int at) { return r * 128 + (((at >> 4) ^ (r & 7)) << 4) + (at & 15); }
// Products of a stage, its accumulator kept or begun.  Ahead of them two barriers are asked whether their phase is over: a question costs the thread that asks
// some 200 cycles, which the products' own time hides.  `done` is arrived at if it is the accumulator's last stage, `used` in any case.
#define FEW_BLOCK(KIND)                                                                                                                                       \
    asm volatile(                                                                                                                                             \
        "{\n\t.reg .pred p, q, on, begun, last;\n\t.reg .b64 a1, a2, a3, b1, b2, b3;\n\t"                                                                     \
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%8], %9;\n\t"                                                                                          \
        "mbarrier.test_wait.parity.shared::cta.b64 q, [%10], %11;\n\t"                                                                                        \
        "setp.eq.u32 on, %2, %2;\n\tsetp.ne.u32 begun, %12, 0;\n\tsetp.ne.u32 last, %13, 0;\n\t"                                                             \
        "add.u64 a1, %3, 2;\n\tadd.u64 a2, %3, 4;\n\tadd.u64 a3, %3, 6;\n\tadd.u64 b1, %4, 2;\n\tadd.u64 b2, %4, 4;\n\tadd.u64 b3, %4, 6;\n\t"                  \
        "tcgen05.mma.cta_group::1.kind::" KIND " [%2], %3, %4, %5, begun;\n\t"                                                                                \
        "tcgen05.mma.cta_group::1.kind::" KIND " [%2], a1, b1, %5, on;\n\t"                                                                                   \
        "tcgen05.mma.cta_group::1.kind::" KIND " [%2], a2, b2, %5, on;\n\t"                                                                                   \
        "tcgen05.mma.cta_group::1.kind::" KIND " [%2], a3, b3, %5, on;\n\t"                                                                                   \
        "@last tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%6];\n\t"                                                               \
        "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%7];\n\t"                                                                     \
        "selp.u32 %0, 1, 0, p;\n\tselp.u32 %1, 1, 0, q;\n\t}"                                                                                                \
        : "=r"(over0), "=r"(over1)                                                                                                                            \
        : "r"(d), "l"(a), "l"(b), "r"(idesc), "r"(done), "r"(used), "r"(bar0), "r"(parity0), "r"(bar1), "r"(parity1), "r"(begun), "r"(last)                   \
        : "memory")
template <bool FP8>
__device__ __forceinline__ void few_block(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t begun, uint32_t last, uint32_t done, uint32_t used, uint32_t bar0,
                                          uint32_t parity0, uint32_t bar1, uint32_t parity1, uint32_t &over0, uint32_t &over1) {
    if constexpr (FP8) FEW_BLOCK("f8f6f4");
    else FEW_BLOCK("f16");
}
#undef FEW_BLOCK
template <bool FP8>
__device__ __forceinline__ uint32_t few_idesc(int n) {
    return FP8 ? (1u << 4) | (static_cast<uint32_t>(n >> 3) << 17) | (8u << 24) : tc_idesc(n);
}
template <int COLS>
__device__ __forceinline__ void few_ld(uint32_t at, uint32_t *v) {  // columns of tensor memory, behind them tcgen05.wait::ld
#pragma unroll
    for (int c = 0; c < COLS; c += 4)
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v[c]), "=r"(v[c + 1]), "=r"(v[c + 2]), "=r"(v[c + 3]) : "r"(at + c) : "memory");
}
__device__ __forceinline__ void few_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// The chosen experts in ascending order and the tokens that chose each, in ascending order: a token's place is its column.  Both launches make these for
// themselves.
struct FewLists {
    uint32_t *words;   // [32]: a bit for every expert, and behind them whether a token names one again; zero at the start
    uint32_t *tokens;  // [most]: the tokens of an active expert, zero at the start
    int *active;       // [most]
    uint16_t *column;  // [most][32]: token * 256 + choice
    int *count;
};
struct FewListsSmem {  // from `at` on, a multiple of 4
    int words, tokens, active, count, column, end;
    __host__ __device__ FewListsSmem(int at, int tokens_, int top, int experts) {
        const int most = tokens_ * top < experts ? tokens_ * top : experts;
        words = at, tokens = words + 132, active = tokens + most * 4, count = active + most * 4, column = count + 4, end = (column + most * 64 + 15) / 16 * 16;
    }
    __device__ FewLists lists(unsigned char *smem) const {
        return {reinterpret_cast<uint32_t *>(smem + words), reinterpret_cast<uint32_t *>(smem + tokens), reinterpret_cast<int *>(smem + active),
                reinterpret_cast<uint16_t *>(smem + column), reinterpret_cast<int *>(smem + count)};
    }
    __device__ void clear(unsigned char *smem) const {  // words and tokens lie side by side
        for (int i = threadIdx.x; i < (active - words) / 4; i += kFewThreads) reinterpret_cast<uint32_t *>(smem + words)[i] = 0;
    }
};
// All threads of the CTA, a pair each; behind a barrier after clear() and the last write of idx and gate, which are in shared memory.  Whether the pair has an
// expert's product.  A token that names an expert twice (scores of minus infinity are equal, and the first of them comes again) has it once, with the sum of its
// weights: the first launch, with CHOICES, joins them, and the later ones become -1.
template <bool CHOICES>
__device__ __forceinline__ bool few_lists(const FewArgs &a, const FewLists &l, int *idx, float *gate) {
    static_assert(kFewPairs <= kFewThreads, "a pair a thread");
    const int p = threadIdx.x, lane = p & 31, t = p / a.top, k = p % a.top;
    int e = p < a.tokens * a.top ? idx[p] : a.experts;
    bool again = false;
    if constexpr (CHOICES) {
        for (int j = 1; j <= k && e < a.experts; ++j)
            if (idx[p - j] == e) e = a.experts, again = true;
        if (again) l.words[32] = 1;
    }
    const bool live = static_cast<uint32_t>(e) < static_cast<uint32_t>(a.experts);
    if (live) atomicOr(&l.words[e >> 5], 1u << (e & 31));
    __syncthreads();
    const bool join = CHOICES && l.words[32] && live;
    float weight = 0.f;
    if (join) {
        weight = gate[p];
        for (int j = 1; k + j < a.top; ++j)
            if (idx[p + j] == e) weight += gate[p + j];
    }
    const uint32_t word = l.words[lane];
    int before = __popc(word);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += v;
    }
    if (p == 31) *l.count = before;
    before -= __popc(word);
    const int at = live ? e >> 5 : 0, first = __shfl_sync(0xffffffffu, before, at);
    const int pos = first + __popc(__shfl_sync(0xffffffffu, word, at) & ((1u << (e & 31)) - 1));
    if (live) l.active[pos] = e, atomicOr(&l.tokens[pos], 1u << t);
    __syncthreads();
    if (join) gate[p] = weight;  // read by all before the barrier
    if (again) idx[p] = -1;
    if (live) l.column[pos * 32 + __popc(l.tokens[pos] & ((1u << t) - 1))] = (uint16_t)(t * 256 + k);
    __syncthreads();
    return live;
}

// Barriers of either launch: the ring's, the accumulators', the second launch's columns'.
struct FewBars {
    uint32_t full, empty, acc_full, acc_empty, cols_full, cols_empty, part_full, part_empty;
    volatile int *dead;
    uint32_t *tmem;
    static constexpr int kBytes = 16 * kFewMostStages + 64 + 64 + 16;
    __device__ FewBars(unsigned char *smem, int at) {
        full = g_smem_u32(smem + at), empty = full + 8 * kFewMostStages, acc_full = empty + 8 * kFewMostStages, acc_empty = acc_full + 32, cols_full = acc_empty + 32;
        cols_empty = cols_full + 16, part_full = cols_empty + 16, part_empty = part_full + 16;
        dead = reinterpret_cast<volatile int *>(smem + at + 16 * kFewMostStages + 128);
        tmem = reinterpret_cast<uint32_t *>(smem + at + 16 * kFewMostStages + 132);
    }
};
constexpr int kFewBuffers = 4;  // accumulators, of bf16 experts 2 are used

// ---- first launch ----------------------------------------------------------------------------------------------------

constexpr int kFewCluster = 4;  // of 2 (all 148 SMs) 1 token took 30.5 us for 29.1, 32 tokens the same
// Columns of the products, for eight tokens each; e4m3: the first terms of all tokens, then the second.
__host__ __device__ constexpr int few_columns(int nt, bool fp8) { return fp8 ? 16 * nt : nt <= 2 ? 16 : 32; }
__host__ __device__ constexpr int few_router_sums(int nt) { return 16 * (nt * 8 + 2); }  // of a warp: 16 rows
constexpr int few_tmem(int columns) { return columns <= 32 ? 32 : columns <= 64 ? 64 : columns <= 128 ? 128 : 256; }

struct FewFirstSmem {
    int cols, cols_block, ring, stages, sums, router, logits, most, idx, gate, bars, total;
    FewListsSmem lists;
    __host__ __device__ FewFirstSmem(int tokens, int nt, int dim, int outputs, int experts, int top, int groups, bool fp8, int room) : lists(0, tokens, top, experts) {
        const int n = few_columns(nt, fp8);
        cols = 0;
        cols_block = nt * (fp8 ? 2048 : 1024);  // of 128 bytes of the reduction; bf16: what the columns past the last token hold does not matter
        sums = (fp8 ? (dim + 127) / 128 * cols_block : (dim + 63) / 64 * cols_block + n * 128);
        most = sums + (fp8 ? n / 2 : n) * 256;
        idx = most + kFewTokens * 4;
        gate = idx + tokens * top * 4;
        lists = FewListsSmem(gate + tokens * top * 4, tokens, top, experts);
        bars = lists.end;
        ring = (bars + FewBars::kBytes + 1023) / 1024 * 1024;
        // the router's sums and logits are done with when the ring's first copies are asked for
        router = ring;
        logits = router + kFewWarps * few_router_sums(nt) * 4;
        const int early = logits + (tokens * (2 * outputs + groups) + tokens) * 4;
        stages = (room - ring) / kFewStage;
        if (stages > kFewMostStages) stages = kFewMostStages;
        total = ring + stages * kFewStage;
        if (total < early) total = early;
    }
};

template <bool FP8, bool GATED, int NT>
__global__ void __launch_bounds__(kFewThreads, 1)
moe_few_first_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map0, const __grid_constant__ CUtensorMap map1, const FewArgs a) {
    extern __shared__ __align__(1024) unsigned char few_smem[];
    constexpr int BUFFERS = FP8 ? kFewBuffers : 2, ENTRIES = FP8 ? 128 : 64;  // of the reduction, in a stage
    constexpr int N = few_columns(NT, FP8), COLS = N / 2, SUMS = FP8 ? COLS / 2 : COLS /* of a thread */, TMEM = few_tmem(N * BUFFERS);
    const FewFirstSmem at(a.tokens, NT, a.dim, a.outputs, a.experts, a.top, a.group_count, FP8, a.room);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
    uint32_t rank, ranks;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
    // Another CTA's shared memory may be written once that CTA runs: arrived at here, waited for ahead of the first such store.
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    float *logits = reinterpret_cast<float *>(few_smem + at.logits), *router_red = reinterpret_cast<float *>(few_smem + at.router);
    const int per_token = 2 * a.outputs + a.group_count;
    float *side = logits + a.tokens * per_token, *gate = reinterpret_cast<float *>(few_smem + at.gate);
    uint32_t *most = reinterpret_cast<uint32_t *>(few_smem + at.most);
    int *idx = reinterpret_cast<int *>(few_smem + at.idx);
    const FewLists lists = at.lists.lists(few_smem);
    const FewBars bars(few_smem, at.bars);
    at.lists.clear(few_smem);
    if (warp == 1 && lane == 0) {
        for (int i = 0; i < at.stages; ++i) g_mbar_init(bars.full + 8 * i, GATED ? 2 : 1), g_mbar_init(bars.empty + 8 * i, 1);
        for (int i = 0; i < BUFFERS; ++i) g_mbar_init(bars.acc_full + 8 * i, 1), g_mbar_init(bars.acc_empty + 8 * i, 8);
        g_mbar_init(bars.cols_full, 1);
        *bars.dead = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_x) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map0) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map1) : "memory");
    }
    if (warp == 2) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(g_smem_u32(bars.tmem)), "n"(TMEM) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    g_tc_fence_before();
    __syncthreads();
    g_tc_fence_after();
    const uint32_t tmem = *bars.tmem;

    tl::griddep_wait();
    tl::griddep_launch();  // the second launch reads nothing ahead of its own wait
    // ---- the tokens, 64 entries of all of them a copy: bf16 columns as they are
    const int rows = a.outputs + (a.side_w ? 1 : 0), pieces = (a.dim + 63) / 64;
    // 16 of the router's rows are shared by all warps, or by eight where there are more than the cluster has at once
    const int parts = rows > 16 * static_cast<int>(ranks) ? 8 : 16, part = warp & (parts - 1), group = parts == 8 ? warp >> 3 : 0, groups = kFewWarps / parts;
    if (warp == 1 && g_elect_one()) {
        g_mbar_expect_tx(bars.cols_full, pieces * NT * 1024 + (few_starved() ? 16 : 0));
        for (int i = 0; i < pieces; ++i) tl::g_tma_load_2d(g_smem_u32(few_smem + at.cols) + i * NT * 1024, &map_x, i * 128, 0, bars.cols_full);
    }
    __syncwarp();
    if (tid == 0) a.lost[blockIdx.x] = 0;
    if (blockIdx.x == 0)
        for (int i = tid; i < (a.dim + 127) / 128 * kFewTokens; i += kFewThreads) a.finished[i] = 0;
    // ---- the router's rows, 16 for eight or all warps, which share the reduction
    constexpr int AT_ONCE = 4;
    uint4 wa[AT_ONCE][2], wb[AT_ONCE][2];
    auto row_of = [&](int r) { return reinterpret_cast<const uint8_t *>(r < a.outputs ? a.router + (size_t)r * a.dim : r < rows ? a.side_w : nullptr); };
    auto ask = [&](int m, int s0) {
        const uint8_t *ra = row_of(m * 16 + g), *rb = row_of(m * 16 + g + 8);
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int o = (s0 + u * parts) * 128 + c * 64 + t4 * 16;
                wa[u][c] = ra && o < a.dim * 2 ? few_ldg(ra + o) : make_uint4(0, 0, 0, 0);
                wb[u][c] = rb && o < a.dim * 2 ? few_ldg(rb + o) : make_uint4(0, 0, 0, 0);
            }
    };
    const int m_first = rank * groups + group;
    ask(m_first, part);
    tc_wait(bars.cols_full, 0, bars.dead, few_starved() ? 1000 : 1u << 22);  // given up: see the end of this kernel
    const unsigned char *raw = few_smem + at.cols;
    auto entries = [&](int b, int t) {  // four of a token, of 128 that a warp has
        return *reinterpret_cast<const uint2 *>(raw + (b * 2 + (lane >> 4)) * NT * 1024 + few_swizzled(t, (lane & 15) * 8));
    };
    if constexpr (FP8)  // the tokens' largest magnitudes
        for (int t = warp; t < 8 * NT; t += kFewWarps) {  // zeros behind the last
            uint32_t top = 0;
            for (int i = lane >> 3; i < pieces; i += 4) {
                const uint4 v = *reinterpret_cast<const uint4 *>(raw + i * NT * 1024 + t * 128 + (lane & 7) * 16);
                top = __vmaxu2(top, __vmaxu2(__vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu), __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu)));
            }
            top = __reduce_max_sync(0xffffffffu, max(top & 0xffffu, top >> 16));
            if (lane == 0) most[t] = top;
        }
    bool waited = false;
    for (int m = m_first; (m - group) * 16 < rows; m += ranks * groups) {
        float acc[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
        for (int s = part; s < pieces; s += AT_ONCE * parts) {
            if (m != m_first || s != part) ask(m, s);
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u) {
                if (s + u * parts >= pieces) break;
                uint4 x[2][NT];
#pragma unroll
                for (int c = 0; c < 2; ++c)
#pragma unroll
                    for (int n = 0; n < NT; ++n) x[c][n] = *reinterpret_cast<const uint4 *>(raw + (s + u * parts) * NT * 1024 + few_swizzled(n * 8 + g, c * 64 + t4 * 16));
#pragma unroll
                for (int c = 0; c < 2; ++c)
#pragma unroll
                    for (int n = 0; n < NT; ++n) few_mma(acc[n], wa[u][c], wb[u][c], x[c][n]);
            }
        }
        constexpr int RED = few_router_sums(NT) / 16;
        float *mine = router_red + warp * 16 * RED;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            *reinterpret_cast<float2 *>(mine + g * RED + n * 8 + 2 * t4) = make_float2(acc[n][0], acc[n][1]);
            *reinterpret_cast<float2 *>(mine + (g + 8) * RED + n * 8 + 2 * t4) = make_float2(acc[n][2], acc[n][3]);
        }
        __syncthreads();
        if (!waited) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // all CTAs of the cluster run
        waited = true;
        const int m0 = m - group;
        for (int i = tid; i < groups * 16 * NT * 8; i += kFewThreads) {
            const int in = i % (16 * NT * 8), r = (m0 + i / (16 * NT * 8)) * 16 + in / (NT * 8), t = in % (NT * 8);
            if (r >= rows || t >= a.tokens) continue;
            float z = 0.f;
#pragma unroll 8
            for (int w = 0; w < parts; ++w) z += router_red[((i / (16 * NT * 8) * parts + w) * 16 + in / (NT * 8)) * RED + t];
            if (r < a.outputs && a.router_bias) z += to_f(a.router_bias[r]);
            const uint32_t to = static_cast<uint32_t>(__cvta_generic_to_shared(r < a.outputs ? logits + t * per_token + r : side + t));
            for (uint32_t c = 0; c < ranks; ++c)
                asm volatile("{\n\t.reg .b32 ra;\n\tmapa.shared::cluster.u32 ra, %0, %1;\n\tst.shared::cluster.f32 [ra], %2;\n\t}" ::"r"(to), "r"(c), "f"(z) : "memory");
        }
        __syncthreads();
    }
    if (!waited) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    // ---- the columns of e4m3 experts, in the place of the tokens: a warp takes 128 entries of all of them
    if constexpr (FP8) {
        __syncthreads();  // the largest magnitudes; the router has read the tokens
        for (int b = warp; b * 2 < pieces; b += kFewWarps) {
            const bool there = b * 2 + (lane >> 4) < pieces;
            unsigned char *to = few_smem + at.cols + b * at.cols_block;
            for (int t0 = 0; t0 < a.tokens; t0 += 4) {  // a token's two terms stand where its 128 entries stood
                uint2 v[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    v[u] = make_uint2(0, 0);
                    if (there) v[u] = entries(b, t0 + u);
                }
                __syncwarp();
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    // at most 256 in magnitude; a half holds eight bits of what counts
                    const float up = few_exp2(8 - few_exponent(__uint_as_float(most[t0 + u] << 16)));
                    const float2 lo = tl::unpack2<bf16>(v[u].x), hi = tl::unpack2<bf16>(v[u].y);
                    const __half2 h0 = __floats2half2_rn(lo.x * up, lo.y * up), h1 = __floats2half2_rn(hi.x * up, hi.y * up);
                    const uint32_t q0 = __nv_cvt_halfraw2_to_fp8x2(h0, __NV_SATFINITE, __NV_E4M3), q1 = __nv_cvt_halfraw2_to_fp8x2(h1, __NV_SATFINITE, __NV_E4M3);
                    const __half2 sixteen = __float2half2_rn(16.f);
                    const __half2 r0 = __hmul2(__hsub2(h0, __half2(__nv_cvt_fp8x2_to_halfraw2(q0, __NV_E4M3))), sixteen);
                    const __half2 r1 = __hmul2(__hsub2(h1, __half2(__nv_cvt_fp8x2_to_halfraw2(q1, __NV_E4M3))), sixteen);
                    *reinterpret_cast<uint32_t *>(to + few_swizzled(t0 + u, lane * 4)) = q0 | q1 << 16;
                    *reinterpret_cast<uint32_t *>(to + few_swizzled(8 * NT + t0 + u, lane * 4)) =
                        __nv_cvt_halfraw2_to_fp8x2(r0, __NV_SATFINITE, __NV_E4M3) | static_cast<uint32_t>(__nv_cvt_halfraw2_to_fp8x2(r1, __NV_SATFINITE, __NV_E4M3)) << 16;
                }
            }
        }
        tl::g_fence_proxy_async();
    }
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");

    // ---- the choice, by every CTA for itself
    for (int t = warp; t < a.tokens; t += kFewWarps) {
        float *z = logits + t * per_token;
        moe_choose(z, z + a.outputs, z + 2 * a.outputs, lane, a.outputs, a.top, a.scoring, a.choice_bias, a.weight_scale, a.group_count, a.group_keep, idx + t * a.top,
                   gate + t * a.top);
    }
    __syncthreads();
    if (blockIdx.x == 0 && a.side_w && tid < a.tokens) a.side[tid] = sigmoid(side[tid]);
    tl::g_fence_proxy_async();  // the logits have been read, copies may come over them
    few_lists<true>(a, lists, idx, gate);
    if (blockIdx.x == 0 && tid < a.tokens * a.top) a.idx[tid] = idx[tid], a.gate[tid] = gate[tid];

    // ---- the first products: tiles of 64 features with their gates, or 128 without
    constexpr int FEATURES = GATED ? 64 : 128;
    const int count = *lists.count, tiles_of = (a.ff + FEATURES - 1) / FEATURES, tiles = count * tiles_of, blocks = (a.dim + ENTRIES - 1) / ENTRIES;
    const int scale_cols = (a.dim + 127) / 128, scale_rows = (a.ff + 127) / 128;
    if (warp == 0 || (GATED && warp == 3)) {
        if (g_elect_one()) {
            int s = 0;
            uint32_t ph = 1;
            bool ok = true;
            for (int tile = blockIdx.x; ok && tile < tiles; tile += gridDim.x) {
                const int e = lists.active[tile / tiles_of], f0 = tile % tiles_of * FEATURES;
                for (int b = 0; b < blocks; ++b) {
                    if (!(ok = tc_wait_one(bars.empty + 8 * s, ph, bars.dead))) break;
                    g_mbar_expect_tx(bars.full + 8 * s, GATED ? kFewStage / 2 : kFewStage);
                    tl::g_tma_load_3d(g_smem_u32(few_smem + at.ring) + s * kFewStage + (warp == 3 ? kFewStage / 2 : 0), warp == 3 ? &map1 : &map0, b * 128, f0, e,
                            bars.full + 8 * s);
                    if (++s == at.stages) s = 0, ph ^= 1u;
                }
            }
        }
    } else if (warp == 1) {
        if (g_elect_one()) {
            int s = 0, buf = 0;
            uint32_t ph = 0, acc_ph = 1;
            bool ok = true;
            const uint32_t ring = g_smem_u32(few_smem + at.ring), cols = g_smem_u32(few_smem + at.cols);
            uint32_t acc_free = 0, there = 0;  // asked ahead
            for (int tile = blockIdx.x; ok && tile < tiles; tile += gridDim.x)
                for (int b = 0; b < blocks; ++b) {
                    if ((FP8 || b == 0) && !acc_free) ok = tc_wait_one(bars.acc_empty + 8 * buf, acc_ph, bars.dead);
                    if (ok && !there) ok = tc_wait_one(bars.full + 8 * s, ph, bars.dead);
                    if (!ok) break;
                    g_tc_fence_after();
                    const uint64_t w = g_smem_desc_sw128(ring + s * kFewStage, 0, 1024), x = g_smem_desc_sw128(cols + b * at.cols_block, 0, 1024);
                    const uint32_t d = tmem + buf * N, done = bars.acc_full + 8 * buf, used = bars.empty + 8 * s;
                    const bool last = FP8 || b == blocks - 1;
                    if (++s == at.stages) s = 0, ph ^= 1u;
                    if (last && ++buf == BUFFERS) buf = 0, acc_ph ^= 1u;
                    few_block<FP8>(d, w, x, few_idesc<FP8>(N), !FP8 && b > 0, last, done, used, bars.acc_empty + 8 * buf, acc_ph, bars.full + 8 * s, ph, acc_free, there);
                }
        }
    } else if (warp >= 8) {
        const int quarter = warp & 3, half = (warp - 8) >> 2, me = tid - 256;
        float *sums = reinterpret_cast<float *>(few_smem + at.sums);  // [token][64]
        int buf = 0;
        uint32_t acc_ph = 0;
        for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
            const int pos = tile / tiles_of, e = lists.active[pos], f0 = tile % tiles_of * FEATURES;
            float acc[SUMS];
#pragma unroll
            for (int c = 0; c < SUMS; ++c) acc[c] = 0.f;
            bool ok = true;
            const uint32_t from = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + half * SUMS;
            if constexpr (FP8) {
                // the rows' block of scales: a gate's (or, without gates, all), the up projection's
                const float *scales = (GATED && quarter >= 2 ? a.s1 : a.s0) + ((size_t)e * scale_rows + (f0 >> 7)) * scale_cols;
                float next = __ldg(scales);
                for (int b = 0; b < blocks; ++b) {
                    const float scale = next;
                    if (b + 1 < blocks) next = __ldg(scales + b + 1);
                    ok &= tc_wait(bars.acc_full + 8 * buf, acc_ph, bars.dead);
                    g_tc_fence_after();
                    uint32_t v[COLS];
                    few_ld<SUMS>(from + buf * N, v), few_ld<SUMS>(from + buf * N + N / 2, v + SUMS);
                    few_ld_wait();
                    g_tc_fence_before();
                    __syncwarp();
                    if (lane == 0) g_mbar_arrive(bars.acc_empty + 8 * buf);
#pragma unroll
                    for (int c = 0; c < SUMS; ++c) acc[c] = fmaf(fmaf(__uint_as_float(v[c + SUMS]), 0.0625f, __uint_as_float(v[c])), scale, acc[c]);
                    if (++buf == BUFFERS) buf = 0, acc_ph ^= 1u;
                }
            } else {
                ok &= tc_wait(bars.acc_full + 8 * buf, acc_ph, bars.dead);
                g_tc_fence_after();
                uint32_t v[COLS];
                few_ld<COLS>(from + buf * N, v);
                few_ld_wait();
                g_tc_fence_before();
                __syncwarp();
                if (lane == 0) g_mbar_arrive(bars.acc_empty + 8 * buf);
#pragma unroll
                for (int c = 0; c < SUMS; ++c) acc[c] = __uint_as_float(v[c]);
                if (++buf == BUFFERS) buf = 0, acc_ph ^= 1u;
            }
            const float bad = tc_verdict(ok, bars.dead);
            // two passes of half of the features each: what they hand over takes half of the memory
            const int columns = __popc(lists.tokens[pos]), here = min(FEATURES, a.ff - f0);
            for (int pass = 0; pass < 2; ++pass) {
                const bool mine = GATED ? (quarter & 1) == pass : (quarter >> 1) == pass;
                if (mine) {
                    const int at_row = GATED ? (quarter >> 1) * 32 + lane : (quarter & 1) * 32 + lane;
#pragma unroll
                    for (int c = 0; c < SUMS; ++c) sums[(half * SUMS + c) * 64 + at_row] = acc[c];
                }
                asm volatile("bar.sync 1, 256;" ::: "memory");
                for (int i = me; i < columns * (FEATURES / 2); i += 256) {
                    const int in = i % (FEATURES / 2), f = pass * (FEATURES / 2) + in, c = lists.column[pos * 32 + i / (FEATURES / 2)], t = c >> 8;
                    if (f >= here) continue;
                    auto of = [&](int r) {
                        if constexpr (!FP8) return sums[t * 64 + r];
                        // a token with an infinity or a NaN has none of its numbers
                        const uint32_t m = most[t] << 16;
                        const float scale = m < 0x7f800000u ? few_exp2(few_exponent(__uint_as_float(m)) - 8) : __int_as_float(0x7fffffff);
                        return sums[t * 64 + r] * scale;
                    };
                    const float v = of(in);
                    float y;
                    if constexpr (GATED) y = gated_pair(v, of(in + 32), a.act, a.limit, a.slope);
                    else y = a.act == 2 ? (v > 0.f ? v * v : v == v ? 0.f : v) : act_apply(v, a.act);
                    float *to = a.inner + ((size_t)t * a.top + (c & 255)) * a.ld_inner + f0;
                    to[f] = y * bad;
                    if (f0 + here == a.ff && f >= here - 16)  // zeros behind the last features
                        for (int z = a.ff + here - 1 - f; z < a.ld_inner; z += min(here, 16)) to[z - f0] = 0.f;
                }
                asm volatile("bar.sync 1, 256;" ::: "memory");  // read before the next are written
            }
        }
    }
    __syncwarp();
    g_tc_fence_before();
    __syncthreads();
    // A CTA without its tokens has given its cluster logits that are none, and the cluster took other experts than the rest of the grid: rows of `inner` that nobody
    // writes, or two write.  No mark of the numbers themselves reaches these, so the second launch makes no output of a layer of which a wait was given up.
    if (tid == 0 && *bars.dead) a.lost[blockIdx.x] = 1;
    if (warp == 2) {
        tc_settle(bars.dead);
        g_tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(TMEM) : "memory");
    }
}

// ---- second launch ---------------------------------------------------------------------------------------------------

constexpr int kFewSecondN = 32;  // the most columns of an item: terms times tokens

// Terms of an inner number, and the tokens of an item.  Three terms of bf16 hold all bits of an fp32 number, and so do six of e4m3, four bits each (off by 2^-24, or by 2^-37
// of the largest of its block of 128).  Over 8 bits an output that is rounded to bf16, off by 2^-8, hides what three leave out of the numbers it adds up (2^-12, 2^-25) and has
// these: 1 token 28.7 us for 29.7, 32 tokens 135 for 143.  Five tokens of three terms are 16 columns, which fit beside the ring for a whole reduction and are half as
// many to take out as 32: with ten tokens an item, 16 tokens over 16 bits took 168 us for 155, 32 took 220 for 199; the few experts with more tokens come out of L2 again.
__host__ __device__ constexpr int few_terms(bool fp8, bool wide) { return fp8 && wide ? 6 : 3; }
constexpr int kFewGroup = 5;
static_assert(kFewGroup * few_terms(true, true) <= kFewSecondN && (kFewTokens + kFewGroup - 1) / kFewGroup <= 8, "an item's columns; groups of an expert, in three bits");

struct FewSecondSmem {
    int cols, factors, sums, idx, gate, need, group, bars, ring, stages, total;
    static constexpr int kCols = kFewItemCols + 4096, kFactors = kFewItemBlocks * kFewSecondN * 4;  // of either place of an item's columns
    FewListsSmem lists;
    __host__ __device__ FewSecondSmem(int tokens, int experts, int top, int room) : lists(0, tokens, top, experts) {
        cols = 0;
        factors = cols + 2 * kCols;
        sums = factors + 2 * kFactors;
        idx = sums + kFewSecondN * 128 * 4;
        gate = idx + tokens * top * 4;
        need = gate + tokens * top * 4;
        group = need + kFewTokens * 4;
        lists = FewListsSmem((group + tokens * top * 4 + 4 + 3) / 4 * 4, tokens, top, experts);
        bars = lists.end;
        ring = (bars + FewBars::kBytes + 1023) / 1024 * 1024;
        stages = (room - ring) / kFewStage;
        if (stages > kFewMostStages) stages = kFewMostStages;
        total = ring + stages * kFewStage;
    }
};

// Four columns of a token's output (a row has a multiple of eight).  A few choices' numbers are asked for together: one at a time, each waits for memory while
// the weights stream.
template <typename OUT>
__device__ __forceinline__ void few_output(const FewArgs &a, int t, int d, int pairs, const int *idx, const float *gate) {
    if (d >= a.dim) return;
    float y[4] = {0.f, 0.f, 0.f, 0.f};
    constexpr int AT_ONCE = 4;
    for (int k0 = t * a.top; k0 < (t + 1) * a.top; k0 += AT_ONCE) {
        float4 z[AT_ONCE];
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) z[u] = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int s = 0; s < a.splits; ++s) {
            uint4 w[AT_ONCE];
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u) {
                w[u] = make_uint4(0, 0, 0, 0);
                if (k0 + u < (t + 1) * a.top && static_cast<uint32_t>(idx[k0 + u]) < static_cast<uint32_t>(a.experts))
                    w[u] = tl::ld_cg(reinterpret_cast<const uint4 *>(a.part + ((size_t)s * pairs + k0 + u) * a.dim + d));
            }
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u) z[u].x += __uint_as_float(w[u].x), z[u].y += __uint_as_float(w[u].y), z[u].z += __uint_as_float(w[u].z), z[u].w += __uint_as_float(w[u].w);
        }
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) {
            const float g = k0 + u < (t + 1) * a.top && static_cast<uint32_t>(idx[k0 + u]) < static_cast<uint32_t>(a.experts) ? gate[k0 + u] : 0.f;
            y[0] = fmaf(g, z[u].x, y[0]), y[1] = fmaf(g, z[u].y, y[1]), y[2] = fmaf(g, z[u].z, y[2]), y[3] = fmaf(g, z[u].w, y[3]);
        }
    }
    if (a.experts < a.outputs) {
        float x[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) x[c] = to_f(tl::ld_cg(a.x + (size_t)t * a.dim + d + c));
        for (int k = t * a.top; k < (t + 1) * a.top; ++k)
            if (idx[k] >= a.experts && idx[k] < a.outputs)
#pragma unroll
                for (int c = 0; c < 4; ++c) y[c] = fmaf(gate[k], x[c], y[c]);
    }
    if (a.shared) {  // all four on their way before the first is used
        float shared[4], side = 1.f;
#pragma unroll
        for (int c = 0; c < 4; ++c) shared[c] = to_f(tl::ld_cg(a.shared + (size_t)t * a.dim + d + c));
        if (a.side_w) side = tl::ld_cg(a.side + t);
#pragma unroll
        for (int c = 0; c < 4; ++c) y[c] = fmaf(side, shared[c], y[c]);
    }
    for (int k = t * a.top; k < (t + 1) * a.top; ++k)  // a choice that is no output at all: the token's logits are no numbers
        if (idx[k] >= a.outputs) y[0] = y[1] = y[2] = y[3] = __int_as_float(0x7fffffff);
#pragma unroll
    for (int c = 0; c < 4; ++c) static_cast<OUT *>(a.out)[(size_t)t * a.dim + d + c] = from_f<OUT>(y[c]);
}

template <bool FP8, typename OUT>
__global__ void __launch_bounds__(kFewThreads, 1)
moe_few_second_kernel(const __grid_constant__ CUtensorMap map, const FewArgs a) {
    extern __shared__ __align__(1024) unsigned char few_smem[];
    constexpr int TERMS = few_terms(FP8, sizeof(OUT) == 4), GROUP = kFewGroup, BUFFERS = FP8 ? kFewBuffers : 2, TMEM = kFewSecondN * BUFFERS, ENTRIES = FP8 ? 128 : 64;
    const FewSecondSmem at(a.tokens, a.experts, a.top, a.room);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, pairs = a.tokens * a.top;
    float *sums = reinterpret_cast<float *>(few_smem + at.sums), *gate = reinterpret_cast<float *>(few_smem + at.gate), *factors = reinterpret_cast<float *>(few_smem + at.factors);
    int *need = reinterpret_cast<int *>(few_smem + at.need);  // [tokens]: the partial sums of an output
    int *idx = reinterpret_cast<int *>(few_smem + at.idx), *group = reinterpret_cast<int *>(few_smem + at.group);  // group: [groups] position * 8 + number
    const FewLists lists = at.lists.lists(few_smem);
    const FewBars bars(few_smem, at.bars);
    at.lists.clear(few_smem);
    if (warp == 1 && lane == 0) {
        for (int i = 0; i < at.stages; ++i) g_mbar_init(bars.full + 8 * i, 1), g_mbar_init(bars.empty + 8 * i, 1);
        for (int i = 0; i < BUFFERS; ++i) g_mbar_init(bars.acc_full + 8 * i, 1), g_mbar_init(bars.acc_empty + 8 * i, 8);
        for (int i = 0; i < 2; ++i) g_mbar_init(bars.cols_full + 8 * i, 4), g_mbar_init(bars.cols_empty + 8 * i, 1 + 8);  // by the warps that write; by the products, and the sums
        for (int i = 0; i < 2; ++i) g_mbar_init(bars.part_full + 8 * i, 1), g_mbar_init(bars.part_empty + 8 * i, 2);
        *bars.dead = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map) : "memory");
    }
    if (warp == 2) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(g_smem_u32(bars.tmem)), "n"(TMEM) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tl::griddep_wait();
    tl::griddep_launch();
    const int mark = tid < a.first_ctas ? tl::ld_cg(a.lost + tid) : 0;  // asked for ahead of the choices: one behind the other cost a microsecond
    if (tid < pairs) {
        const int e = tl::ld_cg(a.idx + tid);
        const float weight = tl::ld_cg(a.gate + tid);
        idx[tid] = e, gate[tid] = weight;
    }
    if (tid < kFewTokens) need[tid] = 0;
    g_tc_fence_before();
    const bool lost = __syncthreads_or(mark);
    g_tc_fence_after();
    const uint32_t tmem = *bars.tmem;
    if (lost)
        for (int i = blockIdx.x * kFewThreads + tid; i < a.tokens * a.dim; i += gridDim.x * kFewThreads) static_cast<OUT *>(a.out)[i] = from_f<OUT>(__int_as_float(0x7fffffff));
    if (few_lists<false>(a, lists, idx, gate)) atomicAdd(&need[tid / a.top], a.splits);
    const int count = *lists.count;
    if (warp == 0) {  // the experts' groups of up to GROUP tokens, in order
        int n = 0;
        for (int p0 = 0; p0 < count; p0 += 32) {
            const int mine = p0 + lane < count ? (__popc(lists.tokens[p0 + lane]) + GROUP - 1) / GROUP : 0;
            int before = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, before, o);
                if (lane >= o) before += v;
            }
            for (int j = 0; j < mine; ++j) group[n + before - mine + j] = (p0 + lane) * 8 + j;
            n += __shfl_sync(0xffffffffu, before, 31);
        }
        if (lane == 0) group[pairs] = n;
    }
    __syncthreads();
    const int groups = group[pairs], outs = (a.dim + 127) / 128, of_group = outs * a.splits, items = lost ? 0 : groups * of_group, blocks = (a.ff + ENTRIES - 1) / ENTRIES;
    const int scale_cols = (a.ff + 127) / 128, scale_rows = (a.dim + 127) / 128;
    struct Item {
        int pos, first, tokens, n, m, split, b0, b1;  // n: columns of the products; b0, b1: blocks of the reduction
    };
    auto item_of = [&](int i) {
        Item it;
        const int entry = group[i / of_group], r = i % of_group;
        it.pos = entry >> 3, it.first = (entry & 7) * GROUP, it.tokens = min(GROUP, __popc(lists.tokens[it.pos]) - it.first), it.n = (it.tokens * TERMS + 15) & ~15;
        it.m = r / a.splits, it.split = r % a.splits;
        it.b0 = blocks * it.split / a.splits, it.b1 = blocks * (it.split + 1) / a.splits;
        return it;
    };
    if (warp == 0) {
        if (g_elect_one()) {
            int s = 0;
            uint32_t ph = 1;
            bool ok = true;
            for (int i = blockIdx.x; ok && i < items; i += gridDim.x) {
                const Item it = item_of(i);
                for (int b = it.b0; b < it.b1; ++b) {
                    if (!(ok = tc_wait_one(bars.empty + 8 * s, ph, bars.dead))) break;
                    g_mbar_expect_tx(bars.full + 8 * s, kFewStage);
                    tl::g_tma_load_3d(g_smem_u32(few_smem + at.ring) + s * kFewStage, &map, b * 128, it.m * 128, lists.active[it.pos], bars.full + 8 * s);
                    if (++s == at.stages) s = 0, ph ^= 1u;
                }
            }
        }
    } else if (warp == 1) {
        if (g_elect_one()) {
            int s = 0, buf = 0, place = 0;
            uint32_t ph = 0, acc_ph = 1, cols_ph = 0;
            bool ok = true;
            uint32_t acc_free = 0, there = 0;  // asked ahead
            const uint32_t ring = g_smem_u32(few_smem + at.ring);
            for (int i = blockIdx.x; ok && i < items; i += gridDim.x) {
                const Item it = item_of(i);
                const int cols_block = (it.tokens * TERMS + 7) / 8 * 1024;
                const uint32_t cols = g_smem_u32(few_smem + at.cols) + place * FewSecondSmem::kCols;
                if (!(ok = tc_wait_one(bars.cols_full + 8 * place, cols_ph, bars.dead))) break;
                for (int b = it.b0; b < it.b1; ++b) {
                    if ((FP8 || b == it.b0) && !acc_free) ok = tc_wait_one(bars.acc_empty + 8 * buf, acc_ph, bars.dead);
                    if (ok && !there) ok = tc_wait_one(bars.full + 8 * s, ph, bars.dead);
                    if (!ok) break;
                    g_tc_fence_after();
                    const uint64_t w = g_smem_desc_sw128(ring + s * kFewStage, 0, 1024), h = g_smem_desc_sw128(cols + (b - it.b0) * cols_block, 0, 1024);
                    const uint32_t d = tmem + buf * kFewSecondN, done = bars.acc_full + 8 * buf, used = bars.empty + 8 * s;
                    const bool last = FP8 || b == it.b1 - 1;
                    if (++s == at.stages) s = 0, ph ^= 1u;
                    if (last && ++buf == BUFFERS) buf = 0, acc_ph ^= 1u;
                    few_block<FP8>(d, w, h, few_idesc<FP8>(it.n), !FP8 && b > it.b0, last, done, used, bars.acc_empty + 8 * buf, acc_ph, bars.full + 8 * s, ph, acc_free, there);
                }
                g_tc_commit(bars.cols_empty + 8 * place);
                if (++place == 2) place = 0, cols_ph ^= 1u;
            }
        }
    } else if (warp >= 4 && warp < 8) {  // the columns of an item, two items ahead at most
        int place = 0;
        uint32_t cols_ph = 1;
        for (int i = blockIdx.x; i < items; i += gridDim.x) {
            const Item it = item_of(i);
            const int cols_block = (it.tokens * TERMS + 7) / 8 * 1024, here = it.b1 - it.b0;
            unsigned char *cols = few_smem + at.cols + place * FewSecondSmem::kCols;
            float *factor = factors + place * (FewSecondSmem::kFactors / 4);
            const float *scales = FP8 ? a.s2 + ((size_t)lists.active[it.pos] * scale_rows + it.m) * scale_cols : nullptr;
            if (!tc_wait(bars.cols_empty + 8 * place, cols_ph, bars.dead)) break;
            const int runs = FP8 ? here : (here + 1) / 2, all = it.tokens * runs;  // of 128 entries
            constexpr int H_AT_ONCE = 4;
            for (int j0 = warp - 4; j0 < all; j0 += 4 * H_AT_ONCE) {
                float v[H_AT_ONCE][4], scale[H_AT_ONCE];
#pragma unroll
                for (int u = 0; u < H_AT_ONCE; ++u) {
                    const int j = j0 + 4 * u, c = j / runs, r = j - c * runs, k = it.b0 * ENTRIES + r * 128 + lane * 4;
                    v[u][0] = v[u][1] = v[u][2] = v[u][3] = scale[u] = 0.f;
                    if (c < it.tokens) {
                        const int column = lists.column[it.pos * 32 + it.first + c];
                        if (k < a.ld_inner) {
                            const uint4 w = tl::ld_cg(reinterpret_cast<const uint4 *>(a.inner + ((size_t)(column >> 8) * a.top + (column & 255)) * a.ld_inner + k));
                            v[u][0] = __uint_as_float(w.x), v[u][1] = __uint_as_float(w.y), v[u][2] = __uint_as_float(w.z), v[u][3] = __uint_as_float(w.w);
                        }
                        if constexpr (FP8) scale[u] = __ldg(scales + it.b0 + r);
                    }
                }
#pragma unroll
                for (int u = 0; u < H_AT_ONCE; ++u) {
                    const int j = j0 + 4 * u, c = j / runs, r = j - c * runs;
                    if (c >= it.tokens) break;
                    if constexpr (FP8) {
                        const uint32_t most = __reduce_max_sync(0xffffffffu, few_most4(v[u]));
                        const int e = few_exponent(__uint_as_float(most));
                        const float up = few_exp2(8 - e);
#pragma unroll
                        for (int q = 0; q < 4; ++q) v[u][q] *= up;
                        float f = most < 0x7f800000u ? few_exp2(e - 8) * scale[u] : __int_as_float(0x7fffffff);  // of a term
#pragma unroll
                        for (int term = 0; term < TERMS; ++term, f *= 0.0625f) {
                            *reinterpret_cast<uint32_t *>(cols + r * cols_block + few_swizzled(term * it.tokens + c, lane * 4)) = few_term(v[u]);
                            if (lane == 0) factor[r * kFewSecondN + term * it.tokens + c] = f;
                        }
                    } else {
                        const int b = r * 2 + (lane >> 4);
                        if (b < here) {
#pragma unroll
                            for (int term = 0; term < TERMS; ++term) {
                                uint32_t w[2];
#pragma unroll
                                for (int q = 0; q < 2; ++q) {
                                    w[q] = tl::pack2<bf16>(v[u][2 * q], v[u][2 * q + 1]);
                                    const float2 f = tl::unpack2<bf16>(w[q]);
                                    // an infinity has no further terms
                                    v[u][2 * q] = fabsf(f.x) < INFINITY ? v[u][2 * q] - f.x : 0.f, v[u][2 * q + 1] = fabsf(f.y) < INFINITY ? v[u][2 * q + 1] - f.y : 0.f;
                                }
                                *reinterpret_cast<uint2 *>(cols + b * cols_block + few_swizzled(term * it.tokens + c, (lane & 15) * 8)) = make_uint2(w[0], w[1]);
                            }
                        }
                    }
                }
            }
            tl::g_fence_proxy_async();
            __syncwarp();
            if (lane == 0) g_mbar_arrive(bars.cols_full + 8 * place);
            if (++place == 2) place = 0, cols_ph ^= 1u;
        }
    } else if (warp == 2 || warp == 3) {  // the tokens whose last partial sums an item's were: all of them, in order; a token a warp
        int slot = 0;
        uint32_t ph = 0;
        for (int i = blockIdx.x; i < items; i += gridDim.x) {
            const Item it = item_of(i);
            if (!tc_wait(bars.part_full + 8 * slot, ph, bars.dead)) {  // nobody else makes these outputs: what is not counted here never becomes whole
                for (int c = warp - 2; c < it.tokens; c += 2)
                    for (int d = it.m * 128 + lane; d < min(a.dim, it.m * 128 + 128); d += 32)
                        static_cast<OUT *>(a.out)[(size_t)(lists.column[it.pos * 32 + it.first + c] >> 8) * a.dim + d] = from_f<OUT>(__int_as_float(0x7fffffff));
                if (++slot == 2) slot = 0, ph ^= 1u;
                continue;
            }
            const int c = lane * 2 + warp - 2;
            bool last = false;
            if (c < it.tokens) {
                const int t = lists.column[it.pos * 32 + it.first + c] >> 8;
                uint32_t before;  // the release is for what the sums' warps wrote ahead of the barrier
                asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(a.finished + it.m * kFewTokens + t) : "memory");
                last = before == static_cast<uint32_t>(need[t] - 1);
            }
            uint32_t whole = __ballot_sync(0xffffffffu, last);
            __threadfence();  // the other lanes read behind the acquiring lane
            for (; whole; whole &= whole - 1)
                few_output<OUT>(a, lists.column[it.pos * 32 + it.first + (__ffs(whole) - 1) * 2 + warp - 2] >> 8, it.m * 128 + lane * 4, pairs, idx, gate);
            if (lane == 0) g_mbar_arrive(bars.part_empty + 8 * slot);
            if (++slot == 2) slot = 0, ph ^= 1u;
        }
    } else if (warp >= 8) {
        const int quarter = warp & 3, half = (warp - 8) >> 2, row = quarter * 32 + lane, me = tid - 256;
        int buf = 0, place = 0, slot = 0;
        uint32_t acc_ph = 0, cols_ph = 0, part_ph = 1;
        for (int i = blockIdx.x; i < items; i += gridDim.x) {
            const Item it = item_of(i);
            bool ok = tc_wait(bars.cols_full + 8 * place, cols_ph, bars.dead);  // their factors
            const float *factor = factors + place * (FewSecondSmem::kFactors / 4);
            auto add = [&](auto wide) {  // the columns of this half: 8, or 16
                constexpr int COLS = decltype(wide)::value;
                float acc[COLS];
#pragma unroll
                for (int c = 0; c < COLS; ++c) acc[c] = 0.f;
                const uint32_t from = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + half * COLS;
                for (int b = it.b0; b < (FP8 ? it.b1 : it.b0 + 1); ++b) {
                    [[maybe_unused]] float4 f[COLS / 4];
                    if constexpr (FP8) {
#pragma unroll
                        for (int c = 0; c < COLS / 4; ++c) f[c] = *reinterpret_cast<const float4 *>(factor + (b - it.b0) * kFewSecondN + half * COLS + c * 4);
                    }
                    ok &= tc_wait(bars.acc_full + 8 * buf, acc_ph, bars.dead);
                    g_tc_fence_after();
                    uint32_t v[COLS];
                    few_ld<COLS>(from + buf * kFewSecondN, v);
                    few_ld_wait();
                    g_tc_fence_before();
                    __syncwarp();
                    if (lane == 0) g_mbar_arrive(bars.acc_empty + 8 * buf);
#pragma unroll
                    for (int c = 0; c < COLS; ++c) {
                        if constexpr (FP8) acc[c] = fmaf(__uint_as_float(v[c]), c % 4 == 0 ? f[c / 4].x : c % 4 == 1 ? f[c / 4].y : c % 4 == 2 ? f[c / 4].z : f[c / 4].w, acc[c]);
                        else acc[c] = __uint_as_float(v[c]);
                    }
                    if (++buf == BUFFERS) buf = 0, acc_ph ^= 1u;
                }
#pragma unroll
                for (int c = 0; c < COLS; ++c) sums[(half * COLS + c) * 128 + row] = acc[c];
            };
            if (it.n == 16) add(std::integral_constant<int, 8>());
            else add(std::integral_constant<int, 16>());
            __syncwarp();  // every lane has used its factors: the sums that are in memory hold them
            if (lane == 0) g_mbar_arrive(bars.cols_empty + 8 * place);
            if (++place == 2) place = 0, cols_ph ^= 1u;
            const float bad = tc_verdict(ok, bars.dead);
            asm volatile("bar.sync 1, 256;" ::: "memory");
            for (int j = me; j < it.tokens * 128; j += 256) {
                const int r = j & 127, c = j >> 7, column = lists.column[it.pos * 32 + it.first + c], d = it.m * 128 + r;
                float y = sums[c * 128 + r];
#pragma unroll
                for (int term = 1; term < TERMS; ++term) y += sums[(term * it.tokens + c) * 128 + r];
                if (d < a.dim) a.part[((size_t)it.split * pairs + (column >> 8) * a.top + (column & 255)) * a.dim + d] = y * bad;
            }
            // written by all of these warps: two other warps see to what follows from it, two items behind at most
            asm volatile("bar.sync 1, 256;" ::: "memory");
            if (warp == 8) {
                tc_wait(bars.part_empty + 8 * slot, part_ph, bars.dead);
                if (lane == 0) g_mbar_arrive(bars.part_full + 8 * slot);
            }
            if (++slot == 2) slot = 0, part_ph ^= 1u;
        }
        for (int j = blockIdx.x * 8 + warp - 8; j < a.tokens * outs; j += gridDim.x * 8)  // tokens without an expert's product
            if (!lost && need[j / outs] == 0) few_output<OUT>(a, j / outs, j % outs * 128 + lane * 4, pairs, idx, gate);
    }
    __syncwarp();
    g_tc_fence_before();
    __syncthreads();
    if (warp == 2) {
        tc_settle(bars.dead);
        g_tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(TMEM) : "memory");
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------

constexpr int kFewSmem = 227 * 1024, kFewMostGrid = kFewThreads;  // the second launch reads a mark a thread

// CTAs of the first launch: as many clusters as are resident at once, which a device's SMs in groups decide (132 CTAs of a B200).
template <typename K>
static int few_grid(K kernel) {
    static std::atomic<int> known[64];
    int device = 0;
    cudaGetDevice(&device);
    if (device >= 0 && device < 64 && known[device].load(std::memory_order_acquire) > 0) return known[device].load(std::memory_order_relaxed);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(kFewCluster), cfg.blockDim = dim3(kFewThreads), cfg.dynamicSmemBytes = kFewSmem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = kFewCluster, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr, cfg.numAttrs = 1;
    int clusters = 0;
    if (cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg) != cudaSuccess || clusters <= 0) {
        cudaGetLastError();
        clusters = std::max(1, sm_count() / (2 * kFewCluster));  // fewer are slower, not wrong
    }
    const int grid = std::min(clusters * kFewCluster, kFewMostGrid);
    if (device >= 0 && device < 64) known[device].store(grid, std::memory_order_release);
    return grid;
}

// Two stages of the ring at least: one on its way while one is used.
static bool few_fits(int tokens, int nt, int dim, int outputs, int experts, int top, int groups, bool fp8) {
    const FewFirstSmem a(tokens, nt, dim, outputs, experts, top, groups, fp8, kFewSmem);
    const FewSecondSmem b(tokens, experts, top, kFewSmem);
    return a.stages >= 2 && a.total <= kFewSmem && b.stages >= 2 && b.total <= kFewSmem;
}

static int few_inner_ld(int ff) { return (ff + 15) / 16 * 16; }
static int few_nt(int tokens) { return ceil_div(tokens, 8); }
static int few_blocks(int ff, bool fp8) { return ceil_div(ff, fp8 ? 128 : 64); }

// Parts of the second product's reduction: as many as an item's columns need, or more where they let the SMs end closer together, by the blocks that the busiest
// takes (and six more an item for what it costs besides), if no two tokens choose the same expert.  The number of experts does not matter: it changes no bits.  Nor does
// the device: the 148 SMs that this was made for are written in, for a token's parts, and the order in which they are added, to be the same wherever it runs.
// 1 token, 6 of 64 experts of 1408 x 2048: in one part 29.0 us (bf16 37.2), in three 30.7 (38.6).
static int few_splits(int tokens, int dim, int top, int ff, bool fp8, bool wide) {
    const int blocks = few_blocks(ff, fp8), outs = ceil_div(dim, 128);
    const int cols_block = ceil_div(std::min(tokens, kFewGroup) * few_terms(fp8, wide), 8) * 1024, fewest = ceil_div(blocks, kFewItemCols / cols_block);
    int best = fewest;
    long long least = 0;
    for (int s = fewest; s <= std::max(fewest, std::min(blocks, 8)); ++s) {
        const long long time = (long long)ceil_div(tokens * top * outs * s, 148) * (ceil_div(blocks, s) + 6);
        if (s == fewest || time < least) best = s, least = time;
    }
    return best;
}

static size_t few_align(size_t n) { return (n + 15) & ~(size_t)15; }
static size_t few_bytes(int tokens, int dim, int top, int ff, bool fp8) {
    const size_t pairs = (size_t)tokens * top;
    return few_align(pairs * 4) * 2 + few_align((size_t)tokens * 4) + few_align((size_t)ceil_div(dim, 128) * kFewTokens * 4) + kFewMostGrid * 4 + pairs * few_inner_ld(ff) * 4 +
           (size_t)std::max(few_splits(tokens, dim, top, ff, fp8, false), few_splits(tokens, dim, top, ff, fp8, true)) * pairs * dim * 4;
}

template <typename K>
static int few_ready(K kernel, tl::PerDevice &ready) {
    int device = 0;
    cudaGetDevice(&device);
    if (ready(device, [&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kFewSmem) == cudaSuccess; })) return TL_OK;
    cudaGetLastError();
    return tl::fail(TL_ECUDA, "moe_few: no shared memory");
}

template <typename K, typename... A>
static int few_launch(K kernel, int grid, int cluster, int smem, cudaStream_t st, const A &...args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid), cfg.blockDim = dim3(kFewThreads), cfg.dynamicSmemBytes = smem, cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr, cfg.numAttrs = tl::use_pdl() ? 2 : 1;
    cudaLaunchKernelEx(&cfg, kernel, args...);
    TL_LAUNCH_CHECK("moe_few");
    return TL_OK;
}

template <bool FP8, int NT>
static int few_run(const CUtensorMap &mx, const CUtensorMap &m0, const CUtensorMap &m1, const CUtensorMap &m2, FewArgs a, bool gated, bool wide, cudaStream_t st) {
    static tl::PerDevice with, without, second16, second32;
    auto first = [&](auto kernel, tl::PerDevice &ready) {
        if (int e = few_ready(kernel, ready)) return e;
        a.first_ctas = few_grid(kernel);
        const int smem = FewFirstSmem(a.tokens, NT, a.dim, a.outputs, a.experts, a.top, a.group_count, FP8, kFewSmem).total;
        return few_launch(kernel, a.first_ctas, kFewCluster, smem, st, mx, m0, m1, a);
    };
    auto second = [&](auto kernel, tl::PerDevice &ready) {
        if (int e = few_ready(kernel, ready)) return e;
        return few_launch(kernel, sm_count(), 1, FewSecondSmem(a.tokens, a.experts, a.top, kFewSmem).total, st, m2, a);
    };
    if (int e = gated ? first(moe_few_first_kernel<FP8, true, NT>, with) : first(moe_few_first_kernel<FP8, false, NT>, without)) return e;
    return wide ? second(moe_few_second_kernel<FP8, float>, second32) : second(moe_few_second_kernel<FP8, bf16>, second16);
}

long long few_gave_up() { return tl::read_gave_up(); }

}  // namespace tlb

using namespace tlb;

extern "C" {

int tlb_moe_few_tokens(int dim, int outputs, int experts, int top, int group_count, int fp8) {
    if (dim <= 0 || dim > kFewWidth || outputs <= 0 || outputs > kFewOutputs || experts <= 0 || experts > outputs || top <= 0 || top > outputs || top > 255 || group_count < 0 ||
        group_count > outputs)
        return 0;
    int tokens = std::min(kFewTokens, kFewPairs / top);
    while (tokens > 0 && !few_fits(tokens, few_nt(tokens), dim, outputs, experts, top, group_count, fp8 != 0)) --tokens;
    return tokens;
}

size_t tlb_moe_few_workspace(int tokens, int dim, int experts, int top, int ff, int fp8) {
    return tokens <= 0 || dim <= 0 || top <= 0 || experts <= 0 || ff <= 0 ? 0 : few_bytes(tokens, dim, top, ff, fp8 != 0);
}

int tlb_moe_few(const tlb_moe_few_layer *l, const void *x, int tokens, const void *shared, void *out, int out_f32, void *workspace, size_t workspace_bytes, void *stream) {
    if (tokens <= 0) return TL_OK;
    if (!l || !x || !l->router || !l->w_up || !l->w_down || !out || !workspace || l->ff <= 0 || l->ff > (1 << 20) || l->scoring < 0 || l->scoring > 2 || (l->side_w && !shared))
        return tl::fail(TL_EINVAL, "moe_few: bad argument");
    const int dim = l->dim, ff = l->ff, top = l->top, experts = l->experts, outputs = l->outputs, groups = l->group_count, fp8 = l->fp8, size = fp8 ? 1 : 2;
    if (tokens > tlb_moe_few_tokens(dim, outputs, experts, top, groups, fp8)) return tl::fail(TL_EINVAL, "moe_few: %d tokens are too many for these sizes", tokens);
    if (l->group_keep < 0 || l->group_keep > groups || (groups > 0 && (outputs % groups || l->group_keep * (outputs / groups) < top)))
        return tl::fail(TL_EINVAL, "moe_few: bad groups");
    if (l->w_gate ? (l->act != 0 && l->act != 1 && l->act != 3) || (l->act == 3 && !(l->limit > 0.f)) : l->act < 0 || l->act > 2)
        return tl::fail(TL_EINVAL, "moe_few: bad activation");
    if (fp8 && (!l->s_up || !l->s_down || (l->w_gate && !l->s_gate))) return tl::fail(TL_EINVAL, "moe_few: 8-bit weights without scales");
    if (dim % 8 || l->ld_in < dim * size || l->ld_out < ff * size || l->ld_in % 16 || l->ld_out % 16 || !tl::aligned16(x) || !tl::aligned16(l->router) ||
        !tl::aligned16(l->side_w) || !tl::aligned16(l->w_gate) || !tl::aligned16(l->w_up) || !tl::aligned16(l->w_down) || !tl::aligned16(workspace))
        return tl::fail(TL_EINVAL, "moe_few: rows must be whole 16-byte pieces");
    if (workspace_bytes < few_bytes(tokens, dim, top, ff, fp8 != 0)) return tl::fail(TL_EINVAL, "moe_few: workspace too small");
    const size_t pairs = (size_t)tokens * top;
    FewArgs a{};
    a.x = (const bf16 *)x, a.router = (const bf16 *)l->router, a.router_bias = (const bf16 *)l->router_bias, a.choice_bias = (const bf16 *)l->choice_bias;
    a.side_w = (const bf16 *)l->side_w, a.tokens = tokens, a.dim = dim, a.outputs = outputs, a.experts = experts, a.top = top, a.scoring = l->scoring, a.group_count = groups;
    a.group_keep = l->group_keep, a.weight_scale = l->weight_scale;
    a.s0 = l->w_gate ? l->s_gate : l->s_up, a.s1 = l->w_gate ? l->s_up : nullptr, a.s2 = l->s_down;
    a.ff = ff;
    a.act = l->act, a.limit = l->limit, a.slope = l->slope, a.shared = (const bf16 *)shared, a.out = out;
    uint8_t *at = (uint8_t *)workspace;
    a.idx = (int32_t *)at, at += few_align(pairs * 4);
    a.gate = (float *)at, at += few_align(pairs * 4);
    a.side = (float *)at, at += few_align((size_t)tokens * 4);
    a.finished = (uint32_t *)at, at += few_align((size_t)ceil_div(dim, 128) * kFewTokens * 4);
    a.lost = (int32_t *)at, at += kFewMostGrid * 4;
    a.inner = (float *)at, a.ld_inner = few_inner_ld(ff), at += pairs * a.ld_inner * 4;
    a.part = (float *)at, a.splits = few_splits(tokens, dim, top, ff, fp8 != 0, out_f32 != 0), a.room = kFewSmem;
    // what lies between a row's last number and the next row is read as zeros
    const uint64_t in = (uint64_t)dim * size, inner = (uint64_t)ff * size;
    CUtensorMap mx, m0, m1, m2;
    const int nt = few_nt(tokens);
    if (int e = tc_map_bytes(&mx, x, (uint64_t)dim * 2, tokens, (uint64_t)dim * 2, 8 * nt)) return e;
    if (int e = tc_map_bytes3(&m0, l->w_gate ? l->w_gate : l->w_up, in, ff, experts, l->ld_in, l->w_gate ? 64 : 128)) return e;
    if (int e = tc_map_bytes3(&m1, l->w_up, in, ff, experts, l->ld_in, 64)) return e;
    if (int e = tc_map_bytes3(&m2, l->w_down, inner, dim, experts, l->ld_out, 128)) return e;
    const cudaStream_t st = as_stream(stream);
    const bool gated = l->w_gate != nullptr, wide = out_f32 != 0;
    switch (nt + (fp8 ? 4 : 0)) {
        case 1: return few_run<false, 1>(mx, m0, m1, m2, a, gated, wide, st);
        case 2: return few_run<false, 2>(mx, m0, m1, m2, a, gated, wide, st);
        case 3: return few_run<false, 3>(mx, m0, m1, m2, a, gated, wide, st);
        case 4: return few_run<false, 4>(mx, m0, m1, m2, a, gated, wide, st);
        case 5: return few_run<true, 1>(mx, m0, m1, m2, a, gated, wide, st);
        case 6: return few_run<true, 2>(mx, m0, m1, m2, a, gated, wide, st);
        case 7: return few_run<true, 3>(mx, m0, m1, m2, a, gated, wide, st);
        default: return few_run<true, 4>(mx, m0, m1, m2, a, gated, wide, st);
    }
}

#ifdef TLB_FEW_STARVED
int tlb_few_starve(int cta) { return cudaMemcpyToSymbol(g_few_starved, &cta, sizeof(cta)) == cudaSuccess ? TL_OK : TL_ECUDA; }
long long tlb_few_starved_waits(void) { return few_gave_up(); }
#endif

}  // extern "C"
