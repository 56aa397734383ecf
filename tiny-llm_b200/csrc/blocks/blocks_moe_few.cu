// A whole mixture-of-experts layer for the few tokens of a decoding step, in two launches, over experts of bf16 numbers or of e4m3 numbers
// with one scale for each block of 128 x 128.
//
//   first launch:  logits = router . x, the choice, inner[pair] = act(gate_e x) * (up_e x)        pair = (token, choice)
//   second launch: y[t] = sum over choices  weight * (down_e inner[pair])  (+ identity experts, + shared expert)
//
// Bound by HBM: every matrix of a chosen expert is read once.  So the features of all chosen experts are one list that is cut into equal runs,
// whatever the number of tokens and experts, and a warp keeps several 2 KB pieces of weights on their way in registers.  The arithmetic
// is m16n8k16 products of the tensor cores' warp form with the weights as the 16 rows, the tokens as the columns: at 1 to 32 columns they
// need a small part of the SM's issue slots, and a column is a token for all experts, so a piece's B operand is an indexed read.
//
// Order of the reduction index: a lane holds 16 consecutive bytes of a row (one load), which is what it contributes to the products' k index,
// of both operands alike; no operand is ever shuffled.
//
// e4m3 numbers become fp16 exactly; then x (a power of two for each token) and the inner rows (a power of two for each block of 128)
// are fp16 as well, off by 2^-11 of the value or 2^-24 of the row's or block's largest (x's own numbers of 8 bits only by the latter).  bf16
// numbers meet bf16 ones: x is as it came, and an inner row is two bf16 terms, off by 2^-16.  Sums are fp32 throughout; with 8 bits the 128 of a block are added before their scale multiplies them.
//
// No CTA waits for another outside its cluster: the cluster's CTAs share the router's rows, exchange the logits through shared memory, and every
// CTA makes the same choices for itself.  The second launch reads the choices and the inner rows behind the wait for the first.
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <atomic>

#include "../per_device.h"
#include "blocks_moe.cuh"

namespace tlb {

constexpr int kFewThreads = 512, kFewWarps = 16;
constexpr int kFewTokens = 32, kFewPairs = 512, kFewOutputs = 1024;
constexpr int kFewTeams = 4, kFewTeam = 4;  // first launch: teams of a CTA, each with its own run of features; warps of a team, which share the reduction

struct FewArgs {
    const bf16 *x, *router, *router_bias, *choice_bias, *side_w;
    int tokens, dim, outputs /* of the router */, experts, top, scoring, group_count, group_keep;
    float weight_scale;
    const uint8_t *w0, *w1, *w2;  // gate, up (w1 NULL: w0 is the up projection), down
    const float *s0, *s1, *s2;    // block scales
    int ff, ld_in, ld_out;        // bytes from row to row of w0 / w1 and of w2
    int bytes_in, bytes_out;      // of a row that are read: whole pieces of 16, zero behind the last number
    int act;
    float limit, slope;
    const bf16 *shared;
    void *out;
    // between the launches
    int32_t *idx;      // [tokens, top]
    float *gate;       // [tokens, top]
    float *side;       // [tokens]
    float *inner;      // [tokens * top, ld_inner], zero behind ff
    int ld_inner, runs;  // runs of features: teams of the first launch
    int room;            // bytes of shared memory that a launch may use
    int prefetch;        // bytes that a CTA of the first launch asks into L2 for the second
};

// ---- small things ----------------------------------------------------------------------------------------------------

__device__ __forceinline__ uint4 few_ldg(const uint8_t *p) {  // weights: read once
    uint4 r;
    asm volatile("ld.global.nc.L1::no_allocate.L2::128B.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
    return r;
}
template <bool FP8>
__device__ __forceinline__ void few_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (FP8)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// four e4m3 numbers -> two pairs of fp16 ones
__device__ __forceinline__ void few_wide(uint32_t v, uint32_t &lo, uint32_t &hi) {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}" : "=r"(lo), "=r"(hi) : "r"(v));
}
__device__ __forceinline__ uint32_t few_half2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
// 2^e with |v| 2^-e in [0.5, 1) for a normal v, within what fp32 holds both ways
__device__ __forceinline__ int few_exponent(float most) {
    const int e = static_cast<int>(__float_as_uint(most) >> 23) - 126;
    return most < INFINITY ? min(126, max(-100, e)) : 0;  // an infinity or NaN stays what it is
}
__device__ __forceinline__ float few_exp2(int e) { return __int_as_float((e + 127) << 23); }

// A warp's piece of 16 rows, 128 bytes of each: four copies of four whole lines (cp.async) into a place of the warp's own, so that a piece is waited for by
// counting one's copies, without a barrier of the CTA.  Behind it the scales of rows 0-7 and 8-15.  A lane then has rows g = lane / 4 and g + 8, 16 bytes at
// t * 16 (t = lane % 4) of either half; odd rows keep their halves exchanged, which spares those reads bank conflicts.
struct FewPiece {
    uint4 a[2], b[2];  // rows g, g + 8
    float2 scale;
};
constexpr int kFewPiece = 2048, kFewPlace = kFewWarps * (kFewPiece + 8);  // bytes of a piece, of one place of all warps
__device__ __forceinline__ void few_copy16(uint32_t to, const uint8_t *from, bool there) {  // not there: zeros, nothing is read
    const int bytes = there ? 16 : 0;
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void few_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// The queue: `depth` places in turn.  place: this warp's share of the first one.
struct FewQueue {
    uint32_t place;
    const unsigned char *at;
    uint32_t scales;  // bytes from this warp's piece to its scales
    int depth, ask, take;
    __device__ FewQueue(unsigned char *smem, int from, int depth_, int warp)
        : place(static_cast<uint32_t>(__cvta_generic_to_shared(smem + from + warp * kFewPiece))), at(smem + from + warp * kFewPiece),
          scales((kFewWarps - warp) * kFewPiece + warp * 8), depth(depth_), ask(0), take(0) {}
    // low, high: this lane's 16 bytes of rows lane / 8 of the first and of the second eight; l0, l1, h0, h1: whether they and those four rows further on are there
    __device__ __forceinline__ void copy(const uint8_t *low, const uint8_t *high, size_t four, bool l0, bool l1, bool h0, bool h1) const {
        __syncwarp();  // the place's last piece has been used by all lanes
        const int lane = threadIdx.x & 31;
        const uint32_t to = place + ask * kFewPlace + (lane >> 3) * 128 + (((lane & 7) ^ (lane >> 1 & 4)) << 4);
        few_copy16(to, low, l0), few_copy16(to + 512, low + four, l1), few_copy16(to + 1024, high, h0), few_copy16(to + 1536, high + four, h1);
    }
    __device__ __forceinline__ void copy_scale(const float *from) const {  // lanes 0 and 1
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(place + ask * kFewPlace + scales + (threadIdx.x & 31) * 4), "l"(from) : "memory");
    }
    __device__ __forceinline__ void asked() {
        few_commit();
        if (++ask == depth) ask = 0;
    }
    template <bool FP8>
    __device__ __forceinline__ FewPiece next() {
        switch (depth) {  // all but the newest depth - 1 of this thread's groups are there
            case 2: asm volatile("cp.async.wait_group 1;" ::: "memory"); break;
            case 3: asm volatile("cp.async.wait_group 2;" ::: "memory"); break;
            case 4: asm volatile("cp.async.wait_group 3;" ::: "memory"); break;
            case 5: asm volatile("cp.async.wait_group 4;" ::: "memory"); break;
            default: asm volatile("cp.async.wait_group 5;" ::: "memory"); break;
        }
        __syncwarp();
        const int lane = threadIdx.x & 31, g = lane >> 2;
        const unsigned char *from = at + take * kFewPlace + g * 128 + ((lane & 3) << 4);
        FewPiece p;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const unsigned char *half = from + ((c ^ (g & 1)) << 6);
            p.a[c] = *reinterpret_cast<const uint4 *>(half), p.b[c] = *reinterpret_cast<const uint4 *>(half + 1024);
        }
        if constexpr (FP8) p.scale = *reinterpret_cast<const float2 *>(at + take * kFewPlace + scales);
        if (++take == depth) take = 0;
        return p;
    }
};
constexpr int kFewDepth = 6;  // the most places

// The products of half a piece (64 bytes of each row) with one tile of eight columns: x, the lane's 16 bytes' worth of column g.
template <bool FP8>
__device__ __forceinline__ void few_half(const uint4 &a, const uint4 &b, const uint32_t (&x)[FP8 ? 8 : 4], float (&d)[4]) {
    const uint32_t wa[4] = {a.x, a.y, a.z, a.w}, wb[4] = {b.x, b.y, b.z, b.w};
    if constexpr (FP8) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t a0, a2, b0, b2;
            few_wide(wa[j], a0, a2), few_wide(wb[j], b0, b2);
            few_mma<true>(d, a0, b0, a2, b2, x[2 * j], x[2 * j + 1]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 2; ++j) few_mma<false>(d, wa[2 * j], wb[2 * j], wa[2 * j + 1], wb[2 * j + 1], x[2 * j], x[2 * j + 1]);
    }
}

// The chosen experts in ascending order and the tokens that chose each, in ascending order: a token's place is its column.  Both launches make these for
// themselves.
struct FewLists {
    uint32_t *words;   // [32]: a bit for every expert, zero at the start
    uint32_t *tokens;  // [most]: the tokens of an active expert, zero at the start
    int *active;       // [most]
    uint16_t *column;  // [most][32]: token * 256 + choice
    int *count;
};
struct FewListsSmem {  // from `at` on, a multiple of 4
    int words, tokens, active, count, column, end;
    __host__ __device__ FewListsSmem(int at, int tokens_, int top, int experts) {
        const int most = tokens_ * top < experts ? tokens_ * top : experts;
        words = at, tokens = words + 128, active = tokens + most * 4, count = active + most * 4, column = count + 4, end = (column + most * 64 + 15) / 16 * 16;
    }
    __device__ FewLists lists(unsigned char *smem) const {
        return {reinterpret_cast<uint32_t *>(smem + words), reinterpret_cast<uint32_t *>(smem + tokens), reinterpret_cast<int *>(smem + active),
                reinterpret_cast<uint16_t *>(smem + column), reinterpret_cast<int *>(smem + count)};
    }
    __device__ void clear(unsigned char *smem) const {  // words and tokens lie side by side
        for (int i = threadIdx.x; i < (active - words) / 4; i += kFewThreads) reinterpret_cast<uint32_t *>(smem + words)[i] = 0;
    }
};
// All threads of the CTA, a pair each; behind a barrier after clear() and the last write of idx, which is in shared memory.
__device__ __forceinline__ void few_lists(const FewArgs &a, const int *idx, const FewLists &l) {
    static_assert(kFewPairs <= kFewThreads, "a pair a thread");
    const int p = threadIdx.x, lane = p & 31, t = p / a.top, k = p % a.top;
    int e = p < a.tokens * a.top ? idx[p] : a.experts;
    for (int j = 1; j <= k && e < a.experts; ++j)  // a token that names an expert twice (equal logits of minus infinity) has it once, by its first choice
        if (idx[p - j] == e) e = a.experts;
    const bool live = e < a.experts;
    if (live) atomicOr(&l.words[e >> 5], 1u << (e & 31));
    __syncthreads();
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
    if (live) l.column[pos * 32 + __popc(l.tokens[pos] & ((1u << t) - 1))] = (uint16_t)(t * 256 + k);
    __syncthreads();
}

// Features 0 .. total - 1 in `runs` runs that differ by one at most.
__device__ __forceinline__ int few_run_start(int total, int runs, int v) { return v * (total / runs) + min(v, total % runs); }
// ---- first launch ----------------------------------------------------------------------------------------------------

constexpr int kFewCluster = 4;

static inline __host__ __device__ int few_x_stride(int dim, bool fp8) {  // bytes of a token's row in shared memory: its 16-byte reads meet no bank conflict
    return (dim + 127) / 128 * 256 + (fp8 ? 16 : 64);
}
struct FewFirstSmem {
    int x, red, most, idx, gate, queue, logits, depth, total;
    FewListsSmem lists;
    __host__ __device__ FewFirstSmem(int tokens, int nt, int dim, int outputs, int experts, int top, int groups, bool fp8, int room) : lists(0, tokens, top, experts) {
        x = 0;
        red = x + tokens * few_x_stride(dim, fp8);
        const int teams = 2 * kFewWarps * 16 * 8 * 4, router = kFewWarps * 16 * nt * 8 * 4;  // sums of a tile's eight columns, in turn in two places; the router's sums
        most = red + teams;
        idx = most + kFewTokens * 4;
        gate = idx + tokens * top * 4;
        lists = FewListsSmem(gate + tokens * top * 4, tokens, top, experts);
        // the router's sums and logits are done with when the queue's first copies are asked for
        queue = lists.end;
        logits = queue + router;
        const int early = router + (tokens * (2 * outputs + groups) + tokens) * 4;
        depth = (room - queue) / kFewPlace;
        if (depth > kFewDepth) depth = kFewDepth;
        const int late = depth * kFewPlace;
        total = queue + (early > late ? early : late);
    }
};

template <bool FP8, bool GATED, int NT>
__global__ void __launch_bounds__(kFewThreads, 1)
moe_few_first_kernel(const FewArgs a) {
    extern __shared__ __align__(128) unsigned char few_smem[];
    const FewFirstSmem at(a.tokens, NT, a.dim, a.outputs, a.experts, a.top, a.group_count, FP8, a.room);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
    const int stride = few_x_stride(a.dim, FP8);
    uint32_t rank, ranks;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
    // Another CTA's shared memory may be written once that CTA runs: arrived at here, waited for ahead of the first such store.
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    float *logits = reinterpret_cast<float *>(few_smem + at.logits), *router_red = reinterpret_cast<float *>(few_smem + at.queue);
    const int per_token = 2 * a.outputs + a.group_count;
    float *side = logits + a.tokens * per_token, *gate = reinterpret_cast<float *>(few_smem + at.gate);
    uint32_t *most = reinterpret_cast<uint32_t *>(few_smem + at.most);
    int *idx = reinterpret_cast<int *>(few_smem + at.idx);
    const FewLists lists = at.lists.lists(few_smem);
    at.lists.clear(few_smem);
    if (tid < kFewTokens) most[tid] = 0;
    __syncthreads();

    tl::griddep_wait();
    tl::griddep_launch();  // the second launch reads nothing ahead of its own wait
    // ---- the router's rows, 16 for eight warps each, which share the reduction; a CTA of the cluster every ranks-th 32 of them
    const int rows = a.outputs + (a.side_w ? 1 : 0), pieces = (a.dim * 2 + 127) / 128, part = warp & 7;
    constexpr int AT_ONCE = 4;
    uint4 wa[AT_ONCE][2], wb[AT_ONCE][2];
    auto row_of = [&](int r) { return reinterpret_cast<const uint8_t *>(r < a.outputs ? a.router + (size_t)r * a.dim : r < rows ? a.side_w : nullptr); };
    auto ask = [&](int m, int s0) {
        const uint8_t *ra = row_of(m * 16 + g), *rb = row_of(m * 16 + g + 8);
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int o = (s0 + u * 8) * 128 + c * 64 + t4 * 16;
                wa[u][c] = ra && o < a.dim * 2 ? few_ldg(ra + o) : make_uint4(0, 0, 0, 0);
                wb[u][c] = rb && o < a.dim * 2 ? few_ldg(rb + o) : make_uint4(0, 0, 0, 0);
            }
    };
    const int m_first = rank * 2 + (warp >> 3);
    ask(m_first, part);
    // ---- the tokens' rows, 256 entries a warp, zero behind the last one, and (8 bits) their largest magnitudes
    const int entries = (a.dim + 127) / 128 * 128, segs = (entries + 255) / 256;
    constexpr int X_AT_ONCE = 4;
    for (int i0 = warp; i0 < a.tokens * segs; i0 += X_AT_ONCE * kFewWarps) {
        uint4 v[X_AT_ONCE];
#pragma unroll
        for (int u = 0; u < X_AT_ONCE; ++u) {
            const int i = i0 + u * kFewWarps, t = i / segs, d = (i - t * segs) * 256 + lane * 8;
            v[u] = make_uint4(0, 0, 0, 0);
            if (t < a.tokens && d < a.dim) v[u] = tl::ld_cg(reinterpret_cast<const uint4 *>(a.x + (size_t)t * a.dim + d));
        }
#pragma unroll
        for (int u = 0; u < X_AT_ONCE; ++u) {
            const int i = i0 + u * kFewWarps, t = i / segs, d = (i - t * segs) * 256 + lane * 8;
            if (t >= a.tokens) break;
            if (d < entries) *reinterpret_cast<uint4 *>(few_smem + t * stride + d * 2) = v[u];
            if constexpr (FP8) {
                const uint32_t c[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
                uint32_t top = 0;  // of the 15 bits of a magnitude, which are in order; an infinity is above all numbers, a NaN above that
#pragma unroll
                for (int j = 0; j < 4; ++j) top = max(top, max(c[j] & 0x7fffu, c[j] >> 16 & 0x7fffu));
                top = __reduce_max_sync(0xffffffffu, top);
                if (lane == 0) atomicMax(&most[t], top);
            }
        }
    }
    __syncthreads();
    bool waited = false;
    for (int m = m_first; (m - (warp >> 3)) * 16 < rows; m += ranks * 2) {
        float acc[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
        for (int s = part; s < pieces; s += AT_ONCE * 8) {
            if (m != m_first || s != part) ask(m, s);
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u)
                if (s + u * 8 < pieces)
#pragma unroll
                    for (int c = 0; c < 2; ++c)
#pragma unroll
                        for (int n = 0; n < NT; ++n) {  // columns past the last token: the last one, not used
                            const uint4 v = *reinterpret_cast<const uint4 *>(few_smem + min(n * 8 + g, a.tokens - 1) * stride + (s + u * 8) * 128 + c * 64 + t4 * 16);
                            const uint32_t x[4] = {v.x, v.y, v.z, v.w};
                            few_half<false>(wa[u][c], wb[u][c], x, acc[n]);
                        }
        }
        float *mine = router_red + warp * 16 * NT * 8;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            *reinterpret_cast<float2 *>(mine + g * NT * 8 + n * 8 + 2 * t4) = make_float2(acc[n][0], acc[n][1]);
            *reinterpret_cast<float2 *>(mine + (g + 8) * NT * 8 + n * 8 + 2 * t4) = make_float2(acc[n][2], acc[n][3]);
        }
        __syncthreads();
        if (!waited) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // all CTAs of the cluster run
        waited = true;
        const int m0 = m - (warp >> 3);
        for (int i = tid; i < 2 * 16 * NT * 8; i += kFewThreads) {
            const int in = i % (16 * NT * 8), r = (m0 + i / (16 * NT * 8)) * 16 + in / (NT * 8), t = in % (NT * 8);
            if (r >= rows || t >= a.tokens) continue;
            float z = 0.f;
#pragma unroll
            for (int w = 0; w < 8; ++w) z += router_red[(i / (16 * NT * 8) * 8 + w) * 16 * NT * 8 + in];
            if (r < a.outputs && a.router_bias) z += to_f(a.router_bias[r]);
            const uint32_t to = static_cast<uint32_t>(__cvta_generic_to_shared(r < a.outputs ? logits + t * per_token + r : side + t));
            for (uint32_t c = 0; c < ranks; ++c)
                asm volatile("{\n\t.reg .b32 ra;\n\tmapa.shared::cluster.u32 ra, %0, %1;\n\tst.shared::cluster.f32 [ra], %2;\n\t}" ::"r"(to), "r"(c), "f"(z) : "memory");
        }
        __syncthreads();
    }
    if (!waited) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    if constexpr (FP8) {  // the rows as fp16 times a power of two; the router is done with them
        for (int i = warp; i < a.tokens * segs; i += kFewWarps) {
            const int t = i / segs, d = i % segs * 256 + lane * 8;
            const float down = few_exp2(-few_exponent(__uint_as_float(most[t] << 16)));
            if (d < entries) {
                uint4 *p = reinterpret_cast<uint4 *>(few_smem + t * stride + d * 2);
                const uint4 u = *p;
                const uint32_t c[4] = {u.x, u.y, u.z, u.w};
                uint32_t o[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 f = tl::unpack2<bf16>(c[j]);
                    o[j] = few_half2(f.x * down, f.y * down);
                }
                *p = make_uint4(o[0], o[1], o[2], o[3]);
            }
        }
    }
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");

    // ---- the choice, by every CTA for itself
    for (int t = warp; t < a.tokens; t += kFewWarps) {
        float *z = logits + t * per_token;
        moe_choose(z, z + a.outputs, z + 2 * a.outputs, lane, a.outputs, a.top, a.scoring, a.choice_bias, a.weight_scale, a.group_count, a.group_keep, idx + t * a.top,
                   gate + t * a.top);
    }
    __syncthreads();
    if (blockIdx.x == 0) {
        for (int p = tid; p < a.tokens * a.top; p += kFewThreads) a.idx[p] = idx[p], a.gate[p] = gate[p];
        if (a.side_w && tid < a.tokens) a.side[tid] = sigmoid(side[tid]);
    }
    few_lists(a, idx, lists);

    // ---- the first products: a team takes its run of the chosen experts' features, up to 8 (with a gate; else 16) of one expert at a time
    constexpr int TILE = GATED ? 8 : 16;
    const int team = warp / kFewTeam, sub = warp % kFewTeam, run = blockIdx.x * kFewTeams + team, total = *lists.count * a.ff;
    const int blocks_in = (a.bytes_in + 127) / 128, iters = (blocks_in + kFewTeam - 1) / kFewTeam;
    const int scale_cols = (a.dim + 127) / 128, scale_rows = (a.ff + 127) / 128;
    struct Tile {
        int pos, row, here, left;
    };
    auto cut = [&](Tile &s) { s.here = min(min(TILE, a.ff - s.row), min(s.left, 128 - (s.row & 127))); };  // within one block of scales
    auto advance = [&](Tile &s) {
        s.left -= s.here, s.row += s.here;
        if (s.row == a.ff) s.row = 0, ++s.pos;
        cut(s);
    };
    Tile tile;
    {
        const int f0 = few_run_start(total, a.runs, run), f1 = few_run_start(total, a.runs, run + 1);
        tile.left = f1 - f0, tile.pos = f0 / a.ff, tile.row = f0 % a.ff;
        cut(tile);
    }
    FewQueue queue(few_smem, at.queue, at.depth, warp);
    Tile ahead = tile;
    const uint8_t *low = nullptr, *high = nullptr;  // this lane's 16 bytes of the next piece
    const float *scale = nullptr;
    int byte = 0, piece = 0;
    const size_t four = (size_t)4 * a.ld_in;
    auto enter = [&] {
        if (ahead.left <= 0) return;
        const int e = lists.active[ahead.pos];
        const size_t row = (size_t)e * a.ff + ahead.row + (lane >> 3);
        byte = sub * 128 + (lane & 7) * 16, piece = sub;
        low = a.w0 + row * a.ld_in + byte, high = GATED ? a.w1 + row * a.ld_in + byte : low + 2 * four;
        if constexpr (FP8) scale = (GATED && lane == 1 ? a.s1 : a.s0) + ((size_t)e * scale_rows + (ahead.row >> 7)) * scale_cols + sub;
    };
    enter();
    auto issue = [&] {
        if (ahead.left > 0) {
            const bool in = byte < a.bytes_in;
            const int left = in ? ahead.here - (lane >> 3) : 0;
            queue.copy(low, high, four, left > 0, left > 4, left > (GATED ? 0 : 8), left > (GATED ? 4 : 12));
            if (FP8 && lane < 2 && piece < blocks_in) queue.copy_scale(scale);
            if constexpr (FP8) scale += kFewTeam;
            low += kFewTeam * 128, high += kFewTeam * 128, byte += kFewTeam * 128, piece += kFewTeam;
            if (piece - sub >= iters * kFewTeam) {
                advance(ahead), enter();
                if (ahead.left <= 0) {
                    // the last weights of this launch are on their way: the first of the next one's are asked into L2 behind them
                    const int d0 = (int)((long long)a.dim * blockIdx.x / gridDim.x), d1 = (int)((long long)a.dim * (blockIdx.x + 1) / gridDim.x);
                    const int bytes = (d1 - d0) * a.ld_out, experts = bytes > 0 ? min(*lists.count, a.prefetch / bytes) : 0;
                    for (int q = warp + lane * kFewWarps; q < experts; q += 32 * kFewWarps)
                        asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(a.w2 + ((size_t)lists.active[q] * a.dim + d0) * a.ld_out), "r"(bytes) : "memory");
                }
            }
        }
        queue.asked();  // an empty group where nothing is left: the count of groups stays that of the places
    };
    float acc[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
    int it = 0, turn = 0;
    const int i128 = sub * 32 + lane, f8 = i128 & 7, col8 = i128 >> 3 & 7;  // the first 64 threads of a team finish a feature (two without a gate) of a column each
    auto finish = [&](int columns) {  // the tile's sums over the team's warps, the activation, the inner rows
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            if (n * 8 >= columns) break;
            float *sums = reinterpret_cast<float *>(few_smem + at.red) + ((turn ^= 1) * kFewTeams + team) * kFewTeam * 128, *mine = sums + sub * 128;
            *reinterpret_cast<float2 *>(mine + g * 8 + 2 * t4) = make_float2(acc[n][0], acc[n][1]);
            *reinterpret_cast<float2 *>(mine + (g + 8) * 8 + 2 * t4) = make_float2(acc[n][2], acc[n][3]);
            acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
            // one barrier for each use of either place: a place is written again only behind the other's
            asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "n"(kFewTeam * 32) : "memory");
            if (i128 < 64) {
                const int col = n * 8 + col8;
                if (col < columns) {
                    const int c = lists.column[tile.pos * 32 + col], t = c >> 8;
                    float v[2] = {};
#pragma unroll
                    for (int w = 0; w < kFewTeam; ++w) v[0] += sums[w * 128 + f8 * 8 + col8], v[1] += sums[w * 128 + (f8 + 8) * 8 + col8];
                    if constexpr (FP8) {
                        const float up = few_exp2(few_exponent(__uint_as_float(most[t] << 16)));
                        v[0] *= up, v[1] *= up;
                    }
                    float *to = a.inner + ((size_t)t * a.top + (c & 255)) * a.ld_inner + tile.row;
                    if constexpr (GATED) {
                        if (f8 < tile.here) {
                            to[f8] = gated_pair(v[0], v[1], a.act, a.limit, a.slope);
                        }
                    } else {
#pragma unroll
                        for (int u = 0; u < 2; ++u)
                            if (f8 + 8 * u < tile.here) {
                                to[f8 + 8 * u] = a.act == 2 ? (v[u] > 0.f ? v[u] * v[u] : v[u] == v[u] ? 0.f : v[u]) : act_apply(v[u], a.act);
                            }
                    }
                    if (tile.row + tile.here == a.ff)
                        for (int z = a.ff + f8; z < a.ld_inner; z += 8) to[z - tile.row] = 0.f;
                }
            }
        }
        advance(tile);
    };
    for (int i = 0; i < at.depth; ++i) issue();
    while (tile.left > 0) {
        const int columns = __popc(lists.tokens[tile.pos]);
        int row[NT];  // this lane's columns' rows; past the last column the first token's, not used
#pragma unroll
        for (int n = 0; n < NT; ++n) row[n] = (n * 8 + g < columns ? lists.column[tile.pos * 32 + n * 8 + g] >> 8 : 0) * stride + t4 * (FP8 ? 32 : 16);
        for (it = 0; it < iters; ++it) {
            const FewPiece p = queue.next<FP8>();
            const int b = sub + it * kFewTeam;
            if (b < blocks_in) {
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    if (n * 8 >= columns) break;
                    if constexpr (FP8) {
                        float d[2][4] = {};
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const unsigned char *from = few_smem + row[n] + b * 256 + c * 128;
                            const uint4 u = *reinterpret_cast<const uint4 *>(from), v = *reinterpret_cast<const uint4 *>(from + 16);
                            const uint32_t x[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
                            few_half<true>(p.a[c], p.b[c], x, d[c]);
                        }
                        const float sb = GATED ? p.scale.y : p.scale.x;
                        acc[n][0] = fmaf(d[0][0] + d[1][0], p.scale.x, acc[n][0]), acc[n][1] = fmaf(d[0][1] + d[1][1], p.scale.x, acc[n][1]);
                        acc[n][2] = fmaf(d[0][2] + d[1][2], sb, acc[n][2]), acc[n][3] = fmaf(d[0][3] + d[1][3], sb, acc[n][3]);
                    } else {
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const uint4 u = *reinterpret_cast<const uint4 *>(few_smem + row[n] + b * 128 + c * 64);
                            const uint32_t x[4] = {u.x, u.y, u.z, u.w};
                            few_half<false>(p.a[c], p.b[c], x, acc[n]);
                        }
                    }
                }
            }
            issue();
        }
        finish(columns);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
}

// ---- second launch ---------------------------------------------------------------------------------------------------

struct FewSecondSmem {
    int sums, idx, factor, queue, depth, total;
    FewListsSmem lists;
    __host__ __device__ FewSecondSmem(int tokens, int experts, int top, bool fp8, int room) : lists(0, tokens, top, experts) {
        sums = 0;
        idx = sums + kFewWarps * few_sum_stride(tokens) * 4;
        factor = idx + tokens * top * 4;
        lists = FewListsSmem(factor + tokens * top * 4, tokens, top, experts);
        queue = lists.end;
        depth = (room - queue) / kFewPlace;
        if (depth > kFewDepth) depth = kFewDepth;
        total = queue + depth * kFewPlace;
    }
    // a warp's sums, [token][17] (16 rows, and one place that keeps the tokens' from falling into the same banks)
    static __host__ __device__ int few_sum_stride(int tokens) { return (tokens * 17 + 3) / 4 * 4; }
};

template <bool FP8, int NT, typename OUT>
__global__ void __launch_bounds__(kFewThreads, 1)
moe_few_second_kernel(const FewArgs a) {
    extern __shared__ __align__(128) unsigned char few_smem[];
    const FewSecondSmem at(a.tokens, a.experts, a.top, FP8, a.room);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
    const int sum_stride = FewSecondSmem::few_sum_stride(a.tokens);
    float *sums = reinterpret_cast<float *>(few_smem + at.sums) + warp * sum_stride, *factor = reinterpret_cast<float *>(few_smem + at.factor);
    int *idx = reinterpret_cast<int *>(few_smem + at.idx);
    const FewLists lists = at.lists.lists(few_smem);
    at.lists.clear(few_smem);
    for (int i = lane; i < sum_stride; i += 32) sums[i] = 0.f;
    tl::griddep_wait();
    tl::griddep_launch();
    const int pairs = a.tokens * a.top;
    if (tid < pairs) idx[tid] = tl::ld_cg(a.idx + tid), factor[tid] = tl::ld_cg(a.gate + tid);
    __syncthreads();
    few_lists(a, idx, lists);
    const int count = *lists.count;

    const int col0 = (int)((long long)a.dim * blockIdx.x / gridDim.x), col1 = (int)((long long)a.dim * (blockIdx.x + 1) / gridDim.x);
    const int blocks_out = (a.bytes_out + 127) / 128, scale_cols = (a.ff + 127) / 128, scale_rows = (a.dim + 127) / 128;
    for (int c0 = col0; c0 < col1; c0 += 16) {
        const int here = min(16, col1 - c0);
        const int turn_row = 128 - (c0 & 127);  // rows from here on have the next block's scales
        // an expert's block b goes to warp (expert * blocks + b) % 16, whichever experts are chosen beside it
        struct Step {
            int pos, b;
        };
        auto enter = [&](Step &s) {
            while (s.pos < count) {
                s.b = (warp - lists.active[s.pos] * blocks_out) & (kFewWarps - 1);
                if (s.b < blocks_out) return;
                ++s.pos;
            }
        };
        auto next = [&](Step &s) {
            s.b += kFewWarps;
            if (s.b >= blocks_out) ++s.pos, enter(s);
        };
        Step now{0, 0}, ahead{0, 0};
        enter(now), enter(ahead);
        FewQueue queue(few_smem, at.queue, at.depth, warp);
        const size_t four = (size_t)4 * a.ld_out;
        const uint8_t *lane_w = a.w2 + ((size_t)c0 + (lane >> 3)) * a.ld_out + (lane & 7) * 16;
        const float *lane_s = FP8 ? a.s2 + (size_t)min((c0 >> 7) + lane, scale_rows - 1) * scale_cols : nullptr;  // lanes 0 and 1: of this block and the next
        auto issue = [&] {
            if (ahead.pos < count) {
                const int e = lists.active[ahead.pos];
                const uint8_t *low = lane_w + (size_t)e * a.dim * a.ld_out + ahead.b * 128;
                const int left = ahead.b * 128 + (lane & 7) * 16 < a.bytes_out ? here - (lane >> 3) : 0;
                queue.copy(low, low + 2 * four, four, left > 0, left > 4, left > 8, left > 12);
                if (FP8 && lane < 2) queue.copy_scale(lane_s + (size_t)e * scale_rows * scale_cols + ahead.b);
                next(ahead);
            }
            queue.asked();
        };
        for (int i = 0; i < at.depth; ++i) issue();
        constexpr int ENTRIES = FP8 ? 16 : 8;  // of either half of a block, a lane's
        float h[2][ENTRIES];
        auto fetch = [&](const Step &s, int n) {  // a column's inner numbers; of a column that is not there: zeros
            const bool mine = n * 8 + g < __popc(lists.tokens[s.pos]);
            const int c = mine ? lists.column[s.pos * 32 + n * 8 + g] : 0;
            const float *row = a.inner + ((size_t)(c >> 8) * a.top + (c & 255)) * a.ld_inner;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int k = s.b * 8 * ENTRIES + u * 4 * ENTRIES + t4 * ENTRIES;
#pragma unroll
                for (int i = 0; i < ENTRIES; i += 4) {
                    uint4 v = make_uint4(0, 0, 0, 0);
                    if (mine && k < a.ld_inner) v = tl::ld_cg(reinterpret_cast<const uint4 *>(row + k + i));
                    h[u][i] = __uint_as_float(v.x), h[u][i + 1] = __uint_as_float(v.y), h[u][i + 2] = __uint_as_float(v.z), h[u][i + 3] = __uint_as_float(v.w);
                }
            }
        };
        if (now.pos < count) fetch(now, 0);
        while (now.pos < count) {
            const FewPiece p = queue.next<FP8>();
            const float scale_a = FP8 && g < turn_row ? p.scale.x : p.scale.y, scale_b = FP8 && g + 8 < turn_row ? p.scale.x : p.scale.y;
            const int columns = __popc(lists.tokens[now.pos]);
            const uint16_t *column = lists.column + now.pos * 32;
            Step later = now;
            next(later);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                if (n * 8 >= columns) break;
                if (n > 0) fetch(now, n);
                constexpr int TERMS = FP8 ? 1 : 2, WORDS = FP8 ? 8 : 4;
                uint32_t x[2][TERMS][WORDS];
                float down = 1.f;
                int e = 0;
                if constexpr (FP8) {  // a power of two for a column's 128 numbers of this block, which the block's promotion takes back
                    uint32_t most = 0;
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int i = 0; i < ENTRIES; ++i) most = max(most, __float_as_uint(h[u][i]) & 0x7fffffffu);
                    most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
                    most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
                    e = few_exponent(__uint_as_float(most)), down = few_exp2(-e);
                }
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int i = 0; i < WORDS; ++i) {
                        const float lo = h[u][2 * i], hi = h[u][2 * i + 1];
                        if constexpr (FP8) {
                            x[u][0][i] = few_half2(lo * down, hi * down);
                        } else {
                            x[u][0][i] = tl::pack2<bf16>(lo, hi);
                            const float2 f = tl::unpack2<bf16>(x[u][0][i]);
                            // an infinity has no second term
                            x[u][1][i] = tl::pack2<bf16>(fabsf(f.x) < INFINITY ? lo - f.x : 0.f, fabsf(f.y) < INFINITY ? hi - f.y : 0.f);
                        }
                    }
                if (n == 0 && columns <= 8 && later.pos < count) fetch(later, 0);  // on its way under the products
                float d[2][4] = {};
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int term = 0; term < TERMS; ++term) few_half<FP8>(p.a[u], p.b[u], x[u][term], d[u]);
#pragma unroll
                for (int v = 0; v < 2; ++v) {
                    const int col = n * 8 + 2 * t4 + v;
                    const int up = FP8 ? __shfl_sync(0xffffffffu, e, (2 * t4 + v) * 4) : 0;
                    if (col < columns) {
                        const int t = column[col] >> 8;
                        const float f = factor[t * a.top + (column[col] & 255)] * few_exp2(up);
                        float *to = sums + t * 17 + g;
                        to[0] = fmaf(d[0][v] + d[1][v], FP8 ? f * scale_a : f, to[0]), to[8] = fmaf(d[0][2 + v] + d[1][2 + v], FP8 ? f * scale_b : f, to[8]);
                    }
                }
            }
            __syncwarp();  // the next expert's column of a token may be another lane's
            if (columns > 8 && later.pos < count) fetch(later, 0);
            now = later;
            issue();
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncthreads();
        const float *all = reinterpret_cast<const float *>(few_smem + at.sums);
        for (int i = tid; i < 16 * a.tokens; i += kFewThreads) {
            const int r = i % 16, t = i / 16;
            if (r >= here) continue;
            float y = 0.f;
#pragma unroll
            for (int w = 0; w < kFewWarps; ++w) y += all[w * sum_stride + t * 17 + r];
            const int d = c0 + r;
            for (int k = 0; k < a.top; ++k) {
                const int e = idx[t * a.top + k];
                if (e < a.experts) continue;
                // an identity expert; no output at all: the token's logits are no numbers
                y = e < a.outputs ? fmaf(factor[t * a.top + k], to_f(tl::ld_cg(a.x + (size_t)t * a.dim + d)), y) : __int_as_float(0x7fffffff);
            }
            if (a.shared) y = fmaf(a.side_w ? tl::ld_cg(a.side + t) : 1.f, to_f(tl::ld_cg(a.shared + (size_t)t * a.dim + d)), y);
            static_cast<OUT *>(a.out)[(size_t)t * a.dim + d] = from_f<OUT>(y);
        }
        if (c0 + 16 < col1) {
            __syncthreads();
            for (int i = lane; i < sum_stride; i += 32) sums[i] = 0.f;
            __syncwarp();
        }
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------

constexpr int kFewSmem = 227 * 1024, kFewMostGrid = 1024;

// CTAs of the first launch: as many clusters as are resident at once, which a device's SMs in groups decide (132 CTAs of a B200; in pairs all 148 are, but then
// every CTA reads half of the router's rows: 1 token of the benchmark's experts 30.2 us in 8 bits against 28.6, 32 tokens 183 and 184).
template <typename K>
static int few_grid(K kernel, int smem) {
    static std::atomic<int> known[64];
    int device = 0;
    cudaGetDevice(&device);
    if (device >= 0 && device < 64 && known[device].load(std::memory_order_acquire) > 0) return known[device].load(std::memory_order_relaxed);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(kFewCluster), cfg.blockDim = dim3(kFewThreads), cfg.dynamicSmemBytes = smem;
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

// Two places of the queue at least: a piece on its way while one is used.
static bool few_fits(const FewFirstSmem &s) { return s.depth >= 2 && s.total <= kFewSmem; }
constexpr int kFewPrefetch = 40 << 20;  // a third of L2

static int few_inner_ld(int ff) { return (ff + 15) / 16 * 16; }
static int few_nt(int tokens) { return tokens <= 8 ? 1 : tokens <= 16 ? 2 : 4; }

static size_t few_align(size_t n) { return (n + 15) & ~(size_t)15; }
static size_t few_bytes(int tokens, int top, int ff) {
    const size_t pairs = (size_t)tokens * top;
    return few_align(pairs * 4) * 2 + few_align((size_t)tokens * 4) + pairs * few_inner_ld(ff) * 4;
}

template <typename K>
static int few_ready(K kernel, tl::PerDevice &ready) {
    int device = 0;
    cudaGetDevice(&device);
    if (ready(device, [&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kFewSmem) == cudaSuccess; })) return TL_OK;
    cudaGetLastError();
    return tl::fail(TL_ECUDA, "moe_few: no shared memory");
}
template <typename K>
static int few_launch(K kernel, dim3 grid, int cluster, int smem, cudaStream_t st, const FewArgs &a) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid, cfg.blockDim = dim3(kFewThreads), cfg.dynamicSmemBytes = smem, cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr, cfg.numAttrs = tl::use_pdl() ? 2 : 1;
    cudaLaunchKernelEx(&cfg, kernel, a);
    TL_LAUNCH_CHECK("moe_few");
    return TL_OK;
}

template <typename K>
static int few_first(K kernel, tl::PerDevice &ready, int smem, cudaStream_t st, FewArgs &a) {
    if (int e = few_ready(kernel, ready)) return e;
    const int grid = few_grid(kernel, kFewSmem);
    a.runs = grid * kFewTeams, a.prefetch = kFewPrefetch / grid;
    return few_launch(kernel, dim3(grid), kFewCluster, smem, st, a);
}
template <typename K>
static int few_second(K kernel, tl::PerDevice &ready, int smem, cudaStream_t st, const FewArgs &a) {
    if (int e = few_ready(kernel, ready)) return e;
    return few_launch(kernel, dim3(std::min(sm_count(), a.dim)), 1, smem, st, a);
}
template <bool FP8, int NT>
static int few_run(FewArgs &a, int first_smem, bool wide, cudaStream_t st) {
    static tl::PerDevice gated, plain, second16, second32;
    if (int e = a.w1 ? few_first(moe_few_first_kernel<FP8, true, NT>, gated, first_smem, st, a) : few_first(moe_few_first_kernel<FP8, false, NT>, plain, first_smem, st, a)) return e;
    const int smem = FewSecondSmem(a.tokens, a.experts, a.top, FP8, kFewSmem).total;
    return wide ? few_second(moe_few_second_kernel<FP8, NT, float>, second32, smem, st, a) : few_second(moe_few_second_kernel<FP8, NT, bf16>, second16, smem, st, a);
}

}  // namespace tlb

using namespace tlb;

extern "C" {

int tlb_moe_few_tokens(int dim, int outputs, int experts, int top, int group_count, int fp8) {
    if (dim <= 0 || outputs <= 0 || outputs > kFewOutputs || experts <= 0 || experts > outputs || top <= 0 || top > outputs || top > 255 || group_count < 0) return 0;
    int tokens = std::min(kFewTokens, kFewPairs / top);
    while (tokens > 0 && !few_fits(FewFirstSmem(tokens, few_nt(tokens), dim, outputs, experts, top, group_count, fp8 != 0, kFewSmem))) --tokens;
    return tokens;
}

size_t tlb_moe_few_workspace(int tokens, int top, int experts, int ff) {
    return tokens <= 0 || top <= 0 || experts <= 0 || ff <= 0 ? 0 : few_bytes(tokens, top, ff);
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
    if (workspace_bytes < few_bytes(tokens, top, ff)) return tl::fail(TL_EINVAL, "moe_few: workspace too small");
    const size_t pairs = (size_t)tokens * top;
    FewArgs a{};
    a.x = (const bf16 *)x, a.router = (const bf16 *)l->router, a.router_bias = (const bf16 *)l->router_bias, a.choice_bias = (const bf16 *)l->choice_bias;
    a.side_w = (const bf16 *)l->side_w, a.tokens = tokens, a.dim = dim, a.outputs = outputs, a.experts = experts, a.top = top, a.scoring = l->scoring, a.group_count = groups;
    a.group_keep = l->group_keep, a.weight_scale = l->weight_scale;
    a.w0 = (const uint8_t *)(l->w_gate ? l->w_gate : l->w_up), a.w1 = (const uint8_t *)(l->w_gate ? l->w_up : nullptr), a.w2 = (const uint8_t *)l->w_down;
    a.s0 = l->w_gate ? l->s_gate : l->s_up, a.s1 = l->w_gate ? l->s_up : nullptr, a.s2 = l->s_down;
    a.ff = ff, a.ld_in = l->ld_in, a.ld_out = l->ld_out, a.bytes_in = (int)few_align((size_t)dim * size), a.bytes_out = (int)few_align((size_t)ff * size);
    a.act = l->act, a.limit = l->limit, a.slope = l->slope, a.shared = (const bf16 *)shared, a.out = out;
    uint8_t *at = (uint8_t *)workspace;
    a.idx = (int32_t *)at, at += few_align(pairs * 4);
    a.gate = (float *)at, at += few_align(pairs * 4);
    a.side = (float *)at, at += few_align((size_t)tokens * 4);
    a.inner = (float *)at, a.ld_inner = few_inner_ld(ff), a.room = kFewSmem;
    const int nt = few_nt(tokens), smem = FewFirstSmem(tokens, nt, dim, outputs, experts, top, groups, fp8 != 0, kFewSmem).total;
    const cudaStream_t st = as_stream(stream);
    if (fp8) return nt == 1 ? few_run<true, 1>(a, smem, out_f32, st) : nt == 2 ? few_run<true, 2>(a, smem, out_f32, st) : few_run<true, 4>(a, smem, out_f32, st);
    return nt == 1 ? few_run<false, 1>(a, smem, out_f32, st) : nt == 2 ? few_run<false, 2>(a, smem, out_f32, st) : few_run<false, 4>(a, smem, out_f32, st);
}

}  // extern "C"
