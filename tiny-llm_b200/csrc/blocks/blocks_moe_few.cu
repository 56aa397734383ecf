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
// e4m3 numbers become fp16 exactly; then x (a power of two for each token) and the inner rows (a power of two for each pair, from the largest
// magnitude that the first launch leaves) are fp16 as well, off by 2^-11 of the value or 2^-24 of the row's largest (x's own numbers of 8 bits only by the latter).  bf16
// numbers meet bf16 ones: x is as it came, and an inner row is two bf16 terms, off by 2^-16.  Sums are fp32 throughout; with 8 bits the 128 of a block are added before their scale multiplies them.
//
// No CTA waits for another outside its cluster: the cluster's CTAs share the router's rows, exchange the logits through shared memory, and every
// CTA makes the same choices for itself.  The second launch reads the choices and the inner rows behind the wait for the first.
#include <cuda_fp16.h>
#include <cuda_fp8.h>

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
    float *most;       // e4m3: [(run of features) + (position of the expert)][32], the largest magnitude of a token's inner row in that run
    int ld_inner, runs;  // runs of features: teams of the first launch
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

// A warp's piece of 16 rows: 128 bytes of each.  A lane has rows g = lane / 4 and g + 8, 16 bytes at t * 16 (t = lane % 4) of either half.
struct FewPiece {
    uint4 a[2], b[2];  // rows g, g + 8
    float sa, sb;      // their scales
};
template <bool FP8>
__device__ __forceinline__ void few_load(FewPiece &p, const uint8_t *row_a, const uint8_t *row_b, int at, int bytes) {
    const uint4 none = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        const int o = at + c * 64;
        p.a[c] = row_a && o < bytes ? few_ldg(row_a + o) : none;
        p.b[c] = row_b && o < bytes ? few_ldg(row_b + o) : none;
    }
}
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

// The chosen experts in ascending order and which choice of theirs a token has: both launches make these for themselves.
struct FewLists {
    int *active;      // [kFewPairs]
    uint8_t *choice;  // [kFewPairs][32]: choice + 1 of a token, 0: not chosen
    int *count;
};
// All threads of the CTA; place [experts] is scratch.  idx: the choices, in shared memory.
__device__ __forceinline__ void few_lists(const FewArgs &a, const int *idx, short *place, const FewLists &l) {
    const int tid = threadIdx.x, lane = tid & 31;
    for (int e = tid; e < a.experts; e += kFewThreads) place[e] = -1;
    for (int i = tid; i < min(a.experts, a.tokens * a.top) * 8; i += kFewThreads) reinterpret_cast<uint32_t *>(l.choice)[i] = 0;
    __syncthreads();
    for (int p = tid; p < a.tokens * a.top; p += kFewThreads)
        if (idx[p] < a.experts) place[idx[p]] = 0;
    __syncthreads();
    if (tid < 32) {
        int n = 0;
        for (int e0 = 0; e0 < a.experts; e0 += 32) {
            const int e = e0 + lane;
            const bool here = e < a.experts && place[e] == 0;
            const uint32_t all = __ballot_sync(0xffffffffu, here);
            if (here) {
                const int at = n + __popc(all & ((1u << lane) - 1));
                l.active[at] = e, place[e] = (short)at;
            }
            n += __popc(all);
        }
        if (lane == 0) *l.count = n;
    }
    __syncthreads();
    if (tid < a.tokens)  // a token that names an expert twice (equal logits of minus infinity) has it once, by its first choice
        for (int k = 0; k < a.top; ++k) {
            const int e = idx[tid * a.top + k];
            if (e < a.experts) {
                uint8_t &c = l.choice[place[e] * 32 + tid];
                if (c == 0) c = (uint8_t)(k + 1);
            }
        }
    __syncthreads();
}

// Features 0 .. total - 1 in `runs` runs that differ by one at most.
__device__ __forceinline__ int few_run_start(int total, int runs, int v) { return v * (total / runs) + min(v, total % runs); }
__device__ __forceinline__ int few_run_of(int total, int runs, int f) {
    const int q = total / runs, r = total % runs;
    return f < r * (q + 1) ? f / (q + 1) : r + (f - r * (q + 1)) / q;
}

// ---- first launch ----------------------------------------------------------------------------------------------------

static inline __host__ __device__ int few_x_stride(int dim, bool fp8) {  // bytes of a token's row in shared memory: its 16-byte reads meet no bank conflict
    return (dim + 127) / 128 * 256 + (fp8 ? 16 : 64);
}
struct FewFirstSmem {
    int x, red, logits, times, idx, gate, active, choice, place, flags, total;
    __host__ __device__ FewFirstSmem(int tokens, int nt, int dim, int outputs, int experts, int top, int groups, bool fp8) {
        x = 0;
        red = x + nt * 8 * few_x_stride(dim, fp8);
        const int sums = kFewWarps * 16 * nt * 8 * 4;  // the teams' sums, or the router's
        logits = red + sums;
        const int per_token = 2 * outputs + groups;
        times = logits + (tokens * per_token * 4 + tokens * 4 + 15) / 16 * 16;
        idx = times + nt * 8 * 4;
        gate = idx + tokens * top * 4;
        active = gate + tokens * top * 4;
        const int most = tokens * top < experts ? tokens * top : experts;
        choice = active + (most * 4 + 15) / 16 * 16;
        place = choice + most * 32;
        flags = (place + experts * 2 + 15) / 16 * 16;
        total = flags + 16;
    }
};

template <bool FP8, bool GATED, int NT>
__global__ void __launch_bounds__(kFewThreads, 1)
moe_few_first_kernel(const FewArgs a) {
    extern __shared__ __align__(128) unsigned char few_smem[];
    const FewFirstSmem at(a.tokens, NT, a.dim, a.outputs, a.experts, a.top, a.group_count, FP8);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
    const int stride = few_x_stride(a.dim, FP8);
    uint32_t rank, ranks;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
    float *red = reinterpret_cast<float *>(few_smem + at.red), *logits = reinterpret_cast<float *>(few_smem + at.logits);
    const int per_token = 2 * a.outputs + a.group_count;
    float *side = logits + a.tokens * per_token;
    int *idx = reinterpret_cast<int *>(few_smem + at.idx);
    float *gate = reinterpret_cast<float *>(few_smem + at.gate);

    tl::griddep_wait();
    // the tokens' rows, zero behind the last entry and the last token
    for (int i = tid; i < NT * 8 * (stride / 16); i += kFewThreads) {
        const int t = i / (stride / 16), d = i % (stride / 16) * 8;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (t < a.tokens && d < a.dim) v = tl::ld_cg(reinterpret_cast<const uint4 *>(a.x + (size_t)t * a.dim + d));
        *reinterpret_cast<uint4 *>(few_smem + t * stride + d * 2) = v;
    }
    // The cluster's CTAs are known to run: their shared memory may be written.
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");

    // ---- the router: 16 rows at a time, a CTA of the cluster every ranks-th of them, the reduction dealt to the 16 warps
    const int rows = a.outputs + (a.side_w ? 1 : 0), pieces = (a.dim * 2 + 127) / 128;
    for (int m = rank; m * 16 < rows; m += ranks) {
        float acc[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
        auto row_of = [&](int r) -> const uint8_t * {
            return reinterpret_cast<const uint8_t *>(r < a.outputs ? a.router + (size_t)r * a.dim : r < rows ? a.side_w : nullptr);
        };
        const uint8_t *ra = row_of(m * 16 + g), *rb = row_of(m * 16 + g + 8);
        for (int s = warp; s < pieces; s += 2 * kFewWarps) {
            FewPiece p[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) few_load<false>(p[u], ra, rb, (s + u * kFewWarps) * 128 + t4 * 16, a.dim * 2);
#pragma unroll
            for (int u = 0; u < 2; ++u)
                if (s + u * kFewWarps < pieces)
#pragma unroll
                    for (int c = 0; c < 2; ++c)
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            const uint4 v = *reinterpret_cast<const uint4 *>(few_smem + (n * 8 + g) * stride + (s + u * kFewWarps) * 128 + c * 64 + t4 * 16);
                            const uint32_t x[4] = {v.x, v.y, v.z, v.w};
                            few_half<false>(p[u].a[c], p[u].b[c], x, acc[n]);
                        }
        }
        float *mine = red + warp * 16 * NT * 8;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            *reinterpret_cast<float2 *>(mine + g * NT * 8 + n * 8 + 2 * t4) = make_float2(acc[n][0], acc[n][1]);
            *reinterpret_cast<float2 *>(mine + (g + 8) * NT * 8 + n * 8 + 2 * t4) = make_float2(acc[n][2], acc[n][3]);
        }
        __syncthreads();
        for (int i = tid; i < 16 * NT * 8; i += kFewThreads) {
            const int r = m * 16 + i / (NT * 8), t = i % (NT * 8);
            if (r >= rows || t >= a.tokens) continue;
            float z = 0.f;
#pragma unroll
            for (int w = 0; w < kFewWarps; ++w) z += red[w * 16 * NT * 8 + i];
            if (r < a.outputs && a.router_bias) z += to_f(a.router_bias[r]);
            const uint32_t to = static_cast<uint32_t>(__cvta_generic_to_shared(r < a.outputs ? logits + t * per_token + r : side + t));
            for (uint32_t c = 0; c < ranks; ++c)
                asm volatile("{\n\t.reg .b32 ra;\n\tmapa.shared::cluster.u32 ra, %0, %1;\n\tst.shared::cluster.f32 [ra], %2;\n\t}" ::"r"(to), "r"(c), "f"(z) : "memory");
        }
        __syncthreads();
    }
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");

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
    int *count = reinterpret_cast<int *>(few_smem + at.flags);
    const FewLists lists{reinterpret_cast<int *>(few_smem + at.active), few_smem + at.choice, count};
    few_lists(a, idx, reinterpret_cast<short *>(few_smem + at.place), lists);

    // ---- with 8 bits: the rows as fp16 times a power of two
    float *times = reinterpret_cast<float *>(few_smem + at.times);
    if constexpr (FP8) {
        for (int t = warp; t < NT * 8; t += kFewWarps) {
            float most = 0.f;
            const int entries = (a.dim + 127) / 128 * 128;
            for (int d = lane * 8; d < entries; d += 256) {
                const uint4 u = *reinterpret_cast<const uint4 *>(few_smem + t * stride + d * 2);
                const uint32_t c[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 f = tl::unpack2<bf16>(c[i]);
                    most = fmaxf(most, fmaxf(fabsf(f.x), fabsf(f.y)));
                }
            }
            const int e = few_exponent(warp_max(most));
            const float down = few_exp2(-e);
            for (int d = lane * 8; d < entries; d += 256) {
                uint4 *p = reinterpret_cast<uint4 *>(few_smem + t * stride + d * 2);
                const uint4 u = *p;
                const uint32_t c[4] = {u.x, u.y, u.z, u.w};
                uint32_t o[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 f = tl::unpack2<bf16>(c[i]);
                    o[i] = few_half2(f.x * down, f.y * down);
                }
                *p = make_uint4(o[0], o[1], o[2], o[3]);
            }
            if (lane == 0) times[t] = few_exp2(e);
        }
        __syncthreads();
    }

    // ---- the first products: a team takes its run of the chosen experts' features, up to 8 (with a gate; else 16) of one expert at a time
    constexpr int TILE = GATED ? 8 : 16;
    const int team = warp / kFewTeam, sub = warp % kFewTeam, run = blockIdx.x * kFewTeams + team, total = *count * a.ff;
    const int blocks_in = (a.bytes_in + 127) / 128, iters = (blocks_in + kFewTeam - 1) / kFewTeam;
    const int scale_cols = (a.dim + 127) / 128, scale_rows = (a.ff + 127) / 128;
    struct Tile {
        int pos, row, here, left;
    };
    auto cut = [&](Tile &s) { s.here = min(min(TILE, a.ff - s.row), s.left); };
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
    Tile ahead = tile;
    int ahead_it = 0;
    auto issue = [&](FewPiece &p) {
        if (ahead.left <= 0) return;
        const int e = lists.active[ahead.pos], b = sub + ahead_it * kFewTeam;
        const size_t r0 = (size_t)e * a.ff + ahead.row;
        const int second = GATED ? g : g + 8;
        const bool va = g < ahead.here && b < blocks_in, vb = second < ahead.here && b < blocks_in;
        few_load<FP8>(p, va ? a.w0 + (r0 + g) * a.ld_in : nullptr, vb ? (GATED ? a.w1 : a.w0) + (r0 + second) * a.ld_in : nullptr, b * 128 + t4 * 16, a.bytes_in);
        if constexpr (FP8) {
            const size_t s0 = (size_t)e * scale_rows;
            p.sa = va ? __ldg(a.s0 + (s0 + (ahead.row + g) / 128) * scale_cols + b) : 0.f;
            p.sb = vb ? __ldg((GATED ? a.s1 : a.s0) + (s0 + (ahead.row + second) / 128) * scale_cols + b) : 0.f;
        }
        if (++ahead_it == iters) ahead_it = 0, advance(ahead);
    };
    float acc[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
    int it = 0;
    float largest[NT > 2 ? 2 : 1] = {};
    float *team_red = red + team * kFewTeam * 16 * NT * 8;
    auto report = [&](int pos) {  // the run's share of this expert ends
        const int i = sub * 32 + lane;
        if constexpr (FP8) {
#pragma unroll
            for (int h = 0; h < (NT > 2 ? 2 : 1); ++h) {
                const int col = (i >> 3) + 16 * h;
                if ((i & 7) == 0 && col < NT * 8) a.most[(size_t)(run + pos) * 32 + col] = largest[h];
                largest[h] = 0.f;
            }
        }
    };
    auto finish = [&] {  // the tile's sums over the team's warps, the activation, the inner rows
        float *mine = team_red + sub * 16 * NT * 8;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            *reinterpret_cast<float2 *>(mine + g * NT * 8 + n * 8 + 2 * t4) = make_float2(acc[n][0], acc[n][1]);
            *reinterpret_cast<float2 *>(mine + (g + 8) * NT * 8 + n * 8 + 2 * t4) = make_float2(acc[n][2], acc[n][3]);
            acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
        }
        asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "n"(kFewTeam * 32) : "memory");
        const int i = sub * 32 + lane;
#pragma unroll
        for (int h = 0; h < (NT > 2 ? 2 : 1); ++h) {
            const int f = i & 7, col = (i >> 3) + 16 * h;
            if (col < NT * 8) {
                const int c = lists.choice[tile.pos * 32 + col];
                float v[2] = {};
                for (int w = 0; w < kFewTeam; ++w) v[0] += team_red[w * 16 * NT * 8 + f * NT * 8 + col], v[1] += team_red[w * 16 * NT * 8 + (f + 8) * NT * 8 + col];
                if constexpr (FP8) v[0] *= times[col], v[1] *= times[col];
                float most = 0.f;
                if (c) {
                    float *to = a.inner + ((size_t)col * a.top + c - 1) * a.ld_inner + tile.row;
                    if constexpr (GATED) {
                        if (f < tile.here) {
                            const float y = gated_pair(v[0], v[1], a.act, a.limit, a.slope);
                            to[f] = y, most = fabsf(y);
                        }
                    } else {
#pragma unroll
                        for (int u = 0; u < 2; ++u)
                            if (f + 8 * u < tile.here) {
                                const float y = a.act == 2 ? (v[u] > 0.f ? v[u] * v[u] : v[u] == v[u] ? 0.f : v[u]) : act_apply(v[u], a.act);
                                to[f + 8 * u] = y, most = most < fabsf(y) || y != y ? fabsf(y) : most;
                            }
                    }
                    if (tile.row + tile.here == a.ff)
                        for (int z = a.ff + f; z < a.ld_inner; z += 8) to[z - tile.row] = 0.f;
                }
                if constexpr (FP8) {
#pragma unroll
                    for (int o = 1; o < 8; o <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
                    largest[h] = fmaxf(largest[h], most);
                }
            }
        }
        const int pos = tile.pos;
        advance(tile);
        if (tile.left <= 0 || tile.pos != pos) report(pos);
        asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "n"(kFewTeam * 32) : "memory");
    };
    auto consume = [&](FewPiece &p) -> bool {
        if (tile.left <= 0) return false;
        const int b = sub + it * kFewTeam;
        if (b < blocks_in) {
            float d[NT][4];
            if constexpr (FP8) {
#pragma unroll
                for (int n = 0; n < NT; ++n) d[n][0] = d[n][1] = d[n][2] = d[n][3] = 0.f;
            }
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const unsigned char *row = few_smem + (n * 8 + g) * stride;
                    if constexpr (FP8) {
                        const uint4 u = *reinterpret_cast<const uint4 *>(row + b * 256 + c * 128 + t4 * 32), v = *reinterpret_cast<const uint4 *>(row + b * 256 + c * 128 + t4 * 32 + 16);
                        const uint32_t x[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
                        few_half<true>(p.a[c], p.b[c], x, d[n]);
                    } else {
                        const uint4 u = *reinterpret_cast<const uint4 *>(row + b * 128 + c * 64 + t4 * 16);
                        const uint32_t x[4] = {u.x, u.y, u.z, u.w};
                        few_half<false>(p.a[c], p.b[c], x, acc[n]);
                    }
                }
            if constexpr (FP8) {
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    acc[n][0] = fmaf(d[n][0], p.sa, acc[n][0]), acc[n][1] = fmaf(d[n][1], p.sa, acc[n][1]);
                    acc[n][2] = fmaf(d[n][2], p.sb, acc[n][2]), acc[n][3] = fmaf(d[n][3], p.sb, acc[n][3]);
                }
            }
        }
        issue(p);
        if (++it == iters) it = 0, finish();
        return true;
    };
    FewPiece p0, p1, p2;
    issue(p0), issue(p1), issue(p2);
    while (consume(p0) && consume(p1) && consume(p2)) {}
    tl::griddep_launch();
}

// ---- second launch ---------------------------------------------------------------------------------------------------

struct FewSecondSmem {
    int red, idx, factor, times, active, choice, place, flags, total;
    __host__ __device__ FewSecondSmem(int tokens, int nt, int experts, int top) {
        red = 0;
        idx = red + kFewWarps * 16 * nt * 8 * 4;
        factor = idx + tokens * top * 4;
        times = factor + tokens * top * 4;
        active = times + tokens * top * 4;
        const int most = tokens * top < experts ? tokens * top : experts;
        choice = active + (most * 4 + 15) / 16 * 16;
        place = choice + most * 32;
        flags = (place + experts * 2 + 15) / 16 * 16;
        total = flags + 16;
    }
};

template <bool FP8, int NT, typename OUT>
__global__ void __launch_bounds__(kFewThreads, 1)
moe_few_second_kernel(const FewArgs a) {
    extern __shared__ __align__(128) unsigned char few_smem[];
    const FewSecondSmem at(a.tokens, NT, a.experts, a.top);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
    float *red = reinterpret_cast<float *>(few_smem + at.red), *factor = reinterpret_cast<float *>(few_smem + at.factor), *times = reinterpret_cast<float *>(few_smem + at.times);
    int *idx = reinterpret_cast<int *>(few_smem + at.idx), *count = reinterpret_cast<int *>(few_smem + at.flags);
    const FewLists lists{reinterpret_cast<int *>(few_smem + at.active), few_smem + at.choice, count};
    tl::griddep_wait();
    tl::griddep_launch();
    for (int p = tid; p < a.tokens * a.top; p += kFewThreads) idx[p] = tl::ld_cg(a.idx + p), factor[p] = tl::ld_cg(a.gate + p);
    __syncthreads();
    short *place = reinterpret_cast<short *>(few_smem + at.place);
    few_lists(a, idx, place, lists);
    const int total = *count * a.ff;
    if constexpr (FP8) {  // an inner row's power of two, from what every run of its features left
        for (int p = warp; p < a.tokens * a.top; p += kFewWarps) {
            const int t = p / a.top, e = idx[p];
            if (e >= a.experts) continue;
            const int pos = place[e], f0 = pos * a.ff, v0 = few_run_of(total, a.runs, f0), v1 = few_run_of(total, a.runs, f0 + a.ff - 1);
            float most = 0.f;
            for (int v = v0 + lane; v <= v1; v += 32) {
                const float m = tl::ld_cg(a.most + (size_t)(v + pos) * 32 + t);
                most = most < m ? m : most;
            }
            const int x = few_exponent(warp_max(most));
            if (lane == 0) times[p] = few_exp2(-x), factor[p] *= few_exp2(x);
        }
        __syncthreads();
    }

    const int col0 = (int)((long long)a.dim * blockIdx.x / gridDim.x), col1 = (int)((long long)a.dim * (blockIdx.x + 1) / gridDim.x);
    const int blocks_out = (a.bytes_out + 127) / 128, scale_cols = (a.ff + 127) / 128, scale_rows = (a.dim + 127) / 128;
    for (int c0 = col0; c0 < col1; c0 += 16) {
        const int here = min(16, col1 - c0);
        float acc[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
        // an expert's block b goes to warp (expert * blocks + b) % 16, whichever experts are chosen beside it
        struct Step {
            int pos, b;
        };
        auto enter = [&](Step &s) {
            while (s.pos < *count) {
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
        auto issue = [&](FewPiece &p) {
            if (ahead.pos >= *count) return;
            const int e = lists.active[ahead.pos];
            const uint8_t *row = a.w2 + ((size_t)e * a.dim + c0 + g) * a.ld_out;
            const bool va = g < here, vb = g + 8 < here;
            few_load<FP8>(p, va ? row : nullptr, vb ? row + (size_t)8 * a.ld_out : nullptr, ahead.b * 128 + t4 * 16, a.bytes_out);
            if constexpr (FP8) {
                const size_t s0 = (size_t)e * scale_rows;
                p.sa = va ? __ldg(a.s2 + (s0 + (c0 + g) / 128) * scale_cols + ahead.b) : 0.f;
                p.sb = vb ? __ldg(a.s2 + (s0 + (c0 + g + 8) / 128) * scale_cols + ahead.b) : 0.f;
            }
            next(ahead);
        };
        auto consume = [&](FewPiece &p) -> bool {
            if (now.pos >= *count) return false;
            const uint8_t *choice = lists.choice + now.pos * 32;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const int mine = n * 8 + g < a.tokens ? choice[n * 8 + g] : 0;
                if (NT > 1 && !__any_sync(0xffffffffu, mine)) continue;
                const int pair = (n * 8 + g) * a.top + mine - 1;
                const float *row = a.inner + (size_t)(mine ? pair : 0) * a.ld_inner;
                const float down = FP8 && mine ? times[pair] : 1.f;
                float d[4] = {};
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    constexpr int ENTRIES = FP8 ? 16 : 8;
                    const int k = now.b * (FP8 ? 128 : 64) + c * (FP8 ? 64 : 32) + t4 * ENTRIES;
                    float h[ENTRIES] = {};
                    if (mine && k < a.ld_inner) {
#pragma unroll
                        for (int i = 0; i < ENTRIES; i += 4) {
                            const uint4 u = tl::ld_cg(reinterpret_cast<const uint4 *>(row + k + i));
                            h[i] = __uint_as_float(u.x), h[i + 1] = __uint_as_float(u.y), h[i + 2] = __uint_as_float(u.z), h[i + 3] = __uint_as_float(u.w);
                        }
                    }
                    if constexpr (FP8) {
                        uint32_t x[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) x[i] = few_half2(h[2 * i] * down, h[2 * i + 1] * down);
                        few_half<true>(p.a[c], p.b[c], x, d);
                    } else {
                        uint32_t x[4], low[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            x[i] = tl::pack2<bf16>(h[2 * i], h[2 * i + 1]);
                            const float2 f = tl::unpack2<bf16>(x[i]);
                            // an infinity has no second term
                            low[i] = tl::pack2<bf16>(fabsf(f.x) < INFINITY ? h[2 * i] - f.x : 0.f, fabsf(f.y) < INFINITY ? h[2 * i + 1] - f.y : 0.f);
                        }
                        few_half<false>(p.a[c], p.b[c], x, d);
                        few_half<false>(p.a[c], p.b[c], low, d);
                    }
                }
                // a token that did not choose this expert gets nothing of it, not even a product with zero
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const int t = n * 8 + 2 * t4 + u, k = t < a.tokens ? choice[t] : 0;
                    if (k) {
                        const float f = factor[t * a.top + k - 1];
                        acc[n][u] = fmaf(d[u], FP8 ? f * p.sa : f, acc[n][u]);
                        acc[n][2 + u] = fmaf(d[2 + u], FP8 ? f * p.sb : f, acc[n][2 + u]);
                    }
                }
            }
            next(now);
            issue(p);
            return true;
        };
        FewPiece p0, p1, p2;
        issue(p0), issue(p1), issue(p2);
        while (consume(p0) && consume(p1) && consume(p2)) {}

        __syncthreads();  // the sums of the columns before
        float *mine = red + warp * 16 * NT * 8;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            *reinterpret_cast<float2 *>(mine + g * NT * 8 + n * 8 + 2 * t4) = make_float2(acc[n][0], acc[n][1]);
            *reinterpret_cast<float2 *>(mine + (g + 8) * NT * 8 + n * 8 + 2 * t4) = make_float2(acc[n][2], acc[n][3]);
        }
        __syncthreads();
        for (int i = tid; i < 16 * NT * 8; i += kFewThreads) {
            const int r = i % 16, t = i / 16;
            if (r >= here || t >= a.tokens) continue;
            float y = 0.f;
#pragma unroll
            for (int w = 0; w < kFewWarps; ++w) y += red[w * 16 * NT * 8 + r * NT * 8 + t];
            const int d = c0 + r;
            for (int k = 0; k < a.top; ++k) {
                const int e = idx[t * a.top + k];
                if (e < a.experts) continue;
                // an identity expert; no output at all: the token's logits are no numbers
                y = e < a.outputs ? fmaf(factor[t * a.top + k], to_f(a.x[(size_t)t * a.dim + d]), y) : __int_as_float(0x7fffffff);
            }
            if (a.shared) y = fmaf(a.side_w ? tl::ld_cg(a.side + t) : 1.f, to_f(tl::ld_cg(a.shared + (size_t)t * a.dim + d)), y);
            static_cast<OUT *>(a.out)[(size_t)t * a.dim + d] = from_f<OUT>(y);
        }
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------

constexpr int kFewSmem = 227 * 1024;

// CTAs of a cluster, and how many clusters of the first launch are resident at once.
constexpr int kFewCluster = 4;
static int few_grid() {
    const int sms = sm_count();
    return sms / kFewCluster * kFewCluster;
}

static int few_inner_ld(int ff) { return (ff + 15) / 16 * 16; }
static int few_nt(int tokens) { return tokens <= 8 ? 1 : tokens <= 16 ? 2 : 4; }

static size_t few_align(size_t n) { return (n + 15) & ~(size_t)15; }
static size_t few_bytes(int tokens, int top, int experts, int ff) {
    const size_t pairs = (size_t)tokens * top, runs = (size_t)few_grid() * kFewTeams + std::min<size_t>(pairs, experts);
    return few_align(pairs * 4) * 2 + few_align((size_t)tokens * 4) + pairs * few_inner_ld(ff) * 4 + runs * 32 * 4;
}

template <typename K>
static int few_launch(K kernel, tl::PerDevice &ready, dim3 grid, int cluster, int smem, cudaStream_t st, const FewArgs &a) {
    int device = 0;
    cudaGetDevice(&device);
    if (!ready(device, [&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kFewSmem) == cudaSuccess; })) {
        cudaGetLastError();
        return tl::fail(TL_ECUDA, "moe_few: no shared memory");
    }
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

template <bool FP8, int NT>
static int few_run(const FewArgs &a, int first_smem, bool wide, cudaStream_t st) {
    static tl::PerDevice gated, plain, second16, second32;
    const int grid = few_grid();
    int e = a.w1 ? few_launch(moe_few_first_kernel<FP8, true, NT>, gated, dim3(grid), kFewCluster, first_smem, st, a)
                 : few_launch(moe_few_first_kernel<FP8, false, NT>, plain, dim3(grid), kFewCluster, first_smem, st, a);
    if (e) return e;
    const int smem = FewSecondSmem(a.tokens, NT, a.experts, a.top).total;
    const dim3 cols(std::min(sm_count(), a.dim));
    return wide ? few_launch(moe_few_second_kernel<FP8, NT, float>, second32, cols, 1, smem, st, a)
                : few_launch(moe_few_second_kernel<FP8, NT, bf16>, second16, cols, 1, smem, st, a);
}

}  // namespace tlb

using namespace tlb;

extern "C" {

int tlb_moe_few_tokens(int dim, int outputs, int experts, int top, int group_count, int fp8) {
    if (dim <= 0 || outputs <= 0 || outputs > kFewOutputs || experts <= 0 || experts > outputs || top <= 0 || top > outputs || top > 255 || group_count < 0) return 0;
    int tokens = std::min(kFewTokens, kFewPairs / top);
    while (tokens > 0 && FewFirstSmem(tokens, few_nt(tokens), dim, outputs, experts, top, group_count, fp8 != 0).total > kFewSmem) --tokens;
    return tokens;
}

size_t tlb_moe_few_workspace(int tokens, int top, int experts, int ff) {
    return tokens <= 0 || top <= 0 || experts <= 0 || ff <= 0 ? 0 : few_bytes(tokens, top, experts, ff);
}

int tlb_moe_few(const void *x, const void *router, const void *router_bias, const void *choice_bias, const void *side_w, int tokens, int dim, int outputs, int experts,
                int top, int scoring, float weight_scale, int group_count, int group_keep, const void *w_gate, const void *w_up, const void *w_down, const float *s_gate,
                const float *s_up, const float *s_down, int fp8, int ff, int ld_in, int ld_out, int act, float limit, float slope, const void *shared, void *out, int out_f32,
                void *workspace, size_t workspace_bytes, void *stream) {
    if (tokens <= 0) return TL_OK;
    if (!x || !router || !w_up || !w_down || !out || !workspace || ff <= 0 || ff > (1 << 20) || scoring < 0 || scoring > 2 || (side_w && !shared))
        return tl::fail(TL_EINVAL, "moe_few: bad argument");
    if (tokens > tlb_moe_few_tokens(dim, outputs, experts, top, group_count, fp8)) return tl::fail(TL_EINVAL, "moe_few: %d tokens are too many for these sizes", tokens);
    if (group_keep < 0 || group_keep > group_count || (group_count > 0 && (outputs % group_count || group_keep * (outputs / group_count) < top)))
        return tl::fail(TL_EINVAL, "moe_few: bad groups");
    if (w_gate ? (act != 0 && act != 1 && act != 3) || (act == 3 && !(limit > 0.f)) : act < 0 || act > 2) return tl::fail(TL_EINVAL, "moe_few: bad activation");
    if (fp8 && (!s_up || !s_down || (w_gate && !s_gate))) return tl::fail(TL_EINVAL, "moe_few: 8-bit weights without scales");
    const int size = fp8 ? 1 : 2;
    if (dim % 8 || ld_in < dim * size || ld_out < ff * size || ld_in % 16 || ld_out % 16 || !tl::aligned16(x) || !tl::aligned16(router) || (side_w && !tl::aligned16(side_w)) ||
        (w_gate && !tl::aligned16(w_gate)) || !tl::aligned16(w_up) || !tl::aligned16(w_down) || !tl::aligned16(workspace))
        return tl::fail(TL_EINVAL, "moe_few: rows must be whole 16-byte pieces");
    if (workspace_bytes < few_bytes(tokens, top, experts, ff)) return tl::fail(TL_EINVAL, "moe_few: workspace too small");
    const size_t pairs = (size_t)tokens * top;
    FewArgs a{};
    a.x = (const bf16 *)x, a.router = (const bf16 *)router, a.router_bias = (const bf16 *)router_bias, a.choice_bias = (const bf16 *)choice_bias, a.side_w = (const bf16 *)side_w;
    a.tokens = tokens, a.dim = dim, a.outputs = outputs, a.experts = experts, a.top = top, a.scoring = scoring, a.group_count = group_count, a.group_keep = group_keep;
    a.weight_scale = weight_scale;
    a.w0 = (const uint8_t *)(w_gate ? w_gate : w_up), a.w1 = (const uint8_t *)(w_gate ? w_up : nullptr), a.w2 = (const uint8_t *)w_down;
    a.s0 = w_gate ? s_gate : s_up, a.s1 = w_gate ? s_up : nullptr, a.s2 = s_down;
    a.ff = ff, a.ld_in = ld_in, a.ld_out = ld_out, a.bytes_in = (int)few_align((size_t)dim * size), a.bytes_out = (int)few_align((size_t)ff * size), a.act = act, a.limit = limit, a.slope = slope, a.shared = (const bf16 *)shared, a.out = out;
    uint8_t *at = (uint8_t *)workspace;
    a.idx = (int32_t *)at, at += few_align(pairs * 4);
    a.gate = (float *)at, at += few_align(pairs * 4);
    a.side = (float *)at, at += few_align((size_t)tokens * 4);
    a.inner = (float *)at, a.ld_inner = few_inner_ld(ff), at += pairs * a.ld_inner * 4;
    a.most = (float *)at, a.runs = few_grid() * kFewTeams;
    const int nt = few_nt(tokens), smem = FewFirstSmem(tokens, nt, dim, outputs, experts, top, group_count, fp8 != 0).total;
    const cudaStream_t st = as_stream(stream);
    if (fp8) return nt == 1 ? few_run<true, 1>(a, smem, out_f32, st) : nt == 2 ? few_run<true, 2>(a, smem, out_f32, st) : few_run<true, 4>(a, smem, out_f32, st);
    return nt == 1 ? few_run<false, 1>(a, smem, out_f32, st) : nt == 2 ? few_run<false, 2>(a, smem, out_f32, st) : few_run<false, 4>(a, smem, out_f32, st);
}

}  // extern "C"
