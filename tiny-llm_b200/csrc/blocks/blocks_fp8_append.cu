// A step's keys and values into pages of 8 bits, with the norm and the rotation that keys and queries pass on the way.
//
// Row x of a head (query or key): x' = x / sqrt(mean(x^2) + eps) * w, then every pair (a, b) of the first `dims` entries turns by the angle
// position * base^(-2i / dims): (a c - b s, b c + a s).  Values stay as they are.  A block is the 16 tokens of a head that share a scale: with m the largest
// magnitude of its new rows, scale = max(2^e, the scale before), e the smallest with m <= 448 * 2^e; the scale before counts if the block holds earlier tokens
// of the sequence, whose numbers are then rounded again to the larger scale.  Scales are powers of two, so that this costs a number nothing
// unless it falls among the smallest ones (below 2^-6 of the scale), and it hardly matters whether tokens come one by one or together.
//
// Keys are made as if in 64 bits and then rounded to fp32: a number is rounded to four significant bits next to borders that the last bits of its fp32 value
// decide.  fp8_append_kernel holds them, and the angles' cosines and sines, as sums of two fp32 numbers (at least 2^-32 of a number): the fp64 units take ten times as long.  Only a position times a frequency, and the whole turns in it, are fp64.  Queries keep their type and are made in 32 bits.
//
// A CTA takes one block of one request and key/value head, with the group's query heads: the angles of its at most 16 tokens are made once, in
// shared memory.  A row goes to 8, 16 or 32 lanes; a lane holds four entries of either half of the rotated part, which are each other's partners, or eight of the
// rest.  Everything is asked for at the start; keys and values stay in registers until the block's largest magnitude is known.
// fp8_append_any_kernel takes what that cannot: rows that do not begin on 16 bytes, rotations of dimensions that are no multiple of 8 (2048 tokens of 32 + 8 heads 59 us for 23).
//
// 1 token of 32 + 8 heads of 128 takes 4.3 us: a launch, length, table, rows and angles, one latency behind another.  128 tokens 6.9, 64 requests of one 6.2.  2048 tokens take 22.9 us (46 MB, 2.0 TB/s):
// instructions, 72 % of the issue slots, of which angles for every key/value head are a fourth.  One set of angles for two or four heads took 115 registers for 64 and 24 us at the best.
#include <math.h>

#include <vector>

#include "../per_device.h"
#include "blocks_fp8_cache.cuh"

namespace tlb {

constexpr int kApThreads = 256;
constexpr int kApMostDim = 256;

constexpr int kApParts = 64;  // of a turn, whose cosines and sines are known

struct F8Turns {
    double of[kApMostDim / 2];  // base^(-2i / dims) / (2 pi): turns a position
    float4 part[kApParts];      // cos and sin of k / 64 turns, as sums of two numbers each
};

struct F8Append : tlb_fp8_append_call {
    tlb_fp8_pages pages;
    int group;
    unsigned group_magic, half_magic;  // for divisions by group and rot / 2
    float under_dim;  // 1 / dim
    float2 root, k_more;  // sqrt(dim) and dim * k_eps, as sums of two numbers
    F8Append(const tlb_fp8_pages &p, const tlb_fp8_append_call &c, int g) : tlb_fp8_append_call(c), pages(p), group(g) {
        auto two = [](double v) { return make_float2(static_cast<float>(v), static_cast<float>(v - static_cast<float>(v))); };
        group_magic = f8_magic(kF8Tokens * static_cast<unsigned long long>(g), g), half_magic = f8_magic(kF8Tokens * kApMostDim / 2, c.rot / 2);
        under_dim = 1.f / p.dim;
        root = two(sqrt(static_cast<double>(p.dim))), k_more = two(static_cast<double>(p.dim) * c.k_eps);
    }
};

__device__ __forceinline__ int2 ap_pair(const F8Append &a, int i) { return a.interleaved ? make_int2(2 * i, 2 * i + 1) : make_int2(i, i + a.rot / 2); }

__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Numbers of earlier tokens rounded to the block's larger scale.
__device__ __forceinline__ void ap_again(uint8_t *rows, int pieces, float ratio) {
    for (int i = threadIdx.x; i < pieces; i += kApThreads) {
        uint4 x = tl::ld_cg(reinterpret_cast<const uint4 *>(rows) + i);
        uint32_t *w = reinterpret_cast<uint32_t *>(&x);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            float f[4];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const __half2_raw two = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w[c] >> (16 * e)), __NV_E4M3);
                const float2 v = __half22float2(__half2(two));
                f[2 * e] = v.x * ratio, f[2 * e + 1] = v.y * ratio;
            }
            w[c] = f8_pack4(f[0], f[1], f[2], f[3]);
        }
        reinterpret_cast<uint4 *>(rows)[i] = x;
    }
}

// A number as the sum of two.
struct ApTwo {
    float h, l;
};
__device__ __forceinline__ ApTwo ap_sum(float a, float b) {  // exactly
    const float s = __fadd_rn(a, b), t = __fsub_rn(s, a);
    return {s, __fadd_rn(__fsub_rn(a, __fsub_rn(s, t)), __fsub_rn(b, t))};
}
__device__ __forceinline__ ApTwo ap_times(ApTwo a, ApTwo b) {
    const float p = __fmul_rn(a.h, b.h);
    return {p, fmaf(a.h, b.l, fmaf(a.l, b.h, fmaf(a.h, b.h, -p)))};
}

// cos and sin of `position` * `of` turns: the nearest 64th of a turn, whose values are known, and a rest r of up to 2^-7 turns, theta = 2 pi r below 0.05:
//   sin = theta + theta (-theta^2 / 6 + theta^4 / 120 - theta^6 / 5040),  cos - 1 = -theta^2 / 2 + theta^4 / 24 - theta^6 / 720   (Taylor; the next terms are below 2^-50)
// (x: cos, y: its rest, z: sin, w: its rest), to 2^-32.
__device__ __forceinline__ float4 ap_angle(int position, double of, const float4 *part) {
    const double t = position * of, f = t - rint(t);
    const float fh = static_cast<float>(f), fl = static_cast<float>(f - fh), k = rintf(fh * kApParts);
    const float rh = fmaf(k, -1.f / kApParts, fh);  // exact: both are near
    constexpr double kTurn = 6.283185307179586;
    const ApTwo th = ap_times({rh, fl}, {static_cast<float>(kTurn), static_cast<float>(kTurn - static_cast<float>(kTurn))});
    const float z = th.h * th.h, zl = fmaf(2.f * th.h, th.l, fmaf(th.h, th.h, -z));
    const float sl = fmaf(th.h, z * fmaf(z, fmaf(z, -1.f / 5040.f, 1.f / 120.f), -1.f / 6.f), th.l);
    const float d = fmaf(-0.5f, zl, z * fmaf(z, fmaf(z, -1.f / 720.f, 1.f / 24.f), -0.5f));
    const float4 p = part[static_cast<int>(k) & (kApParts - 1)];
    const ApTwo u = ap_times({p.z, p.w}, {th.h, sl}), v = ap_times({p.x, p.y}, {th.h, sl});
    const ApTwo c = ap_sum(p.x, -u.h), n = ap_sum(p.z, v.h);
    const ApTwo co = ap_sum(c.h, c.l - u.l + p.y + p.x * d), si = ap_sum(n.h, n.l + v.l + p.w + p.z * d);
    return make_float4(co.h, co.l, si.h, si.l);
}

// A lane's 8 entries of a row: four from a0 on, four from b0 on.  ask: of numbers that the launch in front may have written, through L2.
template <typename T>
struct ApRow;
template <>
struct ApRow<bf16> {
    uint2 a, b;
    __device__ __forceinline__ void load(const bf16 *p, int a0, int b0) { a = *reinterpret_cast<const uint2 *>(p + a0), b = *reinterpret_cast<const uint2 *>(p + b0); }
    __device__ __forceinline__ void ask(const bf16 *p, int a0, int b0) { a = tl::ld_cg(reinterpret_cast<const uint2 *>(p + a0)), b = tl::ld_cg(reinterpret_cast<const uint2 *>(p + b0)); }
    __device__ __forceinline__ void zero() { a = b = make_uint2(0, 0); }
    __device__ __forceinline__ void get(float (&x)[8]) const {
        const uint32_t w[4] = {a.x, a.y, b.x, b.y};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = tl::unpack2<bf16>(w[i]);
            x[2 * i] = f.x, x[2 * i + 1] = f.y;
        }
    }
};
template <>
struct ApRow<float> {
    uint4 a, b;
    __device__ __forceinline__ void load(const float *p, int a0, int b0) { a = *reinterpret_cast<const uint4 *>(p + a0), b = *reinterpret_cast<const uint4 *>(p + b0); }
    __device__ __forceinline__ void ask(const float *p, int a0, int b0) { a = tl::ld_cg(reinterpret_cast<const uint4 *>(p + a0)), b = tl::ld_cg(reinterpret_cast<const uint4 *>(p + b0)); }
    __device__ __forceinline__ void zero() { a = b = make_uint4(0, 0, 0, 0); }
    __device__ __forceinline__ void get(float (&x)[8]) const {
        const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(w[i]);
    }
};

// Where a lane's entries lie, and the pairs that they are: entries e and e + 4 (apart), or 2e and 2e + 1 of the eight.
struct ApPlace {
    int a0, b0, pair;  // pair: a quarter of the number of the first one, -1: not rotated
    bool on, side_by_side;
};
// A token's angles: the first of every four pairs, then the second ones and so on, so that lanes side by side read numbers side by side.
__device__ __forceinline__ int ap_angle_at(int pair, int half) { return (pair & 3) * (half >> 2) + (pair >> 2); }
__device__ __forceinline__ ApPlace ap_place(const F8Append &a, int l) {
    const bool turned = 8 * l < a.rot, halves = turned && !a.interleaved;
    return {halves ? 4 * l : 8 * l, halves ? a.rot / 2 + 4 * l : 8 * l + 4, turned ? l : -1, 8 * l < a.pages.dim, a.interleaved != 0};
}

// Norm and rotation in sums of two fp32 numbers.  Whole warps.  1 / sqrt(mean(x^2) + eps) = sqrt(D) / sqrt(sum(x^2) + D eps).
template <typename T, int LP>
__device__ __forceinline__ void ap_key(const ApRow<T> &row, const F8Append &a, const ApPlace &at, const float4 *turn, float (&y)[8]) {
    float x[8];
    row.get(x);
    ApTwo u[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) u[e] = {x[e], 0.f};
    if (a.k_norm) {
        ApTwo s;
        float2 more = a.k_more;
        // Squares of keys beyond 2^60 or of nothing but numbers (and a root of eps) below 2^-38 would leave fp32's range: such a row is brought nearer to 1 and summed again
#pragma unroll 1
        for (int again = 0;; ++again) {
            s = {0.f, 0.f};
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float q = __fmul_rn(x[e], x[e]);
                const ApTwo t = ap_sum(s.h, q);
                s = {t.h, s.l + t.l + fmaf(x[e], x[e], -q)};
            }
#pragma unroll
            for (int o = 1; o < LP; o <<= 1) {
                const float oh = __shfl_xor_sync(0xffffffffu, s.h, o), ol = __shfl_xor_sync(0xffffffffu, s.l, o);
                const ApTwo t = ap_sum(s.h, oh);
                s = {t.h, s.l + ol + t.l};
            }
            const ApTwo all = ap_sum(s.h, more.x);
            s = {all.h, all.l + s.l + more.y};
            const bool large = !(all.h < 0x1p124f), small = all.h < 0x1p-76f;
            if (again == 2 || !__any_sync(0xffffffffu, large || small)) break;
            const float by = large ? 0x1p-70f : small ? 0x1p64f : 1.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] *= by;
            more.x = more.x * by * by, more.y = more.y * by * by;
        }
        // r0 = 1 / sqrt(s) to 2^-22 or so; 1 - s r0^2 makes it better by as many bits again
        const float r0 = rsqrtf(s.h);
        const ApTwo one = ap_times(ap_times({r0, 0.f}, s), {r0, 0.f});
        const float left = (1.f - one.h) - one.l;
        const ApTwo r = ap_times({r0, 0.5f * r0 * left}, {a.root.x, a.root.y});
        if (at.on) {
            ApRow<T> w;
            float g[8];
            w.load(static_cast<const T *>(a.k_norm), at.a0, at.b0), w.get(g);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float p = x[e] * g[e];  // of two bf16 numbers: all of it
                u[e] = ap_times({p, sizeof(T) == 2 ? 0.f : fmaf(x[e], g[e], -p)}, r);
            }
        }
    }
    if (at.pair < 0) {
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = u[e].h + u[e].l;
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float4 t = turn[e * (a.rot >> 3) + at.pair];
        const ApTwo c{t.x, t.y}, n{t.z, t.w};
        const ApTwo p = at.side_by_side ? u[2 * e] : u[e], q = at.side_by_side ? u[2 * e + 1] : u[e + 4];
        const ApTwo pc = ap_times(p, c), qn = ap_times(q, n), qc = ap_times(q, c), pn = ap_times(p, n);
        const ApTwo f = ap_sum(pc.h, -qn.h), g = ap_sum(qc.h, pn.h);
        const float one = f.h + (f.l + (pc.l - qn.l)), two = g.h + (g.l + (qc.l + pn.l));
        if (at.side_by_side) y[2 * e] = one, y[2 * e + 1] = two;
        else y[e] = one, y[e + 4] = two;
    }
}

// The same in 32 bits.
template <typename T, int LP>
__device__ __forceinline__ void ap_query(const ApRow<T> &row, const F8Append &a, const ApPlace &at, const float (&weight)[8], const float4 *turn, float (&y)[8]) {
    float x[8];
    row.get(x);
    if (a.q_norm) {
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) s = fmaf(x[e], x[e], s);
#pragma unroll
        for (int o = 1; o < LP; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        const float r = rsqrtf(fmaf(s, a.under_dim, a.q_eps));
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] *= r * weight[e];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = x[e];
    if (at.pair < 0) return;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float4 t = turn[e * (a.rot >> 3) + at.pair];
        const float c = t.x, n = t.z, p = at.side_by_side ? x[2 * e] : x[e], q = at.side_by_side ? x[2 * e + 1] : x[e + 4];
        const float one = p * c - q * n, two = q * c + p * n;
        if (at.side_by_side) y[2 * e] = one, y[2 * e + 1] = two;
        else y[e] = one, y[e + 4] = two;
    }
}

template <typename T, int LP>  // lanes of a row
__global__ void __launch_bounds__(kApThreads) fp8_append_kernel(const __grid_constant__ F8Append a, const __grid_constant__ F8Turns turns) {
    constexpr int WARPS = kApThreads / 32, RW = 32 / LP, ROWS = WARPS * RW /* at a time */, PASSES = (kF8Tokens + ROWS - 1) / ROWS, AHEAD = 4;
    extern __shared__ __align__(16) unsigned char sm[];
    float4 *angle = reinterpret_cast<float4 *>(sm);  // [tokens][half]
    __shared__ float4 part[kApParts];
    __shared__ double of[kApMostDim / 2];
    __shared__ float most[2][WARPS];
    // (parameters read at 32 places at once are read one after another: once, then from shared memory)
    if (threadIdx.x < kApParts) part[threadIdx.x] = turns.part[threadIdx.x];
    if (threadIdx.x < a.rot / 2) of[threadIdx.x] = turns.of[threadIdx.x];
    tl::griddep_launch();
    tl::griddep_wait();
    const tlb_fp8_pages &pg = a.pages;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, D = pg.dim, half = a.rot / 2, slot_row = warp * RW + lane / LP;
    const int b = blockIdx.z, h = blockIdx.y, G = a.group;
    const ApPlace at = ap_place(a, lane % LP);
    const int ctx = tl::ld_cg(a.lens + b);
    T *q_out = static_cast<T *>(a.q_out) + (static_cast<size_t>(b) * a.tokens * a.heads + static_cast<size_t>(h) * G) * D;
    // an idle slot (or one whose length does not cover the step) appends nothing; its queries come out as zeros
    if (ctx < a.tokens || static_cast<long long>(ctx) > static_cast<long long>(a.max_pages) * pg.page_size) {
        const int l0 = blockIdx.x * kF8Tokens, n = min(a.tokens - l0, kF8Tokens);
        for (int r = slot_row; r < n * G; r += ROWS)
            if (at.on) {
                T *to = q_out + (static_cast<size_t>(l0 + r / G) * a.heads + r % G) * D;
                store4(to + at.a0, make_float4(0.f, 0.f, 0.f, 0.f)), store4(to + at.b0, make_float4(0.f, 0.f, 0.f, 0.f));
            }
        return;
    }
    const int first = ctx - a.tokens, start = (first / kF8Tokens + blockIdx.x) * kF8Tokens;  // of the step, of this block
    const int p0 = max(start, first), n = min(start + kF8Tokens, ctx) - p0, l0 = p0 - first;
    if (n <= 0) return;
    const int page = tl::ld_cg(a.table + static_cast<size_t>(b) * a.max_pages + start / pg.page_size), slot = start % pg.page_size, kept = p0 - start;
    const bool there = static_cast<unsigned>(page) < static_cast<unsigned>(pg.num_pages);

    // everything is asked for: keys, values, the first rows of queries (row r: token r / G, head r % G)
    ApRow<T> kr[PASSES], vr[PASSES], qr[AHEAD];
    const T *k = static_cast<const T *>(a.k) + b * a.k_b + h * a.k_h + l0 * a.k_l, *v = static_cast<const T *>(a.v) + b * a.v_b + h * a.v_h + l0 * a.v_l;
    const T *q = static_cast<const T *>(a.q) + b * a.q_b + static_cast<long long>(h) * G * a.q_h + l0 * a.q_l;
#pragma unroll
    for (int s = 0; s < PASSES; ++s) {
        const int i = s * ROWS + slot_row;
        if (at.on && i < n) kr[s].ask(k + i * a.k_l, at.a0, at.b0), vr[s].ask(v + i * a.v_l, at.a0, at.b0);
        else kr[s].zero(), vr[s].zero();
    }
    auto ask = [&](int r0) {
#pragma unroll
        for (int s = 0; s < AHEAD; ++s) {
            const int r = r0 + s * ROWS + slot_row;
            const int l = f8_div(r, G, a.group_magic);
            if (at.on && r < n * G) qr[s].ask(q + l * a.q_l + (r - l * G) * a.q_h, at.a0, at.b0);
            else qr[s].zero();
        }
    };
    ask(0);
    float before[2] = {0.f, 0.f};
    if (there && kept) before[0] = tl::ld_cg(pg.key_scales + f8_scale_at(pg, page, h, slot)), before[1] = tl::ld_cg(pg.value_scales + f8_scale_at(pg, page, h, slot));
    __syncthreads();
    for (int i = threadIdx.x; i < n * half; i += kApThreads) {
        const int l = f8_div(i, half, a.half_magic);
        angle[l * half + ap_angle_at(i - l * half, half)] = ap_angle(p0 + l, of[i - l * half], part);
    }
    __syncthreads();

    float x[2][PASSES][8], m[2] = {0.f, 0.f};
#pragma unroll
    for (int s = 0; s < PASSES; ++s) {
        const int i = s * ROWS + slot_row;
        if (s * ROWS + warp * RW >= n) continue;  // whole warps
        ap_key<T, LP>(kr[s], a, at, angle + min(i, n - 1) * half, x[0][s]);
        vr[s].get(x[1][s]);
        if (i < n && at.on) {
#pragma unroll
            for (int e = 0; e < 8; ++e) m[0] = f8_most(m[0], fabsf(x[0][s][e])), m[1] = f8_most(m[1], fabsf(x[1][s][e]));
        }
    }
#pragma unroll
    for (int side = 0; side < 2; ++side) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m[side] = f8_most(m[side], __shfl_xor_sync(0xffffffffu, m[side], o));
        if (lane == 0) most[side][warp] = m[side];
    }
    __syncthreads();
    if (there) {
#pragma unroll
        for (int side = 0; side < 2; ++side) {
            float top = 0.f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) top = f8_most(top, most[side][w]);
            const float need = top < INFINITY ? f8_power(f8_exponent(top)) : __int_as_float(0x7fffffff);
            const float scale = f8_most(need, before[side]), under = scale < INFINITY ? 1.f / scale : 0.f;  // NaN if either is
            uint8_t *rows = (side ? pg.values : pg.keys) + f8_row(pg, page, h, slot);
#pragma unroll
            for (int s = 0; s < PASSES; ++s) {
                const int i = s * ROWS + slot_row;
                if (i >= n || !at.on) continue;
                const float(&y)[8] = x[side][s];
                uint2 w = make_uint2(0, 0);
                if (under != 0.f) w = make_uint2(f8_pack4(y[0] * under, y[1] * under, y[2] * under, y[3] * under), f8_pack4(y[4] * under, y[5] * under, y[6] * under, y[7] * under));
                uint8_t *to = rows + static_cast<size_t>(kept + i) * D;
                *reinterpret_cast<uint32_t *>(to + at.a0) = w.x, *reinterpret_cast<uint32_t *>(to + at.b0) = w.y;
            }
            if (kept && scale > before[side]) ap_again(rows, kept * (D / 16), before[side] * under);  // never where either is NaN: the numbers of such a block do not matter
            if (threadIdx.x == 0) (side ? pg.value_scales : pg.key_scales)[f8_scale_at(pg, page, h, slot)] = scale;
        }
    }
    float weight[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) weight[e] = 1.f;
    if (a.q_norm && at.on) {
        ApRow<T> w;
        w.load(static_cast<const T *>(a.q_norm), at.a0, at.b0), w.get(weight);
    }
    for (int r0 = 0; r0 < n * G; r0 += AHEAD * ROWS) {
        if (r0) ask(r0);
#pragma unroll
        for (int s = 0; s < AHEAD; ++s) {
            const int r = r0 + s * ROWS + slot_row, row = min(r, n * G - 1), l = f8_div(row, G, a.group_magic);
            if (r0 + s * ROWS + warp * RW >= n * G) continue;  // whole warps
            float y[8];
            ap_query<T, LP>(qr[s], a, at, weight, angle + l * half, y);
            if (r < n * G && at.on) {
                T *to = q_out + (static_cast<size_t>(l0 + l) * a.heads + row - l * G) * D;
                store4(to + at.a0, make_float4(y[0], y[1], y[2], y[3])), store4(to + at.b0, make_float4(y[4], y[5], y[6], y[7]));
            }
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(kApThreads) fp8_append_any_kernel(const __grid_constant__ F8Append a, const __grid_constant__ F8Turns turns) {
    extern __shared__ __align__(16) unsigned char sm[];
    __shared__ float most[2][kF8Tokens];
    tl::griddep_launch();
    tl::griddep_wait();
    const tlb_fp8_pages &pg = a.pages;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, D = pg.dim, half = a.rot / 2;
    const int b = blockIdx.z, h = blockIdx.y, G = a.group;
    const int ctx = tl::ld_cg(a.lens + b);
    T *q_out = static_cast<T *>(a.q_out) + (static_cast<size_t>(b) * a.tokens * a.heads + static_cast<size_t>(h) * G) * D;
    // an idle slot (or one whose length does not cover the step) appends nothing; its queries come out as zeros
    if (ctx < a.tokens || static_cast<long long>(ctx) > static_cast<long long>(a.max_pages) * pg.page_size) {
        const int l0 = blockIdx.x * kF8Tokens, n = min(a.tokens - l0, kF8Tokens);
        for (int i = threadIdx.x; i < n * G * D; i += kApThreads) q_out[static_cast<size_t>(l0 + i / (G * D)) * a.heads * D + i % (G * D)] = from_f<T>(0.f);
        return;
    }
    const int first = ctx - a.tokens, start = (first / kF8Tokens + blockIdx.x) * kF8Tokens;  // of the step, of this block
    const int p0 = max(start, first), n = min(start + kF8Tokens, ctx) - p0, l0 = p0 - first;
    if (n <= 0) return;

    const int room = min(a.tokens, kF8Tokens);
    double2 *angle = reinterpret_cast<double2 *>(sm);                        // [room][half]: cos, sin
    float *fresh = reinterpret_cast<float *>(angle + static_cast<size_t>(room) * half);  // [2][room][D]: keys, values
    for (int i = threadIdx.x; i < n * half; i += kApThreads) {
        const double t = (p0 + i / half) * turns.of[i % half];
        double s, c;
        sincospi(2.0 * (t - rint(t)), &s, &c);
        angle[i] = make_double2(c, s);
    }
    __syncthreads();

    for (int task = warp; task < n * (G + 2); task += kApThreads / 32) {
        const int i = task / (G + 2), which = task - i * (G + 2);  // group's queries, then key, then value
        const double2 *turn = angle + i * half;
        if (which < G) {
            const T *x = static_cast<const T *>(a.q) + b * a.q_b + (static_cast<long long>(h) * G + which) * a.q_h + (l0 + i) * a.q_l;
            const T *w = static_cast<const T *>(a.q_norm);
            T *y = q_out + (static_cast<size_t>(l0 + i) * a.heads + which) * D;
            float r = 1.f;
            if (w) {
                float s = 0.f;
                for (int d = lane; d < D; d += 32) {
                    const float u = to_f(tl::ld_cg(x + d));
                    s += u * u;
                }
                r = 1.f / sqrtf(warp_sum(s) / D + a.q_eps);
            }
            auto at = [&](int d) {
                const float u = to_f(tl::ld_cg(x + d));
                return w ? u * r * to_f(w[d]) : u;
            };
            for (int j = lane; j < half; j += 32) {
                const int2 e = ap_pair(a, j);
                const float c = static_cast<float>(turn[j].x), s = static_cast<float>(turn[j].y), u = at(e.x), v = at(e.y);
                y[e.x] = from_f<T>(u * c - v * s);
                y[e.y] = from_f<T>(v * c + u * s);
            }
            for (int d = a.rot + lane; d < D; d += 32) y[d] = from_f<T>(at(d));
            continue;
        }
        const bool key = which == G;
        float *y = fresh + (static_cast<size_t>(key ? 0 : room) + i) * D, m = 0.f;
        if (key) {
            const T *x = static_cast<const T *>(a.k) + b * a.k_b + h * a.k_h + (l0 + i) * a.k_l;
            const T *w = static_cast<const T *>(a.k_norm);
            double r = 1.0;
            if (w) {
                double s = 0.0;
                for (int d = lane; d < D; d += 32) {
                    const double u = to_f(tl::ld_cg(x + d));
                    s += u * u;
                }
                r = 1.0 / sqrt(warp_sum_f64(s) / D + a.k_eps);
            }
            auto at = [&](int d) {
                const double u = to_f(tl::ld_cg(x + d));
                return w ? u * r * to_f(w[d]) : u;
            };
            for (int j = lane; j < half; j += 32) {
                const int2 e = ap_pair(a, j);
                const double u = at(e.x), v = at(e.y);
                const float f = static_cast<float>(u * turn[j].x - v * turn[j].y), g = static_cast<float>(v * turn[j].x + u * turn[j].y);
                y[e.x] = f, y[e.y] = g, m = f8_most(m, f8_most(fabsf(f), fabsf(g)));
            }
            for (int d = a.rot + lane; d < D; d += 32) {
                const float f = static_cast<float>(at(d));
                y[d] = f, m = f8_most(m, fabsf(f));
            }
        } else {
            const T *x = static_cast<const T *>(a.v) + b * a.v_b + h * a.v_h + (l0 + i) * a.v_l;
            for (int d = lane; d < D; d += 32) {
                const float f = to_f(tl::ld_cg(x + d));
                y[d] = f, m = f8_most(m, fabsf(f));
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = f8_most(m, __shfl_xor_sync(0xffffffffu, m, o));
        if (lane == 0) most[key ? 0 : 1][i] = m;
    }
    __syncthreads();

    const int page = tl::ld_cg(a.table + static_cast<size_t>(b) * a.max_pages + start / pg.page_size), slot = start % pg.page_size;
    if (page < 0 || page >= pg.num_pages) return;
    const int kept = p0 - start, pieces = D / 16;  // rows of earlier tokens, 16-byte pieces of a row
#pragma unroll
    for (int side = 0; side < 2; ++side) {
        float m = 0.f;
        for (int i = 0; i < n; ++i) m = f8_most(m, most[side][i]);
        float *scale_at = (side ? pg.value_scales : pg.key_scales) + f8_scale_at(pg, page, h, slot);
        uint8_t *rows = (side ? pg.values : pg.keys) + f8_row(pg, page, h, slot);
        const float before = kept ? tl::ld_cg(scale_at) : 0.f;
        const bool fine = m < INFINITY;
        const float need = fine ? f8_power(f8_exponent(m)) : __int_as_float(0x7fffffff);
        const float scale = f8_most(need, before);  // NaN if either is
        const float under = scale < INFINITY ? 1.f / scale : 0.f;
        for (int i = threadIdx.x; i < n * pieces; i += kApThreads) {
            const float4 *x = reinterpret_cast<const float4 *>(fresh + (static_cast<size_t>(side ? room : 0) + i / pieces) * D + i % pieces * 16);
            uint4 out = make_uint4(0, 0, 0, 0);
            if (under != 0.f) {
                uint32_t w[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) w[c] = f8_pack4(x[c].x * under, x[c].y * under, x[c].z * under, x[c].w * under);
                out = make_uint4(w[0], w[1], w[2], w[3]);
            }
            reinterpret_cast<uint4 *>(rows + static_cast<size_t>(kept) * D)[i] = out;
        }
        if (kept && scale > before) {  // never where either is NaN: the numbers of such a block do not matter
            ap_again(rows, kept * pieces, before * under);
        }
        __syncthreads();  // every thread has read the scale before
        if (threadIdx.x == 0) *scale_at = scale;
    }
}

int f8_check_pages(const char *op, const tlb_fp8_pages *p) {
    if (!p || !p->keys || !p->values || !p->key_scales || !p->value_scales) return tl::fail(TL_EINVAL, "%s: no pages", op);
    if (p->num_pages <= 0 || p->heads <= 0 || p->page_size <= 0 || p->page_size % kF8Tokens) return tl::fail(TL_EINVAL, "%s: pages of a multiple of %d slots", op, kF8Tokens);
    if (p->dim <= 0 || p->dim > kApMostDim || p->dim % 16) return tl::fail(TL_EINVAL, "%s: heads of a multiple of 16 entries, at most %d", op, kApMostDim);
    if (!tl::aligned16(p->keys) || !tl::aligned16(p->values)) return tl::fail(TL_EINVAL, "%s: pages must begin on 16 bytes", op);
    if (static_cast<double>(p->num_pages) * p->heads * (p->page_size / kF8Tokens) > 2147483647.0) return tl::fail(TL_EINVAL, "%s: more than 2^31 blocks", op);  // a block's place is an int
    return TL_OK;
}

int f8_check_step(const char *op, const tlb_fp8_pages &p, const int32_t *lens, const int32_t *table, int batch, int max_pages, int tokens) {
    if (static_cast<long long>(max_pages) * p.page_size > 1LL << 30) return tl::fail(TL_EINVAL, "%s: a block table for more than 2^30 tokens", op);  // positions are ints
    if (!lens && !table) return TL_OK;
    if (!lens || !table) return tl::fail(TL_EINVAL, "%s: lengths and block table on the host go together", op);
    std::vector<uint64_t> seen;  // a bit for every page
    try {
        seen.resize((static_cast<size_t>(p.num_pages) + 63) / 64);
    } catch (...) {  // no exception leaves a C entry
        return tl::fail(TL_EINVAL, "%s: no memory for the checks", op);
    }
    for (int b = 0; b < batch; ++b) {
        const int32_t *row = table + static_cast<size_t>(b) * max_pages;
        const long long n = lens[b], live = (n + p.page_size - 1) / p.page_size;
        bool fine = n >= 0 && (n == 0 || n >= tokens) && live <= max_pages;
        for (int i = 0; fine && i < max_pages; ++i) {
            const int32_t id = row[i];
            if (i >= live) {
                fine = id == -1;
            } else if ((fine = id >= 0 && id < p.num_pages && !(seen[id >> 6] >> (id & 63) & 1))) {
                seen[id >> 6] |= uint64_t{1} << (id & 63);
            }
        }
        if (!fine) return tl::fail(TL_EINVAL, "%s: lengths or block table of request %d", op, b);
    }
    return TL_OK;
}

template <typename T>
static int append_launch(const F8Append &a, const F8Turns &turns, cudaStream_t st) {
    static tl::PerDevice ready;
    const int D = a.pages.dim;
    const long long strides = a.q_b | a.q_h | a.q_l | a.k_b | a.k_h | a.k_l | a.v_b | a.v_h | a.v_l;
    auto aligned = [](const void *p) { return p == nullptr || tl::aligned16(p); };
    const bool wide = aligned(a.q) && aligned(a.k) && aligned(a.v) && aligned(a.q_out) && aligned(a.q_norm) && aligned(a.k_norm) && (strides * static_cast<long long>(sizeof(T)) & 15) == 0 &&
                      a.rot % 8 == 0;
    const size_t room = a.tokens < kF8Tokens ? a.tokens : kF8Tokens, angles = room * (a.rot / 2) * 16;
    const auto any = fp8_append_any_kernel<T>;
    const auto rows = D <= 64 ? fp8_append_kernel<T, 8> : D <= 128 ? fp8_append_kernel<T, 16> : fp8_append_kernel<T, 32>;
    int device = 0;
    cudaGetDevice(&device);
    if (!ready(device, [&] { return cudaFuncSetAttribute(any, cudaFuncAttributeMaxDynamicSharedMemorySize, kF8Tokens * kApMostDim * 16) == cudaSuccess; }))
        return tl::fail(TL_ECUDA, "fp8_append: %s", cudaGetErrorString(cudaGetLastError()));
    const dim3 grid((a.tokens + 2 * kF8Tokens - 2) / kF8Tokens, a.pages.heads, a.batch);
    const cudaError_t e = wide ? tl::launch_chained(rows, grid, dim3(kApThreads), angles, st, a, turns)
                               : tl::launch_chained(any, grid, dim3(kApThreads), angles + room * 2 * D * sizeof(float), st, a, turns);
    if (e != cudaSuccess) return tl::fail(TL_ECUDA, "fp8_append: %s", cudaGetErrorString(e));
    TL_LAUNCH_CHECK("fp8_append");
    return TL_OK;
}

}  // namespace tlb

using namespace tlb;

extern "C" int tlb_fp8_append(const tlb_fp8_pages *pages, const tlb_fp8_append_call *c, const int32_t *lens_host, const int32_t *table_host, void *stream) {
    const int rc = f8_check_pages("fp8_append", pages);
    if (rc != TL_OK) return rc;
    if (!c || c->batch < 0 || c->tokens < 0 || c->heads <= 0 || c->heads % pages->heads) return tl::fail(TL_EINVAL, "fp8_append: query heads over %d key/value heads", pages->heads);
    if (c->rot < 0 || c->rot % 2 || c->rot > pages->dim || !(c->base > 0.0)) return tl::fail(TL_EINVAL, "fp8_append: cannot rotate %d of %d entries", c->rot, pages->dim);
    if (c->batch == 0 || c->tokens == 0) return TL_OK;
    if (c->batch > 65535 || pages->heads > 65535 || c->tokens > (1 << 30) || c->max_pages <= 0) return tl::fail(TL_EINVAL, "fp8_append: sizes out of range");
    if (!c->q || !c->q_out || !c->k || !c->v || !c->table || !c->lens) return tl::fail(TL_EINVAL, "fp8_append: missing argument");
    if (const int bad = f8_check_step("fp8_append", *pages, lens_host, table_host, c->batch, c->max_pages, c->tokens)) return bad;
    // the frequencies of this thread's last call; half as many powers otherwise
    static thread_local F8Turns turns;
    static thread_local int turns_rot = -1;
    static thread_local double turns_base = 0.0;
    if (c->rot != turns_rot || c->base != turns_base) {
        for (int i = 0; i < c->rot / 2; ++i) turns.of[i] = pow(c->base, -2.0 * i / c->rot) / (2.0 * M_PI);
        for (int k = 0; k < kApParts; ++k) {
            const double co = cos(2.0 * M_PI * k / kApParts), si = sin(2.0 * M_PI * k / kApParts);
            turns.part[k] = make_float4(static_cast<float>(co), static_cast<float>(co - static_cast<float>(co)), static_cast<float>(si), static_cast<float>(si - static_cast<float>(si)));
        }
        turns_rot = c->rot, turns_base = c->base;
    }
    const F8Append a{*pages, *c, c->heads / pages->heads};
    TLB_DISPATCH(c->dtype, "fp8_append", return append_launch<T>(a, turns, as_stream(stream)));
}
