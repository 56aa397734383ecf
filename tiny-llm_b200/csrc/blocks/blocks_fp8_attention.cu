// Grouped-query attention over pages of 8 bits:  out = softmax(q k^T * scale) v,  k and v a number times its block's scale.
//
// The products run on mma.sync (m16n8k16, f16 in, fp32 out) with the cache as the first operand: 16 keys (a block, so one scale of either side) times 8 columns, a
// column being one (query head of the group, new token).  An e4m3 number is an f16 number, so the cache's side is exact; a column is brought to the top of
// f16's range by a power of two, where bf16 keeps all its bits, and an fp32 query is two such terms.  The scales never meet f16: a block's
// key scale multiplies its scores and its value scale the product of its weights and values, both in fp32.  Weights are exp2 of a number up to the
// column's running maximum (which may lag behind by 2^8 before the sums are scaled again), rounded to f16 for the second product: 2^-12 of a weight, where an output is
// rounded to 2^-9 of itself; fp32 outputs take a second term for the rest.  Running sums are fp32.
//
// A warp takes blocks of 16 keys straight from the pages into registers in the layouts that the products want, without shared memory between: lane (g, t) loads 16-byte
// pieces t, t + 4 .. of key rows g and g + 8, and of the value rows 2t, 2t + 1, 2t + 8, 2t + 9 the g-th eighth.  Which entry of a head a product's k-index means
// is free as long as queries agree; the values' bytes of two keys are interleaved by byte permutation.  Warps of a CTA and CTAs of a cluster share the
// keys of their columns and are joined at the end, in a fixed order.
#include <cooperative_groups.h>

#include "../per_device.h"
#include "blocks_fp8_cache.cuh"
#include "blocks_fp8_attention.cuh"

namespace tlb {

namespace cg = cooperative_groups;

constexpr float kAtLag = 8.f;  // log2: how far a running maximum may lag behind

__device__ __forceinline__ float at_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t at_half2(uint32_t two) {  // two e4m3 numbers (the lower 16 bits) as f16
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<uint16_t>(two)));
    return r;
}
__device__ __forceinline__ uint32_t at_turn(uint32_t v) {  // an 8 x 8 matrix of f16, transposed
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ void at_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t at_pack(float lo, float hi) { return tl::pack2<__half>(lo, hi); }
__device__ __forceinline__ float2 at_rest(uint32_t two, float lo, float hi) {  // what the rounding to f16 left
    const float2 f = tl::unpack2<__half>(two);
    return make_float2(lo - f.x, hi - f.y);
}

// 16 keys of a head, as a lane holds them.
template <int DP>
struct AtBlock {
    uint4 k[2][DP / 64];
    uint32_t v[4][DP / 32];
    float ks, vs;
};

template <int DP>
__device__ __forceinline__ void at_load(AtBlock<DP> &x, const F8Attend &a, int b, int h, int key0, int page, int lane) {
    const tlb_fp8_pages &pg = a.pages;
    const int g = lane >> 2, t = lane & 3, D = pg.dim;
    if (page < 0 || page >= pg.num_pages) page = 0;  // its keys are masked; nothing outside the pages is read
    const int slot = key0 % pg.page_size;
    const uint8_t *k = pg.keys + f8_row(pg, page, h, slot), *v = pg.values + f8_row(pg, page, h, slot);
#pragma unroll
    for (int r = 0; r < DP / 64; ++r) {
        const int d = (4 * r + t) * 16;
#pragma unroll
        for (int i = 0; i < 2; ++i) x.k[i][r] = d < D ? tl::ldg_stream(k + static_cast<size_t>(g + 8 * i) * D + d) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint8_t *row = v + static_cast<size_t>(2 * t + (i & 1) + 4 * (i & 2)) * D;
        if constexpr (DP == 64) {
            const uint2 w = g * 8 < D ? *reinterpret_cast<const uint2 *>(row + g * 8) : make_uint2(0, 0);
            x.v[i][0] = w.x, x.v[i][1] = w.y;
        } else {
#pragma unroll
            for (int p = 0; p < DP / 128; ++p) {
                const int d = g * (DP / 8) + 16 * p;
                const uint4 w = d < D ? tl::ldg_stream(row + d) : make_uint4(0, 0, 0, 0);
                x.v[i][4 * p] = w.x, x.v[i][4 * p + 1] = w.y, x.v[i][4 * p + 2] = w.z, x.v[i][4 * p + 3] = w.w;
            }
        }
    }
    const size_t s = f8_scale_at(pg, page, h, slot);
    x.ks = __ldg(pg.key_scales + s), x.vs = __ldg(pg.value_scales + s);
}

template <typename T, int DP, int NT, int WARPS>
__global__ void __launch_bounds__(WARPS * 32) fp8_attend_kernel(const __grid_constant__ F8Attend a) {
    constexpr bool kTwo = sizeof(T) == 4;  // a second term of queries and weights
    constexpr int KR = DP / 64, COLS = 8 * NT, J = DP / 16;
    extern __shared__ __align__(16) unsigned char sm[];
    float *part = reinterpret_cast<float *>(sm);  // [WARPS][COLS][DP], then maxima and sums [WARPS][COLS]
    float *part_m = part + WARPS * COLS * DP, *part_l = part_m + WARPS * COLS;
    tl::griddep_launch();
    tl::griddep_wait();
    cg::cluster_group cluster = cg::this_cluster();
    const int ranks = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const tlb_fp8_pages &pg = a.pages;
    const int D = pg.dim, G = a.group, L = a.tokens;
    // this CTA: columns of one request and key/value head; column = new token * group + query head
    const unsigned item = blockIdx.x / ranks;
    const int h = static_cast<int>(item % pg.heads), cb = static_cast<int>(item / pg.heads % a.col_blocks), b = static_cast<int>(item / pg.heads / a.col_blocks);
    const int c0 = cb * COLS;
    const int ctx = static_cast<int>(max(0LL, min(static_cast<long long>(a.lens[b]), static_cast<long long>(a.max_pages) * pg.page_size)));
    // keys [0, limit) are seen; a column behind the last one goes along with it, its query is 0 and nothing of it is stored
    auto limit_of = [&](int col) { return a.causal ? max(ctx - L + 1 + min(col, G * L - 1) / G, 0) : ctx; };
    const int low = limit_of(c0), end = min(limit_of(c0 + COLS - 1), ctx);

    // queries: column g of n-tile nt, the entries that this lane's key pieces stand for
    uint32_t qf[NT][KR][4][2], ql[kTwo ? NT : 1][KR][4][2];
    float factor[NT][2], rest[NT][2];  // of columns 2t and 2t + 1: scores in log2; what its rounding left
    int limit[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int col = c0 + 8 * nt + g;
        const bool live = col < G * L;
        const T *q = static_cast<const T *>(a.q) + b * a.q_b + (static_cast<long long>(h) * G + (live ? col % G : 0)) * a.q_h + (live ? col / G : 0) * a.q_l;
        float x[KR][16], m = 0.f;
#pragma unroll
        for (int r = 0; r < KR; ++r) {
            const int d = (4 * r + t) * 16;
#pragma unroll
            for (int e = 0; e < 16; ++e) x[r][e] = live && d < D ? to_f(q[d + e]) : 0.f;
#pragma unroll
            for (int e = 0; e < 16; ++e) m = f8_most(m, fabsf(x[r][e]));
        }
        m = f8_most(m, __shfl_xor_sync(0xffffffffu, m, 1)), m = f8_most(m, __shfl_xor_sync(0xffffffffu, m, 2));
        const int e2 = static_cast<int>(__float_as_uint(m) >> 23);  // 255: no number, whose scores are none either
        const int up = e2 == 255 ? 0 : min(13 + 127 - e2, 100);      // m * 2^up lies in [2^13, 2^14)
        const float times = f8_power(up);
#pragma unroll
        for (int r = 0; r < KR; ++r)
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float u = x[r][4 * s + 2 * e] * times, w = x[r][4 * s + 2 * e + 1] * times;
                    qf[nt][r][s][e] = at_pack(u, w);
                    if constexpr (kTwo) {
                        const float2 z = at_rest(qf[nt][r][s][e], u, w);
                        ql[nt][r][s][e] = at_pack(z.x, z.y);
                    }
                }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const float back = f8_power(-__shfl_sync(0xffffffffu, up, (2 * t + e) * 4));
            factor[nt][e] = a.scale_log2 * back, rest[nt][e] = a.scale_rest * back;
            limit[nt][e] = limit_of(c0 + 8 * nt + 2 * t + e);
        }
    }

    float o[NT][J][4], m_run[NT][2], l_run[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[nt][j][i] = 0.f;
#pragma unroll
        for (int e = 0; e < 2; ++e) m_run[nt][e] = -INFINITY, l_run[nt][e] = 0.f;
    }

    // the cluster's shares of the blocks, then every WARPS-th one
    const int blocks = (end + kF8Tokens - 1) / kF8Tokens, share = (blocks + ranks - 1) / ranks;
    const int begin = min(rank * share, blocks), stop = min(begin + share, blocks);
    const int32_t *table = a.table + static_cast<size_t>(b) * a.max_pages;
    auto page_of = [&](int blk) { return blk < stop ? table[blk * kF8Tokens / pg.page_size] : -1; };
    int at = begin + warp;
    AtBlock<DP> x;
    int page = page_of(at), page_next = page_of(at + WARPS);
    if (at < stop) at_load<DP>(x, a, b, h, at * kF8Tokens, page, lane);
    for (; at < stop; at += WARPS) {
        AtBlock<DP> y = x;
        const int key0 = at * kF8Tokens, here = page;
        page = page_next, page_next = page_of(at + 2 * WARPS);
        if (at + WARPS < stop) at_load<DP>(x, a, b, h, key0 + WARPS * kF8Tokens, page, lane);
        if (here < 0 || here >= pg.num_pages) continue;

        // scores: rows g and g + 8 (keys), columns 2t and 2t + 1
        float sc[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) sc[nt][i] = 0.f;
#pragma unroll
        for (int r = 0; r < KR; ++r) {
            const uint32_t w0[4] = {y.k[0][r].x, y.k[0][r].y, y.k[0][r].z, y.k[0][r].w}, w1[4] = {y.k[1][r].x, y.k[1][r].y, y.k[1][r].z, y.k[1][r].w};
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const uint32_t f[4] = {at_half2(w0[s]), at_half2(w1[s]), at_half2(w0[s] >> 16), at_half2(w1[s] >> 16)};
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    if constexpr (kTwo) {  // every product's sum begins anew: the tensor cores cut what they add up, fp32 additions round
                        float d[4] = {0.f, 0.f, 0.f, 0.f}, c[4] = {0.f, 0.f, 0.f, 0.f};
                        at_mma(d, f, ql[nt][r][s][0], ql[nt][r][s][1]);
                        at_mma(c, f, qf[nt][r][s][0], qf[nt][r][s][1]);
#pragma unroll
                        for (int i = 0; i < 4; ++i) sc[nt][i] += c[i] + d[i];
                    } else {
                        at_mma(sc[nt], f, qf[nt][r][s][0], qf[nt][r][s][1]);
                    }
                }
            }
        }
        float most[NT][2];
        bool grow = false;
        const bool whole = key0 + kF8Tokens <= low;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float f = factor[nt][e] * y.ks;
                const float u = !whole && key0 + g >= limit[nt][e] ? -INFINITY : sc[nt][e] * f, w = !whole && key0 + g + 8 >= limit[nt][e] ? -INFINITY : sc[nt][2 + e] * f;
                most[nt][e] = fmaxf(u, w);
                grow |= most[nt][e] > m_run[nt][e] + kAtLag;
            }
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float m = most[nt][e];
#pragma unroll
                    for (int w = 4; w < 32; w <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, w));
                    m = fmaxf(m, m_run[nt][e]);
                    const float alpha = m == m_run[nt][e] ? 1.f : at_ex2(m_run[nt][e] - m);
                    m_run[nt][e] = m, l_run[nt][e] *= alpha;
#pragma unroll
                    for (int j = 0; j < J; ++j) o[nt][j][e] *= alpha, o[nt][j][2 + e] *= alpha;
                }
        }
        uint32_t p[NT][2], pl[kTwo ? NT : 1][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float w[4];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float m = m_run[nt][e] == -INFINITY ? 0.f : m_run[nt][e], f = factor[nt][e] * y.ks;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float s = sc[nt][2 * i + e];
                    float z = kTwo ? fmaf(s, f, fmaf(s, rest[nt][e] * y.ks, -m)) : fmaf(s, f, -m);
                    if (!whole && key0 + g + 8 * i >= limit[nt][e]) z = -INFINITY;
                    w[2 * i + e] = kTwo ? exp2f(z) : at_ex2(z);
                }
                l_run[nt][e] += w[e] + w[2 + e];
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                p[nt][i] = at_pack(w[2 * i], w[2 * i + 1]);
                if constexpr (kTwo) {
                    const float2 z = at_rest(p[nt][i], w[2 * i], w[2 * i + 1]);
                    pl[nt][i] = at_turn(at_pack(z.x * 2048.f, z.y * 2048.f));  // the rest of a small weight would fall below f16's range
                }
                p[nt][i] = at_turn(p[nt][i]);
            }
        }
        if (key0 + kF8Tokens > ctx) {  // rows behind the last token may hold anything
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (key0 + 2 * t + (i & 1) + 4 * (i & 2) >= ctx)
#pragma unroll
                    for (int w = 0; w < DP / 32; ++w) y.v[i][w] = 0;
        }
        float vs[NT][2];  // a column that sees none of the block takes nothing from a scale that is no number
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) vs[nt][e] = whole || key0 < limit[nt][e] ? y.vs : 0.f;
#pragma unroll
        for (int j = 0; j < J; ++j) {  // entries 2j (rows g) and 2j + 1 (rows g + 8) of the lanes' eighths
            const uint32_t sel = j & 1 ? 0x7362 : 0x5140;
            const uint32_t one = __byte_perm(y.v[0][j >> 1], y.v[1][j >> 1], sel), two = __byte_perm(y.v[2][j >> 1], y.v[3][j >> 1], sel);
            const uint32_t f[4] = {at_half2(one), at_half2(one >> 16), at_half2(two), at_half2(two >> 16)};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float d[4] = {0.f, 0.f, 0.f, 0.f};
                at_mma(d, f, p[nt][0], p[nt][1]);
                if constexpr (kTwo) {
                    float c[4] = {0.f, 0.f, 0.f, 0.f};
                    at_mma(c, f, pl[nt][0], pl[nt][1]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) d[i] = fmaf(c[i], 1.f / 2048.f, d[i]);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) o[nt][j][i] = fmaf(d[i], vs[nt][i & 1], o[nt][j][i]);
            }
        }
    }

    // join the warps
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float l = l_run[nt][e];
#pragma unroll
            for (int w = 4; w < 32; w <<= 1) l += __shfl_xor_sync(0xffffffffu, l, w);
            const int col = 8 * nt + 2 * t + e;
            if (g == 0) part_m[warp * COLS + col] = m_run[nt][e], part_l[warp * COLS + col] = l;
            float *to = part + (static_cast<size_t>(warp) * COLS + col) * DP + g * (DP / 8);
#pragma unroll
            for (int j = 0; j < J; ++j) to[2 * j] = o[nt][j][e], to[2 * j + 1] = o[nt][j][2 + e];
        }
    __syncthreads();
    for (int i = threadIdx.x; i < COLS * DP; i += WARPS * 32) {
        const int col = i / DP;
        float m = -INFINITY, v = 0.f;
        for (int w = 0; w < WARPS; ++w) m = fmaxf(m, part_m[w * COLS + col]);
        for (int w = 0; w < WARPS; ++w)
            if (part_l[w * COLS + col] != 0.f) v = fmaf(part[w * COLS * DP + i], m == -INFINITY ? 1.f : at_ex2(part_m[w * COLS + col] - m), v);
        part[i] = v;
    }
    __syncthreads();
    if (threadIdx.x < COLS) {
        const int col = threadIdx.x;
        float m = -INFINITY, l = 0.f;
        for (int w = 0; w < WARPS; ++w) m = fmaxf(m, part_m[w * COLS + col]);
        for (int w = 0; w < WARPS; ++w) l = fmaf(part_l[w * COLS + col], m == -INFINITY ? 1.f : at_ex2(part_m[w * COLS + col] - m), l);
        part_m[col] = m, part_l[col] = l;
    }
    // join the cluster: each CTA a share of the numbers
    if (ranks > 1) cluster.sync();
    else __syncthreads();
    const int live = min(COLS, G * L - c0), each = (live * D + ranks - 1) / ranks;
    for (int i = rank * each + threadIdx.x; i < min((rank + 1) * each, live * D); i += WARPS * 32) {
        const int col = i / D, d = i - col * D;
        float m = -INFINITY, l = 0.f, v = 0.f;
        for (int r = 0; r < ranks; ++r) m = fmaxf(m, ranks > 1 ? cluster.map_shared_rank(part_m, r)[col] : part_m[col]);
        for (int r = 0; r < ranks; ++r) {
            const float lr = ranks > 1 ? cluster.map_shared_rank(part_l, r)[col] : part_l[col];
            if (lr == 0.f) continue;
            const float mr = ranks > 1 ? cluster.map_shared_rank(part_m, r)[col] : part_m[col], w = m == -INFINITY ? 1.f : at_ex2(mr - m);
            l = fmaf(lr, w, l), v = fmaf((ranks > 1 ? cluster.map_shared_rank(part, r) : part)[col * DP + d], w, v);
        }
        const int c = c0 + col;
        static_cast<T *>(a.out)[((static_cast<size_t>(b) * L + c / G) * a.heads + static_cast<size_t>(h) * G + c % G) * D + d] = from_f<T>(l == 0.f ? 0.f : v / l);
    }
    if (ranks > 1) cluster.sync();  // the others may still read this CTA's shared memory
}

template <typename T, int DP, int NT, int WARPS>
static int attend_launch(F8Attend a, int ranks, cudaStream_t st) {
    static tl::PerDevice ready;
    constexpr int cols = 8 * NT, smem = WARPS * cols * (DP + 2) * 4;
    const auto kernel = fp8_attend_kernel<T, DP, NT, WARPS>;
    int device = 0;
    cudaGetDevice(&device);
    if (!ready(device, [&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) == cudaSuccess; }))
        return tl::fail(TL_ECUDA, "fp8_attention: %s", cudaGetErrorString(cudaGetLastError()));
    a.col_blocks = (a.group * a.tokens + cols - 1) / cols;
    const long long ctas = static_cast<long long>(a.col_blocks) * a.pages.heads * a.batch * ranks;
    if (ctas > 0x7fffffff) return tl::fail(TL_EINVAL, "fp8_attention: sizes out of range");
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(ctas)), cfg.blockDim = dim3(WARPS * 32), cfg.dynamicSmemBytes = smem, cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim = {static_cast<unsigned>(ranks), 1, 1};
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr, cfg.numAttrs = tl::use_pdl() ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a);
    if (e != cudaSuccess) return tl::fail(TL_ECUDA, "fp8_attention: %s", cudaGetErrorString(e));
    TL_LAUNCH_CHECK("fp8_attention");
    return TL_OK;
}

template <typename T>
static int attend_any(const F8Attend &a, cudaStream_t st) {
    const int D = a.pages.dim, rows = a.group * a.tokens;
    const int nt = D > 128 || rows <= 8 ? 1 : 2;
    const long long ctas = static_cast<long long>((rows + 8 * nt - 1) / (8 * nt)) * a.pages.heads * a.batch;
    int ranks = 1;  // as many CTAs as fill the GPU, each with two blocks a warp at the least
    while (ranks < 8 && ctas * ranks < 2 * sm_count() && a.longest > ranks * 2 * 8 * kF8Tokens) ranks *= 2;
    if (D <= 64) return nt == 1 ? attend_launch<T, 64, 1, 8>(a, ranks, st) : attend_launch<T, 64, 2, 8>(a, ranks, st);
    if (D <= 128) return nt == 1 ? attend_launch<T, 128, 1, 8>(a, ranks, st) : attend_launch<T, 128, 2, 8>(a, ranks, st);
    return attend_launch<T, 256, 1, 8>(a, ranks, st);
}

}  // namespace tlb

using namespace tlb;

extern "C" int tlb_fp8_attention(const tlb_fp8_pages *pages, const tlb_fp8_attention_call *c, void *stream) {
    const int rc = f8_check_pages("fp8_attention", pages);
    if (rc != TL_OK) return rc;
    if (!c || c->batch < 0 || c->tokens < 0 || c->heads <= 0 || c->heads % pages->heads) return tl::fail(TL_EINVAL, "fp8_attention: query heads over %d key/value heads", pages->heads);
    if (c->batch == 0 || c->tokens == 0) return TL_OK;
    if (c->max_pages <= 0 || static_cast<long long>(c->heads / pages->heads) * c->tokens > (1 << 30)) return tl::fail(TL_EINVAL, "fp8_attention: sizes out of range");
    if (!c->q || !c->out || !c->table || !c->lens) return tl::fail(TL_EINVAL, "fp8_attention: missing argument");
    const F8Attend a(*pages, *c);
    TLB_DISPATCH(c->dtype, "fp8_attention", return attend_any<T>(a, as_stream(stream)));
}
