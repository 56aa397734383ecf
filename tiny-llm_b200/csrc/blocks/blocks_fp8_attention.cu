// Grouped-query attention over pages of 8 bits:  out = softmax(q k^T * scale) v,  k and v a number times its block's scale.
//
// The products run on mma.sync (m16n8k16, f16 in, fp32 out) with the cache as the first operand: 16 keys (a block, so one scale of either side) times 8 columns, a
// column being one (query head of the group, new token).  An e4m3 number is an f16 number, so the cache's side is exact; a column is brought to the top of
// f16's range by a power of two, where bf16 keeps all its bits, and an fp32 query is two such terms.  A block's key scale multiplies its scores in fp32; its value
// scale multiplies its weights, over a unit of the column's own (kAtLow; fp32 outputs: the product of weights and values).  Weights are exp2 of a number up to the
// column's running maximum (which may lag behind by 2^12 before the sums are scaled again), rounded to f16 for the second product: 2^-11 of a weight or 2^-21 of the largest, where an
// output is rounded to 2^-8 of itself; fp32 outputs take a second term for the rest.  Running sums are fp32.
//
// A warp takes blocks of 16 keys through a ring of its own in shared memory, filled by asynchronous copies, two blocks ahead of the one it works on; it waits for nobody
// else.  Lane (g, t) reads 16-byte pieces t, t + 4 .. of key rows g and g + 8, and of the value rows 2t, 2t + 1, 2t + 8, 2t + 9 the g-th eighth: which entry of a head a product's
// k-index means is free as long as queries agree, and the values' bytes of two keys are interleaved by byte permutation.  The warps of a CTA share its keys and are
// joined in a fixed order.
//
// An item is 8 (or 16) columns of one request and key/value head.  A CTA takes an item; or, where items are few, a cluster does, whose CTAs read each other's sums; or, where
// requests are of unlike length or very long, a CTA takes a piece of one, which leaves a partial result for fp8_attend_join_kernel to add up in order.  Both follow the lengths
// on the device, so a captured launch does.  attend_plan chooses.
//
// 64 requests of 8192 (1.08 GB) take 160 us in replays over the same pages (some of which stay in L2), 175 over others, 6.2 TB/s: HBM.  With fewer, a block is a chain of latencies (1100 cycles of a warp: copies, eight products, exponentials, eight products), so an item of 1970 tokens
// takes 10 us of the 17 of a step of 24 requests.  Not faster: 16 warps a CTA (24 requests 14.8 us, but 30 of 1000 tokens 18.7 for 14.2), rings of six blocks.  Scales of values anywhere within 2^16
// of one another, whose units move again and again, make it 24 requests 19.5, 64 x 8192 168 us.
#include <algorithm>
#include <atomic>

#include "../per_device.h"
#include "blocks_fp8_cache.cuh"
#include "blocks_fp8_attention.cuh"

namespace tlb {

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
__device__ __forceinline__ void at_mma_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {  // nothing to add to
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t at_pack(float lo, float hi) { return tl::pack2<__half>(lo, hi); }
__device__ __forceinline__ float2 at_rest(uint32_t two, float lo, float hi) {  // what the rounding to f16 left
    const float2 f = tl::unpack2<__half>(two);
    return make_float2(lo - f.x, hi - f.y);
}

// 1 over a power of two of 2^-126 to 2^126; one over the next one above what is none.  (A division would be a call: 0.7 us of 6 for one request of 1011 tokens.)
__device__ __forceinline__ float at_under(float v) { return __int_as_float(0x7f000000 - ((__float_as_int(v) + 0x7fffff) & 0x7f800000)); }

constexpr int kAtWarps = 8, kAtStages = 3;
// bf16 outputs.  A column's weights take the block's value scale, over a unit of the column's own, ahead of their rounding to f16, whose smallest step is 2^-24.  The unit is the scale of one of the
// column's blocks; it moves to one of more than 8 times as much (a weight of up to 2^12 is an f16 number then) or of less than 1 / 16 of it, so a weight's error is 2^-11 of itself or 2^-21 of the
// largest weight.  Blocks that a column does not see, or gives no weight, leave its unit alone.  It falls to 2^-80 of the highest it has had, so that the sums stay within fp32's range.
constexpr float kAtLow = 0.0625f, kAtHigh = 8.f, kAtDeep = 0x1p-80f;
constexpr float kAtRowLag = 12.f;  // log2: how far a running maximum may lag behind here
constexpr float kAtUnder = 0x1p-20f;  // sums leave a warp times this: scales of 2^-100 to 2^119 stay within fp32's range

__device__ __forceinline__ void at_copy16(uint32_t to, const void *from) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory"); }

// A block in shared memory: 16 rows of keys, 16 of values.  Rows of 128 bytes have their pieces moved about so that the eight lanes of a reading phase meet
// all banks: a key's halves change places in odd rows (lanes read 4 pieces of 2 rows), a value's pairs of pieces go by the pair of rows (2 pieces of 4 rows).
__host__ __device__ constexpr int at_stage(int dim) { return 2 * kF8Tokens * dim; }
template <bool MOVED>
__device__ __forceinline__ int at_key(int row, int D, int byte) {
    return row * D + (MOVED ? byte ^ ((row & 1) << 6) : byte);
}
template <bool MOVED>
__device__ __forceinline__ int at_value(int row, int D, int byte) {
    return row * D + (MOVED ? byte ^ (((row >> 1) & 3) << 5) : byte);
}

// Of a cluster's CTAs: a barrier, and numbers in the shared memory of the r-th.
__device__ __forceinline__ void at_cluster_sync() { asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ float at_theirs(uint32_t at, int r) {
    float v;
    asm volatile("{\n\t.reg .b32 ra;\n\tmapa.shared::cluster.u32 ra, %1, %2;\n\tld.shared::cluster.f32 %0, [ra];\n\t}" : "=f"(v) : "r"(at), "r"(r) : "memory");
    return v;
}
__device__ __forceinline__ float4 at_theirs4(uint32_t at, int r) {
    float4 v;
    asm volatile("{\n\t.reg .b32 ra;\n\tmapa.shared::cluster.u32 ra, %4, %5;\n\tld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [ra];\n\t}"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(at), "r"(r)
                 : "memory");
    return v;
}

// DIM: entries of a head, 0: as the pages say.  place: of the block among all pages'.
template <int DIM>
__device__ __forceinline__ void at_issue(uint32_t stage, const tlb_fp8_pages &pg, int place, int lane) {
    const int D = DIM ? DIM : pg.dim;
    const size_t byte = static_cast<size_t>(static_cast<unsigned>(place)) * (kF8Tokens * D) + 16 * lane;
    if constexpr (DIM == 128) {
        const uint32_t k = stage + ((16 * lane) ^ ((lane >> 3 & 1) << 6)), v = stage + 16 * D + ((16 * lane) ^ ((lane >> 4) << 5)), w = stage + 16 * D + ((16 * lane) ^ ((lane >> 4) << 5) ^ 64);
#pragma unroll
        for (int i = 0; i < 4; ++i) at_copy16(k + 512 * i, pg.keys + byte + 512 * i), at_copy16((i & 1 ? w : v) + 512 * i, pg.values + byte + 512 * i);
    } else {
        for (int i = lane; i < D; i += 32) {  // 16 rows of D / 16 pieces lie one behind the other
            at_copy16(stage + 16 * i, pg.keys + byte + 16 * (i - lane));
            at_copy16(stage + 16 * D + 16 * i, pg.values + byte + 16 * (i - lane));
        }
    }
}

// Where 32 of a warp's blocks lie, and their scales: a lane knows one of them.  place -1: the page is none, its keys are skipped.
struct AtLook {
    int place;
    float ks, vs;
};

// DP: entries of a head that the lanes' shares make room for; DIM: entries it has, 0: fewer than DP.
template <typename T, int DP, int DIM, int NT>
__global__ void __launch_bounds__(kAtWarps * 32, DP <= 128 && NT == 1 && sizeof(T) == 2 ? 2 : 1) fp8_attend_kernel(const __grid_constant__ F8Attend a) {
    constexpr bool kTwo = sizeof(T) == 4;  // a second term of queries and weights
    constexpr bool kMoved = DIM == 128;
    constexpr int KR = DP / 64, COLS = 8 * NT, J = DP / 16, WARPS = kAtWarps, ROW = DP + 4;
    extern __shared__ __align__(16) unsigned char sm[];
    constexpr int QROW = DP + 8;
    __shared__ __align__(16) __half q_tile[(kTwo ? 2 : 1) * COLS * QROW];
    __shared__ float q_back[COLS];
    // first the warps' rings, then, once all are through,
    float *part = reinterpret_cast<float *>(sm);  // [WARPS][COLS][ROW], then maxima, sums and factors [WARPS][COLS]
    float *part_m = part + WARPS * COLS * ROW, *part_l = part_m + WARPS * COLS, *part_w = part_l + WARPS * COLS;
    tl::griddep_wait();
    tl::griddep_launch();  // behind the wait: the launch that joins the pieces reads the lengths ahead of its own
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const tlb_fp8_pages &pg = a.pages;
    const int D = DIM ? DIM : pg.dim, G = a.group, L = a.tokens;
    int item, rank;  // of a launch without clusters: the CTA's number and 0
    asm("mov.u32 %0, %%clusterid.x;" : "=r"(item));
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    AtPiece mine = at_piece(a, item);
    if (mine.b < 0) return;  // a whole cluster
    if (a.ranks > 1) mine.piece = rank, mine.size = (at_blocks(mine.ctx) + a.ranks - 1) / a.ranks;
    const int b = mine.b, cb = f8_div(mine.item, pg.heads, a.heads_magic), h = mine.item - cb * pg.heads, c0 = cb * COLS, ctx = mine.ctx;
    // keys [0, limit) are seen; a column behind the last one goes along with it, its query is 0 and nothing of it is stored
    auto limit_of = [&](int col) { return a.causal ? max(ctx - L + 1 + f8_div(min(col, G * L - 1), G, a.group_magic), 0) : ctx; };
    const int low = limit_of(c0), end = min(limit_of(c0 + COLS - 1), ctx);
    const int begin = mine.piece * mine.size, stop = min((end + kF8Tokens - 1) / kF8Tokens, begin + mine.size);
    const int32_t *table = a.table + static_cast<size_t>(b) * a.max_pages;
    auto page_at = [&](int blk) { return f8_div(blk, a.page_blocks, a.page_magic); };  // the blk-th block's place in the table
    const int stage_bytes = at_stage(D);
    unsigned char *ring = sm + warp * kAtStages * stage_bytes;
    const uint32_t ring_at = static_cast<uint32_t>(__cvta_generic_to_shared(ring));
    // A warp's share lies side by side, so that a sector of scales is asked for by one warp: with every eighth block a warp's all eight ask L2 for it (64 x 8192 163.5 us for 160, 32000 tokens 21.3 for 20.4)
    const int n_blocks = max(stop - begin, 0), share = n_blocks / WARPS, more = n_blocks % WARPS, count = share + (warp < more), begin_warp = begin + warp * share + min(warp, more);
    auto look = [&](int i0) {
        AtLook x{-1, 0.f, 0.f};
        const int blk = begin_warp + i0 + lane, at = page_at(blk), page = at < a.max_pages ? tl::ld_cg(table + at) : -1;
        if (static_cast<unsigned>(page) < static_cast<unsigned>(pg.num_pages)) {
            x.place = (page * pg.heads + h) * a.page_blocks + blk - at * a.page_blocks;  // fewer than 2^31: they are 16 rows each
            x.ks = tl::ld_cg(pg.key_scales + x.place), x.vs = tl::ld_cg(pg.value_scales + x.place);
        }
        return x;
    };
    auto issue = [&](int stage, bool more, int place) {
        if (more && place >= 0) at_issue<DIM>(ring_at + stage * stage_bytes, pg, place, lane);
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    // queries: eight entries a thread, brought to f16 once for all warps
    static_assert(COLS * DP / 8 <= WARPS * 32, "every entry has a thread");
    const int qcol = threadIdx.x / (DP / 8), qd = threadIdx.x % (DP / 8) * 8;
    float x8[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x8[e] = 0.f;
    if (qcol < COLS && c0 + qcol < G * L && (DIM || qd < D)) {
        const int l = f8_div(c0 + qcol, G, a.group_magic);
        at_query(static_cast<const T *>(a.q) + b * a.q_b + (static_cast<long long>(h) * G + c0 + qcol - l * G) * a.q_h + l * a.q_l + qd, a.wide_rows, x8);
    }
    AtLook now = look(0), next{-1, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < kAtStages - 1; ++i) issue(i, i < count, __shfl_sync(0xffffffffu, now.place, i));

    {
        float m = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) m = f8_most(m, fabsf(x8[e]));
#pragma unroll
        for (int o = 1; o < DP / 8; o <<= 1) m = f8_most(m, __shfl_xor_sync(0xffffffffu, m, o));
        const int e2 = static_cast<int>(__float_as_uint(m) >> 23);  // 255: no number, whose scores are none either
        const int up = e2 == 255 ? 0 : min(13 + 127 - e2, 100);      // m * 2^up lies in [2^13, 2^14)
        const float times = f8_power(up);
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float u = x8[2 * e] * times, w = x8[2 * e + 1] * times;
            hi[e] = at_pack(u, w);
            const float2 z = at_rest(hi[e], u, w);
            lo[e] = at_pack(z.x, z.y);
        }
        if (qcol < COLS) {
            *reinterpret_cast<uint4 *>(q_tile + qcol * QROW + qd) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            if constexpr (kTwo) *reinterpret_cast<uint4 *>(q_tile + (COLS + qcol) * QROW + qd) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            if (qd == 0) q_back[qcol] = f8_power(-up);
        }
    }
    __syncthreads();
    // column g of n-tile nt, the entries that this lane's key pieces stand for
    uint32_t qf[NT][KR][4][2], ql[kTwo ? NT : 1][KR][4][2];
    float factor[NT][2], rest[NT][2];  // of columns 2t and 2t + 1: scores in log2; what its rounding left
    int limit[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int r = 0; r < KR; ++r)
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const uint4 u = *reinterpret_cast<const uint4 *>(q_tile + (8 * nt + g) * QROW + (4 * r + t) * 16 + 8 * s);
                qf[nt][r][2 * s][0] = u.x, qf[nt][r][2 * s][1] = u.y, qf[nt][r][2 * s + 1][0] = u.z, qf[nt][r][2 * s + 1][1] = u.w;
                if constexpr (kTwo) {
                    const uint4 w = *reinterpret_cast<const uint4 *>(q_tile + (COLS + 8 * nt + g) * QROW + (4 * r + t) * 16 + 8 * s);
                    ql[nt][r][2 * s][0] = w.x, ql[nt][r][2 * s][1] = w.y, ql[nt][r][2 * s + 1][0] = w.z, ql[nt][r][2 * s + 1][1] = w.w;
                }
            }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const float back = q_back[8 * nt + 2 * t + e];
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

    float over[NT][2], highest = 0.f;  // 1 over the columns' units (nothing so far: a power of two above all); the largest unit of this lane's columns
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) over[nt][0] = over[nt][1] = 0x1p126f;
    bool strong = false;  // fp32: scores beyond 2^24 were met, which are rounded as their maxima are from then on: what that rounding left would put them above these
    for (int i = 0, stage = 0; i < count; ++i) {
        const int key0 = (begin_warp + i) * kF8Tokens, in_32 = i & 31, ahead = i + kAtStages - 1;
        asm volatile("cp.async.wait_group %0;" ::"n"(kAtStages - 2) : "memory");
        __syncwarp();  // all lanes' copies of this block are there, and all lanes are through with the block before, whose place is next
        if (in_32 == 0 && i + 32 < count) next = look(i + 32);
        const int place_ahead = __shfl_sync(0xffffffffu, (ahead & 31) < in_32 ? next.place : now.place, ahead & 31), stage_ahead = stage ? stage - 1 : kAtStages - 1;
        const unsigned char *block = ring + stage * stage_bytes;
        stage = stage + 1 == kAtStages ? 0 : stage + 1;
        const int place = __shfl_sync(0xffffffffu, now.place, in_32);
        const float2 scales = make_float2(__shfl_sync(0xffffffffu, now.ks, in_32), __shfl_sync(0xffffffffu, now.vs, in_32));
        if (in_32 == 31) now = next;
        if (place < 0) {
            issue(stage_ahead, ahead < count, place_ahead);
            continue;
        }

        // scores: rows g and g + 8 (keys), columns 2t and 2t + 1; of two chains of products
        float sc[NT][4], sd[NT][4];
        if constexpr (kTwo) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < 4; ++i) sc[nt][i] = 0.f;
        }
#pragma unroll
        for (int r = 0; r < KR; ++r) {
            const int d = (4 * r + t) * 16;
            uint4 one = make_uint4(0, 0, 0, 0), two = one;
            if (DIM || d < D) one = *reinterpret_cast<const uint4 *>(block + at_key<kMoved>(g, D, d)), two = *reinterpret_cast<const uint4 *>(block + at_key<kMoved>(g + 8, D, d));
            const uint32_t w0[4] = {one.x, one.y, one.z, one.w}, w1[4] = {two.x, two.y, two.z, two.w};
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                uint32_t f[4];
                at_halves(w0[s], f[0], f[2]), at_halves(w1[s], f[1], f[3]);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    if constexpr (kTwo) {  // every product's sum begins anew: the tensor cores cut what they add up, fp32 additions round
                        float d4[4], c4[4];
                        at_mma_first(d4, f, ql[nt][r][s][0], ql[nt][r][s][1]);
                        at_mma_first(c4, f, qf[nt][r][s][0], qf[nt][r][s][1]);
#pragma unroll
                        for (int i = 0; i < 4; ++i) sc[nt][i] += c4[i] + d4[i];
                    } else {
                        float(&to)[4] = s & 1 ? sd[nt] : sc[nt];
                        if (r == 0 && s < 2) at_mma_first(to, f, qf[nt][r][s][0], qf[nt][r][s][1]);
                        else at_mma(to, f, qf[nt][r][s][0], qf[nt][r][s][1]);
                    }
                }
            }
        }
        issue(stage_ahead, ahead < count, place_ahead);  // while the products are under way
        uint32_t v[4][DP / 32];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = 2 * t + (i & 1) + 4 * (i & 2);
            if constexpr (DP == 64) {
                const uint2 w = DIM || g * 8 < D ? *reinterpret_cast<const uint2 *>(block + 16 * D + row * D + g * 8) : make_uint2(0, 0);
                v[i][0] = w.x, v[i][1] = w.y;
            } else {
#pragma unroll
                for (int c = 0; c < DP / 128; ++c) {
                    const int d = g * (DP / 8) + 16 * c;
                    const uint4 w = DIM || d < D ? *reinterpret_cast<const uint4 *>(block + 16 * D + at_value<kMoved>(row, D, d)) : make_uint4(0, 0, 0, 0);
                    v[i][4 * c] = w.x, v[i][4 * c + 1] = w.y, v[i][4 * c + 2] = w.z, v[i][4 * c + 3] = w.w;
                }
            }
        }

        if constexpr (!kTwo) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) sc[nt][e] += sd[nt][e];
        }
        // scaled to log2, masked scores -inf whatever the factor (which may be no number, 0 or negative)
        float f[NT][2], x[NT][4], vs[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                f[nt][e] = factor[nt][e] * scales.x, vs[nt][e] = kTwo ? scales.y : scales.y * over[nt][e];
                x[nt][e] = __fmul_rn(sc[nt][e], f[nt][e]), x[nt][2 + e] = __fmul_rn(sc[nt][2 + e], f[nt][e]);
            }
        if (key0 + kF8Tokens > low) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    if (key0 + g >= limit[nt][e]) x[nt][e] = -INFINITY;
                    if (key0 + g + 8 >= limit[nt][e]) x[nt][2 + e] = -INFINITY;
                    if (key0 >= limit[nt][e]) vs[nt][e] = 0.f;  // a column that sees none of the block takes nothing from a scale that is no number
                }
            if (key0 + kF8Tokens > ctx) {  // rows behind the last token may hold anything
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (key0 + 2 * t + (i & 1) + 4 * (i & 2) >= ctx)
#pragma unroll
                        for (int w = 0; w < DP / 32; ++w) v[i][w] = 0;
            }
        }
        bool grow = false, move = false;  // of maxima; of units
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                grow |= fmaxf(x[nt][e], x[nt][2 + e]) > m_run[nt][e] + kAtRowLag;
                if constexpr (!kTwo) move |= static_cast<unsigned>(__float_as_int(vs[nt][e]) - __float_as_int(kAtLow)) > static_cast<unsigned>(__float_as_int(kAtHigh) - __float_as_int(kAtLow));
            }
        if (__any_sync(0xffffffffu, grow | move)) {
            float by[NT][2], top[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float m = fmaxf(x[nt][e], x[nt][2 + e]);
#pragma unroll
                    for (int w = 4; w < 32; w <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, w));
                    top[nt][e] = m, m = fmaxf(m, m_run[nt][e]);
                    by[nt][e] = m == m_run[nt][e] ? 1.f : at_ex2(m_run[nt][e] - m);
                    m_run[nt][e] = m, l_run[nt][e] *= by[nt][e];
                    if constexpr (kTwo) strong |= fabsf(m) > 0x1p24f && m > -INFINITY;
                }
            if (!kTwo && __any_sync(0xffffffffu, move)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        if (vs[nt][e] > kAtHigh || (vs[nt][e] < kAtLow && vs[nt][e] > 0.f)) {
                            if (top[nt][e] - m_run[nt][e] < -126.f) {
                                vs[nt][e] = 0.f;  // none of its weights is a number of fp32
                            } else {
                                const float unit = fminf(fmaxf(scales.y, highest * kAtDeep), 0x1p126f), next = at_under(unit);
                                by[nt][e] *= next * at_under(over[nt][e]), over[nt][e] = next, vs[nt][e] = scales.y * next, highest = fmaxf(highest, unit);
                            }
                        }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int j = 0; j < J; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[nt][j][e] *= by[nt][e & 1];
            if constexpr (kTwo) strong = __any_sync(0xffffffffu, strong);
        }
        float left[NT][2];
        if constexpr (kTwo) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) left[nt][e] = rest[nt][e] * scales.x;
            if (strong) {  // the rounded scores themselves
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) sc[nt][e] = x[nt][e], f[nt][e & 1] = 1.f, left[nt][e & 1] = 0.f;
            }
        }
        uint32_t p[NT][2], pl[kTwo ? NT : 1][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float w[4];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float m = m_run[nt][e] == -INFINITY ? 0.f : m_run[nt][e];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float u = x[nt][2 * i + e], s = sc[nt][2 * i + e];
                    if constexpr (kTwo) w[2 * i + e] = exp2f(u == -INFINITY ? u : fmaf(s, f[nt][e], fmaf(s, left[nt][e], -m)));
                    else w[2 * i + e] = at_ex2(u - m);
                }
                l_run[nt][e] += w[e] + w[2 + e];
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                p[nt][i] = kTwo ? at_pack(w[2 * i], w[2 * i + 1]) : at_pack(w[2 * i] * vs[nt][0], w[2 * i + 1] * vs[nt][1]);
                if constexpr (kTwo) {
                    const float2 z = at_rest(p[nt][i], w[2 * i], w[2 * i + 1]);
                    pl[nt][i] = at_turn(at_pack(z.x * 2048.f, z.y * 2048.f));  // the rest of a small weight would fall below f16's range
                }
                p[nt][i] = at_turn(p[nt][i]);
            }
        }
#pragma unroll
        for (int j = 0; j < J; ++j) {  // entries 2j (rows g) and 2j + 1 (rows g + 8) of the lanes' eighths
            const uint32_t sel = j & 1 ? 0x7362 : 0x5140;
            uint32_t f4[4];
            at_halves(__byte_perm(v[0][j >> 1], v[1][j >> 1], sel), f4[0], f4[1]), at_halves(__byte_perm(v[2][j >> 1], v[3][j >> 1], sel), f4[2], f4[3]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                if constexpr (!kTwo) {
                    at_mma(o[nt][j], f4, p[nt][0], p[nt][1]);
                } else {
                    float d[4], c[4];
                    at_mma_first(d, f4, p[nt][0], p[nt][1]);
                    at_mma_first(c, f4, pl[nt][0], pl[nt][1]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[nt][j][e] = fmaf(fmaf(c[e], 1.f / 2048.f, d[e]), vs[nt][e & 1], o[nt][j][e]);
                }
            }
        }
    }

    // join the warps
    const int live = min(COLS, G * L - c0);
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float l = l_run[nt][e];
#pragma unroll
            for (int w = 4; w < 32; w <<= 1) l += __shfl_xor_sync(0xffffffffu, l, w);
            const int col = 8 * nt + 2 * t + e;
            if (g == 0) part_m[warp * COLS + col] = m_run[nt][e], part_l[warp * COLS + col] = kTwo ? l : l * kAtUnder;
            const float unit = kAtUnder * at_under(over[nt][e]);
            if (col < live) {
                float4 *to = reinterpret_cast<float4 *>(part + (warp * COLS + col) * ROW + g * (DP / 8));
#pragma unroll
                for (int j = 0; j < J; j += 2)
                    to[j / 2] = kTwo ? make_float4(o[nt][j][e], o[nt][j][2 + e], o[nt][j + 1][e], o[nt][j + 1][2 + e])
                                     : make_float4(o[nt][j][e] * unit, o[nt][j][2 + e] * unit, o[nt][j + 1][e] * unit, o[nt][j + 1][2 + e] * unit);
            }
        }
    __syncthreads();
    if (threadIdx.x < COLS) {
        const int col = threadIdx.x;
        float m = -INFINITY, l = 0.f;
        for (int w = 0; w < WARPS; ++w) m = fmaxf(m, part_m[w * COLS + col]);
        for (int w = 0; w < WARPS; ++w) {
            const float f = part_m[w * COLS + col] == m ? 1.f : at_ex2(part_m[w * COLS + col] - m);
            part_w[w * COLS + col] = f, l = fmaf(part_l[w * COLS + col], f, l);
        }
        part_m[col] = m, part_l[col] = l;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < live * (DP / 4); i += WARPS * 32) {
        const int col = i / (DP / 4);
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float f = part_w[w * COLS + col];
            const float4 u = reinterpret_cast<const float4 *>(part + (w * COLS + col) * ROW)[i % (DP / 4)];
            v.x = fmaf(u.x, f, v.x), v.y = fmaf(u.y, f, v.y), v.z = fmaf(u.z, f, v.z), v.w = fmaf(u.w, f, v.w);
        }
        reinterpret_cast<float4 *>(part + col * ROW)[i % (DP / 4)] = v;
    }
    __syncthreads();
    if (a.ranks > 1) {
        // the CTAs of a cluster have a share of the item's blocks each; each adds up a share of its numbers, in the order of the ranks
        at_cluster_sync();
        const uint32_t all = static_cast<uint32_t>(__cvta_generic_to_shared(part)), all_m = all + WARPS * COLS * ROW * 4, all_l = all_m + WARPS * COLS * 4;
        for (int i = threadIdx.x * a.ranks + rank; i < live * (D / 4); i += WARPS * 32 * a.ranks) {
            const int col = i / (D / 4), d = i % (D / 4);
            float m = -INFINITY, l = 0.f;
#pragma unroll 8
            for (int r = 0; r < a.ranks; ++r) m = fmaxf(m, at_theirs(all_m + 4 * col, r));
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
            for (int r = 0; r < a.ranks; ++r) {
                const float most = at_theirs(all_m + 4 * col, r), f = most == m ? 1.f : at_ex2(most - m);
                const float4 u = at_theirs4(all + (col * ROW + 4 * d) * 4, r);
                l = fmaf(at_theirs(all_l + 4 * col, r), f, l);
                v.x = fmaf(u.x, f, v.x), v.y = fmaf(u.y, f, v.y), v.z = fmaf(u.z, f, v.z), v.w = fmaf(u.w, f, v.w);
            }
            const int c = c0 + col, at = f8_div(c, G, a.group_magic);
            const float inv = l == 0.f ? 0.f : 1.f / l;
            store4(static_cast<T *>(a.out) + ((static_cast<size_t>(b) * L + at) * a.heads + static_cast<size_t>(h) * G + c - at * G) * D + 4 * d,
                   make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
        }
        at_cluster_sync();  // nobody's memory is read any more
    } else if (mine.pieces > 1) {
        float *to = static_cast<float *>(a.workspace) + static_cast<size_t>(blockIdx.x) * (COLS * (D + 2));
        for (int i = threadIdx.x; i < live * (D / 4); i += WARPS * 32)
            reinterpret_cast<float4 *>(to)[i] = reinterpret_cast<const float4 *>(part + i / (D / 4) * ROW)[i % (D / 4)];
        if (threadIdx.x < live) to[COLS * D + threadIdx.x] = part_m[threadIdx.x], to[COLS * (D + 1) + threadIdx.x] = part_l[threadIdx.x];
    } else {
        for (int i = threadIdx.x; i < live * (D / 4); i += WARPS * 32) {
            const int col = i / (D / 4), d = i % (D / 4), c = c0 + col, l = f8_div(c, G, a.group_magic);
            const float4 v = reinterpret_cast<const float4 *>(part + col * ROW)[d];
            const float inv = part_l[col] == 0.f ? 0.f : 1.f / part_l[col];  // nothing seen: zeros
            store4(static_cast<T *>(a.out) + ((static_cast<size_t>(b) * L + l) * a.heads + static_cast<size_t>(h) * G + c - l * G) * D + 4 * d,
                   make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
        }
    }
}

// Adds up the pieces of an item that has several, up to 16 of its columns a CTA.
constexpr int kAtJoin = 512, kAtJoinColumns = 16;
template <typename T>
__global__ void __launch_bounds__(kAtJoin) fp8_attend_join_kernel(const __grid_constant__ F8Attend a, int cols) {
    extern __shared__ __align__(16) float js[];  // [pieces][16] maxima, then factors; the threads' sums
    __shared__ float sums[kAtJoinColumns];
    const tlb_fp8_pages &pg = a.pages;
    const int D = pg.dim, G = a.group, L = a.tokens, each = pg.heads * a.col_blocks, skip = blockIdx.y * kAtJoinColumns;
    const int b = f8_div(blockIdx.x, each, a.each_magic), item = static_cast<int>(blockIdx.x) - b * each, cb = f8_div(item, pg.heads, a.heads_magic), h = item - cb * pg.heads;
    const int c0 = cb * cols + skip;
    // the lengths are there: this launch begins once the one before it, which makes the pieces, is past its own wait
    int before;
    const int pieces = at_pieces_of(a, b, before);
    tl::griddep_launch();
    tl::griddep_wait();  // also without work: what follows relies on this launch ending after the one before it
    const int live = min(min(cols - skip, kAtJoinColumns), G * L - c0);
    if (pieces <= 1 || live <= 0) return;
    const int size = cols * (D + 2), quads = live * (D / 4), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const float *ws = static_cast<const float *>(a.workspace) + static_cast<size_t>(static_cast<long long>(before) * each + static_cast<long long>(item) * pieces) * size;
    const float *maxima = ws + static_cast<size_t>(cols) * D + skip, *parts = maxima + cols;
    // a column a warp: the maximum over the pieces, their factors
    for (int col = warp; col < live; col += kAtJoin / 32) {
        float m = -INFINITY, l = 0.f;
        for (int k = lane; k < pieces; k += 32) {
            const float v = tl::ld_cg(maxima + static_cast<size_t>(k) * size + col);
            js[k * kAtJoinColumns + col] = v, m = fmaxf(m, v);
        }
        m = tl::warp_max(m);
        for (int k = lane; k < pieces; k += 32) {
            const float v = js[k * kAtJoinColumns + col], f = v == m ? 1.f : at_ex2(v - m);
            js[k * kAtJoinColumns + col] = f, l = fmaf(tl::ld_cg(parts + static_cast<size_t>(k) * size + col), f, l);
        }
        l = tl::warp_sum(l);
        if (lane == 0) sums[col] = l == 0.f ? 0.f : 1.f / l;
    }
    __syncthreads();
    // groups of threads take every groups-th piece
    const int groups = max(kAtJoin / quads, 1), group = threadIdx.x / quads;
    const float *numbers = ws + static_cast<size_t>(skip) * D;
    float4 *both = reinterpret_cast<float4 *>(js + pieces * kAtJoinColumns);
    for (int q0 = 0; q0 < quads; q0 += kAtJoin) {
        const int i = groups > 1 ? threadIdx.x % quads : q0 + threadIdx.x, col = i / (D / 4), d = i % (D / 4);
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (group < groups && i < quads) {
#pragma unroll 8
            for (int k = groups > 1 ? group : 0; k < pieces; k += groups) {
                const uint4 u = tl::ld_cg(reinterpret_cast<const uint4 *>(numbers + static_cast<size_t>(k) * size) + i);
                const float f = js[k * kAtJoinColumns + col];
                v.x = fmaf(__uint_as_float(u.x), f, v.x), v.y = fmaf(__uint_as_float(u.y), f, v.y), v.z = fmaf(__uint_as_float(u.z), f, v.z), v.w = fmaf(__uint_as_float(u.w), f, v.w);
            }
        }
        if (groups > 1) {
            both[threadIdx.x] = v;
            __syncthreads();
            if (group != 0) continue;
            for (int k = 1; k < groups; ++k) {
                const float4 u = both[k * quads + i];
                v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
            }
        }
        if (i >= quads || (groups == 1 && group > 0 && quads <= kAtJoin)) continue;
        const float inv = sums[col];
        const int c = c0 + col, l = f8_div(c, G, a.group_magic);
        store4(static_cast<T *>(a.out) + ((static_cast<size_t>(b) * L + l) * a.heads + static_cast<size_t>(h) * G + c - l * G) * D + 4 * d,
               make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
    }
}

int f8_attend_join(const F8Attend &a, int cols, cudaStream_t st) {
    const unsigned items = static_cast<unsigned>(a.col_blocks) * a.pages.heads * a.batch;
    const size_t sums = static_cast<size_t>(a.most_pieces + 1) * kAtJoinColumns * 4 + kAtJoin * 16;
    const dim3 grid(items, (cols + kAtJoinColumns - 1) / kAtJoinColumns);
    const cudaError_t e = a.dtype == TL_F32 ? tl::launch_chained(fp8_attend_join_kernel<float>, grid, dim3(kAtJoin), sums, st, a, cols)
                                            : tl::launch_chained(fp8_attend_join_kernel<bf16>, grid, dim3(kAtJoin), sums, st, a, cols);
    if (e != cudaSuccess) return tl::fail(TL_ECUDA, "fp8_attention: %s", cudaGetErrorString(e));
    TL_LAUNCH_CHECK("fp8_attention (join)");
    return TL_OK;
}

// CTAs of the kernels that the GPU holds at a time, as far as the division of the work goes: two an SM, one of the wider forms.
static int attend_slots(int dtype, int dim, int rows) { return sm_count() * (dtype == TL_BF16 && dim <= 128 && rows <= 8 ? 2 : 1); }
static int attend_cols(int dim, int rows) { return dim > 128 || rows <= 8 ? 8 : 16; }
constexpr int kAtWhole = 64;  // blocks of a request that is not cut into pieces
constexpr int kAtAlone = 120 * 1024;  // of shared memory: a CTA has its SM to itself
static cudaLaunchConfig_t at_clusters(unsigned ctas, int ranks, int smem, cudaStream_t st, cudaLaunchAttribute (&attr)[2]) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(ctas), cfg.blockDim = dim3(kAtWarps * 32), cfg.dynamicSmemBytes = smem, cfg.stream = st;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ranks, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr, cfg.numAttrs = tl::use_pdl() ? 2 : 1;
    return cfg;
}
// CTAs of a cluster for so few items that all of them are on the GPU at once, an SM each; 1: no clusters.
static int attend_ranks(long long items) {
    constexpr int kMost = 8;  // of 13 one request of 1011 tokens takes 6.5 us for 6.0, of 8000 10.9 for 11.1
    static std::atomic<int> held[64][kMost + 1];  // clusters of so many CTAs that a device holds, and 1 (the division of its SMs into groups decides: 15 of 8, 33 of 4)
    int device = 0;
    if (items <= 0 || items > sm_count() / 2 || cudaGetDevice(&device) != cudaSuccess || device >= 64) return 1;
    for (int ranks = kMost; ranks > 1; --ranks) {
        int known = held[device][ranks].load(std::memory_order_relaxed);
        if (known == 0) {
            const auto kernel = fp8_attend_kernel<bf16, 128, 128, 1>;
            cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kAtAlone);
            cudaLaunchAttribute attr[2];
            const cudaLaunchConfig_t cfg = at_clusters(ranks, ranks, kAtAlone, nullptr, attr);
            int clusters = 0;
            if (cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg) != cudaSuccess) clusters = 0, cudaGetLastError();
            held[device][ranks].store(known = clusters + 1, std::memory_order_relaxed);
        }
        if (items < known) return ranks;
    }
    return 1;
}

// What decides, in microseconds beside what all have in common (bf16, 8 columns, heads of 128; other heads and columns go by the same, which nobody has fitted to them): a CTA takes 0.075 a block; a cluster's joining takes 1.8 and the
// launch that joins pieces 6.5, which stream at 6.2 TB/s whatever the lengths.  Measured, whole / clusters / pieces: one request of 100 tokens 4.3 / 5.8 / -, of 500 6.4 / 5.7 / -,
// of 1011 8.7 / 6.0 / 10.7, of 8000 - / 10.9 / 13.6, of 32000 - / 25.0 / 20.6; 8 of 8000 - / 26.4 / 30.7; 24 of 70 to 1970 17.2 / - / 19.2; 16 of 8000 45 / - / 53.  Without lengths
// clusters are for one or two requests: of more, one may be far longer than the others, which pieces make up for.
static AtPlan attend_plan(const tlb_fp8_pages &p, const tlb_fp8_attention_call &c, const AtLengths &n, bool lens) {
    const long long rows = static_cast<long long>(c.heads / p.heads) * c.tokens;
    const int cols = attend_cols(p.dim, rows <= 8 ? 8 : 9), slots = attend_slots(c.dtype, p.dim, rows <= 8 ? 8 : 9);
    const long long each = (rows + cols - 1) / cols * p.heads, items = each * c.batch;
    const int ranks = items <= 2 * sm_count() ? attend_ranks(each * n.live) : 1;  // idle slots are clusters too, which leave at once
    const bool pieces = n.longest > kAtWhole && items <= 16LL * slots;            // more items than that have no use for pieces
    const size_t workspace = static_cast<size_t>(items + slots) * at_piece_floats(cols, p.dim) * sizeof(float);
    const double whole = n.longest * (c.dtype == TL_BF16 ? 0.075 : 0.18) * (cols == 16 ? 1.3 : 1.0), clusters = ranks > 1 ? 1.8 + whole / ranks : whole,
                 cut = pieces ? 6.5 + static_cast<double>(n.blocks * each) * (2 * kF8Tokens * p.dim / 6.2e6) : whole;
    if (lens ? clusters < whole && clusters <= cut : clusters < whole && ranks == 8) return {ranks, 0, 4 + clusters, false};
    if (lens ? cut < whole : pieces) return {1, workspace, 4 + cut, false};
    // The last items come to an SM beside others, and then both are slower: let these be the short ones (24 requests of 70 to 1970 17.8 -> 16.8 us; 0.3 us where all are alike)
    const bool long_first = lens && c.batch <= 32 && items > sm_count() && n.longest * n.live > n.blocks + n.blocks / 4;
    return {1, 0, ((each * n.live + slots - 1) / slots) * (4 + whole), false, long_first};
}
// Portions of many columns go to the kernel of blocks_fp8_portion.cu unless this one is sooner through, as it is with few items, which clusters divide (16 tokens over 1000 with
// groups of 4: 9.9 us here, 22.6 there; 64 over 1000 12.7 and 24.5, over 3500 26.9 and 26.2; 8 requests of 16 over 1000 24.2 and 30.7, 32 of them 79 and 57).
static AtPlan any_plan(const tlb_fp8_pages &p, const tlb_fp8_attention_call &c, const int32_t *lens) {
    AtLengths n{static_cast<long long>(c.max_pages) * (p.page_size / kF8Tokens), 0, c.batch};
    n.blocks = n.longest * c.batch;
    if (lens) {
        n = {0, 0, 0};
        for (int b = 0; b < c.batch; ++b) {
            const long long one = (std::max(lens[b], 0) + kF8Tokens - 1LL) / kF8Tokens;
            n.longest = std::max(n.longest, one), n.blocks += one, n.live += one > 0;
        }
    }
    const AtPlan rows = attend_plan(p, c, n, lens != nullptr);
    if (!f8_portion_takes(p, c)) return rows;
    const AtPlan portion = f8_portion_plan(p, c, n);
    return rows.time < portion.time ? rows : portion;
}

template <typename T, int DP, int DIM, int NT>
static int attend_launch(F8Attend a, cudaStream_t st) {
    static tl::PerDevice ready;
    constexpr int cols = 8 * NT, joined = kAtWarps * cols * (DP + 4 + 3) * 4, most = kAtWarps * kAtStages * at_stage(DP);
    const auto kernel = fp8_attend_kernel<T, DP, DIM, NT>;
    const int rings = kAtWarps * kAtStages * at_stage(a.pages.dim), smem = rings > joined ? rings : joined;
    int device = 0;
    cudaGetDevice(&device);
    if (!ready(device, [&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, std::max(most > joined ? most : joined, kAtAlone)) == cudaSuccess; }))
        return tl::fail(TL_ECUDA, "fp8_attention: %s", cudaGetErrorString(cudaGetLastError()));
    a.col_blocks = (a.group * a.tokens + cols - 1) / cols;
    const long long items = static_cast<long long>(a.col_blocks) * a.pages.heads * a.batch;
    if (items > 0x3fffffff) return tl::fail(TL_EINVAL, "fp8_attention: sizes out of range");
    a.each_magic = f8_magic(items + a.slots, a.pages.heads * a.col_blocks);
    cudaError_t e;
    if (a.ranks > 1) {
        cudaLaunchAttribute attr[2];
        const cudaLaunchConfig_t cfg = at_clusters(static_cast<unsigned>(items * a.ranks), a.ranks, std::max(smem, kAtAlone), st, attr);
        e = cudaLaunchKernelEx(&cfg, kernel, a);
    } else {
        e = tl::launch_chained(kernel, dim3(static_cast<unsigned>(items + (a.workspace ? a.slots : 0))), dim3(kAtWarps * 32), smem, st, a);
    }
    if (e != cudaSuccess) return tl::fail(TL_ECUDA, "fp8_attention: %s", cudaGetErrorString(e));
    TL_LAUNCH_CHECK("fp8_attention");
    if (!a.workspace) return TL_OK;
    return f8_attend_join(a, cols, st);
}

template <typename T, int DP, int DIM>
static int attend_columns(const F8Attend &a, cudaStream_t st) {
    if constexpr (DP <= 128)
        if (attend_cols(DP, a.group * a.tokens) == 16) return attend_launch<T, DP, DIM, 2>(a, st);
    return attend_launch<T, DP, DIM, 1>(a, st);
}

template <typename T>
static int attend_any(F8Attend a, bool portion, cudaStream_t st) {
    const int D = a.pages.dim;
    a.wide_rows = tl::aligned16(a.q) && ((a.q_b | a.q_h | a.q_l) * static_cast<long long>(sizeof(T)) & 15) == 0;
    a.page_blocks = a.pages.page_size / kF8Tokens;
    a.page_magic = f8_magic(static_cast<unsigned long long>(a.max_pages) * a.page_blocks + 64, a.page_blocks);  // the first pages are looked up ahead of the length
    a.group_magic = f8_magic(static_cast<unsigned long long>(a.group) * a.tokens, a.group);
    a.heads_magic = f8_magic(static_cast<unsigned long long>(a.pages.heads) * ((a.group * a.tokens + 7) / 8), a.pages.heads);
    a.slots = attend_slots(a.dtype, D, a.group * a.tokens), a.most_pieces = 128, a.whole = kAtWhole;
    if (portion) return f8_portion(a, st);
    if (D <= 64) return D == 64 ? attend_columns<T, 64, 64>(a, st) : attend_columns<T, 64, 0>(a, st);
    if (D <= 128) return D == 128 ? attend_columns<T, 128, 128>(a, st) : attend_columns<T, 128, 0>(a, st);
    return attend_launch<T, 256, 0, 1>(a, st);
}

}  // namespace tlb

using namespace tlb;

extern "C" size_t tlb_fp8_attention_workspace(const tlb_fp8_pages *pages, const tlb_fp8_attention_call *c, const int32_t *lens_host) {
    if (f8_check_pages("fp8_attention", pages) != TL_OK || !c || c->heads <= 0 || c->tokens <= 0 || c->batch <= 0) return 0;
    return any_plan(*pages, *c, lens_host).workspace;
}

extern "C" int tlb_fp8_attention(const tlb_fp8_pages *pages, const tlb_fp8_attention_call *c, const int32_t *lens_host, const int32_t *table_host, void *workspace,
                                 size_t workspace_bytes, void *stream) {
    const int rc = f8_check_pages("fp8_attention", pages);
    if (rc != TL_OK) return rc;
    if (!c || c->batch < 0 || c->tokens < 0 || c->heads <= 0 || c->heads % pages->heads) return tl::fail(TL_EINVAL, "fp8_attention: query heads over %d key/value heads", pages->heads);
    if (c->batch == 0 || c->tokens == 0) return TL_OK;
    if (c->max_pages <= 0 || static_cast<long long>(c->heads / pages->heads) * c->tokens > (1 << 30)) return tl::fail(TL_EINVAL, "fp8_attention: sizes out of range");
    if (!c->q || !c->out || !c->table || !c->lens) return tl::fail(TL_EINVAL, "fp8_attention: missing argument");
    if (const int bad = f8_check_step("fp8_attention", *pages, lens_host, table_host, c->batch, c->max_pages, c->tokens)) return bad;
    const AtPlan plan = any_plan(*pages, *c, lens_host);
    if (lens_host && !workspace && plan.workspace) return tl::fail(TL_EWORKSPACE, "fp8_attention: a workspace is needed");
    if (workspace && plan.workspace && (workspace_bytes < plan.workspace || !tl::aligned16(workspace)))
        return tl::fail(TL_EWORKSPACE, "fp8_attention: the workspace must have %zu bytes, from a boundary of 16 on", plan.workspace);
    F8Attend a(*pages, *c, plan.workspace ? workspace : nullptr);  // without one no item is in pieces
    a.ranks = plan.ranks, a.long_first = plan.long_first;
    TLB_DISPATCH(c->dtype, "fp8_attention", return attend_any<T>(a, plan.portion, as_stream(stream)));
}
