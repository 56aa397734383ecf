// Rows of e4m3 numbers times a matrix of them on the 5th-generation tensor cores: tcgen05.mma (kind::f8f6f4) fed by TMA.
//
//   out[t, n] = sum over blocks b of 128 of  sx[b, t] * sw[n / 128, b] * (sum over k in b of q[t, k] w[n, k])
//
// The inner sum is exact products added in the tensor cores, over one block at a time: four instructions of 32, into an accumulator that
// starts from zero.  The outer sum is kept in registers, in fp32: the epilogue's warps take every block's accumulator out of tensor memory
// and add it times the two scales.  128 rows of the matrix are a tile's M side (a lane each, and one scale for all of them), BN tokens its
// N side, so the second scale is a column's: a warp has its columns' products of scales in shared memory, a broadcast read for four.
//
// Warps: 0 and 3 TMA of the matrix and of the rows (boxes of 128 bytes, 128-byte swizzle: one block of the reduction a stage), 1 the products, the sums from 4 on: 8, or 16
// above 64 tokens, where a block's accumulator would otherwise wait for its turn in two long chains of reads of tensor memory.
//
// Few tokens make few tiles: then the CTAs of a cluster share a tile's blocks and add their sums through each other's shared memory, every
// sum in rank order, so no memory and no atomics stand between two launches, and the result does not depend on their timing.
//
// Up to four rows are rounded in this launch, by every CTA its own blocks of them: a launch less (1 row of 2560 -> 6144: 9.0 -> 7.8 us).
//
// 1 row of 2560 -> 6144: 7.8 us, 2.0 TB/s, one latency behind another (rows, their rounding, the first boxes, a cluster's sums); of 2560 -> 151936: 63 us, 6.15 TB/s,
// bound by HBM.  24 rows of 4096 -> 2560: 9.5 us with the rounding's launch.  Above 64 tokens a block takes 0.56 us of an SM, bound as the pairs' kernel is by the way
// round from a finished accumulator to an empty one.
#include <algorithm>

#include "blocks_fp8.cuh"
#include "blocks_tc.cuh"
#include "../per_device.h"

namespace tlb {

constexpr int kF8WeightBytes = 128 * 128;

// Where the rows come from: rounded by a launch before, or (few rows) rounded here, by every CTA its own blocks of them, once for all its tiles.
constexpr int kF8Tma = 0, kF8Plain = 1, kF8Gated = 2;
constexpr int kF8OwnRows = 8, kF8OwnBlocks = 32;  // the most rows, and blocks of the reduction of a CTA

template <int BN, bool OWN>
struct F8Tile {
    static constexpr int kStage = kF8WeightBytes + (OWN ? 0 : BN * 128);
    static constexpr int kPerSm = BN <= 64 ? 2 : 1;
    static constexpr int kSumWarps = BN <= 64 ? 8 : 16, kThreads = (4 + kSumWarps) * 32;
    static constexpr int kCols = BN / (kSumWarps / 4);  // of a warp
    static constexpr int kBuffers = 4;           // accumulators
    static constexpr int kTmem = BN * kBuffers;  // columns: 64, 128, 256, 512
    static constexpr int kFactors = kSumWarps * kCols * 4;
    static constexpr int kOwn = OWN ? kF8OwnBlocks * kF8OwnRows * (kF8Block + 4) : 0;  // rows that the kernel rounds itself, and their scales
    static constexpr int kStages = std::min(8, (227 * 1024 / kPerSm - 1024 - kFactors - kOwn - 512) / kStage);
    static constexpr int kSmem = kStages * kStage + kFactors + kOwn + 256;
};

struct F8Args {
    F8Rows x;  // kF8Own: the rows as they come; of it x, ldx, gated, act, limit, slope
    const float *sx, *sw;
    const void *bias;
    void *out;
    int ld_sx, rows, n, k_blocks, m_blocks, tiles, splits;
    int second;  // the launch before is one of these products or the rows' rounding, which waited for what was before it: the matrix is older than both
};

// C consecutive columns (8 or 16) of the warp's lanes, without the wait.
__device__ __forceinline__ void f8_ld(uint32_t at, uint32_t (&v)[8]) { tc_ld8(at, v); }
__device__ __forceinline__ void f8_ld(uint32_t at, uint32_t (&v)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]),
                   "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                 : "r"(at)
                 : "memory");
}
// A block's four products of 32 into `d`, from zero, their completion reported to `done` (the accumulator is full) and `used` (the stage may be written), and whether
// two barriers' phases are over.  Asking a barrier takes 180 cycles, whatever the answer: the questions for the next block are on their way while this one's
// products are issued, and their answers are looked at last.
__device__ __forceinline__ void f8_block(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t done, uint32_t used, uint32_t bar0, uint32_t parity0, uint32_t bar1,
                                         uint32_t parity1, uint32_t &over0, uint32_t &over1) {
    asm volatile(
        "{\n\t.reg .pred p, q, on, off;\n\t.reg .b64 a1, a2, a3, b1, b2, b3;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%8], %9;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 q, [%10], %11;\n\t"
        "setp.eq.u32 on, %2, %2;\n\tsetp.ne.u32 off, %2, %2;\n\t"
        "add.u64 a1, %3, 2;\n\tadd.u64 a2, %3, 4;\n\tadd.u64 a3, %3, 6;\n\tadd.u64 b1, %4, 2;\n\tadd.u64 b2, %4, 4;\n\tadd.u64 b3, %4, 6;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%2], %3, %4, %5, off;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%2], a1, b1, %5, on;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%2], a2, b2, %5, on;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%2], a3, b3, %5, on;\n\t"
        "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%6];\n\t"
        "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%7];\n\t"
        "selp.u32 %0, 1, 0, p;\n\tselp.u32 %1, 1, 0, q;\n\t}"
        : "=r"(over0), "=r"(over1)
        : "r"(d), "l"(a), "l"(b), "r"(idesc), "r"(done), "r"(used), "r"(bar0), "r"(parity0), "r"(bar1), "r"(parity1)
        : "memory");
}
// e4m3 x e4m3 -> f32, 128 rows, n columns, both K-major
__host__ __device__ constexpr uint32_t f8_idesc(int n) { return (1u << 4) | (static_cast<uint32_t>(n >> 3) << 17) | (8u << 24); }

// Four numbers of a row from column k on, zero behind the last one; of gated rows (fp32, 128 of the gate and 128 of the up projection in turn) the gated ones.
template <typename X, int ROWS>
__device__ __forceinline__ float4 f8_four(const F8Rows &r, int row, int k, bool whole) {
    const X *from = static_cast<const X *>(r.x) + (size_t)row * r.ldx;
    if constexpr (ROWS == kF8Gated) {
        const int at = k / kF8Block * 2 * kF8Block + k % kF8Block;
        const uint4 g = tl::ld_cg(reinterpret_cast<const uint4 *>(from + at)), u = tl::ld_cg(reinterpret_cast<const uint4 *>(from + at + kF8Block));
        auto pair = [&](uint32_t a, uint32_t b, int i) { return k + i < r.cols ? gated_pair(__uint_as_float(a), __uint_as_float(b), r.act, r.limit, r.slope) : 0.f; };
        return make_float4(pair(g.x, u.x, 0), pair(g.y, u.y, 1), pair(g.z, u.z, 2), pair(g.w, u.w, 3));
    } else if (whole && k + 4 <= r.cols) {
        if constexpr (sizeof(X) == 4) {
            const uint4 v = tl::ld_cg(reinterpret_cast<const uint4 *>(from + k));
            return make_float4(__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w));
        } else {
            uint2 v;
            asm volatile("ld.global.cg.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(from + k) : "memory");
            const float2 a = tl::unpack2<X>(v.x), b = tl::unpack2<X>(v.y);
            return make_float4(a.x, a.y, b.x, b.y);
        }
    } else {
        float v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = k + i < r.cols ? to_f(tl::ld_cg(from + k + i)) : 0.f;
        return make_float4(v[0], v[1], v[2], v[3]);
    }
}

template <typename T, int BN, int ROWS = kF8Tma, typename X = T>
__global__ void __launch_bounds__(F8Tile<BN, ROWS != kF8Tma>::kThreads, F8Tile<BN, ROWS != kF8Tma>::kPerSm)
fp8_product_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_q, const F8Args a) {
    constexpr bool OWN = ROWS != kF8Tma;
    using Tile = F8Tile<BN, OWN>;
    constexpr int COLS = Tile::kCols, STEP = COLS < 16 ? 8 : 16;  // columns of a warp, of one read of tensor memory
    extern __shared__ __align__(1024) unsigned char f8_smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t base = g_smem_u32(f8_smem);
    const uint32_t own = base + Tile::kStages * Tile::kStage;  // [block][8 rows of 128 bytes, in the swizzled order]
    float *own_scales = reinterpret_cast<float *>(f8_smem + Tile::kStages * Tile::kStage + (OWN ? kF8OwnBlocks * kF8OwnRows * kF8Block : 0));  // [block][8]
    float *factors = reinterpret_cast<float *>(f8_smem + Tile::kStages * Tile::kStage + Tile::kOwn);
    const uint32_t bars = base + Tile::kStages * Tile::kStage + Tile::kFactors + Tile::kOwn;
    const uint32_t full = bars, empty = full + 64, acc_full = empty + 64, acc_empty = acc_full + 32, rows_there = acc_empty + 32;
    volatile int *dead = reinterpret_cast<volatile int *>(f8_smem + Tile::kStages * Tile::kStage + Tile::kFactors + Tile::kOwn + 200);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(const_cast<int *>(dead)) + 1;

    if (warp == 0 && lane == 0) {
        for (int i = 0; i < Tile::kStages; ++i) g_mbar_init(full + 8 * i, OWN ? 1 : 2), g_mbar_init(empty + 8 * i, 1);  // full: either kind of copies
        g_mbar_init(rows_there, 10);
        for (int i = 0; i < Tile::kBuffers; ++i) g_mbar_init(acc_full + 8 * i, 1), g_mbar_init(acc_empty + 8 * i, Tile::kSumWarps);
        *dead = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_w) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_q) : "memory");
    }
    if (warp == 2) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(g_smem_u32(tmem_slot)), "n"(Tile::kTmem) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    g_tc_fence_before();
    __syncthreads();
    g_tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if constexpr (OWN) {  // a second product of a feed-forward may ask for its matrix meanwhile
        if (!a.second) tl::griddep_wait();
        tl::griddep_launch();
    }
    const int rank = blockIdx.x % a.splits, first = blockIdx.x / a.splits, step = gridDim.x / a.splits;
    const int kb0 = (int)((long long)a.k_blocks * rank / a.splits), kb1 = (int)((long long)a.k_blocks * (rank + 1) / a.splits);

    // A thread by itself for each role: with the whole warp in the loop a block cost twice the cycles.
    if constexpr (OWN) {
        if (warp >= 2) {  // the rows of this CTA's blocks, one of either a warp at a time, two on their way
            const bool whole = ROWS == kF8Gated || (a.x.ldx % 4 == 0 && (reinterpret_cast<uintptr_t>(a.x.x) & (4 * sizeof(X) - 1)) == 0);
            if (a.second) tl::griddep_wait();
            const int blocks = kb1 - kb0, pieces = a.rows * blocks;
            for (int i0 = warp - 2; i0 < pieces; i0 += 20) {
                float4 v[2];
#pragma unroll
                for (int u = 0; u < 2; ++u)
                    if (i0 + 10 * u < pieces) v[u] = f8_four<X, ROWS>(a.x, (i0 + 10 * u) / blocks, (kb0 + (i0 + 10 * u) % blocks) * kF8Block + lane * 4, whole);
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    if (i0 + 10 * u >= pieces) break;
                    const int t = (i0 + 10 * u) / blocks, b = (i0 + 10 * u) % blocks;
                    // magnitudes are in the order of their bits, an infinity above all numbers and a NaN above that
                    const uint32_t most = __reduce_max_sync(0xffffffffu, max(max(__float_as_uint(v[u].x) & 0x7fffffffu, __float_as_uint(v[u].y) & 0x7fffffffu),
                                                                             max(__float_as_uint(v[u].z) & 0x7fffffffu, __float_as_uint(v[u].w) & 0x7fffffffu)));
                    const F8Scale f = f8_scale(__uint_as_float(most));
                    if (lane == 0) own_scales[b * kF8OwnRows + t] = f.scale;
                    const uint32_t q = f8_pack4(__fmul_rn(v[u].x, f.times), __fmul_rn(v[u].y, f.times), __fmul_rn(v[u].z, f.times), __fmul_rn(v[u].w, f.times));
                    *reinterpret_cast<uint32_t *>(f8_smem + Tile::kStages * Tile::kStage + (b * kF8OwnRows + t) * kF8Block + (((lane >> 2) ^ t) << 4) + (lane & 3) * 4) = q;
                }
            }
            tl::g_fence_proxy_async();
            __syncwarp();
            if (lane == 0) g_mbar_arrive(rows_there);
            asm volatile("bar.sync 1, 320;" ::: "memory");  // the scales, for the warps that add
        }
    }
    if (warp == 0 || (!OWN && warp == 3)) {  // the matrix's copies and the rows'
        if (g_elect_one()) {
            int s = 0;
            uint32_t ph = 1;
            bool ok = true;
            if (warp == 3 || !a.second) tl::griddep_wait();
            for (int tile = first; ok && tile < a.tiles; tile += step)
                for (int kb = kb0; kb < kb1; ++kb) {
                    if (!(ok = tc_wait_one(empty + 8 * s, ph, dead))) break;
                    g_mbar_expect_tx(full + 8 * s, warp == 0 ? kF8WeightBytes : BN * 128);
                    if (warp == 0) g_tma_load_2d(base + s * Tile::kStage, &map_w, kb * 128, tile % a.m_blocks * 128, full + 8 * s);
                    else g_tma_load_2d(base + s * Tile::kStage + kF8WeightBytes, &map_q, kb * 128, tile / a.m_blocks * BN, full + 8 * s);
                    if (++s == Tile::kStages) s = 0, ph ^= 1u;
                }
        }
    } else if (warp == 1) {
        if (g_elect_one()) {
            int s = 0, buf = 0;
            uint32_t ph = 0, acc_ph = 1;
            bool ok = !OWN || tc_wait_one(rows_there, 0, dead);
            uint32_t acc_free = 0, there = 0;  // of the next block's, as far as is known
            for (int tile = first; ok && tile < a.tiles; tile += step)
                for (int kb = kb0; kb < kb1; ++kb) {
                    if (!(ok = (acc_free || tc_wait_one(acc_empty + 8 * buf, acc_ph, dead)) && (there || tc_wait_one(full + 8 * s, ph, dead)))) break;
                    g_tc_fence_after();
                    const uint64_t w = g_smem_desc_sw128(base + s * Tile::kStage, 0, 1024),
                                   // own rows: columns 8-15 are what lies behind the block, and not used
                                   q = OWN ? g_smem_desc_sw128(own + (kb - kb0) * kF8OwnRows * kF8Block, 0, 1024) : g_smem_desc_sw128(base + s * Tile::kStage + kF8WeightBytes, 0, 1024);
                    const uint32_t d = tmem + buf * BN, done = acc_full + 8 * buf, used = empty + 8 * s;
                    if (++s == Tile::kStages) s = 0, ph ^= 1u;
                    if (++buf == Tile::kBuffers) buf = 0, acc_ph ^= 1u;
                    f8_block(d, w, q, f8_idesc(BN), done, used, acc_empty + 8 * buf, acc_ph, full + 8 * s, ph, acc_free, there);
                }
        }
    } else if (warp >= 4) {
        const int quarter = warp & 3, part = (warp - 4) >> 2;
        float *mine = factors + (warp - 4) * COLS;
        int buf = 0;
        uint32_t acc_ph = 0;
        tl::griddep_wait();
        for (int tile = first; tile < a.tiles; tile += step) {
            const int m = tile % a.m_blocks, col0 = tile / a.m_blocks * BN + part * COLS, f = m * 128 + quarter * 32 + lane;
            constexpr int PER = (COLS + 31) / 32;
            float acc[COLS], next[PER], next_w = 0.f;
#pragma unroll
            for (int i = 0; i < COLS; ++i) acc[i] = 0.f;
            auto fetch = [&](int kb) {
                next_w = a.sw[(size_t)m * a.k_blocks + kb];
#pragma unroll
                for (int i = 0; i < PER; ++i) {
                    const int c = lane + 32 * i;
                    if constexpr (!OWN) next[i] = c < COLS && col0 + c < a.rows ? tl::ld_cg(a.sx + (size_t)kb * a.ld_sx + col0 + c) : 0.f;
                }
            };
            if (kb0 < kb1) fetch(kb0);
            bool ok = true;
            for (int kb = kb0; kb < kb1; ++kb) {
                if constexpr (!OWN) {
#pragma unroll
                    for (int i = 0; i < PER; ++i)
                        if (lane + 32 * i < COLS) mine[lane + 32 * i] = next[i] * next_w;
                    if (kb + 1 < kb1) fetch(kb + 1);
                    __syncwarp();
                    ok &= tc_wait(acc_full + 8 * buf, acc_ph, dead);
                } else {  // the block's scales were written before its products
                    const float this_w = next_w;
                    if (kb + 1 < kb1) fetch(kb + 1);
                    ok &= tc_wait(acc_full + 8 * buf, acc_ph, dead);
                    if (lane < COLS) mine[lane] = col0 + lane < a.rows ? own_scales[(kb - kb0) * kF8OwnRows + col0 + lane] * this_w : 0.f;
                    __syncwarp();
                }
                g_tc_fence_after();
                const uint32_t at = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + buf * BN + part * COLS;
#pragma unroll
                for (int c = 0; c < COLS; c += STEP) {
                    uint32_t v[STEP];
                    f8_ld(at + c, v);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                    for (int i = 0; i < STEP; i += 4) {
                        const float4 s4 = *reinterpret_cast<const float4 *>(mine + c + i);
                        acc[c + i] = fmaf(__uint_as_float(v[i]), s4.x, acc[c + i]);
                        acc[c + i + 1] = fmaf(__uint_as_float(v[i + 1]), s4.y, acc[c + i + 1]);
                        acc[c + i + 2] = fmaf(__uint_as_float(v[i + 2]), s4.z, acc[c + i + 2]);
                        acc[c + i + 3] = fmaf(__uint_as_float(v[i + 3]), s4.w, acc[c + i + 3]);
                    }
                }
                g_tc_fence_before();
                __syncwarp();
                if (lane == 0) g_mbar_arrive(acc_empty + 8 * buf);
                if (++buf == Tile::kBuffers) buf = 0, acc_ph ^= 1u;
            }
            const float bad = tc_verdict(ok, dead);
            if (a.splits == 1) {
                const float b = a.bias && f < a.n ? to_f(static_cast<const T *>(a.bias)[f]) : 0.f;
                T *out = static_cast<T *>(a.out) + (size_t)col0 * a.n + f;
#pragma unroll
                for (int c = 0; c < COLS; ++c)
                    if (f < a.n && col0 + c < a.rows) out[(size_t)c * a.n] = from_f<T>((acc[c] + b) * bad);
            } else {  // the stages are done with: the last accumulator came behind all products
                float *sums = reinterpret_cast<float *>(f8_smem) + part * COLS * 128 + quarter * 32 + lane;
#pragma unroll
                for (int c = 0; c < COLS; ++c) sums[c * 128] = acc[c] * bad;
            }
        }
    }
    __syncwarp();  // also behind a role whose wait gave up
    if (a.splits > 1) {  // one tile a cluster; a CTA adds its share of the tokens
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        const int share = BN / a.splits, m = first % a.m_blocks, col0 = first / a.m_blocks * BN + rank * share;
        for (int i = threadIdx.x; i < share * 32; i += Tile::kThreads) {
            const int c = i >> 5, f = m * 128 + (i & 31) * 4, at = ((rank * share + c) * 128 + (i & 31) * 4) * 4;
            if (col0 + c >= a.rows) break;
            float sum[4] = {};
            for (int p = 0; p < a.splits; ++p) {
                float v[4];
                asm volatile("{\n\t.reg .b32 ra;\n\tmapa.shared::cluster.u32 ra, %4, %5;\n\tld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [ra];\n\t}"
                             : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3])
                             : "r"(base + at), "r"(p)
                             : "memory");
#pragma unroll
                for (int j = 0; j < 4; ++j) sum[j] += v[j];
            }
            const float bad = tc_verdict(true, dead);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (f + j < a.n) static_cast<T *>(a.out)[(size_t)(col0 + c) * a.n + f + j] = from_f<T>((sum[j] + (a.bias ? to_f(static_cast<const T *>(a.bias)[f + j]) : 0.f)) * bad);
        }
        __syncwarp();
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
    g_tc_fence_before();
    __syncthreads();
    if (warp == 2) {
        tc_settle(dead);
        g_tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(Tile::kTmem) : "memory");
    }
}

// The CTAs that share a tile's blocks, so that few tiles fill the SMs; two blocks each at least.
static int f8_splits(long long tiles, int k_blocks, int room) {
    int splits = 1;
    while (splits < 8 && tiles * splits * 2 <= room && k_blocks >= 4 * splits) splits *= 2;
    return splits;
}

template <typename T, int BN, int ROWS = kF8Tma, typename X = T>
static int f8_launch(const F8Product &p, cudaStream_t st, const F8Rows *x = nullptr) {
    using Tile = F8Tile<BN, ROWS != kF8Tma>;
    static_assert(Tile::kStages >= 3 && Tile::kStages <= 8 && Tile::kStages * Tile::kStage >= BN * 128 * 4, "the sums of a split tile lie over the stages");
    CUtensorMap mw, mq;
    if (int e = tc_map_bytes(&mw, p.w, p.ldw, p.n, p.ldw, 128)) return e;
    if (ROWS != kF8Tma) mq = mw;  // not read
    else if (int e = tc_map_bytes(&mq, p.q, p.ldq, p.rows, p.ldq, BN)) return e;
    F8Args a{x ? *x : F8Rows{}, p.sx, p.sw, p.bias, p.out, p.ld_sx, p.rows, p.n, ceil_div(p.k, kF8Block), ceil_div(p.n, 128), 0, 1, ROWS != kF8Plain};
    const long long tiles = (long long)a.m_blocks * ceil_div(p.rows, BN);
    if (tiles > 0x3fffffff) return tl::fail(TL_EINVAL, "fp8_product: too large");
    a.tiles = (int)tiles;
    const int room = sm_count() * Tile::kPerSm;
    a.splits = f8_splits(tiles, a.k_blocks, room);
    static tl::PerDevice ready;
    int device = 0;
    cudaGetDevice(&device);
    if (!ready(device, [&] { return cudaFuncSetAttribute(fp8_product_kernel<T, BN, ROWS, X>, cudaFuncAttributeMaxDynamicSharedMemorySize, Tile::kSmem) == cudaSuccess; })) {
        cudaGetLastError();
        return tl::fail(TL_ECUDA, "fp8_product: no shared memory");
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(a.splits > 1 ? tiles * a.splits : std::min<long long>(tiles, room)));
    cfg.blockDim = dim3(Tile::kThreads);
    cfg.dynamicSmemBytes = Tile::kSmem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = a.splits, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = tl::use_pdl() ? 2 : 1;
    cudaLaunchKernelEx(&cfg, fp8_product_kernel<T, BN, ROWS, X>, mw, mq, a);
    TL_LAUNCH_CHECK("fp8_product");
    return TL_OK;
}

// Which kernel, by the time that its rounds of tiles take: blocks of a CTA one after another, times what one takes, by measurement over 200 to 700 rows of 2560 to
// 9728 numbers and 2560 to 19456 outputs (us a block: 32 tokens 0.48, 64 0.66, 128 0.56, a pair's 256 x 256 0.58).  Up to 128 rows the smallest tile that holds them
// all, which reads the matrix once, was the fastest throughout.
static int f8_tile(const F8Product &p) {
    for (int bn : {16, 32, 64, 128})
        if (p.rows <= bn) return bn;
    const int k_blocks = ceil_div(p.k, kF8Block), sms = sm_count();
    const struct {
        int tokens, outputs, room;
        float block;
    } kinds[] = {{32, 128, 2 * sms, 0.48f}, {64, 128, 2 * sms, 0.66f}, {128, 128, sms, 0.56f}};
    int best = 256;
    float least = f8_pairs_width(p.rows, p.n).block * k_blocks;
    for (const auto &t : kinds) {
        const long long tiles = (long long)ceil_div(p.n, t.outputs) * ceil_div(p.rows, t.tokens);
        const int splits = f8_splits(tiles, k_blocks, t.room);
        const float time = (float)((tiles * splits + t.room - 1) / t.room) * ceil_div(k_blocks, splits) * t.block;
        if (time < least) least = time, best = t.tokens;
    }
    return best;
}

int f8_product(const F8Product &p, cudaStream_t st) {
    const int tile = f8_tile(p);
    if (tile == 256) return f8_pairs(p, st);
    TLB_DISPATCH(p.dtype, "fp8_product", return tile == 16 ? f8_launch<T, 16>(p, st) : tile == 32 ? f8_launch<T, 32>(p, st) : tile == 64 ? f8_launch<T, 64>(p, st)
                                                                                                               : f8_launch<T, 128>(p, st));
    return TL_OK;
}

// The rows as they come, rounded by the product's own warps, whose blocks of a CTA have to fit beside its stages: one launch in place of two.  2560 -> 6144, us with
// one launch and two: 1 row 7.8 and 9.0, 4 rows 8.6 and 9.3, 8 rows 10.1 and 9.5.
bool f8_own(const F8Product &p) {
    const int k_blocks = ceil_div(p.k, kF8Block);
    return p.rows <= 4 && ceil_div(k_blocks, f8_splits(ceil_div(p.n, 128), k_blocks, 2 * sm_count())) <= kF8OwnBlocks;
}
int f8_product_own(const F8Product &p, const F8Rows &x, cudaStream_t st) {
    if (x.gated) TLB_DISPATCH(p.dtype, "fp8_product", return (f8_launch<T, 16, kF8Gated, float>(p, st, &x)));
    else if (x.dtype == p.dtype) TLB_DISPATCH(p.dtype, "fp8_product", return (f8_launch<T, 16, kF8Plain, T>(p, st, &x)));
    else return (f8_launch<float, 16, kF8Plain, bf16>(p, st, &x));  // the first product of a feed-forward
    return TL_OK;
}

long long f8_gave_up() {
    const long long one = tl::read_gave_up(), pairs = f8_pairs_gave_up();
    return one < 0 || pairs < 0 ? -1 : one + pairs;
}

}  // namespace tlb
