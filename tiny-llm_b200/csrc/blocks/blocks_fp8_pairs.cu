// Many rows of e4m3 numbers times a matrix of them, on pairs of CTAs (tcgen05.mma, cta_group::2, kind::f8f6f4).
//
// What is computed is blocks_fp8_product.cu's sum over blocks of 128.  A tile is 256 tokens by 256 rows of the matrix (or 224, 192, 160: f8_pairs_width); either CTA
// of a pair loads its 128 tokens and half of the matrix rows, 32 KB for a block's 512 cycles of tensor work (one CTA by itself would load 48 KB: more than L2
// hands an SM in that time).  The tokens are the M side: a token's scale is a lane's and a block scale holds for a run of columns, so taking a block's accumulator
// over into the sums, which live in registers, is one multiply-add an entry.  Eight warps do it, 128 columns each (16 warps with 64 took 30 % longer: the SM's issue
// slots went into what a warp does a block beside the multiply-adds; two multiply-adds an instruction, fma.rn.f32x2, took longer than two).  Two accumulators of
// all columns (three of 160) take turns: one is multiplied into while another is taken over; asking the sums' barrier ahead as the products' thread does changed nothing.
//
// 8192 x 4096 -> 9472: 306 us, 2070 TF/s; 4096 x 9728 -> 2560: 142 us with the rounding (1440 TF/s: 192 tiles of 224 for 74 pairs are three rounds for 2.6).  Bound by
// the way round from a finished accumulator to an empty one (0.62 us a block where its products alone take 0.3): the wait, two trips to tensor memory, the word back.
//
// 12 warps: 0 and 3 TMA, 1 the products (leader) or the news that the own stage is there (peer), 4-11 the sums.  The first four give registers to the others.
//
// kGated: the matrix rows are 128 of a gate and the 128 of an up projection that belong to them; a thread then has both of 64 features of its token, and what
// is stored are the gated rows, rounded to e4m3 with one scale for the 128, which two warps find together.
#include <algorithm>
#include <cmath>

#include "blocks_fp8.cuh"
#include "blocks_tc.cuh"
#include "../per_device.h"

namespace tlb {

constexpr int kPrSumWarps = 8;
constexpr int kPrThreads = (4 + kPrSumWarps) * 32;
constexpr int kPrStages = 6;
constexpr int kPrStage = 2 * 128 * 128;
constexpr int kPrOutStride = 68, kPrOut = 32 * kPrOutStride;  // a warp's staging rows: 64 bytes, and 4 that keep the lanes' words in different banks
constexpr int kPrMost = 2 * 128 * 4;                          // kGated: the two warps' maxima of every token
constexpr int kPrSmem = kPrStages * kPrStage + kPrSumWarps * kPrOut + kPrMost + 256;

struct F8PairArgs {
    const float *sx, *sw;
    const void *bias;
    void *out;
    int ld_sx, rows, n, k_blocks, m_tiles, tiles;
    bool aligned;  // rows of `out` are whole 32-byte pieces
    // kGated
    uint8_t *q;
    float *scales;
    int ldq, ld_scales, ff, act;
    float limit, slope;
};

__device__ __forceinline__ uint32_t pr_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// A block's four products of 32 into `d`, from zero, their completion reported to both CTAs' `done` (the accumulator is full) and `used` (the stage may be
// written), and whether two barriers' phases are over.  Asking a barrier takes 180 cycles, whatever the answer: the questions for the next block are on their way
// while this one's products are issued, and their answers are looked at last.
template <int N>
__device__ __forceinline__ void pr_block(uint32_t d, uint64_t a, uint64_t b, uint32_t done, uint32_t used, uint32_t bar0, uint32_t parity0, uint32_t bar1, uint32_t parity1,
                                         uint32_t &over0, uint32_t &over1) {
    constexpr uint32_t idesc = (1u << 4) | (static_cast<uint32_t>(N >> 3) << 17) | ((256u >> 4) << 24);  // e4m3 x e4m3 -> f32, 256 x N, both K-major
    asm volatile(
        "{\n\t.reg .pred p, q, on, off;\n\t.reg .b64 a1, a2, a3, b1, b2, b3;\n\t.reg .b16 both;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%8], %9;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 q, [%10], %11;\n\t"
        "setp.eq.u32 on, %2, %2;\n\tsetp.ne.u32 off, %2, %2;\n\t"
        "add.u64 a1, %3, 2;\n\tadd.u64 a2, %3, 4;\n\tadd.u64 a3, %3, 6;\n\tadd.u64 b1, %4, 2;\n\tadd.u64 b2, %4, 4;\n\tadd.u64 b3, %4, 6;\n\tmov.b16 both, 3;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%2], %3, %4, %5, off;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%2], a1, b1, %5, on;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%2], a2, b2, %5, on;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%2], a3, b3, %5, on;\n\t"
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%6], both;\n\t"
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%7], both;\n\t"
        "selp.u32 %0, 1, 0, p;\n\tselp.u32 %1, 1, 0, q;\n\t}"
        : "=r"(over0), "=r"(over1)
        : "r"(d), "l"(a), "l"(b), "r"(idesc), "r"(done), "r"(used), "r"(bar0), "r"(parity0), "r"(bar1), "r"(parity1)
        : "memory");
}
__device__ __forceinline__ void pr_store32(void *p, const uint32_t (&v)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}

template <int COLS>
__device__ __forceinline__ void pr_ld(uint32_t at, uint32_t (&v)[32]) {  // without the wait
    if constexpr (COLS == 32) tl::g_tmem_ld32_nowait(at, v);
    else if constexpr (COLS == 16)
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                     : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]),
                       "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                     : "r"(at)
                     : "memory");
}

template <typename T, bool GATED, int N>
__global__ void __launch_bounds__(kPrThreads, 1)
fp8_pairs_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_w, const F8PairArgs a) {
    static_assert(N % 32 == 0 && N >= 160 && N <= 256 && (!GATED || N == 256), "an accumulator's second run");
    extern __shared__ __align__(1024) unsigned char pr_smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rank = (int)pr_rank();
    const int unit = blockIdx.x >> 1, units = gridDim.x >> 1;
    const uint32_t base = g_smem_u32(pr_smem);
    constexpr int kBars = kPrStages * kPrStage + kPrSumWarps * kPrOut + kPrMost;
    const uint32_t full = base + kBars, empty = full + 8 * kPrStages, acc_full = empty + 8 * kPrStages, acc_empty = acc_full + 32;
    constexpr int BUFFERS = N == 160 ? 3 : 2, APART = N == 160 ? 160 : 256;  // accumulators, of 512 columns
    volatile int *dead = reinterpret_cast<volatile int *>(pr_smem + kBars + 16 * kPrStages + 64);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(const_cast<int *>(dead)) + 1;
    if (warp == 1 && lane == 0) {
        for (int i = 0; i < kPrStages; ++i) g_mbar_init(full + 8 * i, rank == 0 ? 3 : 2), g_mbar_init(empty + 8 * i, 1);  // both kinds of copies, and on the leader's the peer's word
        for (int i = 0; i < BUFFERS; ++i) g_mbar_init(acc_full + 8 * i, 1), g_mbar_init(acc_empty + 8 * i, 2 * kPrSumWarps);  // both CTAs' warps, on the leader's
        *dead = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_q) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_w) : "memory");
    }
    if (warp == 2) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(g_smem_u32(tmem_slot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    g_tc_fence_before();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");  // both CTAs' barriers are ready
    g_tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    auto arrive_leader = [&](uint32_t bar) {  // what it reports is in the arriving CTA's own memory, ordered there
        asm volatile("{\n\t.reg .b32 ra;\n\tmapa.shared::cluster.u32 ra, %0, 0;\n\tmbarrier.arrive.shared::cluster.b64 _, [ra];\n\t}" ::"r"(bar) : "memory");
    };
    // Tiles of one band of matrix rows follow one another: the band stays in L2 while the tokens pass.
    auto token0 = [&](int tile) { return tile % a.m_tiles * 256 + rank * 128; };
    auto row0 = [&](int tile) { return tile / a.m_tiles * N; };

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
        // A thread by itself for each role: with the whole warp in the loop a block cost twice the cycles.
        if (warp == 0 || warp == 3) {  // the matrix's copies and the rows': one thread gets a box of 16 KB under way in 380 cycles, two get two
            if (g_elect_one()) {
                int s = 0;
                uint32_t ph = 1;
                bool ok = true;
                if (warp == 3) tl::griddep_wait();  // the matrix is older than the rows' launch, which may still be running
                for (int tile = unit; ok && tile < a.tiles; tile += units)
                    for (int kb = 0; kb < a.k_blocks; ++kb) {
                        if (!(ok = tc_wait_one(empty + 8 * s, ph, dead))) break;
                        g_mbar_expect_tx(full + 8 * s, warp == 0 ? N / 2 * 128 : 128 * 128);
                        if (warp == 0) g_tma_load_2d(base + s * kPrStage + 128 * 128, &map_w, kb * 128, row0(tile) + rank * (N / 2), full + 8 * s);
                        else g_tma_load_2d(base + s * kPrStage, &map_q, kb * 128, token0(tile), full + 8 * s);
                        if (++s == kPrStages) s = 0, ph ^= 1u;
                    }
            }
        } else if (warp == 1 && rank == 0) {
            if (g_elect_one()) {
                int s = 0, buf = 0;
                uint32_t ph = 0, acc_ph = 1;
                bool ok = true;
                uint32_t acc_free = 0, there = 0;  // of the next block's, as far as is known
                for (int tile = unit; ok && tile < a.tiles; tile += units)
                    for (int kb = 0; kb < a.k_blocks; ++kb) {
                        if (!(ok = (acc_free || tc_wait_one(acc_empty + 8 * buf, acc_ph, dead)) && (there || tc_wait_one(full + 8 * s, ph, dead)))) break;
                        g_tc_fence_after();
                        const uint64_t q = g_smem_desc_sw128(base + s * kPrStage, 0, 1024), w = g_smem_desc_sw128(base + s * kPrStage + 128 * 128, 0, 1024);
                        const uint32_t d = tmem + buf * APART, done = acc_full + 8 * buf, used = empty + 8 * s;
                        if (++s == kPrStages) s = 0, ph ^= 1u;
                        if (++buf == BUFFERS) buf = 0, acc_ph ^= 1u;
                        pr_block<N>(d, q, w, done, used, acc_empty + 8 * buf, acc_ph, full + 8 * s, ph, acc_free, there);
                    }
            }
        } else if (warp == 1) {
            if (g_elect_one()) {
                int s = 0;
                uint32_t ph = 0;
                bool ok = true;
                for (int tile = unit; ok && tile < a.tiles; tile += units)
                    for (int kb = 0; kb < a.k_blocks; ++kb) {
                        if (!(ok = tc_wait_one(full + 8 * s, ph, dead))) break;
                        arrive_leader(full + 8 * s);
                        if (++s == kPrStages) s = 0, ph ^= 1u;
                    }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");  // 4 x 40 + 8 x 232 <= 12 x 168 a lane
        // this warp's two runs of matrix rows, 64 of the first 128 and half of the others (of 256: a gate's and the up projection's of the same features).
        // The rows of a tile of 256 have two scales a block; of others every 32 or 16 have one.
        constexpr int NB = (N - 128) / 2, RUN_A = N == 256 ? 64 : 32, RUN_B = N == 256 ? 64 : 16, SA = 64 / RUN_A, SB = NB / RUN_B;
        constexpr int B0 = NB < 32 ? NB : 32, B1 = NB - B0;  // of the second run, a read of tensor memory each
        const int quarter = warp & 3, half = (warp - 4) >> 2, row_a = half * 64, row_b = 128 + half * NB;
        int buf = 0;
        uint32_t acc_ph = 0;
        tl::griddep_wait();
        for (int tile = unit; tile < a.tiles; tile += units) {
            const int t0 = token0(tile), r0 = row0(tile), t = t0 + quarter * 32 + lane;
            float acc_a[64], acc_b[NB];
#pragma unroll
            for (int i = 0; i < 64; ++i) acc_a[i] = 0.f;
#pragma unroll
            for (int i = 0; i < NB; ++i) acc_b[i] = 0.f;
            // of tokens and matrix rows past the end: the last ones', for sums that are not stored
            const float *sx = a.sx + min(t, a.rows - 1);
            const int last = (a.n + 127) / 128 - 1;
            auto scales_of = [&](int row) { return a.sw + (size_t)min((r0 + row) >> 7, last) * a.k_blocks; };
            const float *sw_a[SA], *sw_b[SB];
            float next_x = tl::ld_cg(sx), next_a[SA], next_b[SB];
#pragma unroll
            for (int i = 0; i < SA; ++i) sw_a[i] = scales_of(row_a + i * RUN_A), next_a[i] = __ldg(sw_a[i]);
#pragma unroll
            for (int i = 0; i < SB; ++i) sw_b[i] = scales_of(row_b + i * RUN_B), next_b[i] = __ldg(sw_b[i]);
            bool ok = true;
            for (int kb = 0; kb < a.k_blocks; ++kb) {
                float fa[SA], fb[SB];
#pragma unroll
                for (int i = 0; i < SA; ++i) fa[i] = next_x * next_a[i];
#pragma unroll
                for (int i = 0; i < SB; ++i) fb[i] = next_x * next_b[i];
                if (kb + 1 < a.k_blocks) {
                    next_x = tl::ld_cg(sx + (size_t)(kb + 1) * a.ld_sx);
#pragma unroll
                    for (int i = 0; i < SA; ++i) next_a[i] = __ldg(sw_a[i] + kb + 1);
#pragma unroll
                    for (int i = 0; i < SB; ++i) next_b[i] = __ldg(sw_b[i] + kb + 1);
                }
                ok &= tc_wait(acc_full + 8 * buf, acc_ph, dead);
                g_tc_fence_after();
                const uint32_t at = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + buf * APART;
                uint32_t v[2][32];  // two reads on their way, and again two as soon as their places are free: the accumulator is empty after half of the additions
                pr_ld<32>(at + row_a, v[0]);
                pr_ld<32>(at + row_a + 32, v[1]);
                tl::g_tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 32; ++i) acc_a[i] = fmaf(__uint_as_float(v[0][i]), fa[0], acc_a[i]);
                pr_ld<B0>(at + row_b, v[0]);
#pragma unroll
                for (int i = 0; i < 32; ++i) acc_a[32 + i] = fmaf(__uint_as_float(v[1][i]), fa[SA - 1], acc_a[32 + i]);
                pr_ld<B1>(at + row_b + B0, v[1]);
                tl::g_tmem_ld_wait();
                g_tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if (rank == 0) g_mbar_arrive(acc_empty + 8 * buf);
                    else arrive_leader(acc_empty + 8 * buf);
                }
#pragma unroll
                for (int i = 0; i < NB; ++i) acc_b[i] = fmaf(__uint_as_float(i < 32 ? v[0][i] : v[1][i - 32]), fb[i / RUN_B], acc_b[i]);
                if (++buf == BUFFERS) buf = 0, acc_ph ^= 1u;
            }
            const float bad = tc_verdict(ok, dead);
            if constexpr (GATED) {
                float *most = reinterpret_cast<float *>(pr_smem + kPrStages * kPrStage + kPrSumWarps * kPrOut);  // [part][token]
                const int f0 = (r0 >> 1) + row_a;
                float largest = 0.f;
#pragma unroll
                for (int i = 0; i < 64; ++i) {
                    acc_a[i] = f0 + i < a.ff ? gated_pair(acc_a[i], acc_b[i], a.act, a.limit, a.slope) * bad : 0.f;
                    largest = f8_most(largest, fabsf(acc_a[i]));
                }
                most[half * 128 + quarter * 32 + lane] = largest;
                asm volatile("bar.sync %0, 64;" ::"r"(1 + quarter) : "memory");  // the two warps of these tokens
                largest = f8_most(largest, most[(half ^ 1) * 128 + quarter * 32 + lane]);
                asm volatile("bar.sync %0, 64;" ::"r"(1 + quarter) : "memory");  // read by both before the next tile's are written
                const F8Scale s = f8_scale(largest);
                if (t < a.rows) {
                    if (half == 0) a.scales[(size_t)(r0 >> 8) * a.ld_scales + t] = s.scale;
                    uint8_t *to = a.q + (size_t)t * a.ldq + f0;
#pragma unroll
                    for (int i = 0; i < 64; i += 16)
                        if (f0 + i < a.ldq) {  // a multiple of 16
                            uint32_t w[4];
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                w[j] = f8_pack4(__fmul_rn(acc_a[i + 4 * j], s.times), __fmul_rn(acc_a[i + 4 * j + 1], s.times), __fmul_rn(acc_a[i + 4 * j + 2], s.times),
                                                __fmul_rn(acc_a[i + 4 * j + 3], s.times));
                            *reinterpret_cast<uint4 *>(to + i) = make_uint4(w[0], w[1], w[2], w[3]);
                        }
                }
            } else {
                constexpr int PER = 32 / (int)sizeof(T);  // of 32 bytes
                const int c_a = r0 + row_a, c_b = r0 + row_b;
                if (a.bias) {
#pragma unroll
                    for (int i = 0; i < 64; ++i) {
                        if (c_a + i < a.n) acc_a[i] += to_f(static_cast<const T *>(a.bias)[c_a + i]);
                        if (i < NB && c_b + i < a.n) acc_b[i < NB ? i : 0] += to_f(static_cast<const T *>(a.bias)[c_b + i]);
                    }
                }
                auto piece = [&](const float *v, uint32_t (&w)[8]) {  // PER numbers
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        if constexpr (sizeof(T) == 2) w[j] = tl::pack2<T>(v[2 * j] * bad, v[2 * j + 1] * bad);
                        else w[j] = __float_as_uint(v[j] * bad);
                    }
                };
                T *out = static_cast<T *>(a.out);
                if (a.aligned) {
                    if (t < a.rows) {
#pragma unroll
                        for (int i = 0; i < 64; i += PER) {  // a piece is whole or not at all
                            uint32_t w[8];
                            piece(acc_a + i, w);
                            if (c_a + i < a.n) pr_store32(out + (size_t)t * a.n + c_a + i, w);
                            if (i >= NB) continue;
                            piece(acc_b + i, w);
                            if (c_b + i < a.n) pr_store32(out + (size_t)t * a.n + c_b + i, w);
                        }
                    }
                } else {  // through staging rows of 64 bytes, so that lanes lie along the columns
                    unsigned char *stage = pr_smem + kPrStages * kPrStage + (warp - 4) * kPrOut;
                    constexpr int COLS = 64 / (int)sizeof(T);
#pragma unroll
                    for (int i = 0; i < 64 + NB; i += COLS) {  // the last may be half of a row
                        __syncwarp();
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            uint32_t w[8];
                            const int k = i + h * PER;
                            if (k >= 64 + NB) continue;
                            piece(k < 64 ? acc_a + k : acc_b + k - 64, w);
#pragma unroll
                            for (int j = 0; j < 8; ++j) *reinterpret_cast<uint32_t *>(stage + lane * kPrOutStride + h * 32 + j * 4) = w[j];
                        }
                        __syncwarp();
                        const int c = i < 64 ? c_a + i + lane % COLS : i + lane % COLS < 64 + NB ? c_b + i - 64 + lane % COLS : a.n;
#pragma unroll 4
                        for (int r = lane / COLS; r < 32; r += 32 / COLS) {
                            const int tr = t0 + quarter * 32 + r;
                            if (tr < a.rows && c < a.n) out[(size_t)tr * a.n + c] = *reinterpret_cast<const T *>(stage + r * kPrOutStride + lane % COLS * sizeof(T));
                        }
                    }
                }
            }
        }
    }
    __syncwarp();  // also behind a role whose wait gave up
    g_tc_fence_before();
    __syncthreads();
    if (warp == 2) tc_settle(dead);
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");  // the other CTA is done with this one's memory
    if (warp == 2) {
        g_tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

template <typename T, bool GATED, int N>
static int pr_launch(const F8Product &p, F8PairArgs &a, cudaStream_t st) {
    CUtensorMap mq, mw;
    if (int e = tc_map_bytes(&mq, p.q, p.ldq, p.rows, p.ldq, 128)) return e;
    if (int e = tc_map_bytes(&mw, p.w, p.ldw, p.n, p.ldw, N / 2)) return e;
    a.sx = p.sx, a.sw = p.sw, a.ld_sx = p.ld_sx, a.rows = p.rows, a.n = p.n, a.k_blocks = ceil_div(p.k, kF8Block), a.m_tiles = ceil_div(p.rows, 256);
    const long long tiles = (long long)a.m_tiles * ceil_div(p.n, N);
    if (tiles > 0x3fffffff) return tl::fail(TL_EINVAL, "fp8_product: too large");
    a.tiles = (int)tiles;
    static tl::PerDevice ready;
    int device = 0;
    cudaGetDevice(&device);
    if (!ready(device, [&] { return cudaFuncSetAttribute(fp8_pairs_kernel<T, GATED, N>, cudaFuncAttributeMaxDynamicSharedMemorySize, kPrSmem) == cudaSuccess; })) {
        cudaGetLastError();
        return tl::fail(TL_ECUDA, "fp8_product: no shared memory");
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(2 * (unsigned)std::min<long long>(tiles, sm_count() / 2));
    cfg.blockDim = dim3(kPrThreads);
    cfg.dynamicSmemBytes = kPrSmem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = tl::use_pdl() ? 2 : 1;
    cudaLaunchKernelEx(&cfg, fp8_pairs_kernel<T, GATED, N>, mq, mw, a);
    TL_LAUNCH_CHECK("fp8_product");
    return TL_OK;
}

// The width of the tiles: the one whose tiles the pairs are done with first, by what a block of a tile took where every pair had many (8192 x 4096 -> 9472: widths
// 256, 224, 192 took 322, 359, 368 us; 2048 x 9728 -> 2560 with 160 74).  2048 x 9728 -> 2560, 80 tiles of 256 for 74 pairs or 128 of 160: 90 us or 74; 512 x 2560 ->
// 9728: 32 or 24.
F8PairsWidth f8_pairs_width(int rows, int n) {
    F8PairsWidth best{256, INFINITY};
    for (const F8PairsWidth &w : {F8PairsWidth{256, 0.62f}, F8PairsWidth{224, 0.60f}, F8PairsWidth{192, 0.54f}, F8PairsWidth{160, 0.46f}}) {
        const long long tiles = (long long)ceil_div(n, w.outputs) * ceil_div(rows, 256);
        const float time = (float)((tiles + sm_count() / 2 - 1) / (sm_count() / 2)) * w.block;
        if (time < best.block) best = {w.outputs, time};
    }
    return best;
}

int f8_pairs(const F8Product &p, cudaStream_t st) {
    F8PairArgs a{};
    a.bias = p.bias, a.out = p.out;
    const size_t size = p.dtype == TL_BF16 ? 2 : 4;
    a.aligned = (p.n * size) % 32 == 0 && (reinterpret_cast<uintptr_t>(p.out) & 31) == 0;
    switch (f8_pairs_width(p.rows, p.n).outputs) {
        case 160: TLB_DISPATCH(p.dtype, "fp8_product", return (pr_launch<T, false, 160>(p, a, st))); break;
        case 192: TLB_DISPATCH(p.dtype, "fp8_product", return (pr_launch<T, false, 192>(p, a, st))); break;
        case 224: TLB_DISPATCH(p.dtype, "fp8_product", return (pr_launch<T, false, 224>(p, a, st))); break;
        default: TLB_DISPATCH(p.dtype, "fp8_product", return (pr_launch<T, false, 256>(p, a, st)));
    }
    return TL_OK;
}

int f8_pairs_gated(const F8Product &p, const F8Rows &to, cudaStream_t st) {
    F8PairArgs a{};
    a.q = to.q, a.scales = to.scales, a.ldq = to.ldq, a.ld_scales = to.ld_scales, a.ff = to.cols, a.act = to.act, a.limit = to.limit, a.slope = to.slope;
    return pr_launch<float, true, 256>(p, a, st);
}

long long f8_pairs_gave_up() { return tl::read_gave_up(); }

}  // namespace tlb
