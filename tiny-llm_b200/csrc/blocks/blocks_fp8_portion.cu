// Attention of many columns (prompt portions) over pages of 8 bits on the 5th-generation tensor cores, bf16 queries, heads of 64 or 128 entries.
//
// The arithmetic is that of blocks_fp8_attention.cu; the operands of both products are f16 here too, so that nothing is lost ahead of the weights' rounding (2^-11):
// a query row is brought to the top of f16's range by a power of two, keys and values are their e4m3 numbers times their block's scale over the largest
// scale of the CTA's blocks, which is exact down to 2^-15 of that.  Where the CTA's scales lie further apart (keys' or values'), f16 would lose the small ones, also for rows that
// see nothing of the large ones; where scores may pass 2^23, weights would be above f16's largest number.  Then the operands are the numbers as they are, a tile is one block of 16 keys, and a row's own fp32 scores and weights take the scales.  A block whose
// scale is no number counts as zeros in the products, and the rows that see it are made NaN at the end.
//
// A CTA takes 256 columns of one request and key/value head, or a piece of their keys, as two sets of 128 rows (tensor-memory lanes) that work on the same keys, so that one's
// exponentials run beside the other's products and the cache's numbers are turned into operands once for both.  Per 64 keys:
//   warps 8-15   turn keys (the first four) and values into f16 operand tiles (128-byte swizzle) of two stages each, the next tile's bytes on their way in registers meanwhile
//   warps 16, 17 tcgen05.mma, one elected lane, a set each: S = Q K^T into one of two score buffers, O += P V; the next tile's scores are issued ahead of this tile's values.
//                (One warp for both sets took 2000 cycles to issue a tile's 24 products of 32 cycles each.)
//   warps 0-7    softmax, thread = row: scores from tensor memory, 2^x of them over a running maximum that may lag behind by 2^15, P as f16 back over its own scores
//   warps 20-23  rescale the output's rows whose maximum grew, while the softmax goes on (with queries of heavy tails one warp in eight has such a row: 127 us -> 115 for 2048 tokens over 3500)
//
// 2048 tokens over 3500 (32 over 8 heads of 128) take 106 us, 785 TF/s; 128 tokens 28, of which 6 are the prologue and 5 the launch that joins the pieces.  Block by block (one block with a scale 2^20 times the others') they take
// 433 and 58.  A tile of 256 columns and 64 keys takes 2400 cycles, 2120 if nothing is
// rescaled, where its exponentials and its products take 1024 each: the softmax's own chain is 1600, the products' 1750 (a step of 64 keys reads the queries from shared memory again, which
// is 4 KB for 32 cycles of work).  Leaving out half of the products or all exponentials brings 2120 to 2050 and 1950 only.
#include "../per_device.h"
#include "blocks_fp8_attention.cuh"
#include "blocks_tc.cuh"

namespace tlb {

using tl::g_fence_proxy_async;
using tl::g_tmem_ld32;
using tl::g_tmem_st32;
using tl::g_tmem_st_wait;

constexpr int kPoKeys = 64;
constexpr int kPoSet = 128;  // rows of a set
constexpr int kPoStages = 2;  // of operand tiles, a power of two; four take as long
// Registers are moved between groups of four warps (128, 128, 72, 72, 32 and 48 are six times the launch's 80); warps 18 and 19 have nothing to do.
constexpr int kPoThreads = 24 * 32;
constexpr int kPoColumns = 512;      // of tensor memory; a set's half: two score buffers of 64, the output from 128 on
constexpr uint32_t kPoHalf = 256, kPoOut = 128;

// Asynchronous copies; zeros where `there` is false.
__device__ __forceinline__ void po_copy16(uint32_t to, const void *from, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ float po_max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// Two fp32 numbers side by side: one instruction for both.
__device__ __forceinline__ uint64_t po_two(float x, float y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ float2 po_each(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t po_fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t po_add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// 16 columns of the warp's 32 lanes.
__device__ __forceinline__ void po_st16(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
                 "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
                 : "memory");
}

// 32 columns, on their way until po_ld_wait.
__device__ __forceinline__ void po_ld32(uint32_t taddr, uint32_t *v) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
                 : "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ void po_ld_wait(uint32_t *v) {  // what is read behind it is not read ahead of it
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 64; ++i) asm volatile("" : "+r"(v[i]));
}

constexpr float kPoDeep = 90.f;  // log2: how far a row's unit may fall below the largest it has had: the outputs of 2^28 keys stay below 448 * 2^118
constexpr int kPoApart = 15 << 23;  // the bits of a power of two are this much more than those of one 2^-15 of it: so far f16 holds both sides' numbers

// kind::f16, f16 x f16 -> f32, 128 rows
__host__ __device__ constexpr uint32_t po_idesc(int n, bool b_mn) { return (1u << 4) | ((b_mn ? 1u : 0u) << 16) | (static_cast<uint32_t>(n >> 3) << 17) | (8u << 24); }

template <int DIM>
struct PoShape {
    static constexpr int halves = DIM / 64;                                // 64-column blocks
    static constexpr int q_block = kPoSet * 128, kv_block = kPoKeys * 128;  // bytes
    static constexpr int k_off = 2 * halves * q_block, v_off = k_off + kPoStages * halves * kv_block, bar_off = v_off + kPoStages * halves * kv_block;
    // the row factors and two tiles' factors of the rescaled rows
    static constexpr int row_off = bar_off + 512, smem = row_off + 3 * kPoRows * 4;
    static_assert(2 * kPoStages * halves * kv_block >= kPoRows * DIM * 2, "the queries as they come fit where the operand tiles will be");
};

// 16 e4m3 numbers times `ratio` (two alike), as f16, to the two places of a row.
__device__ __forceinline__ void po_store(unsigned char *one, unsigned char *two, uint4 raw, uint32_t ratio) {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    uint32_t f[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        at_halves(w[i], f[2 * i], f[2 * i + 1]);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const __half2 v = __hmul2(*reinterpret_cast<__half2 *>(&f[2 * i + e]), *reinterpret_cast<const __half2 *>(&ratio));
            f[2 * i + e] = *reinterpret_cast<const uint32_t *>(&v);
        }
    }
    *reinterpret_cast<uint4 *>(one) = make_uint4(f[0], f[1], f[2], f[3]), *reinterpret_cast<uint4 *>(two) = make_uint4(f[4], f[5], f[6], f[7]);
}

template <int DIM>
__global__ void __launch_bounds__(kPoThreads, 1) fp8_portion_kernel(const __grid_constant__ F8Attend a) {
    using Z = PoShape<DIM>;
    constexpr int CH = DIM / 16, PER = kPoKeys * CH / 128;  // 16-byte pieces of a row; of a tile's side, a converting thread's
    extern __shared__ __align__(1024) unsigned char psm[];
    tl::griddep_wait();
    tl::griddep_launch();  // behind the wait: the launch that joins the pieces reads the lengths ahead of its own
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const tlb_fp8_pages &pg = a.pages;
    const int G = a.group, L = a.tokens, columns = G * L;
    const int index = static_cast<int>(gridDim.x - 1 - blockIdx.x);  // late columns, which see most, first
    const AtPiece mine = at_piece(a, index);
    if (mine.b < 0) return;
    const int b = mine.b, cb = f8_div(mine.item, pg.heads, a.heads_magic), h = mine.item - cb * pg.heads, c0 = cb * kPoRows, ctx = mine.ctx;
    // keys [0, limit) are seen; a row behind the last one goes along with it
    auto limit_of = [&](int col) { return a.causal ? max(ctx - L + 1 + f8_div(min(col, columns - 1), G, a.group_magic), 0) : ctx; };
    const int end = min(limit_of(c0 + kPoRows - 1), ctx), begin = mine.piece * mine.size, stop = min((end + kF8Tokens - 1) / kF8Tokens, begin + mine.size);
    const int first = begin * kF8Tokens, past = min(stop * kF8Tokens, end);  // keys [first, past)
    const int32_t *table = a.table + static_cast<size_t>(b) * a.max_pages;
    auto page_at = [&](int blk) { return f8_div(blk, a.page_blocks, a.page_magic); };
    // the scale of block blk, NaN where its page is none
    auto block_at = [&](int blk, int &page) {
        const int at = page_at(blk);
        page = tl::ld_cg(table + at);
        return (static_cast<size_t>(page) * pg.heads + h) * a.page_blocks + (blk - at * a.page_blocks);
    };

    const uint32_t base = g_smem_u32(psm), k_at = base + Z::k_off, v_at = base + Z::v_off, bar = base + Z::bar_off;
    const uint32_t s_full = bar, p_full = bar + 32, pv_done = bar + 64, k_full = bar + 96, k_empty = bar + 128, v_full = bar + 160, v_empty = bar + 192, told = bar + 256;  // two of each, of the first three for either set, of the last for each softmax warp
    volatile int *dead = reinterpret_cast<volatile int *>(psm + Z::bar_off + 224);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(psm + Z::bar_off + 228);
    // largest scales of the CTA's blocks, keys' and values' (bits of positive numbers); whether a scale or page is none; smallest scales; the largest factor of a row
    int *seen = reinterpret_cast<int *>(psm + Z::bar_off + 232);
    float *row_factor = reinterpret_cast<float *>(psm + Z::row_off), *shrink = row_factor + kPoRows;  // [2][kPoRows]
    if (threadIdx.x == 0) {
        for (int i = 0; i < 4; ++i) g_mbar_init(s_full + 8 * i, 1), g_mbar_init(p_full + 8 * i, 8), g_mbar_init(pv_done + 8 * i, 1);
        for (int i = 0; i < kPoStages; ++i) g_mbar_init(k_full + 8 * i, 4), g_mbar_init(k_empty + 8 * i, 2), g_mbar_init(v_full + 8 * i, 4), g_mbar_init(v_empty + 8 * i, 2);
        for (int i = 0; i < 16; ++i) g_mbar_init(told + 8 * i, 1);
        *dead = 0, seen[0] = 0, seen[1] = 0, seen[2] = 0, seen[3] = 0x7f7fffff, seen[4] = 0x7f7fffff, seen[5] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 16) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(g_smem_u32(tmem_slot)), "n"(kPoColumns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    __syncthreads();

    // the converting warps: a thread's i-th piece of a tile is in row (tid + 128 i) / CH, part of the block (tid + 128 i) / (16 CH); it copies, reads and converts
    // its own pieces, so they wait for nobody.  Lane j knows where block j of the tile that is asked for next lies, and the scales of those that were.
    const bool values = warp >= 12;
    const int tid = threadIdx.x & 127;
    const uint8_t *numbers = (values ? pg.values : pg.keys) + 16 * tid;
    const float *scales = values ? pg.value_scales : pg.key_scales;
    int place = -1;  // of a block among all pages' (fewer than 2^31: they are 16 rows each); -1: none
    float scale_next = 0.f;
    uint4 raw[PER];  // the next tile's
    int step = kPoKeys / kF8Tokens;  // blocks of a tile
    auto look_up = [&](int t) {
        const int blk = begin + t * step + lane, at = page_at(blk);
        const int page = lane < step && blk < stop ? tl::ld_cg(table + at) : -1;
        place = static_cast<unsigned>(page) < static_cast<unsigned>(pg.num_pages) ? (page * pg.heads + h) * a.page_blocks + blk - at * a.page_blocks : -1;
    };
    auto ask = [&](int t) {  // of a page that is none: zeros
        scale_next = place < 0 ? 0.f : tl::ld_cg(scales + place);
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int at = __shfl_sync(0xffffffffu, place, (tid + 128 * i) / (kF8Tokens * CH));
            const size_t byte = static_cast<size_t>(static_cast<unsigned>(max(at, 0))) * (kF8Tokens * DIM);
            // the pieces before this thread's i-th that are not of its block
            raw[i] = at >= 0 ? tl::ld_cg(reinterpret_cast<const uint4 *>(numbers + byte + (DIM == 128 ? 0 : -(tid / 64) * 1024))) : make_uint4(0, 0, 0, 0);
        }
    };
    if (warp >= 8 && warp < 16) look_up(0), ask(0), look_up(1);
    // scales of the CTA's blocks, for the largest ones: asked for ahead of the queries, looked at behind them
    auto scales_of = [&](int blk) {
        int page;
        const size_t at = block_at(blk, page);
        const bool there = static_cast<unsigned>(page) < static_cast<unsigned>(pg.num_pages);
        return make_float2(there ? tl::ld_cg(pg.key_scales + at) : NAN, there ? tl::ld_cg(pg.value_scales + at) : NAN);
    };
    auto look_over = [&](float2 s) {  // whole warps
        const int k = s.x < INFINITY ? __float_as_int(s.x) : 0, v = s.y < INFINITY ? __float_as_int(s.y) : 0;
        const int k1 = __reduce_max_sync(0xffffffffu, k), v1 = __reduce_max_sync(0xffffffffu, v);
        const int k0 = __reduce_min_sync(0xffffffffu, k > 0 ? k : 0x7f7fffff), v0 = __reduce_min_sync(0xffffffffu, v > 0 ? v : 0x7f7fffff);
        if (lane == 0 && k1 > 0) atomicMax(seen, k1), atomicMin(seen + 3, k0);
        if (lane == 0 && v1 > 0) atomicMax(seen + 1, v1), atomicMin(seen + 4, v0);
        if (!(s.x < INFINITY) || !(s.y < INFINITY)) seen[2] = 1;
    };
    float2 of_mine = make_float2(0.f, 0.f);
    if (begin + static_cast<int>(threadIdx.x) < stop) of_mine = scales_of(begin + threadIdx.x);
    // queries: 8 entries of either 64 a lane, a row to 8 lanes of the first sixteen warps; first as they are, to where the operand tiles will be
    constexpr int PARTS = DIM / 64, N = kPoRows / (16 * 4);
    unsigned char *mine_q = psm + Z::k_off + threadIdx.x * 16;
    if (warp < 16) {
        const bf16 *q = static_cast<const bf16 *>(a.q) + b * a.q_b + static_cast<long long>(h) * G * a.q_h + lane % 8 * 8;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int col = c0 + (i * 16 + warp) * 4 + lane / 8, l = f8_div(min(col, columns - 1), G, a.group_magic);
            const bf16 *from = q + l * a.q_l + (min(col, columns - 1) - l * G) * a.q_h;
#pragma unroll
            for (int p = 0; p < PARTS; ++p) {
                unsigned char *to = mine_q + (i * PARTS + p) * 8192;
                if (a.wide_rows) {
                    po_copy16(g_smem_u32(to), from + 64 * p, col < columns);
                } else {
#pragma unroll 1
                    for (int e = 0; e < 8; ++e) reinterpret_cast<bf16 *>(to)[e] = col < columns ? tl::ld_cg(from + 64 * p + e) : __float2bfloat16_rn(0.f);
                }
            }
        }
    }
    look_over(of_mine);
    for (int blk = begin + threadIdx.x + kPoThreads; blk - lane < stop; blk += kPoThreads) look_over(blk < stop ? scales_of(blk) : make_float2(0.f, 0.f));
    if (warp < 16) {
        const float sign = a.scale_log2 < 0.f ? -1.f : 1.f;
        asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll 2
        for (int i = 0; i < N; ++i) {
            const int row = (i * 16 + warp) * 4 + lane / 8, j = lane % 8, in_set = row % kPoSet;
            uint4 u[PARTS];
            uint32_t m = 0;  // magnitudes are in the order of their bits, numbers that are none on top
#pragma unroll
            for (int p = 0; p < PARTS; ++p) {
                u[p] = *reinterpret_cast<const uint4 *>(mine_q + (i * PARTS + p) * 8192);
                m = __vmaxu2(m, __vmaxu2(__vmaxu2(u[p].x & 0x7fff7fffu, u[p].y & 0x7fff7fffu), __vmaxu2(u[p].z & 0x7fff7fffu, u[p].w & 0x7fff7fffu)));
            }
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, o));
            const int e2 = static_cast<int>(max(m >> 16, m & 0xffffu) >> 7), up = e2 == 255 ? 0 : min(13 + 127 - e2, 100);
            const float times = f8_power(up) * sign;
            unsigned char *to = psm + row / kPoSet * Z::halves * Z::q_block + in_set * 128 + ((j ^ (in_set & 7)) << 4);
#pragma unroll
            for (int p = 0; p < PARTS; ++p) {
                const float2 y[4] = {tl::unpack2<bf16>(u[p].x), tl::unpack2<bf16>(u[p].y), tl::unpack2<bf16>(u[p].z), tl::unpack2<bf16>(u[p].w)};
                uint4 f;
                f.x = tl::pack2<__half>(y[0].x * times, y[0].y * times), f.y = tl::pack2<__half>(y[1].x * times, y[1].y * times);
                f.z = tl::pack2<__half>(y[2].x * times, y[2].y * times), f.w = tl::pack2<__half>(y[3].x * times, y[3].y * times);
                *reinterpret_cast<uint4 *>(to + p * Z::q_block) = f;
            }
            if (j == 0) {
                row_factor[row] = f8_power(-up);
                if (e2 != 255) atomicMax(seen + 5, __float_as_int(f8_power(-up)));
            }
        }
        g_fence_proxy_async();
    }
    g_tc_fence_before();
    __syncthreads();
    g_tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    // (without any scale: negative); or scores may reach 2^23, where they could come to be half above their own rounded maxima (2^15.5 as a weight): a product is at most 2^14 * 448 for each entry
    const bool apart = seen[0] - seen[3] > kPoApart || seen[1] - seen[4] > kPoApart ||
                       fabsf(a.scale_log2) * __int_as_float(seen[5]) * __int_as_float(seen[0]) > 0x1p23f / (0x1p14f * 448.f * DIM);
    if (apart) step = 1;
    const int n_tiles = max((past - first + step * kF8Tokens - 1) / (step * kF8Tokens), 0);
    // 1 over the largest scales; both are powers of two
    const float top_k = seen[0] && !apart ? __int_as_float(seen[0]) : 1.f, top_v = seen[1] && !apart ? __int_as_float(seen[1]) : 1.f, under_k = 1.f / top_k, under_v = 1.f / top_v;

    if (warp >= 20) {  // ---- rescaling: a quarter of the rows of both sets
        asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
        const int quarter = warp & 3;
        bool ok = true;
        for (int t = 0; ok && t < n_tiles; ++t) {
            const int s = t & 1;
#pragma unroll 1
            for (int set = 0; set < 2; ++set) {
                if (!(ok = tc_wait(told + 8 * (8 * s + 4 * set + quarter), t >> 1 & 1, dead))) break;
                const float alpha = shrink[s * kPoRows + kPoSet * set + 32 * quarter + lane];
                if (__any_sync(0xffffffffu, alpha != 1.f)) {
                    if (!(ok = tc_wait(pv_done + 16 * set + 8 * (s ^ 1), ((t - 1) >> 1) & 1, dead))) break;  // O has to be still meanwhile
                    g_tc_fence_after();
                    const uint32_t out_at = tmem + (static_cast<uint32_t>(32 * quarter) << 16) + set * kPoHalf + kPoOut;
#pragma unroll 1
                    for (int i = 0; i < DIM / 32; ++i) {
                        uint32_t o[32];
                        g_tmem_ld32(out_at + i * 32, o);
#pragma unroll
                        for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * alpha);
                        g_tmem_st32(out_at + i * 32, o);
                    }
                    g_tmem_st_wait();
                    g_tc_fence_before();
                }
                __syncwarp();
                if (lane == 0) g_mbar_arrive(p_full + 16 * set + 8 * s);
            }
        }
    } else if (warp >= 16) {  // ---- products: S_0, then per tile S_(t+1), P_t V_t
        asm volatile("setmaxnreg.dec.sync.aligned.u32 32;");
        constexpr uint32_t idesc_s = po_idesc(kPoKeys, false), idesc_o = po_idesc(DIM, true);
        const int set = warp & 1;
        const uint32_t scores_at = tmem + set * kPoHalf, out_at = scores_at + kPoOut;
        const uint64_t qd = g_smem_desc_sw128(base + set * Z::halves * Z::q_block, 0, 1024), kd0 = g_smem_desc_sw128(k_at, 0, 1024), vd0 = g_smem_desc_sw128(v_at, Z::kv_block, 1024);
        auto scores = [&](int t) {
            const int s = t & 1, k = t & (kPoStages - 1);
            if (!tc_wait(k_full + 8 * k, t / kPoStages & 1, dead)) return false;
            g_tc_fence_after();
            if (g_elect_one()) {
                const uint64_t kd = kd0 + static_cast<uint64_t>(k * Z::halves * (Z::kv_block >> 4));
#pragma unroll
                for (int i = 0; i < DIM / 16; ++i)
                    g_tc_mma(scores_at + s * kPoKeys, qd + (i >> 2) * (Z::q_block >> 4) + 2 * (i & 3), kd + (i >> 2) * (Z::kv_block >> 4) + 2 * (i & 3), idesc_s, i > 0);
                g_tc_commit(s_full + 16 * set + 8 * s);
                g_tc_commit(k_empty + 8 * k);
            }
            __syncwarp();
            return true;
        };
        const bool begun = warp < 18 && n_tiles > 0 && scores(0);
        for (int t = 0; begun && t < n_tiles; ++t) {
            const int s = t & 1, v = t & (kPoStages - 1);
            if (t + 1 < n_tiles && !scores(t + 1)) break;  // its buffer held P_(t-1), read by a product already queued ahead of this one
            if (!tc_wait(v_full + 8 * v, t / kPoStages & 1, dead) || !tc_wait(p_full + 16 * set + 8 * s, t >> 1 & 1, dead)) break;
            g_tc_fence_after();
            if (g_elect_one()) {
                const uint64_t vd = vd0 + static_cast<uint64_t>(v * Z::halves * (Z::kv_block >> 4));
#pragma unroll
                for (int k = 0; k < kPoKeys / 16; ++k) g_tc_mma_ts(out_at, scores_at + s * kPoKeys + 8 * k, vd + k * (2048 >> 4), idesc_o, t > 0 || k > 0);
                g_tc_commit(v_empty + 8 * v);
                g_tc_commit(pv_done + 16 * set + 8 * s);
            }
            __syncwarp();
        }
    } else if (warp >= 8) {  // ---- pages to operands
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        if (apart) look_up(0), ask(0), look_up(1);  // of tiles of one block
        const float under = values ? under_v : under_k;
        unsigned char *tiles = psm + (values ? Z::v_off : Z::k_off);
        const uint32_t full = values ? v_full : k_full, empty = values ? v_empty : k_empty;
        // a thread's first piece in the operand tile; its others lie 128 / CH rows further each, so in the same places of their groups of eight rows.  The second 64 columns'
        // lanes write their second half first: eight lanes meet all banks
        const int row0 = tid / CH, c = tid % CH, odd = (c >> 2) & 1;
        unsigned char *at = tiles + (c >> 2) * Z::kv_block + row0 * 128;
        unsigned char *one = at + (((2 * (c & 3) + odd) ^ (row0 & 7)) << 4), *two = at + (((2 * (c & 3) + 1 - odd) ^ (row0 & 7)) << 4);
        for (int t = 0; t < n_tiles; ++t) {
            const int s = t & (kPoStages - 1), key0 = first + t * step * kF8Tokens;
            const __half2 r2 = __float2half2_rn(scale_next < INFINITY ? (apart ? 1.f : scale_next * under) : 0.f);
            const uint32_t ratio = *reinterpret_cast<const uint32_t *>(&r2);
            if (!tc_wait(empty + 8 * s, (t / kPoStages & 1) ^ 1u, dead)) break;  // the first pass through the stages does not wait
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                uint4 x = raw[i];
                if (key0 + kPoKeys > ctx && key0 + row0 + 128 / CH * i >= ctx) x = make_uint4(0, 0, 0, 0);  // slots behind the last token may hold anything
                if (odd) x = make_uint4(x.z, x.w, x.x, x.y);
                const int by = s * Z::halves * Z::kv_block + 128 / CH * 128 * i;
                po_store(one + by, two + by, x, __shfl_sync(0xffffffffu, ratio, (tid + 128 * i) / (kF8Tokens * CH)));
            }
            g_fence_proxy_async();
            __syncwarp();
            if (lane == 0) g_mbar_arrive(full + 8 * s);
            ask(t + 1), look_up(t + 2);
        }
    } else {  // ---- softmax: thread = row
        asm volatile("setmaxnreg.inc.sync.aligned.u32 128;");
        const int r = threadIdx.x, col = c0 + r, set = warp >> 2;
        const uint32_t s_mine = s_full + 16 * set, p_mine = p_full + 16 * set, pv_mine = pv_done + 16 * set;
        const bool live = col < columns;
        const int limit = min(limit_of(col), past);
        const uint32_t lanes = (static_cast<uint32_t>((warp & 3) * 32) << 16) + set * kPoHalf;
        const float mult = fmaxf(fabsf(a.scale_log2) * row_factor[r] * top_k, 0x1p-126f);  // never 0: a masked score stays -inf
        const bool care = seen[2] != 0;
        float m = -INFINITY, sum = 0.f, back = 1.f;  // back: of the row's output, beside what it is divided by
        bool ok = true;
        // Scales far apart.  A tile is a block: its key scale goes into the scores, its value scale into the weights, which are rounded over a unit of the row's own, 2^mo.  The unit follows the block's
        // largest weight times scale, up and down, so no block takes anything from another one, nor from a row that does not see it (or gives it no weight).
        if (apart) {
            float mo = -INFINITY, highest = -INFINITY;
            const float unit = fabsf(a.scale_log2) * row_factor[r];
            for (int t = 0; t < n_tiles; ++t) {
                const int key0 = first + t * kF8Tokens, s2 = t & 1;
                if (!(ok = tc_wait(s_mine + 8 * s2, t >> 1 & 1, dead))) break;
                g_tc_fence_after();
                const uint32_t mine_s = tmem + lanes + s2 * kPoKeys;
                int page;
                const size_t at_block = block_at(key0 / kF8Tokens, page);
                const bool there = static_cast<unsigned>(page) < static_cast<unsigned>(pg.num_pages);
                const float ks = there ? tl::ld_cg(pg.key_scales + at_block) : 0.f, vs = there ? tl::ld_cg(pg.value_scales + at_block) : 0.f;
                const bool fine = ks < INFINITY && vs < INFINITY;
                const int sees = there ? min(max(limit - key0, 0), kF8Tokens) : 0;  // keys of the block
                if (sees > 0 && !fine) sum = NAN;
                const float mult = fmaxf(unit * (fine ? ks : 0.f), 0x1p-126f), lift = fine ? log2f(vs) : -INFINITY;
                uint32_t s[32], pk[16];
                g_tmem_ld32(mine_s, s);
                // scores are rounded ahead of the subtraction, as the maximum is: one of 2^28 could be 2^4 above it otherwise
                float top = -INFINITY;
#pragma unroll
                for (int c = 0; c < kF8Tokens; ++c) {
                    const float x = __fmul_rn(__uint_as_float(s[c]), mult);
                    s[c] = __float_as_uint(c < sees ? x : -INFINITY), top = c < sees ? fmaxf(top, x) : top;
                }
                if (top > m + kAtLag || (m == -INFINITY && top > m)) sum *= m == -INFINITY ? 1.f : at_ex2(m - top), m = top;
                const float at = m == -INFINITY ? 0.f : m;
                // weights below 2^-126 of the largest are none
                const float most = ceilf(top - at < -126.f ? -INFINITY : top + lift), next = most == -INFINITY ? mo : fmaxf(most, highest - kPoDeep);
                shrink[s2 * kPoRows + r] = mo == -INFINITY || next == mo ? 1.f : at_ex2(mo - next);  // without anything so far the output is 0
                mo = next, highest = fmaxf(highest, mo);
                __syncwarp();
                if (lane == 0) g_mbar_arrive(told + 8 * (8 * s2 + warp));
                const float by = most == -INFINITY ? -INFINITY : lift + (at - mo);
#pragma unroll
                for (int c = 0; c < 16; ++c) pk[c] = 0;
#pragma unroll
                for (int c = 0; c < kF8Tokens; c += 2) {
                    const float x = __fsub_rn(__uint_as_float(s[c]), at), y = __fsub_rn(__uint_as_float(s[c + 1]), at);
                    sum += at_ex2(x) + at_ex2(y);
                    pk[c / 2] = tl::pack2<__half>(at_ex2(x + by), at_ex2(y + by));
                }
                po_st16(mine_s, pk);
#pragma unroll
                for (int c = 0; c < 8; ++c) pk[c] = 0;
                po_st16(mine_s + 16, pk);  // the tile's other keys
                g_tmem_st_wait();
                g_tc_fence_before();
                __syncwarp();
                if (lane == 0) g_mbar_arrive(p_mine + 8 * s2);
            }
            back = mo == -INFINITY ? 0.f : exp2f(0.5f * (mo - m));  // twice: the whole may be beyond fp32's range
        }
        for (int t = apart ? n_tiles : 0; t < n_tiles; ++t) {
            const int key0 = first + t * kPoKeys, s2 = t & 1;
            if (!(ok = tc_wait(s_mine + 8 * s2, t >> 1 & 1, dead))) break;
            g_tc_fence_after();
            const uint32_t mine_s = tmem + lanes + s2 * kPoKeys;
            const bool cut = __any_sync(0xffffffffu, key0 + kPoKeys > limit);
            unsigned hidden = 0;  // blocks whose page is none
            if (care) {           // such a page hides its keys; a scale that is none makes the row NaN
#pragma unroll 1
                for (int g = 0; g < 4; ++g) {
                    const int key = key0 + kF8Tokens * g;
                    if (key >= past) continue;
                    int page;
                    const size_t at = block_at(key / kF8Tokens, page);
                    if (static_cast<unsigned>(page) >= static_cast<unsigned>(pg.num_pages)) hidden |= 1u << g;
                    else if (key < limit && !(tl::ld_cg(pg.key_scales + at) < INFINITY && tl::ld_cg(pg.value_scales + at) < INFINITY)) sum = NAN;
                }
            }
            uint32_t s[64];
            po_ld32(mine_s, s), po_ld32(mine_s + 32, s + 32), po_ld_wait(s);
            if (cut || hidden) {
#pragma unroll
                for (int c = 0; c < 64; ++c)
                    if (key0 + c >= limit || (hidden >> (c / 16) & 1)) s[c] = 0xff800000u;
            }
            float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int c = 0; c < 64; c += 8)
#pragma unroll
                for (int e = 0; e < 4; ++e) tops[e] = po_max3(tops[e], __uint_as_float(s[c + 2 * e]), __uint_as_float(s[c + 2 * e + 1]));
            const float top = po_max3(fmaxf(tops[0], tops[1]), tops[2], tops[3]) * mult;
            const bool grow = top > m + kAtLag || (m == -INFINITY && top > m);
            // the sums so far shrink where the maximum grows, the output by the warps above, which find the factors here
            const float alpha = t == 0 || !grow || m == -INFINITY ? 1.f : at_ex2(m - top);
            m = grow ? top : m, sum *= alpha;
            shrink[s2 * kPoRows + r] = alpha;
            __syncwarp();
            if (lane == 0) g_mbar_arrive(told + 8 * (8 * s2 + warp));
            const float at = m == -INFINITY ? 0.f : m;
            const uint64_t mult2 = po_two(mult, mult), minus = po_two(-at, -at);
            uint64_t sums[2] = {0, 0};  // two pairs of zeros
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                uint32_t pk[16];
#pragma unroll
                for (int c = 0; c < 32; c += 2) {
                    const float2 z = po_each(po_fma2(po_two(__uint_as_float(s[32 * i + c]), __uint_as_float(s[32 * i + c + 1])), mult2, minus));
                    const float x = at_ex2(z.x), y = at_ex2(z.y);
                    pk[c / 2] = tl::pack2<__half>(x, y);
                    sums[(c >> 1) & 1] = po_add2(sums[(c >> 1) & 1], po_two(x, y));
                }
                po_st16(mine_s + 16 * i, pk);  // column c = keys 2 c and 2 c + 1; over scores that have been read
            }
            const float2 both = po_each(po_add2(sums[0], sums[1]));
            sum += both.x + both.y;
            g_tmem_st_wait();
            g_tc_fence_before();
            __syncwarp();
            if (lane == 0) g_mbar_arrive(p_mine + 8 * s2);
        }
        if (n_tiles > 0) {
            ok = ok && tc_wait(pv_mine + 8 * ((n_tiles - 1) & 1), ((n_tiles - 1) >> 1) & 1, dead);
            g_tc_fence_after();
        }
        const float verdict = tc_verdict(ok, dead) * top_v;
        const bool whole = mine.pieces == 1;
        const float inv = (whole ? (sum == 0.f ? 0.f : 1.f / sum) : 1.f) * verdict * back;
        float *part = whole ? nullptr : static_cast<float *>(a.workspace) + index * at_piece_floats(kPoRows, DIM);
        // Rows leave by way of the set's queries, whose products are through, a warp's 32 rows side by side: a warp stores whole rows that way, not 32 pieces of 16 bytes
        // (2048 tokens over 3500: 115 and 106 us, 128 tokens 34 and 28).  16-byte piece u of row i lies at u ^ (i & 7).
        constexpr int U = DIM / 8, ROW = DIM * 2;
        unsigned char *stage = psm + (set * kPoSet + (warp & 3) * 32) * ROW;
        auto column = [&](int i, float (&o)[32]) {
            if (n_tiles > 0) {
                uint32_t u[32];
                g_tmem_ld32(tmem + lanes + kPoOut + i * 32, u);
#pragma unroll
                for (int c = 0; c < 32; ++c) o[c] = __uint_as_float(u[c]) * inv * back;
            } else {
#pragma unroll
                for (int c = 0; c < 32; ++c) o[c] = 0.f;
            }
        };
        auto put = [&](int u, uint4 v) { *reinterpret_cast<uint4 *>(stage + lane * ROW + ((u ^ (lane & 7)) << 4)) = v; };
        auto take = [&](auto to) {  // to(row): where it begins
            __syncwarp();
#pragma unroll 4
            for (int i = lane / U; i < 32; i += 32 / U) {
                const int row = r - lane + i;
                const uint4 v = *reinterpret_cast<const uint4 *>(stage + i * ROW + (((lane % U) ^ (i & 7)) << 4));
                if (c0 + row < columns) reinterpret_cast<uint4 *>(to(row))[lane % U] = v;
            }
            __syncwarp();
        };
        if (whole) {
#pragma unroll 1
            for (int i = 0; i < DIM / 32; ++i) {
                float o[32];
                column(i, o);
#pragma unroll
                for (int c = 0; c < 32; c += 8)
                    put(4 * i + c / 8, make_uint4(tl::pack2<bf16>(o[c], o[c + 1]), tl::pack2<bf16>(o[c + 2], o[c + 3]), tl::pack2<bf16>(o[c + 4], o[c + 5]), tl::pack2<bf16>(o[c + 6], o[c + 7])));
            }
            take([&](int row) {
                const int l = f8_div(c0 + row, G, a.group_magic);
                return static_cast<bf16 *>(a.out) + ((static_cast<size_t>(b) * L + l) * a.heads + static_cast<size_t>(h) * G + c0 + row - l * G) * DIM;
            });
        } else {
#pragma unroll 1
            for (int i = 0; i < DIM / 32; ++i) {
                float o[32];
                column(i, o);
#pragma unroll
                for (int c = 0; c < 32; c += 4)
                    put(8 * (i % (DIM / 64)) + c / 4, make_uint4(__float_as_uint(o[c]), __float_as_uint(o[c + 1]), __float_as_uint(o[c + 2]), __float_as_uint(o[c + 3])));
                if ((i + 1) % (DIM / 64) == 0) take([&](int row) { return part + row * DIM + (i * 32 / (DIM / 2)) * (DIM / 2); });  // half a row
            }
        }
        if (live && !whole) part[kPoRows * DIM + r] = m, part[kPoRows * (DIM + 1) + r] = sum;
    }
    g_tc_fence_before();
    __syncthreads();
    if (warp == 16) {
        tc_settle(dead);
        g_tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(kPoColumns) : "memory");
    }
}

bool f8_portion_takes(const tlb_fp8_pages &p, const tlb_fp8_attention_call &c) {
    return c.dtype == TL_BF16 && (p.dim == 64 || p.dim == 128) && static_cast<long long>(c.heads / p.heads) * c.tokens > 32;
}

template <int DIM>
static int portion_launch(const F8Attend &a, unsigned ctas, cudaStream_t st) {
    static tl::PerDevice ready;
    using Z = PoShape<DIM>;
    int device = 0;
    cudaGetDevice(&device);
    if (!ready(device, [&] {
            return cudaFuncSetAttribute(fp8_portion_kernel<DIM>, cudaFuncAttributeMaxDynamicSharedMemorySize, Z::smem) == cudaSuccess &&
                   cudaFuncSetAttribute(fp8_portion_kernel<DIM>, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared) == cudaSuccess;
        }))
        return tl::fail(TL_ECUDA, "fp8_attention: %s", cudaGetErrorString(cudaGetLastError()));
    const cudaError_t e = tl::launch_chained(fp8_portion_kernel<DIM>, dim3(ctas), dim3(kPoThreads), Z::smem, st, a);
    if (e != cudaSuccess) return tl::fail(TL_ECUDA, "fp8_attention: %s", cudaGetErrorString(e));
    TL_LAUNCH_CHECK("fp8_attention (portion)");
    return a.workspace ? f8_attend_join(a, kPoRows, st) : TL_OK;
}

// A CTA takes 9 us and 1.3 for every 64 keys; with pieces, which are about as many as SMs, and the launch that joins them it is 20 beside the keys.
AtPlan f8_portion_plan(const tlb_fp8_pages &p, const tlb_fp8_attention_call &c, const AtLengths &n) {
    const long long each = (static_cast<long long>(c.heads / p.heads) * c.tokens + kPoRows - 1) / kPoRows * p.heads, items = each * c.batch, slots = sm_count();
    const double block = 1.3 * kF8Tokens / kPoKeys;
    if (items > slots || n.longest <= kPoWhole)  // more items than a cut would serve
        return {1, 0, ((each * n.live + slots - 1) / slots) * (9 + n.longest * block), true};
    return {1, static_cast<size_t>(items + slots) * at_piece_floats(kPoRows, p.dim) * sizeof(float), 20 + static_cast<double>(n.blocks * each) / slots * block, true};
}

int f8_portion(F8Attend a, cudaStream_t st) {
    a.slots = sm_count(), a.most_pieces = 32, a.granule = kPoKeys / kF8Tokens, a.whole = kPoWhole, a.least = kPoLeast;
    a.col_blocks = (a.group * a.tokens + kPoRows - 1) / kPoRows;
    const long long items = static_cast<long long>(a.col_blocks) * a.pages.heads * a.batch;
    if (items > 0x3fffffff) return tl::fail(TL_EINVAL, "fp8_attention: sizes out of range");
    const unsigned ctas = static_cast<unsigned>(items + (a.workspace ? a.slots : 0));
    a.each_magic = f8_magic(ctas, a.pages.heads * a.col_blocks);
    return a.pages.dim == 64 ? portion_launch<64>(a, ctas, st) : portion_launch<128>(a, ctas, st);
}

long long f8_portion_gave_up() { return tl::read_gave_up(); }

}  // namespace tlb
