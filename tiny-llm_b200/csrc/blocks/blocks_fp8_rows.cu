// Rows of numbers rounded to e4m3, one scale for each run of 128, and the entry points of the products over 8-bit weights.
//
// A half warp takes a run: eight numbers a lane (one or two 16-byte loads), their largest by four exchanges, eight bytes out.  Bound by
// HBM: a number is read once and a byte written.
// Few rows are bound by the launch.
#include "blocks_fp8.cuh"

namespace tlb {

constexpr int kRowsThreads = 256;

template <typename T, bool WIDE>
__device__ __forceinline__ void rows_load(const T *p, int left, float (&v)[8]) {
    if constexpr (WIDE && sizeof(T) == 2) {
        const uint4 u = tl::ld_cg(reinterpret_cast<const uint4 *>(p));
        const uint32_t c[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = tl::unpack2<T>(c[i]);
            v[2 * i] = f.x, v[2 * i + 1] = f.y;
        }
    } else if constexpr (WIDE) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint4 u = tl::ld_cg(reinterpret_cast<const uint4 *>(p) + i);
            v[4 * i] = __uint_as_float(u.x), v[4 * i + 1] = __uint_as_float(u.y), v[4 * i + 2] = __uint_as_float(u.z), v[4 * i + 3] = __uint_as_float(u.w);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < left ? to_f(tl::ld_cg(p + i)) : 0.f;
    }
}

// WIDE: every group of eight is whole and aligned to 16 bytes.
template <typename T, bool GATED, bool WIDE>
__global__ void __launch_bounds__(kRowsThreads)
fp8_rows_kernel(const T *x, long long ldx, int rows, int cols, int act, float limit, float slope, uint8_t *q, int ldq, float *scales, int ld_scales) {
    const unsigned runs = (cols + kF8Block - 1) / kF8Block, total = rows * runs, lane = threadIdx.x & 15;
    const unsigned mine = blockIdx.x * (kRowsThreads / 16) + (threadIdx.x >> 4);  // a thread's number itself does not fit into 32 bits
    tl::griddep_wait();
    tl::griddep_launch();  // behind the wait: what a dependent reads ahead of its own is older than this launch
    const bool live = mine < total;  // a half warp as one
    const unsigned row = live ? mine / runs : 0, run = live ? mine - row * runs : 0;
    const int k = run * kF8Block + lane * 8, left = live ? cols - k : 0;
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.f;
    if (left > 0) {
        if constexpr (GATED) {  // the columns of a whole run are there, those past the last feature are zero
            const T *from = x + row * ldx + run * 2 * kF8Block + lane * 8;
            float g[8], up[8];
            rows_load<T, WIDE>(from, 8, g);
            rows_load<T, WIDE>(from + kF8Block, 8, up);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = i < left ? gated_pair(g[i], up[i], act, limit, slope) : 0.f;
        } else {
            rows_load<T, WIDE>(x + row * ldx + k, left, v);
        }
    }
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) most = f8_most(most, fabsf(v[i]));
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) most = f8_most(most, __shfl_xor_sync(0xffffffffu, most, o));
    const F8Scale s = f8_scale(most);
    if (!live) return;
    if (lane == 0) scales[(size_t)run * ld_scales + row] = s.scale;
    if (k >= ldq) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __fmul_rn(v[i], s.times);
    *reinterpret_cast<uint2 *>(q + (size_t)row * ldq + k) = make_uint2(f8_pack4(v[0], v[1], v[2], v[3]), f8_pack4(v[4], v[5], v[6], v[7]));
}

// The same for many rows of whole groups of 16, which the instructions of a run's two quotients and of finding it bound in the form above (4096 rows of 9728:
// 64 % of the issue slots at half of HBM's rate).  Here eight lanes take a run, 16 numbers each, a warp eight runs, neighbours in their row-by-row order; eight lanes
// make the quotients of all eight, and one division finds the first.
template <typename T>
__global__ void __launch_bounds__(kRowsThreads)
fp8_many_rows_kernel(const T *x, long long ldx, int rows, int cols, uint8_t *q, int ldq, float *scales, int ld_scales) {
    const unsigned runs = (cols + kF8Block - 1) / kF8Block, total = rows * runs, lane = threadIdx.x & 31;
    const unsigned first = (blockIdx.x * (kRowsThreads / 32) + (threadIdx.x >> 5)) * 8;
    tl::griddep_wait();
    tl::griddep_launch();
    if (first >= total) return;
    const unsigned row0 = first / runs, run0 = first - row0 * runs;
    auto place = [&](unsigned i, unsigned &row, unsigned &run) {  // of the warp's run i
        row = row0, run = run0 + i;
        while (run >= runs) run -= runs, ++row;
    };
    float v[2][16], most[2];
    unsigned row[2], run[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const unsigned i = u * 4 + (lane >> 3);
        place(i, row[u], run[u]);
        const int k = run[u] * kF8Block + (lane & 7) * 16;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float half[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            if (first + i < total && k < cols) rows_load<T, true>(x + row[u] * ldx + k + h * 8, 8, half);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[u][h * 8 + j] = half[j];
        }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        most[u] = 0.f;
#pragma unroll
        for (int j = 0; j < 16; ++j) most[u] = f8_most(most[u], fabsf(v[u][j]));
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) most[u] = f8_most(most[u], __shfl_xor_sync(0xffffffffu, most[u], o));
    }
    const float a = __shfl_sync(0xffffffffu, most[0], (lane & 3) * 8), b = __shfl_sync(0xffffffffu, most[1], (lane & 3) * 8);
    const F8Scale s = f8_scale(lane & 4 ? b : a);  // of the warp's run lane & 7
    if (lane < 8 && first + lane < total) {
        unsigned at_row, at_run;
        place(lane, at_row, at_run);
        scales[(size_t)at_run * ld_scales + at_row] = s.scale;
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const unsigned i = u * 4 + (lane >> 3);
        const float times = __shfl_sync(0xffffffffu, s.times, i);
        const int k = run[u] * kF8Block + (lane & 7) * 16;
        if (first + i >= total || k >= ldq) continue;
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            w[j] = f8_pack4(__fmul_rn(v[u][4 * j], times), __fmul_rn(v[u][4 * j + 1], times), __fmul_rn(v[u][4 * j + 2], times), __fmul_rn(v[u][4 * j + 3], times));
        *reinterpret_cast<uint4 *>(q + (size_t)row[u] * ldq + k) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

int f8_rows(const F8Rows &a, cudaStream_t st) {
    const long long runs = (long long)a.rows * ceil_div(a.cols, kF8Block);
    if (runs > 0x7fffff00LL) return tl::fail(TL_EINVAL, "fp8_rows: too many rows");
#define TLB_ROWS(T, G, W)                                                                                                                                          \
    tl::launch_chained(fp8_rows_kernel<T, G, W>, dim3((unsigned)((runs + 15) / 16)), dim3(kRowsThreads), 0, st, (const T *)a.x, a.ldx, a.rows, a.cols, a.act, a.limit, \
                       a.slope, a.q, a.ldq, a.scales, a.ld_scales)
    if (a.gated) {
        TLB_ROWS(float, true, true);
    } else {
        const size_t es = a.dtype == TL_BF16 ? 2 : 4;
        const bool wide = a.cols % 8 == 0 && (a.ldx * es) % 16 == 0 && tl::aligned16(a.x);
        if (wide && a.cols % 16 == 0 && runs >= 32 * 1024) {  // below, fewer numbers a warp put more warps to work
            const dim3 grid((unsigned)((runs + kRowsThreads / 4 - 1) / (kRowsThreads / 4)));
            TLB_DISPATCH(a.dtype, "fp8_rows", tl::launch_chained(fp8_many_rows_kernel<T>, grid, dim3(kRowsThreads), 0, st, (const T *)a.x, a.ldx, a.rows, a.cols, a.q, a.ldq, a.scales, a.ld_scales));
        } else {
            TLB_DISPATCH(a.dtype, "fp8_rows", if (wide) TLB_ROWS(T, false, true); else TLB_ROWS(T, false, false));
        }
    }
#undef TLB_ROWS
    TL_LAUNCH_CHECK("fp8_rows");
    return TL_OK;
}

// Above this many rows the first product of a feed-forward leaves its gated rows rounded, below it fp32 sums and a launch that gates and rounds them.
constexpr int kF8Fused = 128;

// The rounded rows of one product in a caller's scratch: bytes, then scales.
static size_t f8_rows_bytes(int rows, int cols) {
    return (size_t)rows * f8_up(cols, 16) + (size_t)ceil_div(cols, kF8Block) * f8_up(rows, 4) * sizeof(float);
}

}  // namespace tlb

using namespace tlb;

extern "C" {

size_t tlb_fp8_linear_workspace(int rows, int k) { return rows <= 0 || k <= 0 ? 0 : f8_rows_bytes(rows, k); }

int tlb_fp8_linear(const void *x, long long ldx, const void *w, int ldw, const float *sw, const void *bias, void *out, int rows, int n, int k, void *workspace,
                   size_t workspace_bytes, int dtype, void *stream) {
    if (rows <= 0) return TL_OK;
    if (!x || !w || !sw || !out || !workspace || n <= 0 || k <= 0 || ldx < k || ldw < k || ldw % 16 || !tl::aligned16(w) || !tl::aligned16(workspace))
        return tl::fail(TL_EINVAL, "fp8_linear: bad argument");
    if (dtype != TL_F32 && dtype != TL_BF16) return tl::fail(TL_EDTYPE, "fp8_linear: dtype must be float32 or bfloat16");
    if (workspace_bytes < tlb_fp8_linear_workspace(rows, k)) return tl::fail(TL_EINVAL, "fp8_linear: workspace too small");
    const int ldq = f8_up(k, 16), ld_sx = f8_up(rows, 4);
    uint8_t *q = (uint8_t *)workspace;
    float *sx = (float *)(q + (size_t)rows * ldq);
    const F8Rows from{x, ldx, rows, k, dtype, false, 0, 0.f, 1.f, q, ldq, sx, ld_sx};
    const F8Product product{q, sx, ldq, ld_sx, rows, (const uint8_t *)w, sw, ldw, n, k, bias, out, dtype};
    if (f8_own(product)) return f8_product_own(product, from, as_stream(stream));
    if (int e = f8_rows(from, as_stream(stream))) return e;
    return f8_product(product, as_stream(stream));
}

size_t tlb_fp8_gated_mlp_workspace(int rows, int dim, int ff) {
    if (rows <= 0 || dim <= 0 || ff <= 0) return 0;
    return ((f8_rows_bytes(rows, dim) + 15) & ~(size_t)15) + ((f8_rows_bytes(rows, ff) + 15) & ~(size_t)15) +
           (rows > kF8Fused ? 0 : (size_t)rows * 2 * f8_up(ff, kF8Block) * sizeof(float));
}

int tlb_fp8_gated_mlp(const void *x, long long ldx, const void *w_gate_up, int ld_gate_up, const float *s_gate_up, const void *w_down, int ld_down, const float *s_down,
                      void *out, int rows, int dim, int ff, int act, float limit, float slope, void *workspace, size_t workspace_bytes, int dtype, void *stream) {
    if (rows <= 0) return TL_OK;
    if (!x || !w_gate_up || !s_gate_up || !w_down || !s_down || !out || !workspace || dim <= 0 || ff <= 0 || ldx < dim || ld_gate_up < dim || ld_gate_up % 16 ||
        ld_down < ff || ld_down % 16 || !tl::aligned16(w_gate_up) || !tl::aligned16(w_down) || !tl::aligned16(workspace) || (act != 0 && act != 1 && act != 3) ||
        (act == 3 && !(limit > 0.f)))
        return tl::fail(TL_EINVAL, "fp8_gated_mlp: bad argument");
    if (dtype != TL_F32 && dtype != TL_BF16) return tl::fail(TL_EDTYPE, "fp8_gated_mlp: dtype must be float32 or bfloat16");
    if (workspace_bytes < tlb_fp8_gated_mlp_workspace(rows, dim, ff)) return tl::fail(TL_EINVAL, "fp8_gated_mlp: workspace too small");
    const cudaStream_t st = as_stream(stream);
    const int ld_sx = f8_up(rows, 4), wide = 2 * f8_up(ff, kF8Block);
    uint8_t *q = (uint8_t *)workspace, *q2 = q + ((f8_rows_bytes(rows, dim) + 15) & ~(size_t)15);
    float *sx = (float *)(q + (size_t)rows * f8_up(dim, 16)), *sx2 = (float *)(q2 + (size_t)rows * f8_up(ff, 16));
    float *inner = (float *)(q2 + ((f8_rows_bytes(rows, ff) + 15) & ~(size_t)15));
    const F8Rows from{x, ldx, rows, dim, dtype, false, 0, 0.f, 1.f, q, f8_up(dim, 16), sx, ld_sx};
    const F8Product first{q, sx, f8_up(dim, 16), ld_sx, rows, (const uint8_t *)w_gate_up, s_gate_up, ld_gate_up, wide, dim, nullptr, inner, TL_F32};
    const F8Rows gated{inner, wide, rows, ff, TL_F32, true, act, limit, slope, q2, f8_up(ff, 16), sx2, ld_sx};
    const F8Product second{q2, sx2, f8_up(ff, 16), ld_sx, rows, (const uint8_t *)w_down, s_down, ld_down, dim, ff, nullptr, out, dtype};
    if (f8_own(first) && f8_own(second)) {
        if (int e = f8_product_own(first, from, st)) return e;
        return f8_product_own(second, gated, st);
    }
    if (int e = f8_rows(from, st)) return e;
    if (rows > kF8Fused) {
        if (int e = f8_pairs_gated(first, gated, st)) return e;
    } else {
        if (int e = f8_product(first, st)) return e;
        if (int e = f8_rows(gated, st)) return e;
    }
    return f8_product(second, st);
}

}  // extern "C"
