// A step's keys and values into pages of 8 bits, with the norm and the rotation that keys and queries pass on the way.
//
// Row x of a head (query or key): x' = x / sqrt(mean(x^2) + eps) * w, then every pair (a, b) of the first `dims` entries turns by the angle
// position * base^(-2i / dims): (a c - b s, b c + a s).  Values stay as they are.  A block is the 16 tokens of a head that share a scale: with m the largest
// magnitude of its new rows, scale = max(2^e, the scale before), e the smallest with m <= 448 * 2^e; the scale before counts if the block holds earlier tokens
// of the sequence, whose numbers are then rounded again to the larger scale.  Scales are powers of two, so that this costs a number nothing
// unless it falls among the smallest ones (below 2^-6 of the scale), and it hardly matters whether tokens come one by one or together.
//
// Angles are made in 64 bits (a far position times a frequency), and so are the keys: a number is rounded to four significant bits next to borders that the last
// bits of its fp32 value decide.  Queries keep their type and are made in 32 bits.
//
// A CTA takes one block of one request and key/value head, with the group's query heads: the angles of its at most 16 tokens are made once, in
// shared memory, a warp takes a row at a time, and the new keys and values wait in shared memory until the block's largest magnitude is known.
#include <math.h>

#include "../per_device.h"
#include "blocks_fp8_cache.cuh"

namespace tlb {

constexpr int kApThreads = 256;
constexpr int kApMostDim = 256;

struct F8Turns {
    double of[kApMostDim / 2];  // base^(-2i / dims) / (2 pi): turns a position
};

struct F8Append : tlb_fp8_append_call {
    tlb_fp8_pages pages;
    int group;
    F8Append(const tlb_fp8_pages &p, const tlb_fp8_append_call &c, int g) : tlb_fp8_append_call(c), pages(p), group(g) {}
};

__device__ __forceinline__ int2 ap_pair(const F8Append &a, int i) { return a.interleaved ? make_int2(2 * i, 2 * i + 1) : make_int2(i, i + a.rot / 2); }

__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

template <typename T>
__global__ void __launch_bounds__(kApThreads) fp8_append_kernel(const __grid_constant__ F8Append a, const __grid_constant__ F8Turns turns) {
    extern __shared__ __align__(16) unsigned char sm[];
    __shared__ float most[2][kF8Tokens];
    tl::griddep_launch();
    tl::griddep_wait();
    const tlb_fp8_pages &pg = a.pages;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, D = pg.dim, half = a.rot / 2;
    const int b = blockIdx.z, h = blockIdx.y, G = a.group;
    const int ctx = a.lens[b];
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
                for (int d = lane; d < D; d += 32) s += to_f(x[d]) * to_f(x[d]);
                r = 1.f / sqrtf(warp_sum(s) / D + a.q_eps);
            }
            auto at = [&](int d) { return w ? to_f(x[d]) * r * to_f(w[d]) : to_f(x[d]); };
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
                for (int d = lane; d < D; d += 32) s += static_cast<double>(to_f(x[d])) * to_f(x[d]);
                r = 1.0 / sqrt(warp_sum_f64(s) / D + a.k_eps);
            }
            auto at = [&](int d) { return w ? to_f(x[d]) * r * to_f(w[d]) : static_cast<double>(to_f(x[d])); };
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
                const float f = to_f(x[d]);
                y[d] = f, m = f8_most(m, fabsf(f));
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = f8_most(m, __shfl_xor_sync(0xffffffffu, m, o));
        if (lane == 0) most[key ? 0 : 1][i] = m;
    }
    __syncthreads();

    const int page = a.table[static_cast<size_t>(b) * a.max_pages + start / pg.page_size], slot = start % pg.page_size;
    if (page < 0 || page >= pg.num_pages) return;
    const int kept = p0 - start, pieces = D / 16;  // rows of earlier tokens, 16-byte pieces of a row
#pragma unroll
    for (int side = 0; side < 2; ++side) {
        float m = 0.f;
        for (int i = 0; i < n; ++i) m = f8_most(m, most[side][i]);
        float *scale_at = (side ? pg.value_scales : pg.key_scales) + f8_scale_at(pg, page, h, slot);
        uint8_t *rows = (side ? pg.values : pg.keys) + f8_row(pg, page, h, slot);
        const float before = kept ? *scale_at : 0.f;
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
            const float ratio = before * under;
            for (int i = threadIdx.x; i < kept * pieces; i += kApThreads) {
                uint4 x = reinterpret_cast<uint4 *>(rows)[i];
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
        __syncthreads();  // every thread has read the scale before
        if (threadIdx.x == 0) *scale_at = scale;
    }
}

int f8_check_pages(const char *op, const tlb_fp8_pages *p) {
    if (!p || !p->keys || !p->values || !p->key_scales || !p->value_scales) return tl::fail(TL_EINVAL, "%s: no pages", op);
    if (p->num_pages <= 0 || p->heads <= 0 || p->page_size <= 0 || p->page_size % kF8Tokens) return tl::fail(TL_EINVAL, "%s: pages of a multiple of %d slots", op, kF8Tokens);
    if (p->dim <= 0 || p->dim > kApMostDim || p->dim % 16) return tl::fail(TL_EINVAL, "%s: heads of a multiple of 16 entries, at most %d", op, kApMostDim);
    if (!tl::aligned16(p->keys) || !tl::aligned16(p->values)) return tl::fail(TL_EINVAL, "%s: pages must begin on 16 bytes", op);
    return TL_OK;
}

template <typename T>
static int append_launch(const F8Append &a, const F8Turns &turns, cudaStream_t st) {
    static tl::PerDevice ready;
    const size_t room = a.tokens < kF8Tokens ? a.tokens : kF8Tokens;
    const size_t smem = room * (static_cast<size_t>(a.rot / 2) * 16 + 2u * a.pages.dim * 4);
    int device = 0;
    cudaGetDevice(&device);
    if (!ready(device, [&] { return cudaFuncSetAttribute(fp8_append_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, kF8Tokens * (kApMostDim * 8 + kApMostDim * 8)) == cudaSuccess; }))
        return tl::fail(TL_ECUDA, "fp8_append: %s", cudaGetErrorString(cudaGetLastError()));
    const int blocks = (a.tokens + 2 * kF8Tokens - 2) / kF8Tokens;
    const cudaError_t e = tl::launch_chained(fp8_append_kernel<T>, dim3(blocks, a.pages.heads, a.batch), dim3(kApThreads), smem, st, a, turns);
    if (e != cudaSuccess) return tl::fail(TL_ECUDA, "fp8_append: %s", cudaGetErrorString(e));
    TL_LAUNCH_CHECK("fp8_append");
    return TL_OK;
}

}  // namespace tlb

using namespace tlb;

extern "C" int tlb_fp8_append(const tlb_fp8_pages *pages, const tlb_fp8_append_call *c, void *stream) {
    const int rc = f8_check_pages("fp8_append", pages);
    if (rc != TL_OK) return rc;
    if (!c || c->batch < 0 || c->tokens < 0 || c->heads <= 0 || c->heads % pages->heads) return tl::fail(TL_EINVAL, "fp8_append: query heads over %d key/value heads", pages->heads);
    if (c->rot < 0 || c->rot % 2 || c->rot > pages->dim || !(c->base > 0.0)) return tl::fail(TL_EINVAL, "fp8_append: cannot rotate %d of %d entries", c->rot, pages->dim);
    if (c->batch == 0 || c->tokens == 0) return TL_OK;
    if (c->batch > 65535 || pages->heads > 65535 || c->tokens > (1 << 30) || c->max_pages <= 0) return tl::fail(TL_EINVAL, "fp8_append: sizes out of range");
    if (!c->q || !c->q_out || !c->k || !c->v || !c->table || !c->lens) return tl::fail(TL_EINVAL, "fp8_append: missing argument");
    // the frequencies of this thread's last call; half as many powers otherwise
    static thread_local F8Turns turns;
    static thread_local int turns_rot = -1;
    static thread_local double turns_base = 0.0;
    if (c->rot != turns_rot || c->base != turns_base) {
        for (int i = 0; i < c->rot / 2; ++i) turns.of[i] = pow(c->base, -2.0 * i / c->rot) / (2.0 * M_PI);
        turns_rot = c->rot, turns_base = c->base;
    }
    const F8Append a{*pages, *c, c->heads / pages->heads};
    TLB_DISPATCH(c->dtype, "fp8_append", return append_launch<T>(a, turns, as_stream(stream)));
}
