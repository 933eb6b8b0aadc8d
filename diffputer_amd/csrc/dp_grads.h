// Global norm of many gradient tensors, and clipping by it.
//
//   norm = sqrt(sum over tensors and elements of g^2)   or   max |g|
//   coef = min(1, limit / (norm + 1e-6)),  g <- g coef  (in place; nothing is written when coef is 1)
//
// Two passes over memory: k_grad_norm leaves one partial per workgroup, k_grad_clip reduces the partials (each workgroup
// for itself, in one fixed order: same bits everywhere) and scales.  Bound by memory, in small sets by the two launches: 0.8 GB of float32
// within the limit 135 us (5.9 TB/s), 2^27 bf16 numbers in 301 tensors clipped in 156 to 170 us on three cards (0.27 GB read,
// then read and written: 4.7 to 5.1 TB/s), 42 MB in 14 tensors in 25.6 us, 0.3 MB in 10.  Sums are float64; squares are added up in float32 within pairs
// (float32) or fours (bf16, whose squares are exact), two roundings at most, and only those go to float64: one conversion per
// element held the kernel to 1.25 elements per ps, 2.5 TB/s in bf16.  A group outside [2^-96, inf) takes the long way, element
// by element in float64: no square overflows or vanishes.
#pragma once
#include "dp_util.h"

namespace dp {

// One tensor of the table that travels in the kernel's arguments (no upload, nothing a captured graph could outlive).
struct GradEntry {
    uint64_t base;             // address rounded down to 16
    uint64_t bytes;            // from `base` to the end of the tensor
    uint32_t chunk0;           // first chunk of this tensor
    uint16_t head;             // bytes between `base` and the first element (< 16)
    uint16_t bf16;             // element type: 1 = bf16, 0 = float32
};
constexpr int GN_MAX = 160;    // entries per launch: 24 bytes each, under the 4 KiB of kernel arguments
struct GradTable {
    int n;
    uint32_t chunks;
    GradEntry e[GN_MAX];
};
constexpr int GN_CHUNK = 16384;                                  // bytes of one chunk: 4 loads of 16 bytes per thread
constexpr int GN_THREADS = 256;
// Workgroups of a launch, eight per CU: four per CU read 0.8 GB in 166 us, eight in 134 (6.0 TB/s); chunks of 32 KiB or 8 KiB
// change nothing there and lose 1 to 2 us at 0.3 MB and 42 MB.
constexpr int GN_MAX_BLOCKS = 2048;

// The entry that holds a chunk (a walk along the table, 40 entries per chunk where 301 tensors share a launch or two, took 30 us
// of 185): lane l keeps the first chunks of entries l, l + 64 and l + 128 and the wave counts those that are not
// behind it.
struct GnFirst {
    uint32_t c[(GN_MAX + 63) / 64];
    __device__ __forceinline__ explicit GnFirst(const GradTable& t) {
#pragma unroll
        for (int k = 0; k < (GN_MAX + 63) / 64; ++k) {
            const int i = k * 64 + (threadIdx.x & 63);
            c[k] = i < t.n ? t.e[i].chunk0 : ~0u;
        }
    }
    __device__ __forceinline__ int find(uint32_t chunk) const {
        int n = -1;
#pragma unroll
        for (int k = 0; k < (GN_MAX + 63) / 64; ++k) n += __popcll(__ballot(c[k] <= chunk));
        return n;
    }
};

__device__ __forceinline__ double gn_join(int inf, double a, double b) {
    if (!inf) return a + b;
    return (b > a || b != b) ? b : a;                            // NaN wins
}
__device__ __forceinline__ void gn_take(int inf, double& a, float v) {
    if (!inf) a = fma((double)v, (double)v, a);
    else a = gn_join(1, a, (double)fabsf(v));
}

// sum of the squares (or the maximum) of 16 bytes
__device__ __forceinline__ void gn_take16(int inf, bool bf, double& a, const uint32_t (&w)[4]) {
    float x[8];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        x[2 * k] = __builtin_bit_cast(float, bf ? w[k] << 16 : w[k]);
        x[2 * k + 1] = __builtin_bit_cast(float, w[k] & 0xffff0000u);
    }
    const float g0 = bf ? fmaf(x[0], x[0], x[1] * x[1]) + fmaf(x[2], x[2], x[3] * x[3]) : fmaf(x[0], x[0], x[2] * x[2]);
    const float g1 = bf ? fmaf(x[4], x[4], x[5] * x[5]) + fmaf(x[6], x[6], x[7] * x[7]) : fmaf(x[4], x[4], x[6] * x[6]);
    const float lo = 0x1p-96f, hi = 0x1.fffffep127f;
    if (!inf && g0 >= lo && g1 >= lo && g0 <= hi && g1 <= hi) {
        a += (double)g0;
        a += (double)g1;
    } else if ((w[0] | w[1] | w[2] | w[3]) & (bf ? 0x7fff7fffu : 0x7fffffffu)) {              // not all zeros
        for (int k = 0; k < (bf ? 8 : 4); ++k) gn_take(inf, a, bf ? x[k] : x[2 * k]);
    }
}

// sum (or maximum) over the workgroup, valid in every thread
__device__ __forceinline__ double gn_block(int inf, double v, double* red) {
    for (int o = 32; o; o >>= 1) v = gn_join(inf, v, __shfl_xor(v, o));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
    for (int w = 1; w < GN_THREADS / 64; ++w) v = gn_join(inf, v, red[w]);
    return v;
}

__global__ __launch_bounds__(GN_THREADS) void k_grad_norm(GradTable t, double* part, int inf) {
    __shared__ double red[GN_THREADS / 64];
    double a = 0.0;
    const GnFirst first(t);
    for (uint32_t c = blockIdx.x; c < t.chunks; c += gridDim.x) {
        const GradEntry e = t.e[first.find(c)];
        const uint64_t off0 = (uint64_t)(c - e.chunk0) * GN_CHUNK;
        const char* const base = (const char*)e.base;
        const int es = e.bf16 ? 2 : 4;
#pragma unroll 8
        for (int v = 0; v < GN_CHUNK / 16 / GN_THREADS; ++v) {
            const uint64_t o = off0 + (uint64_t)(v * GN_THREADS + threadIdx.x) * 16;
            if (o >= e.head && o + 16 <= e.bytes) {
                const uint4 q = *(const uint4*)(base + o);
                const uint32_t w[4] = {q.x, q.y, q.z, q.w};
                gn_take16(inf, e.bf16, a, w);
            } else {
                for (uint64_t b = o < e.head ? e.head : o; b < o + 16 && b < e.bytes; b += es)
                    gn_take(inf, a, e.bf16 ? bf2f(*(const bf16_t*)(base + b)) : *(const float*)(base + b));
            }
        }
    }
    a = gn_block(inf, a, red);
    if (threadIdx.x == 0) part[blockIdx.x] = a;
}

__device__ __forceinline__ double gn_total(const double* part, int nparts, int inf, double* red) {
    double a = 0.0;
    for (int i = threadIdx.x; i < nparts; i += GN_THREADS) a = gn_join(inf, a, part[i]);
    a = gn_block(inf, a, red);
    return inf ? a : sqrt(a);
}

__global__ __launch_bounds__(GN_THREADS) void k_grad_total(const double* part, int nparts, int inf, float* norm) {
    __shared__ double red[GN_THREADS / 64];
    const double total = gn_total(part, nparts, inf, red);
    if (threadIdx.x == 0) *norm = (float)total;
}

// The table names the tensors from the last to the first, and a tensor's chunks are taken from its end: the end of what
// k_grad_norm read is what the caches still hold.
__global__ __launch_bounds__(GN_THREADS) void k_grad_clip(GradTable t, const double* part, int nparts, int inf, double limit, float* norm) {
    __shared__ double red[GN_THREADS / 64];
    const GnFirst first(t);
    const double total = gn_total(part, nparts, inf, red);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)total;
    const double cd = limit / (total + 1e-6);
    if (cd >= 1.0) return;                                       // within the limit (a NaN coefficient goes on, and marks every element)
    const float coef = (float)cd;
    if (coef == 1.0f) return;
    for (uint32_t c = blockIdx.x; c < t.chunks; c += gridDim.x) {
        const GradEntry e = t.e[first.find(c)];
        const uint64_t off0 = (uint64_t)((uint32_t)((e.bytes - 1) / GN_CHUNK) - (c - e.chunk0)) * GN_CHUNK;
        char* const base = (char*)e.base;
        const int es = e.bf16 ? 2 : 4;
#pragma unroll 8
        for (int v = 0; v < GN_CHUNK / 16 / GN_THREADS; ++v) {
            const uint64_t o = off0 + (uint64_t)(v * GN_THREADS + threadIdx.x) * 16;
            if (o >= e.head && o + 16 <= e.bytes) {
                uint4 q = *(const uint4*)(base + o);
                uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    if (e.bf16) w[k] = pack_bf16x2(__builtin_bit_cast(float, w[k] << 16) * coef, __builtin_bit_cast(float, w[k] & 0xffff0000u) * coef);
                    else w[k] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(float, w[k]) * coef);
                }
                *(uint4*)(base + o) = make_uint4(w[0], w[1], w[2], w[3]);
            } else {
                for (uint64_t b = o < e.head ? e.head : o; b < o + 16 && b < e.bytes; b += es) {
                    if (e.bf16) *(bf16_t*)(base + b) = f2bf(bf2f(*(const bf16_t*)(base + b)) * coef);
                    else *(float*)(base + b) *= coef;
                }
            }
        }
    }
}

}  // namespace dp
