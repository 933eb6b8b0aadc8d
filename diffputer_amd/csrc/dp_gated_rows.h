// Gated projection of few rows (M <= 64: requests of one or some rows): bound by reading both weights once.
//
//   h[m, n] = act(x[m] . Wg[n] + bg[n]) * (x[m] . Wu[n] + bu[n])
//
// One launch, nothing to join behind it: a workgroup of 8 waves owns CB columns of h, its waves share the contraction (units
// of 64 k's in bf16, 32 in float32, in turn, so that neighbouring bytes of a row are read at the same time), each lane loads
// 16 bytes of a weight row straight into the matrix instruction's layout, and the waves' sums are added in order through LDS.
// CB = 16: 16 gate and 16 up rows, two fragments; CB = 8 (narrow layers, twice the workgroups): 8 gate and 8 up rows in one.
// x is read by every workgroup, from the L2.  The next round's weights are in flight under this one's products.
// Measured, bf16: 24 x 4096 x 8192 30 us, 134 MB of weights at 4.5 TB/s (a large copy moves 4.7); 1 x 1024 x 2048 4.2 us, of which
// about 3 are a launch's own.
#pragma once
#include "dp_gated_lds.h"

namespace dp {

constexpr int GR_WAVES = 8, GR_MAX_ROWS = 64;

// 16 bytes of a row from element k on, at any alignment; with END, elements at `end` and behind are zeros
template <typename T> struct GrLoad;
template <> struct GrLoad<bf16_t> {
    typedef bf16x8 V;
    static __device__ __forceinline__ f32x4 mul(V w, V x, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, x, c, 0, 0, 0); }
};
template <> struct GrLoad<float> {
    typedef f32x4 V;
    static __device__ __forceinline__ f32x4 mul(V w, V x, f32x4 c) {
#pragma unroll
        for (int s = 0; s < 4; ++s) c = __builtin_amdgcn_mfma_f32_16x16x4f32(w[s], x[s], c, 0, 0, 0);
        return c;
    }
};
template <typename T, bool END> __device__ __forceinline__ typename GrLoad<T>::V gr_get(const T* p, int k, int end) {
    constexpr int E = 16 / sizeof(T);
    typename GrLoad<T>::V v;
    if (!END || k + E <= end) __builtin_memcpy(&v, p + k, 16);
    else
#pragma unroll
        for (int e = 0; e < E; ++e) {
            T t = 0;
            if (k + e < end) t = p[k + e];
            v[e] = t;
        }
    return v;
}

template <typename T, int MT, int CB>
__global__ __launch_bounds__(GR_WAVES * 64, MT > 2 ? 2 : 4) void k_gated_rows(GlArgs p) {
    using L = GrLoad<T>;
    using V = typename L::V;
    constexpr int F = CB / 8;                                    // weight fragments: gate and up, or one with both
    constexpr int E = 16 / sizeof(T), STEP = 4 * E, U = MT == 1 && F == 1 ? 4 : 2;       // elements of a lane's load, of a fragment's; fragments of a round
    __shared__ f32x4 red[GR_WAVES][F][MT][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
    const int n0 = blockIdx.x * CB, K = (int)p.C, M = (int)p.I;
    const T *w[F], *x[MT];
#pragma unroll
    for (int f = 0; f < F; ++f) {
        const int half = F == 2 ? f : r >> 3, n = n0 + (F == 2 ? r : r & 7);
        w[f] = (const T*)p.B[half].p + (int64_t)(n < p.J ? n : p.J - 1) * p.B[half].ld;
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int m = t * 16 + r;
        x[t] = (const T*)p.A[0].p + (int64_t)(m < M ? m : M - 1) * p.A[0].ld;
    }
    f32x4 acc[F][MT];
#pragma unroll
    for (int f = 0; f < F; ++f)
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[f][t] = (f32x4){0.f, 0.f, 0.f, 0.f};
    // a round: U fragments of each row, two and two next to each other; the next round's weights are in flight under this one's products
    constexpr int ROUND = GR_WAVES * U * STEP;
    auto k_of = [&](int k0, int s) { return k0 + (s & 1) * STEP + (s >> 1) * (GR_WAVES * 2 * STEP) + q * E; };
    constexpr int SPAN = (U / 2 - 1) * (GR_WAVES * 2 * STEP) + 2 * STEP;      // a wave's round reads within [k0, k0 + SPAN)
    V wf[2][U][F], xf[U][MT];
    auto load = [&](auto end, V (*wd)[F], V (*xd)[MT], int k0) {
#pragma unroll
        for (int s = 0; s < U; ++s) {
            if (wd)
#pragma unroll
                for (int f = 0; f < F; ++f) wd[s][f] = gr_get<T, decltype(end)::value>(w[f], k_of(k0, s), K);
            if (xd)
#pragma unroll
                for (int t = 0; t < MT; ++t) xd[s][t] = gr_get<T, decltype(end)::value>(x[t], k_of(k0, s), K);
        }
    };
    auto load_at = [&](V (*wd)[F], V (*xd)[MT], int k0) {
        if (k0 + SPAN <= K) load(std::false_type{}, wd, xd, k0);
        else load(std::true_type{}, wd, xd, k0);
    };
    auto round = [&](const V (&cur)[U][F], V (&next)[U][F], int k0) {
        load_at(nullptr, xf, k0);
        if (k0 + ROUND < K) load_at(next, nullptr, k0 + ROUND);
#pragma unroll
        for (int s = 0; s < U; ++s)
#pragma unroll
            for (int f = 0; f < F; ++f)
#pragma unroll
                for (int t = 0; t < MT; ++t) acc[f][t] = L::mul(cur[s][f], xf[s][t], acc[f][t]);
    };
    int k0 = wave * 2 * STEP;
    if (k0 < K) load_at(wf[0], nullptr, k0);
    for (; k0 < K; k0 += 2 * ROUND) {
        round(wf[0], wf[1], k0);
        if (k0 + ROUND < K) round(wf[1], wf[0], k0 + ROUND);
    }
#pragma unroll
    for (int f = 0; f < F; ++f)
#pragma unroll
        for (int t = 0; t < MT; ++t) red[wave][f][t][lane] = acc[f][t];
    __syncthreads();
    // lane: row (lane & 15), rows 4 (lane >> 4) + 0..3 of the fragment
    for (int i = threadIdx.x; i < MT * 16 * CB / 4; i += GR_WAVES * 64) {
        const int t = i / (4 * CB), l = i % (4 * CB);
        const int m = t * 16 + (l & 15), n = n0 + (l >> 4) * 4, cnt = p.J - n < 4 ? p.J - n : 4;
        if (m >= M || cnt <= 0) continue;
        f32x4 g = red[0][0][t][l], u = F == 2 ? red[0][F - 1][t][l] : red[0][0][t][l + 32];
#pragma unroll
        for (int v = 1; v < GR_WAVES; ++v) {
            g += red[v][0][t][l];
            u += F == 2 ? red[v][F - 1][t][l] : red[v][0][t][l + 32];
        }
        gl_fwd_store<T>(p, m, n, cnt, g, u);
    }
}

}  // namespace dp
