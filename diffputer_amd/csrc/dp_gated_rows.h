// Gated projection of few rows (M <= 64: requests of one or some rows): bound by reading both weights once.
//
//   h[m, n] = act(x[m] . Wg[n] + bg[n]) * (x[m] . Wu[n] + bu[n])
//
// One launch, nothing to join behind it: a workgroup of 8 waves owns CB columns of h, its waves share the contraction (units
// of 64 k's in bf16, 32 in float32, in turn, so that neighbouring bytes of a row are read at the same time), each lane loads
// 16 bytes of a weight row straight into the matrix instruction's layout, and the waves' sums are added in order through LDS.
// CB = 16: 16 gate and 16 up rows, two fragments; CB = 8 (narrow layers, twice the workgroups): 8 gate and 8 up rows in one.
// x is read by every workgroup, from the L2.
#pragma once
#include "dp_gated_lds.h"

namespace dp {

constexpr int GR_WAVES = 8, GR_MAX_ROWS = 64;

// 16 bytes of row `p` from element k on; elements at `end` and behind are zeros
template <typename T, bool VEC> struct GrLoad;
template <bool VEC> struct GrLoad<bf16_t, VEC> {
    typedef bf16x8 V;
    static __device__ __forceinline__ V get(const bf16_t* p, int k, int end) {
        if (VEC) {                                               // end % 8 == 0: all or nothing
            const bool in = k < end;
            V v = *(const V*)(p + (in ? k : 0));
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = in ? v[e] : (short)0;
            return v;
        }
        V v;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = k + e < end ? (short)p[k + e] : (short)0;
        return v;
    }
    static __device__ __forceinline__ f32x4 mul(V w, V x, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, x, c, 0, 0, 0); }
};
template <bool VEC> struct GrLoad<float, VEC> {
    typedef f32x4 V;
    static __device__ __forceinline__ V get(const float* p, int k, int end) {
        if (VEC) {                                               // end % 4 == 0
            const bool in = k < end;
            V v = *(const V*)(p + (in ? k : 0));
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = in ? v[e] : 0.f;
            return v;
        }
        V v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = k + e < end ? p[k + e] : 0.f;
        return v;
    }
    static __device__ __forceinline__ f32x4 mul(V w, V x, f32x4 c) {
#pragma unroll
        for (int s = 0; s < 4; ++s) c = __builtin_amdgcn_mfma_f32_16x16x4f32(w[s], x[s], c, 0, 0, 0);
        return c;
    }
};

template <typename T, int MT, int CB, bool VEC>
__global__ __launch_bounds__(GR_WAVES * 64, MT > 2 ? 2 : 4) void k_gated_rows(GlArgs p) {
    using L = GrLoad<T, VEC>;
    using V = typename L::V;
    constexpr int F = CB / 8;                                    // weight fragments: gate and up, or one with both
    constexpr int E = 16 / sizeof(T), STEP = 4 * E, U = MT == 1 ? 4 : 2;       // elements of a lane's load, of a fragment's; fragments of a round
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
    // a round: U fragments of each row, two and two next to each other
    for (int k0 = wave * 2 * STEP; k0 < K; k0 += GR_WAVES * U * STEP) {
        V wf[U][F], xf[U][MT];
#pragma unroll
        for (int s = 0; s < U; ++s) {
            const int k = k0 + (s & 1) * STEP + (s >> 1) * (GR_WAVES * 2 * STEP) + q * E;
#pragma unroll
            for (int f = 0; f < F; ++f) wf[s][f] = L::get(w[f], k, K);
#pragma unroll
            for (int t = 0; t < MT; ++t) xf[s][t] = L::get(x[t], k, K);
        }
#pragma unroll
        for (int s = 0; s < U; ++s)
#pragma unroll
            for (int f = 0; f < F; ++f)
#pragma unroll
                for (int t = 0; t < MT; ++t) acc[f][t] = L::mul(wf[s][f], xf[s][t], acc[f][t]);
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
