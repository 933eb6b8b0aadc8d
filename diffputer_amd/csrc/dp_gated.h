// Gated projection h = act(x Wg^T + bg) * (x Wu^T + bu) and its backward: the three products that carry it, and the
// elementwise passes between them.
//
//   forward   g = x Wg^T + bg, u = x Wu^T + bu, h = act(g) u                  x [M, K], W [N, K], h [M, N]
//   backward  du = dh act(g), dg = dh u act'(g)                               (k_gated_dgu, with the column sums for db)
//             dx = dg Wg + du Wu          one product over a contraction of 2 N
//             dWg = dg^T x, dWu = du^T x  two products over the rows
//
// All three are C(i, j) = sum_k A(i, k) B(j, k) with each operand either "row" laid out (k contiguous) or "column" laid
// out (i or j contiguous, as a transposed product finds its operands in memory).
#pragma once
#include <type_traits>

#include "dp_util.h"

namespace dp {

enum { GL_FWD = 0, GL_DX = 1, GL_DW = 2 };
enum { GL_ACT_NONE = 0, GL_ACT_SILU = 1, GL_ACT_GELU = 2 };

// ---- scalar types --------------------------------------------------------------------------------------------------
template <typename T> struct GlType;
template <> struct GlType<float> {
    static __device__ __forceinline__ float get(float v) { return v; }
    static __device__ __forceinline__ float put(float v) { return v; }
};
template <> struct GlType<bf16_t> {
    static __device__ __forceinline__ float get(bf16_t v) { return bf2f(v); }
    static __device__ __forceinline__ bf16_t put(float v) { return f2bf(v); }
};

// ---- activations, float32 ------------------------------------------------------------------------------------------
// silu(g) = g s(g), s = 1 / (1 + e^-g): e^-g overflows to inf below -88, where s is 0 and the product the right -0;
// gelu(g) = g Phi(g), Phi = erfc(-g / sqrt 2) / 2 (erfc keeps the relative accuracy of the left tail that 1 + erf loses).
// At g = -inf both products are 0 * inf = NaN; plain torch expressions give the same.
// float32 results take erfcf, expf and a division; for bf16 results the hardware's 2^x and reciprocal do (|g| 2^-24 + 2^-22 of s: at
// most 2^-17 where s is not 0, against half a step of 2^-9): what a 256-tile launch takes beyond its K-tiles fell from 18.9 to
// 11.4 us with them.  Phi is e^(-g^2 / 2) t P(t) there, t = 1 / (1 + 0.3076 |g|), for g < 0 (1 - that for g > 0), P fitted to
// the function's tail e^(x^2) erfc(x) by least relative maximum: 2^-18 of it, 2^-16.7 of Phi with the exponential, down to -13.4.
template <typename T> __device__ __forceinline__ float gl_sigmoid(float g) {
    if (sizeof(T) == 4) return 1.0f / (1.0f + expf(-g));
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(g * -1.44269504088896340736f));
}
template <typename T> __device__ __forceinline__ float gl_exp(float x) {
    return sizeof(T) == 4 ? expf(x) : __builtin_amdgcn_exp2f(x * 1.44269504088896340736f);
}
// Phi(g), with e = e^(-g^2 / 2)
template <typename T> __device__ __forceinline__ float gl_phi(float g, float e) {
    if (sizeof(T) == 4) return 0.5f * erfcf(-0.70710678118654752f * g);
    const float t = __builtin_amdgcn_rcpf(fmaf(0.30759145f, fabsf(g), 1.0f));
    float q = -0.075778842f;
    q = fmaf(q, t, 0.19164754f);
    q = fmaf(q, t, 0.0053418200f);
    q = fmaf(q, t, 0.13728017f);
    q = fmaf(q, t, 0.11853294f);
    q = fmaf(q, t, 0.12297484f);
    q *= e * t;
    return g < 0.0f ? q : 1.0f - q;
}
template <typename T, int ACT> __device__ __forceinline__ float gl_act(float g) {
    if (ACT == GL_ACT_SILU) return g * gl_sigmoid<T>(g);
    if (ACT == GL_ACT_GELU) return g * gl_phi<T>(g, gl_exp<T>(-0.5f * g * g));
    return g;
}
template <typename T, int ACT> __device__ __forceinline__ void gl_act_grad(float g, float& a, float& da) {
    if (ACT == GL_ACT_SILU) {
        const float s = gl_sigmoid<T>(g);
        a = g * s;
        da = s * (1.0f + g * (1.0f - s));
    } else if (ACT == GL_ACT_GELU) {
        const float e = gl_exp<T>(-0.5f * g * g), p = gl_phi<T>(g, e);
        a = g * p;
        da = p + g * (0.39894228040143268f * e);
    } else {
        a = g;
        da = 1.0f;
    }
}
// calls f with the activation as a constant
template <typename F> __device__ __forceinline__ void gl_with_act(int act, F f) {
    if (act == GL_ACT_SILU) f(std::integral_constant<int, GL_ACT_SILU>{});
    else if (act == GL_ACT_GELU) f(std::integral_constant<int, GL_ACT_GELU>{});
    else f(std::integral_constant<int, GL_ACT_NONE>{});
}

// ---- operands ------------------------------------------------------------------------------------------------------
// row layout:    element (i, k) at p[i * ld + k]     (k contiguous)
// column layout: element (i, k) at p[k * ld + i]     (i contiguous)
struct GlOp {
    const void* p;
    int64_t ld;
    int64_t cols;              // elements of a row that exist
};

// One product launch.  GL_FWD: A = x (row), B[0] / B[1] = Wg / Wu (row): columns 0..n-1 of the gate and of the up product.
// GL_DX: A[s] = dg / du planes (row), B[s] = Wg / Wu (column), s = contraction segment.  GL_DW: A[z] = dg / du plane
// (column), B[0] = x (column), z = which weight.
// Split launches (splits > 1): slice s takes K-tiles [s, s + 1) * kt_per of the contraction and writes float32 sums to
// part[s][plane][rows][ldp]; k_gated_join adds the slices in order, so results do not depend on timing.
struct GlArgs {
    GlOp A[2], B[2];
    int64_t I;                 // rows of C
    int J;                     // columns of C (of one plane)
    int64_t C;                 // contraction length of one segment
    int kt_per, splits;        // K-tiles per slice, slices
    int zfirst;                // GL_DW: first plane of this launch (0, or 1 where only the up weight's gradient is asked for)
    // outputs
    void* out[2];              // GL_FWD: h in out[0]; GL_DX: dx; GL_DW: dWg, dWu
    int64_t ldo;
    float* part;               // split launches: partial sums
    int64_t ldp;
    void* pre;                 // GL_FWD, training: g and u for the backward pass (GlPre)
    const void* bias[2];
    int act;
};

// four columns of one row, at any alignment of their elements (the loads and stores of this chip take it)
template <typename T> struct GlVec;
template <> struct GlVec<float> { typedef f32x4 V; static __device__ __forceinline__ V put(f32x4 v) { return v; } static __device__ __forceinline__ f32x4 get(V v) { return v; } };
template <> struct GlVec<bf16_t> {
    typedef uint2 V;
    static __device__ __forceinline__ V put(f32x4 v) { return make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])); }
    static __device__ __forceinline__ f32x4 get(V v) {
        return (f32x4){__builtin_bit_cast(float, v.x << 16), __builtin_bit_cast(float, v.x & 0xffff0000u), __builtin_bit_cast(float, v.y << 16), __builtin_bit_cast(float, v.y & 0xffff0000u)};
    }
};
template <typename T> __device__ __forceinline__ void gl_put4(T* o, f32x4 v, int cnt) {
    if (cnt >= 4) {
        const typename GlVec<T>::V q = GlVec<T>::put(v);
        __builtin_memcpy(o, &q, sizeof q);
    } else
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (r < cnt) o[r] = GlType<T>::put(v[r]);
}
template <typename T> __device__ __forceinline__ f32x4 gl_get4(const T* o, int cnt) {
    if (cnt >= 4) {
        typename GlVec<T>::V q;
        __builtin_memcpy(&q, o, sizeof q);
        return GlVec<T>::get(q);
    }
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int r = 0; r < 4; ++r)
        if (r < cnt) v[r] = GlType<T>::get(o[r]);
    return v;
}
// the biases of columns n .. n + cnt - 1
template <typename T> __device__ __forceinline__ void gl_bias(const GlArgs& p, int n, int cnt, f32x4& bg, f32x4& bu) {
    bg = bu = (f32x4){0.f, 0.f, 0.f, 0.f};
    if (p.bias[0]) bg = gl_get4((const T*)p.bias[0] + n, cnt);
    if (p.bias[1]) bu = gl_get4((const T*)p.bias[1] + n, cnt);
}
// The projections g and u as the forward pass leaves them for the backward pass, by groups of 4 columns (G = N / 4 rounded up):
//   float32   g[4], u[4]: two planes [M][G] of 16 bytes
//   bf16      20 bits of each (sign, exponent, 11 bits of the fraction; rounded, half away from zero): a plane [M][G] of 16 bytes with the
//             upper 16 bits of g[4] and u[4], and a plane [M][G] of 4 bytes with the next 4 bits of each, whole blocks of 8 groups
//             in the order 0 4 1 5 2 6 3 7: a lane of the tile kernels has groups q and q + 4 and stores both at once (with 16 bytes
//             per row and store the forward product of 4096 x 1024 x 2048 wrote 69 MB to memory, for 59 of results).
// Half a step of 20 bits is 2^-12: dg = dh u act'(g) is off by a sixteenth of the rounding to bf16 that it gets as an operand
// anyway, and neither float32's exponents nor inf and NaN are lost, as they would be in 16 bits of either kind (numbers within 2^-13
// of float32's largest become inf).  Against float32 planes the
// forward pass writes and the backward pass reads 20 instead of 32 bytes per group.
template <typename T> struct GlPre;
template <> struct GlPre<float> {
    static __host__ __device__ int64_t bytes(int64_t M, int64_t G) { return M * G * 32; }
    static __device__ __forceinline__ void put(void* pre, int64_t M, int64_t G, int64_t m, int n, f32x4 g, f32x4 u) {
        f32x4* const p = (f32x4*)pre + m * G + (n >> 2);
        p[0] = g;
        p[M * G] = u;
    }
    static __device__ __forceinline__ void get(const void* pre, int64_t M, int64_t G, int64_t m, int n, f32x4& g, f32x4& u) {
        const f32x4* const p = (const f32x4*)pre + m * G + (n >> 2);
        g = p[0];
        u = p[M * G];
    }
};
template <> struct GlPre<bf16_t> {
    static __host__ __device__ int64_t bytes(int64_t M, int64_t G) { return M * G * 20; }
    static __device__ __forceinline__ uint32_t* low(const void* pre, int64_t M, int64_t G, int64_t m, int g) {
        const int block = g & ~7;
        return (uint32_t*)((char*)pre + M * G * 16) + m * G + (block + 8 <= G ? block | (g & 3) << 1 | (g >> 2 & 1) : g);
    }
    // stores the upper bits, returns the next ones
    static __device__ __forceinline__ uint32_t put_high(void* pre, int64_t G, int64_t m, int n, f32x4 g, f32x4 u) {
        uint32_t b[8], low = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            b[e] = __builtin_bit_cast(uint32_t, e < 4 ? g[e] : u[e - 4]) + 0x800u;             // carries into the exponent as a rounding does
            low |= ((b[e] >> 12) & 15u) << (4 * e);
        }
        uint4 hi;
        hi.x = __builtin_amdgcn_perm(b[1], b[0], 0x07060302u);
        hi.y = __builtin_amdgcn_perm(b[3], b[2], 0x07060302u);
        hi.z = __builtin_amdgcn_perm(b[5], b[4], 0x07060302u);
        hi.w = __builtin_amdgcn_perm(b[7], b[6], 0x07060302u);
        ((uint4*)pre)[m * G + (n >> 2)] = hi;
        return low;
    }
    static __device__ __forceinline__ void put(void* pre, int64_t M, int64_t G, int64_t m, int n, f32x4 g, f32x4 u) {
        *low(pre, M, G, m, n >> 2) = put_high(pre, G, m, n, g, u);
    }
    // columns n .. and n + 16 .., n in the first half of a block of 32
    static __device__ __forceinline__ void put2(void* pre, int64_t M, int64_t G, int64_t m, int n, const f32x4 (&g)[2], const f32x4 (&u)[2]) {
        const uint32_t l[2] = {put_high(pre, G, m, n, g[0], u[0]), put_high(pre, G, m, n + 16, g[1], u[1])};
        const int first = n >> 2;
        uint32_t* const at = low(pre, M, G, m, first);
        if ((first & ~7) + 8 <= G) __builtin_memcpy(at, l, 8);
        else {
            at[0] = l[0];
            at[4] = l[1];
        }
    }
    static __device__ __forceinline__ void get(const void* pre, int64_t M, int64_t G, int64_t m, int n, f32x4& g, f32x4& u) {
        const int64_t at = m * G + (n >> 2);
        const uint4 hi = ((const uint4*)pre)[at];
        const uint32_t low = *GlPre::low(pre, M, G, m, n >> 2);
        const uint32_t h[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t b = (e & 1 ? h[e >> 1] & 0xffff0000u : h[e >> 1] << 16) | ((low >> (4 * e)) & 15u) << 12;
            if (e < 4) g[e] = __builtin_bit_cast(float, b);
            else u[e - 4] = __builtin_bit_cast(float, b);
        }
    }
};
// h of row m, columns n .. n + cnt - 1 (n a multiple of 4), from both finished projections
template <typename T, int ACT> __device__ __forceinline__ void gl_fwd_put(const GlArgs& p, int64_t m, int n, int cnt, f32x4 g, f32x4 u) {
    if (p.pre) GlPre<T>::put(p.pre, p.I, (p.J + 3) >> 2, m, n, g, u);
    f32x4 v;
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = gl_act<T, ACT>(g[r]) * u[r];
    T* const h = (T*)p.out[0];
    gl_put4(h + m * p.ldo + n, v, cnt);
}
// the same of columns n .. and n + 16 .. (bf16 tile kernels), n < J in the first half of a block of 32
template <int ACT> __device__ __forceinline__ void gl_fwd_put2(const GlArgs& p, int64_t m, int n, const f32x4 (&g)[2], const f32x4 (&u)[2]) {
    const bool both = n + 16 < p.J;
    if (p.pre) {
        if (both) GlPre<bf16_t>::put2(p.pre, p.I, (p.J + 3) >> 2, m, n, g, u);
        else GlPre<bf16_t>::put(p.pre, p.I, (p.J + 3) >> 2, m, n, g[0], u[0]);
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        f32x4 v;
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = gl_act<bf16_t, ACT>(g[j][r]) * u[j][r];
        if (j == 0 || both) gl_put4((bf16_t*)p.out[0] + m * p.ldo + n + 16 * j, v, p.J - n - 16 * j);
    }
}
template <typename T> __device__ __forceinline__ void gl_fwd_store(const GlArgs& p, int64_t m, int n, int cnt, f32x4 g, f32x4 u) {
    f32x4 bg, bu;
    gl_bias<T>(p, n, cnt, bg, bu);
    gl_with_act(p.act, [&](auto act) { gl_fwd_put<T, decltype(act)::value>(p, m, n, cnt, g + bg, u + bu); });
}

// ---- general product: any size, stride and alignment ------------------------------------------------------------------
// 64 x 64 x 32 tile, 4 waves of 32 x 32, operands through registers into LDS as [row][k] (element loads with bounds checks).
// GL_FWD: columns 0..31 of the tile are 32 gate columns, 32..63 the up columns of the same places, so that one lane ends
// with g and u of the same elements.
// TA: type of A.  bf16 layers' dg and du are float32 here and multiplied as bf16 hi + lo, two products, so that there is no rounding
// between the gradient of h and the sums.
constexpr int GG_T = 64, GG_K = 32;
struct GgArgs {
    GlArgs g;
    int ti, tj, wgs;           // tiles along I and J; workgroups: tiles x slices x planes
};
template <typename T> struct GgShape {
    static constexpr int LD = sizeof(T) == 2 ? GG_K + 8 : GG_K + 1, PART = GG_T * LD;         // row stride; elements of an operand
};
template <typename T, typename TA, int MODE>
__device__ __forceinline__ void gg_product(const GgArgs& q, int block, T* smem) {
    constexpr bool BF = sizeof(T) == 2, HILO = BF && sizeof(TA) == 4;
    constexpr int LD = GgShape<T>::LD;
    constexpr bool A_ROW = MODE != GL_DW, B_ROW = MODE == GL_FWD;
    T *const sa = smem, *const sb = smem + GgShape<T>::PART, *const slo = smem + 2 * GgShape<T>::PART;
    const GlArgs& p = q.g;
    const int bx = block % q.ti, by = block / q.ti % q.tj, bz = block / q.ti / q.tj;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave >> 1, wn = wave & 1;
    const int64_t i0 = (int64_t)bx * GG_T;
    const int j0 = by * (MODE == GL_FWD ? GG_T / 2 : GG_T);
    const int slice = bz % p.splits, plane = p.zfirst + bz / p.splits;
    const int segs = MODE == GL_DX ? 2 : 1;
    const int64_t nk = ceil_div<int64_t>(p.C, GG_K);
    const int64_t kt0 = (int64_t)slice * p.kt_per, kt1 = kt0 + p.kt_per < nk * segs ? kt0 + p.kt_per : nk * segs;

    TA ra[8];
    T rb[8];
    auto load8 = [&](auto* r, const auto* src, int64_t valid) {    // `valid` of the 8 elements exist
        if (valid >= 8) {
            __builtin_memcpy(r, src, 8 * sizeof *r);
            return;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            r[e] = 0;
            if (e < valid) r[e] = src[e];
        }
    };
    // row layout: thread = (row tid / 4, 8 k's from (tid % 4) * 8); column layout: thread = (k tid / 8, 8 rows from (tid % 8) * 8)
    auto fetch = [&](int64_t kt) {
        const int seg = kt >= nk ? 1 : 0;
        const int64_t k0 = (kt - seg * nk) * GG_K;
        const GlOp A = p.A[MODE == GL_DX ? seg : MODE == GL_DW ? plane : 0];
        if (A_ROW) {
            const int64_t i = i0 + (tid >> 2), k = k0 + (tid & 3) * 8;
            load8(ra, (const TA*)A.p + i * A.ld + k, i < p.I ? p.C - k : 0);
        } else {
            const int64_t k = k0 + (tid >> 3), i = i0 + (tid & 7) * 8;
            load8(ra, (const TA*)A.p + k * A.ld + i, k < p.C ? p.I - i : 0);
        }
        if (B_ROW) {
            const int row = tid >> 2, half = row >> 5;
            const int64_t j = j0 + (row & 31), k = k0 + (tid & 3) * 8;
            load8(rb, (const T*)p.B[half].p + j * p.B[half].ld + k, j < p.J ? p.C - k : 0);
        } else {
            const GlOp B = p.B[MODE == GL_DX ? seg : 0];
            const int64_t k = k0 + (tid >> 3);
            const int j = j0 + (tid & 7) * 8;
            load8(rb, (const T*)B.p + k * B.ld + j, k < p.C ? p.J - j : 0);
        }
    };
    auto put8 = [&](T* s, const T* r, bool row) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (row) s[(tid >> 2) * LD + (tid & 3) * 8 + e] = r[e];
            else s[((tid & 7) * 8 + e) * LD + (tid >> 3)] = r[e];
        }
    };

    f32x4 acc[2][2];                                               // [m-tile][column half]
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
    if (kt0 < kt1) fetch(kt0);
    for (int64_t kt = kt0; kt < kt1; ++kt) {
        __syncthreads();
        if constexpr (HILO) {
            T hi[8], lo[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                hi[e] = f2bf(ra[e]);
                const float left = ra[e] - bf2f(hi[e]);
                lo[e] = __builtin_isfinite(left) ? f2bf(left) : (T)0;          // inf and NaN are in hi
            }
            put8(sa, hi, A_ROW);
            put8(slo, lo, A_ROW);
        } else put8(sa, ra, A_ROW);
        put8(sb, rb, B_ROW);
        __syncthreads();
        if (kt + 1 < kt1) fetch(kt + 1);
        const int r = lane & 15, q = lane >> 4;
        if constexpr (BF) {
            bf16x8 a[2], b[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                a[i] = *(const bf16x8*)&sa[(wm * 32 + i * 16 + r) * LD + q * 8];
                b[i] = *(const bf16x8*)&sb[(i * 32 + wn * 16 + r) * LD + q * 8];
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[j], a[i], acc[i][j], 0, 0, 0);
            if constexpr (HILO) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const bf16x8 l = *(const bf16x8*)&slo[(wm * 32 + i * 16 + r) * LD + q * 8];
#pragma unroll
                    for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[j], l, acc[i][j], 0, 0, 0);
                }
            }
        } else {
#pragma unroll
            for (int kk = 0; kk < GG_K / 4; ++kk) {
                float a[2], b[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    a[i] = sa[(wm * 32 + i * 16 + r) * LD + kk * 4 + q];
                    b[i] = sb[(i * 32 + wn * 16 + r) * LD + kk * 4 + q];
                }
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(b[j], a[i], acc[i][j], 0, 0, 0);
            }
        }
    }
    // lane: row (lane & 15) of each 16 x 16 tile, columns 4 (lane >> 4) + 0..3
    const int cl = wn * 16 + (lane >> 4) * 4;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int64_t m = i0 + wm * 32 + i * 16 + (lane & 15);
        if (m >= p.I) continue;
        if (MODE == GL_FWD && p.splits == 1) {
            const int n = j0 + cl, cnt = p.J - n < 4 ? p.J - n : 4;
            if (cnt > 0) gl_fwd_store<T>(p, m, n, cnt, acc[i][0], acc[i][1]);
            continue;
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int n = j0 + (MODE == GL_FWD ? 0 : j * 32) + cl;
            const int pl = MODE == GL_FWD ? j : MODE == GL_DW ? plane : 0;
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (n + r < p.J) {
                    if (p.splits > 1) p.part[(((int64_t)slice * 2 + pl) * p.I + m) * p.ldp + n + r] = acc[i][j][r];
                    else ((T*)p.out[pl])[m * p.ldo + n + r] = GlType<T>::put(acc[i][j][r]);
                }
        }
    }
}

template <typename T, typename TA, int MODE>
__global__ __launch_bounds__(256) void k_gated_mm(GgArgs q) {
    __shared__ __attribute__((aligned(16))) T smem[3 * GgShape<T>::PART];
    const int64_t b = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
    if (b < q.wgs) gg_product<T, TA, MODE>(q, (int)b, smem);
}

// Joins the slices of a split launch, in order: 4 columns of one row per step.
template <typename T, int MODE>
__device__ __forceinline__ void gl_join(const GlArgs& p, int planes, int64_t first, int64_t step) {
    const int64_t per_row = ceil_div(p.J, 4), rows = p.I * planes, total = rows * per_row;
    const int64_t stride = 2 * p.I * p.ldp;
    for (int64_t t = first; t < total; t += step) {
        const int64_t row = t / per_row;
        const int n = (int)(t - row * per_row) * 4, cnt = p.J - n < 4 ? p.J - n : 4;
        const int pl = p.zfirst + (int)(row / p.I);
        const int64_t m = row % p.I;
        const float* a = p.part + ((int64_t)pl * p.I + m) * p.ldp + n;
        f32x4 s0 = *(const f32x4*)a, s1 = (f32x4){0.f, 0.f, 0.f, 0.f};
        const float* b = a + p.I * p.ldp;                          // GL_FWD: the up plane
        if (MODE == GL_FWD) s1 = *(const f32x4*)b;
#pragma unroll 8
        for (int s = 1; s < p.splits; ++s) {
            s0 += *(const f32x4*)(a + s * stride);
            if (MODE == GL_FWD) s1 += *(const f32x4*)(b + s * stride);
        }
        if (MODE == GL_FWD) gl_fwd_store<T>(p, m, n, cnt, s0, s1);
        else gl_put4((T*)p.out[pl] + m * p.ldo + n, s0, cnt);
    }
}
template <typename T, int MODE>
__global__ __launch_bounds__(256) void k_gated_join(GlArgs p, int planes) {
    gl_join<T, MODE>(p, planes, (int64_t)blockIdx.x * 256 + threadIdx.x, (int64_t)gridDim.x * 256);
}
// both backward products of one launch: the first `n_dx` workgroups dx, the others dW
template <typename T>
__global__ __launch_bounds__(256) void k_gated_join_both(GlArgs dx, GlArgs dw, int n_dx) {
    const int b = blockIdx.x;
    if (b < n_dx) gl_join<T, GL_DX>(dx, 1, (int64_t)b * 256 + threadIdx.x, (int64_t)n_dx * 256);
    else gl_join<T, GL_DW>(dw, 2, (int64_t)(b - n_dx) * 256 + threadIdx.x, (int64_t)(gridDim.x - n_dx) * 256);
}

// copies of up to three matrices whose rows are not 16-byte aligned: [rows][ldd], columns C..ldd - 1 zero
struct GlPack {
    struct { const void* src; void* dst; int64_t ld, rows; } m[3];
    int64_t ldd;
    int C, n;
};
template <typename T> __device__ __forceinline__ void gl_pack(const GlPack& p, int64_t b, int64_t blocks) {
    constexpr int E = 16 / sizeof(T);
    const int64_t per = p.ldd / E;
    const int64_t n0 = p.m[0].rows, n1 = n0 + p.m[1].rows, total = (n1 + p.m[2].rows) * per;
    for (int64_t t = b * 256 + threadIdx.x; t < total; t += blocks * 256) {
        int64_t r = t / per;
        const int64_t c = (t - r * per) * E;
        // (selections: a table that is indexed at run time would be copied to private memory first)
        const T* src = (const T*)(r < n0 ? p.m[0].src : r < n1 ? p.m[1].src : p.m[2].src);
        T* const dst = (T*)(r < n0 ? p.m[0].dst : r < n1 ? p.m[1].dst : p.m[2].dst);
        const int64_t ld = r < n0 ? p.m[0].ld : r < n1 ? p.m[1].ld : p.m[2].ld;
        r -= r < n0 ? 0 : r < n1 ? n0 : n1;
        src += r * ld + c;
        T v[E];
        if (c + E <= p.C) __builtin_memcpy(v, src, 16);
        else
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = c + e < p.C ? src[e] : (T)0;
        __builtin_memcpy(__builtin_assume_aligned(dst + r * p.ldd + c, 16), v, 16);
    }
}
template <typename T>
__global__ __launch_bounds__(256) void k_gated_pack(GlPack p) { gl_pack<T>(p, blockIdx.x, gridDim.x); }

// ---- backward, elementwise: du = dh act(g), dg = dh u act'(g), and their column sums ------------------------------------
// Bound by memory: 11 bytes per element in bf16 (5 of pre, 2 of dh, 4 of dg and du), 16384 x 8192 in 300 us = 4.9 TB/s.
// Block = tx column groups of 4 x (256 / tx) row lanes, `rows` rows; blocks behind the last row block make the copies that the
// products read (one launch for both: 1537 x 777 x 1203 in bf16, copies in a launch of their own, 5.8 us).  dgu: two planes [M][ldg] of TD, columns N..ldg - 1
// zero.  db: the column sums of the unrounded values: written here if one block has all rows, else left as partial sums
// colpart [row block][2][ldg] (gl_colsum).
struct GlDgu {
    const void* pre;
    const void* dh;
    void* dgu;
    float* colpart;
    void* db[2];
    int64_t lddh, ldg, M;
    int N, act, tx, rows, nblk;
};
template <typename T, typename TD>
__global__ __launch_bounds__(256) void k_gated_dgu(GlDgu p, GlPack pack) {
    __shared__ f32x4 red[2][256];
    if ((int)blockIdx.y >= p.nblk) {
        gl_pack<T>(pack, (int64_t)(blockIdx.y - p.nblk) * gridDim.x + blockIdx.x, (int64_t)(gridDim.y - p.nblk) * gridDim.x);
        return;
    }
    const int cx = threadIdx.x % p.tx, ry = threadIdx.x / p.tx, ty = 256 / p.tx;
    const int n = (blockIdx.x * p.tx + cx) * 4, cnt = p.N - n;
    const int64_t r0 = (int64_t)blockIdx.y * p.rows, r1 = r0 + p.rows < p.M ? r0 + p.rows : p.M;
    TD* const dgu = (TD*)p.dgu;
    f32x4 sg = {0.f, 0.f, 0.f, 0.f}, su = {0.f, 0.f, 0.f, 0.f};
    if (n < p.ldg) gl_with_act(p.act, [&](auto act) {
        // R rows at a time, all their loads before the first store (which could hit what is loaded, as far as the compiler knows)
        constexpr int R = 2;
        for (int64_t m0 = r0 + ry; m0 < r1; m0 += R * ty) {
            f32x4 g[R], u[R], d[R];
#pragma unroll
            for (int k = 0; k < R; ++k) {
                const int64_t m = m0 + k * ty;
                g[k] = u[k] = d[k] = (f32x4){0.f, 0.f, 0.f, 0.f};
                if (m < r1 && cnt > 0) {
                    GlPre<T>::get(p.pre, p.M, (p.N + 3) >> 2, m, n, g[k], u[k]);
                    d[k] = gl_get4((const T*)p.dh + m * p.lddh + n, cnt);
                }
            }
#pragma unroll
            for (int k = 0; k < R; ++k) {
                const int64_t m = m0 + k * ty;
                f32x4 dg = {0.f, 0.f, 0.f, 0.f}, du = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (e < cnt) {
                        float a, da;
                        gl_act_grad<T, decltype(act)::value>(g[k][e], a, da);
                        du[e] = d[k][e] * a;
                        dg[e] = d[k][e] * u[k][e] * da;
                    }
                if (m < r1) {
                    *(typename GlVec<TD>::V*)(dgu + m * p.ldg + n) = GlVec<TD>::put(dg);
                    *(typename GlVec<TD>::V*)(dgu + (p.M + m) * p.ldg + n) = GlVec<TD>::put(du);
                    sg += dg;
                    su += du;
                }
            }
        }
    });
    if (!p.db[0] && !p.db[1]) return;
    red[0][threadIdx.x] = sg;
    red[1][threadIdx.x] = su;
    __syncthreads();
    if (ry == 0 && n < p.ldg) {
        for (int k = 1; k < ty; ++k) {
            sg += red[0][k * p.tx + cx];
            su += red[1][k * p.tx + cx];
        }
        if (p.nblk == 1) {
            if (p.db[0] && cnt > 0) gl_put4((T*)p.db[0] + n, sg, cnt);
            if (p.db[1] && cnt > 0) gl_put4((T*)p.db[1] + n, su, cnt);
        } else {
            float* c = p.colpart + (int64_t)blockIdx.y * 2 * p.ldg + n;
            *(f32x4*)c = sg;
            *(f32x4*)(c + p.ldg) = su;
        }
    }
}

// db[n] = sum of the row blocks' partial sums: a workgroup has 64 columns (16 groups of 4) of one plane and THREADS / 16 lanes, lanes
// joined in order.  Workgroups [0, n) of it, the last ones of a launch of both products where there is one (2 to 5 us of a launch saved).
struct GlColsum {
    const float* colpart;
    void* db[2];
    int64_t ldg;
    int nblk, N, n;
};
template <typename T, int THREADS> __device__ __forceinline__ void gl_colsum(const GlColsum& p, int b, f32x4 (*red)[16]) {
    const int c = threadIdx.x & 15, y = threadIdx.x >> 4;
    const int n = (b >> 1) * 64 + c * 4, pl = b & 1, cnt = p.N - n;
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    if (cnt > 0)
#pragma unroll 8
        for (int k = y; k < p.nblk; k += THREADS / 16) s += *(const f32x4*)(p.colpart + ((int64_t)k * 2 + pl) * p.ldg + n);
    red[y][c] = s;
    __syncthreads();
    T* const out = (T*)p.db[pl];
    if (y == 0 && cnt > 0 && out) {
        for (int k = 1; k < THREADS / 16; ++k) s += red[k][c];
        gl_put4(out + n, s, cnt);
    }
}
template <typename T>
__global__ __launch_bounds__(256) void k_gated_colsum(GlColsum p) {
    __shared__ f32x4 red[16][16];
    gl_colsum<T, 256>(p, blockIdx.x, red);
}

// both backward products of a small layer, and the column sums
template <typename T>
__global__ __launch_bounds__(256) void k_gated_mm_both(GgArgs dx, GgArgs dw, GlColsum cs) {
    __shared__ __attribute__((aligned(16))) T smem[3 * GgShape<T>::PART];
    const int b = blockIdx.x;
    if (b < dx.wgs) gg_product<T, float, GL_DX>(dx, b, smem);
    else if (b < dx.wgs + dw.wgs) gg_product<T, float, GL_DW>(dw, b - dx.wgs, smem);
    else gl_colsum<T, 256>(cs, b - dx.wgs - dw.wgs, (f32x4(*)[16])smem);
}

template <typename T>
__global__ __launch_bounds__(256) void k_gated_zero(T* a, int64_t n) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) a[i] = (T)0;
}

}  // namespace dp
