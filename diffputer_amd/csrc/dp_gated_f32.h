// float32 tile products of the gated projection (dp_gated.h has the three products and their operands): T x T tile of products,
// 32 deep, 4 waves of T / 2 x T / 2 by v_mfma_f32_32x32x2_f32 (T = 128) or v_mfma_f32_16x16x4_f32 (T = 64): k-ordered chains
// of float32 fused multiply-adds.
//
// The float32 matrix pipe takes 64 cycles for 4096 products, 16 times the bf16 one: a K-tile of T = 128 is 4096 cycles of it
// per wave against 32 KiB of loads and 64 LDS reads, so one K-tile of loads in flight and one barrier per K-tile keep it
// fed, and two workgroups share a CU.  T = 64 is for products with too few tiles of 128 to fill the chip.  Operands go
// straight into LDS as in the bf16 tile kernels (rows that do not exist lie behind the buffer's end and arrive as zeros), 16
// bytes a lane where rows start on 16 bytes, else 4: element-wise loads are four times the instructions and still fit under
// the products.
//   Measured: T = 128 takes 3.8 us for a K-tile of two workgroups on every CU, 141 TFLOP/s of the pipe's 157 (a library product of
//   4096^3: 140, 8192^3: 153); both backward products of 8192 x 1024 x 4096 2.0 ms (136 TFLOP/s), of 4096 x 1024 x 2048 0.49 to
//   0.56 ms.  Results leave through LDS by whole rows: stores of 32 bytes a row wrote 212 MB to memory for 101 MB of results.
//   With G = 64 / (T / 4) lane groups of T / 4 lanes, a lane reads four k's of its row or column, the group's 4 (G g + group) ..
//   + 3: step s of the four multiplies the G k's 4 (G g + group) + s (both operands agree on that, and a sum over k does not
//   ask for more).
//   row layout (k contiguous): LDS rows of 128 bytes, 16-byte chunk c of row r at c ^ ((r >> 1) & 7), one ds_read_b128;
//   column layout: LDS holds k rows of 4 T bytes as they are in memory, four ds_read_b32; the bytes of k row k are stored with
//   their place xor'ed by T * ((k / 4) % G), so that the G k's of a read use all banks.
#pragma once
#include "dp_gated_lds.h"

namespace dp {

constexpr int GF_K = 32, GF_THREADS = 256;
template <int T> struct GfShape {
    static constexpr int TS = T / 4, G = 64 / TS;                // matrix tile, lane groups
    static constexpr int OP = T * GF_K * 4, LDS = 4 * OP;        // bytes of one operand's K-tile; two buffers
};
template <int TS> struct GfAcc;
template <> struct GfAcc<32> {
    typedef f32x16 V;
    static __device__ __forceinline__ V mul(float b, float a, V c) { return __builtin_amdgcn_mfma_f32_32x32x2f32(b, a, c, 0, 0, 0); }
};
template <> struct GfAcc<16> {
    typedef f32x4 V;
    static __device__ __forceinline__ V mul(float b, float a, V c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(b, a, c, 0, 0, 0); }
};

template <int MODE, int T, bool VEC>
__device__ __forceinline__ void gf_product(const GtArgs& q, int b, int count, char* smem) {
    using S = GfShape<T>;
    using Acc = GfAcc<S::TS>;
    constexpr bool A_ROW = MODE != GL_DW, B_ROW = MODE == GL_FWD;
    constexpr unsigned OUTSIDE = 0x80000000u;
    constexpr int TS = S::TS, G = S::G, OP = S::OP;
    constexpr int EL = VEC ? 16 : 4;                             // bytes per lane and load
    constexpr int NL = OP / (64 * EL) / 4;                       // loads per wave, operand and K-tile
    const GlArgs& p = q.g;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave >> 1, wn = wave & 1;
    const bool split = p.splits > 1;
    int slice, plane, ti, tj;
    gt_tile<MODE>(q, b, count, slice, plane, ti, tj);
    const int64_t i0 = (int64_t)ti * T;
    const int j0 = tj * (MODE == GL_FWD ? T / 2 : T);
    const int nk = (int)((p.C + GF_K - 1) / GF_K);
    const int kt0 = slice * p.kt_per, kt1 = min(kt0 + p.kt_per, nk * (MODE == GL_DX ? 2 : 1));

    // load `n` of a wave covers bytes (wave * NL + n) * 64 * EL .. of the operand's image; this lane's EL of them
    const int64_t lda = p.A[MODE == GL_DW ? plane : 0].ld * 4, ldb = p.B[0].ld * 4;
    unsigned va[NL], vb[NL];
    bool tail_out[NL];                                           // row layout: past the end in the last K-tile
    const int left = (int)(p.C - (int64_t)(nk - 1) * GF_K);      // k's of a segment's last K-tile
#pragma unroll
    for (int n = 0; n < NL; ++n) {
        const int byte = (wave * NL + n) * 64 * EL + lane * EL;
        const int r = byte >> 7, in_r = (((byte >> 4) & 7) ^ ((r >> 1) & 7)) * 16 + (byte & 15);      // row layout: row, byte within the row
        const int k = byte / (4 * T), in_k = (byte % (4 * T)) ^ (((k >> 2) & (G - 1)) * T);    // column layout: k, byte within the k row
        va[n] = A_ROW ? (unsigned)(r * lda + in_r) : (unsigned)(k * lda + in_k);
        vb[n] = B_ROW ? (unsigned)((r & (MODE == GL_FWD ? T / 2 - 1 : T - 1)) * ldb + in_r) : (unsigned)(k * ldb + in_k);
        tail_out[n] = in_r / 4 >= left;
    }
    auto stage = [&](int kt) {
        const int seg = MODE == GL_DX && kt >= nk ? 1 : 0;
        const int64_t kk = kt - seg * nk;
        const bool last = kk == nk - 1;
        char* const dst = smem + ((kt - kt0) & 1) * 2 * OP + wave * NL * 64 * EL;
        {
            const GlOp& op = p.A[MODE == GL_DX ? seg : MODE == GL_DW ? plane : 0];
            const char* const base = (const char*)op.p;
            const auto buf = gt_buffer(base + (A_ROW ? i0 * lda + kk * (GF_K * 4) : kk * GF_K * lda + i0 * 4), base + (A_ROW ? p.I - 1 : p.C - 1) * lda + op.cols * 4);
#pragma unroll
            for (int n = 0; n < NL; ++n)
                gt_load<EL>(buf, dst + n * 64 * EL, A_ROW && last && tail_out[n] ? OUTSIDE : va[n]);
        }
        // FWD: waves 0 and 1 load gate rows, waves 2 and 3 up rows
        const GlOp& op = p.B[MODE == GL_FWD ? wave >> 1 : MODE == GL_DX ? seg : 0];
        const char* const base = (const char*)op.p;
        const auto buf = gt_buffer(base + (B_ROW ? j0 * ldb + kk * (GF_K * 4) : kk * GF_K * ldb + (int64_t)j0 * 4), base + (B_ROW ? p.J - 1 : p.C - 1) * ldb + op.cols * 4);
#pragma unroll
        for (int n = 0; n < NL; ++n)
            gt_load<EL>(buf, dst + OP + n * 64 * EL, B_ROW && last && tail_out[n] ? OUTSIDE : vb[n]);
    };

    const int r = lane % TS, grp = lane / TS;
    typename Acc::V acc[2][2];                                   // [rows wm * T / 2 + TS i][columns b * T / 2 + wn * TS]
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int e = 0; e < TS * TS / 64; ++e) acc[i][h][e] = 0.f;

    stage(kt0);
    GT_VMCNT(0);
    __builtin_amdgcn_s_barrier();
#pragma clang loop unroll(disable)
    for (int kt = kt0; kt < kt1; ++kt) {
        const char* const sa = smem + ((kt - kt0) & 1) * 2 * OP;
        const char* const sb = sa + OP;
        if (kt + 1 < kt1) stage(kt + 1);
#pragma unroll
        for (int g = 0; g < GF_K / (4 * G); ++g) {
            f32x4 av[2], bv[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int ra = wm * (T / 2) + i * TS + r, rb = i * (T / 2) + wn * TS + r;
                if (A_ROW) av[i] = *(const f32x4*)(sa + ra * 128 + (((G * g + grp) ^ ((r >> 1) & 7)) << 4));
                else
#pragma unroll
                    for (int s = 0; s < 4; ++s) av[i][s] = *(const float*)(sa + (4 * (G * g + grp) + s) * (4 * T) + ((ra * 4) ^ (grp * T)));
                if (B_ROW) bv[i] = *(const f32x4*)(sb + rb * 128 + (((G * g + grp) ^ ((r >> 1) & 7)) << 4));
                else
#pragma unroll
                    for (int s = 0; s < 4; ++s) bv[i][s] = *(const float*)(sb + (4 * (G * g + grp) + s) * (4 * T) + ((rb * 4) ^ (grp * T)));
            }
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int h = 0; h < 2; ++h) acc[i][h] = Acc::mul(bv[h][s], av[i][s], acc[i][h]);
        }
        GL_SYNC(0);                                              // the next tile is there, and this one's slot has been read by every wave
    }

    // A lane holds row r, columns 8 e + 4 grp + 0..3 of each TS x TS tile: 32 bytes of a row side by side.  The tiles go through the wave's
    // own part of LDS and leave by whole rows of 4 TS bytes.
    constexpr int ROWB = TS * 4 + 16, LPR = TS / 4, RP = 64 / LPR;         // bytes of a row there; lanes of a row; rows at a time
    static_assert(4 * 2 * TS * ROWB <= S::LDS, "the tiles of all waves fit");
    char* const mine = smem + wave * 2 * TS * ROWB;
    float* const out = (float*)p.out[MODE == GL_DW ? plane : 0];
    const int cl = wn * TS + lane % LPR * 4;
    f32x4 bg, bu;
    if (MODE == GL_FWD && !split && j0 + cl < p.J) gl_bias<float>(p, j0 + cl, p.J - j0 - cl, bg, bu);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int e = 0; e < TS * TS / 256; ++e)
                *(f32x4*)(mine + (h * TS + r) * ROWB + (8 * e + 4 * grp) * 4) = (f32x4){acc[i][h][4 * e], acc[i][h][4 * e + 1], acc[i][h][4 * e + 2], acc[i][h][4 * e + 3]};
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
#pragma unroll
        for (int k = 0; k < TS / RP; ++k) {
            const int row = k * RP + lane / LPR;
            const int64_t m = i0 + wm * (T / 2) + i * TS + row;
            f32x4 v[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) v[h] = *(const f32x4*)(mine + (h * TS + row) * ROWB + lane % LPR * 16);
            if (m >= p.I) continue;
            if (MODE == GL_FWD && !split) {
                if (j0 + cl < p.J)
                    gl_with_act(p.act, [&](auto act) { gl_fwd_put<float, decltype(act)::value>(p, m, j0 + cl, p.J - j0 - cl, v[0] + bg, v[1] + bu); });
                continue;
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int n = j0 + (MODE == GL_FWD ? 0 : h * (T / 2)) + cl, pl = MODE == GL_FWD ? h : plane;
                if (n >= p.J) continue;
                if (split) *(f32x4*)(p.part + (((int64_t)slice * 2 + pl) * p.I + m) * p.ldp + n) = v[h];
                else gl_put4(out + m * p.ldo + n, v[h], p.J - n);
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
}

template <int MODE, int T, bool VEC>
__global__ __launch_bounds__(GF_THREADS) void k_gated_f32(GtArgs q) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    gf_product<MODE, T, VEC>(q, blockIdx.x, gridDim.x, smem);
}
template <int T, bool VEC>
__global__ __launch_bounds__(GF_THREADS) void k_gated_f32_both(GtArgs dx, GtArgs dw, int n0, int dx_first, GlColsum cs) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int b = blockIdx.x, all = gridDim.x - cs.n, first = b < n0, at = first ? b : b - n0, count = first ? n0 : all - n0;
    if (b >= all) return gl_colsum<float, GF_THREADS>(cs, b - all, (f32x4(*)[16])smem);
    if (first == dx_first) gf_product<GL_DX, T, VEC>(dx, at, count, smem);
    else gf_product<GL_DW, T, VEC>(dw, at, count, smem);
}

}  // namespace dp
