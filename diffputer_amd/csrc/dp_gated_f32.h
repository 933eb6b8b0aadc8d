// float32 tile products of the gated projection (dp_gated.h has the three products and their operands): 128 x 128 tile of
// products, 32 deep, 4 waves of 64 x 64, v_mfma_f32_32x32x2_f32 (a k-ordered chain of float32 fused multiply-adds).
//
// The float32 matrix pipe takes 64 cycles for 4096 products, 16 times the bf16 one: a K-tile is 4096 cycles of it per wave
// against 32 KiB of loads and 64 LDS reads, so one K-tile of loads in flight and one barrier per K-tile keep it fed, and two
// workgroups share a CU.  Operands go straight into LDS as in the bf16 tile kernels (rows that do not exist lie behind the
// buffer's end and arrive as zeros), 16 bytes a lane where rows start on 16 bytes, else 4: element-wise loads are four times
// the instructions and still fit under the products.
//   row layout (k contiguous): LDS rows of 128 bytes, 16-byte chunk c of row r at c ^ (r & 7); a lane reads four k's of its
//     row at once, lanes 0..31 the k's 8 q .. 8 q + 3 and lanes 32..63 the next four: step s of the four multiplies the
//     k's 8 q + s and 8 q + 4 + s (both operands agree on that, and a sum over k does not ask for more).
//   column layout: LDS holds k rows of 512 bytes as they are in memory, a lane reads one k of its column; rows with
//     (k & 4) are stored with the two 128-byte parts of every 256 swapped, so that the two k's of a read use all banks.
#pragma once
#include "dp_gated_tile.h"

namespace dp {

constexpr int GF_T = 128, GF_K = 32, GF_THREADS = 256;
constexpr int GF_OP = GF_T * GF_K * 4;                           // bytes of one operand's K-tile
constexpr int GF_LDS = 4 * GF_OP;

template <int MODE, bool VEC, bool SPLIT>
__global__ __launch_bounds__(GF_THREADS) void k_gated_f32(GtArgs q) {
    constexpr bool A_ROW = MODE != GL_DW, B_ROW = MODE == GL_FWD;
    constexpr unsigned OUTSIDE = 0x80000000u;
    constexpr int EL = VEC ? 16 : 4;                             // bytes per lane and load
    constexpr int NL = GF_OP / (64 * EL) / 4;                    // loads per wave, operand and K-tile
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const GlArgs& p = q.g;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave >> 1, wn = wave & 1;
    int slice;
    const int tile = gt_slice<SPLIT>(p, slice);
    int plane, ti, tj;
    gt_tile<MODE>(q, tile, plane, ti, tj);
    const int64_t i0 = (int64_t)ti * GF_T;
    const int j0 = tj * (MODE == GL_FWD ? GF_T / 2 : GF_T);
    const int nk = (int)((p.C + GF_K - 1) / GF_K);
    const int all = nk * (MODE == GL_DX ? 2 : 1);
    const int kt0 = SPLIT ? slice * p.kt_per : 0, kt1 = SPLIT ? min(kt0 + p.kt_per, all) : all;

    // load `n` of a wave covers bytes (wave * NL + n) * 64 * EL .. of the operand's image; this lane's EL of them
    const int64_t lda = p.A[MODE == GL_DW ? plane : 0].ld * 4, ldb = p.B[0].ld * 4;
    unsigned va[NL], vb[NL];
    bool tail_out[NL];                                           // row layout: past the end in the last K-tile
    const int left = (int)(p.C - (int64_t)(nk - 1) * GF_K);      // k's of a segment's last K-tile
#pragma unroll
    for (int n = 0; n < NL; ++n) {
        const int byte = (wave * NL + n) * 64 * EL + lane * EL;
        const int r = byte >> 7, in_r = (((byte >> 4) & 7) ^ (r & 7)) * 16 + (byte & 15);      // row layout: row, byte within the row
        const int k = byte >> 9, in_k = (byte & 511) ^ (((k >> 2) & 1) << 7);                  // column layout: k, byte within the k row
        // FWD: rows 0..63 of the B image are gate rows, 64..127 up rows: handled by base and row below
        va[n] = A_ROW ? (unsigned)(r * lda + in_r) : (unsigned)(k * lda + in_k);
        vb[n] = B_ROW ? (unsigned)((r & (MODE == GL_FWD ? 63 : 127)) * ldb + in_r) : (unsigned)(k * ldb + in_k);
        tail_out[n] = in_r / 4 >= left;
    }
    auto stage = [&](int kt) {
        const int seg = MODE == GL_DX && kt >= nk ? 1 : 0;
        const int64_t kk = kt - seg * nk;
        const bool last = kk == nk - 1;
        char* const dst = smem + ((kt - kt0) & 1) * 2 * GF_OP + wave * NL * 64 * EL;
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
            gt_load<EL>(buf, dst + GF_OP + n * 64 * EL, B_ROW && last && tail_out[n] ? OUTSIDE : vb[n]);
    };

    const int r32 = lane & 31, half = lane >> 5;
    f32x16 acc[2][2];                                            // [rows wm * 64 + 32 i][columns 64 b + wn * 32]
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][b][e] = 0.f;

    stage(kt0);
    GT_VMCNT(0);
    __builtin_amdgcn_s_barrier();
#pragma clang loop unroll(disable)
    for (int kt = kt0; kt < kt1; ++kt) {
        const char* const sa = smem + ((kt - kt0) & 1) * 2 * GF_OP;
        const char* const sb = sa + GF_OP;
        if (kt + 1 < kt1) stage(kt + 1);
#pragma unroll
        for (int g = 0; g < GF_K / 8; ++g) {
            f32x4 a[2], b[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (A_ROW) a[i] = *(const f32x4*)(sa + (wm * 64 + i * 32 + r32) * 128 + (((2 * g + half) ^ (r32 & 7)) << 4));
                else
#pragma unroll
                    for (int s = 0; s < 4; ++s) a[i][s] = *(const float*)(sa + (8 * g + 4 * half + s) * 512 + (((wm * 64 + i * 32 + r32) * 4) ^ (half << 7)));
                if (B_ROW) b[i] = *(const f32x4*)(sb + (i * 64 + wn * 32 + r32) * 128 + (((2 * g + half) ^ (r32 & 7)) << 4));
                else
#pragma unroll
                    for (int s = 0; s < 4; ++s) b[i][s] = *(const float*)(sb + (8 * g + 4 * half + s) * 512 + (((i * 64 + wn * 32 + r32) * 4) ^ (half << 7)));
            }
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(b[j][s], a[i][s], acc[i][j], 0, 0, 0);
        }
        GT_VMCNT(0);
        __builtin_amdgcn_s_barrier();
    }

    // lane: row (lane & 31), columns 8 e + 4 half + 0..3 of each 32 x 32 tile
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int64_t m = i0 + wm * 64 + i * 32 + r32;
        if (m >= p.I) continue;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int cl = wn * 32 + 8 * e + 4 * half;
            if (MODE == GL_FWD && !SPLIT) {
                const int n = j0 + cl, cnt = p.J - n < 4 ? p.J - n : 4;
                const float g[4] = {acc[i][0][4 * e], acc[i][0][4 * e + 1], acc[i][0][4 * e + 2], acc[i][0][4 * e + 3]};
                const float u[4] = {acc[i][1][4 * e], acc[i][1][4 * e + 1], acc[i][1][4 * e + 2], acc[i][1][4 * e + 3]};
                if (cnt > 0) gl_fwd_store<float>(p, m, n, cnt, g, u);
                continue;
            }
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const int n = j0 + (MODE == GL_FWD ? 0 : b * 64) + cl, pl = MODE == GL_FWD ? b : plane;
                if (n >= p.J) continue;
                const f32x4 v = {acc[i][b][4 * e], acc[i][b][4 * e + 1], acc[i][b][4 * e + 2], acc[i][b][4 * e + 3]};
                if (SPLIT) {
                    *(f32x4*)(p.part + (((int64_t)slice * 2 + pl) * p.I + m) * p.ldp + n) = v;
                } else {
                    float* const o = (float*)p.out[MODE == GL_DW ? plane : 0] + m * p.ldo + n;
                    if ((p.ldo & 3) == 0 && ((uintptr_t)o & 15) == 0 && n + 4 <= p.J) *(f32x4*)o = v;
                    else
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (n + r < p.J) o[r] = v[r];
                }
            }
        }
    }
}

}  // namespace dp
