// bf16 products of the gated projection in 128 x 128 tiles (dp_gated.h has the three products and their operands): 4 waves of
// 64 x 64, K-steps of 32 in a ring of five LDS slots, two workgroups per CU.
//
// Made for products with fewer than 256 tiles of 256 x 256, and taken wherever the host's estimate says it is faster (whole rounds
// of 256 tiles that end badly, layers narrower than such a tile).  With one or two workgroups on a CU it is bound by the latency of a
// K-step, not by the matrix pipes: nothing of a step waits for itself.  While a step's products run, the fragments of the next one are read into a second set of registers
// and the loads of the step five ahead go out, interleaved with the products; the only waits are one per step, for loads
// that went out four steps before and for reads whose latency the products have covered, and one barrier.  64 k's take 0.46 us
// with one workgroup on a CU in four (the four-phase schedule of the 256 x 256 kernel at this tile: 0.92), 0.55 with one on
// each (1.02), 1.16 with two on each (1.20).  There the tiles' way into LDS is the bound: 64 KiB per 64 k's and pair of
// workgroups, 1024 cycles at 64 bytes each, as long as the products; with loads of no bytes the same steps take 0.73.  Both backward products of 4096 x 1024 x 2048, 512
// workgroups: 68 us (1 010 TFLOP/s).
//   step s:   { load step s + 5 into the slot of step s ; read fragments of s + 1 ; products of s ; wait ; barrier }
//   RAW  step s + 1 was loaded in step s - 4 and waited for (all but the three newest steps' loads) at the end of step s - 1;
//   WAR  the slot of step s was read in step s - 1, whose end every wave has passed with its reads done.
// Steps past the end are "loaded" with no bytes (zeros, no traffic): every count holds for any number of steps.
// Masking as in the 256 x 256 kernel: what does not exist lies behind the buffer's end, or is asked for there.
// GL_FWD: the first 64 B rows are gate rows, the others the up rows of the same columns: one lane ends with g and u of the same
// elements.
#pragma once
#include "dp_gated_lds.h"

namespace dp {

constexpr int GS_T = 128, GS_THREADS = 256;
constexpr int GS_NB = 5, GS_STEP = GS_T * 128, GS_LDS = GS_NB * GS_STEP;   // ring slots; bytes of a slot (A, then B)
constexpr int GS_MI = GS_T / 32, GS_NJ = GS_T / 64, GS_NP = GS_T / 64;     // m-tiles; n-tiles of a half; loads of a wave, operand and step

template <int MODE>
__device__ __forceinline__ void gs_product(const GtArgs& q, int b, int count, char* smem) {
    constexpr bool A_ROW = MODE != GL_DW, B_ROW = MODE == GL_FWD;
    constexpr int T = GS_T, NB = GS_NB, STEP = GS_STEP, MI = GS_MI, NJ = GS_NJ, NP = GS_NP, NI = 2 * NP;
    constexpr unsigned OUTSIDE = 0x80000000u;
    const GlArgs& p = q.g;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave >> 1, wn = wave & 1;
    const bool split = p.splits > 1;
    int slice, plane, ti, tj;
    gt_tile<MODE>(q, b, count, slice, plane, ti, tj);
    const int64_t i0 = (int64_t)ti * T;
    const int j0 = tj * (MODE == GL_FWD ? T / 2 : T);
    const int nk = (int)((p.C + 31) >> 5);                                 // K-steps of a segment
    const int kt0 = slice * p.kt_per, kt1 = min(kt0 + p.kt_per, nk * (MODE == GL_DX ? 2 : 1));

    // ---- loads: a wave moves pieces wave, wave + 4, .. (1 KiB) of each operand's T x 32 image ----
    //   row layout: piece = 16 rows x 64 B, 16-byte chunk c of row r at c ^ turn(r / 4 % 4)
    //   column layout: k rows of 2 T bytes, piece = 512 / T of them, 32-byte slot s of k row k at s ^ g(k)
    const int64_t lda = p.A[MODE == GL_DW ? plane : 0].ld * 2, ldb = p.B[0].ld * 2;            // bytes
    constexpr int KR = 512 / T, CH = T / 8;                                // k rows of a piece, 16-byte chunks of a k row
    auto g_of = [](int k) { return (k & 3) | ((k >> 3) & 1) << 2; };
    // ds_read_b128 takes lanes 0-3, 12-15, 20-23 and 24-27 at a time (and 4-7, 8-11, 16-19, 28-31; the upper half alike): with 0, 2, 3, 1 their
    // 16 chunks lie in 16 places, with 0, 1, 2, 3 in 8
    auto turn = [](int x) { return ((x ^ x >> 1) & 1) << 1 | x >> 1; };
    const int r16 = lane >> 2, c4 = (lane & 3) ^ turn(lane >> 4);
    unsigned va[NP], vb[NP];
#pragma unroll
    for (int s = 0; s < NP; ++s) {
        const int piece = wave + s * 4;
        const int k = piece * KR + lane / CH, c = (lane % CH) ^ (2 * g_of(k));
        const int rb = MODE == GL_FWD ? (piece * 16 + r16) & (T / 2 - 1) : piece * 16 + r16;   // FWD: row within the gate's or the up's half
        va[s] = A_ROW ? (unsigned)((piece * 16 + r16) * lda + c4 * 16) : (unsigned)(k * lda + c * 16);
        vb[s] = B_ROW ? (unsigned)(rb * ldb + c4 * 16) : (unsigned)(k * ldb + c * 16);
    }
    const bool tail_out = B_ROW && (p.C & 31) && c4 * 8 >= (int)(p.C & 31);                    // chunks past the contraction's end, last K-step

    // A stream walks an operand K-step by K-step.  Row layout: rows that do not exist lie behind `full` bytes whatever the step.
    // Column layout: a step has 32 k rows, the segment's last one `last` bytes.
    struct Stream { u32x4 at; unsigned full, last; };
    auto open = [&](const GlOp& op, bool row, int64_t first, int64_t size, int64_t kk) {
        const int64_t ld = op.ld * 2;
        Stream st;
        st.at = gl_buffer((const char*)op.p + (row ? first * ld + kk * 64 : kk * 32 * ld + first * 2));
        st.full = gl_clip(row ? (size - 1 - first) * ld + op.cols * 2 : 31 * ld + (op.cols - first) * 2);
        st.last = row ? st.full : gl_clip((p.C - 1 - (int64_t)(nk - 1) * 32) * ld + (op.cols - first) * 2);
        return st;
    };
    auto seg_of = [&](int kt) { return MODE == GL_DX && kt >= nk ? 1 : 0; };
    auto open_a = [&](int kt) { return open(p.A[MODE == GL_DX ? seg_of(kt) : MODE == GL_DW ? plane : 0], A_ROW, i0, p.I, kt - seg_of(kt) * nk); };
    auto open_b = [&](int kt, int half) { return open(p.B[MODE == GL_FWD ? half : seg_of(kt)], B_ROW, j0, p.J, kt - seg_of(kt) * nk); };
    Stream sa = open_a(kt0), sb = open_b(kt0, 0), su = sb;
    if (MODE == GL_FWD) su = open_b(kt0, 1);
    const int64_t step_a = A_ROW ? 64 : 32 * lda, step_b = B_ROW ? 64 : 32 * ldb;
    int skt = kt0;                                                         // next K-step to load
    unsigned slot_in = gt_lds(smem);                                       // its slot
    const unsigned lds0 = slot_in;
    bool s_tail;
    auto stage_begin = [&]() {
        const int kk = skt - seg_of(skt) * nk;
        const bool live = skt < kt1, last = kk == nk - 1;
        sa.at[2] = !live ? 0u : last ? sa.last : sa.full;
        sb.at[2] = !live ? 0u : last ? sb.last : sb.full;
        if (MODE == GL_FWD) su.at[2] = !live ? 0u : su.full;
        s_tail = last;
    };
    auto stage_one = [&](int i) {                                          // load i of NI
        const bool is_b = i >= NP;
        const int s = is_b ? i - NP : i;
        unsigned vo = is_b ? vb[s] : va[s];
        if (B_ROW && s_tail && tail_out) vo = OUTSIDE;
        const unsigned dst = slot_in + (is_b ? STEP / 2 : 0) + (wave + s * 4) * 1024;
        if (!is_b) gl_load_lds(sa.at, vo, dst);
        else if (MODE == GL_FWD && s >= NP / 2) gl_load_lds(su.at, vo, dst);
        else gl_load_lds(sb.at, vo, dst);
    };
    auto stage_end = [&]() {
        ++skt;
        gl_advance(sa.at, step_a);
        gl_advance(sb.at, step_b);
        if (MODE == GL_FWD) gl_advance(su.at, step_b);
        if (MODE == GL_DX && __builtin_expect(skt == nk, 0)) {
            asm volatile("");                                              // a branch, not a selection computed every time
            sa = open_a(skt);
            sb = open_b(skt, 0);
        }
        slot_in += STEP;
        if (slot_in == lds0 + NB * STEP) slot_in = lds0;
    };

    // ---- fragment reads: an LDS byte address (column layout: the tile's number is xor'ed into the slot bits), and constant offsets ----
    const unsigned foff = (lane & 15) * 64 + (((lane >> 4) ^ turn((lane >> 2) & 3)) << 4);
    const int krow = (lane >> 4) * 8 + ((lane >> 2) & 3);
    const unsigned fc = krow * T * 2 + (g_of(krow) << 5) + (lane & 3) * 8;
    const unsigned fa = A_ROW ? foff + wm * MI * 1024 : fc ^ (wm * MI << 5), fb = B_ROW ? foff + wn * NJ * 1024 : fc ^ (wn * NJ << 5);
    typedef const DP_LDS_AS char* LdsAt;
    auto frag = [&](bool row, unsigned at, int off, int t) {
        if (row) return *(const DP_LDS_AS bf16x8*)((LdsAt)(uintptr_t)at + (off + t * 1024));
        const LdsAt c = (LdsAt)(uintptr_t)(at ^ (t << 5)) + off;
        const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((DP_LDS_AS bf16x4*)c), hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((DP_LDS_AS bf16x4*)(c + 4 * T * 2));
        return (bf16x8)__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    struct Frags { bf16x8 a[MI], b[2 * NJ]; };
    unsigned slot_out = lds0;                                              // slot of the K-step to read next
    auto read_one = [&](Frags& f, int n) {                                 // fragment n of MI + 2 NJ
        if (n < MI) f.a[n] = frag(A_ROW, slot_out + fa, 0, n);
        else {
            const int j = n - MI;
            f.b[j] = frag(B_ROW, slot_out + fb, STEP / 2, (j / NJ) * (T / 32) + j % NJ);
        }
    };
    auto read_end = [&]() {
        slot_out += STEP;
        if (slot_out == lds0 + NB * STEP) slot_out = lds0;
    };

    f32x4 acc[MI][2 * NJ];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < 2 * NJ; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};

    // one K-step: in NI groups, a load of the step NB ahead, fragments of the next step, products of this one
    auto step = [&](const Frags& cur, Frags& next) {
        stage_begin();
#pragma unroll
        for (int g = 0; g < NI; ++g) {
            stage_one(g);
#pragma unroll
            for (int n = g * (MI + 2 * NJ) / NI; n < (g + 1) * (MI + 2 * NJ) / NI; ++n) read_one(next, n);
#pragma unroll
            for (int m = g * MI * 2 * NJ / NI; m < (g + 1) * MI * 2 * NJ / NI; ++m)
                acc[m / (2 * NJ)][m % (2 * NJ)] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(cur.b[m % (2 * NJ)], cur.a[m / (2 * NJ)], acc[m / (2 * NJ)][m % (2 * NJ)], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
        stage_end();
        read_end();
        GL_SYNC((NB - 2) * NI);
    };
    Frags f0, f1;
#pragma unroll
    for (int s = 0; s < NB; ++s) {
        stage_begin();
#pragma unroll
        for (int g = 0; g < NI; ++g) stage_one(g);
        stage_end();
    }
    GL_SYNC((NB - 1) * NI);
#pragma unroll
    for (int n = 0; n < MI + 2 * NJ; ++n) read_one(f0, n);
    read_end();
    GL_SYNC((NB - 2) * NI);
    int kt = kt0;
#pragma clang loop unroll(disable)
    for (; kt + 1 < kt1; kt += 2) {
        step(f0, f1);
        step(f1, f0);
    }
    if (kt < kt1) step(f0, f1);
    GT_VMCNT(0);                                                           // nothing may land in LDS behind the workgroup's end

    // ---- epilogue: lane holds row (lane & 15), columns 4 (lane >> 4) + 0..3 of each 16 x 16 tile ----
    const int cl = wn * NJ * 16 + (lane >> 4) * 4;
    const int64_t mrow = i0 + wm * (T / 2) + (lane & 15);
    if (split) {
#pragma unroll
        for (int i = 0; i < MI; ++i) {
            const int64_t m = mrow + i * 16;
            if (m >= p.I) continue;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    const int n = j0 + (MODE == GL_FWD ? 0 : h * (T / 2)) + cl + j * 16, pl = MODE == GL_FWD ? h : plane;
                    // ldp is a multiple of 4: four columns that start inside a row end inside its padding
                    if (n < p.J) *(f32x4*)(p.part + (((int64_t)slice * 2 + pl) * p.I + m) * p.ldp + n) = acc[i][h * NJ + j];
                }
        }
    } else if constexpr (MODE == GL_FWD) {
        static_assert(NJ == 2, "two tiles side by side");
        const int n = j0 + cl;
        if (n < p.J) gl_with_act(p.act, [&](auto act) {
            f32x4 bg[2], bu[2];
            gl_bias<bf16_t>(p, n, p.J - n, bg[0], bu[0]);
            gl_bias<bf16_t>(p, n + 16, p.J - n - 16, bg[1], bu[1]);
#pragma unroll
            for (int i = 0; i < MI; ++i) {
                const int64_t m = mrow + i * 16;
                const f32x4 g[2] = {acc[i][0] + bg[0], acc[i][1] + bg[1]}, u[2] = {acc[i][NJ] + bu[0], acc[i][NJ + 1] + bu[1]};
                if (m < p.I) gl_fwd_put2<decltype(act)::value>(p, m, n, g, u);
            }
        });
    } else {
        bf16_t* const out = (bf16_t*)p.out[MODE == GL_DW ? plane : 0];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const int n = j0 + h * (T / 2) + cl + j * 16, cnt = p.J - n;
                if (cnt <= 0) continue;
#pragma unroll
                for (int i = 0; i < MI; ++i) {
                    const int64_t m = mrow + i * 16;
                    if (m < p.I) gl_put4(out + m * p.ldo + n, acc[i][h * NJ + j], cnt);
                }
            }
    }
}

template <int MODE>
__global__ __launch_bounds__(GS_THREADS, 2) void k_gated_ring(GtArgs q) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    gs_product<MODE>(q, blockIdx.x, gridDim.x, smem);
}
// both backward products in one launch, the longer contraction first: workgroups [0, n0) the one, then the
// other, then the column sums
__global__ __launch_bounds__(GS_THREADS, 2) static void k_gated_ring_both(GtArgs dx, GtArgs dw, int n0, int dx_first, GlColsum cs) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int b = blockIdx.x, all = gridDim.x - cs.n, first = b < n0, at = first ? b : b - n0, count = first ? n0 : all - n0;
    if (b >= all) return gl_colsum<bf16_t, GS_THREADS>(cs, b - all, (f32x4(*)[16])smem);
    if (first == dx_first) gs_product<GL_DX>(dx, at, count, smem);
    else gs_product<GL_DW>(dw, at, count, smem);
}

}  // namespace dp
