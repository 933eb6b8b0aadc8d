// bf16 products of the gated projection that fill the chip with 256 x 256 tiles (dp_gated.h has the three products and their
// operands): 64 deep, 8 waves of 128 x 64, one workgroup per CU.
//
//   * A K-tile is four half-tiles in LDS, A0 A1 B0 B1 (128 rows of A or of B, 64 deep), two K-tiles deep.  Each half-tile
//     is loaded straight into LDS (buffer loads, 16 bytes a lane) 5 to 6 phases before it is read, and the loads stay in
//     flight across barriers (counted vmcnt).  Rows or k's that do not exist lie behind the buffer's last byte: the range
//     check returns zeros for them, which is all the masking that ragged sizes need.
//   * A K-tile is four phases, one quadrant (A half x B half) of matrix instructions each:
//       phase   LDS reads                 loads issued         quadrant    landed after the phase's vmcnt
//       c0      B0(t), A0(t)              -                    A0 B0       -
//       c1      -                         A1(t+1), B1(t+2)     A0 B1       A1(t)
//       c2      A1(t)                     A0(t+2)              A1 B1       B1(t+1)
//       c3      B1(t+1)                   B0(t+2)              A1 B0       A0(t+1), B0(t+1)
//     A half-tile is read after the vmcnt of every wave and a barrier; its slot is loaded again at least two phases after
//     its last read, whose lgkmcnt(0) every wave has passed by then.  K-tiles past the end are "loaded" from an empty
//     buffer (zeros, no traffic), so that every count holds for any number of K-tiles.
//   * The waves of the lower half run one barrier behind, so that one wave of a SIMD multiplies while its partner reads LDS.
//   * Row layout (k contiguous): LDS rows of 128 bytes, 16-byte chunk c of row r at c ^ (r & 7); fragments by
//     ds_read_b128.  Column layout (a transposed product's operand): LDS holds the k rows as they are in memory, and
//     ds_read_b64_tr_b16 turns 4 k's x 16 columns into a fragment's k order while reading, 32-byte slot s of k row k at
//     s ^ g(k), with g spread so that the 8 rows of a half wave's read lie in 8 different slots.
//   * Bound by the matrix pipes, and on a full chip by the power that they may draw: a K-tile takes 1.07 us with 64 workgroups
//     and 1.36 with 256, 0.85 being the pipes' own time at 2.4 GHz.  256 tiles of K = 4096 take 98 us (1 403 TFLOP/s; a
//     library product of 8192^3 reaches 1 404), both backward products of 16384 x 4096 x 8192 3.1 ms (1 420 TFLOP/s), the
//     forward product there 1.75 ms (1 260) with h and the projections for the backward pass, 0.94 GB, written beside it.
//   * Why 128 x 64 per wave: 24 fragments are read from LDS for 64 matrix instructions, three quarters of what LDS delivers
//     meanwhile (64 x 64 per wave: all of it).  128 x 128 per wave (4 waves, accumulators in AGPRs) has the same K-loop and
//     takes 16.5 us beyond it instead of 11.
//   * GL_FWD: B0 are the gate's rows and B1 the up's rows for the same columns of h: one lane ends with g and u of the
//     same elements, and the activation and the product are lane-local.
#pragma once
#include "dp_gated_lds.h"

namespace dp {

constexpr int GT_T = 256, GT_THREADS = 512;
constexpr int GT_NW = 8, GT_WN = 4;                                        // waves; waves along the columns (2 along the rows)
constexpr int GT_HR = GT_T / 2, GT_HB = GT_HR * 128;                       // rows and bytes of a half-tile
constexpr int GT_MI = GT_HR / 32, GT_NJ = GT_HR / GT_WN / 16;              // 16 x 16 tiles of a wave's quadrant
constexpr int GT_LDS = 8 * GT_HB;

// tiles (and slices) b, b + step, .. of the product, neighbouring ones on one XCD; returns how far behind its end the walk is
template <int MODE>
__device__ __forceinline__ int gt_product(const GtArgs& q, int b, int step, char* smem) {
    constexpr bool A_ROW = MODE != GL_DW, B_ROW = MODE == GL_FWD;
    constexpr int HR = GT_HR, HB = GT_HB, MI = GT_MI, NJ = GT_NJ, NW = GT_NW, WN = GT_WN;
    constexpr unsigned OUTSIDE = 0x80000000u;                              // an offset behind every buffer
    const GlArgs& p = q.g;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / WN, wn = wave % WN;

    const bool split = p.splits > 1;
    const int nk = (int)((p.C + 63) >> 6);                                 // K-tiles of a segment
    struct Tile { int slice, plane, j0, kt0, kt1; int64_t i0; };
    auto locate = [&](int at) {
        Tile t;
        int ti, tj;
        gt_tile<MODE>(q, at, q.wgs, t.slice, t.plane, ti, tj);
        t.i0 = (int64_t)ti * GT_T;
        t.j0 = tj * (MODE == GL_FWD ? HR : GT_T);
        t.kt0 = t.slice * p.kt_per;
        t.kt1 = min(t.kt0 + p.kt_per, nk * (MODE == GL_DX ? 2 : 1));
        return t;
    };

    // ---- loads: a wave moves pieces `wave` and `wave + NW` (1 KiB each) of every half-tile ----
    //   row layout: piece = 8 rows x 128 B; column layout: piece = 4 k rows x 256 B
    const int64_t lda = p.A[0].ld * 2, ldb = p.B[0].ld * 2;                // bytes (both planes and both weights have the same)
    auto g_of = [](int k) { return (k & 3) | ((k >> 3) & 1) << 2; };
    const int r8 = lane >> 3, c8 = (lane & 7) ^ r8;                        // row layout: row of the piece, chunk of memory
    unsigned va[2], vb[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        const int piece = wave + s * NW, k = piece * 4 + (lane >> 4), c = (lane & 15) ^ (2 * g_of(k));
        va[s] = A_ROW ? (unsigned)((piece * 8 + r8) * lda + c8 * 16) : (unsigned)(k * lda + c * 16);
        vb[s] = B_ROW ? (unsigned)((piece * 8 + r8) * ldb + c8 * 16) : (unsigned)(k * ldb + c * 16);
    }
    const bool tail_out = B_ROW && (p.C & 63) && c8 * 8 >= (int)(p.C & 63);                    // chunks past the contraction's end, last K-tile

    // A half-tile's stream walks its rows or columns K-tile by K-tile.  Row layout: rows that do not exist lie behind `full` bytes whatever
    // the K-tile.  Column layout: a K-tile has 64 k rows, the segment's last one `last` bytes.
    struct Stream { u32x4 at; unsigned full, last; int kt; };
    auto seg_of = [&](int kt) { return MODE == GL_DX && kt >= nk ? 1 : 0; };
    auto open = [&](const Tile& t, bool is_b, int h, int kt) {
        const bool row = is_b ? B_ROW : A_ROW;
        const int seg = seg_of(kt);
        const GlOp& op = is_b ? p.B[MODE == GL_FWD ? h : seg] : p.A[MODE == GL_DX ? seg : MODE == GL_DW ? t.plane : 0];
        const int64_t ld = op.ld * 2, size = is_b ? p.J : p.I, kk = kt - seg * nk;
        const int64_t first = (is_b ? t.j0 : t.i0) + (MODE == GL_FWD && is_b ? 0 : h * HR);        // first row / column of the half
        Stream st;
        st.at = gl_buffer((const char*)op.p + (row ? first * ld + kk * 128 : kk * 64 * ld + first * 2));
        st.full = gl_clip(row ? (size - 1 - first) * ld + op.cols * 2 : 63 * ld + (op.cols - first) * 2);
        if (first >= (row ? size : op.cols)) st.full = 0;
        st.last = row || st.full == 0 ? st.full : gl_clip((p.C - 1 - (int64_t)(nk - 1) * 64) * ld + (op.cols - first) * 2);
        st.kt = kt;
        return st;
    };
    Stream sa[2], sb[2];
    Tile in;                                                               // the tile that is loaded
    const int64_t step_a = A_ROW ? 128 : 64 * lda, step_b = B_ROW ? 128 : 64 * ldb;
    const unsigned lds0 = gt_lds(smem);
    auto stage = [&](bool is_b, int h) {                                   // the next K-tile of a half; past the last one: no bytes
        Stream& st = is_b ? sb[h] : sa[h];
        const bool last = st.kt - seg_of(st.kt) * nk == nk - 1;
        st.at[2] = st.kt >= in.kt1 ? 0u : last ? st.last : st.full;
        const unsigned dst = lds0 + (unsigned)((((st.kt - in.kt0) & 1) * 4 + (is_b ? 2 : 0) + h) * HB + wave * 1024);
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            unsigned vo = is_b ? vb[s] : va[s];
            if (B_ROW && last && tail_out) vo = OUTSIDE;
            gl_load_lds(st.at, vo, dst + s * NW * 1024);
        }
        ++st.kt;
        gl_advance(st.at, is_b ? step_b : step_a);
        if (MODE == GL_DX && __builtin_expect(st.kt == nk, 0)) {
            asm volatile("");                                              // a branch, not a selection computed every time
            st = open(in, is_b, h, st.kt);
        }
    };

    // ---- fragment reads: an LDS byte address per k-step (row layout) or per 16 columns (column layout: the tile's number is xor'ed
    // into the slot bits), and constant offsets ----
    const unsigned foff = (lane & 15) * 128 + (((lane >> 4) ^ (lane & 7)) << 4);
    const int krow = (lane >> 4) * 8 + ((lane >> 2) & 3);
    const unsigned fc = krow * 256 + (g_of(krow) << 5) + (lane & 3) * 8;
    const unsigned fa = A_ROW ? foff + wm * MI * 2048 : fc ^ (wm * MI << 5), fb = B_ROW ? foff + wn * NJ * 2048 : fc ^ (wn * NJ << 5);
    typedef const DP_LDS_AS char* LdsAt;
    auto frag = [&](bool row, unsigned at, int off, int ks, int t) {       // k-step ks, 16-row tile t of the wave's, half-tile at byte `off`
        if (row) return *(const DP_LDS_AS bf16x8*)((LdsAt)(uintptr_t)(at ^ (ks * 64)) + (off + t * 2048));
        const LdsAt c = (LdsAt)(uintptr_t)(at ^ (t << 5)) + (off + ks * 8192);
        const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((DP_LDS_AS bf16x4*)c), hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((DP_LDS_AS bf16x4*)(c + 1024));
        return (bf16x8)__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    bf16x8 af[2][MI], b0[2][NJ], b1[2][NJ];
    auto read_a = [&](unsigned buf, int h) {
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int i = 0; i < MI; ++i) af[ks][i] = frag(A_ROW, buf + fa, h * HB, ks, i);
    };
    auto read_b = [&](bf16x8 (&d)[2][NJ], unsigned buf, int h) {
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int j = 0; j < NJ; ++j) d[ks][j] = frag(B_ROW, buf + fb, (2 + h) * HB, ks, j);
    };

    f32x4 acc[2][MI][2][NJ];                                               // [A half][m-tile][B half][n-tile]
#define GT_MFMA(ha, hb, bfr)                                                                                    \
    do {                                                                                                        \
        asm volatile("" ::: "memory");                                                                          \
        __builtin_amdgcn_s_barrier();                                                                           \
        __builtin_amdgcn_s_waitcnt(0xc07f);      /* lgkmcnt(0) */                                               \
        __builtin_amdgcn_sched_barrier(0);                                                                      \
        __builtin_amdgcn_s_setprio(1);                                                                          \
        _Pragma("unroll") for (int ks = 0; ks < 2; ++ks) _Pragma("unroll") for (int i = 0; i < MI; ++i)         \
            _Pragma("unroll") for (int j = 0; j < NJ; ++j)                                                      \
                acc[ha][i][hb][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bfr[ks][j], af[ks][i], acc[ha][i][hb][j], 0, 0, 0); \
        __builtin_amdgcn_s_setprio(0);                                                                          \
        __builtin_amdgcn_sched_barrier(0);                                                                      \
        __builtin_amdgcn_s_barrier();                                                                           \
        asm volatile("" ::: "memory");                                                                          \
    } while (0)

    // The first loads of a tile: where there is one before it, they are in flight while that one's results are stored.
    auto begin = [&](int at) {
        in = locate(at);
        for (int h = 0; h < 2; ++h) {
            sa[h] = open(in, false, h, in.kt0);
            sb[h] = open(in, true, h, in.kt0);
        }
        stage(true, 1); stage(false, 0); stage(true, 0); stage(false, 1);
        stage(true, 1); stage(false, 0); stage(true, 0);
    };
    if (b < q.wgs) begin(b);
    bool first = true;
#pragma clang loop unroll(disable)
    for (; b < q.wgs; b += step, first = false) {
        const Tile cur = in;
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int j = 0; j < NJ; ++j) acc[a][i][b][j] = (f32x4){0.f, 0.f, 0.f, 0.f};

        if (first) GT_VMCNT(8);                                                // B1, A0, B0 of the first K-tile
        else GT_VMCNT(0);                                                      // (the last tile's stores are behind them)
        __builtin_amdgcn_s_barrier();
        if (wm == 1) __builtin_amdgcn_s_barrier();                             // the lower half runs one barrier behind
        asm volatile("" ::: "memory");
        read_b(b1, lds0, 1);
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_s_waitcnt(0xc07f);
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        unsigned par = 0;
#pragma clang loop unroll(disable)
        for (int kt = cur.kt0; kt < cur.kt1; ++kt, par ^= 4 * HB) {
            const unsigned buf = lds0 + par, nbuf = lds0 + (par ^ 4 * HB);
            read_b(b0, buf, 0);                                                // c0
            read_a(buf, 0);
            GT_MFMA(0, 0, b0);
            stage(false, 1);                                                   // c1: A1(t+1), B1(t+2)
            stage(true, 1);
            GT_VMCNT(10);
            GT_MFMA(0, 1, b1);
            read_a(buf, 1);                                                    // c2
            stage(false, 0);
            GT_VMCNT(10);
            GT_MFMA(1, 1, b1);
            read_b(b1, nbuf, 1);                                               // c3
            stage(true, 0);
            GT_VMCNT(8);
            GT_MFMA(1, 0, b0);
        }
        if (wm == 0) __builtin_amdgcn_s_barrier();                 // as many barriers as the lower half
        GT_VMCNT(0);                                                           // nothing may land in LDS behind the workgroup's end
        if (b + step < q.wgs) begin(b + step);

        // ---- epilogue: lane holds row (lane & 15), columns 4 (lane >> 4) + 0..3 of each 16 x 16 tile ----
        const int cl = wn * NJ * 16 + (lane >> 4) * 4;
        const int64_t mrow = cur.i0 + wm * (HR / 2) + (lane & 15);
        if (split) {
#pragma unroll
            for (int a = 0; a < 2; ++a)
#pragma unroll
                for (int i = 0; i < MI; ++i) {
                    const int64_t m = mrow + a * HR + i * 16;
                    if (m >= p.I) continue;
#pragma unroll
                    for (int b = 0; b < 2; ++b)
#pragma unroll
                        for (int j = 0; j < NJ; ++j) {
                            const int n = cur.j0 + (MODE == GL_FWD ? 0 : b * HR) + cl + j * 16, pl = MODE == GL_FWD ? b : cur.plane;
                            // ldp is a multiple of 4: four columns that start inside a row end inside its padding
                            if (n < p.J) *(f32x4*)(p.part + (((int64_t)cur.slice * 2 + pl) * p.I + m) * p.ldp + n) = acc[a][i][b][j];
                        }
                }
        } else if constexpr (MODE == GL_FWD) {
            static_assert(NJ == 2, "two tiles side by side");
            const int n = cur.j0 + cl;
            if (n < p.J) gl_with_act(p.act, [&](auto act) {
                f32x4 bg[2], bu[2];
                gl_bias<bf16_t>(p, n, p.J - n, bg[0], bu[0]);
                gl_bias<bf16_t>(p, n + 16, p.J - n - 16, bg[1], bu[1]);
#pragma unroll
                for (int a = 0; a < 2; ++a)
#pragma unroll
                    for (int i = 0; i < MI; ++i) {
                        const int64_t m = mrow + a * HR + i * 16;
                        const f32x4 g[2] = {acc[a][i][0][0] + bg[0], acc[a][i][0][1] + bg[1]}, u[2] = {acc[a][i][1][0] + bu[0], acc[a][i][1][1] + bu[1]};
                        if (m < p.I) gl_fwd_put2<decltype(act)::value>(p, m, n, g, u);
                    }
            });
        } else {
            bf16_t* const out = (bf16_t*)p.out[MODE == GL_DW ? cur.plane : 0];
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    const int n = cur.j0 + b * HR + cl + j * 16, cnt = p.J - n;
                    if (cnt <= 0) continue;
#pragma unroll
                    for (int a = 0; a < 2; ++a)
#pragma unroll
                        for (int i = 0; i < MI; ++i) {
                            const int64_t m = mrow + a * HR + i * 16;
                            if (m < p.I) gl_put4(out + m * p.ldo + n, acc[a][i][b][j], cnt);
                        }
                }
        }
    }
#undef GT_MFMA
    return b - q.wgs;
}

template <int MODE>
__global__ __launch_bounds__(GT_THREADS) void k_gated_tile(GtArgs q) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    gt_product<MODE>(q, blockIdx.x, gridDim.x, smem);
}
// both backward products in one launch, the longer contraction first, and the column sums
__global__ __launch_bounds__(GT_THREADS) static void k_gated_tile_both(GtArgs dx, GtArgs dw, int dx_first, GlColsum cs) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int step = gridDim.x - cs.n;
    int b = blockIdx.x;
    if (b >= step) return gl_colsum<bf16_t, GT_THREADS>(cs, b - step, (f32x4(*)[16])smem);
#pragma clang loop unroll(disable)
    for (int k = 0; k < 2; ++k) b = (k == 0) == (dx_first != 0) ? gt_product<GL_DX>(dx, b, step, smem) : gt_product<GL_DW>(dw, b, step, smem);
}

}  // namespace dp
