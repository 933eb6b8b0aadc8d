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

// Fragments of column-laid-out half-tiles: for every 16-column tile and k-step two reads of 4 k's each, in one statement that
// ends with their wait (KS, HI: byte offsets of the second k-step and of a fragment's second four k's).
template <int KS, int HI> __device__ __forceinline__ void gt_tr4(bf16x4 (&a)[2][4][2], const unsigned (&ra)[4]) {
    asm volatile("ds_read_b64_tr_b16 %0, %16\n\t" "ds_read_b64_tr_b16 %1, %16 offset:%20\n\t"
                 "ds_read_b64_tr_b16 %4, %17\n\t" "ds_read_b64_tr_b16 %5, %17 offset:%20\n\t"
                 "ds_read_b64_tr_b16 %8, %18\n\t" "ds_read_b64_tr_b16 %9, %18 offset:%20\n\t"
                 "ds_read_b64_tr_b16 %12, %19\n\t" "ds_read_b64_tr_b16 %13, %19 offset:%20\n\t"
                 "ds_read_b64_tr_b16 %2, %16 offset:%21\n\t" "ds_read_b64_tr_b16 %3, %16 offset:%22\n\t"
                 "ds_read_b64_tr_b16 %6, %17 offset:%21\n\t" "ds_read_b64_tr_b16 %7, %17 offset:%22\n\t"
                 "ds_read_b64_tr_b16 %10, %18 offset:%21\n\t" "ds_read_b64_tr_b16 %11, %18 offset:%22\n\t"
                 "ds_read_b64_tr_b16 %14, %19 offset:%21\n\t" "ds_read_b64_tr_b16 %15, %19 offset:%22\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(a[0][0][0]), "=&v"(a[0][0][1]), "=&v"(a[1][0][0]), "=&v"(a[1][0][1]), "=&v"(a[0][1][0]), "=&v"(a[0][1][1]), "=&v"(a[1][1][0]),
                   "=&v"(a[1][1][1]), "=&v"(a[0][2][0]), "=&v"(a[0][2][1]), "=&v"(a[1][2][0]), "=&v"(a[1][2][1]), "=&v"(a[0][3][0]), "=&v"(a[0][3][1]),
                   "=&v"(a[1][3][0]), "=&v"(a[1][3][1])
                 : "v"(ra[0]), "v"(ra[1]), "v"(ra[2]), "v"(ra[3]), "n"(HI), "n"(KS), "n"(KS + HI)
                 : "memory");
}
template <int KS, int HI> __device__ __forceinline__ void gt_tr2(bf16x4 (&a)[2][2][2], const unsigned (&ra)[2]) {
    asm volatile("ds_read_b64_tr_b16 %0, %8\n\t" "ds_read_b64_tr_b16 %1, %8 offset:%10\n\t"
                 "ds_read_b64_tr_b16 %4, %9\n\t" "ds_read_b64_tr_b16 %5, %9 offset:%10\n\t"
                 "ds_read_b64_tr_b16 %2, %8 offset:%11\n\t" "ds_read_b64_tr_b16 %3, %8 offset:%12\n\t"
                 "ds_read_b64_tr_b16 %6, %9 offset:%11\n\t" "ds_read_b64_tr_b16 %7, %9 offset:%12\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(a[0][0][0]), "=&v"(a[0][0][1]), "=&v"(a[1][0][0]), "=&v"(a[1][0][1]), "=&v"(a[0][1][0]), "=&v"(a[0][1][1]), "=&v"(a[1][1][0]), "=&v"(a[1][1][1])
                 : "v"(ra[0]), "v"(ra[1]), "n"(HI), "n"(KS), "n"(KS + HI)
                 : "memory");
}
template <int KS, int HI> __device__ __forceinline__ void gt_tr4_2(bf16x4 (&a)[2][4][2], const unsigned (&ra)[4], bf16x4 (&b)[2][2][2], const unsigned (&rb)[2]) {
    asm volatile("ds_read_b64_tr_b16 %0, %24\n\t" "ds_read_b64_tr_b16 %1, %24 offset:%30\n\t"
                 "ds_read_b64_tr_b16 %4, %25\n\t" "ds_read_b64_tr_b16 %5, %25 offset:%30\n\t"
                 "ds_read_b64_tr_b16 %8, %26\n\t" "ds_read_b64_tr_b16 %9, %26 offset:%30\n\t"
                 "ds_read_b64_tr_b16 %12, %27\n\t" "ds_read_b64_tr_b16 %13, %27 offset:%30\n\t"
                 "ds_read_b64_tr_b16 %16, %28\n\t" "ds_read_b64_tr_b16 %17, %28 offset:%30\n\t"
                 "ds_read_b64_tr_b16 %20, %29\n\t" "ds_read_b64_tr_b16 %21, %29 offset:%30\n\t"
                 "ds_read_b64_tr_b16 %2, %24 offset:%31\n\t" "ds_read_b64_tr_b16 %3, %24 offset:%32\n\t"
                 "ds_read_b64_tr_b16 %6, %25 offset:%31\n\t" "ds_read_b64_tr_b16 %7, %25 offset:%32\n\t"
                 "ds_read_b64_tr_b16 %10, %26 offset:%31\n\t" "ds_read_b64_tr_b16 %11, %26 offset:%32\n\t"
                 "ds_read_b64_tr_b16 %14, %27 offset:%31\n\t" "ds_read_b64_tr_b16 %15, %27 offset:%32\n\t"
                 "ds_read_b64_tr_b16 %18, %28 offset:%31\n\t" "ds_read_b64_tr_b16 %19, %28 offset:%32\n\t"
                 "ds_read_b64_tr_b16 %22, %29 offset:%31\n\t" "ds_read_b64_tr_b16 %23, %29 offset:%32\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(a[0][0][0]), "=&v"(a[0][0][1]), "=&v"(a[1][0][0]), "=&v"(a[1][0][1]), "=&v"(a[0][1][0]), "=&v"(a[0][1][1]), "=&v"(a[1][1][0]),
                   "=&v"(a[1][1][1]), "=&v"(a[0][2][0]), "=&v"(a[0][2][1]), "=&v"(a[1][2][0]), "=&v"(a[1][2][1]), "=&v"(a[0][3][0]), "=&v"(a[0][3][1]),
                   "=&v"(a[1][3][0]), "=&v"(a[1][3][1]), "=&v"(b[0][0][0]), "=&v"(b[0][0][1]), "=&v"(b[1][0][0]), "=&v"(b[1][0][1]), "=&v"(b[0][1][0]),
                   "=&v"(b[0][1][1]), "=&v"(b[1][1][0]), "=&v"(b[1][1][1])
                 : "v"(ra[0]), "v"(ra[1]), "v"(ra[2]), "v"(ra[3]), "v"(rb[0]), "v"(rb[1]), "n"(HI), "n"(KS), "n"(KS + HI)
                 : "memory");
}
__device__ __forceinline__ bf16x8 gt_join(const bf16x4 (&f)[2]) { return __builtin_shufflevector(f[0], f[1], 0, 1, 2, 3, 4, 5, 6, 7); }

// workgroup `b` of the launch's `count` that run this product: its tile and slice, neighbouring tiles on one XCD
template <int MODE>
__device__ __forceinline__ void gt_product(const GtArgs& q, int b, int count, char* smem) {
    constexpr bool A_ROW = MODE != GL_DW, B_ROW = MODE == GL_FWD;
    constexpr int HR = GT_HR, HB = GT_HB, MI = GT_MI, NJ = GT_NJ, NW = GT_NW, WN = GT_WN;
    constexpr unsigned OUTSIDE = 0x80000000u;                              // an offset behind every buffer
    const GlArgs& p = q.g;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / WN, wn = wave % WN;

    const bool split = p.splits > 1;
    int slice, plane, ti, tj;
    gt_tile<MODE>(q, b, count, slice, plane, ti, tj);
    const int64_t i0 = (int64_t)ti * GT_T;
    const int j0 = tj * (MODE == GL_FWD ? HR : GT_T);

    const int nk = (int)((p.C + 63) >> 6);                                 // K-tiles of a segment
    const int kt0 = slice * p.kt_per, kt1 = min(kt0 + p.kt_per, nk * (MODE == GL_DX ? 2 : 1));

    // ---- loads: a wave moves pieces `wave` and `wave + NW` (1 KiB each) of every half-tile ----
    //   row layout: piece = 8 rows x 128 B; column layout: piece = 1024 / (2 HR) k rows x 2 HR bytes
    const int64_t lda = p.A[MODE == GL_DW ? plane : 0].ld * 2, ldb = p.B[0].ld * 2;            // bytes
    constexpr int KR = 1024 / (2 * HR), CH = HR / 8;                       // k rows per piece, 16-byte chunks per k row
    auto g_of = [](int k) { return (k & 3) | ((k >> 3) & 1) << 2; };
    unsigned va[2], vb[2];
    const int r8 = lane >> 3, c8 = (lane & 7) ^ r8;                        // row layout: row of the piece, chunk of memory
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        const int piece = wave + s * NW;
        const int k = piece * KR + lane / CH, c = (lane % CH) ^ (2 * g_of(k));
        va[s] = A_ROW ? (unsigned)((piece * 8 + r8) * lda + c8 * 16) : (unsigned)(k * lda + c * 16);
        vb[s] = B_ROW ? (unsigned)((piece * 8 + r8) * ldb + c8 * 16) : (unsigned)(k * ldb + c * 16);
    }
    // row layout, last K-tile of a contraction that is no multiple of 64: chunks past its end
    const int tail = B_ROW && (p.C & 63) ? nk - 1 : -1;
    const bool tail_out = c8 * 8 >= (int)(p.C & 63);

    auto stage = [&](bool is_b, int kt, int h) {
        const bool row = is_b ? B_ROW : A_ROW;
        const bool live = kt < kt1;
        const int seg = MODE == GL_DX && kt >= nk ? 1 : 0;
        const int64_t kk = kt - seg * nk;
        const GlOp& op = is_b ? p.B[MODE == GL_FWD ? h : seg] : p.A[MODE == GL_DX ? seg : MODE == GL_DW ? plane : 0];
        const int64_t ld = is_b ? ldb : lda, size = is_b ? p.J : p.I;
        const int64_t at = (is_b ? j0 : i0) + (MODE == GL_FWD && is_b ? 0 : h * HR);           // first row / column of the half
        const char* const base = (const char*)op.p;
        const char* const from = base + (row ? at * ld + kk * 128 : kk * 64 * ld + at * 2);
        const char* const end = base + (row ? size - 1 : p.C - 1) * ld + op.cols * 2;
        const auto buf = gt_buffer(from, live ? end : from);
        char* const dst = smem + (((kt - kt0) & 1) * 4 + (is_b ? 2 : 0) + h) * HB + wave * 1024;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            unsigned vo = is_b ? vb[s] : va[s];
            if (row && B_ROW && kt == tail && tail_out) vo = OUTSIDE;
            gt_load<16>(buf, dst + s * NW * 1024, vo);
        }
    };

    // ---- fragment reads ----
    //   row layout: row (lane & 15) of a 16-row tile, chunk ks * 4 + lane / 16, swizzled: an address per k-step
    //   column layout: lane = (k row (lane >> 2) & 3 of four, 8 bytes lane & 3 of the tile's 32): an address per 16-column tile
    const int foff = (lane & 15) * 128 + (((lane >> 4) ^ (lane & 7)) << 4);
    const int krow = (lane >> 4) * 8 + ((lane >> 2) & 3);
    unsigned ra[A_ROW ? 2 : MI], rb[B_ROW ? 2 : NJ];
    if (A_ROW) { ra[0] = wm * (HR / 2) * 128 + foff; ra[1] = ra[0] ^ 64; }
    else
#pragma unroll
        for (int i = 0; i < MI; ++i) ra[i] = krow * HR * 2 + (((wm * MI + i) ^ g_of(krow)) << 5) + (lane & 3) * 8;
    if (B_ROW) { rb[0] = wn * NJ * 2048 + foff; rb[1] = rb[0] ^ 64; }
    else
#pragma unroll
        for (int j = 0; j < NJ; ++j) rb[j] = krow * HR * 2 + (((wn * NJ + j) ^ g_of(krow)) << 5) + (lane & 3) * 8;
    constexpr int KS = 32 * HR * 2, HI = 4 * HR * 2;
    const unsigned lds0 = gt_lds(smem);
    bf16x8 af[2][MI], b0[2][NJ], b1[2][NJ];
    // A half `ha` of buffer `buf` into af and / or B half `hb` into d (-1: none); with column-laid-out operands the reads have
    // landed when this returns, with row-laid-out ones they are in flight
    auto read = [&](const char* buf, int ha, bf16x8 (*d)[NJ], int hb) {
        if (A_ROW && ha >= 0)
#pragma unroll
            for (int ks = 0; ks < 2; ++ks)
#pragma unroll
                for (int i = 0; i < MI; ++i) af[ks][i] = *(const bf16x8*)(buf + ha * HB + ra[A_ROW ? ks : 0] + i * 2048);
        if (B_ROW && hb >= 0)
#pragma unroll
            for (int ks = 0; ks < 2; ++ks)
#pragma unroll
                for (int j = 0; j < NJ; ++j) d[ks][j] = *(const bf16x8*)(buf + (2 + hb) * HB + rb[B_ROW ? ks : 0] + j * 2048);
        if constexpr (!B_ROW) {
            const unsigned at = lds0 + (unsigned)(buf - smem);
            bf16x4 ta[2][MI][2], tb[2][NJ][2];
            unsigned xa[MI], xb[NJ];
            if constexpr (!A_ROW)
                if (ha >= 0)
#pragma unroll
                    for (int i = 0; i < MI; ++i) xa[i] = at + ha * HB + ra[i];
            if (hb >= 0)
#pragma unroll
                for (int j = 0; j < NJ; ++j) xb[j] = at + (2 + hb) * HB + rb[j];
            if constexpr (A_ROW) {
                if (hb >= 0) gt_tr2<KS, HI>(tb, xb);
            } else if (ha >= 0) {
                if (hb >= 0) gt_tr4_2<KS, HI>(ta, xa, tb, xb);
                else gt_tr4<KS, HI>(ta, xa);
            } else if (hb >= 0) gt_tr2<KS, HI>(tb, xb);
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
                if (!A_ROW && ha >= 0)
#pragma unroll
                    for (int i = 0; i < MI; ++i) af[ks][i] = gt_join(ta[ks][i]);
                if (hb >= 0)
#pragma unroll
                    for (int j = 0; j < NJ; ++j) d[ks][j] = gt_join(tb[ks][j]);
            }
        }
    };

    f32x4 acc[2][MI][2][NJ];                                               // [A half][m-tile][B half][n-tile]
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int j = 0; j < NJ; ++j) acc[a][i][b][j] = (f32x4){0.f, 0.f, 0.f, 0.f};

#define GT_MFMA(ha, hb, bfr)                                                                                    \
    do {                                                                                                        \
        __builtin_amdgcn_s_barrier();                                                                           \
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");                                                      \
        __builtin_amdgcn_sched_barrier(0);                                                                      \
        __builtin_amdgcn_s_setprio(1);                                                                          \
        _Pragma("unroll") for (int ks = 0; ks < 2; ++ks) _Pragma("unroll") for (int i = 0; i < MI; ++i)         \
            _Pragma("unroll") for (int j = 0; j < NJ; ++j)                                                      \
                acc[ha][i][hb][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bfr[ks][j], af[ks][i], acc[ha][i][hb][j], 0, 0, 0); \
        __builtin_amdgcn_s_setprio(0);                                                                          \
        __builtin_amdgcn_sched_barrier(0);                                                                      \
        __builtin_amdgcn_s_barrier();                                                             \
    } while (0)

    stage(true, kt0, 1); stage(false, kt0, 0); stage(true, kt0, 0); stage(false, kt0, 1);
    stage(true, kt0 + 1, 1); stage(false, kt0 + 1, 0); stage(true, kt0 + 1, 0);
    GT_VMCNT(8);                                                           // B1, A0, B0 of the first K-tile
    __builtin_amdgcn_s_barrier();
    if (wm == 1) __builtin_amdgcn_s_barrier();                 // the lower half runs one barrier behind
    read(smem, -1, b1, 1);
    __builtin_amdgcn_s_barrier();
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
#pragma clang loop unroll(disable)
    for (int kt = kt0; kt < kt1; ++kt) {
        const char* const buf = smem + ((kt - kt0) & 1) * 4 * HB;
        const char* const nbuf = smem + ((kt + 1 - kt0) & 1) * 4 * HB;
        read(buf, 0, b0, 0);                                               // c0
        GT_MFMA(0, 0, b0);
        stage(false, kt + 1, 1);                                           // c1
        stage(true, kt + 2, 1);
        GT_VMCNT(10);
        GT_MFMA(0, 1, b1);
        stage(false, kt + 2, 0);                                           // c2
        read(buf, 1, nullptr, -1);
        GT_VMCNT(10);
        GT_MFMA(1, 1, b1);
        stage(true, kt + 2, 0);                                            // c3
        read(nbuf, -1, b1, 1);
        GT_VMCNT(8);
        GT_MFMA(1, 0, b0);
    }
    if (wm == 0) __builtin_amdgcn_s_barrier();                 // as many barriers as the lower half
    GT_VMCNT(0);                                                           // nothing may land in LDS behind the workgroup's end
#undef GT_MFMA

    // ---- epilogue: lane holds row (lane & 15), columns 4 (lane >> 4) + 0..3 of each 16 x 16 tile ----
    const int cl = wn * NJ * 16 + (lane >> 4) * 4;
    const int64_t mrow = i0 + wm * (HR / 2) + (lane & 15);
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
                        const int n = j0 + (MODE == GL_FWD ? 0 : b * HR) + cl + j * 16, pl = MODE == GL_FWD ? b : plane;
                        // ldp is a multiple of 4: four columns that start inside a row end inside its padding
                        if (n < p.J) *(f32x4*)(p.part + (((int64_t)slice * 2 + pl) * p.I + m) * p.ldp + n) = acc[a][i][b][j];
                    }
            }
        return;
    }
    if constexpr (MODE == GL_FWD) {
        gl_with_act(p.act, [&](auto act) {
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const int n = j0 + cl + j * 16, cnt = p.J - n;
                if (cnt <= 0) continue;
                f32x4 bg, bu;
                gl_bias<bf16_t>(p, n, cnt, bg, bu);
#pragma unroll
                for (int a = 0; a < 2; ++a)
#pragma unroll
                    for (int i = 0; i < MI; ++i) {
                        const int64_t m = mrow + a * HR + i * 16;
                        if (m < p.I) gl_fwd_put<bf16_t, decltype(act)::value>(p, m, n, cnt, acc[a][i][0][j] + bg, acc[a][i][1][j] + bu);
                    }
            }
        });
    } else {
        bf16_t* const out = (bf16_t*)p.out[MODE == GL_DW ? plane : 0];
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const int n = j0 + b * HR + cl + j * 16, cnt = p.J - n;
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

template <int MODE>
__global__ __launch_bounds__(GT_THREADS) void k_gated_tile(GtArgs q) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    gt_product<MODE>(q, blockIdx.x, gridDim.x, smem);
}
// both backward products in one launch, the longer contraction first: workgroups [0, n0) the one, [n0, gridDim) the other
__global__ __launch_bounds__(GT_THREADS) static void k_gated_tile_both(GtArgs dx, GtArgs dw, int n0, int dx_first) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int b = blockIdx.x, first = b < n0, at = first ? b : b - n0, count = first ? n0 : gridDim.x - n0;
    if (first == dx_first) gt_product<GL_DX>(dx, at, count, smem);
    else gt_product<GL_DW>(dw, at, count, smem);
}

}  // namespace dp
