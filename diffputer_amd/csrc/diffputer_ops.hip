// Operators beside the sampler: the gated projection with its backward (dp_gated.h) and the global gradient norm with
// clipping (dp_grads.h).  Host side and C ABI (include/diffputer.h); linked into libdiffputer_hip.so.
#include <math.h>
#include <string.h>

#include <algorithm>
#include <atomic>
#include <mutex>
#include <new>
#include <vector>

#include "dp_gated.h"
#include "dp_gated_f32.h"
#include "dp_gated_ring.h"
#include "dp_gated_rows.h"
#include "dp_gated_tile.h"
#include "dp_grads.h"
#include "dp_util.h"

namespace dp {

static bool aligned(const void* p, size_t a) { return ((uintptr_t)p & (a - 1)) == 0; }

// ---- gated projection -------------------------------------------------------------------------------------------------
constexpr int64_t GL_MAX_DIM = 1 << 20;                          // N and K
constexpr int64_t GL_MAX_ROWS = (int64_t)1 << 29;                // M (exclusive): a grid has fewer than 2^32 threads

static int gl_check(const char* who, int dtype, int64_t M, int N, int K, int act) {
    if (dtype != DP_DTYPE_F32 && dtype != DP_DTYPE_BF16) return fail(DP_EINVAL, "%s: unknown dtype %d", who, dtype);
    if (M < 0 || M >= GL_MAX_ROWS || N < 1 || N > GL_MAX_DIM || K < 1 || K > GL_MAX_DIM)
        return fail(DP_EINVAL, "%s: M=%lld N=%d K=%d: need 0 <= M < 2^29, 1 <= N, K <= 2^20", who, (long long)M, N, K);
    if (act != GL_ACT_NONE && act != GL_ACT_SILU && act != GL_ACT_GELU) return fail(DP_EINVAL, "%s: unknown activation %d", who, act);
    return DP_OK;
}

// tuning knobs (dp_tune, defined in diffputer_hip.hip): "gated_kernel" 0 = by the rule below, 1 = the general kernel, 64 / 128 / 256 = the
// tile kernel of that tile (the nearest one that the type has); "gated_splits" 0 = by the rule, n = that many slices of the
// contraction (as many as there are K-tiles at most)
std::atomic<int> g_gated_kernel{0}, g_gated_splits{0};
// read once by an entry point: everything that a call decides (operands, planes, plans, workspace, launches) is decided by one pair of values
struct GlTune { int kernel, splits; };
static GlTune gl_tune() { return {g_gated_kernel.load(std::memory_order_relaxed), g_gated_splits.load(std::memory_order_relaxed)}; }

// dynamic LDS of the tile kernels, once per device
template <int MODE> static hipError_t gt_attributes() {
    const struct { const void* k; int lds; } all[] = {
        {(const void*)k_gated_tile<MODE>, GT_LDS}, {(const void*)k_gated_ring<MODE>, GS_LDS},
        {(const void*)k_gated_f32<MODE, 128, false>, GfShape<128>::LDS}, {(const void*)k_gated_f32<MODE, 128, true>, GfShape<128>::LDS},
        {(const void*)k_gated_tile_both, GT_LDS}, {(const void*)k_gated_ring_both, GS_LDS},
        {(const void*)k_gated_f32_both<128, false>, GfShape<128>::LDS}, {(const void*)k_gated_f32_both<128, true>, GfShape<128>::LDS}};
    for (const auto& a : all) {
        const hipError_t e = hipFuncSetAttribute(a.k, hipFuncAttributeMaxDynamicSharedMemorySize, a.lds);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}
static int gt_ready() {
    static std::atomic<int> ready[64];
    static std::mutex mutex;
    int dev = 0;
    DP_HIP(hipGetDevice(&dev));
    if (dev < 0 || dev >= 64) return fail(DP_EHIP, "device index %d", dev);
    if (ready[dev].load(std::memory_order_acquire)) return DP_OK;
    std::lock_guard<std::mutex> lock(mutex);
    DP_HIP(gt_attributes<GL_FWD>());
    DP_HIP(gt_attributes<GL_DX>());
    DP_HIP(gt_attributes<GL_DW>());
    ready[dev].store(1, std::memory_order_release);
    return DP_OK;
}

// ---- how a product runs: by the general kernel (T = 0), a tile kernel (T = 64, 128 or 256) or the kernel for few rows
// (GL_ROWS, forward only), and in how many slices of the contraction ----
constexpr int GL_ROWS = 1;
struct GlShape { int mode; int64_t I; int J; int64_t C; int planes; GlTune tune; };
struct GlPlan { int T, kt_per, splits; int64_t ti, tj, wgs; };
static int64_t gl_ldp(int J) { return round_up<int64_t>(J, 4); }
static size_t gl_part_bytes(const GlShape& s) { return (size_t)2 * s.I * gl_ldp(s.J) * 4; }       // one slice: two planes

static GlPlan gl_shape(const GlShape& s, int T, int kdepth, int want) {
    GlPlan pl;
    const int t = T ? T : GG_T;
    const int64_t nk = ceil_div<int64_t>(s.C, kdepth) * (s.mode == GL_DX ? 2 : 1);
    pl.T = T;
    pl.ti = ceil_div<int64_t>(s.I, t);
    pl.tj = ceil_div<int64_t>(s.J, s.mode == GL_FWD ? t / 2 : t);
    if (s.tune.splits) want = s.tune.splits;
    pl.kt_per = (int)ceil_div<int64_t>(nk, std::max<int64_t>(1, std::min<int64_t>(want, nk)));
    pl.splits = (int)ceil_div<int64_t>(nk, pl.kt_per);
    pl.wgs = pl.ti * pl.tj * s.planes * pl.splits;
    return pl;
}

// Microseconds of a launch of up to two products, from what the kernels measured with 64 to 4096 workgroups and K-loops of 16 and
// 64 K-tiles: a K-step of `depth` takes `one` where a workgroup has its CU to itself and `full` where the CU holds `per_cu` of
// them; `fixed` is what a launch takes beyond its K-steps, `round` what every further round of workgroups adds to that (`full_fwd`,
// `round_fwd`: the forward product, whose operands are both row laid out and whose results are activated).  A split launch pays for
// its partial sums, written and read at about 4.5 TB/s (forward 10 and `slice` for each slice: most of them are still in the caches),
// and a launch more.  Over 180 sizes drawn at random (70 to 16384 rows, K 64 to 4096, N 64 to 8192, both types) the choice is on
// average as fast as the best single tile with 1 to 8 slices for everything, at worst 16 % (forward) and 7 % (backward) behind it.
struct GlRate { int T, depth, per_cu; double one, full, full_fwd, fixed, round, round_fwd, slice; };
static const GlRate GL_RATES_BF16[] = {{256, 64, 1, 1.36, 1.36, 1.36, 11.0, 5.0, 5.0, 0.7}, {128, 32, 2, 0.28, 0.50, 0.68, 5.5, 1.0, 2.5, 0.7}};
static const GlRate GL_RATES_F32[] = {{128, GF_K, 2, 2.10, 3.80, 3.80, 9.0, 4.0, 4.0, 0.3}, {64, GF_K, 4, 0.70, 2.05, 2.05, 4.0, 1.0, 1.0, 0.3}};
// (by the fullest CU: 315 workgroups of the float32 tile of 64, 2190 x 1235 x 279, take 58.0 us; in three slices 46.0)
static double gl_step(const GlRate& r, double full, double wgs) {
    const double here = std::min(ceil(wgs / 256.0), (double)r.per_cu);
    return here <= 1 ? r.one : r.one + (full - r.one) * (here - 1) / (r.per_cu - 1);
}
static double gl_cost(const GlRate& r, const GlPlan* pl, const GlShape* s, int n) {
    double wgs = 0, work = 0, join = 0;
    int longer = 0;
    for (int i = 0; i < n; ++i) {
        wgs += (double)pl[i].wgs;
        work += (double)pl[i].wgs * pl[i].kt_per;
        if (pl[i].kt_per > pl[longer].kt_per) longer = i;
        if (pl[i].splits > 1) {
            const double bytes = (double)s[i].I * s[i].J * (s[i].mode == GL_DX ? 1 : 2) * 4 * 2 * pl[i].splits;
            join = std::max(join, 5.0) + (s[i].mode == GL_FWD ? r.slice * pl[i].splits + bytes / 10e6 : bytes / 4.5e6);
        }
    }
    const double full = s[0].mode == GL_FWD ? r.full_fwd : r.full, slots = 256.0 * r.per_cu, most = pl[longer].kt_per, least = n > 1 ? pl[1 - longer].kt_per : most;
    double t;
    if (wgs <= slots) t = least * gl_step(r, full, wgs) + (most - least) * gl_step(r, full, (double)pl[longer].wgs);     // all at once; the longer ones go on alone
    else {                                                        // whole rounds, the last workgroups (short ones), and long ones that outlast the others
        const double last = fmod(wgs, slots), mean = work / slots;
        t = (mean - last * least / slots) * full + (last > 0 ? least * gl_step(r, full, last) : 0);
        t = std::max(t, mean * full + std::max(0.0, most - mean) * r.one);
    }
    return r.fixed + (s[0].mode == GL_FWD ? r.round_fwd : r.round) * std::max(0.0, ceil(wgs / slots) - 1.0) + t + join;
}

// A grid has fewer than 2^32 threads; the kernel of 256 tiles launches a workgroup per CU, which walk on by an int.
static int64_t gl_most(int T) { return T == 256 ? (int64_t)1 << 30 : (int64_t)1 << 22; }
static bool gl_grid_ok(const GlPlan& pl) { return pl.wgs < gl_most(pl.T); }

// The cheapest tile and slices for a launch of `n` products (one, or both of the backward pass); false if no tile's grid fits.
static bool gl_choose(const GlShape* s, int n, int dtype, GlPlan* best) {
    const bool bf = dtype == DP_DTYPE_BF16;
    const int forced = s[0].tune.kernel;
    static const int slices[] = {1, 2, 3, 4, 6, 8, 12, 16, 32, 64};
    double least = 1e300;
    for (int k = 0; k < 2; ++k) {
        const GlRate& r = bf ? GL_RATES_BF16[k] : GL_RATES_F32[k];
        if (forced > 1 && r.T != (bf ? std::max(forced, 128) : std::min(forced, 128))) continue;
        const int kdepth = r.depth;
        GlPlan whole[2];
        int64_t longest = 1;
        for (int i = 0; i < n; ++i) {
            whole[i] = gl_shape(s[i], r.T, kdepth, 1);
            longest = std::max<int64_t>(longest, whole[i].kt_per);
        }
        for (int a : slices) {                                    // the longer contraction in `a` slices, the other in slices as long
            if (a > 1 && longest < 2 * a) break;
            const int64_t per = ceil_div<int64_t>(longest, a);
            GlPlan pl[2];
            bool fits = true;
            for (int i = 0; i < n; ++i) {
                pl[i] = gl_shape(s[i], r.T, kdepth, (int)ceil_div<int64_t>(whole[i].kt_per, per));
                fits = fits && (pl[i].splits == 1 || gl_part_bytes(s[i]) * pl[i].splits <= (size_t)128 << 20);
            }
            if (!fits && a > 1) continue;
            if (!gl_grid_ok(pl[0]) || (n > 1 && (!gl_grid_ok(pl[1]) || pl[0].wgs + pl[1].wgs >= gl_most(r.T)))) continue;
            const double c = gl_cost(r, pl, s, n);
            if (c < least) {
                least = c;
                for (int i = 0; i < n; ++i) best[i] = pl[i];
            }
        }
    }
    return least < 1e300;
}

// The kernel for few rows reads x once per workgroup: with many rows that takes longer than the weights do, and a tile kernel,
// which pads the rows, is faster (us, few-row kernel / tile kernel).  bf16: 4096 x 8192 (K x N) at 24 rows 34 / 34, 32 rows
// 38 to 41 / 37, 64 rows 51 / 38; 1024 x 8192 at 32 rows 10.1 / 10.6, 33 rows 11.3 / 10.9, 64 rows 14.1 / 11.5; 1024 x 4096 at 64 rows
// 8.5 / 11.1.  float32: 4096 x 8192 at 32 rows 79 / 84, 33 rows 98 / 82, 64 rows 126 / 90; 2048 x 2048 at 64 rows
// 21.7 / 19.0; 512 x 1024 at 64 rows 7.5 / 11.0.
static int gr_columns(int J) { return J >= 16 * 256 ? 16 : 8; }                          // columns of a workgroup: narrow layers take twice as many workgroups
static bool gr_slower(const GlShape& s, int dtype) {
    if (dtype == DP_DTYPE_F32) return s.I > 32 && (int64_t)s.J * s.C >= (int64_t)1 << 21;
    return s.I > 32 ? (int64_t)s.J * s.C >= (int64_t)1 << 23 : s.I > 16 && s.I * s.C * 2 * ceil_div(s.J, gr_columns(s.J)) >= (int64_t)1 << 27;
}
static GlPlan gl_plan_new(const GlShape& s, int dtype, bool tile) {
    const int forced = s.tune.kernel;
    if (s.mode == GL_FWD && s.I <= GR_MAX_ROWS && forced == 0 && !(tile && gr_slower(s, dtype))) return {GL_ROWS, 0, 1, 1, 1, 1};
    if (tile && forced != 1) {
        GlPlan pl;
        if (gl_choose(&s, 1, dtype, &pl)) return pl;
    }
    // general kernel: slices until there are about two workgroups per CU, as long as a slice keeps 8 K-tiles
    const int64_t nk = ceil_div<int64_t>(s.C, GG_K) * (s.mode == GL_DX ? 2 : 1), tiles = gl_shape(s, 0, GG_K, 1).wgs;
    const int64_t want = std::min<int64_t>({512 / std::max<int64_t>(tiles, 1), nk / 8, (int64_t)(64 << 20) / std::max<int64_t>(gl_part_bytes(s), 1), 64});
    return gl_shape(s, 0, GG_K, (int)std::max<int64_t>(want, 1));
}
// both backward products, in one launch if they take kernels of one kind and fit a grid
static GlPlan gl_plan(const GlShape& s, int dtype, bool tile);
static bool gl_plan_both_new(const GlShape s[2], int dtype, bool tile, GlPlan pl[2]) {
    if (tile && s[0].tune.kernel != 1 && gl_choose(s, 2, dtype, pl)) return true;
    for (int i = 0; i < 2; ++i) pl[i] = gl_plan(s[i], dtype, tile);
    return pl[0].T == 0 && pl[1].T == 0 && gl_grid_ok(pl[0]) && gl_grid_ok(pl[1]);
}
// A choice takes a microsecond or two and is asked for several times per call (workspace query, check, launch): the last ones are
// remembered by everything that they depend on, sizes and settings.
struct GlKey {
    int64_t I, C;
    int J, mode, planes, dtype, tile, kernel, splits, both;
    bool operator==(const GlKey& o) const {
        return I == o.I && C == o.C && J == o.J && mode == o.mode && planes == o.planes && dtype == o.dtype && tile == o.tile && kernel == o.kernel && splits == o.splits && both == o.both;
    }
};
struct GlMemo { GlKey key; GlPlan pl[2]; bool one; };
static GlMemo& gl_memo(const GlShape& s, int dtype, bool tile, int both, bool& known) {
    static thread_local GlMemo memo[64];
    const GlKey k = {s.I, s.C, s.J, s.mode + 1, s.planes, dtype, tile, s.tune.kernel, s.tune.splits, both};
    GlMemo& m = memo[((uint64_t)(s.I * 31 + s.C) * 31 + (uint64_t)s.J * 7 + (uint64_t)(s.mode * 5 + both * 3 + dtype)) % 64];
    known = m.key == k;
    m.key = k;
    return m;
}
static GlPlan gl_plan(const GlShape& s, int dtype, bool tile) {
    bool known;
    GlMemo& m = gl_memo(s, dtype, tile, 0, known);
    if (!known) m.pl[0] = gl_plan_new(s, dtype, tile);
    return m.pl[0];
}
// (the second product's shape follows from the first's)
static bool gl_plan_both(const GlShape s[2], int dtype, bool tile, GlPlan pl[2]) {
    bool known;
    GlMemo& m = gl_memo(s[0], dtype, tile, 1, known);
    if (!known) {
        GlPlan p[2];
        const bool one = gl_plan_both_new(s, dtype, tile, p);     // may use the memo itself
        GlMemo& again = gl_memo(s[0], dtype, tile, 1, known);
        again.pl[0] = p[0]; again.pl[1] = p[1];
        again.one = one;
    }
    pl[0] = m.pl[0]; pl[1] = m.pl[1];
    return m.one;
}
static size_t gl_split_bytes(const GlShape& s, const GlPlan& c) { return c.splits > 1 ? gl_part_bytes(s) * c.splits : 0; }

static unsigned gt_grid(int64_t tiles) { return (unsigned)std::min<int64_t>(tiles, 256); }        // a CU has room for one workgroup, which walks on
template <int MODE>
static int gt_launch(const GtArgs& q, const GlPlan& pl, bool bf, bool vec, hipStream_t st) {
    const dim3 grid((unsigned)pl.wgs);
    if (bf) {
        if (pl.T == 256) hipLaunchKernelGGL((k_gated_tile<MODE>), dim3(gt_grid(pl.wgs)), dim3(GT_THREADS), GT_LDS, st, q);
        else hipLaunchKernelGGL((k_gated_ring<MODE>), grid, dim3(GS_THREADS), GS_LDS, st, q);
    } else if (pl.T == 128) {
        if (vec) hipLaunchKernelGGL((k_gated_f32<MODE, 128, true>), grid, dim3(GF_THREADS), GfShape<128>::LDS, st, q);
        else hipLaunchKernelGGL((k_gated_f32<MODE, 128, false>), grid, dim3(GF_THREADS), GfShape<128>::LDS, st, q);
    } else {
        if (vec) hipLaunchKernelGGL((k_gated_f32<MODE, 64, true>), grid, dim3(GF_THREADS), GfShape<64>::LDS, st, q);
        else hipLaunchKernelGGL((k_gated_f32<MODE, 64, false>), grid, dim3(GF_THREADS), GfShape<64>::LDS, st, q);
    }
    DP_LAUNCH_CHECK("gated tile kernel");
    return DP_OK;
}

static GtArgs gl_args(GlArgs a, const GlShape& s, const GlPlan& c) {
    a.I = s.I; a.J = s.J; a.C = s.C; a.kt_per = c.kt_per; a.splits = c.splits; a.ldp = gl_ldp(s.J);
    return {a, (int)c.ti, (int)c.tj, 8, (int)c.wgs};
}
static GgArgs gg_args(const GlArgs& a, const GlShape& s, const GlPlan& c) { return {gl_args(a, s, c).g, (int)c.ti, (int)c.tj, (int)c.wgs}; }
static unsigned gl_join_grid(const GlShape& s) { return (unsigned)std::min<int64_t>(ceil_div<int64_t>(s.I * s.planes * ceil_div<int64_t>(s.J, 4), 256), 4096); }

template <typename T, int MT, int CB>
static int gr_launch(const GlArgs& a, hipStream_t st) {
    hipLaunchKernelGGL((k_gated_rows<T, MT, CB>), dim3((unsigned)ceil_div(a.J, CB)), dim3(GR_WAVES * 64), 0, st, a);
    DP_LAUNCH_CHECK("k_gated_rows");
    return DP_OK;
}
template <typename T>
static int gr_rows(const GlArgs& a, hipStream_t st) {
    const bool wide = gr_columns(a.J) == 16;
    if (a.I <= 16) return wide ? gr_launch<T, 1, 16>(a, st) : gr_launch<T, 1, 8>(a, st);
    if (a.I <= 32) return wide ? gr_launch<T, 2, 16>(a, st) : gr_launch<T, 2, 8>(a, st);
    return wide ? gr_launch<T, 4, 16>(a, st) : gr_launch<T, 4, 8>(a, st);
}

// type of the general kernel's A: the planes dg, du are float32 there
template <typename T, int MODE> struct GlPlane { typedef float V; };
template <typename T> struct GlPlane<T, GL_FWD> { typedef T V; };
template <typename T, int MODE>
static int gl_mm(const GlArgs& a, const GlShape& s, const GlPlan& c, bool vec, hipStream_t st) {
    const GtArgs q = gl_args(a, s, c);
    int rc;
    if (c.T == GL_ROWS) return MODE == GL_FWD ? gr_rows<T>(q.g, st) : DP_EINVAL;
    if (c.T == 0) {
        if (c.wgs > INT32_MAX) return fail(DP_EINVAL, "gated projection: %lld tiles", (long long)c.wgs);
        const unsigned across = (unsigned)std::min<int64_t>(c.wgs, 1 << 20);
        hipLaunchKernelGGL((k_gated_mm<T, typename GlPlane<T, MODE>::V, MODE>), dim3(across, (unsigned)ceil_div<int64_t>(c.wgs, across)), dim3(256), 0, st, gg_args(a, s, c));
        DP_LAUNCH_CHECK("k_gated_mm");
    } else if ((rc = gt_ready()) || (rc = gt_launch<MODE>(q, c, sizeof(T) == 2, vec, st))) return rc;
    if (c.splits > 1) {
        hipLaunchKernelGGL((k_gated_join<T, MODE>), dim3(gl_join_grid(s)), dim3(256), 0, st, q.g, s.planes);
        DP_LAUNCH_CHECK("k_gated_join");
    }
    return DP_OK;
}

// both backward products and the column sums in one launch: the longer contraction's workgroups start first
template <typename T>
static int gl_both(const GlArgs a[2], const GlShape s[2], const GlPlan c[2], const GlColsum& cs, bool vec, hipStream_t st) {
    int rc;
    if (c[0].T && (rc = gt_ready())) return rc;
    const GtArgs dx = gl_args(a[0], s[0], c[0]), dw = gl_args(a[1], s[1], c[1]);
    const int dx_first = c[0].kt_per >= c[1].kt_per, n0 = (int)c[dx_first ? 0 : 1].wgs;
    const dim3 grid((unsigned)(c[0].wgs + c[1].wgs + cs.n));
    if (c[0].T == 0) hipLaunchKernelGGL((k_gated_mm_both<T>), grid, dim3(256), 0, st, gg_args(a[0], s[0], c[0]), gg_args(a[1], s[1], c[1]), cs);
    else if (sizeof(T) == 2) {
        if (c[0].T == 256) hipLaunchKernelGGL(k_gated_tile_both, dim3(gt_grid(c[0].wgs + c[1].wgs) + cs.n), dim3(GT_THREADS), GT_LDS, st, dx, dw, dx_first, cs);
        else hipLaunchKernelGGL(k_gated_ring_both, grid, dim3(GS_THREADS), GS_LDS, st, dx, dw, n0, dx_first, cs);
    } else if (c[0].T == 128) {
        if (vec) hipLaunchKernelGGL((k_gated_f32_both<128, true>), grid, dim3(GF_THREADS), GfShape<128>::LDS, st, dx, dw, n0, dx_first, cs);
        else hipLaunchKernelGGL((k_gated_f32_both<128, false>), grid, dim3(GF_THREADS), GfShape<128>::LDS, st, dx, dw, n0, dx_first, cs);
    } else {
        if (vec) hipLaunchKernelGGL((k_gated_f32_both<64, true>), grid, dim3(GF_THREADS), GfShape<64>::LDS, st, dx, dw, n0, dx_first, cs);
        else hipLaunchKernelGGL((k_gated_f32_both<64, false>), grid, dim3(GF_THREADS), GfShape<64>::LDS, st, dx, dw, n0, dx_first, cs);
    }
    DP_LAUNCH_CHECK("gated products");
    const unsigned jx = c[0].splits > 1 ? gl_join_grid(s[0]) : 0, jw = c[1].splits > 1 ? gl_join_grid(s[1]) : 0;
    if (jx + jw) {
        hipLaunchKernelGGL((k_gated_join_both<T>), dim3(jx + jw), dim3(256), 0, st, dx.g, dw.g, (int)jx);
        DP_LAUNCH_CHECK("k_gated_join_both");
    }
    return DP_OK;
}

// 16-byte loads into LDS need rows that start on 16 bytes and end on a whole chunk.  Other operands are copied to the workspace
// (rows padded with zeros) where the product is large enough to pay for it (float32, 4096 x 1025 x 2048 backward: 774 us with
// 4-byte loads of rows that start anywhere, 540 with copies).  Smaller products run on the general kernel in bf16, and with 4-byte
// loads in float32.  The kernel for few rows takes rows of any alignment.
static bool gt_direct(const void* p, int64_t ld, int64_t cols, int chunk) { return aligned(p, 16) && ld % chunk == 0 && cols % chunk == 0; }
// Backward passes of bf16 layers below this M N keep dg and du in float32 (general kernel, bf16 hi + lo).  Rounded, their roundings
// come into each gradient once per term: its error against float64 is 1.35 to 1.6 times that of gradients rounded only at the end, at
// 1 row as at 16384; unrounded 1.00.  What that costs, general / tile kernel in us (M x K x N): 64 x 1024 x 64 11.4 / 9.3,
// 16 x 1024 x 256 17.9 / 11.6, 1 x 1024 x 8000 49 / 32, 8 x 4096 x 1000 32 / 23; with K in the thousands beside M or N in the thousands
// it costs more (1 x 16384 x 8000 652 / 314).  In larger layers it would be the second product's whole time: those are rounded.
constexpr int64_t GL_EXACT_BELOW = 8192;                         // M N
constexpr int64_t GT_PACK_LEAST = (int64_t)1 << 26;              // M N K
constexpr int64_t GT_MAX_LD = 1 << 21;                           // 128 rows of float32 stay within 2^30 bytes
struct GtOperands { bool tile, vec, short_rows, pack_x, pack_w; int64_t ldk; };   // ldk: row stride of the copies
static GtOperands gt_operands(int forced, int dtype, const void* x, int64_t ldx, const void* wg, const void* wu, int64_t ldw, int64_t M, int N, int K) {
    GtOperands o;
    const bool bf = dtype == DP_DTYPE_BF16;
    const int chunk = bf ? 8 : 4;
    const bool x_in = gt_direct(x, ldx, K, chunk), w_in = gt_direct(wg, ldw, K, chunk) && gt_direct(wu, ldw, K, chunk);
    const bool short_rows = o.short_rows = ldx <= GT_MAX_LD && ldw <= GT_MAX_LD;
    o.vec = x_in && w_in;
    o.pack_x = o.pack_w = false;
    o.ldk = round_up<int64_t>(K, chunk);
    const bool large = (double)M * N * K >= (double)GT_PACK_LEAST;
    o.tile = forced != 1 && (bf ? forced || (o.vec && short_rows) || large : short_rows || large);
    if (o.tile && (bf || large || !short_rows)) {
        o.pack_x = !x_in || ldx > GT_MAX_LD || K % chunk;
        o.pack_w = !w_in || ldw > GT_MAX_LD || K % chunk;
        o.vec = true;
    }
    return o;
}
struct Carver {
    char* base;
    size_t off = 0;
    char* take(size_t n) { const size_t o = off; off += round_up<size_t>(n, 256); return base ? base + o : (char*)nullptr; }
};
// x and both weights as the products read them: where they are, or copied to the workspace
struct GlIn {
    GlOp x, wg, wu;
    int64_t M;
    int N, K;
    size_t es;
    GlTune tune;
    GtOperands o;
    char *px, *pw;
    void carve(Carver& c) {
        px = o.pack_x ? c.take((size_t)M * o.ldk * es) : nullptr;
        pw = o.pack_w ? c.take((size_t)2 * N * o.ldk * es) : nullptr;
    }
    // the copies to make, and how many workgroups make them
    GlPack copies(bool need_x, bool need_w, int* blocks) {
        GlPack p = {{}, o.ldk, K, 0};
        int64_t rows = 0;
        auto add = [&](GlOp& op, char* to, int64_t n) {
            p.m[p.n++] = {op.p, to, op.ld, n};
            rows += n;
            op = {to, o.ldk, o.ldk};
        };
        if (o.pack_x && need_x) add(x, px, M);
        if (o.pack_w && need_w) {
            add(wg, pw, N);
            add(wu, pw + (size_t)N * o.ldk * es, N);
        }
        *blocks = (int)std::min<int64_t>(ceil_div<int64_t>(rows * (o.ldk * (int64_t)es / 16), 256), 8192);
        return p;
    }
    // contraction length of the forward product: the copies' padding belongs to it (zeros on both sides)
    int64_t fwd_c() const { return o.pack_x && o.pack_w ? o.ldk : K; }
};
static GlIn gl_in(int dtype, const void* x, int64_t ldx, const void* wg, const void* wu, int64_t ldw, int64_t M, int N, int K) {
    const GlTune tune = gl_tune();
    return {{x, ldx, K}, {wg, ldw, K}, {wu, ldw, K}, M, N, K, dtype == DP_DTYPE_BF16 ? (size_t)2 : (size_t)4, tune, gt_operands(tune.kernel, dtype, x, ldx, wg, wu, ldw, M, N, K), nullptr, nullptr};
}

// forward workspace: copies, partial sums
struct GlFwd { GlShape s; GlPlan plan; float* part; size_t bytes; };
static GlFwd gl_fwd_carve(int dtype, GlIn& in, void* base) {
    GlFwd w;
    // the float32 forward product (both operands row laid out) loses 5 to 10 % to 4-byte loads, less than copies take
    if (dtype == DP_DTYPE_F32 && in.o.short_rows && (in.o.pack_x || in.o.pack_w)) in.o.pack_x = in.o.pack_w = in.o.vec = false;
    w.s = {GL_FWD, in.M, in.N, in.fwd_c(), 1, in.tune};
    // few rows: copies of the weights would cost more than a tile kernel gains
    w.plan = gl_plan(w.s, dtype, in.o.tile && !(in.M <= GR_MAX_ROWS && (in.o.pack_x || in.o.pack_w) && in.tune.kernel == 0));
    if (w.plan.T == GL_ROWS) {                                    // reads rows of any alignment
        in.o.pack_x = in.o.pack_w = false;
        w.s.C = in.K;
    }
    Carver c = {(char*)base};
    in.carve(c);
    w.part = (float*)c.take(gl_split_bytes(w.s, w.plan));
    w.bytes = c.off;
    return w;
}

// backward workspace: copies; the two planes dg, du; partial column sums; partial products
struct GlBwd {
    char* dgu;
    float *colpart, *part[2];
    GlShape s[2];              // dx, dW
    GlPlan plan[2];
    bool both;                 // in one launch
    int plane;                 // type of the planes
    int64_t ldg;
    int tx, rows, nblk;
    size_t bytes;
};
static GlBwd gl_bwd_carve(int dtype, GlIn& in, int planes, bool want_dx, void* base) {
    const int64_t M = in.M;
    const int N = in.N, K = in.K;
    GlBwd w;
    // small layers take the general kernel, whose dg and du are not rounded
    if (dtype == DP_DTYPE_BF16 && M * N < GL_EXACT_BELOW && in.tune.kernel == 0) in.o.tile = in.o.pack_x = in.o.pack_w = false;
    w.s[0] = {GL_DX, M, K, N, 1, in.tune};
    w.s[1] = {GL_DW, N, K, M, planes ? planes : 2, in.tune};
    for (;;) {
        w.both = false;
        if (want_dx && planes == 2) w.both = gl_plan_both(w.s, dtype, in.o.tile, w.plan);
        else for (int i = 0; i < 2; ++i) w.plan[i] = gl_plan(w.s[i], dtype, in.o.tile);
        // The general kernel reads planes of float32, a bf16 tile kernel planes of bf16: where a product that is asked for has no tile
        // whose grid fits, the call takes the general kernel for all of them.
        if (dtype == DP_DTYPE_F32 || !in.o.tile || ((!want_dx || w.plan[0].T) && (!planes || w.plan[1].T))) break;
        in.o.tile = in.o.pack_x = in.o.pack_w = false;
    }
    w.plane = in.o.tile ? dtype : DP_DTYPE_F32;
    Carver c = {(char*)base};
    in.carve(c);
    w.ldg = round_up<int64_t>(N, 64);
    w.tx = (int)std::min<int64_t>(64, w.ldg / 4);                 // 16, 32 or 64 column groups of 4
    if (w.tx == 48) w.tx = 64;
    const int64_t cols = ceil_div<int64_t>(w.ldg, w.tx * 4);
    const int ty = 256 / w.tx;
    // about 1024 workgroups, at least 2 rows per row lane
    w.rows = (int)std::max<int64_t>(2 * ty, ceil_div<int64_t>(M, std::max<int64_t>(1, 1024 / cols)));
    w.nblk = (int)ceil_div<int64_t>(std::max<int64_t>(M, 1), w.rows);
    w.dgu = c.take((size_t)2 * M * w.ldg * (w.plane == DP_DTYPE_BF16 ? 2 : 4));
    w.colpart = (float*)c.take(w.nblk > 1 ? (size_t)w.nblk * 2 * w.ldg * 4 : 0);
    for (int i = 0; i < 2; ++i) w.part[i] = (float*)c.take((i ? planes > 0 : want_dx) ? gl_split_bytes(w.s[i], w.plan[i]) : 0);
    w.bytes = c.off;
    return w;
}

template <typename T>
static int gl_forward(GlArgs a, GlIn& in, const GlFwd& w, hipStream_t st) {
    int blocks;
    const GlPack copies = in.copies(true, true, &blocks);
    if (blocks) {
        hipLaunchKernelGGL((k_gated_pack<T>), dim3((unsigned)blocks), dim3(256), 0, st, copies);
        DP_LAUNCH_CHECK("k_gated_pack");
    }
    a.A[0] = in.x;
    a.B[0] = in.wg; a.B[1] = in.wu;
    a.part = w.part;
    return gl_mm<T, GL_FWD>(a, w.s, w.plan, in.o.vec, st);
}

template <typename T>
static int gl_zero(void* p, int64_t n, hipStream_t st) {
    hipLaunchKernelGGL((k_gated_zero<T>), dim3((unsigned)std::min<int64_t>(ceil_div<int64_t>(n, 256), 2048)), dim3(256), 0, st, (T*)p, n);
    DP_LAUNCH_CHECK("k_gated_zero");
    return DP_OK;
}

template <typename T>
static int gl_no_rows(T* dw[2], T* db[2], int N, int K, hipStream_t st) {      // the sums are empty
    int rc;
    for (int z = 0; z < 2; ++z) {
        if (dw[z] && (rc = gl_zero<T>(dw[z], (int64_t)N * K, st))) return rc;
        if (db[z] && (rc = gl_zero<T>(db[z], N, st))) return rc;
    }
    return DP_OK;
}

template <typename T>
static int gl_backward(int dtype, GlIn& in, const GlBwd& w, const void* pre, const GlOp& dh, T* dx, T* dw[2], T* db[2], int act, hipStream_t st) {
    const int64_t M = in.M;
    const int N = in.N, K = in.K, planes = (dw[0] != nullptr) + (dw[1] != nullptr);
    int rc, blocks;
    const GlPack copies = in.copies(planes > 0, dx != nullptr, &blocks);
    const GlDgu e = {pre, dh.p, w.dgu, w.colpart, {db[0], db[1]}, dh.ld, w.ldg, M, N, act, w.tx, w.rows, w.nblk};
    const unsigned across = (unsigned)ceil_div<int64_t>(w.ldg, w.tx * 4);
    const dim3 grid(across, (unsigned)(w.nblk + ceil_div<int64_t>(blocks, across)));
    if (w.plane == dtype) hipLaunchKernelGGL((k_gated_dgu<T, T>), grid, dim3(256), 0, st, e, copies);
    else hipLaunchKernelGGL((k_gated_dgu<T, float>), grid, dim3(256), 0, st, e, copies);
    DP_LAUNCH_CHECK("k_gated_dgu");
    GlColsum cs = {w.colpart, {db[0], db[1]}, w.ldg, w.nblk, N, (db[0] || db[1]) && w.nblk > 1 ? 2 * ceil_div(N, 64) : 0};
    if (cs.n && !w.both) {
        hipLaunchKernelGGL((k_gated_colsum<T>), dim3((unsigned)cs.n), dim3(256), 0, st, cs);
        DP_LAUNCH_CHECK("k_gated_colsum");
    }
    GlArgs a[2];
    memset(a, 0, sizeof a);
    for (int i = 0; i < 2; ++i) {
        a[i].part = w.part[i];
        a[i].A[0] = {w.dgu, w.ldg, w.ldg};
        a[i].A[1] = {w.dgu + (size_t)M * w.ldg * (w.plane == DP_DTYPE_BF16 ? 2 : 4), w.ldg, w.ldg};
        a[i].ldo = K;
    }
    a[0].B[0] = in.wg; a[0].B[1] = in.wu;
    a[0].out[0] = dx;
    a[1].B[0] = in.x;
    a[1].out[0] = dw[0]; a[1].out[1] = dw[1];
    a[1].zfirst = dw[0] ? 0 : 1;
    if (w.both) return gl_both<T>(a, w.s, w.plan, cs, in.o.vec, st);
    if (dx && (rc = gl_mm<T, GL_DX>(a[0], w.s[0], w.plan[0], in.o.vec, st))) return rc;
    if (planes && (rc = gl_mm<T, GL_DW>(a[1], w.s[1], w.plan[1], in.o.vec, st))) return rc;
    return DP_OK;
}

// ---- gradient norm and clipping -----------------------------------------------------------------------------------------
constexpr int64_t GN_MAX_BYTES = (int64_t)1 << 45;
static int gn_blocks(uint32_t chunks, int cap) { return (int)std::max<int64_t>(1, std::min<int64_t>(chunks, cap)); }

static int gn_check(const char* who, int n, void* const* g, const int64_t* numel, const int* dtype, int norm_type, const void* ws, size_t ws_bytes) {
    if (n < 0 || (n > 0 && (!g || !numel || !dtype))) return fail(DP_EINVAL, "%s: bad tensor list", who);
    if (norm_type != DP_NORM_L2 && norm_type != DP_NORM_MAX) return fail(DP_EINVAL, "%s: unknown norm %d", who, norm_type);
    if (!ws || !aligned(ws, 8) || ws_bytes < dp_grad_workspace_bytes(n)) return fail(DP_EWORKSPACE, "%s: workspace of %zu bytes, need %zu (8-byte aligned)", who, ws_bytes, dp_grad_workspace_bytes(n));
    uint64_t total = 0;                                          // keeps the chunk counter inside 32 bits
    for (int i = 0; i < n; ++i) {
        if (dtype[i] != DP_DTYPE_F32 && dtype[i] != DP_DTYPE_BF16) return fail(DP_EINVAL, "%s: tensor %d: unknown dtype %d", who, i, dtype[i]);
        if (numel[i] < 0 || numel[i] > GN_MAX_BYTES || (total += (uint64_t)numel[i] * 4) > GN_MAX_BYTES) return fail(DP_EINVAL, "%s: tensor %d: %lld elements", who, i, (long long)numel[i]);
        if (numel[i] && (!g[i] || !aligned(g[i], dtype[i] == DP_DTYPE_BF16 ? 2 : 4))) return fail(DP_EINVAL, "%s: tensor %d: null or misaligned pointer", who, i);
    }
    return DP_OK;
}

// next table of at most GN_MAX entries from tensor `i` on (which moves on, forwards or backwards)
static bool gn_next(GradTable& t, int& i, int step, int n, void* const* g, const int64_t* numel, const int* dtype) {
    t.n = 0;
    t.chunks = 0;
    for (; i >= 0 && i < n && t.n < GN_MAX; i += step) {
        if (numel[i] == 0) continue;
        const int64_t es = dtype[i] == DP_DTYPE_BF16 ? 2 : 4;
        const uint64_t p = (uint64_t)g[i], base = p & ~(uint64_t)15;
        GradEntry& e = t.e[t.n++];
        e.base = base;
        e.head = (uint16_t)(p - base);
        e.bytes = e.head + (uint64_t)(numel[i] * es);
        e.chunk0 = t.chunks;
        e.bf16 = es == 2;
        t.chunks += (uint32_t)ceil_div<uint64_t>(e.bytes, GN_CHUNK);
    }
    return t.n > 0;
}

static int gn_launches(int n) { return std::max(1, ceil_div(n, GN_MAX)); }
// blocks per launch: eight per CU, fewer where there are so many launches that their partials would be slow to join
static int gn_cap(int n) { return std::max(16, std::min(GN_MAX_BLOCKS, 4096 / gn_launches(n))); }

// partials of all tensors; returns how many there are
static int gn_norm(int n, void* const* g, const int64_t* numel, const int* dtype, int norm_type, double* part, int* nparts, int* launches, hipStream_t st) {
    GradTable t;
    int i = 0;
    *nparts = *launches = 0;
    const int cap = gn_cap(n);
    while (gn_next(t, i, 1, n, g, numel, dtype)) {
        const int grid = gn_blocks(t.chunks, cap);
        hipLaunchKernelGGL(k_grad_norm, dim3(grid), dim3(GN_THREADS), 0, st, t, part + *nparts, norm_type == DP_NORM_MAX);
        DP_LAUNCH_CHECK("k_grad_norm");
        *nparts += grid;
        ++*launches;
    }
    return DP_OK;
}

}  // namespace dp

using namespace dp;

extern "C" {

size_t dp_gated_linear_pre_bytes(int dtype, int64_t M, int N) {
    if ((dtype != DP_DTYPE_F32 && dtype != DP_DTYPE_BF16) || M < 0 || M >= GL_MAX_ROWS || N < 1 || N > GL_MAX_DIM) { fail(DP_EINVAL, "dp_gated_linear_pre_bytes: dtype=%d M=%lld N=%d", dtype, (long long)M, N); return 0; }
    M = std::max<int64_t>(M, 1);
    return (size_t)(dtype == DP_DTYPE_BF16 ? GlPre<bf16_t>::bytes(M, ceil_div(N, 4)) : GlPre<float>::bytes(M, ceil_div(N, 4)));
}

size_t dp_gated_linear_workspace_bytes(int dtype, const void* x, int64_t ldx, const void* w_gate, const void* w_up, int64_t ldw, int64_t M, int N, int K, int grads) {
    if (gl_check("dp_gated_linear_workspace_bytes", dtype, M, N, K, 0)) return 0;
    if (grads < 0 || grads > 15) { fail(DP_EINVAL, "dp_gated_linear_workspace_bytes: grads %d", grads); return 0; }
    if (M == 0) return 256;
    GlIn in = gl_in(dtype, x, ldx, w_gate, w_up, ldw, M, N, K);
    if (grads == DP_GATED_FORWARD) return std::max<size_t>(gl_fwd_carve(dtype, in, nullptr).bytes, 256);
    return std::max<size_t>(gl_bwd_carve(dtype, in, ((grads & DP_GATED_DW_GATE) != 0) + ((grads & DP_GATED_DW_UP) != 0), (grads & DP_GATED_DX) != 0, nullptr).bytes, 256);
}

int dp_gated_linear_plan(int dtype, const void* x, int64_t ldx, const void* w_gate, const void* w_up, int64_t ldw, int64_t M, int N, int K, int grads, int kernel[3]) {
    const int rc = gl_check("dp_gated_linear_plan", dtype, M, N, K, 0);
    if (rc) return rc;
    if (grads < 0 || grads > 15) return fail(DP_EINVAL, "dp_gated_linear_plan: grads %d", grads);
    if (!kernel) return fail(DP_EINVAL, "dp_gated_linear_plan: null pointer");
    kernel[0] = kernel[1] = kernel[2] = -1;
    if (M == 0) return DP_OK;
    auto name = [](int T) { return T == 0 ? 1 : T == GL_ROWS ? 2 : T; };
    GlIn in = gl_in(dtype, x, ldx, w_gate, w_up, ldw, M, N, K);
    if (grads == DP_GATED_FORWARD) {
        kernel[0] = name(gl_fwd_carve(dtype, in, nullptr).plan.T);
        return DP_OK;
    }
    const int planes = ((grads & DP_GATED_DW_GATE) != 0) + ((grads & DP_GATED_DW_UP) != 0);
    const bool dx = (grads & DP_GATED_DX) != 0;
    const GlBwd w = gl_bwd_carve(dtype, in, planes, dx, nullptr);
    if (dx) kernel[0] = name(w.plan[0].T);
    if (planes) kernel[1] = name(w.plan[1].T);
    kernel[2] = w.plane;
    return DP_OK;
}

int dp_gated_linear(int dtype, const void* x, int64_t ldx, const void* w_gate, const void* w_up, int64_t ldw, const void* b_gate, const void* b_up,
                    void* h, int64_t ldh, void* pre, int64_t M, int N, int K, int act, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = gl_check("dp_gated_linear", dtype, M, N, K, act);
    if (rc) return rc;
    if (M == 0) return DP_OK;
    const size_t es = dtype == DP_DTYPE_BF16 ? 2 : 4;
    if (!x || !w_gate || !w_up || !h) return fail(DP_EINVAL, "dp_gated_linear: null pointer");
    if (ldx < K || ldw < K || ldh < N) return fail(DP_EINVAL, "dp_gated_linear: row strides ldx=%lld ldw=%lld ldh=%lld are shorter than a row (K=%d, N=%d)", (long long)ldx, (long long)ldw, (long long)ldh, K, N);
    for (const void* p : {x, w_gate, w_up, b_gate, b_up, (const void*)h})
        if (!aligned(p, es)) return fail(DP_EINVAL, "dp_gated_linear: a pointer is not aligned to its element");
    if (!aligned(pre, 16)) return fail(DP_EINVAL, "dp_gated_linear: pre must be 16-byte aligned");
    GlIn in = gl_in(dtype, x, ldx, w_gate, w_up, ldw, M, N, K);
    const GlFwd w = gl_fwd_carve(dtype, in, workspace);
    const size_t need = std::max<size_t>(w.bytes, 256);
    if (!workspace || workspace_bytes < need || !aligned(workspace, 256)) return fail(DP_EWORKSPACE, "dp_gated_linear: workspace of %zu bytes, need %zu (256-byte aligned)", workspace_bytes, need);
    GlArgs a;
    memset(&a, 0, sizeof a);
    a.out[0] = h; a.ldo = ldh;
    a.pre = pre;
    a.bias[0] = b_gate; a.bias[1] = b_up;
    a.act = act;
    hipStream_t st = (hipStream_t)stream;
    return dtype == DP_DTYPE_BF16 ? gl_forward<bf16_t>(a, in, w, st) : gl_forward<float>(a, in, w, st);
}

int dp_gated_linear_bwd(int dtype, const void* x, int64_t ldx, const void* w_gate, const void* w_up, int64_t ldw, const void* pre, const void* dh, int64_t lddh,
                        void* dx, void* dw_gate, void* dw_up, void* db_gate, void* db_up, int64_t M, int N, int K, int act,
                        void* workspace, size_t workspace_bytes, void* stream) {
    int rc = gl_check("dp_gated_linear_bwd", dtype, M, N, K, act);
    if (rc) return rc;
    const size_t es = dtype == DP_DTYPE_BF16 ? 2 : 4;
    if (M > 0) {
        if (!x || !w_gate || !w_up || !pre || !dh) return fail(DP_EINVAL, "dp_gated_linear_bwd: null pointer");
        if (ldx < K || ldw < K || lddh < N) return fail(DP_EINVAL, "dp_gated_linear_bwd: row strides ldx=%lld ldw=%lld lddh=%lld are shorter than a row (K=%d, N=%d)", (long long)ldx, (long long)ldw, (long long)lddh, K, N);
        if (!aligned(pre, 16)) return fail(DP_EINVAL, "dp_gated_linear_bwd: pre must be 16-byte aligned");
    }
    for (const void* p : {x, w_gate, w_up, dh, (const void*)dx, (const void*)dw_gate, (const void*)dw_up, (const void*)db_gate, (const void*)db_up})
        if (!aligned(p, es)) return fail(DP_EINVAL, "dp_gated_linear_bwd: a pointer is not aligned to its element");
    hipStream_t st = (hipStream_t)stream;
    bf16_t *dw16[2] = {(bf16_t*)dw_gate, (bf16_t*)dw_up}, *db16[2] = {(bf16_t*)db_gate, (bf16_t*)db_up};
    float *dw32[2] = {(float*)dw_gate, (float*)dw_up}, *db32[2] = {(float*)db_gate, (float*)db_up};
    if (M == 0) return dtype == DP_DTYPE_BF16 ? gl_no_rows<bf16_t>(dw16, db16, N, K, st) : gl_no_rows<float>(dw32, db32, N, K, st);
    GlIn in = gl_in(dtype, x, ldx, w_gate, w_up, ldw, M, N, K);
    const GlBwd w = gl_bwd_carve(dtype, in, (dw_gate != nullptr) + (dw_up != nullptr), dx != nullptr, workspace);
    const size_t need = std::max<size_t>(w.bytes, 256);
    if (!workspace || workspace_bytes < need || !aligned(workspace, 256)) return fail(DP_EWORKSPACE, "dp_gated_linear_bwd: workspace of %zu bytes, need %zu (256-byte aligned)", workspace_bytes, need);
    const GlOp od = {dh, lddh, N};
    return dtype == DP_DTYPE_BF16 ? gl_backward<bf16_t>(dtype, in, w, pre, od, (bf16_t*)dx, dw16, db16, act, st) : gl_backward<float>(dtype, in, w, pre, od, (float*)dx, dw32, db32, act, st);
}

size_t dp_grad_workspace_bytes(int n) { return n < 0 ? 0 : (size_t)(gn_cap(n) * gn_launches(n) + 1) * sizeof(double); }

int dp_grad_norm(int n, const void* const* g, const int64_t* numel, const int* dtype, int norm_type, float* norm, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = gn_check("dp_grad_norm", n, (void* const*)g, numel, dtype, norm_type, workspace, workspace_bytes);
    if (rc) return rc;
    if (!norm) return fail(DP_EINVAL, "dp_grad_norm: null pointer");
    hipStream_t st = (hipStream_t)stream;
    int nparts, launches;
    if ((rc = gn_norm(n, (void* const*)g, numel, dtype, norm_type, (double*)workspace, &nparts, &launches, st))) return rc;
    hipLaunchKernelGGL(k_grad_total, dim3(1), dim3(GN_THREADS), 0, st, (const double*)workspace, nparts, norm_type == DP_NORM_MAX, norm);
    DP_LAUNCH_CHECK("k_grad_total");
    return DP_OK;
}

int dp_clip_grads(int n, void* const* g, const int64_t* numel, const int* dtype, int norm_type, double limit, float* norm, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = gn_check("dp_clip_grads", n, g, numel, dtype, norm_type, workspace, workspace_bytes);
    if (rc) return rc;
    if (!norm) return fail(DP_EINVAL, "dp_clip_grads: null pointer");
    if (!(limit >= 0.0)) return fail(DP_EINVAL, "dp_clip_grads: the limit has to be a number of at least 0");
    try {                                                        // no two tensors may share memory: they are scaled in place
        std::vector<std::pair<uint64_t, uint64_t>> span;
        span.reserve(n);
        for (int i = 0; i < n; ++i)
            if (numel[i]) span.push_back({(uint64_t)g[i], (uint64_t)g[i] + (uint64_t)numel[i] * (dtype[i] == DP_DTYPE_BF16 ? 2 : 4)});
        if (!std::is_sorted(span.begin(), span.end())) std::sort(span.begin(), span.end());
        for (size_t i = 1; i < span.size(); ++i)
            if (span[i].first < span[i - 1].second) return fail(DP_EINVAL, "dp_clip_grads: two of the tensors share memory");
    } catch (const std::bad_alloc&) {
        return fail(DP_EINVAL, "dp_clip_grads: out of host memory for %d tensors", n);
    }
    hipStream_t st = (hipStream_t)stream;
    const int inf = norm_type == DP_NORM_MAX;
    const double* part = (const double*)workspace;
    int nparts, launches;
    if ((rc = gn_norm(n, g, numel, dtype, norm_type, (double*)workspace, &nparts, &launches, st))) return rc;
    GradTable t;
    int i = n - 1;
    if (launches == 0) {
        hipLaunchKernelGGL(k_grad_total, dim3(1), dim3(GN_THREADS), 0, st, part, 0, inf, norm);
        DP_LAUNCH_CHECK("k_grad_total");
    }
    for (int k = 0; gn_next(t, i, -1, n, g, numel, dtype); ++k) {
        hipLaunchKernelGGL(k_grad_clip, dim3(gn_blocks(t.chunks, GN_MAX_BLOCKS)), dim3(GN_THREADS), 0, st, t, part, nparts, inf, limit, k == 0 ? norm : nullptr);
        DP_LAUNCH_CHECK("k_grad_clip");
    }
    return DP_OK;
}

}  // extern "C"
