// Operators beside the sampler: the gated projection with its backward (dp_gated.h) and the global gradient norm with
// clipping (dp_grads.h).  Host side and C ABI (include/diffputer.h); linked into libdiffputer_hip.so.
#include <math.h>
#include <string.h>

#include <algorithm>
#include <new>
#include <vector>

#include "dp_gated.h"
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

// How a product is cut: tiles over C and slices of the contraction.  A launch with few tiles leaves most of the 256 CUs
// idle, so the contraction is cut until there are about two workgroups per CU, as long as a slice keeps 8 K-tiles.
struct GlCut { int kt_per, splits; };
static GlCut gl_cut(int64_t tiles, int64_t nk, int64_t part_bytes) {
    int64_t s = std::min<int64_t>({512 / std::max<int64_t>(tiles, 1), nk / 8, (int64_t)(64 << 20) / std::max<int64_t>(part_bytes, 1), 64});
    if (s <= 1) return {(int)nk, 1};
    const int64_t per = ceil_div<int64_t>(nk, s);
    return {(int)per, (int)ceil_div<int64_t>(nk, per)};
}

struct GlShape { int mode; int64_t I; int J; int64_t C; int planes; };
static int64_t gl_ldp(int J) { return round_up<int64_t>(J, 4); }
static size_t gl_part_bytes(const GlShape& s) { return (size_t)2 * s.I * gl_ldp(s.J) * 4; }       // one slice: two planes
static GlCut gl_plan(const GlShape& s) {
    const int64_t tiles = ceil_div<int64_t>(s.I, GG_T) * ceil_div<int64_t>(s.J, s.mode == GL_FWD ? GG_T / 2 : GG_T) * s.planes;
    return gl_cut(tiles, ceil_div<int64_t>(s.C, GG_K) * (s.mode == GL_DX ? 2 : 1), gl_part_bytes(s));
}
static size_t gl_split_bytes(const GlShape& s) {
    const GlCut c = gl_plan(s);
    return c.splits > 1 ? gl_part_bytes(s) * c.splits : 0;
}

template <typename T, int MODE>
static int gl_mm(GlArgs a, const GlShape& s, hipStream_t st) {
    const GlCut c = gl_plan(s);
    a.I = s.I; a.J = s.J; a.C = s.C; a.kt_per = c.kt_per; a.splits = c.splits; a.ldp = gl_ldp(s.J);
    const int64_t gx = ceil_div<int64_t>(s.I, GG_T), gy = ceil_div<int64_t>(s.J, MODE == GL_FWD ? GG_T / 2 : GG_T);
    hipLaunchKernelGGL((k_gated_mm<T, MODE>), dim3((unsigned)gx, (unsigned)gy, (unsigned)(s.planes * c.splits)), dim3(256), 0, st, a);
    DP_LAUNCH_CHECK("k_gated_mm");
    if (c.splits > 1) {
        const int64_t n = s.I * s.planes * ceil_div<int64_t>(s.J, 4);
        const unsigned grid = (unsigned)std::min<int64_t>(ceil_div<int64_t>(n, 256), 4096);
        hipLaunchKernelGGL((k_gated_join<T, MODE>), dim3(grid), dim3(256), 0, st, a, s.planes);
        DP_LAUNCH_CHECK("k_gated_join");
    }
    return DP_OK;
}

// backward workspace: the two planes dg, du; partial column sums; partial products (dx and dW use the same bytes in turn)
struct GlBwd {
    char* dgu;
    float *colpart, *part;
    int64_t ldg;
    int tx, rows, nblk;
    size_t bytes;
};
static GlBwd gl_bwd_carve(int dtype, int64_t M, int N, int K, void* base) {
    GlBwd w;
    size_t off = 0;
    auto take = [&](size_t n) { const size_t o = off; off += round_up<size_t>(n, 256); return base ? (char*)base + o : (char*)nullptr; };
    w.ldg = round_up<int64_t>(N, 64);
    w.tx = (int)std::min<int64_t>(64, w.ldg / 4);                 // 16, 32, 48 or 64 column groups of 4
    if (w.tx == 48) w.tx = 64;
    const int64_t cols = ceil_div<int64_t>(w.ldg, w.tx * 4);
    const int ty = 256 / w.tx;
    // about 2048 workgroups, at least 4 rows per row lane
    w.rows = (int)std::max<int64_t>(4 * ty, ceil_div<int64_t>(M, std::max<int64_t>(1, 2048 / cols)));
    w.nblk = (int)ceil_div<int64_t>(std::max<int64_t>(M, 1), w.rows);
    w.dgu = take((size_t)2 * M * w.ldg * (dtype == DP_DTYPE_BF16 ? 2 : 4));
    w.colpart = (float*)take((size_t)w.nblk * 2 * w.ldg * 4);
    w.part = (float*)take(std::max(gl_split_bytes({GL_DX, M, K, N, 1}), gl_split_bytes({GL_DW, N, K, M, 2})));
    w.bytes = off;
    return w;
}

template <typename T>
static int gl_forward(const GlArgs& a, int64_t M, int N, int K, hipStream_t st) {
    return gl_mm<T, GL_FWD>(a, {GL_FWD, M, N, K, 1}, st);
}

template <typename T>
static int gl_zero(void* p, int64_t n, hipStream_t st) {
    hipLaunchKernelGGL((k_gated_zero<T>), dim3((unsigned)std::min<int64_t>(ceil_div<int64_t>(n, 256), 2048)), dim3(256), 0, st, (T*)p, n);
    DP_LAUNCH_CHECK("k_gated_zero");
    return DP_OK;
}

template <typename T>
static int gl_backward(int dtype, const GlOp& x, const GlOp& wg, const GlOp& wu, const float* pre, const GlOp& dh, T* dx, T* dw[2], T* db[2],
                       int64_t M, int N, int K, int act, void* ws, hipStream_t st) {
    int rc;
    if (M == 0) {                                                // no rows: the sums are empty
        for (int z = 0; z < 2; ++z) {
            if (dw[z] && (rc = gl_zero<T>(dw[z], (int64_t)N * K, st))) return rc;
            if (db[z] && (rc = gl_zero<T>(db[z], N, st))) return rc;
        }
        return DP_OK;
    }
    const GlBwd w = gl_bwd_carve(dtype, M, N, K, ws);
    T* const dgu = (T*)w.dgu;
    const bool bias = db[0] || db[1];
    hipLaunchKernelGGL((k_gated_dgu<T>), dim3((unsigned)ceil_div<int64_t>(w.ldg, w.tx * 4), (unsigned)w.nblk), dim3(256), 0, st, pre, gl_ldp(N),
                       (const T*)dh.p, dh.ld, dgu, w.ldg, bias ? w.colpart : (float*)nullptr, M, N, act, w.tx, w.rows);
    DP_LAUNCH_CHECK("k_gated_dgu");
    if (bias) {
        hipLaunchKernelGGL((k_gated_colsum<T>), dim3((unsigned)ceil_div(N, 64), 2), dim3(256), 0, st, w.colpart, w.nblk, w.ldg, db[0], db[1], N);
        DP_LAUNCH_CHECK("k_gated_colsum");
    }
    GlArgs a;
    memset(&a, 0, sizeof a);
    a.part = w.part;
    a.A[0] = {dgu, w.ldg};
    a.A[1] = {dgu + (size_t)M * w.ldg, w.ldg};
    if (dx) {
        a.B[0] = wg; a.B[1] = wu;
        a.out[0] = dx; a.ldo = K;
        if ((rc = gl_mm<T, GL_DX>(a, {GL_DX, M, K, N, 1}, st))) return rc;
    }
    if (dw[0] || dw[1]) {
        a.B[0] = x;
        a.out[0] = dw[0]; a.out[1] = dw[1]; a.ldo = K;
        a.zfirst = dw[0] ? 0 : 1;
        if ((rc = gl_mm<T, GL_DW>(a, {GL_DW, N, K, M, dw[0] && dw[1] ? 2 : 1}, st))) return rc;
    }
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

// next table of at most GN_MAX entries from tensor `i` on (which moves on)
static bool gn_next(GradTable& t, int& i, int n, void* const* g, const int64_t* numel, const int* dtype) {
    t.n = 0;
    t.chunks = 0;
    for (; i < n && t.n < GN_MAX; ++i) {
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
static int gn_cap(int n) { return std::max(1, GN_MAX_BLOCKS / ceil_div(std::max(n, 1), GN_MAX)); }     // blocks per launch

// partials of all tensors; returns how many there are
static int gn_norm(int n, void* const* g, const int64_t* numel, const int* dtype, int norm_type, double* part, int* nparts, int* launches, hipStream_t st) {
    GradTable t;
    int i = 0;
    *nparts = *launches = 0;
    const int cap = gn_cap(n);
    while (gn_next(t, i, n, g, numel, dtype)) {
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

size_t dp_gated_linear_pre_bytes(int64_t M, int N) {
    if (M < 0 || M >= GL_MAX_ROWS || N < 1 || N > GL_MAX_DIM) { fail(DP_EINVAL, "dp_gated_linear_pre_bytes: M=%lld N=%d", (long long)M, N); return 0; }
    return (size_t)std::max<int64_t>(M, 1) * 2 * gl_ldp(N) * 4;
}

size_t dp_gated_linear_workspace_bytes(int dtype, int64_t M, int N, int K, int backward) {
    if (gl_check("dp_gated_linear_workspace_bytes", dtype, M, N, K, 0)) return 0;
    const size_t need = M == 0 ? 0 : backward ? gl_bwd_carve(dtype, M, N, K, nullptr).bytes : gl_split_bytes({GL_FWD, M, N, K, 1});
    return std::max<size_t>(need, 256);
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
    const size_t need = dp_gated_linear_workspace_bytes(dtype, M, N, K, 0);
    if (!workspace || workspace_bytes < need || !aligned(workspace, 256)) return fail(DP_EWORKSPACE, "dp_gated_linear: workspace of %zu bytes, need %zu (256-byte aligned)", workspace_bytes, need);
    GlArgs a;
    memset(&a, 0, sizeof a);
    a.A[0] = {x, ldx};
    a.B[0] = {w_gate, ldw};
    a.B[1] = {w_up, ldw};
    a.out[0] = h; a.ldo = ldh;
    a.part = (float*)workspace;
    a.pre = (float*)pre; a.ldpre = gl_ldp(N);
    a.bias[0] = b_gate; a.bias[1] = b_up;
    a.act = act;
    hipStream_t st = (hipStream_t)stream;
    return dtype == DP_DTYPE_BF16 ? gl_forward<bf16_t>(a, M, N, K, st) : gl_forward<float>(a, M, N, K, st);
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
        const size_t need = dp_gated_linear_workspace_bytes(dtype, M, N, K, 1);
        if (!workspace || workspace_bytes < need || !aligned(workspace, 256)) return fail(DP_EWORKSPACE, "dp_gated_linear_bwd: workspace of %zu bytes, need %zu (256-byte aligned)", workspace_bytes, need);
    }
    for (const void* p : {x, w_gate, w_up, dh, (const void*)dx, (const void*)dw_gate, (const void*)dw_up, (const void*)db_gate, (const void*)db_up})
        if (!aligned(p, es)) return fail(DP_EINVAL, "dp_gated_linear_bwd: a pointer is not aligned to its element");
    const GlOp ox = {x, ldx}, og = {w_gate, ldw}, ou = {w_up, ldw}, od = {dh, lddh};
    hipStream_t st = (hipStream_t)stream;
    if (dtype == DP_DTYPE_BF16) {
        bf16_t *dw[2] = {(bf16_t*)dw_gate, (bf16_t*)dw_up}, *db[2] = {(bf16_t*)db_gate, (bf16_t*)db_up};
        return gl_backward<bf16_t>(dtype, ox, og, ou, (const float*)pre, od, (bf16_t*)dx, dw, db, M, N, K, act, workspace, st);
    }
    float *dw[2] = {(float*)dw_gate, (float*)dw_up}, *db[2] = {(float*)db_gate, (float*)db_up};
    return gl_backward<float>(dtype, ox, og, ou, (const float*)pre, od, (float*)dx, dw, db, M, N, K, act, workspace, st);
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

int dp_clip_grads(int n, void* const* g, const int64_t* numel, const int* dtype, int norm_type, float limit, float* norm, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = gn_check("dp_clip_grads", n, g, numel, dtype, norm_type, workspace, workspace_bytes);
    if (rc) return rc;
    if (!norm) return fail(DP_EINVAL, "dp_clip_grads: null pointer");
    if (!(limit >= 0.0f)) return fail(DP_EINVAL, "dp_clip_grads: the limit has to be a number of at least 0");
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
    int i = 0;
    if (launches == 0) {
        hipLaunchKernelGGL(k_grad_total, dim3(1), dim3(GN_THREADS), 0, st, part, 0, inf, norm);
        DP_LAUNCH_CHECK("k_grad_total");
    }
    for (int k = 0; gn_next(t, i, n, g, numel, dtype); ++k) {
        hipLaunchKernelGGL(k_grad_clip, dim3(gn_blocks(t.chunks, 2048)), dim3(GN_THREADS), 0, st, t, part, nparts, inf, limit, k == 0 ? norm : nullptr);
        DP_LAUNCH_CHECK("k_grad_clip");
    }
    return DP_OK;
}

}  // extern "C"
