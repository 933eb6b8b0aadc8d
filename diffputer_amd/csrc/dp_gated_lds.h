// What the tile kernels of the gated projection share: their arguments, the order of the tiles, and loads from a bounded buffer
// straight into LDS.
#pragma once
#include "dp_gated.h"
#include "dp_gemm_bf16.h"

namespace dp {

typedef __attribute__((ext_vector_type(4))) short bf16x4;

struct GtArgs {
    GlArgs g;
    int nti, ntj;              // tiles along I and J
    int group;                 // tile rows that are walked together (shared B panels stay in the XCD's L2)
};

__device__ __forceinline__ unsigned gt_lds(const void* p) { return (unsigned)(size_t)(DP_LDS_AS const char*)p; }   // LDS byte address

#define GT_VMCNT(n) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(n) : "memory")

// byte range [p, end) as a buffer; reads behind it return 0
__device__ __forceinline__ __amdgpu_buffer_rsrc_t gt_buffer(const char* p, const char* end) {
    const int64_t n = end - p;
    const int hi = (int)(n >> 32);
    const unsigned lo = (unsigned)n;
    const unsigned bytes = hi < 0 ? 0u : hi > 0 || lo > 0x7fffffffu ? 0x7fffffffu : lo;
    return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, (int)bytes, 0x00027000);
}

// EL bytes per lane from the buffer's byte `off` on into LDS, lane after lane from `dst` on
template <int EL> __device__ __forceinline__ void gt_load(__amdgpu_buffer_rsrc_t buf, char* dst, unsigned off) {
    if constexpr (EL == 16) __builtin_amdgcn_raw_ptr_buffer_load_lds(buf, (DP_LDS_AS void*)dst, 16, (int)off, 0, 0, 0);
    else __builtin_amdgcn_raw_ptr_buffer_load_lds(buf, (DP_LDS_AS void*)dst, 4, (int)off, 0, 0, 0);
}

// workgroup -> slice, and tile -> (plane, row, column): groups of q.group tile rows, column by column within a group
template <int MODE> __device__ __forceinline__ void gt_tile(const GtArgs& q, int b, int count, int& slice, int& plane, int& ti, int& tj) {
    const int t = xcd_remap(b, count), tiles = count / q.g.splits, tile = t % tiles;
    slice = __builtin_amdgcn_readfirstlane(t / tiles);
    const int per_plane = q.nti * q.ntj;
    plane = MODE == GL_DW ? q.g.zfirst + __builtin_amdgcn_readfirstlane(tile / per_plane) : 0;
    const int tp = tile % per_plane, gsz = q.group * q.ntj, grp = tp / gsz, in = tp - grp * gsz;
    const int rows_here = min(q.group, q.nti - grp * q.group);
    ti = __builtin_amdgcn_readfirstlane(grp * q.group + in % rows_here);
    tj = __builtin_amdgcn_readfirstlane(in / rows_here);
}

// copies of up to three matrices whose rows are not 16-byte aligned: [rows][ldd], columns C..ldd - 1 zero
struct GlPack {
    struct { const bf16_t* src; bf16_t* dst; int64_t ld, rows; } m[3];
    int64_t ldd;
    int C, n;
};
__global__ __launch_bounds__(256) static void k_gated_pack(GlPack p) {
    const int64_t per = p.ldd / 8;
    int64_t total = 0;
    for (int i = 0; i < p.n; ++i) total += p.m[i].rows * per;
    for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < total; t += (int64_t)gridDim.x * 256) {
        int64_t r = t / per;
        const int64_t c = (t - r * per) * 8;
        int i = 0;
        while (r >= p.m[i].rows) r -= p.m[i++].rows;
        const bf16_t* const src = p.m[i].src + r * p.m[i].ld + c;
        bf16x8 v;
        if (c + 8 <= p.C) __builtin_memcpy(&v, src, 16);
        else
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = c + e < p.C ? (short)src[e] : (short)0;
        *(bf16x8*)(p.m[i].dst + r * p.ldd + c) = v;
    }
}

}  // namespace dp
