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
    int wgs;                   // tiles x slices x planes
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

// A buffer's descriptor in four scalar registers: base, bytes, type.  Kept whole so that walking on is an addition in place.
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ u32x4 gl_buffer(const char* base) { return (u32x4){(unsigned)(uint64_t)base, (unsigned)((uint64_t)base >> 32) & 0xffffu, 0u, 0x00027000u}; }
__device__ __forceinline__ void gl_advance(u32x4& rs, int64_t bytes) {     // addresses have 48 bits: nothing carries into the upper half of the second word
    const uint64_t b = ((uint64_t)rs[1] << 32 | rs[0]) + (uint64_t)bytes;
    rs[0] = (unsigned)b;
    rs[1] = (unsigned)(b >> 32);
}
// 16 bytes per lane from byte `off` of the buffer to LDS byte `lds` on; zeros where a lane is outside.  In assembly so that the
// compiler does not wait for loads in flight before every LDS read (there is no register result: the waits for what arrives in
// LDS are the counted ones below).
__device__ __forceinline__ void gl_load_lds(u32x4 rs, unsigned off, unsigned lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(off), "s"(rs) : "memory");
}
__device__ __forceinline__ unsigned gl_clip(int64_t n) { return n <= 0 ? 0u : n > 0x7fffffff ? 0x7fffffffu : (unsigned)n; }

    // all but the newest `n` loads into LDS and every LDS read of this wave done, in all waves (a wait that the compiler knows, so
    // that it does not wait again for the fragments)
#define GL_SYNC(n)                                                                                              \
    do {                                                                                                        \
        asm volatile("" ::: "memory");                                                                          \
        __builtin_amdgcn_s_waitcnt(((n) & 15) | (((n) >> 4) << 14) | (7 << 4));                                 \
        __builtin_amdgcn_s_barrier();                                                                           \
        asm volatile("" ::: "memory");                                                                          \
    } while (0)

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

}  // namespace dp
