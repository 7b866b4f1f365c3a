// Shared by the sequence operators (rotary.hip, layer_norm.hip, decay_attn.hip): (B, T, J, H, D) views and vectors of VE values.
#pragma once
#include "common.h"

// VE consecutive elements <-> fp32 registers, one access of VE * sizeof(T) bytes wherever they start (this hardware's vector accesses of
// global memory need no alignment of their own)
template <typename V> __device__ __forceinline__ V ld_any(const void* p) { V v; __builtin_memcpy(&v, p, sizeof(V)); return v; }
template <typename V> __device__ __forceinline__ void st_any(void* p, const V& v) { __builtin_memcpy(p, &v, sizeof(V)); }
template <int VE> __device__ __forceinline__ void ldv(float (&v)[VE], const float* p) {
    if constexpr (VE == 4) {
        const float4 u = ld_any<float4>(p);
        v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
    } else if constexpr (VE == 2) {
        const float2 u = ld_any<float2>(p);
        v[0] = u.x; v[1] = u.y;
    } else {
        static_assert(VE == 1, "1, 2 or 4 values of fp32");
        v[0] = *p;
    }
}
template <int VE> __device__ __forceinline__ void ldv(float (&v)[VE], const bf16_t* p) {
    if constexpr (VE == 8) {
        const uint4 u = ld_any<uint4>(p);
        h16x2_unpack(u.x, v[0], v[1]); h16x2_unpack(u.y, v[2], v[3]); h16x2_unpack(u.z, v[4], v[5]); h16x2_unpack(u.w, v[6], v[7]);
    } else if constexpr (VE == 4) {
        const uint2 u = ld_any<uint2>(p);
        h16x2_unpack(u.x, v[0], v[1]); h16x2_unpack(u.y, v[2], v[3]);
    } else if constexpr (VE == 2) {
        h16x2_unpack(ld_any<uint32_t>(p), v[0], v[1]);
    } else {
        static_assert(VE == 1, "1, 2, 4 or 8 values of 16 bits");
        v[0] = bf2f(*p);
    }
}
template <int VE> __device__ __forceinline__ void stv(float* p, const float (&v)[VE]) {
    if constexpr (VE == 4) st_any<float4>(p, make_float4(v[0], v[1], v[2], v[3]));
    else if constexpr (VE == 2) st_any<float2>(p, make_float2(v[0], v[1]));
    else *p = v[0];
}
template <int VE> __device__ __forceinline__ void stv(bf16_t* p, const float (&v)[VE]) {
    if constexpr (VE == 8) st_any<uint4>(p, make_uint4(pack_h16x2(v[0], v[1]), pack_h16x2(v[2], v[3]), pack_h16x2(v[4], v[5]), pack_h16x2(v[6], v[7])));
    else if constexpr (VE == 4) st_any<uint2>(p, make_uint2(pack_h16x2(v[0], v[1]), pack_h16x2(v[2], v[3])));
    else if constexpr (VE == 2) st_any<uint32_t>(p, pack_h16x2(v[0], v[1]));
    else *p = f2bf(v[0]);
}

// element (b, t, j, h, 0) of a view
__device__ __forceinline__ long seq_at(const gast_seq& s, long b, long t, long j, long h) { return b * s.b + t * s.t + j * s.j + h * s.h; }

// the widest vector (in elements, at most `most`) that every row of a view starts on
static inline int seq_align(const gast_seq& s, int elem_bytes, int most) {
    int ve = most;
    while (ve > 1 && (((uintptr_t)s.p % (uintptr_t)(ve * elem_bytes)) || s.b % ve || s.t % ve || s.j % ve || s.h % ve)) ve >>= 1;
    return ve;
}
