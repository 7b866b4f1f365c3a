// Causal linear attention with a decay for each head, forward, backward and one token at a time.
//
//   S_t = lambda S_(t-1) + k_t v_t',   o_t = scale q_t' S_t,   lambda = exp(log_decay)
//
// Every pass is one recurrence in three roles,   out_i = oscale * a_i' X_i,   X_i = lambda X_(i-1) + bscale * b_i c_i' :
//   o   a = q,  b = k,  c = v    forward in time            dq  a = do, b = v,  c = k    forward in time (X = S')
//   dv  a = k,  b = q,  c = do   backward in time           dk  a = v,  b = do, c = q    backward in time (X = the transposed one of dv)
// Forward in time the carry is decayed before it is used (o_t sees lambda S_(t-1)), backward in time the gradient of the last state is
// used as it is and the decay follows: d state = lambda * (the recurrence's end).
#include <algorithm>
#include <atomic>
#include <type_traits>
#include "seq_common.h"

namespace {

// ------------------------------------------------------------------------------------------------ whole sequences, by chunks of 32 tokens
// Inside a chunk the recurrence is products of matrices (i, j tokens of the chunk, X the state before it, n its tokens):
//   out_i = sum_j [j before or at i] lambda^|i-j| (a_i b_j) c_j + lambda^(steps to i) a_i X,     X' = lambda^n X + sum_j lambda^(steps from j) b_j c_j'
// A wave owns 32 columns of X (and of c and out) and keeps them in accumulators; the waves of a block share a, b, c of the chunk in LDS.
// The 32x32 matrix instructions leave result rows 8 (r / 4) + 4 (lane / 32) + r % 4 in register r and the column in lane % 32, and take
// operands with the row (or column) in lane % 32 and any order of the summed index that both sides agree on.  Every operand here is held in
// that same order -- 16 values a lane for 32 summed indexes -- so scores (summed over d, then over j) and states (made by a sum over j, then
// summed over d) go from one product into the next without leaving their registers.  Only tokens pass through LDS, b and c turned on the way.
// Scores are computed by every wave for itself: at 128 channels 8 of a wave's 52 matrix instructions a chunk (16 bits), against a barrier and an
// LDS round trip.
//
// Arithmetic.  fp32: fp32 matrix instructions.  16 bits: products of stored values are exact in fp32; scores and states, which are fp32,
// meet 16-bit operands as three bf16 parts that hold all of their 24 bits; in the binary16 flavour the stored operand is split into two bf16
// parts as well (exactly; binary16 parts of a state would overflow at 65504).  So the 16-bit types compute as fp32 does, and only results are
// rounded to the type.  Two parts (2^-17 of each score and state) are faster, 15 - 17 % with 128 channels a head (512 heads, 1024 tokens, bf16: 154
// against 183 us, with gradients 585 against 705), 5 - 12 % with 64, but what is left of terms that nearly cancel is then off by 2^-17 of the terms.
//
// What bounds it, on a full card (two waves a SIMD, 1024 tokens, without gradients; a copy of the same bytes takes 112 us at 16 bits, 224 fp32):
//   bf16  1024 heads of 64: 136 us, memory (3.9 TB/s); 512 of 128: 183 us, issue (823 vector, 62 matrix and 54 LDS instructions a wave and chunk:
//         the splits into parts are most of them)
//   fp16  64: 181 us, 128: 257 us: issue, both sides of a product are split
//   fp32  2048 heads of 32: 314 us and 1024 of 64: 309 us, memory and LDS; 512 of 128: 480 us, of which 355 are matrix instructions (208 of 64
//         cycles a wave and chunk)
// 16 heads of 128 channels and 32768 tokens (bf16) are cut into 32 segments: 80 us of sums, 14 of joining them, 177 of outputs.
constexpr int CT = 32;               // tokens of a chunk
constexpr int TS = CT + 4;           // row pitch of the turned tiles (elements): rows start 18 / 36 banks apart, no two of a read collide

template <typename T> struct Frag;
template <> struct Frag<float> { float x[16]; };
template <> struct Frag<bf16_t> { uint4 x[2]; };
struct Parts { uint4 x[3][2]; };                       // x = x[0] + x[1] + x[2], bf16 parts that hold all of its 24 bits

// 16 values of a row of an LDS tile: elements 8 q + 4 (lane / 32) + 0 .. 3, q = 0 .. 3
__device__ __forceinline__ Frag<float> ld_frag(const float* row, int half) {
    Frag<float> f;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const float4 v = *(const float4*)(row + 8 * q + 4 * half);
        f.x[4 * q] = v.x; f.x[4 * q + 1] = v.y; f.x[4 * q + 2] = v.z; f.x[4 * q + 3] = v.w;
    }
    return f;
}
__device__ __forceinline__ Frag<bf16_t> ld_frag(const bf16_t* row, int half) {
    Frag<bf16_t> f;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const uint2 a = *(const uint2*)(row + 16 * q + 4 * half), b = *(const uint2*)(row + 16 * q + 8 + 4 * half);
        f.x[q] = make_uint4(a.x, a.y, b.x, b.y);
    }
    return f;
}
// 16 values of a column: of a tile's rows (fp32, RS apart; p is the column's first value), or of a turned tile (16 bits; p is the column's row)
template <int RS> __device__ __forceinline__ Frag<float> ld_column(const float* p, int half) {
    Frag<float> f;
#pragma unroll
    for (int i = 0; i < 16; ++i) f.x[i] = p[(8 * (i >> 2) + 4 * half + (i & 3)) * RS];
    return f;
}
template <int RS> __device__ __forceinline__ Frag<bf16_t> ld_column(const bf16_t* p, int half) { return ld_frag(p, half); }
__device__ __forceinline__ void unpack(const Frag<float>& f, float (&v)[16]) {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = f.x[i];
}
__device__ __forceinline__ void unpack(const Frag<bf16_t>& f, float (&v)[16]) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        h16x2_unpack(f.x[q].x, v[8 * q], v[8 * q + 1]); h16x2_unpack(f.x[q].y, v[8 * q + 2], v[8 * q + 3]);
        h16x2_unpack(f.x[q].z, v[8 * q + 4], v[8 * q + 5]); h16x2_unpack(f.x[q].w, v[8 * q + 6], v[8 * q + 7]);
    }
}
// two bf16 of two values, and what they leave of them (exact).  The empty statement keeps hipcc from converting the low half a second time.
__device__ __forceinline__ uint32_t take2(float& a, float& b) {
    uint32_t u = pack_bf16x2(a, b);
    asm("" : "+v"(u));
    a -= __uint_as_float(u << 16);
    b -= __uint_as_float(u & 0xffff0000u);
    return u;
}
template <typename V> __device__ __forceinline__ Parts parts16(const V& v) {
    Parts s;
    float w[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i] = v[i];
#pragma unroll
    for (int k = 0; k < 3; ++k)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            uint32_t u[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) u[e] = take2(w[8 * q + 2 * e], w[8 * q + 2 * e + 1]);
            s.x[k][q] = make_uint4(u[0], u[1], u[2], u[3]);
        }
    return s;
}

// c += A B over 32 summed indexes, both as stored
__device__ __forceinline__ void mma(f32x16& c, const Frag<bf16_t>& a, const Frag<bf16_t>& b) {
    c = mfma_h16(a.x[0], b.x[0], c);
    c = mfma_h16(a.x[1], b.x[1], c);
}
__device__ __forceinline__ void mma(f32x16& c, const Frag<float>& a, const Frag<float>& b) {
#pragma unroll
    for (int i = 0; i < 16; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.x[i], b.x[i], c, 0, 0, 0);
}
// c += A B with one side in fp32 (16 values in the same order): rows from the fp32 side (mma_fs) or from the stored one (mma_sf)
template <typename V> __device__ __forceinline__ void mma_fs(f32x16& c, const V& a, const Frag<float>& b) {
#pragma unroll
    for (int i = 0; i < 16; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b.x[i], c, 0, 0, 0);
}
template <typename V> __device__ __forceinline__ void mma_sf(f32x16& c, const Frag<float>& a, const V& b) {
#pragma unroll
    for (int i = 0; i < 16; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.x[i], b[i], c, 0, 0, 0);
}
#ifdef GAST_H16_F16
// a binary16 value is two bf16 parts (exactly)
struct Stored {
    uint4 hi[2], lo[2];
    __device__ __forceinline__ explicit Stored(const Frag<bf16_t>& f) {
        float v[16];
        unpack(f, v);
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            uint32_t h[4], l[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                h[e] = take2(v[8 * q + 2 * e], v[8 * q + 2 * e + 1]);
                l[e] = pack_bf16x2(v[8 * q + 2 * e], v[8 * q + 2 * e + 1]);
            }
            hi[q] = make_uint4(h[0], h[1], h[2], h[3]);
            lo[q] = make_uint4(l[0], l[1], l[2], l[3]);
        }
    }
};
#endif
// (the product of the smallest parts of both sides, 2^-24 of a term, is left out)
__device__ __forceinline__ void mma_fs(f32x16& c, const Parts& a, const Frag<bf16_t>& b) {
#ifdef GAST_H16_F16
    const Stored p(b);
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        c = mfma_pair<1>(a.x[2][q], p.hi[q], c);
        c = mfma_pair<1>(a.x[1][q], p.lo[q], c);
        c = mfma_pair<1>(a.x[1][q], p.hi[q], c);
        c = mfma_pair<1>(a.x[0][q], p.lo[q], c);
        c = mfma_pair<1>(a.x[0][q], p.hi[q], c);
    }
#else
#pragma unroll
    for (int k = 2; k >= 0; --k)
#pragma unroll
        for (int q = 0; q < 2; ++q) c = mfma_pair<1>(a.x[k][q], b.x[q], c);
#endif
}
__device__ __forceinline__ void mma_sf(f32x16& c, const Frag<bf16_t>& a, const Parts& b) {
#ifdef GAST_H16_F16
    const Stored p(a);
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        c = mfma_pair<1>(p.hi[q], b.x[2][q], c);
        c = mfma_pair<1>(p.lo[q], b.x[1][q], c);
        c = mfma_pair<1>(p.hi[q], b.x[1][q], c);
        c = mfma_pair<1>(p.lo[q], b.x[0][q], c);
        c = mfma_pair<1>(p.hi[q], b.x[0][q], c);
    }
#else
#pragma unroll
    for (int k = 2; k >= 0; --k)
#pragma unroll
        for (int q = 0; q < 2; ++q) c = mfma_pair<1>(a.x[q], b.x[k][q], c);
#endif
}
// X[q] += A[q] B for every q (bf16: one after the other, so that none waits for the one before)
template <int G> __device__ __forceinline__ void mma_into(f32x16 (&X)[G], const Frag<bf16_t> (&a)[G], const Parts& b) {
#ifdef GAST_H16_F16
#pragma unroll
    for (int q = 0; q < G; ++q) {
        const Stored p(a[q]);
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            X[q] = mfma_pair<1>(p.hi[s], b.x[2][s], X[q]);
            X[q] = mfma_pair<1>(p.lo[s], b.x[1][s], X[q]);
            X[q] = mfma_pair<1>(p.hi[s], b.x[1][s], X[q]);
            X[q] = mfma_pair<1>(p.lo[s], b.x[0][s], X[q]);
            X[q] = mfma_pair<1>(p.hi[s], b.x[0][s], X[q]);
        }
    }
#else
#pragma unroll
    for (int k = 2; k >= 0; --k)
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int q = 0; q < G; ++q) X[q] = mfma_pair<1>(a[q].x[s], b.x[k][s], X[q]);
#endif
}
// the fp32 side of a product, prepared once where several products share it
template <typename T> struct Prepared;
template <> struct Prepared<float> {
    float v[16];
    template <typename V> __device__ __forceinline__ void set(const V& x) {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = x[i];
    }
};
template <> struct Prepared<bf16_t> { Parts v; template <typename V> __device__ __forceinline__ void set(const V& x) { v = parts16(x); } };

// Infinities and NaN among stored values: whether there are any; c += where they stand (ones) times which tokens are seen (sees(i): element i);
// c += A B with zeros in their place.  These run for chunks that hold some; the fences keep their operands from being made all at once, for
// the sake of the registers of everything else.
__device__ __forceinline__ bool any_wild(const Frag<float>& f) {
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) t = fmaf(f.x[i], 0.f, t);
    return t != 0.f;
}
template <typename F> __device__ __forceinline__ void mma_wild(f32x16& c, const Frag<float>& f, const F& sees) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        c = __builtin_amdgcn_mfma_f32_32x32x2f32(fabsf(f.x[i]) < INFINITY ? 0.f : 1.f, sees(i) ? 1.f : 0.f, c, 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
    }
}
__device__ __forceinline__ void mma_tame(f32x16& c, const Frag<float>& f, const float (&b)[16]) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        c = __builtin_amdgcn_mfma_f32_32x32x2f32(fabsf(f.x[i]) < INFINITY ? f.x[i] : 0.f, b[i], c, 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
    }
}
// (16 bits: an exponent of all ones carries into the sign's place)
#ifdef GAST_H16_F16
constexpr uint32_t H_CARRY = 0x04000400u, H_ONE = 0x3c00u;
#else
constexpr uint32_t H_CARRY = 0x00800080u, H_ONE = 0x3f80u;
#endif
__device__ __forceinline__ uint32_t wild2(uint32_t x) { return ((x & 0x7fff7fffu) + H_CARRY) & 0x80008000u; }
__device__ __forceinline__ bool any_wild(const Frag<bf16_t>& f) {
    return (wild2(f.x[0].x) | wild2(f.x[0].y) | wild2(f.x[0].z) | wild2(f.x[0].w) | wild2(f.x[1].x) | wild2(f.x[1].y) | wild2(f.x[1].z) | wild2(f.x[1].w)) != 0;
}
template <typename F> __device__ __forceinline__ void mma_wild(f32x16& c, const Frag<bf16_t>& f, const F& sees) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        auto one = [](uint32_t x) { return (wild2(x) >> 15) * H_ONE; };
        auto see = [&](int i) { return (sees(i) ? H_ONE : 0u) | (sees(i + 1) ? H_ONE << 16 : 0u); };
        c = mfma_h16(make_uint4(one(f.x[q].x), one(f.x[q].y), one(f.x[q].z), one(f.x[q].w)),
                     make_uint4(see(8 * q), see(8 * q + 2), see(8 * q + 4), see(8 * q + 6)), c);
        __builtin_amdgcn_sched_barrier(0);
    }
}
__device__ __forceinline__ void mma_tame(f32x16& c, const Frag<bf16_t>& f, const Parts& b) {
    auto tame = [](uint32_t x) { return x & ~((wild2(x) >> 15) * 0xffffu); };
    Frag<bf16_t> t;
#pragma unroll
    for (int q = 0; q < 2; ++q) t.x[q] = make_uint4(tame(f.x[q].x), tame(f.x[q].y), tame(f.x[q].z), tame(f.x[q].w));
    mma_sf(c, t, b);
    __builtin_amdgcn_sched_barrier(0);
}

// The 32 x DP tokens of one tensor on their way from memory to LDS: 16 elements a thread of NW waves.  16 bits: 8 channels of two rows,
// so that a turned word holds both; four lanes read 64 contiguous bytes and the turned words of a wave fall into 64 different banks.
struct View { const void* p; long t; int D; };           // token 0 of the sequence, its stride, channels
template <typename T> struct Stage;
template <> struct Stage<bf16_t> {
    static constexpr int NV = 2, VE = 8;
    uint4 x[NV];
    static __device__ __forceinline__ int row(int lane, int k) { return (lane >> 2) * 2 + k; }
    static __device__ __forceinline__ int chan(int wv, int lane, int) { return (wv * 4 + (lane & 3)) * 8; }
    __device__ __forceinline__ void none(int k) { x[k] = make_uint4(0, 0, 0, 0); }
    __device__ __forceinline__ void vec(int k, const char* p) { __builtin_memcpy(&x[k], p, 16); }
    __device__ __forceinline__ void drop(int k, int n) {       // the first n elements
        uint4 v = x[k];
        if (n & 1) v = make_uint4(v.x >> 16 | v.y << 16, v.y >> 16 | v.z << 16, v.z >> 16 | v.w << 16, v.w >> 16);
        if (n & 2) v = make_uint4(v.y, v.z, v.w, 0);
        if (n & 4) v = make_uint4(v.z, v.w, 0, 0);
        x[k] = v;
    }
    __device__ __forceinline__ void some(int k, const bf16_t* p, int n) {
        uint32_t w[4] = {0, 0, 0, 0};
        for (int e = 0; e < 8 && e < n; ++e) w[e >> 1] |= (uint32_t)p[e] << 16 * (e & 1);
        x[k] = make_uint4(w[0], w[1], w[2], w[3]);
    }
    template <int RS> __device__ __forceinline__ void rows(bf16_t* tile, int wv, int lane) const {
        bf16_t* p = tile + (lane >> 2) * 2 * RS + (wv * 4 + (lane & 3)) * 8;
#pragma unroll
        for (int k = 0; k < 2; ++k, p += RS) {
            *(uint2*)p = make_uint2(x[k].x, x[k].y);
            *(uint2*)(p + 4) = make_uint2(x[k].z, x[k].w);
        }
    }
    __device__ __forceinline__ void turned(bf16_t* tile, int wv, int lane) const {
        uint32_t* p = (uint32_t*)(tile + (wv * 4 + (lane & 3)) * 8 * TS) + (lane >> 2);
        const uint32_t a[4] = {x[0].x, x[0].y, x[0].z, x[0].w}, b[4] = {x[1].x, x[1].y, x[1].z, x[1].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            p[(2 * e) * (TS / 2)] = __builtin_amdgcn_perm(b[e], a[e], 0x05040100u);
            p[(2 * e + 1) * (TS / 2)] = __builtin_amdgcn_perm(b[e], a[e], 0x07060302u);
        }
    }
};
template <> struct Stage<float> {
    static constexpr int NV = 4, VE = 4;
    float4 x[NV];
    static __device__ __forceinline__ int row(int lane, int k) { return (lane >> 2) + 16 * (k >> 1); }
    static __device__ __forceinline__ int chan(int wv, int lane, int k) { return (wv * 8 + (lane & 3) + 4 * (k & 1)) * 4; }
    __device__ __forceinline__ void none(int k) { x[k] = make_float4(0.f, 0.f, 0.f, 0.f); }
    __device__ __forceinline__ void vec(int k, const char* p) { __builtin_memcpy(&x[k], p, 16); }
    __device__ __forceinline__ void drop(int k, int n) {
        float4 v = x[k];
        if (n & 1) v = make_float4(v.y, v.z, v.w, 0.f);
        if (n & 2) v = make_float4(v.z, v.w, 0.f, 0.f);
        x[k] = v;
    }
    __device__ __forceinline__ void some(int k, const float* p, int n) {
        x[k] = make_float4(p[0], n > 1 ? p[1] : 0.f, n > 2 ? p[2] : 0.f, n > 3 ? p[3] : 0.f);
    }
    template <int RS> __device__ __forceinline__ void rows(float* tile, int wv, int lane) const {
#pragma unroll
        for (int k = 0; k < 4; ++k) *(float4*)(tile + row(lane, k) * RS + chan(wv, lane, k)) = x[k];
    }
};
// The loads of a chunk are issued while the one before is worked on, so they stand in straight code (a join of two paths would wait for
// them): every lane reads 16 bytes at a block-uniform base plus a 32-bit offset, at a row and channels that exist (the last vector of a row
// ends with the row), and what is behind the chunk's end or the head's last channel becomes zero on the way to LDS.  Rows may start
// anywhere: this hardware's 16-byte accesses need no alignment of their own.
template <typename T>
__device__ __forceinline__ void bring(Stage<T>& s, const View& v, int t0, int n, int wv, int lane) {
    const char* base = (const char*)v.p + (long)t0 * v.t * (int)sizeof(T);
#pragma unroll
    for (int k = 0; k < Stage<T>::NV; ++k) {
        const int d = Stage<T>::chan(wv, lane, k), row = min(Stage<T>::row(lane, k), n - 1);
        s.vec(k, base + (uint32_t)(row * (int)v.t + min(d, v.D - Stage<T>::VE)) * (uint32_t)sizeof(T));
    }
}
template <typename T>
__device__ __forceinline__ void trim(Stage<T>& s, const View& v, int n, int wv, int lane) {
#pragma unroll
    for (int k = 0; k < Stage<T>::NV; ++k) {
        const int d = Stage<T>::chan(wv, lane, k);
        if (v.D % Stage<T>::VE) s.drop(k, max(d + Stage<T>::VE - v.D, 0));
        if (Stage<T>::row(lane, k) >= n || d >= v.D) s.none(k);
    }
}
// heads shorter than a vector, tokens that lie too far apart: element by element, not ahead of time
template <typename T>
__device__ __forceinline__ void bring_odd(Stage<T>& s, const View& v, int t0, int n, int wv, int lane) {
#pragma unroll
    for (int k = 0; k < Stage<T>::NV; ++k) {
        const int d = Stage<T>::chan(wv, lane, k), row = Stage<T>::row(lane, k);
        s.none(k);
        if (row < n && d < v.D) s.some(k, (const T*)v.p + (long)(t0 + row) * v.t + d, v.D - d);
    }
}

// Y (32 columns of out by 32 tokens, the token in lane % 32) to memory.  fp32: four registers are 16 bytes of a row, and go out as they are.
__device__ __forceinline__ void put_tile(const f32x16& Y, float*, float* O, long st, int t0, int n, int c0, int D, int lane) {
    const int row = lane & 31;
    float* p = O + (long)(t0 + row) * st + c0 + 4 * (lane >> 5);
    const int left = D - c0 - 4 * (lane >> 5);
    if (row >= n) return;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const float4 y = make_float4(Y[4 * q], Y[4 * q + 1], Y[4 * q + 2], Y[4 * q + 3]);
        if (8 * q + 4 <= left) __builtin_memcpy(p + 8 * q, &y, 16);
        else
#pragma unroll
            for (int e = 0; e < 3; ++e)
                if (8 * q + e < left) p[8 * q + e] = Y[4 * q + e];
    }
}
// 16 bits: by way of LDS, so that a row leaves in 16-byte pieces
__device__ __forceinline__ void put_tile(const f32x16& Y, bf16_t* tile, bf16_t* O, long st, int t0, int n, int c0, int D, int lane) {
#pragma unroll
    for (int q = 0; q < 4; ++q)
        st4(tile + (lane & 31) * TS + 8 * q + 4 * (lane >> 5), make_float4(Y[4 * q], Y[4 * q + 1], Y[4 * q + 2], Y[4 * q + 3]));
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int row = lane / 4 + 16 * k, e = (lane % 4) * 8;
        if (row >= n || c0 + e >= D) continue;
        const bf16_t* s = tile + row * TS + e;
        bf16_t* p = O + (long)(t0 + row) * st + c0 + e;
        if (c0 + e + 8 <= D) {
            const uint2 u = *(const uint2*)s, w = *(const uint2*)(s + 4);
            const uint4 y = make_uint4(u.x, u.y, w.x, w.y);
            __builtin_memcpy(p, &y, 16);
        } else {
            for (int x = 0; x < 8 && c0 + e + x < D; ++x) p[x] = s[x];
        }
    }
}
// rows [t0, t1) of out are behind the sequence's end: zero (by nthr threads)
template <typename T>
__device__ __forceinline__ void put_zeros(T* O, long st, int t0, int t1, int D, int tid, int nthr) {
    constexpr int VE = 16 / sizeof(T);
    const int nv = (D + VE - 1) / VE;
    for (long i = tid; i < (long)(t1 - t0) * nv; i += nthr) {
        const long t = i / nv;
        const int e = (int)(i - t * nv) * VE;
        T* p = O + (t0 + t) * st + e;
        if (e + VE <= D) __builtin_memset(p, 0, 16);
        else
            for (int x = 0; x < VE && e + x < D; ++x) p[x] = (T)0;
    }
}

// Which tensors a kernel stages and what its groups of DP / 32 waves do with them.
//   ONE    in = a, b, c, one group                                                (o, and dq)
//   TWO    in = q, do, k, v: group 0 makes dv, group 1 dk                         (both run backward in time)
//   THREE  in = q, do, k, v: group 2 makes dq as well                             (sequences of one chunk: no state to hand on to dq)
//   SUMS   in = -, b, c: only X, from zero, of each segment
enum { ONE, TWO, THREE, SUMS };

struct Role {
    gast_seq out;
    const float* xin;                // X before the first token in this direction, [head][segment][D1][D2], or null: zero
    float* xout;                     // X behind the last, or null
    int turn, reverse, D1, D2;       // turn: xin is held as [D2][D1]
    float fp, fk, fo;                // factors of scores, of what enters X, of what the carried X gives
};

struct ChunkArgs {
    gast_seq in[4];
    int D[4], vec[4];                // channels; can be read by vectors
    Role role[3];
    const float* log_decay;
    const int32_t* lengths;
    int B, T, J, H, nseg, L, skip_last;     // segments of L tokens; skip_last: nobody reads the sums of the last one in this direction
};

// LDS of a kernel, in elements: tiles as rows, turned tiles, output tiles of the waves (ONE: over the wave's own columns of c; fp32: none).
// 16 bits need the turned tiles because an operand's register holds two tokens; fp32 reads columns of the rows, value by value, which takes LDS
// as long as 16 bytes at a time, and has no room and no writes for them.
template <typename T, int DP, int MODE> struct Lay {
    static constexpr bool TURNED = sizeof(T) == 2;
    static constexpr int NW = DP / 32, RS = DP + 4, ROWS = CT * RS, TURN = TURNED ? DP * TS : ROWS;
    static constexpr int GROUPS = MODE == TWO ? 2 : MODE == THREE ? 3 : 1, NT = GROUPS * NW * 64;
    static constexpr int NROWS = MODE == ONE ? (TURNED ? 2 : 3) : MODE == SUMS ? (TURNED ? 0 : 2) : 4, NTURN = !TURNED ? 0 : MODE == THREE ? 3 : 2;
    static constexpr int TILES = NROWS * ROWS + NTURN * TURN;
};

// exp(g n) to two steps of fp32, however long n is: the product's rounding is carried along
__device__ __forceinline__ float power(float g, float n) {
    const float x = g * n, rest = fmaf(g, n, -x), e = expf(x), p = fmaf(e, rest, e);
    return n == 0.f ? 1.f : e > 0.f && e < INFINITY ? p : e;        // (minus infinity: lambda^0 is 1 all the same)
}
// The state is held as X = unit[p] * Xh, unit[p] = lambda^(32 p), p = chunks since the accumulators were last brought up to date: decaying them
// costs nothing until unit leaves [2^-8, 2^8].  What enters is divided by the unit, what leaves multiplied.
constexpr int PERIOD = 32;                                 // ... or until this many chunks
struct Powers {
    float up[CT + 4];                                      // lambda^k, k = 0 .. 32
    float down[2 * CT];                                    // lambda^(31 - k), 0 behind
    float unit[PERIOD + 4], per_unit[PERIOD + 4];
};
template <typename T, int DP, int MODE, bool STATE> struct Lds {
    using L = Lay<T, DP, MODE>;
    static constexpr int OUT = sizeof(T) == 2 && (MODE == TWO || MODE == THREE) ? L::NT / 64 * 32 * TS : 0;
    // two sets of tiles (one barrier a chunk instead of two) where the waves that the registers allow still fit: 20 KB a wave
    static constexpr int NBUF = STATE && (2 * L::TILES + OUT) * (int)sizeof(T) <= 20 * 1024 * L::GROUPS * L::NW ? 2 : 1;
    Powers pw;
    T tiles[NBUF * L::TILES + OUT];
};

// Two waves a SIMD where X lives in registers; four without a state (128 windows of 27 frames, 17 joints, 4 heads of 32 channels, fp32: the
// backward pass takes 76 us with three, 72 with four, 93 with five, where registers spill).
template <typename T, int DP, int MODE, bool VEC, bool STATE>
__global__ void __launch_bounds__((Lay<T, DP, MODE>::NT), (STATE ? 2 : 4)) chunk_kernel(const ChunkArgs g) {
    using L = Lay<T, DP, MODE>;
    constexpr int NW = L::NW, RS = L::RS, G = DP / 32;
    constexpr bool BWD = MODE == TWO || MODE == THREE;
    // 16 bits: operands are read and split a step ahead.  fp32: when they are needed -- its products are long and its operands take twice the
    // registers (512 heads of 128 channels, 1024 tokens: 585 -> 489 us) -- and rows of X behind the last channel are left out (32 x 128 channels:
    // 473 -> 249 us; at 16 bits the branches cost equal heads 2 to 3 % and gained unequal ones 4 to 17 %)
    constexpr bool AHEAD = sizeof(T) == 2;
    extern __shared__ __align__(16) char lds[];
    using M = Lds<T, DP, MODE, STATE>;
    M& m = *(M*)lds;
    constexpr int NBUF = M::NBUF, TURN0 = L::NROWS * L::ROWS;
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, col = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), grp = wave / NW, wv = wave % NW;
    const uint32_t heads = (uint32_t)g.B * g.J * g.H, bid = xcd_remap(blockIdx.x, gridDim.x);
    const uint32_t seg = g.nseg > 1 ? bid / heads : 0, hd = bid - seg * heads, bj = hd / (uint32_t)g.H, h = hd - bj * g.H, b = bj / (uint32_t)g.J, j = bj - b * g.J;
    const Role& ro = g.role[BWD ? grp : 0];
    const bool rev = MODE == ONE ? false : MODE == TWO ? true : MODE == THREE ? grp < 2 : ro.reverse;
    const int len = g.lengths ? min(max(g.lengths[b], 0), g.T) : g.T;
    const int s0 = (int)seg * g.L, s1 = min(s0 + g.L, g.T), e1 = min(s1, len), count = max(e1 - s0, 0);     // tokens [s0, e1), padding behind them
    const int nchunk = (count + CT - 1) / CT;
    if (MODE == SUMS && (!count || (g.skip_last && (rev ? s0 == 0 : e1 == len)))) return;
    const float lg = g.log_decay[h];
    // ---- roles: dv (a, b, c) = (k, q, do), dk (v, do, q), dq (do, v, k); turned tiles of BWD: q, do (, k)
    const int ia = BWD ? (grp == 0 ? 2 : grp == 1 ? 3 : 1) : 0, ib = BWD ? (grp == 0 ? 0 : grp == 1 ? 1 : 3) : 1, ic = BWD ? (grp == 0 ? 1 : grp == 1 ? 0 : 2) : 2;
    // offsets in a set of tiles: rows, and columns of turned tiles or of rows
    constexpr int COL0 = L::TURNED ? TURN0 : MODE == ONE ? L::ROWS : 0, CS = L::TURNED ? TS : 1;       // (the columns of b of ONE and SUMS; a column's step)
    // (v has no turned tile: the dq waves of THREE hand no state on, and make theirs of k)
    const int oa = ia * L::ROWS, ob = ib * L::ROWS, obT = COL0 + (BWD ? (L::TURNED ? min(ib, 2) : ib) : 0) * L::TURN;
    const int oc = COL0 + (BWD ? ic : 1) * L::TURN + wv * 32 * CS;                                // (this wave's 32 columns of c)
    const int c0 = wv * 32 + col, D1 = ro.D1, D2 = ro.D2;
    const bool works = wv * 32 < D2;

    // ---- which tensors this group of waves brings in: ONE and SUMS all, TWO (q, k) and (do, v), THREE (q, v), do, k
    constexpr int NS = MODE == ONE ? 3 : 2;
    const int st[3] = {MODE == ONE ? 0 : MODE == SUMS ? 1 : grp, MODE == ONE ? 1 : MODE == SUMS ? 2 : MODE == TWO ? 2 + grp : grp ? -1 : 3, 2};
    View in[NS];
    Stage<T> stage[NS];
    bool whole = true;
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        const int k = max(st[i], 0);
        in[i] = View{(const T*)g.in[k].p + seq_at(g.in[k], b, 0, j, h), g.in[k].t, g.D[k]};
        whole = whole && g.D[k] == DP;
    }
    auto fetch = [&](int c) {
        const int t0 = s0 + c * CT, n = min(CT, e1 - t0);
        if constexpr (VEC)
#pragma unroll
            for (int i = 0; i < NS; ++i) bring<T>(stage[i], in[i], t0, n, wv, lane);      // (THREE: two groups bring in nothing new the second time)
    };
    auto place = [&](int c, T* tiles) {
        const int t0 = s0 + c * CT, n = min(CT, e1 - t0);
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            if (st[i] < 0) continue;
            if constexpr (VEC) { if (!whole || n < CT) trim<T>(stage[i], in[i], n, wv, lane); }
            else bring_odd<T>(stage[i], in[i], t0, n, wv, lane);
            if (!L::TURNED || (MODE == ONE ? i < 2 : MODE != SUMS)) stage[i].template rows<RS>(tiles + (MODE == SUMS ? i : st[i]) * L::ROWS, wv, lane);
            if constexpr (L::TURNED)
                if (MODE == ONE ? i > 0 : MODE == SUMS || st[i] < L::NTURN) stage[i].turned(tiles + TURN0 + (BWD ? st[i] : st[i] - 1) * L::TURN, wv, lane);
        }
    };
    const int c_first = rev && MODE != THREE ? nchunk - 1 : 0;
    if (nchunk) fetch(c_first);
    Powers& pw = m.pw;
    if (tid <= CT) {
        const float p = tid <= count ? power(lg, (float)tid) : 0.f;         // (a growing one may overflow where there are no tokens: no inf times 0)
        pw.up[tid] = p;
        if constexpr (STATE) {
            const float u = power(lg, 32.f * tid);
            pw.unit[tid] = u;
            pw.per_unit[tid] = 1.f / u;
            if (tid < CT) {
                pw.down[CT - 1 - tid] = p;
                pw.down[CT + tid] = 0.f;
            }
        }
    }
    const float steps = 5.545f / (32.f * fabsf(lg));       // ln 2^8
    const int period = steps >= PERIOD ? PERIOD : max((int)steps, 1);
    int p = 0;
    f32x16 X[G];
#pragma unroll
    for (int q = 0; q < G; ++q) X[q] = f32x16{};
    if (STATE && MODE != SUMS && ro.xin && works) {
        const float* xin = ro.xin + ((long)hd * g.nseg + seg) * (D1 * D2);
        const int sd = ro.turn ? 1 : D2;
        xin += min(c0, D2 - 1) * (ro.turn ? D1 : 1);       // (columns behind the last repeat it: nothing of theirs is stored)
#pragma unroll
        for (int q = 0; q < G; ++q)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int d = 32 * q + 8 * (r >> 2) + 4 * half + (r & 3);
                const float x = xin[min(d, D1 - 1) * sd];
                X[q][r] = d < D1 ? x : 0.f;
            }
    }
    if (nchunk) place(c_first, m.tiles);
    __syncthreads();
    // lambda^|i - j| of the scores this lane holds, for tokens j = 8 (r / 4) + 4 half + r % 4 and i = col; 0 where i does not see j
    float pd[16];
    if constexpr (MODE != SUMS)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int gap = (8 * (r >> 2) + 4 * half + (r & 3) - col) * (rev ? 1 : -1);
            pd[r] = gap >= 0 ? pw.up[abs(gap)] * ro.fp : 0.f;
        }
    T* const O = (T*)ro.out.p + (MODE == SUMS ? 0 : seq_at(ro.out, b, 0, j, h));
    for (int c = 0; c < nchunk; ++c) {
        const int ch = rev ? nchunk - 1 - c : c, next = c + 1 < nchunk ? (rev ? ch - 1 : ch + 1) : ch, t0 = s0 + ch * CT, n = min(CT, e1 - t0);
        T* const tiles = m.tiles + (NBUF == 2 ? (c & 1) * L::TILES : 0);
        // backward in time the gradient of the last state meets the last token undecayed
        const int first = rev && t0 + n == len ? 1 : 0, steps_on = n - first;
        const bool renew = p + 1 >= period || steps_on < CT;
        const int pa = renew ? 0 : p + 1;                   // the unit afterwards
        if constexpr (STATE) fetch(next);                  // (the last chunk once more: no branch here)
        if (works) {
            const T *ta = tiles + oa + col * RS, *tb = tiles + ob + col * RS, *tbT = tiles + obT + col * CS;
            T* const tc = tiles + oc;
            // ---- P[j][i] = b_j a_i, Y[e][i] = sum_d X[d][e] a_i[d].  What one step's products need is read and split during the step before.
            f32x16 P = {}, Y = {};
            const Frag<T> fc = ld_column<RS>(tc + col * CS, half);
            Frag<T> fk[G];
            Prepared<T> pv;
            auto enter = [&] {                             // c as it enters the state, and the other side of that product
                if constexpr (AHEAD)
#pragma unroll
                    for (int q = 0; q < G; ++q) fk[q] = ld_column<RS>(tbT + 32 * q * CS, half);
                float v[16];
                unpack(fc, v);
                const float w = ro.fk * pw.per_unit[pa];
                const float* in_by = (rev ? pw.up : pw.down + CT - n) + 4 * half;      // token k enters with lambda^k, or lambda^(n - 1 - k)
#pragma unroll
                for (int r = 0; r < 16; ++r) v[r] *= in_by[8 * (r >> 2) + (r & 3)] * w;
                pv.set(v);
            };
            if constexpr (MODE != SUMS) {
                Frag<T> fa = ld_frag(ta, half), fb = ld_frag(tb, half), na = fa, nb = fb;
                Prepared<T> px, nx;
                if constexpr (STATE) px.set(X[0]);
#pragma unroll
                for (int q = 0; q < G; ++q) {
                    if (!AHEAD && q && 32 * q >= D1) break;
                    if (AHEAD && q + 1 < G) na = ld_frag(ta + 32 * (q + 1), half), nb = ld_frag(tb + 32 * (q + 1), half);
                    mma(P, fb, fa);
                    if constexpr (STATE) {
                        mma_fs(Y, px.v, fa);
                        if (q + 1 < G) nx.set(X[q + 1]);
                        else if (AHEAD) enter();
                    }
                    if (!AHEAD && q + 1 < G) na = ld_frag(ta + 32 * (q + 1), half), nb = ld_frag(tb + 32 * (q + 1), half);
                    fa = na; fb = nb; px = nx;
                }
            }
            if constexpr (MODE == SUMS || (STATE && !AHEAD)) enter();
            if constexpr (STATE)
                if (renew) {
                    const float f = pw.unit[p] * pw.up[steps_on];
#pragma unroll
                    for (int q = 0; q < G; ++q) X[q] *= f;
                }
            // ---- X += b c; meanwhile the scores, and Y[e][i] += sum_j c_j[e] P[j][i]
            if constexpr (STATE && AHEAD) {
                mma_into<G>(X, fk, pv.v);
            } else if constexpr (STATE) {
#pragma unroll
                for (int q = 0; q < G; ++q) {
                    if (q && 32 * q >= D1) break;
                    mma_sf(X[q], ld_column<RS>(tbT + 32 * q * CS, half), pv.v);
                }
            }
            if constexpr (MODE != SUMS) {
                float sc[16];
#pragma unroll
                for (int r = 0; r < 16; ++r) sc[r] = pd[r] != 0.f ? P[r] * pd[r] : 0.f;
                Prepared<T> pp;
                pp.set(sc);
                if constexpr (STATE) Y *= pw.up[max((rev ? n - 1 - col : col) + 1 - first, 0)] * pw.unit[p] * ro.fo;
                // A score of zero is no mask for an infinity or NaN of a token that i does not see: those chunks are worked on with zeros in
                // their place, and only outputs that see one of them take the product as it is.  (One that enters the state is seen there.)
                bool wild;
                if constexpr (STATE) wild = !(fabsf(X[0][0]) < INFINITY);
                else wild = any_wild(fc);
                if (__any(wild)) {
                    f32x16 Z = {};
                    mma_wild(Z, fc, [&](int r) { return (8 * (r >> 2) + 4 * half + (r & 3) - col) * (rev ? 1 : -1) >= 0; });
                    uint32_t at = 0;
#pragma unroll
                    for (int r = 0; r < 16; ++r) at |= Z[r] != 0.f ? 1u << r : 0u;
                    Z = Y;
                    mma_tame(Z, fc, pp.v);
                    mma_sf(Y, fc, pp.v);
#pragma unroll
                    for (int r = 0; r < 16; ++r) Y[r] = at >> r & 1 ? Y[r] : Z[r];
                } else {
                    mma_sf(Y, fc, pp.v);
                }
                put_tile(Y, BWD ? m.tiles + NBUF * L::TILES + wave * 32 * TS : tc, O, ro.out.t, t0, n, wv * 32, D2, lane);
            }
        }
        if constexpr (STATE) {
            p = pa;
            if (c + 1 < nchunk) {
                if constexpr (NBUF == 1) __syncthreads();
                place(next, m.tiles + (NBUF == 2 ? ((c + 1) & 1) * L::TILES : 0));
                __syncthreads();
            }
        }
    }
    if (MODE != SUMS && s1 > max(e1, s0)) put_zeros<T>(O, ro.out.t, max(e1, s0), s1, D2, tid - grp * NW * 64, NW * 64);
    if (STATE && ro.xout && works) {
        float* xo = ro.xout + ((long)hd * g.nseg + seg) * (D1 * D2);
        const float f = pw.unit[p] * (MODE != SUMS && rev && len ? pw.up[1] : 1.f);
        if (c0 >= D2) return;
#pragma unroll
        for (int q = 0; q < G; ++q)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int d = 32 * q + 8 * (r >> 2) + 4 * half + (r & 3);
                if (d < D1) xo[d * D2 + c0] = X[q][r] * f;
            }
    }
}

// The states before every segment (in place of the segments' sums) and behind the last: one thread an element, segment by segment.
struct JoinArgs {
    float* ws;                       // [head][segment][D1 D2]
    const float* first;              // [head][D1 D2], the state before the first segment in this direction, or null
    float* last;
    const float* log_decay;
    const int32_t* lengths;
    int T, J, H, nseg, L, size, reverse;
};
__global__ void __launch_bounds__(256) join_kernel(const JoinArgs g) {
    const long hd = blockIdx.x;
    const int i = blockIdx.y * 256 + threadIdx.x;
    const int h = (int)(hd % g.H);
    const long b = hd / g.H / g.J;
    const int len = g.lengths ? min(max(g.lengths[b], 0), g.T) : g.T;
    if (i >= g.size) return;
    const float lg = g.log_decay[h];
    const int n = (len + g.L - 1) / g.L;                   // segments that hold tokens
    float x = g.first ? g.first[hd * g.size + i] : 0.f;
    float* w = g.ws + hd * g.nseg * g.size + i;
    const float whole = power(lg, (float)g.L), last = power(lg, (float)(len - (n - 1) * g.L - (g.reverse ? 1 : 0)));
    for (int k0 = 0; k0 < n; k0 += 8) {                    // eight sums on their way at once
        float e[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int at = min(k0 + k, n - 1);
            e[k] = w[(long)(g.reverse ? n - 1 - at : at) * g.size];
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            if (k0 + k >= n) break;
            const int s = g.reverse ? n - 1 - k0 - k : k0 + k;
            w[(long)s * g.size] = x;
            // (the sums of the segment that comes last are only there where somebody wants the state behind it)
            x = k0 + k + 1 == n && !g.last ? 0.f : fmaf(s == n - 1 ? last : whole, x, e[k]);
        }
    }
    if (g.last) g.last[hd * g.size + i] = g.reverse && len ? power(lg, 1.f) * x : x;
}

// One token: the state is read and written once (that is the whole cost: 8 Dk Dv bytes a head; 2048 heads of 128 x 128 in 57 us, 4.7 TB/s, the
// rate of a copy).  NT threads a head, VE columns a thread, the
// rows spread over the other threads and summed through LDS.  Small states have heads of 64 threads, so that no thread is without work.
template <typename T, int VE, int NT>
__global__ void __launch_bounds__(256) step_kernel(const gast_decay_args p) {
    __shared__ float sq[256 / NT][GAST_DECAY_MAX_D], sk[256 / NT][GAST_DECAY_MAX_D], so[256 * VE];
    const int tid = threadIdx.x % NT, grp = threadIdx.x / NT, Dk = p.Dk, Dv = p.Dv, nv = Dv / VE;
    const long heads = (long)p.B * p.J * p.H, hd = NT == 256 ? blockIdx.x : min((long)blockIdx.x * (256 / NT) + grp, heads - 1);
    const bool mine = NT == 256 || (long)blockIdx.x * (256 / NT) + grp < heads;
    const int h = (int)(hd % p.H), j = (int)(hd / p.H % p.J);
    const long b = hd / p.H / p.J;
    T* O = (T*)p.o.p + seq_at(p.o, b, 0, j, h);
    const bool live = mine && !(p.lengths && p.lengths[b] < 1);
    if (mine && !live)
        for (int e = tid; e < Dv; e += NT) Elem<T>::st(O + e, 0.f);
    if (NT == 256 && !live) return;
    const T *Q = (const T*)p.q.p + seq_at(p.q, b, 0, j, h), *K = (const T*)p.k.p + seq_at(p.k, b, 0, j, h), *V = (const T*)p.v.p + seq_at(p.v, b, 0, j, h);
    if (live)
        for (int d = tid; d < Dk; d += NT) {
            sq[grp][d] = Elem<T>::ld(Q + d) * p.scale;
            sk[grp][d] = Elem<T>::ld(K + d);
        }
    __syncthreads();
    // a lambda near 1 takes effect as lambda - 1: rounded itself, it would be off the same way at every token (10^4 tokens: 2^-11 of a state)
    const float lg = p.log_decay[h];
    const bool near = fabsf(lg) < 0.6931f;
    const float f = near ? expm1f(lg) : expf(lg);
    const int rows = NT / nv, c = tid % nv, r0 = tid / nv;
    float* S = (float*)p.state + hd * Dk * Dv + c * VE;
    float o[VE], v[VE];
#pragma unroll
    for (int i = 0; i < VE; ++i) o[i] = 0.f;
    if (live && r0 < rows) {
#pragma unroll
        for (int i = 0; i < VE; ++i) v[i] = Elem<T>::ld(V + c * VE + i);
#pragma unroll 8
        for (int d = r0; d < Dk; d += rows) {
            float x[VE];
            ldv<VE>(x, S + d * Dv);
#pragma unroll
            for (int i = 0; i < VE; ++i) {
                x[i] = fmaf(f, x[i], fmaf(sk[grp][d], v[i], near ? x[i] : 0.f));
                o[i] = fmaf(sq[grp][d], x[i], o[i]);
            }
            stv<VE>(S + d * Dv, x);
        }
#pragma unroll
        for (int i = 0; i < VE; ++i) so[grp * NT * VE + (r0 * nv + c) * VE + i] = o[i];
    }
    __syncthreads();
    if (live)
        for (int e = tid; e < Dv; e += NT) {
            float t = 0.f;
            for (int r = 0; r < rows; ++r) t += so[grp * NT * VE + r * Dv + e];
            Elem<T>::st(O + e, t);
        }
}

int check(const gast_decay_args* p) {
    if (!p || p->B < 1 || p->T < 1 || p->J < 1 || p->H < 1 || p->Dk < 1 || p->Dv < 1 || !p->log_decay) return GAST_EINVAL;
    if (p->dtype != GAST_F32 && p->dtype != GAST_BF16) return GAST_EINVAL;
    if (!p->q.p || !p->k.p || !p->v.p) return GAST_EINVAL;
    if (p->Dk > GAST_DECAY_MAX_D || p->Dv > GAST_DECAY_MAX_D || p->T > (1 << 30)) return GAST_ERANGE;
    return 0;
}

// How the tokens are cut into segments, each with blocks of its own that start from the state before it.  In units of one chunk's work of a
// block: a cut reads two of the tensors twice (half a chunk's work for each chunk), hands a state of D x D fp32 over four times for each segment
// (as many bytes as D / 16 chunks of 16-bit tokens have, D / 32 of fp32), and has two launches more (about 6 chunks' time, 4 of the longer fp32
// ones).  A CU runs eight waves' worth of blocks at once, two to a SIMD; a last round that is not full still takes half of one.
// Measured, uncut and cut: 16 heads of 128 channels and 32768 tokens (bf16, forward) 2234 us in two segments, 313 in 32; forward and backward in fp32,
// 12 heads of 16 and 530 tokens 203 and 44 in 17, 128 heads of 64 and 362 tokens 189 and 140 in 6.
struct Cut { int dp, nseg, L; };
Cut cut(int dtype, long heads, int T, int Dk, int Dv) {
    const int D = Dk > Dv ? Dk : Dv;
    Cut c;
    c.dp = (D + 31) / 32 * 32;
    const long slots = 256 * (8 * 32 / c.dp), chunks = (T + CT - 1L) / CT;
    const double state = 2 + c.dp / (dtype == GAST_F32 ? 32.0 : 16.0), launches = dtype == GAST_F32 ? 4 : 6;
    auto rounds = [&](long blocks) {
        const long full = blocks / slots, rest = blocks % slots;
        return !rest ? (double)full : !full ? 1.0 : full + std::max(0.5, (double)rest / slots);
    };
    double best = (double)chunks;
    long nseg = 1;
    for (long n = 2; n <= 64 && n <= chunks && heads < slots; ++n) {
        const long len = (chunks + n - 1) / n;
        const double t = rounds(heads * ((chunks + len - 1) / len)) * (1.5 * len + state) + launches;
        if (t < best) {
            best = t;
            nseg = n;
        }
    }
    c.L = (int)((chunks + nseg - 1) / nseg * CT);
    c.nseg = (T + c.L - 1) / c.L;
    return c;
}

template <typename T, int DP, int MODE, bool VEC, bool STATE>
int launch(const ChunkArgs& g, hipStream_t s) {
    using L = Lay<T, DP, MODE>;
    constexpr int bytes = (int)sizeof(Lds<T, DP, MODE, STATE>);
    const long blocks = (long)g.B * g.J * g.H * g.nseg;
    if (blocks > 0x7fffffffL) return GAST_ERANGE;
    static_assert(bytes <= 160 * 1024, "LDS of a CU");
    if (bytes > 64 * 1024) {
        static std::atomic<bool> done[64];
        int dev = 0;
        if (hipError_t e = hipGetDevice(&dev)) return (int)e;
        if (dev >= 64 || !done[dev].load(std::memory_order_acquire)) {       // (an attribute of the device; a racing first call repeats it)
            if (hipError_t e = hipFuncSetAttribute((const void*)chunk_kernel<T, DP, MODE, VEC, STATE>, hipFuncAttributeMaxDynamicSharedMemorySize, bytes)) return (int)e;
            if (dev < 64) done[dev].store(true, std::memory_order_release);
        }
    }
    hipLaunchKernelGGL((chunk_kernel<T, DP, MODE, VEC, STATE>), dim3((unsigned)blocks), dim3(L::NT), bytes, s, g);
    GAST_CHECK_LAUNCH();
    return 0;
}
template <typename T, int MODE, bool VEC, bool STATE>
int launch_dp(const ChunkArgs& g, int dp, hipStream_t s) {
    if (dp == 32) return launch<T, 32, MODE, VEC, STATE>(g, s);
    if (dp == 64) return launch<T, 64, MODE, VEC, STATE>(g, s);
    if constexpr (MODE != THREE) return dp == 96 ? launch<T, 96, MODE, VEC, STATE>(g, s) : launch<T, 128, MODE, VEC, STATE>(g, s);
    return GAST_EINVAL;
}
// VEC: every tensor that is brought in can be read by vectors.  STATE: there is a state to start from, to return or to hand to a second chunk.
template <typename T, int MODE>
int launch_any(const ChunkArgs& g, int dp, hipStream_t s) {
    const bool vec = (MODE == SUMS || g.vec[0]) && g.vec[1] && g.vec[2] && (MODE == ONE || MODE == SUMS || g.vec[3]);
    if constexpr (MODE == ONE || MODE == THREE) {
        bool state = g.T > CT;
        for (const Role& r : g.role) state = state || r.xin || r.xout;
        if (!state) return vec ? launch_dp<T, MODE, true, false>(g, dp, s) : launch_dp<T, MODE, false, false>(g, dp, s);
    }
    return vec ? launch_dp<T, MODE, true, true>(g, dp, s) : launch_dp<T, MODE, false, true>(g, dp, s);
}

ChunkArgs chunk_args(const gast_decay_args& g, const Cut& c) {
    ChunkArgs a = {};
    a.log_decay = g.log_decay; a.lengths = g.lengths; a.B = g.B; a.T = g.T; a.J = g.J; a.H = g.H; a.nseg = c.nseg; a.L = c.L;
    return a;
}
void put_in(ChunkArgs& a, int i, const gast_seq& s, int D, int dtype) {
    const int es = dtype == GAST_F32 ? 4 : 2;
    a.in[i] = s;
    a.D[i] = D;
    a.vec[i] = D >= 16 / es && s.t >= 0 && (CT * s.t + GAST_DECAY_MAX_D) * es < (1L << 31);      // (a vector fits, offsets fit 32 bits)
}
Role role_of(const gast_seq& out, int D1, int D2, int reverse, float scale) {
    Role r = {};
    r.out = out; r.D1 = D1; r.D2 = D2; r.reverse = reverse;
    r.fp = scale; r.fk = reverse ? scale : 1.f; r.fo = reverse ? 1.f : scale;
    return r;
}

// sums of the segments of b c' and the states between them, into ws
template <typename T>
int states(const gast_decay_args& g, const Cut& c, const gast_seq& b, const gast_seq& cc, int reverse, const float* first, float* last, float* ws, hipStream_t s) {
    ChunkArgs a = chunk_args(g, c);
    put_in(a, 1, b, g.Dk, g.dtype);
    put_in(a, 2, cc, g.Dv, g.dtype);
    a.role[0] = role_of(gast_seq{}, g.Dk, g.Dv, reverse, g.scale);
    a.role[0].xout = ws;
    a.skip_last = !last;
    if (int rc = launch_any<T, SUMS>(a, c.dp, s)) return rc;
    JoinArgs j = {ws, first, last, g.log_decay, g.lengths, g.T, g.J, g.H, c.nseg, c.L, g.Dk * g.Dv, reverse};
    hipLaunchKernelGGL(join_kernel, dim3((unsigned)((long)g.B * g.J * g.H), (unsigned)((j.size + 255) / 256)), dim3(256), 0, s, j);
    GAST_CHECK_LAUNCH();
    return 0;
}

template <typename T>
int forward(const gast_decay_args& g, hipStream_t s) {
    const Cut c = cut(g.dtype, (long)g.B * g.J * g.H, g.T, g.Dk, g.Dv);
    ChunkArgs a = chunk_args(g, c);
    put_in(a, 0, g.q, g.Dk, g.dtype);
    put_in(a, 1, g.k, g.Dk, g.dtype);
    put_in(a, 2, g.v, g.Dv, g.dtype);
    a.role[0] = role_of(g.o, g.Dk, g.Dv, 0, g.scale);
    if (c.nseg > 1) {
        if (int rc = states<T>(g, c, g.k, g.v, 0, g.state, g.state_out, g.ws, s)) return rc;
        a.role[0].xin = g.ws;
    } else {
        a.role[0].xin = g.state;
        a.role[0].xout = g.state_out;
    }
    return launch_any<T, ONE>(a, c.dp, s);
}

template <typename T>
int backward(const gast_decay_args& g, hipStream_t s) {
    const Cut c = cut(g.dtype, (long)g.B * g.J * g.H, g.T, g.Dk, g.Dv);
    const float *before = g.state, *behind = g.dstate_out;
    if (c.nseg > 1) {
        if (int rc = states<T>(g, c, g.q, g.d_o, 1, g.dstate_out, g.dstate, g.ws, s)) return rc;
        before = g.ws_fwd;
        behind = g.ws;
    }
    ChunkArgs a = chunk_args(g, c);
    put_in(a, 0, g.q, g.Dk, g.dtype);
    put_in(a, 1, g.d_o, g.Dv, g.dtype);
    put_in(a, 2, g.k, g.Dk, g.dtype);
    put_in(a, 3, g.v, g.Dv, g.dtype);
    a.role[0] = role_of(g.dv, g.Dk, g.Dv, 1, g.scale);
    a.role[0].xin = behind;
    a.role[0].xout = c.nseg > 1 ? nullptr : g.dstate;
    a.role[1] = role_of(g.dk, g.Dv, g.Dk, 1, g.scale);
    a.role[1].xin = behind;
    a.role[1].turn = 1;
    Role dq = role_of(g.dq, g.Dv, g.Dk, 0, g.scale);
    dq.xin = before;
    dq.turn = 1;
    if (g.T <= CT && c.dp <= 64) {
        a.role[2] = dq;
        return launch_any<T, THREE>(a, c.dp, s);
    }
    if (int rc = launch_any<T, TWO>(a, c.dp, s)) return rc;
    ChunkArgs d = chunk_args(g, c);
    put_in(d, 0, g.d_o, g.Dv, g.dtype);
    put_in(d, 1, g.v, g.Dv, g.dtype);
    put_in(d, 2, g.k, g.Dk, g.dtype);
    d.role[0] = dq;
    return launch_any<T, ONE>(d, c.dp, s);
}

}  // namespace

extern "C" int gast_decay_fwd(const gast_decay_args* args, gast_stream_t stream) {
    if (int rc = check(args)) return rc;
    if (!args->o.p || (!args->ws && gast_decay_ws_floats(args->dtype, args->B, args->T, args->J, args->H, args->Dk, args->Dv))) return GAST_EINVAL;
    return args->dtype == GAST_F32 ? forward<float>(*args, (hipStream_t)stream) : forward<bf16_t>(*args, (hipStream_t)stream);
}

extern "C" int gast_decay_bwd(const gast_decay_args* args, gast_stream_t stream) {
    if (int rc = check(args)) return rc;
    if (!args->d_o.p || !args->dq.p || !args->dk.p || !args->dv.p) return GAST_EINVAL;
    if ((!args->ws || !args->ws_fwd) && gast_decay_ws_floats(args->dtype, args->B, args->T, args->J, args->H, args->Dk, args->Dv)) return GAST_EINVAL;
    return args->dtype == GAST_F32 ? backward<float>(*args, (hipStream_t)stream) : backward<bf16_t>(*args, (hipStream_t)stream);
}

extern "C" long gast_decay_ws_floats(int dtype, int B, int T, int J, int H, int Dk, int Dv) {
    const long heads = (long)B * J * H;
    if (heads < 1 || T < 1 || Dk < 1 || Dv < 1) return 0;
    const Cut c = cut(dtype, heads, T, Dk, Dv);
    return c.nseg > 1 ? heads * c.nseg * Dk * Dv : 0;
}

extern "C" int gast_decay_step(const gast_decay_args* args, gast_stream_t stream) {
    if (int rc = check(args)) return rc;
    if (!args->o.p || !args->state || args->T != 1) return GAST_EINVAL;
    const gast_decay_args& g = *args;
    const long heads = (long)g.B * g.J * g.H;
    if (heads > 0x7fffffffL) return GAST_ERANGE;
    const hipStream_t s = (hipStream_t)stream;
    const int ve = (uintptr_t)g.state % 16 == 0 && g.Dv % 4 == 0 ? 4 : 1;
    // 64 threads a head for states of up to 256 vectors (67456 heads of 16 x 16: 104 -> 42 us, 34816 of 32 x 32: 72 -> 57), 256 for larger ones
    // (34816 of 31 x 64: 122 -> 109) and where there are too few heads to fill the card (17 of 32 x 32 either way 4 us of kernel)
    const bool small = g.Dk * g.Dv <= ve * 256 && g.Dv <= 64 * ve && heads >= 1024;
    const dim3 grid((unsigned)(small ? (heads + 3) / 4 : heads)), blk(256);
    auto go = [&](auto t, auto v) {
        using T = decltype(t);
        constexpr int VE = decltype(v)::value;
        if (small) hipLaunchKernelGGL((step_kernel<T, VE, 64>), grid, blk, 0, s, g);
        else hipLaunchKernelGGL((step_kernel<T, VE, 256>), grid, blk, 0, s, g);
    };
    if (g.dtype == GAST_F32) {
        if (ve == 4) go(float{}, std::integral_constant<int, 4>{});
        else go(float{}, std::integral_constant<int, 1>{});
    } else {
        if (ve == 4) go(bf16_t{}, std::integral_constant<int, 4>{});
        else go(bf16_t{}, std::integral_constant<int, 1>{});
    }
    GAST_CHECK_LAUNCH();
    return 0;
}
