// Layer norm, alone or of a residual stream plus a dropped-out branch, forward and backward.
//
//   s = residual + drop(x)  (rounded to the storage type: the next layer reads it)      mean, var over the C channels of a row
//   y = (s - mean) rstd gamma + beta,   rstd = 1 / sqrt(var + eps)
//   dxhat = dy gamma;   ds = dstream + rstd (dxhat - mean(dxhat) - xhat mean(dxhat xhat));   dx = ds * dropout multiplier
//   dgamma = sum_rows dy xhat,   dbeta = sum_rows dy
//
// Bound by memory: every tensor is read or written once.  A group of G lanes holds one row in registers (up to 16 values a lane), so the
// variance is the second pass over registers, not over memory; statistics and sums are fp32.  The dropout mask is the library's counter
// stream, computed again in the backward pass and never stored.  dgamma / dbeta: a group keeps the sums of the columns it owns in
// registers over all its rows, groups of a block meet in LDS, blocks in a partial row each, and a second launch adds the partial rows in a
// fixed order (no atomics: run-to-run the same bits).
// Measured: 8192 rows of 4096 (bf16, dropout) 53 us forward = 5.0 TB/s, 76 + 6 us backward = 4.4 TB/s (a copy reaches 4.8); 58752 rows of 128
// (fp32) 12 us forward, 16 + 4 us backward.
#include "seq_common.h"

namespace {

constexpr int MAXV = 16;             // values of a row that one lane holds

// the dropout multipliers of elements e .. e + VE - 1 of their tensor: drop_mul for e < 2^33, beyond that the high word of e / 2 enters the
// key.  Two neighbours share a hash, so a vector of VE >= 2 (e even) makes VE / 2 of them.
__device__ __forceinline__ uint32_t drop_word(uint32_t key, unsigned long pair) { return hash32((uint32_t)pair ^ (key + (uint32_t)(pair >> 32) * 0xC2B2AE35u)); }
template <int VE>
__device__ __forceinline__ void drop_vec(float (&m)[VE], uint32_t key, uint32_t thresh, float inv_keep, long e) {
    if constexpr (VE == 1) {
        const uint32_t h = drop_word(key, (unsigned long)e >> 1);
        m[0] = ((e & 1) ? h >> 16 : h & 0xffffu) >= thresh ? inv_keep : 0.f;
    } else {
#pragma unroll
        for (int i = 0; i < VE; i += 2) {
            const uint32_t h = drop_word(key, ((unsigned long)e + i) >> 1);
            m[i] = (h & 0xffffu) >= thresh ? inv_keep : 0.f;
            m[i + 1] = (h >> 16) >= thresh ? inv_keep : 0.f;
        }
    }
}
// the stream's value as it is stored: x m + r rounded to fp32, and that to the type.  (The empty statement keeps the binary16 build from
// fusing both into one instruction that rounds once, which is another value now and then.)
template <typename T> __device__ __forceinline__ float stored(float v) {
    asm("" : "+v"(v));
    return Elem<T>::rnd(v);
}
// VE parameters from column c on (fp32, on the same alignment as the rows), or `none`
template <int VE> __device__ __forceinline__ void ld_par(float (&w)[VE], const float* p, int c, float none) {
    constexpr int VF = VE < 4 ? VE : 4;
#pragma unroll
    for (int k = 0; k < VE; k += VF) {
        float4 u = make_float4(none, none, none, none);
        if (p) {
            if constexpr (VF == 4) u = *(const float4*)(p + c + k);
            else if constexpr (VF == 2) { const float2 v = *(const float2*)(p + c + k); u.x = v.x; u.y = v.y; }
            else u.x = p[c + k];
        }
        w[k] = u.x;
        if constexpr (VF > 1) w[k + 1] = u.y;
        if constexpr (VF > 2) { w[k + 2] = u.z; w[k + 3] = u.w; }
    }
}

// sum over the G lanes that hold a row (G <= 64: lanes of a wave; else the whole block of G threads); every lane gets it
template <int G>
__device__ __forceinline__ float group_sum(float v, float* red) {
#pragma unroll
    for (int o = (G < 64 ? G : 64) / 2; o; o >>= 1) v += __shfl_xor(v, o, 64);
    if constexpr (G > 64) {
        constexpr int NW = G / 64;
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) v += red[w];
    }
    return v;
}

struct NormArgs {
    const void *X, *Res, *dY, *dSt;
    void *S, *Y, *dX, *dS;
    long ldx, ldr, lds, ldy, lddy, ldds, lddx, lddsum, rows;
    int C, use_drop;
    const float *gamma, *beta;
    float *mean, *rstd;
    float eps;
    uint32_t salt;
    gast_dropout drop;
    float* ws;
};

// NC vectors of VE values per lane cover the row: G * NC * VE >= C.  A block walks over rows with gamma and beta in registers.  Loads stand
// in straight code (a join of two paths would wait for them): lanes and groups behind the end read the last vector of the last row.
template <typename T, int VE, int NC, int G, bool ADD>
__global__ void __launch_bounds__(G > 256 ? G : 256) norm_fwd_kernel(const NormArgs a) {
    constexpr int GPB = G > 256 ? 1 : 256 / G;
    __shared__ float red[2][2][G > 64 ? G / 64 : 1];
    const int lane = threadIdx.x % G, C = a.C, nvec = C / VE;
    const float inv = 1.f / (float)C;
    const uint32_t key = ADD && a.use_drop ? drop_key(a.drop, a.salt) : 0u;
    int at[NC];
    float w[NC][VE], b[NC][VE];
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        at[i] = min(i * G + lane, nvec - 1) * VE;
        ld_par<VE>(w[i], a.gamma, at[i], 1.f);
        ld_par<VE>(b[i], a.beta, at[i], 0.f);
    }
    int par = 0;
    for (long r0 = (long)blockIdx.x * GPB; r0 < a.rows; r0 += (long)gridDim.x * GPB, par ^= 1) {        // (block-uniform: barriers inside)
        const long row = r0 + threadIdx.x / G, in = min(row, a.rows - 1);
        const bool on = row < a.rows;
        const T* x = (const T*)a.X + in * a.ldx;
        float s[NC][VE];
#pragma unroll
        for (int i = 0; i < NC; ++i) ldv<VE>(s[i], x + at[i]);
        if constexpr (ADD) {
            const T* r = (const T*)a.Res + in * a.ldr;
            float q[NC][VE];
#pragma unroll
            for (int i = 0; i < NC; ++i) ldv<VE>(q[i], r + at[i]);
            if (a.use_drop) {
#pragma unroll
                for (int i = 0; i < NC; ++i) {
                    float m[VE];
                    drop_vec<VE>(m, key, a.drop.thresh, a.drop.inv_keep, row * C + at[i]);
                    // what a 0 multiplies is gone even where it is not finite
#pragma unroll
                    for (int e = 0; e < VE; ++e) s[i][e] = stored<T>(fmaf(m[e] == 0.f ? 0.f : s[i][e], m[e], q[i][e]));
                }
            } else {
#pragma unroll
                for (int i = 0; i < NC; ++i)
#pragma unroll
                    for (int e = 0; e < VE; ++e) s[i][e] = stored<T>(s[i][e] + q[i][e]);
            }
            T* so = (T*)a.S + in * a.lds;
#pragma unroll
            for (int i = 0; i < NC; ++i)
                if (on && i * G + lane < nvec) stv<VE>(so + at[i], s[i]);
        }
        if (nvec < NC * G)
#pragma unroll
            for (int i = 0; i < NC; ++i)
#pragma unroll
                for (int e = 0; e < VE; ++e) s[i][e] = i * G + lane < nvec ? s[i][e] : 0.f;
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < NC; ++i)
#pragma unroll
            for (int e = 0; e < VE; ++e) t += s[i][e];
        const float mean = group_sum<G>(t, red[par][0]) * inv;
        t = 0.f;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            float u = 0.f;
#pragma unroll
            for (int e = 0; e < VE; ++e) u = fmaf(s[i][e] - mean, s[i][e] - mean, u);
            t += i * G + lane < nvec ? u : 0.f;
        }
        const float rstd = 1.f / sqrtf(group_sum<G>(t, red[par][1]) * inv + a.eps);
        if (!on) continue;
        T* y = (T*)a.Y + row * a.ldy;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            if (i * G + lane >= nvec) continue;
            float d[VE];
#pragma unroll
            for (int e = 0; e < VE; ++e) d[e] = fmaf((s[i][e] - mean) * rstd, w[i][e], b[i][e]);
            stv<VE>(y + at[i], d);
        }
        if (a.mean && lane == 0) {
            a.mean[row] = mean;
            a.rstd[row] = rstd;
        }
    }
}

// rows longer than the registers of a block: the row is read three times (from L2 after the first)
template <typename T>
__global__ void __launch_bounds__(1024) norm_fwd_long_kernel(const NormArgs a) {
    __shared__ float red[2][16];
    const int C = a.C;
    const long row = blockIdx.x;
    const T* x = (const T*)a.X + row * a.ldx;
    T* so = (T*)a.S + row * a.lds;
    float t = 0.f;
    if (a.Res) {
        const T* r = (const T*)a.Res + row * a.ldr;
        const uint32_t key = a.use_drop ? drop_key(a.drop, a.salt) : 0u;
        for (int c = threadIdx.x; c < C; c += 1024) {
            float v = Elem<T>::ld(x + c);
            const float q = Elem<T>::ld(r + c);
            if (a.use_drop) {
                float m[1];
                drop_vec<1>(m, key, a.drop.thresh, a.drop.inv_keep, row * C + c);
                v = m[0] == 0.f ? q : fmaf(v, m[0], q);
            } else {
                v += q;
            }
            v = stored<T>(v);
            Elem<T>::st(so + c, v);
            t += v;
        }
        x = so;                        // (each thread reads back what it wrote itself)
    } else {
        for (int c = threadIdx.x; c < C; c += 1024) t += Elem<T>::ld(x + c);
    }
    const float inv = 1.f / (float)C;
    const float mean = group_sum<1024>(t, red[0]) * inv;
    t = 0.f;
    for (int c = threadIdx.x; c < C; c += 1024) {
        const float d = Elem<T>::ld(x + c) - mean;
        t = fmaf(d, d, t);
    }
    const float rstd = 1.f / sqrtf(group_sum<1024>(t, red[1]) * inv + a.eps);
    T* y = (T*)a.Y + row * a.ldy;
    for (int c = threadIdx.x; c < C; c += 1024)
        Elem<T>::st(y + c, fmaf((Elem<T>::ld(x + c) - mean) * rstd, a.gamma ? a.gamma[c] : 1.f, a.beta ? a.beta[c] : 0.f));
    if (a.mean && threadIdx.x == 0) {
        a.mean[row] = mean;
        a.rstd[row] = rstd;
    }
}

// g = dY gamma, xhat -> dS, dX row by row; the sums of dY xhat and dY per column stay in w0, w1 (registers of the lane that owns it)
// (ADD: there is the stream's own gradient dSt.)
template <typename T, int VE, int NC, int G, bool ADD>
__global__ void __launch_bounds__(G > 256 ? G : 256) norm_bwd_kernel(const NormArgs a) {
    constexpr int GPB = G > 256 ? 1 : 256 / G;
    constexpr int NT = G > 256 ? G : 256;
    __shared__ float red[2][2][G > 64 ? G / 64 : 1];
    __shared__ float meet[GPB > 1 ? NT * NC * VE : 1];
    const int lane = threadIdx.x % G, grp = threadIdx.x / G, C = a.C, nvec = C / VE;
    const float inv = 1.f / (float)C;
    const uint32_t key = a.use_drop ? drop_key(a.drop, a.salt) : 0u;
    int at[NC];
    float w0[NC][VE], w1[NC][VE], gm[NC][VE];
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        at[i] = min(i * G + lane, nvec - 1) * VE;
        ld_par<VE>(gm[i], a.gamma, at[i], 1.f);
#pragma unroll
        for (int e = 0; e < VE; ++e) w0[i][e] = w1[i][e] = 0.f;
    }
    const T *dY = (const T*)(a.dY ? a.dY : a.S), *S = (const T*)a.S;            // (without dY the norm has no gradient: zeros below)
    const long lddy = a.dY ? a.lddy : a.lds;
    int par = 0;
    for (long r0 = (long)blockIdx.x * GPB; r0 < a.rows; r0 += (long)gridDim.x * GPB, par ^= 1) {        // (block-uniform: barriers inside)
        const long row = r0 + grp, in = min(row, a.rows - 1);
        const bool on = row < a.rows;
        float g[NC][VE], h[NC][VE], st[NC][VE];
#pragma unroll
        for (int i = 0; i < NC; ++i) ldv<VE>(h[i], S + in * a.lds + at[i]);
#pragma unroll
        for (int i = 0; i < NC; ++i) ldv<VE>(g[i], dY + in * lddy + at[i]);
        if constexpr (ADD)
#pragma unroll
            for (int i = 0; i < NC; ++i) ldv<VE>(st[i], (const T*)a.dSt + in * a.ldds + at[i]);
        float mean = a.mean[in], rstd = a.rstd[in];
        if (!a.dY) {                                     // (the stream's gradient passes as it is, in rows with infinities too)
            mean = rstd = 0.f;
#pragma unroll
            for (int i = 0; i < NC; ++i)
#pragma unroll
                for (int e = 0; e < VE; ++e) h[i][e] = 0.f;
        }
        if (!on || nvec < NC * G || !a.dY)
#pragma unroll
            for (int i = 0; i < NC; ++i)
#pragma unroll
                for (int e = 0; e < VE; ++e) g[i][e] = on && i * G + lane < nvec && a.dY ? g[i][e] : 0.f;
        float t0 = 0.f, t1 = 0.f;
#pragma unroll
        for (int i = 0; i < NC; ++i)
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                h[i][e] = (h[i][e] - mean) * rstd;
                w0[i][e] = fmaf(g[i][e], h[i][e], w0[i][e]);
                w1[i][e] += g[i][e];
                g[i][e] *= gm[i][e];
                t0 += g[i][e];
                t1 = fmaf(g[i][e], h[i][e], t1);
            }
        t0 = group_sum<G>(t0, red[par][0]) * inv;
        t1 = group_sum<G>(t1, red[par][1]) * inv;
        if (!on) continue;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            if (i * G + lane >= nvec) continue;
            float d[VE];
#pragma unroll
            for (int e = 0; e < VE; ++e) d[e] = ADD ? fmaf(rstd, g[i][e] - t0 - h[i][e] * t1, st[i][e]) : rstd * (g[i][e] - t0 - h[i][e] * t1);
            if (a.dS) stv<VE>((T*)a.dS + row * a.lddsum + at[i], d);
            if (a.dX) {
                if (a.use_drop) {
                    float m[VE];
                    drop_vec<VE>(m, key, a.drop.thresh, a.drop.inv_keep, row * C + at[i]);
#pragma unroll
                    for (int e = 0; e < VE; ++e) d[e] = m[e] == 0.f ? 0.f : d[e] * m[e];
                }
                stv<VE>((T*)a.dX + row * a.lddx + at[i], d);
            }
        }
    }
    if (a.ws) {
        float* out = a.ws + (long)blockIdx.x * 2 * C;
        for (int k = 0; k < 2; ++k, out += C) {
            if constexpr (GPB > 1) {
                __syncthreads();
#pragma unroll
                for (int i = 0; i < NC; ++i)
#pragma unroll
                    for (int e = 0; e < VE; ++e) meet[(grp * G * NC + i * G + lane) * VE + e] = k ? w1[i][e] : w0[i][e];
                __syncthreads();
                for (int c = threadIdx.x; c < C; c += NT) {
                    float t = 0.f;
#pragma unroll
                    for (int q = 0; q < GPB; ++q) t += meet[q * G * NC * VE + c];
                    out[c] = t;
                }
            } else {
#pragma unroll
                for (int i = 0; i < NC; ++i)
                    if (i * G + lane < nvec)
#pragma unroll
                        for (int e = 0; e < VE; ++e) out[(i * G + lane) * VE + e] = k ? w1[i][e] : w0[i][e];
            }
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(1024) norm_bwd_long_kernel(const NormArgs a) {
    __shared__ float red[2][2][16];
    const int C = a.C;
    const float inv = 1.f / (float)C;
    const uint32_t key = a.use_drop ? drop_key(a.drop, a.salt) : 0u;
    float* out = a.ws ? a.ws + (long)blockIdx.x * 2 * C : nullptr;
    int par = 0;
    bool first = true;
    for (long row = blockIdx.x; row < a.rows; row += gridDim.x, par ^= 1, first = false) {
        const T* s = (const T*)a.S + row * a.lds;
        const T* dy = a.dY ? (const T*)a.dY + row * a.lddy : nullptr;
        const float mean = dy ? a.mean[row] : 0.f, rstd = dy ? a.rstd[row] : 0.f;       // (without dY nothing of the row counts, infinities neither)
        float t0 = 0.f, t1 = 0.f;
        for (int c = threadIdx.x; c < C; c += 1024) {
            const float y = dy ? Elem<T>::ld(dy + c) : 0.f, h = dy ? (Elem<T>::ld(s + c) - mean) * rstd : 0.f, g = a.gamma ? y * a.gamma[c] : y;
            if (out) {                                   // (this block's partial row; column c belongs to this thread alone)
                out[c] = first ? y * h : fmaf(y, h, out[c]);
                out[C + c] = first ? y : out[C + c] + y;
            }
            t0 += g;
            t1 = fmaf(g, h, t1);
        }
        t0 = group_sum<1024>(t0, red[par][0]) * inv;
        t1 = group_sum<1024>(t1, red[par][1]) * inv;
        for (int c = threadIdx.x; c < C; c += 1024) {
            const float y = dy ? Elem<T>::ld(dy + c) : 0.f, h = dy ? (Elem<T>::ld(s + c) - mean) * rstd : 0.f, g = a.gamma ? y * a.gamma[c] : y;
            float d = fmaf(rstd, g - t0 - h * t1, a.dSt ? Elem<T>::ld((const T*)a.dSt + row * a.ldds + c) : 0.f);
            if (a.dS) Elem<T>::st((T*)a.dS + row * a.lddsum + c, d);
            if (a.dX) {
                if (a.use_drop) {
                    float m[1];
                    drop_vec<1>(m, key, a.drop.thresh, a.drop.inv_keep, row * C + c);
                    d = m[0] == 0.f ? 0.f : d * m[0];
                }
                Elem<T>::st((T*)a.dX + row * a.lddx + c, d);
            }
        }
    }
}

// dgamma[c] = sum_b ws[b][0][c], dbeta[c] = sum_b ws[b][1][c]: 32 columns x 32 row lanes a block, a fixed order
__global__ void __launch_bounds__(1024) norm_wsum_kernel(const float* __restrict__ ws, int nblk, int C, float* dgamma, float* dbeta) {
    __shared__ float sred[32][33];
    const int cx = threadIdx.x & 31, ry = threadIdx.x >> 5;
    const long n = (long)blockIdx.x * 32 + cx, ncol = 2L * C;
    float t = 0.f;
    if (n < ncol) {
#pragma unroll 8
        for (int r = ry; r < nblk; r += 32) t += ws[r * ncol + n];
    }
    sred[ry][cx] = t;
    __syncthreads();
    if (ry == 0 && n < ncol) {
        t = 0.f;
#pragma unroll
        for (int r = 0; r < 32; ++r) t += sred[r][cx];
        float* o = n < C ? (dgamma ? dgamma + n : nullptr) : (dbeta ? dbeta + (n - C) : nullptr);
        if (o) *o = t;
    }
}

// How a row is held: vectors of ve values, G lanes, NC vectors a lane (at most MAXV values); G = 0: the long kernels.
// The narrowest group that can hold the row: 32 lanes, a wave, then 256 .. 1024 threads.
// A row has 32 lanes at least, and a width that is no multiple of a vector has narrower ones, which is slow for short rows and for odd widths of
// 16 bits (64 MB a tensor, forward, fp32 / bf16: C = 8 0.9 / 0.4 TB/s, 32 3.3 / 1.4, 64 5.3 / 2.7, 87 4.0 / 2.2, 128 6.4 / 4.8, 4095 5.8 / 1.8, 4096 6.3 / 5.9).
struct Shape { int ve, G, NC; };

Shape shape_of(int C, int ve) {
    while (ve > 1 && C % ve) ve >>= 1;
    const int nvec = C / ve, ncmax = MAXV / ve;
    Shape s = {ve, 0, 1};
    if (nvec <= 32) s.G = 32;
    else
        for (int G = 64; G <= 1024; G *= (G == 64 ? 4 : 2))
            if (nvec <= G * ncmax) {
                s.G = G;
                while (s.NC * G < nvec) s.NC *= 2;
                break;
            }
    return s;
}

// parameters are read in vectors of min(ve, 4) floats
int par_align(const void* p, int ve) {
    while (ve > 1 && p && (uintptr_t)p % ((ve < 4 ? ve : 4) * 4)) ve >>= 1;
    return ve;
}
int row_align(const void* p, long ld, int es, int ve) {
    while (ve > 1 && (p && (((uintptr_t)p % (uintptr_t)(ve * es)) || ld % ve))) ve >>= 1;
    return ve;
}

constexpr int LONG_BLOCKS = 256;
// blocks of the backward pass: each leaves a partial row of 2 C sums (8 C bytes), so there are no more than one for every 64 C bytes or so of
// S, dY and dX -- the partial rows stay below an eighth of the tensors -- and no more than fill the card
long bwd_blocks(long rows, int C, int es, int G) {
    if (!G) return rows < LONG_BLOCKS ? rows : LONG_BLOCKS;
    const int gpb = G > 256 ? 1 : 256 / G;
    long n = (rows + gpb - 1) / gpb;
    const long most = G > 256 ? 256L * 2048 / G / 2 : 1024, lean = rows * es * 3 / 64 + 1;
    if (n > most) n = most;
    if (n > lean) n = lean;
    return n < 1 ? 1 : n;
}

template <typename T, int VE, int NC, int G>
void run(const NormArgs& a, bool bwd, long nblk, hipStream_t s) {
    constexpr int NT = G > 256 ? G : 256, GPB = G > 256 ? 1 : 256 / G;
    if (bwd) {
        if (a.dSt) hipLaunchKernelGGL((norm_bwd_kernel<T, VE, NC, G, true>), dim3((unsigned)nblk), dim3(NT), 0, s, a);
        else hipLaunchKernelGGL((norm_bwd_kernel<T, VE, NC, G, false>), dim3((unsigned)nblk), dim3(NT), 0, s, a);
        return;
    }
    const long need = (a.rows + GPB - 1) / GPB, most = 8L * 256 * 256 / NT;       // (no more than run at once: gamma and beta are read once each)
    const dim3 grid((unsigned)(need < most ? need : most));
    if (a.Res) hipLaunchKernelGGL((norm_fwd_kernel<T, VE, NC, G, true>), grid, dim3(NT), 0, s, a);
    else hipLaunchKernelGGL((norm_fwd_kernel<T, VE, NC, G, false>), grid, dim3(NT), 0, s, a);
}
// (only what shape_of picks is built: every NC for a wave, NC > MAXV / VE / 4 for 256 threads, the largest beyond)
template <typename T, int VE, int NC>
void run_g(const NormArgs& a, int G, bool bwd, long nblk, hipStream_t s) {
    constexpr int most = MAXV / VE;
    if constexpr (NC == 1) { if (G == 32) return run<T, VE, NC, 32>(a, bwd, nblk, s); }
    if constexpr (NC > most / 4) { if (G == 256) return run<T, VE, NC, 256>(a, bwd, nblk, s); }
    if constexpr (NC == most) {
        if (G == 512) return run<T, VE, NC, 512>(a, bwd, nblk, s);
        if (G == 1024) return run<T, VE, NC, 1024>(a, bwd, nblk, s);
    }
    run<T, VE, NC, 64>(a, bwd, nblk, s);
}
template <typename T, int VE, int NC = MAXV / VE>
void run_nc(const NormArgs& a, const Shape& sh, bool bwd, long nblk, hipStream_t s) {
    if constexpr (NC > 1) { if (sh.NC < NC) return run_nc<T, VE, NC / 2>(a, sh, bwd, nblk, s); }
    run_g<T, VE, NC>(a, sh.G, bwd, nblk, s);
}
template <typename T>
void run_all(const NormArgs& a, const Shape& sh, bool bwd, long nblk, hipStream_t s) {
    if (!sh.G) {
        if (bwd) hipLaunchKernelGGL((norm_bwd_long_kernel<T>), dim3((unsigned)nblk), dim3(1024), 0, s, a);
        else hipLaunchKernelGGL((norm_fwd_long_kernel<T>), dim3((unsigned)a.rows), dim3(1024), 0, s, a);
        return;
    }
    if constexpr (sizeof(T) == 2) { if (sh.ve == 8) return run_nc<T, 8>(a, sh, bwd, nblk, s); }
    if (sh.ve == 4) return run_nc<T, 4>(a, sh, bwd, nblk, s);
    if (sh.ve == 2) return run_nc<T, 2>(a, sh, bwd, nblk, s);
    run_nc<T, 1>(a, sh, bwd, nblk, s);
}

}  // namespace

extern "C" int gast_layer_norm_fwd(int dtype, const void* X, long ldx, const void* residual, long ldr, long rows, int C, const float* gamma,
                                   const float* beta, float eps, int use_drop, uint32_t salt, gast_dropout drop, void* S, long lds, void* Y,
                                   long ldy, float* mean, float* rstd, gast_stream_t stream) {
    if (!X || !Y || rows < 1 || C < 1 || (residual && !S) || (use_drop && (!residual || !drop.seed)) || (!mean != !rstd)) return GAST_EINVAL;
    if (dtype != GAST_F32 && dtype != GAST_BF16) return GAST_EINVAL;
    if (rows > 0x7fffffffL) return GAST_ERANGE;
    const int es = dtype == GAST_F32 ? 4 : 2;
    int ve = row_align(X, ldx, es, 16 / es);
    ve = row_align(Y, ldy, es, ve);
    if (residual) ve = row_align(S, lds, es, row_align(residual, ldr, es, ve));
    ve = par_align(gamma, par_align(beta, ve));
    const Shape sh = shape_of(C, ve);
    NormArgs a = {};
    a.X = X; a.ldx = ldx; a.Res = residual; a.ldr = ldr; a.rows = rows; a.C = C; a.gamma = gamma; a.beta = beta; a.eps = eps;
    a.use_drop = use_drop; a.salt = salt; a.drop = drop; a.S = S; a.lds = lds; a.Y = Y; a.ldy = ldy; a.mean = mean; a.rstd = rstd;
    if (dtype == GAST_F32) run_all<float>(a, sh, false, 0, (hipStream_t)stream);
    else run_all<bf16_t>(a, sh, false, 0, (hipStream_t)stream);
    GAST_CHECK_LAUNCH();
    return 0;
}

extern "C" long gast_layer_norm_bwd_ws_floats(long rows, int C) {
    const long lean = rows * 12 / 64 + 1 > LONG_BLOCKS ? rows * 12 / 64 + 1 : LONG_BLOCKS;        // (bwd_blocks at any alignment and type)
    const long most = rows < 1024 ? rows : 1024;
    return (most < lean ? most : lean) * 2 * C;
}

extern "C" int gast_layer_norm_bwd(int dtype, const void* dY, long lddy, const void* dStream, long ldds, const void* S, long lds, long rows,
                                   int C, const float* gamma, const float* mean, const float* rstd, int use_drop, uint32_t salt,
                                   gast_dropout drop, void* dX, long lddx, void* dS, long lddsum, float* dgamma, float* dbeta, float* ws,
                                   gast_stream_t stream) {
    if (!S || !mean || !rstd || rows < 1 || C < 1 || (use_drop && !drop.seed) || ((dgamma || dbeta) && !ws)) return GAST_EINVAL;
    if (dtype != GAST_F32 && dtype != GAST_BF16) return GAST_EINVAL;
    if (rows > 0x7fffffffL) return GAST_ERANGE;
    const int es = dtype == GAST_F32 ? 4 : 2;
    int ve = row_align(S, lds, es, 16 / es);
    ve = row_align(dY, lddy, es, ve);
    ve = row_align(dStream, ldds, es, ve);
    ve = row_align(dX, lddx, es, ve);
    ve = row_align(dS, lddsum, es, ve);
    ve = par_align(gamma, ve);
    const Shape sh = shape_of(C, ve);
    NormArgs a = {};
    a.dY = dY; a.lddy = lddy; a.dSt = dStream; a.ldds = ldds; a.S = (void*)S; a.lds = lds; a.rows = rows; a.C = C; a.gamma = gamma;
    a.mean = (float*)mean; a.rstd = (float*)rstd; a.use_drop = use_drop; a.salt = salt; a.drop = drop; a.dX = dX; a.lddx = lddx;
    a.dS = dS; a.lddsum = lddsum; a.ws = dgamma || dbeta ? ws : nullptr;
    const long nblk = bwd_blocks(rows, C, es, sh.G);
    const hipStream_t s = (hipStream_t)stream;
    if (dtype == GAST_F32) run_all<float>(a, sh, true, nblk, s);
    else run_all<bf16_t>(a, sh, true, nblk, s);
    GAST_CHECK_LAUNCH();
    if (a.ws) {
        hipLaunchKernelGGL(norm_wsum_kernel, dim3((unsigned)((2L * C + 31) / 32)), dim3(1024), 0, s, a.ws, (int)nblk, C, dgamma, dbeta);
        GAST_CHECK_LAUNCH();
    }
    return 0;
}
