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
#include "seq_common.h"

namespace {

constexpr int MAXV = 16;             // values of a row that one lane holds

// the dropout multiplier of element e of its tensor: drop_mul for e < 2^33, beyond that the high word of e / 2 enters the key
__device__ __forceinline__ float drop_mul64(uint32_t key, uint32_t thresh, float inv_keep, long e) {
    const uint32_t hi = (uint32_t)((unsigned long)e >> 33);
    const uint32_t h = hash32((uint32_t)((unsigned long)e >> 1) ^ (key + hi * 0xC2B2AE35u));
    const uint32_t bits = (e & 1) ? (h >> 16) : (h & 0xffffu);
    return bits >= thresh ? inv_keep : 0.f;
}
template <int VE>
__device__ __forceinline__ void drop_vec(float (&m)[VE], uint32_t key, uint32_t thresh, float inv_keep, long e) {
#pragma unroll
    for (int i = 0; i < VE; ++i) m[i] = drop_mul64(key, thresh, inv_keep, e + i);
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

// NC vectors of VE values per lane cover the row: G * NC * VE >= C
template <typename T, int VE, int NC, int G>
__global__ void __launch_bounds__(G > 256 ? G : 256) norm_fwd_kernel(const NormArgs a) {
    constexpr int GPB = G > 256 ? 1 : 256 / G;
    __shared__ float red[2][G > 64 ? G / 64 : 1];
    const int lane = threadIdx.x % G, C = a.C, nvec = C / VE;
    const long row = (long)blockIdx.x * GPB + threadIdx.x / G;
    const bool on = row < a.rows;
    float s[NC][VE];
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
        for (int e = 0; e < VE; ++e) s[i][e] = 0.f;
    if (on) {
        const T* x = (const T*)a.X + row * a.ldx;
#pragma unroll
        for (int i = 0; i < NC; ++i)
            if (i * G + lane < nvec) ldv<VE>(s[i], x + (i * G + lane) * VE);
        if (a.Res) {
            const T* r = (const T*)a.Res + row * a.ldr;
            T* so = (T*)a.S + row * a.lds;
            float q[NC][VE];
#pragma unroll
            for (int i = 0; i < NC; ++i)
                if (i * G + lane < nvec) ldv<VE>(q[i], r + (i * G + lane) * VE);
            const uint32_t key = a.use_drop ? drop_key(a.drop, a.salt) : 0u;
#pragma unroll
            for (int i = 0; i < NC; ++i) {
                if (i * G + lane >= nvec) continue;
                const int c0 = (i * G + lane) * VE;
                float m[VE];
                if (a.use_drop) drop_vec<VE>(m, key, a.drop.thresh, a.drop.inv_keep, row * C + c0);
                // one rounding of x m + r to fp32, one to the storage type; what a 0 multiplies is gone even where it is not finite
#pragma unroll
                for (int e = 0; e < VE; ++e)
                    s[i][e] = Elem<T>::rnd(a.use_drop ? (m[e] == 0.f ? q[i][e] : fmaf(s[i][e], m[e], q[i][e])) : s[i][e] + q[i][e]);
                stv<VE>(so + c0, s[i]);
            }
        }
    }
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
        for (int e = 0; e < VE; ++e) t += s[i][e];
    const float inv = 1.f / (float)C;
    const float mean = group_sum<G>(t, red[0]) * inv;
    t = 0.f;
#pragma unroll
    for (int i = 0; i < NC; ++i)
        if (i * G + lane < nvec)
#pragma unroll
            for (int e = 0; e < VE; ++e) t = fmaf(s[i][e] - mean, s[i][e] - mean, t);
    const float rstd = 1.f / sqrtf(group_sum<G>(t, red[1]) * inv + a.eps);
    if (!on) return;
    T* y = (T*)a.Y + row * a.ldy;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        if (i * G + lane >= nvec) continue;
        const int c0 = (i * G + lane) * VE;
        float w[VE], b[VE];
#pragma unroll
        for (int e = 0; e < VE; ++e) {
            w[e] = a.gamma ? a.gamma[c0 + e] : 1.f;
            b[e] = a.beta ? a.beta[c0 + e] : 0.f;
        }
#pragma unroll
        for (int e = 0; e < VE; ++e) w[e] = fmaf((s[i][e] - mean) * rstd, w[e], b[e]);
        stv<VE>(y + c0, w);
    }
    if (a.mean && lane == 0) {
        a.mean[row] = mean;
        a.rstd[row] = rstd;
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
                const float m = drop_mul64(key, a.drop.thresh, a.drop.inv_keep, row * C + c);
                v = m == 0.f ? q : fmaf(v, m, q);
            } else {
                v += q;
            }
            v = Elem<T>::rnd(v);
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
template <typename T, int VE, int NC, int G>
__global__ void __launch_bounds__(G > 256 ? G : 256) norm_bwd_kernel(const NormArgs a) {
    constexpr int GPB = G > 256 ? 1 : 256 / G;
    constexpr int NT = G > 256 ? G : 256;
    __shared__ float red[2][2][G > 64 ? G / 64 : 1];
    __shared__ float meet[GPB > 1 ? NT * NC * VE : 1];
    const int lane = threadIdx.x % G, grp = threadIdx.x / G, C = a.C, nvec = C / VE;
    const float inv = 1.f / (float)C;
    const uint32_t key = a.use_drop ? drop_key(a.drop, a.salt) : 0u;
    float w0[NC][VE], w1[NC][VE];
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
        for (int e = 0; e < VE; ++e) w0[i][e] = w1[i][e] = 0.f;
    int par = 0;
    for (long r0 = (long)blockIdx.x * GPB; r0 < a.rows; r0 += (long)gridDim.x * GPB, par ^= 1) {        // (block-uniform: barriers inside)
        const long row = r0 + grp;
        const bool on = row < a.rows;
        float g[NC][VE], h[NC][VE], st[NC][VE];
#pragma unroll
        for (int i = 0; i < NC; ++i)
#pragma unroll
            for (int e = 0; e < VE; ++e) g[i][e] = h[i][e] = st[i][e] = 0.f;
        float mean = 0.f, rstd = 0.f;
        if (on) {
            mean = a.mean[row];
            rstd = a.rstd[row];
            if (a.dY) {
                const T* dy = (const T*)a.dY + row * a.lddy;
#pragma unroll
                for (int i = 0; i < NC; ++i)
                    if (i * G + lane < nvec) ldv<VE>(g[i], dy + (i * G + lane) * VE);
            }
            const T* s = (const T*)a.S + row * a.lds;
#pragma unroll
            for (int i = 0; i < NC; ++i)
                if (i * G + lane < nvec) ldv<VE>(h[i], s + (i * G + lane) * VE);
            if (a.dSt) {
                const T* d = (const T*)a.dSt + row * a.ldds;
#pragma unroll
                for (int i = 0; i < NC; ++i)
                    if (i * G + lane < nvec) ldv<VE>(st[i], d + (i * G + lane) * VE);
            }
        }
        float t0 = 0.f, t1 = 0.f;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            if (i * G + lane >= nvec) continue;
            const int c0 = (i * G + lane) * VE;
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                h[i][e] = (h[i][e] - mean) * rstd;
                w0[i][e] = fmaf(g[i][e], h[i][e], w0[i][e]);
                w1[i][e] += g[i][e];
                if (a.gamma) g[i][e] *= a.gamma[c0 + e];
                t0 += g[i][e];
                t1 = fmaf(g[i][e], h[i][e], t1);
            }
        }
        t0 = group_sum<G>(t0, red[par][0]) * inv;
        t1 = group_sum<G>(t1, red[par][1]) * inv;
        if (!on) continue;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            if (i * G + lane >= nvec) continue;
            const int c0 = (i * G + lane) * VE;
            float d[VE];
#pragma unroll
            for (int e = 0; e < VE; ++e) d[e] = fmaf(rstd, g[i][e] - t0 - h[i][e] * t1, st[i][e]);
            if (a.dS) stv<VE>((T*)a.dS + row * a.lddsum + c0, d);
            if (a.dX) {
                if (a.use_drop) {
                    float m[VE];
                    drop_vec<VE>(m, key, a.drop.thresh, a.drop.inv_keep, row * C + c0);
#pragma unroll
                    for (int e = 0; e < VE; ++e) d[e] = m[e] == 0.f ? 0.f : d[e] * m[e];
                }
                stv<VE>((T*)a.dX + row * a.lddx + c0, d);
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
        const float mean = a.mean[row], rstd = a.rstd[row];
        float t0 = 0.f, t1 = 0.f;
        for (int c = threadIdx.x; c < C; c += 1024) {
            const float y = dy ? Elem<T>::ld(dy + c) : 0.f, h = (Elem<T>::ld(s + c) - mean) * rstd, g = a.gamma ? y * a.gamma[c] : y;
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
            const float y = dy ? Elem<T>::ld(dy + c) : 0.f, h = (Elem<T>::ld(s + c) - mean) * rstd, g = a.gamma ? y * a.gamma[c] : y;
            float d = fmaf(rstd, g - t0 - h * t1, a.dSt ? Elem<T>::ld((const T*)a.dSt + row * a.ldds + c) : 0.f);
            if (a.dS) Elem<T>::st((T*)a.dS + row * a.lddsum + c, d);
            if (a.dX) {
                if (a.use_drop) {
                    const float m = drop_mul64(key, a.drop.thresh, a.drop.inv_keep, row * C + c);
                    d = m == 0.f ? 0.f : d * m;
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

int row_align(const void* p, long ld, int es, int ve) {
    while (ve > 1 && (p && (((uintptr_t)p % (uintptr_t)(ve * es)) || ld % ve))) ve >>= 1;
    return ve;
}

constexpr int LONG_BLOCKS = 256;
// blocks of the backward pass: each leaves a partial row of 2 C sums, so there are no more than one for every 64 KB or so it reads --
// the partial rows stay below an eighth of the tensors -- and no more than fill the card
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
    if (bwd) hipLaunchKernelGGL((norm_bwd_kernel<T, VE, NC, G>), dim3((unsigned)nblk), dim3(NT), 0, s, a);
    else hipLaunchKernelGGL((norm_fwd_kernel<T, VE, NC, G>), dim3((unsigned)((a.rows + GPB - 1) / GPB)), dim3(NT), 0, s, a);
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
