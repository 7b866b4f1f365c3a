// Rotary positions: pairs of channels of every head turned by the angle position * frequency.
//
//   (x_a, x_b) -> scale * (x_a cos - x_b sin, x_a sin + x_b cos),   angle = position * freq[f],   f < R / 2
//   half layout: (a, b) = (f, f + R / 2);  interleaved: (2 f, 2 f + 1);  channels R .. D are copied
//
// The backward pass is the same launch with the angle negated: a rotation's transpose.
// One pass over the data, bound by memory: a block first makes the cosines and sines of its tokens (one per token and frequency, in LDS; the
// angle is reduced to a fraction of a turn in 64 bits, so positions of millions keep 1e-7 of a turn), then streams every head of those tokens
// past them with up to 16 bytes per lane and access.  Without the LDS step each head would pay for its own cosines: at 40 heads of 128 that is
// 20 times the arithmetic.  Measured: 16384 tokens of 32 + 8 heads of 128 channels, 64 of them turned (bf16): 67 us, 5.0 TB/s, what a copy reaches.
#include "seq_common.h"

namespace {

constexpr int NTHR = 256;
constexpr int MAX_CS = 1024;                         // cosines of a block: one token of the longest heads, or several
static_assert(MAX_CS >= GAST_ROTARY_MAX_D / 2, "a token's cosines");

struct RotaryArgs {
    gast_rotary_job j[GAST_ROTARY_MAX_BATCH];
    const void* pos;
    const double* freqs;
    long pos_b, pos_t, ntok;
    int n, pos64, T, J, D, R, TT, RL;
    float scale, sign;
};

// v[i ..] to y[i ..], i > 0 where a vector's first elements are somebody else's
template <int VE, typename T> __device__ __forceinline__ void put(T* y, const float (&v)[VE], int first) {
    if (first <= 0) {
        stv<VE>(y, v);
        return;
    }
#pragma unroll
    for (int i = 1; i < VE; ++i)
        if (i >= first) Elem<T>::st(y + i, v[i]);
}

// VE: elements per access.  INTER with VE >= 2 turns VE / 2 pairs inside one vector; every other form turns VE pairs between two.
// Where the channels are not a multiple of VE the last vector starts earlier, and only what the one before it leaves is stored.
template <typename T, int VE, bool INTER>
__global__ void __launch_bounds__(NTHR) rotary_kernel(const RotaryArgs a) {
    __shared__ float2 cs[MAX_CS];
    constexpr bool INSIDE = INTER && VE > 1;
    constexpr int NP = INSIDE ? VE / 2 : VE;         // pairs of a unit
    const int tid = threadIdx.x, R = a.R, R2 = R >> 1, D = a.D;
    const long tok0 = (long)blockIdx.x * a.TT;
    const int ntok = (int)min((long)a.TT, a.ntok - tok0);
    const long b0 = tok0 / a.T;
    const uint32_t t0 = (uint32_t)(tok0 - b0 * a.T);
    for (int i = tid; i < ntok * R2; i += NTHR) {
        const int tt = i / R2, f = i - tt * R2;
        const uint32_t db = (t0 + tt) / (uint32_t)a.T, t = t0 + tt - db * (uint32_t)a.T;
        const long at = (b0 + db) * a.pos_b + t * a.pos_t;
        const double pos = a.pos64 ? (double)((const int64_t*)a.pos)[at] : (double)((const int32_t*)a.pos)[at];
        double turns = pos * a.freqs[f] * 0.15915494309189533577;       // 1 / (2 pi)
        turns -= rint(turns);
        const float near = (float)turns, rest = 6.28318531f * (float)(turns - (double)near);       // (what fp32 leaves of the angle: small sines keep their bits)
        float s, c;
        sincospif(2.f * near, &s, &c);
        cs[i] = make_float2(fmaf(-rest, s, c) * a.scale, fmaf(rest, c, s) * a.scale * a.sign);
    }
    __syncthreads();
    // units of a row: the rotated ones, then the copied tail in pieces of the same size
    const int UP = (R2 + NP - 1) / NP, step = INSIDE ? VE : 2 * VE, UT = (D - R + step - 1) / step, U = UP + UT;
    for (int z = blockIdx.z; z < a.n; z += gridDim.z) {
        const gast_rotary_job& job = a.j[z];
        const int H = job.H, rows = a.J * H;
        const T* __restrict__ X = (const T*)job.x.p;
        T* __restrict__ Y = (T*)job.y.p;
        for (int idx = tid; idx < ntok * a.RL * U; idx += NTHR) {
            const int u = idx % U, q = idx / U, rl = q % a.RL, tt = q / a.RL;
            const uint32_t db = (t0 + tt) / (uint32_t)a.T;
            const long b = b0 + db, t = t0 + tt - db * (uint32_t)a.T;
            const bool turn = u < UP;
            int o0, o1, skip0 = 0, skip1 = 0;            // where the vectors start, and how much of them is not this unit's
            float c[NP], s[NP];
            if (turn) {
                const int p = min(u * NP, R2 - NP), twice = INTER ? 2 : 1;
                o0 = p * twice;
                o1 = INTER ? o0 + 1 : o0 + R2;
                skip0 = skip1 = (u * NP - p) * (INSIDE ? 2 : 1);
#pragma unroll
                for (int i = 0; i < NP; ++i) {
                    const float2 v = cs[tt * R2 + p + i];
                    c[i] = v.x; s[i] = v.y;
                }
            } else {
                const int e0 = R + (u - UP) * step, e1 = e0 + VE;
                o0 = min(e0, D - VE);
                o1 = e1 < D ? min(e1, D - VE) : D;
                skip0 = e0 - o0;
                skip1 = e1 - o1;
#pragma unroll
                for (int i = 0; i < NP; ++i) c[i] = 1.f, s[i] = 0.f;
            }
            const bool two = !INSIDE && o1 < D;
            const long xb = b * job.x.b + t * job.x.t, yb = b * job.y.b + t * job.y.t;
#pragma unroll 2
            for (int r = rl + a.RL * blockIdx.y; r < rows; r += a.RL * gridDim.y) {
                const int j = r / H, h = r - j * H;
                const T* x = X + xb + j * job.x.j + h * job.x.h;
                T* y = Y + yb + j * job.y.j + h * job.y.h;
                float p[VE], w[VE];
                ldv<VE>(p, x + o0);
                if constexpr (INSIDE) {
#pragma unroll
                    for (int i = 0; i < VE; i += 2) {
                        w[i] = turn ? p[i] * c[i / 2] - p[i + 1] * s[i / 2] : p[i];           // (a copy, not a turn by zero: infinities stay)
                        w[i + 1] = turn ? p[i] * s[i / 2] + p[i + 1] * c[i / 2] : p[i + 1];
                    }
                    put<VE>(y + o0, w, skip0);
                } else {
                    float p1[VE], w1[VE];
#pragma unroll
                    for (int i = 0; i < VE; ++i) p1[i] = 0.f;
                    if (two) ldv<VE>(p1, x + o1);
#pragma unroll
                    for (int i = 0; i < VE; ++i) {
                        w[i] = turn ? p[i] * c[i] - p1[i] * s[i] : p[i];
                        w1[i] = turn ? p[i] * s[i] + p1[i] * c[i] : p1[i];
                    }
                    put<VE>(y + o0, w, skip0);
                    if (two) put<VE>(y + o1, w1, skip1);
                }
            }
        }
    }
}

template <typename T, int VE>
void launch(const RotaryArgs& a, int interleaved, dim3 grid, hipStream_t s) {
    if (interleaved) hipLaunchKernelGGL((rotary_kernel<T, VE, true>), grid, dim3(NTHR), 0, s, a);
    else hipLaunchKernelGGL((rotary_kernel<T, VE, false>), grid, dim3(NTHR), 0, s, a);
}

}  // namespace

extern "C" int gast_rotary_multi(int dtype, const gast_rotary_job* jobs, int n, int B, int T, int J, int D, int R, int interleaved,
                                 const void* positions, int pos64, long pos_b, long pos_t, const double* freqs, float scale, int backward,
                                 gast_stream_t stream) {
    if (!jobs || n < 1 || n > GAST_ROTARY_MAX_BATCH || !positions || !freqs || B < 1 || T < 1 || J < 1 || R < 2 || (R & 1) || R > D) return GAST_EINVAL;
    if (D > GAST_ROTARY_MAX_D) return GAST_ERANGE;
    if (dtype != GAST_F32 && dtype != GAST_BF16) return GAST_EINVAL;
    RotaryArgs a;
    const int es = dtype == GAST_F32 ? 4 : 2;
    // vectors: as wide as both parts of a row allow (their starts need no alignment)
    int ve = 16 / es, maxH = 1;
    for (int i = 0; i < n; ++i) {
        if (!jobs[i].x.p || !jobs[i].y.p || jobs[i].H < 1) return GAST_EINVAL;
        if ((long)J * jobs[i].H > (1L << 24)) return GAST_ERANGE;
        a.j[i] = jobs[i];
        if (jobs[i].H > maxH) maxH = jobs[i].H;
    }
    while (ve > 1 && ((interleaved ? R : R / 2) < ve || (D > R && D - R < ve))) ve >>= 1;
    a.n = n; a.pos = positions; a.pos64 = pos64; a.pos_b = pos_b; a.pos_t = pos_t;
    a.freqs = freqs; a.scale = scale; a.sign = backward ? -1.f : 1.f;
    a.T = T; a.J = J; a.D = D; a.R = R; a.ntok = (long)B * T;
    const int R2 = R / 2, np = interleaved && ve > 1 ? ve / 2 : ve, step = interleaved && ve > 1 ? ve : 2 * ve;
    const int U = (R2 + np - 1) / np + (D - R + step - 1) / step;
    // tokens of a block: four units of the longest job a thread or more, while 2048 blocks are left
    long tt = (4L * NTHR + (long)J * maxH * U - 1) / ((long)J * maxH * U);
    if (tt < NTHR / R2) tt = NTHR / R2;
    if (tt > MAX_CS / R2) tt = MAX_CS / R2;
    if (tt > 16 && tt > a.ntok / 2048) tt = a.ntok / 2048 > 16 ? a.ntok / 2048 : 16;
    a.TT = (int)(tt > a.ntok ? a.ntok : tt);
    a.RL = NTHR / (a.TT * U) > 1 ? NTHR / (a.TT * U) : 1;
    const long bx = (a.ntok + a.TT - 1) / a.TT;
    if (bx > 0x7fffffffL) return GAST_ERANGE;
    // few tokens: the rows of a token are split over blocks, each of which makes the cosines again
    const int maxsplit = (int)(((long)J * maxH + a.RL - 1) / a.RL);
    long by = 1024 / (bx * n);
    by = by < 1 ? 1 : by > maxsplit ? maxsplit : by;
    // few heads and many tokens: a block turns all jobs by the cosines it has made (497k tokens of 2 + 2 heads of 14 channels, fp32: 237 -> 140 us
    // both ways, with more tokens a block).  With many heads the cosines are cheap and blocks of one job are faster (32 + 8 heads of 128: 75 against 67 us).
    const bool share = 4L * R2 > (long)J * maxH * U && bx * by >= 1024;
    const dim3 grid((unsigned)bx, (unsigned)by, (unsigned)(share ? 1 : n));
    const hipStream_t s = (hipStream_t)stream;
    if (dtype == GAST_F32) {
        if (ve == 4) launch<float, 4>(a, interleaved, grid, s);
        else if (ve == 2) launch<float, 2>(a, interleaved, grid, s);
        else launch<float, 1>(a, interleaved, grid, s);
    } else {
        if (ve == 8) launch<bf16_t, 8>(a, interleaved, grid, s);
        else if (ve == 4) launch<bf16_t, 4>(a, interleaved, grid, s);
        else if (ve == 2) launch<bf16_t, 2>(a, interleaved, grid, s);
        else launch<bf16_t, 1>(a, interleaved, grid, s);
    }
    GAST_CHECK_LAUNCH();
    return 0;
}
