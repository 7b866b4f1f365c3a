// Rotary positions: pairs of channels of every head turned by the angle position * frequency.
//
//   (x_a, x_b) -> scale * (x_a cos - x_b sin, x_a sin + x_b cos),   angle = position * freq[f],   f < R / 2
//   half layout: (a, b) = (f, f + R / 2);  interleaved: (2 f, 2 f + 1);  channels R .. D are copied
//
// The backward pass is the same launch with the angle negated: a rotation's transpose.
// One pass over the data, bound by memory: a block first makes the cosines and sines of its tokens (one per token and frequency, in LDS; the
// angle is reduced to a fraction of a turn in 64 bits, so positions of millions keep 1e-7 of a turn), then streams every head of those tokens
// past them with up to 16 bytes per lane and access.  Without the LDS step each head would pay for its own cosines: at 40 heads of 128 that is
// 20 times the arithmetic.
#include "seq_common.h"

namespace {

constexpr int NTHR = 256;
constexpr int MAX_R2 = GAST_ROTARY_MAX_D / 2;

struct RotaryArgs {
    gast_rotary_job j[GAST_ROTARY_MAX_BATCH];
    const void* pos;
    const double* freqs;
    long pos_b, pos_t, ntok;
    int pos64, T, J, D, R, TT, RL;
    float scale, sign;
};

// VE: elements per access.  INTER with VE >= 2 turns VE / 2 pairs inside one vector; every other form turns VE pairs between two.
template <typename T, int VE, bool INTER>
__global__ void __launch_bounds__(NTHR) rotary_kernel(const RotaryArgs a) {
    __shared__ float2 cs[NTHR > MAX_R2 ? NTHR : MAX_R2];
    constexpr bool INSIDE = INTER && VE > 1;
    constexpr int NP = INSIDE ? VE / 2 : VE;         // pairs of a unit
    const gast_rotary_job& job = a.j[blockIdx.z];
    const int tid = threadIdx.x, R = a.R, R2 = R >> 1, D = a.D, H = job.H, rows = a.J * H;
    const long tok0 = (long)blockIdx.x * a.TT;
    const int ntok = (int)min((long)a.TT, a.ntok - tok0);
    for (int i = tid; i < ntok * R2; i += NTHR) {
        const int tt = i / R2, f = i - tt * R2;
        const long b = (tok0 + tt) / a.T, t = (tok0 + tt) - b * a.T, at = b * a.pos_b + t * a.pos_t;
        const double pos = a.pos64 ? (double)((const int64_t*)a.pos)[at] : (double)((const int32_t*)a.pos)[at];
        double turns = pos * a.freqs[f] * 0.15915494309189533577;       // 1 / (2 pi)
        turns -= rint(turns);
        float s, c;
        sincospif(2.f * (float)turns, &s, &c);
        cs[i] = make_float2(c * a.scale, s * a.scale * a.sign);
    }
    __syncthreads();
    // units of a row: the rotated ones, then the copied tail in pieces of the same size
    const int UP = R2 / NP, step = INSIDE ? VE : 2 * VE, UT = (D - R + step - 1) / step, U = UP + UT;
    const T* __restrict__ X = (const T*)job.x.p;
    T* __restrict__ Y = (T*)job.y.p;
    for (int idx = tid; idx < ntok * a.RL * U; idx += NTHR) {
        const int u = idx % U, q = idx / U, rl = q % a.RL, tt = q / a.RL;
        const long b = (tok0 + tt) / a.T, t = (tok0 + tt) - b * a.T;
        const bool turn = u < UP;
        int o0, o1;
        float c[NP], s[NP];
        if (turn) {
            o0 = INSIDE ? u * VE : INTER ? 2 * u : u * VE;
            o1 = INTER ? 2 * u + 1 : o0 + R2;
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                const float2 v = cs[tt * R2 + u * NP + i];
                c[i] = v.x; s[i] = v.y;
            }
        } else {
            o0 = R + (u - UP) * step;
            o1 = o0 + VE;
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
                stv<VE>(y + o0, w);
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
                stv<VE>(y + o0, w);
                if (two) stv<VE>(y + o1, w1);
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
    // vectors: as wide as every row's start and both parts of a row allow
    int ve = 16 / es, maxH = 1;
    for (int i = 0; i < n; ++i) {
        if (!jobs[i].x.p || !jobs[i].y.p || jobs[i].H < 1) return GAST_EINVAL;
        if ((long)J * jobs[i].H > (1L << 24)) return GAST_ERANGE;
        a.j[i] = jobs[i];
        const int ax = seq_align(jobs[i].x, es, ve), ay = seq_align(jobs[i].y, es, ve);
        ve = ax < ay ? ax : ay;
        if (jobs[i].H > maxH) maxH = jobs[i].H;
    }
    while (ve > 1 && ((interleaved ? R : R / 2) % ve || (D - R) % ve)) ve >>= 1;
    a.pos = positions; a.pos64 = pos64; a.pos_b = pos_b; a.pos_t = pos_t;
    a.freqs = freqs; a.scale = scale; a.sign = backward ? -1.f : 1.f;
    a.T = T; a.J = J; a.D = D; a.R = R; a.ntok = (long)B * T;
    const int R2 = R / 2, np = interleaved && ve > 1 ? ve / 2 : ve, step = interleaved && ve > 1 ? ve : 2 * ve;
    const int U = R2 / np + (D - R + step - 1) / step;
    a.TT = R2 >= NTHR ? 1 : NTHR / R2 > 16 ? 16 : NTHR / R2;
    if (a.TT > a.ntok) a.TT = (int)a.ntok;
    a.RL = NTHR / (a.TT * U) > 1 ? NTHR / (a.TT * U) : 1;
    const long bx = (a.ntok + a.TT - 1) / a.TT;
    if (bx > 0x7fffffffL) return GAST_ERANGE;
    // few tokens: the rows of a token are split over blocks, each of which makes the cosines again
    const int maxsplit = (int)(((long)J * maxH + a.RL - 1) / a.RL);
    long by = 1024 / (bx * n);
    by = by < 1 ? 1 : by > maxsplit ? maxsplit : by;
    const dim3 grid((unsigned)bx, (unsigned)by, (unsigned)n);
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
