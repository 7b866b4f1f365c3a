// Causal linear attention with a decay for each head, forward, backward and one token at a time.
//
//   S_t = lambda S_(t-1) + k_t v_t',   o_t = scale q_t' S_t,   lambda = exp(log_decay)
//
// Every pass is one recurrence in three roles,   out_i = oscale * a_i' X_i,   X_i = lambda X_(i-1) + bscale * b_i c_i' :
//   o   a = q,  b = k,  c = v    forward in time            dq  a = do, b = v,  c = k    forward in time (X = S')
//   dv  a = k,  b = q,  c = do   backward in time           dk  a = v,  b = do, c = q    backward in time (X = the transposed one of dv)
// Forward in time the carry is decayed before it is used (o_t sees lambda S_(t-1)), backward in time the gradient of the last state is
// used as it is and the decay follows: d state = lambda * (the recurrence's end).
#include "seq_common.h"

namespace {

struct ScanArgs {
    gast_seq a, b, c, out;
    const float* xin;        // [B][J][H][D1][D2] (xin_t: [D2][D1]), or null: zero
    float* xout;             // [B][J][H][D1][D2] or null
    const float* log_decay;
    const int32_t* lengths;
    int B, T, J, H, D1, D2, xin_t, reverse;
    float bscale, oscale;
};

constexpr int TS = 16;       // tokens staged at a time
constexpr int EC = 64;       // columns of X that a block owns

// The recurrence as it stands: a block owns EC columns of one head's X; wave p holds rows 32 p .. 32 p + 31 of them in registers.
template <typename T>
__global__ void __launch_bounds__(256) scan_kernel(const ScanArgs p) {
    __shared__ float sa[TS][GAST_DECAY_MAX_D], sb[TS][GAST_DECAY_MAX_D], sc[TS][EC], so[4][TS][EC];
    const int tid = threadIdx.x, e = tid & 63, w = tid >> 6, D1 = p.D1, D2 = p.D2;
    const int nct = (D2 + EC - 1) / EC, ct = blockIdx.x % nct, e0 = ct * EC;
    const long hd = blockIdx.x / nct;                   // (b, j, h)
    const int h = (int)(hd % p.H), j = (int)(hd / p.H % p.J);
    const long b = hd / p.H / p.J;
    const float lam = expf(p.log_decay[h]);
    const int len = p.lengths ? min(max(p.lengths[b], 0), p.T) : p.T;
    const bool col = e0 + e < D2;
    float X[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) {
        const int d = w * 32 + i;
        X[i] = 0.f;
        if (p.xin && d < D1 && col) X[i] = p.xin[hd * D1 * D2 + (p.xin_t ? (long)(e0 + e) * D1 + d : (long)d * D2 + e0 + e)];
        if (!p.reverse && len) X[i] *= lam;
    }
    const T *A = (const T*)p.a.p + seq_at(p.a, b, 0, j, h), *Bp = (const T*)p.b.p + seq_at(p.b, b, 0, j, h), *Cp = (const T*)p.c.p + seq_at(p.c, b, 0, j, h);
    T* O = (T*)p.out.p + seq_at(p.out, b, 0, j, h);
    for (int t0 = 0; t0 < len; t0 += TS) {
        const int n = min(TS, len - t0);
        for (int i = tid; i < n * D1; i += 256) {
            const int q = i / D1, d = i - q * D1, t = p.reverse ? len - 1 - t0 - q : t0 + q;
            sa[q][d] = Elem<T>::ld(A + t * p.a.t + d);
            sb[q][d] = Elem<T>::ld(Bp + t * p.b.t + d) * p.bscale;
        }
        for (int i = tid; i < n * EC; i += 256) {
            const int q = i / EC, c = i - q * EC, t = p.reverse ? len - 1 - t0 - q : t0 + q;
            sc[q][c] = e0 + c < D2 ? Elem<T>::ld(Cp + t * p.c.t + e0 + c) : 0.f;
        }
        __syncthreads();
        for (int q = 0; q < n; ++q) {
            const float c = sc[q][e];
            float o = 0.f;
            const bool decay = t0 + q > 0;
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                const int d = w * 32 + i;
                if (d < D1) {
                    X[i] = fmaf(sb[q][d], c, decay ? lam * X[i] : X[i]);
                    o = fmaf(sa[q][d], X[i], o);
                }
            }
            so[w][q][e] = o;
        }
        __syncthreads();
        for (int i = tid; i < n * EC; i += 256) {
            const int q = i / EC, c = i - q * EC, t = p.reverse ? len - 1 - t0 - q : t0 + q;
            if (e0 + c < D2) Elem<T>::st(O + t * p.out.t + e0 + c, p.oscale * (so[0][q][c] + so[1][q][c] + so[2][q][c] + so[3][q][c]));
        }
    }
    for (long i = tid; i < (long)(p.T - len) * EC; i += 256) {
        const long t = len + i / EC;
        const int c = (int)(i % EC);
        if (e0 + c < D2) Elem<T>::st(O + t * p.out.t + e0 + c, 0.f);
    }
    if (p.xout && col)
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            const int d = w * 32 + i;
            if (d < D1) p.xout[hd * D1 * D2 + (long)d * D2 + e0 + e] = p.reverse && len ? lam * X[i] : X[i];
        }
}

template <typename T>
int scan(const ScanArgs& p, hipStream_t s) {
    const long blocks = (long)p.B * p.J * p.H * ((p.D2 + EC - 1) / EC);
    if (blocks > 0x7fffffffL) return GAST_ERANGE;
    hipLaunchKernelGGL((scan_kernel<T>), dim3((unsigned)blocks), dim3(256), 0, s, p);
    GAST_CHECK_LAUNCH();
    return 0;
}

// One token: a block per head, the state is read and written once (that is the whole cost: 8 Dk Dv bytes), VE columns a thread, the rows
// spread over the other threads and summed through LDS.
template <typename T, int VE>
__global__ void __launch_bounds__(256) step_kernel(const gast_decay_args p) {
    __shared__ float sq[GAST_DECAY_MAX_D], sk[GAST_DECAY_MAX_D], so[256 * VE];
    const int tid = threadIdx.x, Dk = p.Dk, Dv = p.Dv, nv = Dv / VE;
    const long hd = blockIdx.x;
    const int h = (int)(hd % p.H), j = (int)(hd / p.H % p.J);
    const long b = hd / p.H / p.J;
    T* O = (T*)p.o.p + seq_at(p.o, b, 0, j, h);
    if (p.lengths && p.lengths[b] < 1) {
        for (int e = tid; e < Dv; e += 256) Elem<T>::st(O + e, 0.f);
        return;
    }
    const T *Q = (const T*)p.q.p + seq_at(p.q, b, 0, j, h), *K = (const T*)p.k.p + seq_at(p.k, b, 0, j, h), *V = (const T*)p.v.p + seq_at(p.v, b, 0, j, h);
    for (int d = tid; d < Dk; d += 256) {
        sq[d] = Elem<T>::ld(Q + d) * p.scale;
        sk[d] = Elem<T>::ld(K + d);
    }
    __syncthreads();
    const float lam = expf(p.log_decay[h]);
    const int rows = 256 / nv, c = tid % nv, r0 = tid / nv;
    float* S = (float*)p.state + hd * Dk * Dv + c * VE;
    float o[VE], v[VE];
#pragma unroll
    for (int i = 0; i < VE; ++i) o[i] = 0.f;
    if (r0 < rows) {
#pragma unroll
        for (int i = 0; i < VE; ++i) v[i] = Elem<T>::ld(V + c * VE + i);
#pragma unroll 8
        for (int d = r0; d < Dk; d += rows) {
            float x[VE];
            ldv<VE>(x, S + d * Dv);
#pragma unroll
            for (int i = 0; i < VE; ++i) {
                x[i] = fmaf(sk[d], v[i], lam * x[i]);
                o[i] = fmaf(sq[d], x[i], o[i]);
            }
            stv<VE>(S + d * Dv, x);
        }
#pragma unroll
        for (int i = 0; i < VE; ++i) so[(r0 * nv + c) * VE + i] = o[i];
    }
    __syncthreads();
    for (int e = tid; e < Dv; e += 256) {
        float t = 0.f;
        for (int r = 0; r < rows; ++r) t += so[r * Dv + e];
        Elem<T>::st(O + e, t);
    }
}

int check(const gast_decay_args* p) {
    if (!p || p->B < 1 || p->T < 1 || p->J < 1 || p->H < 1 || p->Dk < 1 || p->Dv < 1 || !p->log_decay) return GAST_EINVAL;
    if (p->dtype != GAST_F32 && p->dtype != GAST_BF16) return GAST_EINVAL;
    if (!p->q.p || !p->k.p || !p->v.p) return GAST_EINVAL;
    if (p->Dk > GAST_DECAY_MAX_D || p->Dv > GAST_DECAY_MAX_D) return GAST_ERANGE;
    return 0;
}

ScanArgs roles(const gast_decay_args& g, const gast_seq& a, const gast_seq& b, const gast_seq& c, const gast_seq& out, int D1, int D2) {
    ScanArgs p = {};
    p.a = a; p.b = b; p.c = c; p.out = out; p.D1 = D1; p.D2 = D2;
    p.log_decay = g.log_decay; p.lengths = g.lengths; p.B = g.B; p.T = g.T; p.J = g.J; p.H = g.H;
    p.bscale = p.oscale = 1.f;
    return p;
}

template <typename T>
int forward(const gast_decay_args& g, hipStream_t s) {
    ScanArgs p = roles(g, g.q, g.k, g.v, g.o, g.Dk, g.Dv);
    p.xin = g.state; p.xout = g.state_out; p.oscale = g.scale;
    return scan<T>(p, s);
}

template <typename T>
int backward(const gast_decay_args& g, hipStream_t s) {
    ScanArgs p = roles(g, g.d_o, g.v, g.k, g.dq, g.Dv, g.Dk);
    p.xin = g.state; p.xin_t = 1; p.oscale = g.scale;
    if (int rc = scan<T>(p, s)) return rc;
    p = roles(g, g.k, g.q, g.d_o, g.dv, g.Dk, g.Dv);
    p.reverse = 1; p.xin = g.dstate_out; p.xout = g.dstate; p.bscale = g.scale;
    if (int rc = scan<T>(p, s)) return rc;
    p = roles(g, g.v, g.d_o, g.q, g.dk, g.Dv, g.Dk);
    p.reverse = 1; p.xin = g.dstate_out; p.xin_t = 1; p.bscale = g.scale;
    return scan<T>(p, s);
}

}  // namespace

extern "C" int gast_decay_fwd(const gast_decay_args* args, gast_stream_t stream) {
    if (int rc = check(args)) return rc;
    if (!args->o.p) return GAST_EINVAL;
    return args->dtype == GAST_F32 ? forward<float>(*args, (hipStream_t)stream) : forward<bf16_t>(*args, (hipStream_t)stream);
}

extern "C" int gast_decay_bwd(const gast_decay_args* args, gast_stream_t stream) {
    if (int rc = check(args)) return rc;
    if (!args->d_o.p || !args->dq.p || !args->dk.p || !args->dv.p) return GAST_EINVAL;
    return args->dtype == GAST_F32 ? backward<float>(*args, (hipStream_t)stream) : backward<bf16_t>(*args, (hipStream_t)stream);
}

extern "C" long gast_decay_ws_floats(int B, int T, int J, int H, int Dk, int Dv, int backward) { return 0; }

extern "C" int gast_decay_step(const gast_decay_args* args, gast_stream_t stream) {
    if (int rc = check(args)) return rc;
    if (!args->o.p || !args->state || args->T != 1) return GAST_EINVAL;
    const gast_decay_args& g = *args;
    const long blocks = (long)g.B * g.J * g.H;
    if (blocks > 0x7fffffffL) return GAST_ERANGE;
    const int ve = ((uintptr_t)g.state % 16 == 0 && g.Dv % 4 == 0) ? 4 : 1;
    const hipStream_t s = (hipStream_t)stream;
    const dim3 grid((unsigned)blocks), blk(256);
    if (g.dtype == GAST_F32) {
        if (ve == 4) hipLaunchKernelGGL((step_kernel<float, 4>), grid, blk, 0, s, g);
        else hipLaunchKernelGGL((step_kernel<float, 1>), grid, blk, 0, s, g);
    } else {
        if (ve == 4) hipLaunchKernelGGL((step_kernel<bf16_t, 4>), grid, blk, 0, s, g);
        else hipLaunchKernelGGL((step_kernel<bf16_t, 1>), grid, blk, 0, s, g);
    }
    GAST_CHECK_LAUNCH();
    return 0;
}
