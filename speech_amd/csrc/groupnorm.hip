// Group normalisation with an activation, channels last, forward and backward:
//     y = act( (x - mean) * rstd * gamma[c] + beta[c] + residual ),   act = identity, ReLU or SiLU,
// mean and rstd over the positions and the C / G channels of one (sample, group).  x is [N][F][T][C] with unit channel stride; with
// `lengths` only frames t < lengths[n] count and are written as values, the others become zero.  The batch-independent normalisation of
// the conv stack's blocks (the reference normalises those over the batch, net.py:24-25) and of a recurrent layer's output.
//
// HBM-bound: forward reads x (and the residual) and writes y; the statistics need x before the first output, so x is read twice -- the
// second time from the Infinity Cache at the conv stack's size (61 MB).  The backward reads gy, x and the residual twice for the same reason.
// Measured at [32][40][751][32] bf16 with SiLU and residual: statistics 18.6 us, apply 32 (5.8 TB/s), backward statistics 44 (5.6), backward
// apply 43 (5.7); rows, 24032 x 1024 bf16, 8 groups: forward 22 us (4.5 TB/s), backward 36 (4.1) + 7.4 for the parameters' gradients.
// Two routes, chosen by the shape alone:
//   rows    one position a sample (F * T == 1): a (sample, group) is a contiguous segment that a team of lanes holds in registers; one
//           read, one write, two-pass statistics.
//   blocks  everything else: a statistics kernel over (sample, split) and an apply kernel that merges the splits' partials itself.
// Statistics: a thread takes kU positions at a time as a triple (count, mean, M2 around that mean) and adds it to its own by Chan's formula;
// triples of threads and splits are merged as sums of w * mean and of M2 + w * (mean - mean_all)^2.  Every term of M2 is positive and nothing
// is subtracted from it: a large mean costs no digits, nor does a click, in the first frame or elsewhere.  (One sum of squares of differences to
// the first value lost them where that value was the click: 1.4e-4 of rstd after 469 positions.)  All sums are f32 in a fixed order.
#include "common.h"

namespace sp {

constexpr int kGnMaxC = 2048;
constexpr int kGnThreads = 256;
constexpr int kGnMaxSplit = 64;

struct GnShape {
    int N, F, T, C, G, Cg, act;
    const int32_t* lengths;
};
struct GnStr { int64_t n, f, t; };

template <typename T, int VW> struct alignas(sizeof(T) * VW) GnRaw { T e[VW]; };

template <typename T, int VW> __device__ __forceinline__ void gn_ld(const T* p, float (&f)[VW]) {
    const GnRaw<T, VW> r = *reinterpret_cast<const GnRaw<T, VW>*>(p);
#pragma unroll
    for (int i = 0; i < VW; ++i) f[i] = Elem<T>::f(r.e[i]);
}
template <typename T, int VW> __device__ __forceinline__ void gn_get(const GnRaw<T, VW>& r, float (&f)[VW]) {
#pragma unroll
    for (int i = 0; i < VW; ++i) f[i] = Elem<T>::f(r.e[i]);
}
template <typename T, int VW> __device__ __forceinline__ void gn_st(T* p, const float (&f)[VW]) {
    GnRaw<T, VW> r;
#pragma unroll
    for (int i = 0; i < VW; ++i) Elem<T>::st(&r.e[i], f[i]);
    *reinterpret_cast<GnRaw<T, VW>*>(p) = r;
}

// v_rcp_f32 is good to one unit in the last place; the exact division costs ten instructions an element
template <int VW> __device__ __forceinline__ void gn_act(float (&v)[VW], int act) {
    if (act == SP_ACT_RELU) {
#pragma unroll
        for (int i = 0; i < VW; ++i) v[i] = v[i] <= 0.f ? 0.f : v[i];   // NaN stays NaN
    } else if (act == SP_ACT_SILU) {
#pragma unroll
        for (int i = 0; i < VW; ++i) v[i] *= __builtin_amdgcn_rcpf(1.f + __expf(-v[i]));
    }
}
// g *= act'(pre)
template <int VW> __device__ __forceinline__ void gn_act_grad(float (&g)[VW], const float (&pre)[VW], int act) {
    if (act == SP_ACT_RELU) {
#pragma unroll
        for (int i = 0; i < VW; ++i) g[i] = pre[i] > 0.f ? g[i] : 0.f;
    } else if (act == SP_ACT_SILU) {
#pragma unroll
        for (int i = 0; i < VW; ++i) {
            const float s = __builtin_amdgcn_rcpf(1.f + __expf(-pre[i]));
            g[i] *= s * (1.f + pre[i] * (1.f - s));
        }
    }
}

// Positions [lo, hi) of a sample walked by rows of threads, kU positions at a time: their loads are all in flight before the first is used
// (one position at a time moved 2.3-2.8 TB/s on the 61 MB tensors of the conv stack).  Offsets advance by additions; a tensor whose frames
// follow each other through the bands (the usual layout) needs no correction at a band's end.
constexpr int kU = 4, kUb = 1;      // forward; backward (three tensors and the channel sums in registers)
struct GnWalk {
    int p, hi, step, t, dt, T;
    __device__ __forceinline__ GnWalk(int p_, int hi_, int step_, int T_) : p(p_), hi(hi_), step(step_), t(p_ % T_), dt(step_ % T_), T(T_) {}
    __device__ __forceinline__ bool more() const { return p < hi; }
};
struct GnPos {          // offsets of one tensor along a walk
    int64_t off, inc, wrap, first;
    __device__ __forceinline__ GnPos(GnStr s, int n, const GnWalk& w)
        : off(n * s.n + (int64_t)(w.p / w.T) * s.f + (int64_t)w.t * s.t), inc((int64_t)(w.step / w.T) * s.f + (int64_t)w.dt * s.t), wrap(s.f - (int64_t)w.T * s.t), first(off) {}
    // a position outside (behind the walk's end or the utterance's) is loaded from the walk's first position instead, and not used
    __device__ __forceinline__ int64_t at(bool in) const { return in ? off : first; }
    __device__ __forceinline__ void next(bool wrapped) { off += inc + (wrapped ? wrap : 0); }
};

template <typename... P> __device__ __forceinline__ void gn_next(GnWalk& w, P&... pos) {
    w.p += w.step;
    w.t += w.dt;
    const bool wrapped = w.t >= w.T;
    if (wrapped) w.t -= w.T;
    (pos.next(wrapped), ...);
}

// For groups g0 .. g1: sums of part(g, lane, width) over the lanes of a wave, handed to done(g, sum) in one lane.  Waves take the groups in
// turn: with one thread a group, the walk over 64 partial results alone took 30 us (each load waited for the one before).
__device__ __forceinline__ float gn_wave_sum(float v) {      // sums over 16 lanes by rotations inside the register, then over the four rows
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x128, 0xf, 0xf, false));
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x124, 0xf, 0xf, false));
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x122, 0xf, 0xf, false));
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x121, 0xf, 0xf, false));
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}
template <typename A, typename B> __device__ __forceinline__ void gn_group_sums(int g0, int g1, A&& part, B&& done) {
    const int lane = threadIdx.x & 63;
    for (int g = g0 + (int)(threadIdx.x >> 6); g <= g1; g += kGnThreads / 64) {
        const float v = gn_wave_sum(part(g, lane, 64));
        if (lane == 0) done(g, v);
    }
}

// Sums of every thread's NV values over the rows (threads cpb apart) that hold the same chunk.  They end in red[w * cpb * NV + chunk * NV + i],
// to be added over the w < (the result) that is returned: one per wave where a wave holds whole rows (sums by lane exchange, one barrier;
// the tree through LDS that other widths take has eight), one otherwise.
template <int NV> __device__ __forceinline__ int gn_row_sums(float (&v)[NV], float* red, int cpb, int row, int rows) {
    if (cpb <= 64 && (cpb & (cpb - 1)) == 0) {
        for (int o = cpb; o < 64; o <<= 1)
#pragma unroll
            for (int i = 0; i < NV; ++i) v[i] += __shfl_xor(v[i], o);
        const int lane = threadIdx.x & 63;
        if (lane < cpb)
#pragma unroll
            for (int i = 0; i < NV; ++i) red[((threadIdx.x >> 6) * cpb + lane) * NV + i] = v[i];
        __syncthreads();
        return kGnThreads / 64;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) red[threadIdx.x * NV + i] = v[i];
    __syncthreads();
    for (int o = 128; o > 0; o >>= 1) {
        if (row < o && row + o < rows) {
#pragma unroll
            for (int i = 0; i < NV; ++i) red[threadIdx.x * NV + i] += red[(threadIdx.x + o * cpb) * NV + i];
        }
        __syncthreads();
    }
    return 1;
}

// ---- block route --------------------------------------------------------------------------------------
// thread = (row, chunk of VW channels); a chunk lies inside a group or holds whole groups
template <typename T, int VW>
__global__ __launch_bounds__(kGnThreads) void gn_stats_kernel(const T* __restrict__ x, GnStr xs, GnShape s, int nsplit,
                                                              float* __restrict__ part) {
    __shared__ float red[kGnThreads * VW];
    __shared__ float gmean[kGnMaxC];
    const int n = blockIdx.x / nsplit, split = blockIdx.x % nsplit;
    const int P = s.F * s.T, nch = s.C / VW;
    const int per = (P + nsplit - 1) / nsplit, lo = split * per, hi = min(P, lo + per);
    const int len = s.lengths ? min(max(s.lengths[n], 0), s.T) : s.T;
    const int cpb = min(nch, kGnThreads);                 // chunks walked at a time
    const int rows = kGnThreads / cpb, row = threadIdx.x / cpb;
    for (int cb = 0; cb < nch; cb += cpb) {
        const int chunk = cb + threadIdx.x % cpb;
        const bool on = row < rows && chunk < nch;
        float mean[VW], sq[VW];
        int cnt = 0;
#pragma unroll
        for (int i = 0; i < VW; ++i) { mean[i] = 0.f; sq[i] = 0.f; }
        if (on) {
            const T* base = x + chunk * VW;
            GnWalk w(lo + row, hi, rows, s.T);
            GnPos px(xs, n, w);
            while (w.more()) {
                GnRaw<T, VW> raw[kU];
                bool on[kU];
                int nb = 0;
#pragma unroll
                for (int u = 0; u < kU; ++u) {
                    on[u] = w.more() && w.t < len;
                    nb += on[u];
                    raw[u] = *reinterpret_cast<const GnRaw<T, VW>*>(base + px.at(on[u]));
                    gn_next(w, px);
                }
                if (nb == 0) continue;
                const float rb = 1.f / (float)nb, part = (float)nb / (float)(cnt + nb), rest = (float)cnt * part;
                cnt += nb;
                float mb[VW], d[kU][VW];
#pragma unroll
                for (int i = 0; i < VW; ++i) mb[i] = 0.f;
#pragma unroll
                for (int u = 0; u < kU; ++u) {
                    gn_get<T, VW>(raw[u], d[u]);
#pragma unroll
                    for (int i = 0; i < VW; ++i) {
                        d[u][i] = on[u] ? d[u][i] : 0.f;
                        mb[i] += d[u][i];
                    }
                }
#pragma unroll
                for (int i = 0; i < VW; ++i) {
                    mb[i] *= rb;
                    const float away = mb[i] - mean[i];
                    mean[i] += away * part;
                    sq[i] += away * away * rest;
                }
#pragma unroll
                for (int u = 0; u < kU; ++u)
#pragma unroll
                    for (int i = 0; i < VW; ++i) {
                        const float e = on[u] ? d[u][i] - mb[i] : 0.f;
                        sq[i] += e * e;
                    }
            }
        }
        // positions below p that are counted: whole bands of len frames and the last one's
        const auto counted = [&](int p) { return p / s.T * len + min(p % s.T, len); };
        const float c_all = hi > lo ? (float)(counted(hi) - counted(lo)) : 0.f;
        float sum[VW];
#pragma unroll
        for (int i = 0; i < VW; ++i) sum[i] = (float)cnt * mean[i];
        __syncthreads();                                       // the pass before has read its sums
        const int nw = gn_row_sums<VW>(sum, red, cpb, row, rows);
        // channels of this pass: [cb * VW, cb * VW + cpb * VW); with more than 256 chunks (VW 1, 2 and 4 with C > 256, 512 and 1024) a group may lie in
        // two passes, each of which writes a triple for its part of the channels
        const int c0 = cb * VW, c1 = min(s.C, c0 + cpb * VW);
        const int g0 = c0 / s.Cg, g1 = (c1 - 1) / s.Cg;
        const float winv = c_all > 0.f ? 1.f / c_all : 0.f;
        gn_group_sums(g0, g1, [&](int g, int lane, int width) {
            const int a = max(c0, g * s.Cg), b = min(c1, (g + 1) * s.Cg);
            float m = 0.f;
            for (int c = a + lane; c < b; c += width)
                for (int w = 0; w < nw; ++w) m += red[w * cpb * VW + c - c0];
            return m;
        }, [&](int g, float m) { gmean[g - g0] = m * winv / (float)(min(c1, (g + 1) * s.Cg) - max(c0, g * s.Cg)); });
        __syncthreads();
#pragma unroll
        for (int i = 0; i < VW; ++i) {
            const int c = chunk * VW + i;
            const float d = on ? mean[i] - gmean[c / s.Cg - g0] : 0.f;
            sum[i] = on && cnt ? sq[i] + (float)cnt * d * d : 0.f;
        }
        gn_row_sums<VW>(sum, red, cpb, row, rows);
        gn_group_sums(g0, g1, [&](int g, int lane, int width) {
            const int a = max(c0, g * s.Cg), b = min(c1, (g + 1) * s.Cg);
            float m2 = 0.f;
            for (int c = a + lane; c < b; c += width)
                for (int w = 0; w < nw; ++w) m2 += red[w * cpb * VW + c - c0];
            return m2;
        }, [&](int g, float m2) {
            // slot: one per (sample, split, pass-part of the group)
            const int sub = cb / cpb, nsub = (nch + cpb - 1) / cpb;
            float* o = part + (((int64_t)n * nsplit + split) * nsub + sub) * s.G * 3 + g * 3;
            o[0] = c_all * (float)(min(c1, (g + 1) * s.Cg) - max(c0, g * s.Cg)); o[1] = gmean[g - g0]; o[2] = m2;
        });
        if (nch > cpb) {   // groups that this pass does not touch hold no weight
            const int sub = cb / cpb, nsub = (nch + cpb - 1) / cpb;
            for (int g = threadIdx.x; g < s.G; g += kGnThreads)
                if (g < g0 || g > g1) part[(((int64_t)n * nsplit + split) * nsub + sub) * s.G * 3 + g * 3] = 0.f;
        }
        __syncthreads();
    }
}

// mean and rstd of every group of sample n from the splits' triples, into LDS: a wave a group, a lane a part
__device__ __forceinline__ void gn_merge(const float* __restrict__ part, int n, int nparts, int G, float eps, float* mean, float* rstd) {
    const int lane = threadIdx.x & 63;
    for (int g = threadIdx.x >> 6; g < G; g += kGnThreads / 64) {
        const float* p = part + (int64_t)n * nparts * G * 3 + g * 3;
        float w = 0.f, m = 0.f;
        for (int i = lane; i < nparts; i += 64) {
            const float wi = p[(int64_t)i * G * 3], mi = p[(int64_t)i * G * 3 + 1];
            w += wi;
            m += wi > 0.f ? wi * mi : 0.f;
        }
        w = gn_wave_sum(w);
        m = gn_wave_sum(m);
        const float inv = w > 0.f ? 1.f / w : 0.f;
        m *= inv;
        float m2 = 0.f;
        for (int i = lane; i < nparts; i += 64) {
            const float wi = p[(int64_t)i * G * 3], d = p[(int64_t)i * G * 3 + 1] - m, qi = p[(int64_t)i * G * 3 + 2];
            m2 += wi > 0.f ? qi + wi * d * d : 0.f;
        }
        m2 = gn_wave_sum(m2);
        if (lane == 0) {
            mean[g] = m;
            rstd[g] = rsqrtf(m2 * inv + eps);
        }
    }
    __syncthreads();
}

template <typename T, int VW, bool RES>
__global__ __launch_bounds__(kGnThreads) void gn_apply_kernel(const T* __restrict__ x, GnStr xs, const T* __restrict__ res, GnStr rs,
                                                              const float* __restrict__ gamma, const float* __restrict__ beta, GnShape s,
                                                              float eps, const float* __restrict__ part, int nsplit, int nparts, T* __restrict__ y,
                                                              GnStr ys, float* __restrict__ mean_out, float* __restrict__ rstd_out) {
    __shared__ float mean[kGnMaxC], rstd[kGnMaxC];
    const int n = blockIdx.x / nsplit, split = blockIdx.x % nsplit;
    gn_merge(part, n, nparts, s.G, eps, mean, rstd);
    if (split == 0 && mean_out)
        for (int g = threadIdx.x; g < s.G; g += kGnThreads) { mean_out[(int64_t)n * s.G + g] = mean[g]; rstd_out[(int64_t)n * s.G + g] = rstd[g]; }
    const int P = s.F * s.T, nch = s.C / VW;
    const int len = s.lengths ? min(max(s.lengths[n], 0), s.T) : s.T;
    const int cpb = min(nch, kGnThreads), rows = kGnThreads / cpb, row = threadIdx.x / cpb;
    const int per = (P + nsplit - 1) / nsplit, lo = split * per, hi = min(P, lo + per);
    for (int cb = 0; cb < nch; cb += cpb) {
        const int chunk = cb + threadIdx.x % cpb;
        if (row >= rows || chunk >= nch) continue;
        float mu[VW], a[VW], b[VW];
#pragma unroll
        for (int i = 0; i < VW; ++i) {
            const int c = chunk * VW + i;
            mu[i] = mean[c / s.Cg];
            a[i] = rstd[c / s.Cg] * gamma[c];
            b[i] = beta[c];
        }
        GnWalk w(lo + row, hi, rows, s.T);
        GnPos px(xs, n, w), pr(rs, n, w), py(ys, n, w);
        while (w.more()) {
            GnRaw<T, VW> rx[kU], rr[kU];
            int64_t at[kU];
            bool on[kU], in[kU];
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                on[u] = w.more();
                in[u] = on[u] && w.t < len;
                at[u] = py.off;
                rx[u] = *reinterpret_cast<const GnRaw<T, VW>*>(x + px.at(in[u]) + chunk * VW);
                if (RES) rr[u] = *reinterpret_cast<const GnRaw<T, VW>*>(res + pr.at(in[u]) + chunk * VW);
                gn_next(w, px, pr, py);
            }
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                if (!on[u]) continue;
                float o[VW];
#pragma unroll
                for (int i = 0; i < VW; ++i) o[i] = 0.f;
                if (in[u]) {
                    float v[VW], z[VW];
                    gn_get<T, VW>(rx[u], v);
                    if (RES) gn_get<T, VW>(rr[u], z);
#pragma unroll
                    for (int i = 0; i < VW; ++i) o[i] = (v[i] - mu[i]) * a[i] + b[i] + (RES ? z[i] : 0.f);
                    gn_act<VW>(o, s.act);
                }
                gn_st<T, VW>(y + at[u] + chunk * VW, o);
            }
        }
    }
}

// Backward, first pass: g = gy * act'(pre) (written as the residual's gradient), per (sample, split): channel sums of g and of g * xhat,
// and the same weighted with gamma per group.
template <typename T, int VW, bool RES>
__global__ __launch_bounds__(kGnThreads) void gn_bwd_stats_kernel(const T* __restrict__ gy, GnStr gs, const T* __restrict__ x, GnStr xs,
                                                                  const T* __restrict__ res, GnStr rs, const float* __restrict__ gamma,
                                                                  const float* __restrict__ beta, const float* __restrict__ mean,
                                                                  const float* __restrict__ rstd, GnShape s, int nsplit,
                                                                  T* __restrict__ gres, GnStr grs, float* __restrict__ cpart,
                                                                  float* __restrict__ gpart) {
    __shared__ float red[kGnThreads * VW * 2];
    const int n = blockIdx.x / nsplit, split = blockIdx.x % nsplit;
    const int P = s.F * s.T, nch = s.C / VW;
    const int per = (P + nsplit - 1) / nsplit, lo = split * per, hi = min(P, lo + per);
    const int len = s.lengths ? min(max(s.lengths[n], 0), s.T) : s.T;
    const int cpb = min(nch, kGnThreads), rows = kGnThreads / cpb, row = threadIdx.x / cpb;
    float* cp = cpart + ((int64_t)n * nsplit + split) * s.C * 2;
    for (int cb = 0; cb < nch; cb += cpb) {
        const int chunk = cb + threadIdx.x % cpb;
        const bool on = row < rows && chunk < nch;
        float sb[VW], sx[VW];
#pragma unroll
        for (int i = 0; i < VW; ++i) { sb[i] = 0.f; sx[i] = 0.f; }
        if (on) {
            float mu[VW], r[VW], gm[VW], bt[VW];
#pragma unroll
            for (int i = 0; i < VW; ++i) {
                const int c = chunk * VW + i;
                mu[i] = mean[(int64_t)n * s.G + c / s.Cg];
                r[i] = rstd[(int64_t)n * s.G + c / s.Cg];
                gm[i] = gamma[c];
                bt[i] = beta[c];
            }
            GnWalk w(lo + row, hi, rows, s.T);
            GnPos pg(gs, n, w), px(xs, n, w), pr(rs, n, w), po(grs, n, w);
            while (w.more()) {
                GnRaw<T, VW> rg[kUb], rx[kUb], rr[kUb];
                int64_t at[kUb];
                bool on[kUb], in[kUb];
#pragma unroll
                for (int u = 0; u < kUb; ++u) {
                    on[u] = w.more();
                    in[u] = on[u] && w.t < len;
                    at[u] = po.off;
                    rg[u] = *reinterpret_cast<const GnRaw<T, VW>*>(gy + pg.at(in[u]) + chunk * VW);
                    rx[u] = *reinterpret_cast<const GnRaw<T, VW>*>(x + px.at(in[u]) + chunk * VW);
                    if (RES) rr[u] = *reinterpret_cast<const GnRaw<T, VW>*>(res + pr.at(in[u]) + chunk * VW);
                    gn_next(w, pg, px, pr, po);
                }
#pragma unroll
                for (int u = 0; u < kUb; ++u) {
                    if (!on[u]) continue;
                    float q[VW];
#pragma unroll
                    for (int i = 0; i < VW; ++i) q[i] = 0.f;
                    if (in[u]) {
                        float v[VW], z[VW];
                        gn_get<T, VW>(rg[u], q);
                        gn_get<T, VW>(rx[u], v);
                        if (RES) gn_get<T, VW>(rr[u], z);
#pragma unroll
                        for (int i = 0; i < VW; ++i) {
                            v[i] = (v[i] - mu[i]) * r[i];
                            z[i] = v[i] * gm[i] + bt[i] + (RES ? z[i] : 0.f);
                        }
                        gn_act_grad<VW>(q, z, s.act);
#pragma unroll
                        for (int i = 0; i < VW; ++i) {
                            sb[i] += q[i];
                            sx[i] += q[i] * v[i];
                        }
                    }
                    if (gres) gn_st<T, VW>(gres + at[u] + chunk * VW, q);
                }
            }
        }
        float sums[2 * VW];
#pragma unroll
        for (int i = 0; i < VW; ++i) { sums[i] = sb[i]; sums[VW + i] = sx[i]; }
        __syncthreads();
        const int nw = gn_row_sums<2 * VW>(sums, red, cpb, row, rows);
        // the total of a channel's sum q, into the first wave's place
        for (int c = threadIdx.x; c < cpb * VW * 2; c += kGnThreads) {
            float t = red[c];
            for (int w = 1; w < nw; ++w) t += red[w * cpb * VW * 2 + c];
            red[c] = t;
            const int ch = cb + c / (2 * VW), q = c / VW & 1;
            if (ch < nch) cp[(ch * VW + c % VW) * 2 + q] = t;
        }
        __syncthreads();
    }
    // per group, weighted with gamma: from LDS where one pass held all channels, else from what the passes wrote (this workgroup's own
    // global writes, visible to it behind the barrier)
    float* go = gpart + ((int64_t)n * nsplit + split) * s.G * 2;
#pragma unroll
    for (int q = 0; q < 2; ++q)
        gn_group_sums(0, s.G - 1, [&](int g, int lane, int width) {
            float a = 0.f;
            for (int c = g * s.Cg + lane; c < (g + 1) * s.Cg; c += width)
                a += gamma[c] * (nch <= kGnThreads ? red[(c / VW * 2 + q) * VW + c % VW] : cp[c * 2 + q]);
            return a;
        }, [&](int g, float a) { go[g * 2 + q] = a; });
}

// out[c] (+)= sum over parts of part[r][c][0 / 1]; a workgroup takes 32 channels, its rows of 32 threads walk the parts
__device__ __forceinline__ void gn_param_reduce(const float* __restrict__ cpart, int64_t nrows, int C, int c0, int accumulate,
                                                float* __restrict__ dgamma, float* __restrict__ dbeta) {
    __shared__ float red[32][32][2];
    const int c = c0 + (threadIdx.x & 31), r0 = threadIdx.x >> 5, nr = blockDim.x >> 5;
    float a = 0.f, b = 0.f;
    if (c < C) {
#pragma unroll 4
        for (int64_t r = r0; r < nrows; r += nr) { a += cpart[(r * C + c) * 2]; b += cpart[(r * C + c) * 2 + 1]; }
    }
    red[r0][threadIdx.x & 31][0] = a;
    red[r0][threadIdx.x & 31][1] = b;
    __syncthreads();
    if (r0 == 0 && c < C) {
        for (int i = 1; i < nr; ++i) { a += red[i][threadIdx.x][0]; b += red[i][threadIdx.x][1]; }
        dbeta[c] = accumulate ? dbeta[c] + a : a;
        dgamma[c] = accumulate ? dgamma[c] + b : b;
    }
}

// Backward, second pass: gx = rstd * (gamma g - mean(gamma g) - xhat mean(gamma g xhat)); the workgroups behind the N * nsplit that do so
// add up the parameter gradients instead, 32 channels each.  g is formed again from gy, x and the residual: reading the written gres back
// would save a read in three but carry its 16-bit rounding into gx.
template <typename T, int VW, bool RES>
__global__ __launch_bounds__(kGnThreads) void gn_bwd_apply_kernel(const T* __restrict__ gy, GnStr gs, const T* __restrict__ x, GnStr xs,
                                                                  const T* __restrict__ res, GnStr rs, const float* __restrict__ gamma,
                                                                  const float* __restrict__ beta, const float* __restrict__ mean,
                                                                  const float* __restrict__ rstd, GnShape s, const float* __restrict__ cpart, const float* __restrict__ gpart,
                                                                  int nsplit, int accumulate, T* __restrict__ gx, GnStr gxs,
                                                                  float* __restrict__ dgamma, float* __restrict__ dbeta) {
    __shared__ float c1[kGnMaxC], c2[kGnMaxC];
    const int n = blockIdx.x / nsplit, split = blockIdx.x % nsplit;
    if (n >= s.N) {
        gn_param_reduce(cpart, (int64_t)s.N * nsplit, s.C, (blockIdx.x - s.N * nsplit) * 32, accumulate, dgamma, dbeta);
        return;
    }
    const int len = s.lengths ? min(max(s.lengths[n], 0), s.T) : s.T;
    const float cinv = len > 0 ? 1.f / ((float)len * (float)s.F * (float)s.Cg) : 0.f;
#pragma unroll
    for (int q = 0; q < 2; ++q)
        gn_group_sums(0, s.G - 1, [&](int g, int lane, int width) {
            float a = 0.f;
            for (int i = lane; i < nsplit; i += width) a += gpart[(((int64_t)n * nsplit + i) * s.G + g) * 2 + q];
            return a;
        }, [&](int g, float a) { (q ? c2 : c1)[g] = a * cinv; });
    __syncthreads();
    const int P = s.F * s.T, nch = s.C / VW;
    const int cpb = min(nch, kGnThreads), rows = kGnThreads / cpb, row = threadIdx.x / cpb;
    const int per = (P + nsplit - 1) / nsplit, lo = split * per, hi = min(P, lo + per);
    for (int cb = 0; cb < nch; cb += cpb) {
        const int chunk = cb + threadIdx.x % cpb;
        if (row >= rows || chunk >= nch) continue;
        float mu[VW], r[VW], gm[VW], bt[VW], k1[VW], k2[VW];
#pragma unroll
        for (int i = 0; i < VW; ++i) {
            const int c = chunk * VW + i, g = c / s.Cg;
            mu[i] = mean[(int64_t)n * s.G + g];
            r[i] = rstd[(int64_t)n * s.G + g];
            gm[i] = gamma[c];
            bt[i] = beta[c];
            k1[i] = c1[g];
            k2[i] = c2[g];
        }
        GnWalk w(lo + row, hi, rows, s.T);
        GnPos pg(gs, n, w), px(xs, n, w), pr(rs, n, w), po(gxs, n, w);
        while (w.more()) {
            GnRaw<T, VW> rg[kUb], rx[kUb], rr[kUb];
            int64_t at[kUb];
            bool on[kUb], in[kUb];
#pragma unroll
            for (int u = 0; u < kUb; ++u) {
                on[u] = w.more();
                in[u] = on[u] && w.t < len;
                at[u] = po.off;
                rg[u] = *reinterpret_cast<const GnRaw<T, VW>*>(gy + pg.at(in[u]) + chunk * VW);
                rx[u] = *reinterpret_cast<const GnRaw<T, VW>*>(x + px.at(in[u]) + chunk * VW);
                if (RES) rr[u] = *reinterpret_cast<const GnRaw<T, VW>*>(res + pr.at(in[u]) + chunk * VW);
                gn_next(w, pg, px, pr, po);
            }
#pragma unroll
            for (int u = 0; u < kUb; ++u) {
                if (!on[u]) continue;
                float o[VW];
#pragma unroll
                for (int i = 0; i < VW; ++i) o[i] = 0.f;
                if (in[u]) {
                    float q[VW], v[VW], z[VW];
                    gn_get<T, VW>(rg[u], q);
                    gn_get<T, VW>(rx[u], v);
                    if (RES) gn_get<T, VW>(rr[u], z);
#pragma unroll
                    for (int i = 0; i < VW; ++i) {
                        v[i] = (v[i] - mu[i]) * r[i];
                        z[i] = v[i] * gm[i] + bt[i] + (RES ? z[i] : 0.f);
                    }
                    gn_act_grad<VW>(q, z, s.act);
#pragma unroll
                    for (int i = 0; i < VW; ++i) o[i] = r[i] * (gm[i] * q[i] - k1[i] - v[i] * k2[i]);
                }
                gn_st<T, VW>(gx + at[u] + chunk * VW, o);
            }
        }
    }
}

// ---- rows route ---------------------------------------------------------------------------------------
// sum over `team` neighbouring lanes (a power of two), in all of them; rows of 16 lanes rotate in the vector ALU, no LDS involved
__device__ __forceinline__ float gn_team_sum(float v, int team) {
    if (team >= 16) {
        v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x128, 0xf, 0xf, false));
        v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x124, 0xf, 0xf, false));
        v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x122, 0xf, 0xf, false));
        v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x121, 0xf, 0xf, false));
        if (team >= 32) v += __shfl_xor(v, 16);
        if (team == 64) v += __shfl_xor(v, 32);
        return v;
    }
    for (int o = team >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// Unit u = (sample u / G, group u % G): Cg contiguous channels held by `team` lanes (a power of two), NCH chunks of VW each.
template <typename T, int VW, int NCH, bool RES>
__global__ __launch_bounds__(kGnThreads) void gn_rows_fwd_kernel(const T* __restrict__ x, int64_t xsn, const T* __restrict__ res, int64_t rsn,
                                                                 const float* __restrict__ gamma, const float* __restrict__ beta, GnShape s,
                                                                 float eps, int team, T* __restrict__ y, int64_t ysn,
                                                                 float* __restrict__ mean_out, float* __restrict__ rstd_out) {
    const int upb = kGnThreads / team, lane = threadIdx.x & (team - 1);
    const float inv = 1.f / (float)s.Cg;
    const uint32_t slot = blockIdx.x * upb + threadIdx.x / team;
    const int g = (int)(slot % s.G), c0 = g * s.Cg, dn = (int)(gridDim.x * upb / s.G);
    float gm[NCH][VW], bt[NCH][VW];
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
        const int c = c0 + min((k * team + lane) * VW, s.Cg - VW);
        gn_ld<float, VW>(gamma + c, gm[k]);
        gn_ld<float, VW>(beta + c, bt[k]);
    }
    GnRaw<T, VW> nx[NCH], nr[NCH];          // the next unit's elements, requested a unit ahead
    auto fetch = [&](int64_t n) {
#pragma unroll
        for (int k = 0; k < NCH; ++k) {
            const int c = c0 + min((k * team + lane) * VW, s.Cg - VW);
            nx[k] = *reinterpret_cast<const GnRaw<T, VW>*>(x + n * xsn + c);
            if (RES) nr[k] = *reinterpret_cast<const GnRaw<T, VW>*>(res + n * rsn + c);
        }
    };
    int n = (int)(slot / s.G);
    if (n < s.N) fetch(n);
    for (; n < s.N; n += dn) {
        const bool dead = s.lengths && s.lengths[n] <= 0;
        GnRaw<T, VW> cr[NCH];
        float v[NCH][VW], sm = 0.f;
#pragma unroll
        for (int k = 0; k < NCH; ++k) {
            gn_get<T, VW>(nx[k], v[k]);
            cr[k] = nr[k];
        }
        if (n + dn < s.N) fetch(n + dn);
#pragma unroll
        for (int k = 0; k < NCH; ++k) {
            const int c = (k * team + lane) * VW;
#pragma unroll
            for (int i = 0; i < VW; ++i) v[k][i] = c < s.Cg && !dead ? v[k][i] : 0.f;
#pragma unroll
            for (int i = 0; i < VW; ++i) sm += v[k][i];
        }
        sm = gn_team_sum(sm, team);
        const float mean = sm * inv;
        float q = 0.f;
#pragma unroll
        for (int k = 0; k < NCH; ++k)
            if ((k * team + lane) * VW < s.Cg) {
#pragma unroll
                for (int i = 0; i < VW; ++i) { v[k][i] -= mean; q += v[k][i] * v[k][i]; }
            }
        q = gn_team_sum(q, team);
        const float rstd = rsqrtf(q * inv + eps);
        if (lane == 0 && mean_out) { mean_out[(int64_t)n * s.G + g] = mean; rstd_out[(int64_t)n * s.G + g] = rstd; }
#pragma unroll
        for (int k = 0; k < NCH; ++k) {
            const int c = (k * team + lane) * VW;
            if (c < s.Cg) {
                float o[VW];
                if (RES) gn_get<T, VW>(cr[k], o);
#pragma unroll
                for (int i = 0; i < VW; ++i) o[i] = v[k][i] * (rstd * gm[k][i]) + bt[k][i] + (RES ? o[i] : 0.f);
                gn_act<VW>(o, s.act);
#pragma unroll
                for (int i = 0; i < VW; ++i) o[i] = dead ? 0.f : o[i];
                gn_st<T, VW>(y + (int64_t)n * ysn + c0 + c, o);
            }
        }
    }
}

// The grid steps by a multiple of G units, so a lane keeps its channels and sums its parameter gradients in registers; slot = unit slot of
// the grid, cpart [slots / G][C][2] because slot % G is the group.
template <typename T, int VW, int NCH, bool RES>
__global__ __launch_bounds__(kGnThreads) void gn_rows_bwd_kernel(const T* __restrict__ gy, int64_t gsn, const T* __restrict__ x, int64_t xsn,
                                                                 const T* __restrict__ res, int64_t rsn, const float* __restrict__ gamma,
                                                                 const float* __restrict__ beta, const float* __restrict__ mean_in,
                                                                 const float* __restrict__ rstd_in, GnShape s, int team, T* __restrict__ gx,
                                                                 int64_t gxsn, T* __restrict__ gres, int64_t grsn, float* __restrict__ cpart) {
    const int upb = kGnThreads / team, lane = threadIdx.x & (team - 1);
    const float inv = 1.f / (float)s.Cg;
    const uint32_t slot = blockIdx.x * upb + threadIdx.x / team;
    const int g = (int)(slot % s.G), c0 = g * s.Cg, dn = (int)(gridDim.x * upb / s.G);
    float gm[NCH][VW], bt[NCH][VW], dg[NCH][VW], db[NCH][VW];
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
        const int c = (k * team + lane) * VW;
#pragma unroll
        for (int i = 0; i < VW; ++i) { gm[k][i] = bt[k][i] = dg[k][i] = db[k][i] = 0.f; }
        if (c < s.Cg) { gn_ld<float, VW>(gamma + c0 + c, gm[k]); gn_ld<float, VW>(beta + c0 + c, bt[k]); }
    }
    GnRaw<T, VW> ng[NCH], nx[NCH], nr[NCH];
    float nmean = 0.f, nrstd = 0.f;
    auto fetch = [&](int64_t n) {
        nmean = mean_in[n * s.G + g];
        nrstd = rstd_in[n * s.G + g];
#pragma unroll
        for (int k = 0; k < NCH; ++k) {
            const int c = c0 + min((k * team + lane) * VW, s.Cg - VW);
            ng[k] = *reinterpret_cast<const GnRaw<T, VW>*>(gy + n * gsn + c);
            nx[k] = *reinterpret_cast<const GnRaw<T, VW>*>(x + n * xsn + c);
            if (RES) nr[k] = *reinterpret_cast<const GnRaw<T, VW>*>(res + n * rsn + c);
        }
    };
    int n = (int)(slot / s.G);
    if (n < s.N) fetch(n);
    for (; n < s.N; n += dn) {
        const bool dead = s.lengths && s.lengths[n] <= 0;
        const float mean = nmean, rstd = nrstd;
        float w[NCH][VW], xh[NCH][VW], zr[NCH][VW], s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int k = 0; k < NCH; ++k) {
            gn_get<T, VW>(ng[k], w[k]);
            gn_get<T, VW>(nx[k], xh[k]);
            if (RES) gn_get<T, VW>(nr[k], zr[k]);
        }
        if (n + dn < s.N) fetch(n + dn);
#pragma unroll
        for (int k = 0; k < NCH; ++k) {
            const int c = (k * team + lane) * VW;
            const bool on = c < s.Cg && !dead;
            float z[VW];
#pragma unroll
            for (int i = 0; i < VW; ++i) {
                w[k][i] = on ? w[k][i] : 0.f;
                xh[k][i] = on ? xh[k][i] : 0.f;
                z[i] = RES && on ? zr[k][i] : 0.f;
            }
            if (on) {
#pragma unroll
                for (int i = 0; i < VW; ++i) {
                    xh[k][i] = (xh[k][i] - mean) * rstd;
                    z[i] += xh[k][i] * gm[k][i] + bt[k][i];
                }
                gn_act_grad<VW>(w[k], z, s.act);
            }
            if (gres && c < s.Cg) gn_st<T, VW>(gres + (int64_t)n * grsn + c0 + c, w[k]);
#pragma unroll
            for (int i = 0; i < VW; ++i) {
                dg[k][i] += w[k][i] * xh[k][i];
                db[k][i] += w[k][i];
                w[k][i] *= gm[k][i];
                s1 += w[k][i];
                s2 += w[k][i] * xh[k][i];
            }
        }
        s1 = gn_team_sum(s1, team);
        s2 = gn_team_sum(s2, team);
        s1 *= inv; s2 *= inv;
#pragma unroll
        for (int k = 0; k < NCH; ++k) {
            const int c = (k * team + lane) * VW;
            if (c < s.Cg) {
                float o[VW];
#pragma unroll
                for (int i = 0; i < VW; ++i) o[i] = dead ? 0.f : rstd * (w[k][i] - s1 - xh[k][i] * s2);
                gn_st<T, VW>(gx + (int64_t)n * gxsn + c0 + c, o);
            }
        }
    }
    float* cp = cpart + (int64_t)(slot / s.G) * s.C * 2 + c0 * 2;
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
        const int c = (k * team + lane) * VW;
        if (c < s.Cg) {
#pragma unroll
            for (int i = 0; i < VW; ++i) { cp[(c + i) * 2] = db[k][i]; cp[(c + i) * 2 + 1] = dg[k][i]; }
        }
    }
}

__global__ __launch_bounds__(1024) void gn_param_kernel(const float* __restrict__ cpart, int64_t nrows, int C, int accumulate,
                                                              float* __restrict__ dgamma, float* __restrict__ dbeta) {
    gn_param_reduce(cpart, nrows, C, blockIdx.x * 32, accumulate, dgamma, dbeta);
}

// ---- host ----------------------------------------------------------------------------------------------
struct GnPlan {
    bool rows;
    int vw;                  // channels a chunk
    int nch, team;           // rows route: chunks a lane, lanes a unit
    int splits, nsub;        // block route
    int grid, gstep;         // rows route: the backward's grid; grids are multiples of gstep, so that a lane keeps its channels
};

// `vw`: the widest vector that the tensors' addresses and strides allow
static GnPlan gn_plan(int64_t N, int F, int T, int C, int G, int vw) {
    GnPlan p{};
    const int Cg = C / G;
    if ((int64_t)F * T == 1) {
        p.vw = vw;
        while (Cg % p.vw) p.vw >>= 1;
        const int chunks = Cg / p.vw;
        int team = 1;
        while (team < 64 && team < chunks) team *= 2;
        const int nch = (chunks + team - 1) / team;
        if (nch <= 4) {
            p.rows = true; p.team = team; p.nch = nch == 3 ? 4 : nch;
            const int upb = kGnThreads / team;
            // one persistent grid; its step is a multiple of G units, so that a lane keeps its channels
            int64_t blocks = (N * G + upb - 1) / upb;
            if (blocks > 768) blocks = 768;
            int step = 1;
            while ((int64_t)step * upb % G) ++step;
            p.gstep = step;
            p.grid = (int)((blocks + step - 1) / step * step);
            return p;
        }
    }
    // a chunk of channels lies inside one group or holds whole groups
    p.vw = vw;
    while (p.vw > 1 && !(C % p.vw == 0 && (Cg % p.vw == 0 || p.vw % Cg == 0))) p.vw >>= 1;
    const int64_t P = (int64_t)F * T;
    // ~768 workgroups on the chip, at least 32 positions each.  Each pays for its reductions; the backward's two passes on 61 MB tensors took
    // 48 + 42 us with 512, 44 + 43 with 768, 46 + 49 with 1024, 49 + 55 with 1536
    int64_t sp = N > 0 ? 768 / N : 1;
    if (sp > kGnMaxSplit) sp = kGnMaxSplit;
    if (sp > (P + 31) / 32) sp = (P + 31) / 32;
    if (sp < 1) sp = 1;
    p.splits = (int)sp;
    const int nch = C / p.vw, cpb = nch < kGnThreads ? nch : kGnThreads;
    p.nsub = (nch + cpb - 1) / cpb;
    return p;
}

static size_t gn_bytes(const GnPlan& p, int64_t N, int C, int G, int backward) {
    if (p.rows) return backward ? align_up((size_t)p.grid * (kGnThreads / p.team) / G * C * 2 * sizeof(float), 256) : 0;
    const size_t parts = (size_t)N * p.splits;
    if (!backward) return align_up(parts * p.nsub * G * 3 * sizeof(float), 256);
    return align_up(parts * C * 2 * sizeof(float), 256) + align_up(parts * G * 2 * sizeof(float), 256);
}

static int gn_check(const char* who, int64_t N, int F, int T, int C, int G, int act, int dtype) {
    SP_CHECK_ARG(N >= 0 && N <= (1 << 22) && F >= 0 && T >= 0 && (int64_t)F * T < (1ll << 31) - 4096,
                 "%s: bad shape N=%lld (at most 2^22) F=%d T=%d", who, (long long)N, F, T);
    SP_CHECK_ARG(C >= 1 && C <= kGnMaxC && G >= 1 && C % G == 0, "%s: C=%d must be a multiple of G=%d and at most %d", who, C, G, kGnMaxC);
    SP_CHECK_ARG(act == SP_ACT_NONE || act == SP_ACT_RELU || act == SP_ACT_SILU, "%s: act %d unknown", who, act);
    SP_CHECK_ARG(dtype == SP_F32 || dtype == SP_BF16 || dtype == SP_F16, "%s: dtype %d not supported (f32, bf16, f16)", who, dtype);
    return SP_OK;
}

// widest vector (8 at most) that addresses and strides allow; gamma and beta are read as f32 vectors
static int gn_align(int esize, const void* const* p, const int64_t* st, int k, const float* gamma, const float* beta) {
    int vw = 8;
    const uintptr_t par = reinterpret_cast<uintptr_t>(gamma) | reinterpret_cast<uintptr_t>(beta);
    for (; vw > 1; vw >>= 1) {
        bool ok = par % (vw * sizeof(float)) == 0;
        for (int i = 0; i < k; ++i) {
            if (!p[i]) continue;
            if (reinterpret_cast<uintptr_t>(p[i]) % (vw * esize)) ok = false;
            for (int j = 0; j < 3; ++j) if (st[3 * i + j] % vw) ok = false;
        }
        if (ok) break;
    }
    return vw;
}

}  // namespace sp

using namespace sp;

#define SP_GN_TYPES(DT, CALL)                                     \
    if (DT == SP_F32) { using T_ = float; CALL }                  \
    else if (DT == SP_F16) { using T_ = __half; CALL }            \
    else { using T_ = __hip_bfloat16; CALL }
#define SP_GN_VW(V, CALL)                          \
    if (V == 8) { constexpr int VW_ = 8; CALL }    \
    else if (V == 4) { constexpr int VW_ = 4; CALL } \
    else if (V == 2) { constexpr int VW_ = 2; CALL } \
    else { constexpr int VW_ = 1; CALL }
#define SP_GN_NCH(K, CALL)                          \
    if (K == 1) { constexpr int NC_ = 1; CALL }     \
    else if (K == 2) { constexpr int NC_ = 2; CALL } \
    else { constexpr int NC_ = 4; CALL }

extern "C" size_t sp_groupnorm_workspace_bytes(int64_t N, int F, int T, int C, int G, int backward) {
    if (gn_check("sp_groupnorm_workspace_bytes", N, F, T, C, G, 0, SP_F32)) return 0;
    size_t most = 0;        // whatever vector width the tensors will allow
    for (int vw = 8; vw; vw >>= 1) {
        const size_t b = gn_bytes(gn_plan(N, F, T, C, G, vw), N, C, G, backward);
        if (b > most) most = b;
    }
    return most;
}

extern "C" int sp_groupnorm_fwd(const void* x, const void* residual, const float* gamma, const float* beta, const int32_t* lengths,
                                const int64_t* strides, int64_t N, int F, int T, int C, int G, float eps, int act, int dtype, void* y,
                                float* mean, float* rstd, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = gn_check("sp_groupnorm_fwd", N, F, T, C, G, act, dtype);
    if (rc) return rc;
    SP_CHECK_ARG(strides, "sp_groupnorm_fwd: null strides");
    SP_CHECK_ARG((mean == nullptr) == (rstd == nullptr), "sp_groupnorm_fwd: mean and rstd are given together or not at all");
    if (N == 0 || F == 0 || T == 0) return SP_OK;
    SP_CHECK_ARG(x && gamma && beta && y, "sp_groupnorm_fwd: null pointer");
    const size_t need = sp_groupnorm_workspace_bytes(N, F, T, C, G, 0);
    if (workspace_bytes < need || (need && !workspace)) return fail(SP_EWORKSPACE, "sp_groupnorm_fwd: workspace %zu < %zu bytes", workspace_bytes, need);
    const GnShape s{(int)N, F, T, C, G, C / G, act, lengths};
    const void* ptrs[3] = {x, residual, y};
    const GnPlan p = gn_plan(N, F, T, C, G, gn_align(dtype == SP_F32 ? 4 : 2, ptrs, strides, 3, gamma, beta));
    const GnStr xs{strides[0], strides[1], strides[2]}, rs{strides[3], strides[4], strides[5]}, ys{strides[6], strides[7], strides[8]};
    hipStream_t st = (hipStream_t)stream;
    if (p.rows) {
        const int upb = kGnThreads / p.team;
        int64_t blocks = (N * G + upb - 1) / upb;
        if (blocks > 2048) blocks = 2048;      // a few units a team, the next one's loads ahead of the present one's work
        blocks = (blocks + p.gstep - 1) / p.gstep * p.gstep;
        SP_GN_TYPES(dtype, SP_GN_VW(p.vw, SP_GN_NCH(p.nch, {
            hipLaunchKernelGGL((residual ? gn_rows_fwd_kernel<T_, VW_, NC_, true> : gn_rows_fwd_kernel<T_, VW_, NC_, false>), dim3((unsigned)blocks), dim3(kGnThreads), 0, st, (const T_*)x, xs.n,
                               (const T_*)residual, rs.n, gamma, beta, s, eps, p.team, (T_*)y, ys.n, mean, rstd); })))
        return check_launch("gn_rows_fwd_kernel");
    }
    SP_GN_TYPES(dtype, SP_GN_VW(p.vw, {
        hipLaunchKernelGGL((gn_stats_kernel<T_, VW_>), dim3((unsigned)N * p.splits), dim3(kGnThreads), 0, st, (const T_*)x, xs, s, p.splits,
                           (float*)workspace);
        hipLaunchKernelGGL((residual ? gn_apply_kernel<T_, VW_, true> : gn_apply_kernel<T_, VW_, false>), dim3((unsigned)N * p.splits), dim3(kGnThreads), 0, st, (const T_*)x, xs,
                           (const T_*)residual, rs, gamma, beta, s, eps, (const float*)workspace, p.splits, p.splits * p.nsub, (T_*)y, ys, mean, rstd); }))
    return check_launch("gn_apply_kernel");
}

extern "C" int sp_groupnorm_bwd(const void* gy, const void* x, const void* residual, const float* gamma, const float* beta,
                                const float* mean, const float* rstd, const int32_t* lengths, const int64_t* strides, int64_t N, int F,
                                int T, int C, int G, int act, int accumulate, int dtype, void* gx, void* gres, float* dgamma,
                                float* dbeta, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = gn_check("sp_groupnorm_bwd", N, F, T, C, G, act, dtype);
    if (rc) return rc;
    SP_CHECK_ARG(strides, "sp_groupnorm_bwd: null strides");
    SP_CHECK_ARG(dgamma && dbeta, "sp_groupnorm_bwd: null pointer");
    hipStream_t st = (hipStream_t)stream;
    if (N == 0 || F == 0 || T == 0) {       // no positions: the parameter gradients are zero
        hipLaunchKernelGGL(gn_param_kernel, dim3((C + 31) / 32), dim3(1024), 0, st, nullptr, (int64_t)0, C, accumulate, dgamma, dbeta);
        return check_launch("gn_param_kernel");
    }
    SP_CHECK_ARG(gy && x && gamma && beta && mean && rstd && gx, "sp_groupnorm_bwd: null pointer");
    const size_t need = sp_groupnorm_workspace_bytes(N, F, T, C, G, 1);
    if (workspace_bytes < need || !workspace) return fail(SP_EWORKSPACE, "sp_groupnorm_bwd: workspace %zu < %zu bytes", workspace_bytes, need);
    const GnShape s{(int)N, F, T, C, G, C / G, act, lengths};
    const void* ptrs[5] = {gy, x, residual, gx, gres};
    const GnPlan p = gn_plan(N, F, T, C, G, gn_align(dtype == SP_F32 ? 4 : 2, ptrs, strides, 5, gamma, beta));
    const GnStr gs{strides[0], strides[1], strides[2]}, xs{strides[3], strides[4], strides[5]}, rs{strides[6], strides[7], strides[8]},
        gxs{strides[9], strides[10], strides[11]}, grs{strides[12], strides[13], strides[14]};
    float* cpart = (float*)workspace;
    if (p.rows) {
        SP_GN_TYPES(dtype, SP_GN_VW(p.vw, SP_GN_NCH(p.nch, {
            hipLaunchKernelGGL((residual ? gn_rows_bwd_kernel<T_, VW_, NC_, true> : gn_rows_bwd_kernel<T_, VW_, NC_, false>), dim3(p.grid), dim3(kGnThreads), 0, st, (const T_*)gy, gs.n, (const T_*)x,
                               xs.n, (const T_*)residual, rs.n, gamma, beta, mean, rstd, s, p.team, (T_*)gx, gxs.n, (T_*)gres, grs.n, cpart); })))
        hipLaunchKernelGGL(gn_param_kernel, dim3((C + 31) / 32), dim3(1024), 0, st, cpart, (int64_t)p.grid * (kGnThreads / p.team) / G, C,
                           accumulate, dgamma, dbeta);
        return check_launch("gn_rows_bwd_kernel");
    }
    float* gpart = (float*)((char*)workspace + align_up((size_t)N * p.splits * C * 2 * sizeof(float), 256));
    SP_GN_TYPES(dtype, SP_GN_VW(p.vw, {
        hipLaunchKernelGGL((residual ? gn_bwd_stats_kernel<T_, VW_, true> : gn_bwd_stats_kernel<T_, VW_, false>), dim3((unsigned)N * p.splits), dim3(kGnThreads), 0, st, (const T_*)gy, gs, (const T_*)x,
                           xs, (const T_*)residual, rs, gamma, beta, mean, rstd, s, p.splits, (T_*)gres, grs, cpart, gpart);
        hipLaunchKernelGGL((residual ? gn_bwd_apply_kernel<T_, VW_, true> : gn_bwd_apply_kernel<T_, VW_, false>), dim3((unsigned)N * p.splits + (C + 31) / 32), dim3(kGnThreads), 0, st,
                           (const T_*)gy, gs, (const T_*)x, xs, (const T_*)residual, rs, gamma, beta, mean, rstd, s, cpart, gpart, p.splits, accumulate, (T_*)gx, gxs, dgamma, dbeta); }))
    return check_launch("gn_bwd_apply_kernel");
}
