// Gated delta rule, chunked (forward and backward) and recurrent.  Per utterance and value head, with a state S [dk][dv] in f32:
//     S_t = a_t S_{t-1} + kh_t u_t^T,   u_t = beta_t (v_t - a_t S_{t-1}^T kh_t),   o_t = S_t^T qh_t,   a_t = exp(g_t)
// kh = k (or k / sqrt(|k|^2 + 1e-6)), qh = scale * q (or normalised alike).  It stands beside the SRU recurrence (net.py:61-72 of the
// reference, which has no such layer).
//
// Chunked form, 64 frames a chunk, G = running sum of g inside the chunk, D_ij = exp(G_i - G_j):
//     N_ij = D_ij kh_i.kh_j (j < i),  P_ij = D_ij qh_i.kh_j (j <= i),  X = (I + N diag(beta))^-1 N     (strictly lower)
//     Vt = V - e^G (Kh S0),  E = Vt - X (beta Vt),  U = beta E,  O = e^G (Qh S0) + P U,  S = e^{G_C} S0 + Kh^T (e^{G_C - G} U)
// X instead of (I + A)^-1: the identity part stays an exact f32 addition, and beta = 0 needs no care.
// Backward, dS and dO given:
//     dU = P^T dO + e^{G_C - G} (Kh dS),  F = dU - X^T (beta dU),  dV = beta F,  dbeta_j = E_j . F_j
//     dS0 = e^{G_C} dS + Qh^T (e^G dO) - Kh^T (e^G dV)
//     dP = dO U^T (j <= i),  dN = -dV U^T (j < i)
//     dQh = e^G dO S0^T + (dP*D) Kh,  dKh = (dP*D)^T Qh + e^{G_C-G} U dS^T - e^G dV S0^T + (dN*D) Kh + (dN*D)^T Kh
//     dg = suffix sums of dO_i.O_i - dV_i.V_i, plus <dS, S_C> at the chunk's end (every other dependence on G cancels)
//
// Arithmetic: the state, the chunk matrices and every sum are f32.  Products run on v_mfma_f32_16x16x32_bf16 with operands split into
// bf16 parts (x = hi + lo [+ lo2]): an input of type bf16 is one exact part, f16 two, f32 three; what is derived (S, U, X, ...) two, for
// f32 inputs three.  Two parts carry 2^-17, so that the f32 results (states, dg, dbeta) keep about 1e-6; one part of everything would be
// four times cheaper on the matrix cores and leave 1e-3.  Outputs of 16-bit type are rounded once.
//
// Kernels: prep (N, P, X of a chunk; all chunks at once) -> scan (walks the chunks with S in registers; a wave owns 32 columns of dv and
// never talks to the others: the accumulator layout of one product is the B operand of the next) ; backward: rscan (the same walk in
// reverse with dS) -> grads (dq, dk, dg, dbeta of a chunk; all chunks at once).  Few frames (streaming, single tokens): one recurrent kernel.
#include "common.h"

namespace sp {

constexpr int kC = 64;              // frames a chunk
constexpr int kRecurrentMax = 32;   // frames up to which the recurrent kernel runs (inference)
constexpr int kLdm = 72;            // row pitch (elements) of a 64 x 64 matrix plane in LDS: 16 rows of 8 bytes fall on distinct banks
constexpr int kVec = 8;             // per-chunk vectors of 64 floats: aq, ak, kb, beta, rk, sq, G (as 64 doubles)
enum { kAq = 0, kAk = 1, kKb = 2, kBe = 3, kRk = 4, kSq = 5, kG64 = 6 };

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef uint32_t u32x4a __attribute__((ext_vector_type(4), may_alias));
typedef uint32_t u32x2a __attribute__((ext_vector_type(2), may_alias));
typedef float f32x4a __attribute__((ext_vector_type(4), may_alias));

struct GdrArgs {
    const void *q, *k, *v;
    const float *g, *beta, *s0;
    const int32_t* lengths;
    int64_t qs[3], ks[3], vs[3], gs[3], bs[3];       // element strides (t, b, h)
    int T, B, Hk, H, r, dk, dv, nc, nsl;             // nsl: slices of 32 columns
    float scale;
    int norm, bidir;
    void* o;
    float* sT;
    // kept between the kernels (and, in training, for the backward)
    float* vec;              // [bh][nc][kVec][64]
    __bf16 *X, *P;           // [bh][nc][planes][64][64]
    float *S0, *E;           // [bh][nc][dk][dv], [bh][nc][64][dv]
    __bf16* olo;             // [T][B][H][dv]: what o's 16-bit rounding dropped
    // backward
    const void* go;
    const float* gsT;
    float* dS;               // [bh][nc][dk][dv]
    float *xpart, *bpart;    // [nsl][bh][nc][64]
    float* apart;            // [nsl][bh][nc]
    void *gq, *gk, *gv;
    float *gg, *gbeta, *gs0;
    int64_t gos[3];
};

// ---- operand fragments --------------------------------------------------------------------------------
template <typename T> struct Gd;
template <> struct Gd<__hip_bfloat16> { static constexpr int PT = 1, PD = 2; };
template <> struct Gd<__half> { static constexpr int PT = 2, PD = 2; };
template <> struct Gd<float> { static constexpr int PT = 3, PD = 3; };

template <int P> struct Frag { bf16x8 p[P]; };

template <int P> __device__ __forceinline__ Frag<P> split(f32x8 v) {
    Frag<P> f;
    f.p[0] = __builtin_convertvector(v, bf16x8);
#pragma unroll
    for (int i = 1; i < P; ++i) {
        v -= __builtin_convertvector(f.p[i - 1], f32x8);
        f.p[i] = __builtin_convertvector(v, bf16x8);
    }
    return f;
}
template <int P> __device__ __forceinline__ Frag<P> split(f32x4 a, f32x4 b) {
    return split<P>(__builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

// acc += a b, the parts whose product matters (i + j below the larger number of parts, or below `CUT`)
template <int PA, int PB, int CUT = (PA > PB ? PA : PB)>
__device__ __forceinline__ f32x4 mma(const Frag<PA>& a, const Frag<PB>& b, f32x4 acc) {
#pragma unroll
    for (int i = 0; i < PA; ++i)
#pragma unroll
        for (int j = 0; j < PB; ++j)
            if (i + j < CUT) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[i], b.p[j], acc, 0, 0, 0);
    return acc;
}

template <typename T> __device__ __forceinline__ float to_f(T v) { return Elem<T>::f(v); }
template <> __device__ __forceinline__ float to_f<__bf16>(__bf16 v) { return (float)v; }

// Operand from rows: lane (i = l & 15, g = l >> 4) takes row r0 + i, columns c0 + 4g .. +3 and c0 + 16 + 4g .. +3.  Both operands of every
// product use this order of the 32 inner indices; it is the order in which two stacked 16 x 16 accumulators hold their rows.
__device__ __forceinline__ Frag<1> row_frag(const __hip_bfloat16* t, int ld, int r0, int c0) {
    const int l = threadIdx.x & 63;
    const __hip_bfloat16* p = t + (r0 + (l & 15)) * ld + c0 + 4 * (l >> 4);
    const u32x2a a = *reinterpret_cast<const u32x2a*>(p), b = *reinterpret_cast<const u32x2a*>(p + 16);
    Frag<1> f;
    const u32x4a w = {a.x, a.y, b.x, b.y};
    f.p[0] = __builtin_bit_cast(bf16x8, w);
    return f;
}
__device__ __forceinline__ Frag<1> row_frag(const __bf16* t, int ld, int r0, int c0) {
    return row_frag(reinterpret_cast<const __hip_bfloat16*>(t), ld, r0, c0);
}
__device__ __forceinline__ f32x8 half8(u32x2a a, u32x2a b) {
    typedef _Float16 h8 __attribute__((ext_vector_type(8)));
    const u32x4a w = {a.x, a.y, b.x, b.y};
    return __builtin_convertvector(__builtin_bit_cast(h8, w), f32x8);
}
__device__ __forceinline__ Frag<2> row_frag(const __half* t, int ld, int r0, int c0) {
    const int l = threadIdx.x & 63;
    const __half* p = t + (r0 + (l & 15)) * ld + c0 + 4 * (l >> 4);
    return split<2>(half8(*reinterpret_cast<const u32x2a*>(p), *reinterpret_cast<const u32x2a*>(p + 16)));
}
__device__ __forceinline__ Frag<3> row_frag(const float* t, int ld, int r0, int c0) {
    const int l = threadIdx.x & 63;
    const float* p = t + (r0 + (l & 15)) * ld + c0 + 4 * (l >> 4);
    return split<3>(*reinterpret_cast<const f32x4a*>(p), *reinterpret_cast<const f32x4a*>(p + 16));
}

// 16-bit transposing LDS read: lane (i, g) gets rows k0 + 4g .. +3 of column m0 + i
__device__ __forceinline__ s16x4 tr4(const void* t, int ld, int k0, int m0) {
    const int l = threadIdx.x & 63, i = l & 15, g = l >> 4;
    const short* p = reinterpret_cast<const short*>(t) + (k0 + 4 * g + (i >> 2)) * ld + m0 + 4 * (i & 3);
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
}
// Operand from columns: lane (i, g) takes column m0 + i, rows k0 + 4g .. +3 and k0 + 16 + 4g .. +3
__device__ __forceinline__ Frag<1> col_frag(const __hip_bfloat16* t, int ld, int k0, int m0) {
    const s16x4 a = tr4(t, ld, k0, m0), b = tr4(t, ld, k0 + 16, m0);
    Frag<1> f;
    f.p[0] = __builtin_bit_cast(bf16x8, (s16x8)__builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    return f;
}
__device__ __forceinline__ Frag<1> col_frag(const __bf16* t, int ld, int k0, int m0) {
    return col_frag(reinterpret_cast<const __hip_bfloat16*>(t), ld, k0, m0);
}
__device__ __forceinline__ Frag<2> col_frag(const __half* t, int ld, int k0, int m0) {
    const s16x4 a = tr4(t, ld, k0, m0), b = tr4(t, ld, k0 + 16, m0);
    return split<2>(half8(__builtin_bit_cast(u32x2a, a), __builtin_bit_cast(u32x2a, b)));
}
__device__ __forceinline__ Frag<3> col_frag(const float* t, int ld, int k0, int m0) {
    const int l = threadIdx.x & 63;
    const float* p = t + (k0 + 4 * (l >> 4)) * ld + m0 + (l & 15);
    f32x8 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) { v[e] = p[e * ld]; v[4 + e] = p[(16 + e) * ld]; }
    return split<3>(v);
}
// planes of a split 64 x 64 matrix in LDS
template <int P> __device__ __forceinline__ Frag<P> plane_rows(const __bf16* t, int r0, int c0) {
    Frag<P> f;
#pragma unroll
    for (int i = 0; i < P; ++i) f.p[i] = row_frag(t + i * kC * kLdm, kLdm, r0, c0).p[0];
    return f;
}
template <int P> __device__ __forceinline__ Frag<P> plane_cols(const __bf16* t, int k0, int m0) {
    Frag<P> f;
#pragma unroll
    for (int i = 0; i < P; ++i) f.p[i] = col_frag(t + i * kC * kLdm, kLdm, k0, m0).p[0];
    return f;
}

// a 16 x 16 tile in the accumulators' layout: lane (i, g) holds rows r0 + 4g .. +3 of column c0 + i
__device__ __forceinline__ f32x4 tile_read(const __hip_bfloat16* t, int ld, int r0, int c0) {
    const s16x4 a = tr4(t, ld, r0, c0);
    f32x4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = __uint_as_float((uint32_t)(uint16_t)a[e] << 16);
    return v;
}
__device__ __forceinline__ f32x4 tile_read(const __half* t, int ld, int r0, int c0) {
    typedef _Float16 h4 __attribute__((ext_vector_type(4)));
    return __builtin_convertvector(__builtin_bit_cast(h4, tr4(t, ld, r0, c0)), f32x4);
}
__device__ __forceinline__ f32x4 tile_read(const float* t, int ld, int r0, int c0) {
    const int l = threadIdx.x & 63;
    const float* p = t + (r0 + 4 * (l >> 4)) * ld + c0 + (l & 15);
    f32x4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = p[e * ld];
    return v;
}
template <typename T> __device__ __forceinline__ void tile_write(T* t, int ld, int r0, int c0, f32x4 v) {
    const int l = threadIdx.x & 63;
    T* p = t + (r0 + 4 * (l >> 4)) * ld + c0 + (l & 15);
#pragma unroll
    for (int e = 0; e < 4; ++e) Elem<T>::st(p + e * ld, v[e]);
}
// a vector's four entries that belong to the rows of a tile
__device__ __forceinline__ f32x4 vec4(const float* v, int r0) { return *reinterpret_cast<const f32x4a*>(v + r0 + 4 * ((threadIdx.x & 63) >> 4)); }

__device__ __forceinline__ void lds_order() { asm volatile("" ::: "memory"); }   // a wave's LDS operations execute in order

// sum over the 16 lanes of a row group, in every lane
__device__ __forceinline__ float row16_sum(float v) {
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x128, 0xf, 0xf, false));
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x124, 0xf, 0xf, false));
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x122, 0xf, 0xf, false));
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x121, 0xf, 0xf, false));
    return v;
}

// ---- frames ---------------------------------------------------------------------------------------------
// position i of a head's walk -> frame: reversed heads walk an utterance's own frames backwards
struct Walk {
    int len;
    bool rev;
    __device__ __forceinline__ int64_t frame(int i) const { return rev && i < len ? len - 1 - i : i; }
};
__device__ __forceinline__ Walk walk_of(const GdrArgs& a, int b, int h) {
    Walk w;
    w.len = a.lengths ? min(max(a.lengths[b], 0), a.T) : a.T;
    w.rev = a.bidir && 2 * h >= a.H;
    return w;
}

// 64 frames x `ncol` columns (multiple of 8) from global rows into LDS [64][ld], columns up to `cols` and frames behind the end zero
template <typename T>
__device__ __forceinline__ void stage(T* dst, int ld, const T* src, int64_t ts, int ncol, int cols, int pos0, Walk w, int tid, int nt) {
    const int vpr = cols >> 3;
    for (int i = tid; i < kC * vpr; i += nt) {
        const int row = i / vpr, c = (i - row * vpr) * 8, p = pos0 + row;
        constexpr int Q = sizeof(T) / 2;       // 16-byte pieces
        u32x4a v[Q];
#pragma unroll
        for (int j = 0; j < Q; ++j) v[j] = u32x4a{0, 0, 0, 0};
        if (p < w.len && c < ncol) {
            const u32x4a* s = reinterpret_cast<const u32x4a*>(src + w.frame(p) * ts + c);
#pragma unroll
            for (int j = 0; j < Q; ++j) v[j] = s[j];
        }
        u32x4a* d = reinterpret_cast<u32x4a*>(dst + row * ld + c);
#pragma unroll
        for (int j = 0; j < Q; ++j) d[j] = v[j];
    }
}
// dense [planes][64][64] bf16 -> LDS planes of pitch kLdm
__device__ __forceinline__ void stage_planes(__bf16* dst, const __bf16* src, int planes, int tid, int nt) {
    for (int i = tid; i < planes * kC * 8; i += nt) {
        const int row = i >> 3, c = (i & 7) * 8;
        *reinterpret_cast<u32x4a*>(dst + row * kLdm + c) = *reinterpret_cast<const u32x4a*>(src + row * kC + c);
    }
}

// ---- prep -----------------------------------------------------------------------------------------------
template <typename T, int DK> struct PrepLds {
    static constexpr int LDK = DK + 8, LDN = kC + 4;
    static constexpr size_t bytes = (size_t)2 * kC * LDK * sizeof(T) + (size_t)2 * kC * LDN * 4 + 4 * 16 * 20 * 4 + kVec * kC * 4;
};

template <typename T, int DK, int NP>
__global__ __launch_bounds__(256) void gdr_prep_kernel(GdrArgs a) {
    extern __shared__ __align__(16) char smem[];
    using L = PrepLds<T, DK>;
    constexpr int PD = Gd<T>::PD, LDK = L::LDK, LDN = L::LDN;
    T* Kl = reinterpret_cast<T*>(smem);
    T* Ql = Kl + kC * LDK;
    float* N = reinterpret_cast<float*>(Ql + kC * LDK);
    float* P = N + kC * LDN;
    float* Tb = P + kC * LDN;                 // [4][16][20]
    float* vec = Tb + 4 * 16 * 20;
    double* G = reinterpret_cast<double*>(vec + kG64 * kC);
    const int c = blockIdx.x % a.nc, bh = blockIdx.x / a.nc, b = bh / a.H, h = bh % a.H, hk = h / a.r;
    const Walk w = walk_of(a, b, h);
    if (c * kC >= w.len) return;
    const int tid = threadIdx.x, l = tid & 63, wave = tid >> 6;
    stage(Kl, LDK, (const T*)a.k + b * a.ks[1] + hk * a.ks[2], a.ks[0], a.dk, DK, c * kC, w, tid, 256);
    stage(Ql, LDK, (const T*)a.q + b * a.qs[1] + hk * a.qs[2], a.qs[0], a.dk, DK, c * kC, w, tid, 256);
    if (wave == 0) {
        const int p = c * kC + l;
        const bool on = p < w.len;
        const int64_t t = on ? w.frame(p) : 0;
        // below -200 a decay is zero in f32 whatever the exact value; the clamp keeps sums and differences finite
        const float gv = on ? a.g[t * a.gs[0] + b * a.gs[1] + h * a.gs[2]] : 0.f;
        double s = gv < -200.f ? -200.0 : (double)gv;      // differences of long sums: 64 bits
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) { const double u = __shfl_up(s, o); if (l >= o) s += u; }
        G[l] = s;
        vec[kBe * kC + l] = on ? a.beta[t * a.bs[0] + b * a.bs[1] + h * a.bs[2]] : 0.f;
    }
    __syncthreads();
    {   // row norms: four lanes a row
        const int row = tid >> 2, part = tid & 3;
        float sk = 0.f, sq = 0.f;
        if (a.norm)
            for (int i = part; i < DK; i += 4) {
                const float kv = to_f(Kl[row * LDK + i]), qv = to_f(Ql[row * LDK + i]);
                sk += kv * kv; sq += qv * qv;
            }
        sk += __shfl_xor(sk, 1); sk += __shfl_xor(sk, 2);
        sq += __shfl_xor(sq, 1); sq += __shfl_xor(sq, 2);
        if (part == 0) {
            const float rk = a.norm ? 1.f / sqrtf(sk + 1e-6f) : 1.f, rq = (a.norm ? 1.f / sqrtf(sq + 1e-6f) : 1.f) * a.scale;
            const float eg = __expf((float)G[row]), ec = __expf((float)(G[kC - 1] - G[row]));
            vec[kAq * kC + row] = eg * rq;
            vec[kAk * kC + row] = eg * rk;
            vec[kKb * kC + row] = ec * rk;
            vec[kRk * kC + row] = rk;
            vec[kSq * kC + row] = rq;
        }
    }
    __syncthreads();
    // wave = block column of N and P
    for (int m = 0; m < 4; ++m) {
        f32x4 kk = {0, 0, 0, 0}, qk = {0, 0, 0, 0};
        if (m >= wave) {
#pragma unroll
            for (int kb = 0; kb < DK / 32; ++kb) {
                const auto bf = row_frag(Kl, LDK, 16 * wave, 32 * kb);
                kk = mma(row_frag(Kl, LDK, 16 * m, 32 * kb), bf, kk);
                qk = mma(row_frag(Ql, LDK, 16 * m, 32 * kb), bf, qk);
            }
            const int j = 16 * wave + (l & 15);
            const float rkj = vec[kRk * kC + j];
            const double gj = G[j];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int i = 16 * m + 4 * (l >> 4) + e;
                const float d = i >= j ? __expf((float)(G[i] - gj)) * rkj : 0.f;
                kk[e] = i > j ? kk[e] * d * vec[kRk * kC + i] : 0.f;
                qk[e] = i >= j ? qk[e] * d * vec[kSq * kC + i] : 0.f;
            }
        }
        tile_write(N, LDN, 16 * m, 16 * wave, kk);
        tile_write(P, LDN, 16 * m, 16 * wave, qk);
    }
    __syncthreads();
    {   // diagonal block `wave` of (I + N diag(beta))^-1 by substitution: lane = column, all lane groups alike
        float t[16];
        const int col = l & 15, base = 16 * wave;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float s = i == col ? 1.f : 0.f;
#pragma unroll
            for (int k = 0; k < i; ++k) s -= N[(base + i) * LDN + base + k] * vec[kBe * kC + base + k] * t[k];
            t[i] = s;
        }
        float* o = Tb + wave * 16 * 20;
        if (l < 16) {
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i * 20 + col] = t[i];
        }
    }
    __syncthreads();
    f32x4 X[4];
    {   // block column j = wave: X_ij = T_i (N_ij - sum_{j <= k < i} N_ik beta_k X_kj), on the f32 matrix instruction
        const int j = wave, g = l >> 4, i16 = l & 15;
        auto times = [&](const f32x4 av, const f32x4 bv, f32x4 acc) {   // inner index 4g + m at step m
#pragma unroll
            for (int m = 0; m < 4; ++m) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(av[m], bv[m], acc, 0, 0, 0);
            return acc;
        };
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            X[i] = f32x4{0, 0, 0, 0};
            if (i < j) continue;
            f32x4 s = {0, 0, 0, 0};
#pragma unroll
            for (int k = 0; k < i; ++k) {
                if (k < j) continue;
                f32x4 av = *reinterpret_cast<const f32x4a*>(N + (16 * i + i16) * LDN + 16 * k + 4 * g);
                av *= *reinterpret_cast<const f32x4a*>(vec + kBe * kC + 16 * k + 4 * g);
                s = times(av, X[k], s);
            }
            const f32x4 rhs = tile_read(N, LDN, 16 * i, 16 * j) - s;
            X[i] = times(*reinterpret_cast<const f32x4a*>(Tb + i * 16 * 20 + i16 * 20 + 4 * g), rhs, f32x4{0, 0, 0, 0});
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) tile_write(N, LDN, 16 * i, 16 * wave, X[i]);
    __syncthreads();
    const int64_t at = (int64_t)bh * a.nc + c;
    __bf16* Xo = a.X + at * PD * kC * kC;
    __bf16* Po = a.P + at * NP * kC * kC;
    for (int i = tid; i < kC * 8; i += 256) {
        const int row = i >> 3, col = (i & 7) * 8;
        const float* x = N + row * LDN + col;
        const float* p = P + row * LDN + col;
        const Frag<PD> xf = split<PD>(*reinterpret_cast<const f32x4a*>(x), *reinterpret_cast<const f32x4a*>(x + 4));
        const Frag<NP> pf = split<NP>(*reinterpret_cast<const f32x4a*>(p), *reinterpret_cast<const f32x4a*>(p + 4));
#pragma unroll
        for (int e = 0; e < PD; ++e) *reinterpret_cast<bf16x8*>(Xo + e * kC * kC + row * kC + col) = xf.p[e];
#pragma unroll
        for (int e = 0; e < NP; ++e) *reinterpret_cast<bf16x8*>(Po + e * kC * kC + row * kC + col) = pf.p[e];
    }
    float* vo = a.vec + at * kVec * kC;
    for (int i = tid; i < kVec * kC; i += 256) vo[i] = vec[i];
}

// ---- scan -----------------------------------------------------------------------------------------------
// rows [64][32 columns of this wave] from LDS to frames of a [T][B][H][dv] tensor, 16 bytes a lane; frames behind the end get nothing
template <typename T>
__device__ __forceinline__ void store_rows(const T* src, int ld, T* dst, int64_t ts, int ncol, int pos0, Walk w) {
    const int l = threadIdx.x & 63;
    constexpr int VE = 16 / sizeof(T), LPR = 32 / VE;       // elements a lane, lanes a row
    for (int r = l / LPR; r < kC; r += 64 / LPR) {
        const int p = pos0 + r, c = (l % LPR) * VE;
        if (p < w.len && c < ncol) *reinterpret_cast<u32x4a*>(dst + w.frame(p) * ts + c) = *reinterpret_cast<const u32x4a*>(src + r * ld + c);
    }
}
template <typename T>
__device__ __forceinline__ void zero_rows(T* dst, int64_t ts, int ncol, int from, int to, int tid, int nt) {
    constexpr int VE = 16 / sizeof(T);
    const int vpr = (ncol + VE - 1) / VE;
    for (int64_t i = tid; i < (int64_t)(to - from) * vpr; i += nt)
        *reinterpret_cast<u32x4a*>(dst + (from + i / vpr) * ts + (i % vpr) * VE) = u32x4a{0, 0, 0, 0};
}

template <typename T, int DK, int NW, int NP> struct ScanLds {
    static constexpr int LDK = DK + 8, LDV = NW * 32 + 8;
    static constexpr size_t bytes = (size_t)kC * (2 * LDK + LDV) * sizeof(T) + (size_t)(Gd<T>::PD + NP) * kC * kLdm * 2 + kVec * kC * 4;
};

template <typename T, int DK, int NW, int NP, bool TRAIN>
__global__ __launch_bounds__(NW * 64) void gdr_scan_kernel(GdrArgs a) {
    extern __shared__ __align__(16) char smem[];
    using L = ScanLds<T, DK, NW, NP>;
    constexpr int PD = Gd<T>::PD, LDK = L::LDK, LDV = L::LDV, KT = DK / 16;
    T* Kl = reinterpret_cast<T*>(smem);
    T* Ql = Kl + kC * LDK;
    T* Vl = Ql + kC * LDK;
    __bf16* Xl = reinterpret_cast<__bf16*>(Vl + kC * LDV);
    __bf16* Pl = Xl + PD * kC * kLdm;
    float* vec = reinterpret_cast<float*>(Pl + NP * kC * kLdm);
    const int groups = (a.nsl + NW - 1) / NW;
    const int bh = blockIdx.x / groups, sg = blockIdx.x % groups, b = bh / a.H, h = bh % a.H, hk = h / a.r;
    const Walk w = walk_of(a, b, h);
    const int tid = threadIdx.x, l = tid & 63, wave = tid >> 6, g = l >> 4, i16 = l & 15;
    const int col0 = (sg * NW + wave) * 32;                 // this wave's columns of dv
    const int vcols = min(a.dv - sg * NW * 32, NW * 32), mycols = a.dv - col0;
    const int64_t state = (int64_t)bh * a.dk * a.dv;
    f32x4 S[KT][2];
#pragma unroll
    for (int m = 0; m < KT; ++m)
#pragma unroll
        for (int ct = 0; ct < 2; ++ct)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int row = 16 * m + 4 * g + e, col = col0 + 16 * ct + i16;
                S[m][ct][e] = a.s0 && row < a.dk && col < a.dv ? a.s0[state + (int64_t)row * a.dv + col] : 0.f;
            }
    const T* kp = (const T*)a.k + b * a.ks[1] + hk * a.ks[2];
    const T* qp = (const T*)a.q + b * a.qs[1] + hk * a.qs[2];
    const T* vp = (const T*)a.v + b * a.vs[1] + h * a.vs[2] + sg * NW * 32;
    const int64_t ots = (int64_t)a.B * a.H * a.dv;
    T* op = (T*)a.o + ((int64_t)b * a.H + h) * a.dv;
    const int ncl = (w.len + kC - 1) / kC;
    for (int c = 0; c < ncl; ++c) {
        const int64_t at = (int64_t)bh * a.nc + c;
        __syncthreads();
        stage(Kl, LDK, kp, a.ks[0], a.dk, DK, c * kC, w, tid, NW * 64);
        stage(Ql, LDK, qp, a.qs[0], a.dk, DK, c * kC, w, tid, NW * 64);
        stage(Vl, LDV, vp, a.vs[0], vcols, NW * 32, c * kC, w, tid, NW * 64);
        stage_planes(Xl, a.X + at * PD * kC * kC, PD, tid, NW * 64);
        stage_planes(Pl, a.P + at * NP * kC * kC, NP, tid, NW * 64);
        for (int i = tid; i < kVec * kC; i += NW * 64) vec[i] = a.vec[at * kVec * kC + i];
        __syncthreads();
        if (mycols <= 0) continue;
        if (TRAIN) {      // the state at the chunk's start, for the backward
            float* so = a.S0 + at * a.dk * a.dv;
#pragma unroll
            for (int m = 0; m < KT; ++m)
#pragma unroll
                for (int ct = 0; ct < 2; ++ct)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int row = 16 * m + 4 * g + e, col = col0 + 16 * ct + i16;
                        if (row < a.dk && col < a.dv) so[(int64_t)row * a.dv + col] = S[m][ct][e];
                    }
        }
        f32x4 ks[4][2], qs[4][2];
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int ct = 0; ct < 2; ++ct) { ks[m][ct] = f32x4{0, 0, 0, 0}; qs[m][ct] = f32x4{0, 0, 0, 0}; }
#pragma unroll
        for (int kb = 0; kb < DK / 32; ++kb) {
            Frag<PD> sb[2];
#pragma unroll
            for (int ct = 0; ct < 2; ++ct) sb[ct] = split<PD>(S[2 * kb][ct], S[2 * kb + 1][ct]);
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                const auto kf = row_frag(Kl, LDK, 16 * m, 32 * kb);
                const auto qf = row_frag(Ql, LDK, 16 * m, 32 * kb);
#pragma unroll
                for (int ct = 0; ct < 2; ++ct) { ks[m][ct] = mma(kf, sb[ct], ks[m][ct]); qs[m][ct] = mma(qf, sb[ct], qs[m][ct]); }
            }
        }
        // Vt in ks; O's first part in qs
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            const f32x4 ak = vec4(vec + kAk * kC, 16 * m), aq = vec4(vec + kAq * kC, 16 * m);
#pragma unroll
            for (int ct = 0; ct < 2; ++ct) {
                ks[m][ct] = tile_read(Vl, LDV, 16 * m, wave * 32 + 16 * ct) - ak * ks[m][ct];
                qs[m][ct] *= aq;
            }
        }
        Frag<PD> uf[2][2];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            const f32x4 b0 = vec4(vec + kBe * kC, 32 * kb), b1 = vec4(vec + kBe * kC, 32 * kb + 16);
#pragma unroll
            for (int ct = 0; ct < 2; ++ct) uf[kb][ct] = split<PD>(b0 * ks[2 * kb][ct], b1 * ks[2 * kb + 1][ct]);
        }
#pragma unroll
        for (int m = 0; m < 4; ++m) {      // E = Vt - X (beta Vt); X is lower triangular: row tiles 0, 1 need the first 32 columns only
            f32x4 xs[2] = {f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}};
#pragma unroll
            for (int kb = 0; kb <= m / 2; ++kb) {
                const Frag<PD> xf = plane_rows<PD>(Xl, 16 * m, 32 * kb);
#pragma unroll
                for (int ct = 0; ct < 2; ++ct) xs[ct] = mma(xf, uf[kb][ct], xs[ct]);
            }
#pragma unroll
            for (int ct = 0; ct < 2; ++ct) ks[m][ct] -= xs[ct];
        }
        if (TRAIN) {
            float* eo = a.E + at * kC * a.dv;
#pragma unroll
            for (int m = 0; m < 4; ++m)
#pragma unroll
                for (int ct = 0; ct < 2; ++ct)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int col = col0 + 16 * ct + i16;
                        if (col < a.dv) eo[(int64_t)(16 * m + 4 * g + e) * a.dv + col] = ks[m][ct][e];
                    }
        }
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            const f32x4 b0 = vec4(vec + kBe * kC, 32 * kb), b1 = vec4(vec + kBe * kC, 32 * kb + 16);
#pragma unroll
            for (int ct = 0; ct < 2; ++ct) {
                ks[2 * kb][ct] *= b0;
                ks[2 * kb + 1][ct] *= b1;
                uf[kb][ct] = split<PD>(ks[2 * kb][ct], ks[2 * kb + 1][ct]);
            }
        }
#pragma unroll
        for (int m = 0; m < 4; ++m) {
#pragma unroll
            for (int kb = 0; kb <= m / 2; ++kb) {
                const Frag<NP> pf = plane_rows<NP>(Pl, 16 * m, 32 * kb);
#pragma unroll
                for (int ct = 0; ct < 2; ++ct) qs[m][ct] = mma(pf, uf[kb][ct], qs[m][ct]);
            }
        }
        // O leaves through this wave's own columns of the V tile, which it has read
        lds_order();
        T* my = Vl + wave * 32;
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int ct = 0; ct < 2; ++ct) tile_write(my, LDV, 16 * m, 16 * ct, qs[m][ct]);
        lds_order();
        store_rows(my, LDV, op + col0, ots, mycols, c * kC, w);
        if (TRAIN && sizeof(T) == 2) {      // what the rounding dropped (dO . O needs O in 32 bits)
#pragma unroll
            for (int m = 0; m < 4; ++m)
#pragma unroll
                for (int ct = 0; ct < 2; ++ct) qs[m][ct] -= tile_read(my, LDV, 16 * m, 16 * ct);
            lds_order();
            __hip_bfloat16* lo = reinterpret_cast<__hip_bfloat16*>(my);
#pragma unroll
            for (int m = 0; m < 4; ++m)
#pragma unroll
                for (int ct = 0; ct < 2; ++ct) tile_write(lo, LDV, 16 * m, 16 * ct, qs[m][ct]);
            lds_order();
            store_rows(lo, LDV, reinterpret_cast<__hip_bfloat16*>(a.olo) + ((int64_t)b * a.H + h) * a.dv + col0, ots, mycols, c * kC, w);
        }
        // S = e^{G_C} S + K^T (kb U)
        const float dec = __expf((float)reinterpret_cast<const double*>(vec + kG64 * kC)[kC - 1]);
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            const f32x4 b0 = vec4(vec + kKb * kC, 32 * kb), b1 = vec4(vec + kKb * kC, 32 * kb + 16);
#pragma unroll
            for (int ct = 0; ct < 2; ++ct) uf[kb][ct] = split<PD>(b0 * ks[2 * kb][ct], b1 * ks[2 * kb + 1][ct]);
        }
#pragma unroll
        for (int m = 0; m < KT; ++m) {
#pragma unroll
            for (int ct = 0; ct < 2; ++ct) S[m][ct] *= dec;
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                const auto kf = col_frag(Kl, LDK, 32 * kb, 16 * m);
#pragma unroll
                for (int ct = 0; ct < 2; ++ct) S[m][ct] = mma(kf, uf[kb][ct], S[m][ct]);
            }
        }
    }
#pragma unroll
    for (int m = 0; m < KT; ++m)
#pragma unroll
        for (int ct = 0; ct < 2; ++ct)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int row = 16 * m + 4 * g + e, col = col0 + 16 * ct + i16;
                if (row < a.dk && col < a.dv) a.sT[state + (int64_t)row * a.dv + col] = S[m][ct][e];
            }
    if (vcols > 0) zero_rows(op + sg * NW * 32, ots, vcols, w.len, a.T, tid, NW * 64);
}

// ---- reverse scan ---------------------------------------------------------------------------------------
template <typename T, int DK, int NW> struct RscanLds {
    static constexpr int LDK = DK + 8, LDV = NW * 32 + 8;
    static constexpr size_t bytes = (size_t)kC * (2 * LDK + 2 * LDV) * sizeof(T) + (size_t)2 * Gd<T>::PD * kC * kLdm * 2 + kVec * kC * 4;
};

template <typename T, int DK, int NW>
__global__ __launch_bounds__(NW * 64) void gdr_rscan_kernel(GdrArgs a) {
    extern __shared__ __align__(16) char smem[];
    using L = RscanLds<T, DK, NW>;
    constexpr int PD = Gd<T>::PD, LDK = L::LDK, LDV = L::LDV, KT = DK / 16;
    T* Kl = reinterpret_cast<T*>(smem);
    T* Ql = Kl + kC * LDK;
    T* Vl = Ql + kC * LDK;
    T* Ol = Vl + kC * LDV;                                  // dO
    __bf16* Xl = reinterpret_cast<__bf16*>(Ol + kC * LDV);
    __bf16* Pl = Xl + PD * kC * kLdm;
    float* vec = reinterpret_cast<float*>(Pl + PD * kC * kLdm);
    const int groups = (a.nsl + NW - 1) / NW;
    const int bh = blockIdx.x / groups, sg = blockIdx.x % groups, b = bh / a.H, h = bh % a.H, hk = h / a.r;
    const Walk w = walk_of(a, b, h);
    const int tid = threadIdx.x, l = tid & 63, wave = tid >> 6, g = l >> 4, i16 = l & 15;
    const int col0 = (sg * NW + wave) * 32;
    const int vcols = min(a.dv - sg * NW * 32, NW * 32), mycols = a.dv - col0;
    const int64_t state = (int64_t)bh * a.dk * a.dv;
    f32x4 S[KT][2];                                         // dS
#pragma unroll
    for (int m = 0; m < KT; ++m)
#pragma unroll
        for (int ct = 0; ct < 2; ++ct)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int row = 16 * m + 4 * g + e, col = col0 + 16 * ct + i16;
                S[m][ct][e] = a.gsT && row < a.dk && col < a.dv ? a.gsT[state + (int64_t)row * a.dv + col] : 0.f;
            }
    const T* kp = (const T*)a.k + b * a.ks[1] + hk * a.ks[2];
    const T* qp = (const T*)a.q + b * a.qs[1] + hk * a.qs[2];
    const T* vp = (const T*)a.v + b * a.vs[1] + h * a.vs[2] + sg * NW * 32;
    const T* gp = (const T*)a.go + b * a.gos[1] + h * a.gos[2] + sg * NW * 32;
    const int64_t ots = (int64_t)a.B * a.H * a.dv;
    T* gvp = (T*)a.gv + ((int64_t)b * a.H + h) * a.dv;
    const int ncl = (w.len + kC - 1) / kC;
    const int slice = sg * NW + wave;
    for (int c = ncl - 1; c >= 0; --c) {
        const int64_t at = (int64_t)bh * a.nc + c;
        __syncthreads();
        stage(Kl, LDK, kp, a.ks[0], a.dk, DK, c * kC, w, tid, NW * 64);
        stage(Ql, LDK, qp, a.qs[0], a.dk, DK, c * kC, w, tid, NW * 64);
        stage(Vl, LDV, vp, a.vs[0], vcols, NW * 32, c * kC, w, tid, NW * 64);
        stage(Ol, LDV, gp, a.gos[0], vcols, NW * 32, c * kC, w, tid, NW * 64);
        stage_planes(Xl, a.X + at * PD * kC * kC, PD, tid, NW * 64);
        stage_planes(Pl, a.P + at * PD * kC * kC, PD, tid, NW * 64);
        for (int i = tid; i < kVec * kC; i += NW * 64) vec[i] = a.vec[at * kVec * kC + i];
        __syncthreads();
        if (mycols <= 0) continue;
        const float dec = __expf((float)reinterpret_cast<const double*>(vec + kG64 * kC)[kC - 1]);
        float anchor = 0.f;
        {   // dS at the chunk's end is what the gradient kernel needs; <dS, S_C> = dec <dS, S0> + sum_j dU2_j . U_j
            float* so = a.dS + at * a.dk * a.dv;
            const float* s0 = a.S0 + at * a.dk * a.dv;
#pragma unroll
            for (int m = 0; m < KT; ++m)
#pragma unroll
                for (int ct = 0; ct < 2; ++ct)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int row = 16 * m + 4 * g + e, col = col0 + 16 * ct + i16;
                        if (row < a.dk && col < a.dv) {
                            so[(int64_t)row * a.dv + col] = S[m][ct][e];
                            anchor += S[m][ct][e] * s0[(int64_t)row * a.dv + col];
                        }
                    }
            anchor *= dec;
        }
        f32x4 du[4][2];
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int ct = 0; ct < 2; ++ct) du[m][ct] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int kb = 0; kb < DK / 32; ++kb) {
            Frag<PD> sb[2];
#pragma unroll
            for (int ct = 0; ct < 2; ++ct) sb[ct] = split<PD>(S[2 * kb][ct], S[2 * kb + 1][ct]);
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                const auto kf = row_frag(Kl, LDK, 16 * m, 32 * kb);
#pragma unroll
                for (int ct = 0; ct < 2; ++ct) du[m][ct] = mma(kf, sb[ct], du[m][ct]);
            }
        }
        f32x4 E[4][2];
        {
            const float* eo = a.E + at * kC * a.dv;
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                const f32x4 kb = vec4(vec + kKb * kC, 16 * m), be = vec4(vec + kBe * kC, 16 * m);
#pragma unroll
                for (int ct = 0; ct < 2; ++ct) {
                    const int col = col0 + 16 * ct + i16;
#pragma unroll
                    for (int e = 0; e < 4; ++e) E[m][ct][e] = col < a.dv ? eo[(int64_t)(16 * m + 4 * g + e) * a.dv + col] : 0.f;
                    du[m][ct] *= kb;
                    const f32x4 p = du[m][ct] * be * E[m][ct];
                    anchor += p[0] + p[1] + p[2] + p[3];
                }
            }
        }
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {      // + P^T dO: column tile m of P has rows >= 16 m
            Frag<Gd<T>::PT> of[2];
#pragma unroll
            for (int ct = 0; ct < 2; ++ct) of[ct] = col_frag(Ol, LDV, 32 * kb, wave * 32 + 16 * ct);
#pragma unroll
            for (int m = 0; m < 2 * kb + 2; ++m) {
                const Frag<PD> pf = plane_cols<PD>(Pl, 32 * kb, 16 * m);
#pragma unroll
                for (int ct = 0; ct < 2; ++ct) du[m][ct] = mma(pf, of[ct], du[m][ct]);
            }
        }
        Frag<PD> wf[2][2];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            const f32x4 b0 = vec4(vec + kBe * kC, 32 * kb), b1 = vec4(vec + kBe * kC, 32 * kb + 16);
#pragma unroll
            for (int ct = 0; ct < 2; ++ct) wf[kb][ct] = split<PD>(b0 * du[2 * kb][ct], b1 * du[2 * kb + 1][ct]);
        }
        float* xo = a.xpart + ((int64_t)slice * a.B * a.H * a.nc + at) * kC;
        float* bo = a.bpart + ((int64_t)slice * a.B * a.H * a.nc + at) * kC;
#pragma unroll
        for (int m = 0; m < 4; ++m) {      // F = dU - X^T (beta dU), dV = beta F
            f32x4 xs[2] = {f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}};
#pragma unroll
            for (int kb = m / 2; kb < 2; ++kb) {
                const Frag<PD> xf = plane_cols<PD>(Xl, 32 * kb, 16 * m);
#pragma unroll
                for (int ct = 0; ct < 2; ++ct) xs[ct] = mma(xf, wf[kb][ct], xs[ct]);
            }
            const f32x4 be = vec4(vec + kBe * kC, 16 * m);
            f32x4 sb = {0, 0, 0, 0}, sx = {0, 0, 0, 0};
#pragma unroll
            for (int ct = 0; ct < 2; ++ct) {
                du[m][ct] -= xs[ct];
                sb += E[m][ct] * du[m][ct];
                du[m][ct] *= be;
                sx += du[m][ct] * tile_read(Vl, LDV, 16 * m, wave * 32 + 16 * ct);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) { sb[e] = row16_sum(sb[e]); sx[e] = row16_sum(sx[e]); }
            if (i16 == 0) {
                *reinterpret_cast<f32x4a*>(bo + 16 * m + 4 * g) = sb;
                *reinterpret_cast<f32x4a*>(xo + 16 * m + 4 * g) = sx;
            }
        }
        anchor = wave_sum(anchor);
        if (l == 0) a.apart[(int64_t)slice * a.B * a.H * a.nc + at] = anchor;
        lds_order();
        T* my = Vl + wave * 32;
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int ct = 0; ct < 2; ++ct) tile_write(my, LDV, 16 * m, 16 * ct, du[m][ct]);
        lds_order();
        store_rows(my, LDV, gvp + col0, ots, mycols, c * kC, w);
        // dS = dec dS + Q^T (aq dO) - K^T (ak dV)
        Frag<PD> qf[2][2];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            const f32x4 k0 = vec4(vec + kAk * kC, 32 * kb), k1 = vec4(vec + kAk * kC, 32 * kb + 16);
            const f32x4 q0 = vec4(vec + kAq * kC, 32 * kb), q1 = vec4(vec + kAq * kC, 32 * kb + 16);
#pragma unroll
            for (int ct = 0; ct < 2; ++ct) {
                wf[kb][ct] = split<PD>(-k0 * du[2 * kb][ct], -k1 * du[2 * kb + 1][ct]);
                qf[kb][ct] = split<PD>(q0 * tile_read(Ol, LDV, 32 * kb, wave * 32 + 16 * ct), q1 * tile_read(Ol, LDV, 32 * kb + 16, wave * 32 + 16 * ct));
            }
        }
#pragma unroll
        for (int m = 0; m < KT; ++m) {
#pragma unroll
            for (int ct = 0; ct < 2; ++ct) S[m][ct] *= dec;
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                const auto kf = col_frag(Kl, LDK, 32 * kb, 16 * m);
                const auto qa = col_frag(Ql, LDK, 32 * kb, 16 * m);
#pragma unroll
                for (int ct = 0; ct < 2; ++ct) S[m][ct] = mma(qa, qf[kb][ct], mma(kf, wf[kb][ct], S[m][ct]));
            }
        }
    }
    if (a.gs0) {
#pragma unroll
        for (int m = 0; m < KT; ++m)
#pragma unroll
            for (int ct = 0; ct < 2; ++ct)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int row = 16 * m + 4 * g + e, col = col0 + 16 * ct + i16;
                    if (row < a.dk && col < a.dv) a.gs0[state + (int64_t)row * a.dv + col] = S[m][ct][e];
                }
    }
    if (vcols > 0) zero_rows(gvp + sg * NW * 32, ots, vcols, w.len, a.T, tid, NW * 64);
}

// ---- gradients of a chunk ---------------------------------------------------------------------------------
template <typename T> struct MatT { using type = float; };
template <> struct MatT<__hip_bfloat16> { using type = __hip_bfloat16; };

template <typename T, int DK> struct GradLds {
    using M = typename MatT<T>::type;
    static constexpr int LDK = DK + 8, LDV = 136, LDM = sizeof(M) == 2 ? 72 : 68;
    static constexpr size_t tiles = (size_t)3 * kC * LDV > (size_t)2 * kC * LDK ? (size_t)3 * kC * LDV : (size_t)2 * kC * LDK;
    static constexpr size_t bytes = tiles * sizeof(T) + (size_t)2 * kC * LDM * sizeof(M) + (kVec + 8 + 1) * kC * 4;
};

template <typename T, int DK>
__global__ __launch_bounds__(256) void gdr_grads_kernel(GdrArgs a) {
    extern __shared__ __align__(16) char smem[];
    using L = GradLds<T, DK>;
    using M = typename L::M;
    constexpr int PT = Gd<T>::PT, LDK = L::LDK, LDV = L::LDV, LDM = L::LDM, NT = DK / 64;
    T* tile = reinterpret_cast<T*>(smem);
    T *Ol = tile, *Dl = tile + kC * LDV, *Ul = tile + 2 * kC * LDV;      // dO, dV, U
    T *Kl = tile, *Ql = tile + kC * LDK;                                  // later
    M* M1 = reinterpret_cast<M*>(tile + L::tiles);
    M* M2 = M1 + kC * LDM;
    float* vec = reinterpret_cast<float*>(M2 + kC * LDM);
    const double* G = reinterpret_cast<const double*>(vec + kG64 * kC);
    float* dots = vec + kVec * kC;                                        // [2][4][64]
    float* ys = dots + 8 * kC;
    const int c = blockIdx.x % a.nc, bk = blockIdx.x / a.nc, b = bk / a.Hk, hk = bk % a.Hk;
    const int tid = threadIdx.x, l = tid & 63, wave = tid >> 6, g = l >> 4, i16 = l & 15;
    const Walk w = walk_of(a, b, hk * a.r);
    const int64_t kts = (int64_t)a.B * a.Hk * a.dk, gts = (int64_t)a.B * a.H;
    T* gqp = (T*)a.gq + ((int64_t)b * a.Hk + hk) * a.dk;
    T* gkp = (T*)a.gk + ((int64_t)b * a.Hk + hk) * a.dk;
    const int p0 = c * kC;
    // frames of this chunk behind the utterance's end: zero gradients
    const int z0 = max(p0, w.len), z1 = min(p0 + kC, a.T);
    if (z0 < z1) {
        zero_rows(gqp, kts, a.dk, z0, z1, tid, 256);
        zero_rows(gkp, kts, a.dk, z0, z1, tid, 256);
        for (int i = tid; i < (z1 - z0) * a.r; i += 256) {
            const int64_t o = (int64_t)(z0 + i / a.r) * gts + (int64_t)b * a.H + hk * a.r + i % a.r;
            a.gg[o] = 0.f;
            a.gbeta[o] = 0.f;
        }
    }
    if (p0 >= w.len) return;
    f32x4 tq[4][NT], tk[4][NT];
#pragma unroll
    for (int m = 0; m < 4; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n) { tq[m][n] = f32x4{0, 0, 0, 0}; tk[m][n] = f32x4{0, 0, 0, 0}; }
    const int64_t ots = (int64_t)a.B * a.H * a.dv, nbh = (int64_t)a.B * a.H;
    for (int hh = 0; hh < a.r; ++hh) {
        const int h = hk * a.r + hh, bh = b * a.H + h;
        const int64_t at = (int64_t)bh * a.nc + c;
        __syncthreads();
        for (int i = tid; i < kVec * kC; i += 256) vec[i] = a.vec[at * kVec * kC + i];
        stage(Ol, LDV, (const T*)a.go + b * a.gos[1] + h * a.gos[2], a.gos[0], a.dv, 128, p0, w, tid, 256);
        stage(Dl, LDV, (const T*)a.gv + (int64_t)bh * a.dv, ots, a.dv, 128, p0, w, tid, 256);
        {
            const float* e = a.E + at * kC * a.dv;
            for (int i = tid; i < kC * 32; i += 256) {
                const int row = i >> 5, col = (i & 31) * 4;
                const float be = a.vec[at * kVec * kC + kBe * kC + row];
                f32x4 v = {0, 0, 0, 0};
                if (col < a.dv && p0 + row < w.len) v = *reinterpret_cast<const f32x4a*>(e + row * a.dv + col);
#pragma unroll
                for (int j = 0; j < 4; ++j) Elem<T>::st(Ul + row * LDV + col + j, v[j] * be);
            }
        }
        __syncthreads();
        {   // dO . O per frame: four lanes a row
            const int row = tid >> 2, part = tid & 3, p = p0 + row;
            float y = 0.f;
            if (p < w.len) {
                const int64_t o = w.frame(p) * ots + (int64_t)bh * a.dv;
                for (int i = part * 4; i < a.dv; i += 16)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        float ov = Elem<T>::ld((const T*)a.o + o + i + j);
                        if (sizeof(T) == 2) ov += (float)a.olo[o + i + j];
                        y += to_f(Ol[row * LDV + i + j]) * ov;
                    }
            }
            y += __shfl_xor(y, 1); y += __shfl_xor(y, 2);
            if (part == 0) ys[row] = y;
        }
        // states: wave = a quarter of dk
        {
            const float* s0 = a.S0 + at * a.dk * a.dv;
            const float* ds = a.dS + at * a.dk * a.dv;
            f32x4 cq[4][NT], ck[4][NT], cd[4][NT];
#pragma unroll
            for (int m = 0; m < 4; ++m)
#pragma unroll
                for (int n = 0; n < NT; ++n) { cq[m][n] = f32x4{0, 0, 0, 0}; ck[m][n] = cq[m][n]; cd[m][n] = cq[m][n]; }
            for (int kb = 0; kb * 32 < a.dv; ++kb) {
                Frag<PT> sf[NT], df[NT];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const int row = (wave * NT + n) * 16 + i16, c0 = 32 * kb + 4 * g, c1 = c0 + 16;
                    f32x4 s_0 = {0, 0, 0, 0}, s_1 = s_0, d_0 = s_0, d_1 = s_0;
                    if (row < a.dk && c0 < a.dv) {
                        s_0 = *reinterpret_cast<const f32x4a*>(s0 + (int64_t)row * a.dv + c0);
                        d_0 = *reinterpret_cast<const f32x4a*>(ds + (int64_t)row * a.dv + c0);
                    }
                    if (row < a.dk && c1 < a.dv) {
                        s_1 = *reinterpret_cast<const f32x4a*>(s0 + (int64_t)row * a.dv + c1);
                        d_1 = *reinterpret_cast<const f32x4a*>(ds + (int64_t)row * a.dv + c1);
                    }
                    sf[n] = split<PT>(s_0, s_1);
                    df[n] = split<PT>(d_0, d_1);
                }
#pragma unroll
                for (int m = 0; m < 4; ++m) {
                    const auto of = row_frag(Ol, LDV, 16 * m, 32 * kb);
                    const auto uf = row_frag(Ul, LDV, 16 * m, 32 * kb);
                    const auto vf = row_frag(Dl, LDV, 16 * m, 32 * kb);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        cq[m][n] = mma(of, sf[n], cq[m][n]);
                        ck[m][n] = mma(uf, df[n], ck[m][n]);
                        cd[m][n] = mma(vf, sf[n], cd[m][n]);
                    }
                }
            }
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                const f32x4 aq = vec4(vec + kAq * kC, 16 * m), ak = vec4(vec + kAk * kC, 16 * m), kb = vec4(vec + kKb * kC, 16 * m);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    tq[m][n] += aq * cq[m][n];
                    tk[m][n] += kb * ck[m][n] - ak * cd[m][n];
                }
            }
        }
        // M1 = dP * D * sq_i * rk_j (lower), M2 = (dN * D * rk_i * rk_j) made symmetric; wave = block column
        for (int m = 0; m < 4; ++m) {
            f32x4 dp = {0, 0, 0, 0}, dn = {0, 0, 0, 0};
            if (m < wave) {
                tile_write(M1, LDM, 16 * m, 16 * wave, dp);
                continue;
            }
            for (int kb = 0; kb * 32 < a.dv; ++kb) {
                const auto uf = row_frag(Ul, LDV, 16 * wave, 32 * kb);
                dp = mma(row_frag(Ol, LDV, 16 * m, 32 * kb), uf, dp);
                dn = mma(row_frag(Dl, LDV, 16 * m, 32 * kb), uf, dn);
            }
            const int j = 16 * wave + i16;
            const float rkj = vec[kRk * kC + j];
            const double gj = G[j];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int i = 16 * m + 4 * g + e;
                const float d = i >= j ? __expf((float)(G[i] - gj)) * rkj : 0.f;
                dp[e] = i >= j ? dp[e] * d * vec[kSq * kC + i] : 0.f;
                dn[e] = i > j ? -dn[e] * d * vec[kRk * kC + i] : 0.f;
                if (i > j) Elem<M>::st(M2 + j * LDM + i, dn[e]);
                if (i >= j) Elem<M>::st(M2 + i * LDM + j, dn[e]);
            }
            tile_write(M1, LDM, 16 * m, 16 * wave, dp);
        }
        __syncthreads();
        stage(Kl, LDK, (const T*)a.k + b * a.ks[1] + hk * a.ks[2], a.ks[0], a.dk, DK, p0, w, tid, 256);
        stage(Ql, LDK, (const T*)a.q + b * a.qs[1] + hk * a.qs[2], a.qs[0], a.dk, DK, p0, w, tid, 256);
        if (wave == 0) {      // dg and dbeta: lane = frame
            float z = ys[l], be = 0.f, an = 0.f;
            for (int s = 0; s < a.nsl; ++s) {
                z -= a.xpart[(s * nbh * a.nc + at) * kC + l];
                be += a.bpart[(s * nbh * a.nc + at) * kC + l];
                an += a.apart[s * nbh * a.nc + at];
            }
            if (p0 + l >= w.len) z = 0.f;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) { const float u = __shfl_down(z, o); if (l + o < 64) z += u; }
            if (p0 + l < w.len) {
                const int64_t o = w.frame(p0 + l) * gts + bh;
                a.gg[o] = z + an;
                a.gbeta[o] = be;
            }
        }
        __syncthreads();
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const int n0 = (wave * NT + n) * 16;
                const auto kf = col_frag(Kl, LDK, 32 * kb, n0);
                const auto qf = col_frag(Ql, LDK, 32 * kb, n0);
#pragma unroll
                for (int m = 0; m < 4; ++m) {
                    tq[m][n] = mma(row_frag(M1, LDM, 16 * m, 32 * kb), kf, tq[m][n]);
                    tk[m][n] = mma(col_frag(M1, LDM, 32 * kb, 16 * m), qf, tk[m][n]);
                    tk[m][n] = mma(row_frag(M2, LDM, 16 * m, 32 * kb), kf, tk[m][n]);
                }
            }
        }
    }
    // through the normalisation: dq = tq - q |q|^-2 (q . tq)  (|.|^2 with its epsilon), dk alike
    if (a.norm) {
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            f32x4 sq = {0, 0, 0, 0}, sk = {0, 0, 0, 0};
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const int n0 = (wave * NT + n) * 16;
                sq += tq[m][n] * tile_read(Ql, LDK, 16 * m, n0);
                sk += tk[m][n] * tile_read(Kl, LDK, 16 * m, n0);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) { sq[e] = row16_sum(sq[e]); sk[e] = row16_sum(sk[e]); }
            if (i16 == 0) {
                *reinterpret_cast<f32x4a*>(dots + wave * kC + 16 * m + 4 * g) = sq;
                *reinterpret_cast<f32x4a*>(dots + (4 + wave) * kC + 16 * m + 4 * g) = sk;
            }
        }
        __syncthreads();
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            f32x4 sq = {0, 0, 0, 0}, sk = {0, 0, 0, 0};
#pragma unroll
            for (int x = 0; x < 4; ++x) { sq += vec4(dots + x * kC, 16 * m); sk += vec4(dots + (4 + x) * kC, 16 * m); }
            const f32x4 rk = vec4(vec + kRk * kC, 16 * m), rq = vec4(vec + kSq * kC, 16 * m) * (1.f / a.scale);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const int n0 = (wave * NT + n) * 16;
                tq[m][n] -= sq * rq * rq * tile_read(Ql, LDK, 16 * m, n0);
                tk[m][n] -= sk * rk * rk * tile_read(Kl, LDK, 16 * m, n0);
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int m = 0; m < 4; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            tile_write(Ql, LDK, 16 * m, (wave * NT + n) * 16, tq[m][n]);
            tile_write(Kl, LDK, 16 * m, (wave * NT + n) * 16, tk[m][n]);
        }
    __syncthreads();
    constexpr int VE = 16 / sizeof(T);
    const int vpr = a.dk / VE;
    for (int i = tid; i < kC * vpr; i += 256) {
        const int row = i / vpr, col = (i % vpr) * VE, p = p0 + row;
        if (p >= w.len) continue;
        const int64_t t = w.frame(p);
        *reinterpret_cast<u32x4a*>(gqp + t * kts + col) = *reinterpret_cast<const u32x4a*>(Ql + row * LDK + col);
        *reinterpret_cast<u32x4a*>(gkp + t * kts + col) = *reinterpret_cast<const u32x4a*>(Kl + row * LDK + col);
    }
}

// ---- recurrent form -------------------------------------------------------------------------------------
// Few frames: a workgroup owns 32 columns of one head's state, in registers: 8 lanes x 4 columns a row, 32 row groups of up to four rows.
// One reduction a frame: k.S and q.S come from the state before the frame, o follows from u.
template <typename T>
__global__ __launch_bounds__(256) void gdr_recurrent_kernel(GdrArgs a) {
    __shared__ float red[2][4][8][12];
    const int bh = blockIdx.x / a.nsl, sl = blockIdx.x % a.nsl, b = bh / a.H, h = bh % a.H, hk = h / a.r;
    const Walk w = walk_of(a, b, h);
    const int tid = threadIdx.x, wave = tid >> 6, cl = tid & 7, rg = tid >> 3;
    const int col = sl * 32 + cl * 4;
    const bool con = col < a.dv;
    const int64_t state = (int64_t)bh * a.dk * a.dv;
    f32x4 S[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = i * 32 + rg;
        S[i] = f32x4{0, 0, 0, 0};
        if (a.s0 && con && row < a.dk) S[i] = *reinterpret_cast<const f32x4a*>(a.s0 + state + (int64_t)row * a.dv + col);
    }
    const T* kp = (const T*)a.k + b * a.ks[1] + hk * a.ks[2];
    const T* qp = (const T*)a.q + b * a.qs[1] + hk * a.qs[2];
    const T* vp = (const T*)a.v + b * a.vs[1] + h * a.vs[2];
    T* op = (T*)a.o + ((int64_t)b * a.H + h) * a.dv;
    const int64_t ots = (int64_t)a.B * a.H * a.dv;
    for (int p = 0; p < w.len; ++p) {
        const int64_t t = w.frame(p);
        float k[4], q[4], acc[11];
        f32x4 v = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = i * 32 + rg;
            k[i] = row < a.dk ? Elem<T>::ld(kp + t * a.ks[0] + row) : 0.f;
            q[i] = row < a.dk ? Elem<T>::ld(qp + t * a.qs[0] + row) : 0.f;
        }
        if (con) {
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = Elem<T>::ld(vp + t * a.vs[0] + col + j);
        }
        const float gv = a.g[t * a.gs[0] + b * a.gs[1] + h * a.gs[2]], be = a.beta[t * a.bs[0] + b * a.bs[1] + h * a.bs[2]];
#pragma unroll
        for (int j = 0; j < 11; ++j) acc[j] = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) { acc[j] += k[i] * S[i][j]; acc[4 + j] += q[i] * S[i][j]; }
            acc[8] += k[i] * k[i];
            acc[9] += q[i] * q[i];
            acc[10] += q[i] * k[i];
        }
#pragma unroll
        for (int j = 0; j < 11; ++j) {
            acc[j] += __shfl_xor(acc[j], 8);
            acc[j] += __shfl_xor(acc[j], 16);
            acc[j] += __shfl_xor(acc[j], 32);
        }
        float(*rd)[8][12] = red[p & 1];
        if ((tid & 63) < 8) {
#pragma unroll
            for (int j = 0; j < 11; ++j) rd[wave][cl][j] = acc[j];
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 11; ++j) acc[j] = rd[0][cl][j] + rd[1][cl][j] + rd[2][cl][j] + rd[3][cl][j];
        const float rk = a.norm ? 1.f / sqrtf(acc[8] + 1e-6f) : 1.f, sq = (a.norm ? 1.f / sqrtf(acc[9] + 1e-6f) : 1.f) * a.scale;
        const float dec = __expf(gv);
        f32x4 u, o;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            u[j] = be * (v[j] - dec * rk * acc[j]);
            o[j] = sq * (dec * acc[4 + j] + rk * acc[10] * u[j]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) S[i] = dec * S[i] + (rk * k[i]) * u;
        if (rg == 0 && con) {
#pragma unroll
            for (int j = 0; j < 4; ++j) Elem<T>::st(op + t * ots + col + j, o[j]);
        }
    }
    if (rg == 0 && con) {
        for (int t = w.len; t < a.T; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) Elem<T>::st(op + t * ots + col + j, 0.f);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = i * 32 + rg;
        if (con && row < a.dk) *reinterpret_cast<f32x4a*>(a.sT + state + (int64_t)row * a.dv + col) = S[i];
    }
}

// ---- host -----------------------------------------------------------------------------------------------
static int gdr_check(const char* who, int T, int B, int Hk, int H, int dk, int dv, int flags, int dtype) {
    SP_CHECK_ARG(T >= 0 && T < (1 << 24) && B >= 0 && Hk >= 1 && H >= 1 && H % Hk == 0, "%s: bad shape T=%d B=%d Hk=%d H=%d (H a multiple of Hk)", who, T, B, Hk, H);
    SP_CHECK_ARG(dk >= 8 && dk <= 128 && dk % 8 == 0 && dv >= 8 && dv <= 128 && dv % 8 == 0, "%s: dk=%d and dv=%d must be multiples of 8 in [8, 128]", who, dk, dv);
    SP_CHECK_ARG((flags & ~(SP_GDR_NORMALIZE | SP_GDR_BIDIRECTIONAL)) == 0, "%s: unknown flags %d", who, flags);
    SP_CHECK_ARG(!(flags & SP_GDR_BIDIRECTIONAL) || Hk % 2 == 0, "%s: both directions need an even number of key heads, not %d", who, Hk);
    SP_CHECK_ARG(dtype == SP_F32 || dtype == SP_BF16 || dtype == SP_F16, "%s: dtype %d not supported (f32, bf16, f16)", who, dtype);
    SP_CHECK_ARG((int64_t)B * H * ((T + kC - 1) / kC + 4) < (1ll << 22), "%s: B=%d x H=%d x %d frames exceed the grid", who, B, H, T);
    return SP_OK;
}

static int parts_d(int dtype) { return dtype == SP_F32 ? 3 : 2; }

struct GdrLayout { size_t vec, X, P, S0, E, olo, end; };
static GdrLayout gdr_saved(int T, int B, int H, int dk, int dv, int dtype, bool train) {
    GdrLayout s{};
    const size_t n = (size_t)B * H * ((T + kC - 1) / kC);
    const int pd = parts_d(dtype), np = train || dtype != SP_BF16 ? pd : 1;
    size_t o = 0;
    auto put = [&](size_t bytes) { const size_t at = o; o = align_up(o + bytes, 256); return at; };
    s.vec = put(n * kVec * kC * 4);
    s.X = put(n * pd * kC * kC * 2);
    s.P = put(n * np * kC * kC * 2);
    if (train) {
        s.S0 = put(n * dk * dv * 4);
        s.E = put(n * kC * dv * 4);
        s.olo = put(dtype == SP_F32 ? 0 : (size_t)T * B * H * dv * 2);
    }
    s.end = o;
    return s;
}
struct GdrBwdLayout { size_t dS, x, b, a, end; };
static GdrBwdLayout gdr_bwd_ws(int T, int B, int H, int dk, int dv) {
    GdrBwdLayout s{};
    const size_t n = (size_t)B * H * ((T + kC - 1) / kC), nsl = (dv + 31) / 32;
    size_t o = 0;
    auto put = [&](size_t bytes) { const size_t at = o; o = align_up(o + bytes, 256); return at; };
    s.dS = put(n * dk * dv * 4);
    s.x = put(n * nsl * kC * 4);
    s.b = put(n * nsl * kC * 4);
    s.a = put(n * nsl * 4);
    s.end = o;
    return s;
}

static bool gdr_aligned(const void* p, const int64_t* st, int dtype) {
    const int64_t ve = dtype == SP_F32 ? 4 : 8;
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && st[0] % ve == 0 && st[1] % ve == 0 && st[2] % ve == 0;
}

template <typename K> static int gdr_launch(K kernel, size_t lds, int64_t blocks, int threads, const GdrArgs& a, hipStream_t s, const char* what) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(threads), lds, s, a);
    return check_launch(what);
}

static void gdr_fill(GdrArgs& a, const void* q, const void* k, const void* v, const float* g, const float* beta, const int32_t* lengths,
                     const int64_t* st, int T, int B, int Hk, int H, int dk, int dv, float scale, int flags) {
    a.q = q; a.k = k; a.v = v; a.g = g; a.beta = beta; a.lengths = lengths;
    for (int i = 0; i < 3; ++i) { a.qs[i] = st[i]; a.ks[i] = st[3 + i]; a.vs[i] = st[6 + i]; a.gs[i] = st[9 + i]; a.bs[i] = st[12 + i]; }
    a.T = T; a.B = B; a.Hk = Hk; a.H = H; a.r = H / Hk; a.dk = dk; a.dv = dv;
    a.nc = (T + kC - 1) / kC; a.nsl = (dv + 31) / 32;
    a.scale = scale;
    a.norm = flags & SP_GDR_NORMALIZE ? 1 : 0;
    a.bidir = flags & SP_GDR_BIDIRECTIONAL ? 1 : 0;
}

template <typename T, int DK, int NP, bool TRAIN> static int gdr_forward(const GdrArgs& a, hipStream_t s) {
    int rc = gdr_launch(gdr_prep_kernel<T, DK, NP>, PrepLds<T, DK>::bytes, (int64_t)a.B * a.H * a.nc, 256, a, s, "gdr_prep_kernel");
    if (rc) return rc;
    constexpr int NW = 4;
    return gdr_launch(gdr_scan_kernel<T, DK, NW, NP, TRAIN>, ScanLds<T, DK, NW, NP>::bytes, (int64_t)a.B * a.H * ((a.nsl + NW - 1) / NW), NW * 64, a,
                      s, "gdr_scan_kernel");
}
template <typename T, int DK> static int gdr_backward(const GdrArgs& a, hipStream_t s) {
    constexpr int NW = sizeof(T) == 4 && DK == 128 ? 2 : 4;
    int rc = gdr_launch(gdr_rscan_kernel<T, DK, NW>, RscanLds<T, DK, NW>::bytes, (int64_t)a.B * a.H * ((a.nsl + NW - 1) / NW), NW * 64, a, s,
                        "gdr_rscan_kernel");
    if (rc) return rc;
    return gdr_launch(gdr_grads_kernel<T, DK>, GradLds<T, DK>::bytes, (int64_t)a.B * a.Hk * a.nc, 256, a, s, "gdr_grads_kernel");
}

}  // namespace sp

using namespace sp;

extern "C" size_t sp_gdr_workspace_bytes(int T, int B, int Hk, int H, int dk, int dv, int dtype, int backward) {
    if (gdr_check("sp_gdr_workspace_bytes", T, B, Hk, H, dk, dv, 0, dtype)) return 0;
    return backward ? gdr_bwd_ws(T, B, H, dk, dv).end : gdr_saved(T, B, H, dk, dv, dtype, false).end;
}
extern "C" size_t sp_gdr_saved_bytes(int T, int B, int Hk, int H, int dk, int dv, int dtype) {
    if (gdr_check("sp_gdr_saved_bytes", T, B, Hk, H, dk, dv, 0, dtype)) return 0;
    return gdr_saved(T, B, H, dk, dv, dtype, true).end;
}

extern "C" int sp_gdr_fwd(const void* q, const void* k, const void* v, const float* g, const float* beta, const float* state,
                          const int32_t* lengths, const int64_t* strides, int T, int B, int Hk, int H, int dk, int dv, float scale, int flags,
                          int dtype, void* o, float* state_out, void* saved, size_t saved_bytes, void* workspace, size_t workspace_bytes,
                          void* stream) {
    int rc = gdr_check("sp_gdr_fwd", T, B, Hk, H, dk, dv, flags, dtype);
    if (rc) return rc;
    if (B == 0) return SP_OK;
    SP_CHECK_ARG(state_out && strides, "sp_gdr_fwd: null pointer");
    SP_CHECK_ARG(T == 0 || (q && k && v && g && beta && o), "sp_gdr_fwd: null pointer");
    SP_CHECK_ARG(reinterpret_cast<uintptr_t>(state) % 16 == 0 && reinterpret_cast<uintptr_t>(state_out) % 16 == 0 && reinterpret_cast<uintptr_t>(o) % 16 == 0,
                 "sp_gdr_fwd: state and o must be 16-byte aligned");
    GdrArgs a{};
    gdr_fill(a, q, k, v, g, beta, lengths, strides, T, B, Hk, H, dk, dv, scale, flags);
    a.s0 = state; a.sT = state_out; a.o = o;
    hipStream_t s = (hipStream_t)stream;
    const bool train = saved != nullptr;
    if (!train && T <= kRecurrentMax) {
        const int64_t blocks = (int64_t)B * H * a.nsl;
        if (dtype == SP_F32) return gdr_launch(gdr_recurrent_kernel<float>, 0, blocks, 256, a, s, "gdr_recurrent_kernel");
        if (dtype == SP_F16) return gdr_launch(gdr_recurrent_kernel<__half>, 0, blocks, 256, a, s, "gdr_recurrent_kernel");
        return gdr_launch(gdr_recurrent_kernel<__hip_bfloat16>, 0, blocks, 256, a, s, "gdr_recurrent_kernel");
    }
    SP_CHECK_ARG(gdr_aligned(q, strides, dtype) && gdr_aligned(k, strides + 3, dtype) && gdr_aligned(v, strides + 6, dtype),
                 "sp_gdr_fwd: q, k, v need 16-byte aligned rows");
    const GdrLayout lay = gdr_saved(T, B, H, dk, dv, dtype, train);
    if (train ? saved_bytes < lay.end : workspace_bytes < lay.end || !workspace)
        return fail(SP_EWORKSPACE, "sp_gdr_fwd: %s %zu < %zu bytes", train ? "saved" : "workspace", train ? saved_bytes : workspace_bytes, lay.end);
    char* base = (char*)(train ? saved : workspace);
    a.vec = (float*)(base + lay.vec); a.X = (__bf16*)(base + lay.X); a.P = (__bf16*)(base + lay.P);
    a.S0 = (float*)(base + lay.S0); a.E = (float*)(base + lay.E); a.olo = (__bf16*)(base + lay.olo);
    const bool wide = dk > 64;
#define SP_GDR_FWD(T_, NP_, TR_) return wide ? gdr_forward<T_, 128, NP_, TR_>(a, s) : gdr_forward<T_, 64, NP_, TR_>(a, s)
    if (train) {
        if (dtype == SP_F32) SP_GDR_FWD(float, 3, true);
        if (dtype == SP_F16) SP_GDR_FWD(__half, 2, true);
        SP_GDR_FWD(__hip_bfloat16, 2, true);
    }
    if (dtype == SP_F32) SP_GDR_FWD(float, 3, false);
    if (dtype == SP_F16) SP_GDR_FWD(__half, 2, false);
    SP_GDR_FWD(__hip_bfloat16, 1, false);
#undef SP_GDR_FWD
}

extern "C" int sp_gdr_bwd(const void* q, const void* k, const void* v, const float* g, const float* beta, const int32_t* lengths,
                          const int64_t* strides, int T, int B, int Hk, int H, int dk, int dv, float scale, int flags, int dtype,
                          const void* o, const void* saved, size_t saved_bytes, const void* go, const float* gstate_out, void* gq, void* gk,
                          void* gv, float* gg, float* gbeta, float* gstate, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = gdr_check("sp_gdr_bwd", T, B, Hk, H, dk, dv, flags, dtype);
    if (rc) return rc;
    if (B == 0) return SP_OK;
    SP_CHECK_ARG(scale != 0.f, "sp_gdr_bwd: scale is zero");
    SP_CHECK_ARG(T > 0, "sp_gdr_bwd: T=0 has nothing to differentiate");
    SP_CHECK_ARG(q && k && v && g && beta && strides && o && saved && go && gq && gk && gv && gg && gbeta && workspace, "sp_gdr_bwd: null pointer");
    SP_CHECK_ARG(gdr_aligned(q, strides, dtype) && gdr_aligned(k, strides + 3, dtype) && gdr_aligned(v, strides + 6, dtype) &&
                     gdr_aligned(go, strides + 15, dtype), "sp_gdr_bwd: q, k, v, go need 16-byte aligned rows");
    const GdrLayout lay = gdr_saved(T, B, H, dk, dv, dtype, true);
    const GdrBwdLayout ws = gdr_bwd_ws(T, B, H, dk, dv);
    if (saved_bytes < lay.end || workspace_bytes < ws.end)
        return fail(SP_EWORKSPACE, "sp_gdr_bwd: saved %zu < %zu or workspace %zu < %zu bytes", saved_bytes, lay.end, workspace_bytes, ws.end);
    GdrArgs a{};
    gdr_fill(a, q, k, v, g, beta, lengths, strides, T, B, Hk, H, dk, dv, scale, flags);
    char* base = (char*)saved;
    a.vec = (float*)(base + lay.vec); a.X = (__bf16*)(base + lay.X); a.P = (__bf16*)(base + lay.P);
    a.S0 = (float*)(base + lay.S0); a.E = (float*)(base + lay.E); a.olo = (__bf16*)(base + lay.olo);
    a.o = (void*)o; a.go = go; a.gsT = gstate_out;
    for (int i = 0; i < 3; ++i) a.gos[i] = strides[15 + i];
    char* wb = (char*)workspace;
    a.dS = (float*)(wb + ws.dS); a.xpart = (float*)(wb + ws.x); a.bpart = (float*)(wb + ws.b); a.apart = (float*)(wb + ws.a);
    a.gq = gq; a.gk = gk; a.gv = gv; a.gg = gg; a.gbeta = gbeta; a.gs0 = gstate;
    hipStream_t s = (hipStream_t)stream;
    const bool wide = dk > 64;
    if (dtype == SP_F32) return wide ? gdr_backward<float, 128>(a, s) : gdr_backward<float, 64>(a, s);
    if (dtype == SP_F16) return wide ? gdr_backward<__half, 128>(a, s) : gdr_backward<__half, 64>(a, s);
    return wide ? gdr_backward<__hip_bfloat16, 128>(a, s) : gdr_backward<__hip_bfloat16, 64>(a, s);
}
