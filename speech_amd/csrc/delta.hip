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
// bf16 parts (x = hi + mid + lo): an input of type bf16 is one exact part, f16 two, f32 three; what is derived (S, U, X, ...) three, which
// is all of an f32's mantissa, wherever a result of 32 bits (states, dg, dbeta) hangs on it.  With two parts those results were off by
// 3e-6 to 1e-5 instead of 3e-7; the f32 matrix instruction costs 5.3 times a bf16 one, three to six bf16 products at most as much.  What
// only reaches a 16-bit output (o, dq, dk) takes two parts.  Outputs of 16-bit type are rounded once.
//
// Kernels: prep (N, P, X of a chunk; all chunks at once) -> scan (walks the chunks with S in registers; a wave owns 16 columns of dv and
// never talks to the others: the accumulator layout of one product is the B operand of the next) ; backward: rscan (the same walk in
// reverse with dS) -> grads (dq, dk, dg, dbeta of a chunk; all chunks at once).  Few frames (streaming, single tokens): one recurrent kernel.
#include "common.h"

#include <initializer_list>
#include <type_traits>

namespace sp {

constexpr int kC = 64;              // frames a chunk
// Frames up to which the recurrent kernel runs (inference).  It costs 3 us + 0.95 us a frame for few heads, the two chunked kernels 17 to
// 20 us for any number up to 64, and their second launch: at 12 frames 14.7 us against 16.6 (8 heads, bf16, dk 64), 14.8 against 20 (dk 128),
// at 16 frames 18.2 against 17; at 12 frames of 256 heads 24.9 against 21.1, of 512 at dk 128 43 against 38, at 8 frames 31 against 39.
constexpr int kRecurrentMax = 12;
constexpr int kLdm = 72;            // row pitch (elements) of a 64 x 64 matrix plane in LDS: 16 rows of 8 bytes fall on distinct banks
constexpr int kVec = 8;             // per-chunk vectors of 64 floats: aq, ak, kb, beta, rk, sq, G (as 64 doubles)
constexpr int kTri = 10 * 256;      // a lower triangular 64 x 64 matrix: ten 16 x 16 blocks (row block major), f32
enum { kAq = 0, kAk = 1, kKb = 2, kBe = 3, kRk = 4, kSq = 5, kG64 = 6 };

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
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
    int T, B, Hk, H, r, dk, dv, nc, nsl;             // nsl: slices of 16 columns of dv
    float scale;
    int norm, bidir, fresh;                          // fresh: the walk began without a state
    void* o;
    float* sT;
    // kept between the kernels (and, in training, for the backward)
    float* vec;              // [bh][nc][kVec][64]
    float *X, *P;            // [bh][nc][kTri]
    float* S0;               // [bh][nc][dk][dv]: the state at the chunk's start
    // backward
    const void* go;
    const float* gsT;
    float* dS;               // [bh][nc][dk][dv]: the state's gradient at the chunk's end
    uint32_t* E;             // [bh][nc][64][dv]: f32; for 16-bit types words of pack_ev
    float *zpart, *bpart;    // [nsl][bh][nc][64]: dO.O - dV.V and E.F over 16 columns
    float* apart;            // [nsl][bh][nc]
    void *gq, *gk, *gv;
    float *gg, *gbeta, *gs0;
    int64_t gos[3];
};

// ---- operand fragments --------------------------------------------------------------------------------
// PT: parts of an input; OP: parts of what is derived, where it reaches a 16-bit output only (S, U, P in o's product)
template <typename T> struct Gd;
template <> struct Gd<__hip_bfloat16> { static constexpr int PT = 1, OP = 2; };
template <> struct Gd<__half> { static constexpr int PT = 2, OP = 2; };
template <> struct Gd<float> { static constexpr int PT = 3, OP = 3; };

template <int P> struct Frag { bf16x8 p[P]; };

// One part is rounded to nearest.  Of several, all but the last are cut off (the upper 16 bits as they stand: one v_perm packs two, and
// three parts of 8 bits are exactly an f32's 24); the last of two is rounded.
__device__ __forceinline__ uint32_t cvt_pk(float a, float b) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const f32x2 v = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
}
template <int P> __device__ __forceinline__ Frag<P> split(f32x8 v) {
    Frag<P> f;
#pragma unroll
    for (int i = 0; i < P; ++i) {
        u32x4a w;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float x = v[2 * j], y = v[2 * j + 1];
            const uint32_t a = __float_as_uint(x), b = __float_as_uint(y);
            if (i + 1 < P || P == 3) w[j] = __builtin_amdgcn_perm(b, a, 0x07060302u);
            else w[j] = cvt_pk(x, y);
            if (i + 1 < P) {
                x -= __uint_as_float(a & 0xFFFF0000u);
                y -= __uint_as_float(b & 0xFFFF0000u);
                v[2 * j] = x;
                v[2 * j + 1] = y;
            }
        }
        f.p[i] = __builtin_bit_cast(bf16x8, w);
    }
    return f;
}
template <int P> __device__ __forceinline__ Frag<P> split(f32x4 a, f32x4 b) {
    return split<P>(__builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

// the parts of four values, as the planes of a matrix in LDS take them
template <int P, typename F> __device__ __forceinline__ void parts4(f32x4 v, F&& put) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
        u32x2a w;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const float x = v[2 * j], y = v[2 * j + 1];
            const uint32_t a = __float_as_uint(x), b = __float_as_uint(y);
            if (i + 1 < P || P == 3) w[j] = __builtin_amdgcn_perm(b, a, 0x07060302u);
            else w[j] = cvt_pk(x, y);
            if (i + 1 < P) {
                v[2 * j] = x - __uint_as_float(a & 0xFFFF0000u);
                v[2 * j + 1] = y - __uint_as_float(b & 0xFFFF0000u);
            }
        }
        put(i, w);
    }
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

// four row tiles' operands for one block of 32 inner indices; one column tile's for both blocks
template <typename T, int P> __device__ __forceinline__ void row_frags(Frag<P> (&f)[4], const T* t, int ld, int c0) {
#pragma unroll
    for (int m = 0; m < 4; ++m) f[m] = row_frag(t, ld, 16 * m, c0);
}
template <typename T, int P> __device__ __forceinline__ void col_frags(Frag<P> (&f)[2], const T* t, int ld, int m0) {
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) f[kb] = col_frag(t, ld, 32 * kb, m0);
}
// the six operands of a lower triangular 64 x 64 matrix: number x is row tile tri_m(x), block tri_k(x); of its transpose, column tile and
// block 3 - tri_m(x), 1 - tri_k(x)
constexpr int tri_m(int x) { return x < 2 ? x : x < 4 ? 2 : 3; }
constexpr int tri_k(int x) { return x == 3 || x == 5; }
template <int P, int A, int B> __device__ __forceinline__ void tri_rows(Frag<P> (&f)[6], const __bf16* t) {
#pragma unroll
    for (int x = A; x < B; ++x) f[x] = plane_rows<P>(t, 16 * tri_m(x), 32 * tri_k(x));
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

__device__ __forceinline__ int opaque(int x) {
    asm volatile("" : "+v"(x));
    return x;
}

// ---- frames ---------------------------------------------------------------------------------------------
// position i of a head's walk -> frame: reversed heads walk an utterance's own frames backwards
struct Walk {
    int len;
    bool rev;
    __device__ __forceinline__ int64_t frame(int i) const { return rev && i < len ? len - 1 - i : i; }
    // the lowest frame of the chunk at position p0 and, for a position p < len of that chunk, the distance from it (0 .. 63): addresses are
    // a uniform 64-bit base and a 32-bit offset a lane (the host refuses frames that lie more than 32 MiB apart)
    __device__ __forceinline__ int64_t low(int p0) const { return rev ? max(0, len - p0 - kC) : p0; }
    __device__ __forceinline__ uint32_t above(int p0, int p) const { return rev ? (uint32_t)(len - 1 - p - max(0, len - p0 - kC)) : (uint32_t)(p - p0); }
};
__device__ __forceinline__ Walk walk_of(const GdrArgs& a, int b, int h) {
    Walk w;
    w.len = a.lengths ? min(max(a.lengths[b], 0), a.T) : a.T;
    w.rev = a.bidir && 2 * h >= a.H;
    return w;
}

// A thread's share of a tile of 64 frames x COLS columns on its way from global memory to LDS: requested a chunk ahead, in registers.
// Loads are unconditional at clamped addresses (a branch around each would serialise them); what lies outside becomes zero on the way out.
// Needs w.len > 0 and ncol >= 8.
template <typename T, int COLS, int NT> struct TileRegs {
    static constexpr int Q = sizeof(T) / 2, N = (kC * COLS / 8 + NT - 1) / NT;
    u32x4a v[N][Q];
    __device__ __forceinline__ void load(const T* src, int64_t ts, int ncol, int pos0, Walk w) {
        const char* base = reinterpret_cast<const char*>(src + w.low(pos0) * ts);
        const int tid = opaque(threadIdx.x);
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int i = tid + n * NT, row = i / (COLS / 8), c = i % (COLS / 8) * 8;
            const uint32_t off = w.above(pos0, min(pos0 + row, w.len - 1)) * (uint32_t)(ts * sizeof(T)) + (uint32_t)(min(c, ncol - 8) * sizeof(T));
            const u32x4a* s = reinterpret_cast<const u32x4a*>(base + off);
#pragma unroll
            for (int j = 0; j < Q; ++j) v[n][j] = s[j];
        }
    }
    __device__ __forceinline__ void store(T* dst, int ld, int ncol, int pos0, int len) const {
        const int tid = opaque(threadIdx.x);
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int i = tid + n * NT, row = i / (COLS / 8), c = i % (COLS / 8) * 8;
            u32x4a* d = reinterpret_cast<u32x4a*>(dst + row * ld + c);
            if (N * NT == kC * COLS / 8 || row < kC) {
                if (pos0 + kC <= len && ncol == COLS) {
#pragma unroll
                    for (int j = 0; j < Q; ++j) d[j] = v[n][j];
                } else {
                    const bool on = pos0 + row < len && c < ncol;
#pragma unroll
                    for (int j = 0; j < Q; ++j) d[j] = on ? v[n][j] : u32x4a{0, 0, 0, 0};
                }
            }
        }
    }
};
// the same for a lower triangular matrix, split into bf16 planes when it is stored
template <int NT> struct TriRegs {
    static constexpr int N = (kTri / 4 + NT - 1) / NT;
    f32x4a v[N];
    __device__ __forceinline__ void load(const float* src) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            v[n] = reinterpret_cast<const f32x4a*>(src)[min((int)threadIdx.x + n * NT, kTri / 4 - 1)];
        }
    }
    template <int P> __device__ __forceinline__ void store(__bf16* dst) const {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int i = threadIdx.x + n * NT, blk = i >> 6;
            if (i < kTri / 4) {
                const int bi = blk >= 6 ? 3 : blk >= 3 ? 2 : blk >= 1 ? 1 : 0, bj = blk - bi * (bi + 1) / 2;
                __bf16* d = dst + (16 * bi + ((i >> 2) & 15)) * kLdm + 16 * bj + 4 * (i & 3);
                parts4<P>(v[n], [&](int e, u32x2a h) { *reinterpret_cast<u32x2a*>(d + e * kC * kLdm) = h; });
            }
        }
    }
};
// the blocks right of the diagonal that products over 32 columns touch: (0, 1) and (2, 3).  A loop that ends lane by lane: in front of
// everything that lives in registers (see gdr_grads_kernel)
__device__ __forceinline__ void clear_upper(__bf16* t, int planes, int tid, int nt) {
    for (int i = tid; i < planes * 64; i += nt) {
        const int pl = i >> 6, row = (i >> 1) & 31, half = i & 1;
        const int r = row & 15, blk = (row >> 4) * 2;
        *reinterpret_cast<u32x4a*>(t + pl * kC * kLdm + (16 * blk + r) * kLdm + 16 * (blk + 1) + 8 * half) = u32x4a{0, 0, 0, 0};
    }
}

// Measured below at T = 751, 256 heads (32 x 8), dk 64, dv 128, bf16, normalised, both directions, unless another shape is named.

// ---- prep -----------------------------------------------------------------------------------------------
// A workgroup forms N, P, the inverse's X and the chunk's vectors for one (head, chunk): 44 us (94 MB: 2.1 TB/s).  Bound by
// its chain of dependent steps (loads, prefix sum, norms, products, substitution), not by bytes or rate: so little LDS (26 KB) and few
// registers (92) that five workgroups share a CU and fill each other's waits; with N and P both kept in LDS it was three, and 53 us.
// X by blocks of 16: the four diagonal blocks of (I + N diag(beta))^-1 by substitution, one a wave, the blocks below them by products on the
// f32 matrix instruction: the inverse multiplies everything behind it, and bf16 parts would have to be formed of each intermediate block.
template <typename T, int DK> struct PrepLds {
    static constexpr int LDK = DK + 8, LDN = kC + 4;
    static constexpr size_t in = (size_t)2 * kC * LDK * sizeof(T), mat = (size_t)kC * LDN * 4;
    static constexpr size_t bytes = (in > mat ? in : mat) + 4 * 16 * 20 * 4 + kVec * kC * 4;
};

// block (i, j) of a lower triangular matrix, from the accumulators' layout
__device__ __forceinline__ void block_store(float* t, int i, int j, f32x4 v) {
    const int l = threadIdx.x & 63;
    float* p = t + (i * (i + 1) / 2 + j) * 256 + 64 * (l >> 4) + (l & 15);
#pragma unroll
    for (int e = 0; e < 4; ++e) p[16 * e] = v[e];
}

template <typename T, int DK>
__global__ __launch_bounds__(256) void gdr_prep_kernel(GdrArgs a) {
    extern __shared__ __align__(16) char smem[];
    using L = PrepLds<T, DK>;
    constexpr int LDK = L::LDK, LDN = L::LDN;
    T* Kl = reinterpret_cast<T*>(smem);
    T* Ql = Kl + kC * LDK;
    float* N = reinterpret_cast<float*>(smem);    // over K and Q once their products are done
    float* Tb = reinterpret_cast<float*>(smem + (L::in > L::mat ? L::in : L::mat));   // [4][16][20]
    float* vec = Tb + 4 * 16 * 20;
    double* G = reinterpret_cast<double*>(vec + kG64 * kC);
    const int c = blockIdx.x % a.nc, bh = blockIdx.x / a.nc, b = bh / a.H, h = bh % a.H, hk = h / a.r;
    const Walk w = walk_of(a, b, h);
    if (c * kC >= w.len) return;
    const int64_t at = (int64_t)bh * a.nc + c;
    const int tid = threadIdx.x, l = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    TileRegs<T, DK, 256> tk, tq;
    tk.load((const T*)a.k + b * a.ks[1] + hk * a.ks[2], a.ks[0], a.dk, c * kC, w);
    tq.load((const T*)a.q + b * a.qs[1] + hk * a.qs[2], a.qs[0], a.dk, c * kC, w);
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
    tk.store(Kl, LDK, a.dk, c * kC, w.len);
    tq.store(Ql, LDK, a.dk, c * kC, w.len);
    __syncthreads();
    {   // row norms: four lanes a row
        const int row = tid >> 2, part = tid & 3;
        float sk = 0.f, sq = 0.f;
        if (a.norm) {
#pragma unroll
            for (int i = 0; i < DK / 32; ++i) {
                T x[8], y[8];
                __builtin_memcpy(x, __builtin_assume_aligned(Kl + row * LDK + 32 * i + 8 * part, 16), sizeof(x));
                __builtin_memcpy(y, __builtin_assume_aligned(Ql + row * LDK + 32 * i + 8 * part, 16), sizeof(y));
#pragma unroll
                for (int e = 0; e < 8; ++e) { sk += to_f(x[e]) * to_f(x[e]); sq += to_f(y[e]) * to_f(y[e]); }
            }
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
    f32x4 kk[4], qk[4];
#pragma unroll
    for (int m = 0; m < 4; ++m) { kk[m] = f32x4{0, 0, 0, 0}; qk[m] = kk[m]; }
#pragma unroll
    for (int kb = 0; kb < DK / 32; ++kb) {
        const auto bf = row_frag(Kl, LDK, 16 * wave, 32 * kb);
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            kk[m] = mma<Gd<T>::PT, Gd<T>::PT, 3>(row_frag(Kl, LDK, 16 * m, 32 * kb), bf, kk[m]);
            qk[m] = mma<Gd<T>::PT, Gd<T>::PT, 3>(row_frag(Ql, LDK, 16 * m, 32 * kb), bf, qk[m]);
        }
    }
    __syncthreads();
    {
        const int j = 16 * wave + (l & 15);
        const float rkj = vec[kRk * kC + j];
        const double gj = G[j];
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            const f32x4 sqi = vec4(vec + kSq * kC, 16 * m), rki = vec4(vec + kRk * kC, 16 * m);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int i = 16 * m + 4 * (l >> 4) + e;
                const float d = __expf((float)(G[i] - gj)) * rkj;      // above the diagonal it may be infinite: selected away
                const float n = kk[m][e] * d * rki[e], p = qk[m][e] * d * sqi[e];
                kk[m][e] = i > j ? n : 0.f;
                qk[m][e] = i >= j ? p : 0.f;
            }
            tile_write(N, LDN, 16 * m, 16 * wave, kk[m]);
            if (m >= wave) block_store(a.P + at * kTri, m, wave, qk[m]);
        }
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
            block_store(a.X + at * kTri, i, j, X[i]);
        }
    }
    float* vo = a.vec + at * kVec * kC;
#pragma unroll
    for (int x = 0; x < kVec * kC / 256; ++x) vo[x * 256 + tid] = vec[x * 256 + tid];
}

// A state's 16 columns in the accumulators' layout from / to rows [dk][dv].  One 32-bit lane offset in bytes, everything else is uniform; dk
// is a multiple of 8, so a lane's four rows lie inside or outside together.
template <int KT> __device__ __forceinline__ void state_load(f32x4 (&S)[KT], const float* p, int dk, int dv, int col0) {
    const int g4 = 4 * ((threadIdx.x & 63) >> 4), col = col0 + (threadIdx.x & 15);
    const char* base = reinterpret_cast<const char*>(p);
    if (dk == 16 * KT && col0 + 16 <= dv) {
        const uint32_t off = (uint32_t)(g4 * dv + col) * 4u;
#pragma unroll
        for (int m = 0; m < KT; ++m)
#pragma unroll
            for (int e = 0; e < 4; ++e) S[m][e] = *reinterpret_cast<const float*>(base + (uint32_t)(16 * m + e) * dv * 4u + off);
    } else {
#pragma unroll
        for (int m = 0; m < KT; ++m) {
            const bool in = 16 * m + g4 < dk && col < dv;
            const uint32_t off = in ? (uint32_t)((16 * m + g4) * dv + col) * 4u : 0u;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float x = *reinterpret_cast<const float*>(base + (uint32_t)(e * dv) * 4u + off);
                S[m][e] = in ? x : 0.f;
            }
        }
    }
}
template <int KT> __device__ __forceinline__ void state_store(const f32x4 (&S)[KT], float* p, int dk, int dv, int col0) {
    const int g4 = 4 * ((threadIdx.x & 63) >> 4), col = col0 + (threadIdx.x & 15);
    char* base = reinterpret_cast<char*>(p);
    const uint32_t off = (uint32_t)(g4 * dv + col) * 4u;
    if (dk == 16 * KT && col0 + 16 <= dv) {
#pragma unroll
        for (int m = 0; m < KT; ++m)
#pragma unroll
            for (int e = 0; e < 4; ++e) *reinterpret_cast<float*>(base + (uint32_t)(16 * m + e) * dv * 4u + off) = S[m][e];
    } else {
#pragma unroll
        for (int m = 0; m < KT; ++m)
            if (16 * m + g4 < dk && col < dv) {
#pragma unroll
                for (int e = 0; e < 4; ++e) *reinterpret_cast<float*>(base + (uint32_t)(16 * m + e) * dv * 4u + off) = S[m][e];
            }
    }
}

// Nothing is scheduled across.  Between two such lines stand the LDS reads of the next products and the matrix instructions of the present
// ones: left alone, the compiler reads one fragment, waits for it, multiplies, and reads the next.
__device__ __forceinline__ void phase_end() { __builtin_amdgcn_sched_barrier(0); }

// ---- scan -----------------------------------------------------------------------------------------------
// rows [64][16 columns of this wave] from LDS to a chunk's frames, 16 bytes a lane
template <typename T>
__device__ __forceinline__ void store_rows(const T* src, int ld, int ncol, T* dst, int64_t ts, int pos0, Walk w) {
    const int l = threadIdx.x & 63;
    constexpr int VE = 16 / sizeof(T), LPR = 16 / VE;       // elements a lane, lanes a row
    char* base = reinterpret_cast<char*>(dst + w.low(pos0) * ts);
#pragma unroll
    for (int x = 0; x < LPR; ++x) {
        const int r = l / LPR + x * (64 / LPR), c = (l % LPR) * VE;
        if (pos0 + r < w.len && c < ncol)
            *reinterpret_cast<u32x4a*>(base + (w.above(pos0, pos0 + r) * (uint32_t)(ts * sizeof(T)) + (uint32_t)(c * sizeof(T)))) =
                *reinterpret_cast<const u32x4a*>(src + r * ld + c);
    }
}
template <typename T>
__device__ __forceinline__ void zero_rows(T* dst, int64_t ts, int ncol, int from, int to, int tid, int nt) {
    constexpr int VE = 16 / sizeof(T);
    const int vpr = (ncol + VE - 1) / VE;
    for (int64_t i = tid; i < (int64_t)(to - from) * vpr; i += nt)
        *reinterpret_cast<u32x4a*>(dst + (from + i / vpr) * ts + (i % vpr) * VE) = u32x4a{0, 0, 0, 0};
}

template <typename T, int DK, int NW> struct ScanLds {
    static constexpr int LDK = DK + 8, LDV = NW * 16 + 8;
    static constexpr size_t bytes = (size_t)kC * (2 * LDK + LDV) * sizeof(T) + (size_t)(3 + Gd<T>::OP) * kC * kLdm * 2 + kVec * kC * 4;
};

// B operands (inner index = rows of the accumulators) of 64 frames: row tiles 2 kb and 2 kb + 1, each scaled by a vector
template <int P> __device__ __forceinline__ void row_operands(Frag<P> (&f)[2], const float* scale, const f32x4 (&t)[4]) {
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) f[kb] = split<P>(vec4(scale, 32 * kb) * t[2 * kb], vec4(scale, 32 * kb + 16) * t[2 * kb + 1]);
}

// A wave owns 16 columns of dv: the state's columns, U's, O's.  Only K, Q, X, P and the vectors are shared (LDS, filled a chunk ahead
// through registers); two barriers a chunk.  A wave whose columns lie behind dv works on zeros and writes nothing: as many steps as the
// others, and no branch around the matrix instructions.
// 100 to 105 us, 12 chunks in turn: 8.5 us a chunk, of which the matrix pipes are busy 18 %.  P takes two parts: with one, o was off by 1.34 times
// its own rounding (bf16: 2.2e-3 of the two-norm instead of 1.66e-3) for 2.5 us less.  Bound by the chain of three dependent products a chunk
// (K S, X, K^T U), with Q S and P U, which feed o alone, behind the same waits, at two waves a SIMD; the states are the only thing that could
// be split further, and every split loads K, Q, X and P again.  Inference at dk 128 (T = 1501, 128 heads, one wave a SIMD): 139 us, 24 chunks (132 with one part of P).
template <typename T, int DK, int NW, bool TRAIN>
__global__ __launch_bounds__(NW * 64) void gdr_scan_kernel(GdrArgs a) {
    extern __shared__ __align__(16) char smem[];
    using L = ScanLds<T, DK, NW>;
    constexpr int NT = NW * 64, PT = Gd<T>::PT, OP = Gd<T>::OP, LDK = L::LDK, LDV = L::LDV, KT = DK / 16;
    constexpr bool AHEAD = PT == 1;      // operands of one part fit the registers ahead of their use
    T* Kl = reinterpret_cast<T*>(smem);
    T* Ql = Kl + kC * LDK;
    T* Vl = Ql + kC * LDK;
    __bf16* Xl = reinterpret_cast<__bf16*>(Vl + kC * LDV);
    __bf16* Pl = Xl + 3 * kC * kLdm;
    float* vec = reinterpret_cast<float*>(Pl + OP * kC * kLdm);
    const int groups = (a.nsl + NW - 1) / NW;
    const int bh = blockIdx.x / groups, sg = blockIdx.x % groups, b = bh / a.H, h = bh % a.H, hk = h / a.r;
    const Walk w = walk_of(a, b, h);
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col0 = (sg * NW + wave) * 16;                        // this wave's columns of dv
    const int vcols = min(a.dv - sg * NW * 16, NW * 16), mycols = a.dv - col0;
    const int64_t state = (int64_t)bh * a.dk * a.dv;
    clear_upper(Xl, 3 + OP, tid, NT);
    f32x4 S[KT];
#pragma unroll
    for (int m = 0; m < KT; ++m) S[m] = f32x4{0, 0, 0, 0};
    if (a.s0) state_load(S, a.s0 + state, a.dk, a.dv, col0);
    const T* kp = (const T*)a.k + b * a.ks[1] + hk * a.ks[2];
    const T* qp = (const T*)a.q + b * a.qs[1] + hk * a.qs[2];
    const T* vp = (const T*)a.v + b * a.vs[1] + h * a.vs[2] + sg * NW * 16;
    const int64_t ots = (int64_t)a.B * a.H * a.dv;
    T* op = (T*)a.o + ((int64_t)b * a.H + h) * a.dv;
    const int ncl = (w.len + kC - 1) / kC;
    TileRegs<T, DK, NT> rk, rq;
    TileRegs<T, NW * 16, NT> rv;
    TriRegs<NT> rx, rp;
    float rvec[kVec * kC / NT];
    auto fetch = [&](int c) {
        const int64_t at = (int64_t)bh * a.nc + c;
        rk.load(kp, a.ks[0], a.dk, c * kC, w);
        rq.load(qp, a.qs[0], a.dk, c * kC, w);
        rv.load(vp, a.vs[0], vcols, c * kC, w);
        rx.load(a.X + at * kTri);
        rp.load(a.P + at * kTri);
#pragma unroll
        for (int i = 0; i < kVec * kC / NT; ++i) rvec[i] = a.vec[at * kVec * kC + i * NT + tid];
    };
    if (ncl > 0) fetch(0);
    for (int c = 0; c < ncl; ++c) {
        const int64_t at = (int64_t)bh * a.nc + c;
        __syncthreads();
        rk.store(Kl, LDK, a.dk, c * kC, w.len);
        rq.store(Ql, LDK, a.dk, c * kC, w.len);
        rv.store(Vl, LDV, vcols, c * kC, w.len);
        rx.template store<3>(Xl);
        rp.template store<OP>(Pl);
#pragma unroll
        for (int i = 0; i < kVec * kC / NT; ++i) vec[i * NT + tid] = rvec[i];
        __syncthreads();
        if (c + 1 < ncl) fetch(c + 1);
        if (TRAIN) state_store(S, a.S0 + at * a.dk * a.dv, a.dk, a.dv, col0);      // for the backward
        f32x4 ks[4], qs[4];
#pragma unroll
        for (int m = 0; m < 4; ++m) { ks[m] = f32x4{0, 0, 0, 0}; qs[m] = ks[m]; }
        Frag<PT> kf[2][4], qf[2][4];
        row_frags(kf[0], Kl, LDK, 0);
        row_frags(qf[0], Ql, LDK, 0);
        Frag<3> xf[6];
        f32x4 vt[4];
#pragma unroll
        for (int kb = 0; kb < DK / 32; ++kb) {
            if (kb + 1 < DK / 32) {
                row_frags(kf[(kb + 1) & 1], Kl, LDK, 32 * (kb + 1));
                row_frags(qf[(kb + 1) & 1], Ql, LDK, 32 * (kb + 1));
            } else {
#pragma unroll
                for (int m = 0; m < 4; ++m) vt[m] = tile_read(Vl, LDV, 16 * m, wave * 16);
                if (AHEAD) tri_rows<3, 0, 3>(xf, Xl);
            }
            const Frag<3> sb = split<3>(S[2 * kb], S[2 * kb + 1]);
            if (AHEAD) phase_end();
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                ks[m] = mma(kf[kb & 1][m], sb, ks[m]);
                qs[m] = mma<PT, 3, OP>(qf[kb & 1][m], sb, qs[m]);
            }
            if (AHEAD) phase_end();
        }
        // Vt in ks; O's first part in qs
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            ks[m] = vt[m] - vec4(vec + kAk * kC, 16 * m) * ks[m];
            qs[m] *= vec4(vec + kAq * kC, 16 * m);
        }
        Frag<3> uf[2];
        row_operands(uf, vec + kBe * kC, ks);
        // E = Vt - X (beta Vt), U = beta E; X is lower triangular: row tiles 0, 1 need the first 32 columns only
        f32x4 xs[4];
#pragma unroll
        for (int m = 0; m < 4; ++m) xs[m] = f32x4{0, 0, 0, 0};
        tri_rows<3, AHEAD ? 3 : 0, 6>(xf, Xl);
        if (AHEAD) phase_end();
#pragma unroll
        for (int x = 0; x < 3; ++x) xs[tri_m(x)] = mma(xf[x], uf[tri_k(x)], xs[tri_m(x)]);
        if (AHEAD) phase_end();
        Frag<OP> pf[6];
        tri_rows<OP, 0, 3>(pf, Pl);
        if (AHEAD) phase_end();
#pragma unroll
        for (int x = 3; x < 6; ++x) xs[tri_m(x)] = mma(xf[x], uf[tri_k(x)], xs[tri_m(x)]);
#pragma unroll
        for (int m = 0; m < 4; ++m) ks[m] = (ks[m] - xs[m]) * vec4(vec + kBe * kC, 16 * m);
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) uf[kb] = split<3>(ks[2 * kb], ks[2 * kb + 1]);
        if (AHEAD) phase_end();
        tri_rows<OP, 3, 6>(pf, Pl);
        constexpr int FIRST = AHEAD && KT > 4 ? 2 : KT;      // of eight tiles of K's operands the registers hold two ahead of their use
        Frag<PT> cf[KT][2];
#pragma unroll
        for (int m = 0; m < FIRST; ++m) col_frags(cf[m], Kl, LDK, 16 * m);
        if (AHEAD) phase_end();
#pragma unroll
        for (int x = 0; x < 6; ++x) qs[tri_m(x)] = mma<OP, 3, OP>(pf[x], uf[tri_k(x)], qs[tri_m(x)]);
        row_operands(uf, vec + kKb * kC, ks);
        if (AHEAD) phase_end();
        // S = e^{G_C} S + K^T (kb U)
        const float dec = __expf((float)reinterpret_cast<const double*>(vec + kG64 * kC)[kC - 1]);
#pragma unroll
        for (int m = 0; m < KT; ++m) {
            if (m + FIRST < KT) col_frags(cf[m + FIRST], Kl, LDK, 16 * (m + FIRST));
            if (FIRST < KT) phase_end();
            S[m] *= dec;
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) S[m] = mma(cf[m][kb], uf[kb], S[m]);
        }
        // O leaves through this wave's own columns of the V tile, which it has read
        lds_order();
        T* my = Vl + wave * 16;
#pragma unroll
        for (int m = 0; m < 4; ++m) tile_write(my, LDV, 16 * m, 0, qs[m]);
        lds_order();
        store_rows(my, LDV, mycols, op + col0, ots, c * kC, w);
    }
    state_store(S, a.sT + state, a.dk, a.dv, col0);
    if (vcols > 0) zero_rows(op + sg * NW * 16, ots, vcols, w.len, a.T, tid, NT);
}

// ---- reverse scan ---------------------------------------------------------------------------------------
template <typename T, int DK, int NW> struct RscanLds {
    static constexpr int LDK = DK + 8, LDV = NW * 16 + 8;
    static constexpr size_t bytes = (size_t)kC * (2 * LDK + 2 * LDV) * sizeof(T) + (size_t)6 * kC * kLdm * 2 + kVec * kC * 4;
};

// What the gradients of q and k take of E and dV.  Of 16-bit types two parts of each (with E in one bf16 part dq and dk were off by 1.34 and 1.47 times
// their own rounding, with dV as it is written, in gv, dk by 1.1 times).  One word holds the upper 24 bits of E, which are its two parts, and the
// eight bits that follow dV's rounded mantissa, as a signed number: four bytes an element as for f32, and no third tensor (one more
// took the reverse scan from 217 to 230 us).
template <typename T> struct BehindT;
template <> struct BehindT<__hip_bfloat16> { static constexpr int SHIFT = 8; };       // f32 bits behind the type's mantissa: 16 and 13, eight of them kept
template <> struct BehindT<__half> { static constexpr int SHIFT = 5; };
template <typename T> __device__ __forceinline__ uint32_t pack_ev(float e, float v) {
    constexpr int S = BehindT<T>::SHIFT;
    T t;
    Elem<T>::st(&t, v);
    const int d = (int)(__float_as_uint(v) - __float_as_uint(to_f(t))) + (1 << (S - 1));
    return (__float_as_uint(e) & 0xFFFFFF00u) | ((uint32_t)max(min(d >> S, 127), -128) & 0xFFu);
}
// what dV's rounded value lacks, exactly (eight bits)
template <typename T> __device__ __forceinline__ float behind(float v, uint32_t word) {
    return __uint_as_float(__float_as_uint(v) + ((uint32_t)((int)(word << 24) >> 24) << BehindT<T>::SHIFT)) - v;
}

// E and O are formed again from the state at the chunk's start: 36 + 84 more matrix instructions a wave and chunk instead of 100 KB more
// traffic a chunk (E in f32 and the rest of O that its rounding dropped, written by the forward and read back).
// 223 to 232 us, 19 us a chunk (f32 at 30 heads, dk 40, dv 72, 301 frames: 76 us): 246 matrix instructions a wave and chunk keep the pipes busy 17 %
// of the time, 439 MB move.  Bound by latency at two waves a SIMD, which 256 registers a lane allow: without the next chunk's loads it took three
// quarters of the time (they find registers only at the chunk's end).
// Measured and not kept: those loads earlier (they spill), their lines touched into the L2 cache a chunk ahead (7 % more).
template <typename T, int DK, int NW>
__global__ __launch_bounds__(NW * 64) void gdr_rscan_kernel(GdrArgs a) {
    extern __shared__ __align__(16) char smem[];
    using L = RscanLds<T, DK, NW>;
    constexpr int NT = NW * 64, PT = Gd<T>::PT, LDK = L::LDK, LDV = L::LDV, KT = DK / 16;
    constexpr bool AHEAD = PT == 1;
    T* Kl = reinterpret_cast<T*>(smem);
    T* Ql = Kl + kC * LDK;
    T* Vl = Ql + kC * LDK;
    T* Ol = Vl + kC * LDV;                                  // dO
    __bf16* Xl = reinterpret_cast<__bf16*>(Ol + kC * LDV);
    __bf16* Pl = Xl + 3 * kC * kLdm;
    float* vec = reinterpret_cast<float*>(Pl + 3 * kC * kLdm);
    const int groups = (a.nsl + NW - 1) / NW;
    const int bh = blockIdx.x / groups, sg = blockIdx.x % groups, b = bh / a.H, h = bh % a.H, hk = h / a.r;
    const Walk w = walk_of(a, b, h);
    const int tid = threadIdx.x, l = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = l >> 4, i16 = l & 15;
    const int slice = sg * NW + wave, col0 = slice * 16;
    const int vcols = min(a.dv - sg * NW * 16, NW * 16), mycols = a.dv - col0;
    const int64_t state = (int64_t)bh * a.dk * a.dv, nat = (int64_t)a.B * a.H * a.nc;
    clear_upper(Xl, 6, tid, NT);
    f32x4 S[KT], s0n[KT];                                   // dS; the next chunk's starting state
#pragma unroll
    for (int m = 0; m < KT; ++m) S[m] = f32x4{0, 0, 0, 0};
    if (a.gsT) state_load(S, a.gsT + state, a.dk, a.dv, col0);
    const T* kp = (const T*)a.k + b * a.ks[1] + hk * a.ks[2];
    const T* qp = (const T*)a.q + b * a.qs[1] + hk * a.qs[2];
    const T* vp = (const T*)a.v + b * a.vs[1] + h * a.vs[2] + sg * NW * 16;
    const T* gp = (const T*)a.go + b * a.gos[1] + h * a.gos[2] + sg * NW * 16;
    const int64_t ots = (int64_t)a.B * a.H * a.dv;
    T* gvp = (T*)a.gv + ((int64_t)b * a.H + h) * a.dv;
    const int ncl = (w.len + kC - 1) / kC;
    TileRegs<T, DK, NT> rk, rq;
    TileRegs<T, NW * 16, NT> rv, ro;
    TriRegs<NT> rx, rp;
    float rvec[kVec * kC / NT];
    auto fetch = [&](int c) {
        const int64_t at = (int64_t)bh * a.nc + c;
        state_load(s0n, a.S0 + at * a.dk * a.dv, a.dk, a.dv, col0);
        rk.load(kp, a.ks[0], a.dk, c * kC, w);
        rq.load(qp, a.qs[0], a.dk, c * kC, w);
        rv.load(vp, a.vs[0], vcols, c * kC, w);
        ro.load(gp, a.gos[0], vcols, c * kC, w);
        rx.load(a.X + at * kTri);
        rp.load(a.P + at * kTri);
#pragma unroll
        for (int i = 0; i < kVec * kC / NT; ++i) rvec[i] = a.vec[at * kVec * kC + i * NT + tid];
    };
    if (ncl > 0) fetch(ncl - 1);
    for (int c = ncl - 1; c >= 0; --c) {
        const int64_t at = (int64_t)bh * a.nc + c;
        __syncthreads();
        rk.store(Kl, LDK, a.dk, c * kC, w.len);
        rq.store(Ql, LDK, a.dk, c * kC, w.len);
        rv.store(Vl, LDV, vcols, c * kC, w.len);
        ro.store(Ol, LDV, vcols, c * kC, w.len);
        rx.template store<3>(Xl);
        rp.template store<3>(Pl);
#pragma unroll
        for (int i = 0; i < kVec * kC / NT; ++i) vec[i * NT + tid] = rvec[i];
        f32x4 s0[KT];
#pragma unroll
        for (int m = 0; m < KT; ++m) s0[m] = s0n[m];
        __syncthreads();
        const float dec = __expf((float)reinterpret_cast<const double*>(vec + kG64 * kC)[kC - 1]);
        float anchor = 0.f;
        {   // dS at the chunk's end is what the gradient kernel needs; <dS, S_C> = dec <dS, S0> + sum_j dU2_j . U_j
            state_store(S, a.dS + at * a.dk * a.dv, a.dk, a.dv, col0);
            f32x4 p = {0, 0, 0, 0};
#pragma unroll
            for (int m = 0; m < KT; ++m) p += S[m] * s0[m];
            anchor = dec * ((p[0] + p[1]) + (p[2] + p[3]));
        }
        f32x4 E[4], O[4], z[4], xs[4];
#pragma unroll
        for (int m = 0; m < 4; ++m) { E[m] = f32x4{0, 0, 0, 0}; O[m] = E[m]; }
        Frag<PT> kf[2][4], qf[2][4];
        Frag<3> tf[6], pf[6], f[2];
        // six operands of a triangular matrix, each read two products ahead of its use; the last two steps read the next matrix's first two
        auto six = [&](auto&& read, auto&& use, auto&& next) {
            if (!AHEAD) { read(0); read(1); }
#pragma unroll
            for (int x = 0; x < 6; ++x) {
                if (x < 4) read(x + 2);
                else if (AHEAD) next(x - 4);
                phase_end();
                use(x);
                phase_end();
            }
        };
        auto x_rows = [&](int x) { tf[x] = plane_rows<3>(Xl, 16 * tri_m(x), 32 * tri_k(x)); };
        auto p_rows = [&](int x) { pf[x] = plane_rows<3>(Pl, 16 * tri_m(x), 32 * tri_k(x)); };
        auto x_cols = [&](int x) { tf[x] = plane_cols<3>(Xl, 32 * (1 - tri_k(x)), 16 * (3 - tri_m(x))); };
        auto p_cols = [&](int x) { pf[x] = plane_cols<3>(Pl, 32 * (1 - tri_k(x)), 16 * (3 - tri_m(x))); };
        row_frags(kf[0], Kl, LDK, 0);
        row_frags(qf[0], Ql, LDK, 0);
#pragma unroll
        for (int kb = 0; kb < DK / 32; ++kb) {
            if (kb + 1 < DK / 32) {
                row_frags(kf[(kb + 1) & 1], Kl, LDK, 32 * (kb + 1));
                row_frags(qf[(kb + 1) & 1], Ql, LDK, 32 * (kb + 1));
            } else if (AHEAD) {
                x_rows(0);
                x_rows(1);
            }
            const Frag<3> sb = split<3>(s0[2 * kb], s0[2 * kb + 1]);
            if (AHEAD) phase_end();
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                E[m] = mma(kf[kb & 1][m], sb, E[m]);
                O[m] = mma(qf[kb & 1][m], sb, O[m]);
            }
            phase_end();
        }
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            E[m] = tile_read(Vl, LDV, 16 * m, wave * 16) - vec4(vec + kAk * kC, 16 * m) * E[m];      // Vt
            O[m] *= vec4(vec + kAq * kC, 16 * m);
            xs[m] = f32x4{0, 0, 0, 0};
        }
        row_operands(f, vec + kBe * kC, E);
        six(x_rows, [&](int x) { xs[tri_m(x)] = mma(tf[x], f[tri_k(x)], xs[tri_m(x)]); }, p_rows);
#pragma unroll
        for (int m = 0; m < 4; ++m) E[m] -= xs[m];
        row_operands(f, vec + kBe * kC, E);                 // U
        six(p_rows, [&](int x) { O[tri_m(x)] = mma(pf[x], f[tri_k(x)], O[tri_m(x)]); },
            [&](int x) {      // K's four row tiles
                kf[0][2 * x] = row_frag(Kl, LDK, 32 * x, 0);
                kf[0][2 * x + 1] = row_frag(Kl, LDK, 32 * x + 16, 0);
            });
        if (!AHEAD) row_frags(kf[0], Kl, LDK, 0);
        f32x4 du[4];
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            z[m] = O[m] * tile_read(Ol, LDV, 16 * m, wave * 16);
            du[m] = f32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int kb = 0; kb < DK / 32; ++kb) {
            if (kb + 1 < DK / 32) row_frags(kf[(kb + 1) & 1], Kl, LDK, 32 * (kb + 1));
            else if (AHEAD) { p_cols(0); p_cols(1); }
            const Frag<3> db = split<3>(S[2 * kb], S[2 * kb + 1]);
            phase_end();
#pragma unroll
            for (int m = 0; m < 4; ++m) du[m] = mma(kf[kb & 1][m], db, du[m]);
            phase_end();
        }
        Frag<PT> of[2];
        col_frags(of, Ol, LDV, wave * 16);
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            du[m] *= vec4(vec + kKb * kC, 16 * m);
            const f32x4 p = du[m] * vec4(vec + kBe * kC, 16 * m) * E[m];
            anchor += (p[0] + p[1]) + (p[2] + p[3]);
        }
        six(p_cols, [&](int x) { du[3 - tri_m(x)] = mma(pf[x], of[1 - tri_k(x)], du[3 - tri_m(x)]); }, x_cols);      // + P^T dO
        row_operands(f, vec + kBe * kC, du);
#pragma unroll
        for (int m = 0; m < 4; ++m) xs[m] = f32x4{0, 0, 0, 0};
        // F = dU - X^T (beta dU), dV = beta F
        six(x_cols, [&](int x) { xs[3 - tri_m(x)] = mma(tf[x], f[1 - tri_k(x)], xs[3 - tri_m(x)]); }, [](int) {});
        f32x4 sb[4];
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            du[m] -= xs[m];
            sb[m] = E[m] * du[m];
            du[m] *= vec4(vec + kBe * kC, 16 * m);
            z[m] -= du[m] * tile_read(Vl, LDV, 16 * m, wave * 16);
#pragma unroll
            for (int e = 0; e < 4; ++e) { sb[m][e] = row16_sum(sb[m][e]); z[m][e] = row16_sum(z[m][e]); }
        }
        anchor = wave_sum(anchor);
        if (i16 == 0 && mycols > 0) {
            float* zo = a.zpart + (slice * nat + at) * kC + 4 * g;
            float* bo = a.bpart + (slice * nat + at) * kC + 4 * g;
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                *reinterpret_cast<f32x4a*>(bo + 16 * m) = sb[m];
                *reinterpret_cast<f32x4a*>(zo + 16 * m) = z[m];
            }
            if (g == 0) a.apart[slice * nat + at] = anchor;
        }
        // dS = dec dS + Q^T (aq dO) - K^T (ak dV)
        Frag<3> of3[2];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            f[kb] = split<3>(-vec4(vec + kAk * kC, 32 * kb) * du[2 * kb], -vec4(vec + kAk * kC, 32 * kb + 16) * du[2 * kb + 1]);
            of3[kb] = split<3>(vec4(vec + kAq * kC, 32 * kb) * tile_read(Ol, LDV, 32 * kb, wave * 16),
                               vec4(vec + kAq * kC, 32 * kb + 16) * tile_read(Ol, LDV, 32 * kb + 16, wave * 16));
        }
        // dV leaves through this wave's own columns of the V tile, which it has read; E (f32) through those of the dO tile
        lds_order();
        T* my = Vl + wave * 16;
#pragma unroll
        for (int m = 0; m < 4; ++m) tile_write(my, LDV, 16 * m, 0, du[m]);
        lds_order();
        store_rows(my, LDV, mycols, gvp + col0, ots, c * kC, w);
        float* eo = (float*)a.E + at * kC * a.dv;
        if constexpr (sizeof(T) == 4) {
            T* me = Ol + wave * 16;
#pragma unroll
            for (int m = 0; m < 4; ++m) tile_write(me, LDV, 16 * m, 0, E[m]);
            lds_order();
            store_rows(me, LDV, mycols, eo + col0, a.dv, 0, Walk{kC, false});
        } else {
#pragma unroll
            for (int m = 0; m < 4; ++m)
#pragma unroll
                for (int e = 0; e < 4; ++e) E[m][e] = __uint_as_float(pack_ev<T>(E[m][e], du[m][e]));
            state_store(E, eo, kC, a.dv, col0);
        }
        phase_end();
        if (c > 0) fetch(c - 1);      // here, not earlier: the tiles in flight take 57 registers a lane, which are free only now
        phase_end();
        Frag<PT> ck[2][2], cq[2][2];
        col_frags(ck[0], Kl, LDK, 0);
        col_frags(cq[0], Ql, LDK, 0);
#pragma unroll
        for (int m = 0; m < KT; ++m) {
            if (m + 1 < KT) {
                col_frags(ck[(m + 1) & 1], Kl, LDK, 16 * (m + 1));
                col_frags(cq[(m + 1) & 1], Ql, LDK, 16 * (m + 1));
            }
            S[m] *= dec;
            phase_end();
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) S[m] = mma(cq[m & 1][kb], of3[kb], mma(ck[m & 1][kb], f[kb], S[m]));
            phase_end();
        }
    }
    if (a.gs0) state_store(S, a.gs0 + state, a.dk, a.dv, col0);
    if (vcols > 0) zero_rows(gvp + sg * NW * 16, ots, vcols, w.len, a.T, tid, NT);
}

// ---- gradients of a chunk ---------------------------------------------------------------------------------
template <typename T, int DK> struct GradLds {
    static constexpr int LDK = DK + 8, LDV = sizeof(T) == 4 ? 132 : 136;
    static constexpr size_t values = (size_t)(sizeof(T) == 4 ? 3 : 5) * kC * LDV * sizeof(T);      // dO, dV, E; 16-bit types: dV's rest, two parts of E
    static constexpr size_t keys = (size_t)2 * kC * LDK * sizeof(T), mat = (size_t)Gd<T>::OP * kC * kLdm * 2, vecs = (kVec + 8) * kC * 4;
    static constexpr bool ROOM = values + keys + mat + vecs <= 160 * 1024;      // K, Q and the matrix stand beside the values, else in their place
    static constexpr size_t at_keys = ROOM ? values : 0, at_mat = at_keys + keys, at_vec = at_mat + mat > values ? at_mat + mat : values;
    static constexpr size_t bytes = at_vec + vecs;
};

template <int P> __device__ __forceinline__ void plane_write(__bf16* t, int r0, int c0, f32x4 v) {
    const int l = threadIdx.x & 63;
    short* p = reinterpret_cast<short*>(t) + (r0 + 4 * (l >> 4)) * kLdm + c0 + (l & 15);
    parts4<P>(v, [&](int i, u32x2a h) {
        short* o = p + i * kC * kLdm;
        o[0] = (short)h.x; o[kLdm] = (short)(h.x >> 16);
        o[2 * kLdm] = (short)h.y; o[3 * kLdm] = (short)(h.y >> 16);
    });
}
// the transpose of a tile: rows and columns exchanged
template <int P> __device__ __forceinline__ void plane_write_t(__bf16* t, int r0, int c0, f32x4 v) {
    const int l = threadIdx.x & 63;
    __bf16* p = t + (c0 + (l & 15)) * kLdm + r0 + 4 * (l >> 4);
    parts4<P>(v, [&](int i, u32x2a h) { *reinterpret_cast<u32x2a*>(p + i * kC * kLdm) = h; });
}

// words of pack_ev and dV's values on their way to LDS: three planes of bf16, E's upper and lower part and dV's rest
template <typename T>
__device__ __forceinline__ void store_ev(const TileRegs<T, 128, 512>& v, const TileRegs<float, 128, 512>& e, __hip_bfloat16* dst, int ld, int ncol) {
    const int tid = opaque(threadIdx.x);
#pragma unroll
    for (int n = 0; n < 2; ++n) {
        const int i = tid + n * 512, row = i / 16, c = i % 16 * 8;
        T t[8];
        __builtin_memcpy(t, &v.v[n][0], sizeof(t));
        f32x8 x, r;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const uint32_t word = e.v[n][k >> 2][k & 3];
            x[k] = __uint_as_float(word & 0xFFFFFF00u);
            r[k] = behind<T>(to_f(t[k]), word);
        }
        const Frag<2> f = split<2>(x);
        const bf16x8 planes[3] = {f.p[0], f.p[1], split<1>(r).p[0]};
#pragma unroll
        for (int p = 0; p < 3; ++p)
            *reinterpret_cast<u32x4a*>(dst + (p * kC + row) * ld + c) = c < ncol ? __builtin_bit_cast(u32x4a, planes[p]) : u32x4a{0, 0, 0, 0};
    }
}

// One workgroup a (key head, chunk), its value heads in turn: shared heads' gradients are sums in registers, in a fixed order.  Eight waves: a
// wave owns a quarter of dk in the products with the states and 16 columns j of the 64 x 64 products, and half of the rows of both.  219 to 226 us
// (one value head a key head; four: 160): 284 MB at 1.3 TB/s, bound by the waits between its phases.  Two parts of E and of dV take 128 KB of LDS, so one
// workgroup a CU; four waves a workgroup, two of them a CU, held one part of each: 173 us, dq off by 1.34 times its own rounding, dk by 1.47.
// Other shapes of the same size, eight waves against four: f32 dk 64 302 us / 363, dk 128 451 / 608, f16 dk 64 245 / 272, dk 128 337 / 415,
// bf16 dk 128 313 / 289 (one part).
template <typename T, int DK>
__global__ __launch_bounds__(512) void gdr_grads_kernel(GdrArgs a) {
    extern __shared__ __align__(16) char smem[];
    using L = GradLds<T, DK>;
    constexpr bool HALF = sizeof(T) == 2;
    using ET = std::conditional_t<HALF, __hip_bfloat16, float>;
    constexpr int PT = Gd<T>::PT, OP = Gd<T>::OP, PE = HALF ? 2 : 3, LDK = L::LDK, LDV = L::LDV, NT = DK / 64;
    constexpr int NTH = 512, AHEAD = 2;                                   // pieces of the states in flight or in use (3: 0 to 4 % slower, 5: 9 %)
    T *Ol = reinterpret_cast<T*>(smem), *Dl = Ol + kC * LDV;              // dO, dV
    ET *El = reinterpret_cast<ET*>(Dl + kC * LDV), *Rl = El + 2 * kC * LDV;      // E (16-bit types: two planes), dV's rest
    T *Kl = reinterpret_cast<T*>(smem + L::at_keys), *Ql = Kl + kC * LDK;
    __bf16* M = reinterpret_cast<__bf16*>(smem + L::at_mat);
    float* vec = reinterpret_cast<float*>(smem + L::at_vec);
    const double* G = reinterpret_cast<const double*>(vec + kG64 * kC);
    float* dots = vec + kVec * kC;                                        // [2][4][64]
    const int c = blockIdx.x % a.nc, bk = blockIdx.x / a.nc, b = bk / a.Hk, hk = bk % a.Hk;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wr = wave >> 2, wc = wave & 3;
    const Walk w = walk_of(a, b, hk * a.r);
    const int64_t kts = (int64_t)a.B * a.Hk * a.dk, gts = (int64_t)a.B * a.H;
    T* gqp = (T*)a.gq + ((int64_t)b * a.Hk + hk) * a.dk;
    T* gkp = (T*)a.gk + ((int64_t)b * a.Hk + hk) * a.dk;
    const int p0 = c * kC;
    // frames of this chunk behind the utterance's end: zero gradients
    const int z0 = max(p0, w.len), z1 = min(p0 + kC, a.T);
    if (z0 < z1) {
        zero_rows(gqp, kts, a.dk, z0, z1, tid, NTH);
        zero_rows(gkp, kts, a.dk, z0, z1, tid, NTH);
        for (int i = tid; i < (z1 - z0) * a.r; i += NTH) {
            const int64_t o = (int64_t)(z0 + i / a.r) * gts + (int64_t)b * a.H + hk * a.r + i % a.r;
            a.gg[o] = 0.f;
            a.gbeta[o] = 0.f;
        }
    }
    if (p0 >= w.len) return;
    f32x4 tq[2][NT], tk[2][NT];                               // rows 32 wr + 16 m + ..
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n) { tq[m][n] = f32x4{0, 0, 0, 0}; tk[m][n] = f32x4{0, 0, 0, 0}; }
    const int64_t ots = (int64_t)a.B * a.H * a.dv, nat = (int64_t)a.B * a.H * a.nc;
    const int r0 = 32 * wr;
    for (int hh = 0; hh < a.r; ++hh) {
        // the lane's number as the loop's own value: what follows from it (masks, addresses) is then formed where it is used, not kept in
        // registers, and out of them in scratch memory, across the loop
        const int l = opaque(tid & 63), g = l >> 4, i16 = l & 15;
        const int h = hk * a.r + hh, bh = b * a.H + h;
        const int64_t at = (int64_t)bh * a.nc + c;
        // the states' rows of one of this wave's tiles of dk: lane = row, 32 columns of dv from 32 kb on
        const float* s0 = a.S0 + at * a.dk * a.dv;
        const float* ds = a.dS + at * a.dk * a.dv;
        auto state_rows = [&](f32x4 (&v)[4], int n, int kb) {
            const int row = (wc * NT + n) * 16 + i16;
            const uint32_t rb = (uint32_t)(min(row, a.dk - 1) * a.dv) * 4u;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const uint32_t off = rb + (uint32_t)min(32 * kb + 16 * x + 4 * g, a.dv - 4) * 4u;
                v[x] = *reinterpret_cast<const f32x4a*>(reinterpret_cast<const char*>(s0) + off);
                v[2 + x] = *reinterpret_cast<const f32x4a*>(reinterpret_cast<const char*>(ds) + off);
            }
        };
        auto state_cut = [&](f32x4 (&v)[4], int n, int kb) {      // what lies outside is zero
            if ((wc * NT + n) * 16 + 16 <= a.dk && 32 * kb + 32 <= a.dv) return;
            const int row = (wc * NT + n) * 16 + i16;
#pragma unroll
            for (int x = 0; x < 4; ++x) v[x] = row < a.dk && 32 * kb + 16 * (x & 1) + 4 * g < a.dv ? v[x] : f32x4{0, 0, 0, 0};
        };
        // operands from rows of E (its parts) and of dV
        auto e_frag = [&](int row, int kb) {
            if constexpr (HALF) {
                Frag<2> f;
                f.p[0] = row_frag(El, LDV, row, 32 * kb).p[0];
                f.p[1] = row_frag(El + kC * LDV, LDV, row, 32 * kb).p[0];
                return f;
            } else return row_frag(El, LDV, row, 32 * kb);
        };
        f32x4 sr[AHEAD][4];
        TileRegs<T, DK, NTH> rk, rq;
        auto load_keys = [&] {
            rk.load((const T*)a.k + b * a.ks[1] + hk * a.ks[2], a.ks[0], a.dk, p0, w);
            rq.load((const T*)a.q + b * a.qs[1] + hk * a.qs[2], a.qs[0], a.dk, p0, w);
        };
        auto store_keys = [&] {
            rk.store(Kl, LDK, a.dk, c * kC, w.len);
            rq.store(Ql, LDK, a.dk, c * kC, w.len);
        };
        __syncthreads();
        {
            TileRegs<T, 128, NTH> ro, rd;
            TileRegs<float, 128, NTH> re;
            const Walk rows = {kC, false};
            ro.load((const T*)a.go + b * a.gos[1] + h * a.gos[2], a.gos[0], a.dv, p0, w);
            rd.load((const T*)a.gv + (int64_t)bh * a.dv, ots, a.dv, p0, w);
            re.load((const float*)a.E + at * kC * a.dv, a.dv, a.dv, 0, rows);
            if (L::ROOM) load_keys();
            // a loop over i = tid, tid + 512, ... would end lane by lane, and at such an exit the compiler has put a copy of a register that
            // lives on (to an accumulation register, where 256 do not suffice) in front of the instruction that turns the lanes on again:
            // the copy wrote nothing.  No loop in this kernel ends lane by lane while the tiles are live.
            static_assert(kVec * kC == NTH, "one entry a thread");
            vec[tid] = a.vec[at * kVec * kC + tid];
#pragma unroll
            for (int i = 0; i + 1 < AHEAD; ++i) state_rows(sr[i], i / 4, i % 4);
            phase_end();
            ro.store(Ol, LDV, a.dv, p0, w.len);
            rd.store(Dl, LDV, a.dv, p0, w.len);
            if constexpr (HALF) store_ev<T>(rd, re, El, LDV, a.dv);
            else re.store(El, LDV, a.dv, 0, kC);
            if (L::ROOM) store_keys();
            phase_end();
        }
        __syncthreads();
        // states: wave = a quarter of dk; U = beta E: its factor goes with the rows
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            f32x4 cq[2], ck[2], cd[2];
#pragma unroll
            for (int m = 0; m < 2; ++m) { cq[m] = f32x4{0, 0, 0, 0}; ck[m] = cq[m]; cd[m] = cq[m]; }
#pragma unroll
            for (int kb = 0; kb < 4; ++kb) {
                const int nx = 4 * n + kb + AHEAD - 1;
                if (nx < 4 * NT) state_rows(sr[nx % AHEAD], nx / 4, nx % 4);
                f32x4 (&cur)[4] = sr[(4 * n + kb) % AHEAD];
                if (kb * 32 < a.dv) {
                    state_cut(cur, n, kb);
                    const Frag<OP> sf = split<OP>(cur[0], cur[1]), df = split<OP>(cur[2], cur[3]);
                    Frag<PT> of[2], vf[2];
                    Frag<PE> uf[2];
                    Frag<1> lf[2], s1;
                    s1.p[0] = sf.p[0];
#pragma unroll
                    for (int m = 0; m < 2; ++m) {
                        of[m] = row_frag(Ol, LDV, r0 + 16 * m, 32 * kb);
                        vf[m] = row_frag(Dl, LDV, r0 + 16 * m, 32 * kb);
                        uf[m] = e_frag(r0 + 16 * m, kb);
                        if constexpr (HALF) lf[m] = row_frag(Rl, LDV, r0 + 16 * m, 32 * kb);
                    }
                    if (PT == 1) phase_end();
#pragma unroll
                    for (int m = 0; m < 2; ++m) {
                        cq[m] = mma<PT, OP, OP>(of[m], sf, cq[m]);
                        ck[m] = mma<PE, OP, OP>(uf[m], df, ck[m]);
                        cd[m] = mma<PT, OP, OP>(vf[m], sf, cd[m]);
                        if constexpr (HALF) cd[m] = mma(lf[m], s1, cd[m]);
                    }
                }
                phase_end();
            }
            phase_end();
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                const f32x4 aq = vec4(vec + kAq * kC, r0 + 16 * m), ak = vec4(vec + kAk * kC, r0 + 16 * m);
                const f32x4 kb = vec4(vec + kKb * kC, r0 + 16 * m) * vec4(vec + kBe * kC, r0 + 16 * m);
                tq[m][n] += aq * cq[m];
                tk[m][n] += kb * ck[m] - ak * cd[m];
            }
        }
        // M1 = dP * D * sq_i * rk_j (lower), M2 = -dV U^T * D * rk_i * rk_j (strictly lower, made symmetric); wc = block column j
        f32x4 dp[2], dn[2];
#pragma unroll
        for (int m = 0; m < 2; ++m) { dp[m] = f32x4{0, 0, 0, 0}; dn[m] = dp[m]; }
#pragma unroll
        for (int kb = 0; kb < 4; ++kb) {
            if (kb * 32 < a.dv) {
                const Frag<PE> uf = e_frag(16 * wc, kb);
                Frag<PT> of[2], vf[2];
                Frag<1> lf[2], u1;
                u1.p[0] = uf.p[0];
#pragma unroll
                for (int m = 0; m < 2; ++m) {
                    of[m] = row_frag(Ol, LDV, r0 + 16 * m, 32 * kb);
                    vf[m] = row_frag(Dl, LDV, r0 + 16 * m, 32 * kb);
                    if constexpr (HALF) lf[m] = row_frag(Rl, LDV, r0 + 16 * m, 32 * kb);
                }
                if (PT == 1) phase_end();
#pragma unroll
                for (int m = 0; m < 2; ++m) {
                    dp[m] = mma<PT, PE, OP>(of[m], uf, dp[m]);
                    dn[m] = mma<PT, PE, OP>(vf[m], uf, dn[m]);
                    if constexpr (HALF) dn[m] = mma(lf[m], u1, dn[m]);
                }
            }
            phase_end();
        }
        if (!L::ROOM) load_keys();
        float part[8], anchor;                                // the slices' partial sums, all at once: a loop over them waited for each
        {
            const float* parts = wave == 0 ? a.zpart : a.bpart;      // the other waves load along
#pragma unroll
            for (int s = 0; s < 8; ++s) part[s] = parts[(min(s, a.nsl - 1) * nat + at) * kC + l];
            anchor = a.apart[min(l & 7, a.nsl - 1) * nat + at];
        }
        phase_end();
        if (!L::ROOM) __syncthreads();                        // the matrix takes the values' place
        {
            const int j = 16 * wc + i16;
            const float rkj = vec[kRk * kC + j] * vec[kBe * kC + j];
            const double gj = G[j];
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                const f32x4 sqi = vec4(vec + kSq * kC, r0 + 16 * m), rki = vec4(vec + kRk * kC, r0 + 16 * m);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int i = r0 + 16 * m + 4 * g + e;
                    const float d = __expf((float)(G[i] - gj)) * rkj;      // above the diagonal it may be infinite: selected away
                    const float p = dp[m][e] * d * sqi[e], n = -dn[m][e] * d * rki[e];
                    dp[m][e] = i >= j ? p : 0.f;
                    dn[m][e] = i > j ? n : 0.f;
                }
                plane_write<OP>(M, r0 + 16 * m, 16 * wc, dp[m]);
                phase_end();
            }
        }
        if (!L::ROOM) store_keys();
        if (wave == 0) {      // dg: lane = frame
            float z = 0.f;
#pragma unroll
            for (int s = 0; s < 8; ++s) z += s < a.nsl ? part[s] : 0.f;
            float an = (l & 7) < a.nsl ? anchor : 0.f;
            an += __shfl_xor(an, 1);
            an += __shfl_xor(an, 2);
            an += __shfl_xor(an, 4);
            if (p0 + l >= w.len) z = 0.f;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) { const float u = __shfl_down(z, o); if (l + o < 64) z += u; }
            if (p0 + l < w.len) {
                const int64_t o = w.frame(p0 + l) * gts + bh;
                a.gg[o] = a.fresh && p0 + l == 0 ? 0.f : z + an;
            }
        }
        if (wave == 1) {      // dbeta
            float be = 0.f;
#pragma unroll
            for (int s = 0; s < 8; ++s) be += s < a.nsl ? part[s] : 0.f;
            if (p0 + l < w.len) a.gbeta[w.frame(p0 + l) * gts + bh] = be;
        }
        __syncthreads();
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const int n0 = (wc * NT + n) * 16;
                const auto kf = col_frag(Kl, LDK, 32 * kb, n0);
                const auto qf = col_frag(Ql, LDK, 32 * kb, n0);
#pragma unroll
                for (int m = 0; m < 2; ++m) {
                    if (kb <= wr) tq[m][n] = mma<OP, PT, OP>(plane_rows<OP>(M, r0 + 16 * m, 32 * kb), kf, tq[m][n]);
                    if (kb >= wr) tk[m][n] = mma<OP, PT, OP>(plane_cols<OP>(M, 32 * kb, r0 + 16 * m), qf, tk[m][n]);
                }
                phase_end();
            }
        __syncthreads();
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            const int bi = 2 * wr + m;
            if (bi < wc) continue;
            if (bi > wc) plane_write<OP>(M, 16 * bi, 16 * wc, dn[m]);
            else {      // the diagonal block: its upper half is the transpose of its lower half
                f32x4 t = dn[m];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    // entry (i, j) of the upper half = lower entry (j, i): lane (j / 4 group, i), element j % 4
                    const int i = 4 * g + e;
                    float up = 0.f;
#pragma unroll
                    for (int x = 0; x < 4; ++x) { const float v = __shfl(dn[m][x], (i16 >> 2) * 16 + i); if ((i16 & 3) == x) up = v; }
                    if (i < i16) t[e] = up;
                }
                plane_write<OP>(M, 16 * bi, 16 * wc, t);
            }
            if (bi > wc) plane_write_t<OP>(M, 16 * bi, 16 * wc, dn[m]);
        }
        __syncthreads();
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const auto kf = col_frag(Kl, LDK, 32 * kb, (wc * NT + n) * 16);
#pragma unroll
                for (int m = 0; m < 2; ++m) tk[m][n] = mma<OP, PT, OP>(plane_rows<OP>(M, r0 + 16 * m, 32 * kb), kf, tk[m][n]);
                phase_end();
            }
    }
    const int l = tid & 63, g = l >> 4, i16 = l & 15;
    // through the normalisation: dq = tq - q |q|^-2 (q . tq)  (|.|^2 with its epsilon), dk alike
    if (a.norm) {
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            f32x4 sq = {0, 0, 0, 0}, sk = {0, 0, 0, 0};
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const int n0 = (wc * NT + n) * 16;
                sq += tq[m][n] * tile_read(Ql, LDK, r0 + 16 * m, n0);
                sk += tk[m][n] * tile_read(Kl, LDK, r0 + 16 * m, n0);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) { sq[e] = row16_sum(sq[e]); sk[e] = row16_sum(sk[e]); }
            if (i16 == 0) {
                *reinterpret_cast<f32x4a*>(dots + wc * kC + r0 + 16 * m + 4 * g) = sq;
                *reinterpret_cast<f32x4a*>(dots + (4 + wc) * kC + r0 + 16 * m + 4 * g) = sk;
            }
        }
        __syncthreads();
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            f32x4 sq = {0, 0, 0, 0}, sk = {0, 0, 0, 0};
#pragma unroll
            for (int x = 0; x < 4; ++x) { sq += vec4(dots + x * kC, r0 + 16 * m); sk += vec4(dots + (4 + x) * kC, r0 + 16 * m); }
            const f32x4 rk = vec4(vec + kRk * kC, r0 + 16 * m), rq = vec4(vec + kSq * kC, r0 + 16 * m) * (1.f / a.scale);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const int n0 = (wc * NT + n) * 16;
                tq[m][n] -= sq * rq * rq * tile_read(Ql, LDK, r0 + 16 * m, n0);
                tk[m][n] -= sk * rk * rk * tile_read(Kl, LDK, r0 + 16 * m, n0);
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            tile_write(Ql, LDK, r0 + 16 * m, (wc * NT + n) * 16, tq[m][n]);
            tile_write(Kl, LDK, r0 + 16 * m, (wc * NT + n) * 16, tk[m][n]);
        }
    __syncthreads();
    constexpr int VE = 16 / sizeof(T);
    const int vpr = a.dk / VE;
    for (int i = tid; i < kC * vpr; i += NTH) {
        const int row = i / vpr, col = (i % vpr) * VE, p = p0 + row;
        if (p >= w.len) continue;
        const int64_t t = w.frame(p);
        *reinterpret_cast<u32x4a*>(gqp + t * kts + col) = *reinterpret_cast<const u32x4a*>(Ql + row * LDK + col);
        *reinterpret_cast<u32x4a*>(gkp + t * kts + col) = *reinterpret_cast<const u32x4a*>(Kl + row * LDK + col);
    }
}

// ---- recurrent form -------------------------------------------------------------------------------------
// One frame of 512 heads of 128 x 128: 14.6 us, 67 MB of state read and written at 4.6 TB/s, HBM-bound.  One frame of 8 heads: 4.9 us, of
// which an empty launch is 3.5; each further frame 0.95 us, one reduction over LDS.
// Few frames: a workgroup owns 32 columns of one head's state, in registers: 8 lanes x 4 columns a row, 32 row groups of four rows.  All
// frames' keys, queries, values and gates are brought to LDS first (a frame's global loads inside the loop cost 1.7 us a frame), with the
// three products of k and q that do not need the state.  One reduction a frame then: k.S and q.S come from the state before the frame, and
// o follows from u.
__device__ __forceinline__ float add_lanes_8_16_32(float v) {       // sum over the eight lanes that agree in their number mod 8
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x128, 0xf, 0xf, false));
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

template <typename T, int NF>      // NF: frames that LDS holds (1 or kRecurrentMax)
__global__ __launch_bounds__(256) void gdr_recurrent_kernel(GdrArgs a) {
    __shared__ __align__(16) float kq[2][NF][128];
    __shared__ __align__(16) float vs[NF][32];
    __shared__ __align__(16) float sc[NF][8];          // decay, beta, 1 / |k|, scale / |q|, qh.kh
    __shared__ __align__(16) float red[2][4][8][8];
    const int ns = (a.dv + 31) >> 5, bh = blockIdx.x / ns, sl = blockIdx.x % ns, b = bh / a.H, h = bh % a.H, hk = h / a.r;
    const Walk w = walk_of(a, b, h);
    const int tid = threadIdx.x, wave = tid >> 6, cl = tid & 7, rg = tid >> 3;
    const int col = sl * 32 + cl * 4, row0 = rg * 4;
    const bool con = col < a.dv && row0 < a.dk;
    const int64_t state = (int64_t)bh * a.dk * a.dv + (int64_t)row0 * a.dv + col;
    f32x4 S[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        S[i] = f32x4{0, 0, 0, 0};
        if (a.s0 && con) S[i] = *reinterpret_cast<const f32x4a*>(a.s0 + state + (int64_t)i * a.dv);
    }
    const T* kp = (const T*)a.k + b * a.ks[1] + hk * a.ks[2];
    const T* qp = (const T*)a.q + b * a.qs[1] + hk * a.qs[2];
    const T* vp = (const T*)a.v + b * a.vs[1] + h * a.vs[2];
    for (int i = tid; i < w.len * 128; i += 256) {
        const int p = i >> 7, c = i & 127;
        const int64_t t = w.frame(p);
        kq[0][p][c] = c < a.dk ? Elem<T>::ld(kp + t * a.ks[0] + c) : 0.f;
        kq[1][p][c] = c < a.dk ? Elem<T>::ld(qp + t * a.qs[0] + c) : 0.f;
    }
    for (int i = tid; i < w.len * 32; i += 256) {
        const int p = i >> 5, c = i & 31;
        vs[p][c] = sl * 32 + c < a.dv ? Elem<T>::ld(vp + w.frame(p) * a.vs[0] + sl * 32 + c) : 0.f;
    }
    __syncthreads();
    for (int p = wave; p < w.len; p += 4) {             // a wave a frame: two entries a lane
        const int l = tid & 63;
        const float k0 = kq[0][p][l], k1 = kq[0][p][64 + l], q0 = kq[1][p][l], q1 = kq[1][p][64 + l];
        const float kk = wave_sum(k0 * k0 + k1 * k1), qq = wave_sum(q0 * q0 + q1 * q1), qk = wave_sum(q0 * k0 + q1 * k1);
        if (l == 0) {
            const int64_t t = w.frame(p);
            const float rk = a.norm ? 1.f / sqrtf(kk + 1e-6f) : 1.f, sq = (a.norm ? 1.f / sqrtf(qq + 1e-6f) : 1.f) * a.scale;
            sc[p][0] = __expf(a.g[t * a.gs[0] + b * a.gs[1] + h * a.gs[2]]);
            sc[p][1] = a.beta[t * a.bs[0] + b * a.bs[1] + h * a.bs[2]];
            sc[p][2] = rk;
            sc[p][3] = sq;
            sc[p][4] = sq * rk * qk;
        }
    }
    __syncthreads();
    T* op = (T*)a.o + ((int64_t)b * a.H + h) * a.dv + col;
    const int64_t ots = (int64_t)a.B * a.H * a.dv;
    const bool writes = rg == 0 && col < a.dv;
    for (int p = 0; p < w.len; ++p) {
        const f32x4 k = *reinterpret_cast<const f32x4a*>(&kq[0][p][row0]), q = *reinterpret_cast<const f32x4a*>(&kq[1][p][row0]);
        const f32x4 v = *reinterpret_cast<const f32x4a*>(&vs[p][cl * 4]), c4 = *reinterpret_cast<const f32x4a*>(&sc[p][0]);
        const float dec = c4[0], be = c4[1], rk = c4[2], sq = c4[3], qk = sc[p][4];
        f32x4 ks = {0, 0, 0, 0}, qs = ks;
#pragma unroll
        for (int i = 0; i < 4; ++i) { ks += k[i] * S[i]; qs += q[i] * S[i]; }
#pragma unroll
        for (int j = 0; j < 4; ++j) { ks[j] = add_lanes_8_16_32(ks[j]); qs[j] = add_lanes_8_16_32(qs[j]); }
        float(*rd)[8][8] = red[p & 1];
        if ((tid & 63) < 8) {
            *reinterpret_cast<f32x4a*>(&rd[wave][cl][0]) = ks;
            *reinterpret_cast<f32x4a*>(&rd[wave][cl][4]) = qs;
        }
        __syncthreads();
        ks = f32x4{0, 0, 0, 0};
        qs = ks;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            ks += *reinterpret_cast<const f32x4a*>(&rd[x][cl][0]);
            qs += *reinterpret_cast<const f32x4a*>(&rd[x][cl][4]);
        }
        const f32x4 u = be * (v - (dec * rk) * ks);
#pragma unroll
        for (int i = 0; i < 4; ++i) S[i] = dec * S[i] + (rk * k[i]) * u;
        if (writes) {
            const f32x4 o = (sq * dec) * qs + qk * u;
#pragma unroll
            for (int j = 0; j < 4; ++j) Elem<T>::st(op + w.frame(p) * ots + j, o[j]);
        }
    }
    if (writes) {
        for (int t = w.len; t < a.T; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) Elem<T>::st(op + t * ots + j, 0.f);
    }
    if (con) {
#pragma unroll
        for (int i = 0; i < 4; ++i) *reinterpret_cast<f32x4a*>(a.sT + state + (int64_t)i * a.dv) = S[i];
    }
}

// ---- host -----------------------------------------------------------------------------------------------
static int gdr_check(const char* who, int T, int B, int Hk, int H, int dk, int dv, int flags, int dtype) {
    SP_CHECK_ARG(T >= 0 && T < (1 << 24) && B >= 0 && Hk >= 1 && H >= 1 && H % Hk == 0, "%s: bad shape T=%d B=%d Hk=%d H=%d (H a multiple of Hk)", who, T, B, Hk, H);
    SP_CHECK_ARG(dk >= 8 && dk <= 128 && dk % 8 == 0 && dv >= 8 && dv <= 128 && dv % 8 == 0, "%s: dk=%d and dv=%d must be multiples of 8 in [8, 128]", who, dk, dv);
    SP_CHECK_ARG((flags & ~(SP_GDR_NORMALIZE | SP_GDR_BIDIRECTIONAL)) == 0, "%s: unknown flags %d", who, flags);
    SP_CHECK_ARG(!(flags & SP_GDR_BIDIRECTIONAL) || Hk % 2 == 0, "%s: both directions need an even number of key heads, not %d", who, Hk);
    SP_CHECK_ARG(dtype == SP_F32 || dtype == SP_BF16 || dtype == SP_F16, "%s: dtype %d not supported (f32, bf16, f16)", who, dtype);
    SP_CHECK_ARG((int64_t)B * H * 128 <= (1ll << 23), "%s: B=%d x H=%d exceed 65536", who, B, H);
    SP_CHECK_ARG((int64_t)B * H * ((T + kC - 1) / kC + 4) < (1ll << 22), "%s: B=%d x H=%d x %d frames exceed the grid", who, B, H, T);
    return SP_OK;
}

struct GdrLayout { size_t vec, X, P, S0, end; };
static GdrLayout gdr_saved(int T, int B, int H, int dk, int dv, bool train) {
    GdrLayout s{};
    const size_t n = (size_t)B * H * ((T + kC - 1) / kC);
    size_t o = 0;
    auto put = [&](size_t bytes) { const size_t at = o; o = align_up(o + bytes, 256); return at; };
    s.vec = put(n * kVec * kC * 4);
    s.X = put(n * kTri * 4);
    s.P = put(n * kTri * 4);
    if (train) s.S0 = put(n * dk * dv * 4);
    s.end = o;
    return s;
}
struct GdrBwdLayout { size_t dS, E, z, b, a, end; };
static GdrBwdLayout gdr_bwd_ws(int T, int B, int H, int dk, int dv) {
    GdrBwdLayout s{};
    const size_t n = (size_t)B * H * ((T + kC - 1) / kC), nsl = (dv + 15) / 16;
    size_t o = 0;
    auto put = [&](size_t bytes) { const size_t at = o; o = align_up(o + bytes, 256); return at; };
    s.dS = put(n * dk * dv * 4);
    s.E = put(n * kC * dv * 4);
    s.z = put(n * nsl * kC * 4);
    s.b = put(n * nsl * kC * 4);
    s.a = put(n * nsl * 4);
    s.end = o;
    return s;
}

static bool gdr_aligned(const void* p, const int64_t* st, int dtype) {
    const int64_t ve = dtype == SP_F32 ? 4 : 8;
    if (st[0] < 0 || st[0] * 4 > (1ll << 25)) return false;
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && st[0] % ve == 0 && st[1] % ve == 0 && st[2] % ve == 0;
}

// every address that the kernels read or write 16 bytes at a time
static bool gdr_at16(std::initializer_list<const void*> ps) {
    for (const void* p : ps) if (reinterpret_cast<uintptr_t>(p) % 16) return false;
    return true;
}

template <typename K> static int gdr_launch(K kernel, size_t lds, int64_t blocks, int threads, const GdrArgs& a, hipStream_t s, const char* what) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(threads), lds, s, a);
    return check_launch(what);
}

// Columns of dv a workgroup of the scans owns: 128 in eight waves (a head's K, Q and matrices are then staged once), or 64 in four where the
// eight would leave CUs idle that the four fill: up to 128 heads.  T = 751, dv 128, both directions, wide against narrow in us, forward (prep
// and scan) and backward (reverse scan and gradients):
//   heads          128                  136                  256
//   bf16 dk 64     147/139  338/299     153/194  374/435     171/215  476/536
//   f16 dk 64      180/157  398/353     183/228  420/530     205/252  538/643
//   f32 dk 64      210/183  -           215/274  -           268/315  -
//   bf16 dk 128    182/170  -           188/242  -           225/282  -
//   f16 dk 128     248/213  -           254/323  -           296/367  -
// Eight waves have 256 registers each.  Where the tiles do not fit those, the narrow form is the faster one at 256 heads as well: the
// reverse scan of dk 128 (bf16 400 us against 358, f16 700 against 525) and of f32 (dk 64: 488 against 420; dk 128 exceeds the LDS), the
// scan of f32 at dk 128 (373 against 358).
static bool gdr_wide(const GdrArgs& a) { return a.nsl > 4 && (int64_t)a.B * a.H > 128; }

static void gdr_fill(GdrArgs& a, const void* q, const void* k, const void* v, const float* g, const float* beta, const int32_t* lengths,
                     const int64_t* st, int T, int B, int Hk, int H, int dk, int dv, float scale, int flags) {
    a.q = q; a.k = k; a.v = v; a.g = g; a.beta = beta; a.lengths = lengths;
    for (int i = 0; i < 3; ++i) { a.qs[i] = st[i]; a.ks[i] = st[3 + i]; a.vs[i] = st[6 + i]; a.gs[i] = st[9 + i]; a.bs[i] = st[12 + i]; }
    a.T = T; a.B = B; a.Hk = Hk; a.H = H; a.r = H / Hk; a.dk = dk; a.dv = dv;
    a.nc = (T + kC - 1) / kC; a.nsl = (dv + 15) / 16;
    a.scale = scale;
    a.norm = flags & SP_GDR_NORMALIZE ? 1 : 0;
    a.bidir = flags & SP_GDR_BIDIRECTIONAL ? 1 : 0;
    a.fresh = flags & SP_GDR_NO_STATE ? 1 : 0;
}

template <typename T, int DK, int NW, bool TRAIN> static int gdr_scan(const GdrArgs& a, hipStream_t s) {
    return gdr_launch(gdr_scan_kernel<T, DK, NW, TRAIN>, ScanLds<T, DK, NW>::bytes, (int64_t)a.B * a.H * ((a.nsl + NW - 1) / NW), NW * 64, a, s,
                      "gdr_scan_kernel");
}
template <typename T, int DK, bool TRAIN> static int gdr_forward(const GdrArgs& a, hipStream_t s) {
    const int rc = gdr_launch(gdr_prep_kernel<T, DK>, PrepLds<T, DK>::bytes, (int64_t)a.B * a.H * a.nc, 256, a, s, "gdr_prep_kernel");
    if (rc) return rc;
    if constexpr (sizeof(T) == 2 || DK == 64)
        if (gdr_wide(a)) return gdr_scan<T, DK, 8, TRAIN>(a, s);
    return gdr_scan<T, DK, 4, TRAIN>(a, s);
}
template <typename T, int DK, int NW> static int gdr_rscan(const GdrArgs& a, hipStream_t s) {
    return gdr_launch(gdr_rscan_kernel<T, DK, NW>, RscanLds<T, DK, NW>::bytes, (int64_t)a.B * a.H * ((a.nsl + NW - 1) / NW), NW * 64, a, s,
                      "gdr_rscan_kernel");
}
template <typename T, int DK> static int gdr_backward(const GdrArgs& a, hipStream_t s) {
    const auto walk = [&] {
        if constexpr (sizeof(T) == 2 && DK == 64)
            if (gdr_wide(a)) return gdr_rscan<T, DK, 8>(a, s);
        return gdr_rscan<T, DK, 4>(a, s);
    };
    if (const int rc = walk()) return rc;
    return gdr_launch(gdr_grads_kernel<T, DK>, GradLds<T, DK>::bytes, (int64_t)a.B * a.Hk * a.nc, 512, a, s, "gdr_grads_kernel");
}

}  // namespace sp

using namespace sp;

extern "C" size_t sp_gdr_workspace_bytes(int T, int B, int Hk, int H, int dk, int dv, int dtype, int backward) {
    if (gdr_check("sp_gdr_workspace_bytes", T, B, Hk, H, dk, dv, 0, dtype)) return 0;
    return backward ? gdr_bwd_ws(T, B, H, dk, dv).end : gdr_saved(T, B, H, dk, dv, false).end;
}
extern "C" size_t sp_gdr_saved_bytes(int T, int B, int Hk, int H, int dk, int dv, int dtype) {
    if (gdr_check("sp_gdr_saved_bytes", T, B, Hk, H, dk, dv, 0, dtype)) return 0;
    return gdr_saved(T, B, H, dk, dv, true).end;
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
    SP_CHECK_ARG(gdr_at16({state, state_out, o, saved, workspace}), "sp_gdr_fwd: state, state_out, o, saved and workspace must be 16-byte aligned");
    GdrArgs a{};
    gdr_fill(a, q, k, v, g, beta, lengths, strides, T, B, Hk, H, dk, dv, scale, flags);
    a.s0 = state; a.sT = state_out; a.o = o;
    hipStream_t s = (hipStream_t)stream;
    const bool train = saved != nullptr;
    if (T == 0 || (!train && T <= kRecurrentMax)) {       // T = 0: the state is copied, and nothing to save
        const int64_t blocks = (int64_t)B * H * ((dv + 31) / 32);
#define SP_GDR_REC(T_) return T == 1 ? gdr_launch(gdr_recurrent_kernel<T_, 1>, 0, blocks, 256, a, s, "gdr_recurrent_kernel") \
                                     : gdr_launch(gdr_recurrent_kernel<T_, kRecurrentMax>, 0, blocks, 256, a, s, "gdr_recurrent_kernel")
        if (dtype == SP_F32) SP_GDR_REC(float);
        if (dtype == SP_F16) SP_GDR_REC(__half);
        SP_GDR_REC(__hip_bfloat16);
#undef SP_GDR_REC
    }
    SP_CHECK_ARG(gdr_aligned(q, strides, dtype) && gdr_aligned(k, strides + 3, dtype) && gdr_aligned(v, strides + 6, dtype),
                 "sp_gdr_fwd: q, k, v need 16-byte aligned rows and at most 2^23 elements from frame to frame");
    const GdrLayout lay = gdr_saved(T, B, H, dk, dv, train);
    if (train ? saved_bytes < lay.end : workspace_bytes < lay.end || !workspace)
        return fail(SP_EWORKSPACE, "sp_gdr_fwd: %s %zu < %zu bytes", train ? "saved" : "workspace", train ? saved_bytes : workspace_bytes, lay.end);
    char* base = (char*)(train ? saved : workspace);
    a.vec = (float*)(base + lay.vec); a.X = (float*)(base + lay.X); a.P = (float*)(base + lay.P); a.S0 = (float*)(base + lay.S0);
    const bool wide = dk > 64;
#define SP_GDR_FWD(T_, TR_) return wide ? gdr_forward<T_, 128, TR_>(a, s) : gdr_forward<T_, 64, TR_>(a, s)
    if (train) {
        if (dtype == SP_F32) SP_GDR_FWD(float, true);
        if (dtype == SP_F16) SP_GDR_FWD(__half, true);
        SP_GDR_FWD(__hip_bfloat16, true);
    }
    if (dtype == SP_F32) SP_GDR_FWD(float, false);
    if (dtype == SP_F16) SP_GDR_FWD(__half, false);
    SP_GDR_FWD(__hip_bfloat16, false);
#undef SP_GDR_FWD
}

extern "C" int sp_gdr_bwd(const void* q, const void* k, const void* v, const float* g, const float* beta, const int32_t* lengths,
                          const int64_t* strides, int T, int B, int Hk, int H, int dk, int dv, float scale, int flags, int dtype,
                          const void* /* o */, const void* saved, size_t saved_bytes, const void* go, const float* gstate_out, void* gq, void* gk,
                          void* gv, float* gg, float* gbeta, float* gstate, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = gdr_check("sp_gdr_bwd", T, B, Hk, H, dk, dv, flags & ~SP_GDR_NO_STATE, dtype);
    if (rc) return rc;
    if (B == 0) return SP_OK;
    SP_CHECK_ARG(scale != 0.f, "sp_gdr_bwd: scale is zero");
    SP_CHECK_ARG(T > 0, "sp_gdr_bwd: T=0 has nothing to differentiate");
    SP_CHECK_ARG(q && k && v && g && beta && strides && saved && go && gq && gk && gv && gg && gbeta && workspace, "sp_gdr_bwd: null pointer");
    SP_CHECK_ARG(gdr_aligned(q, strides, dtype) && gdr_aligned(k, strides + 3, dtype) && gdr_aligned(v, strides + 6, dtype) &&
                     gdr_aligned(go, strides + 15, dtype), "sp_gdr_bwd: q, k, v, go need 16-byte aligned rows and at most 2^23 elements from frame to frame");
    SP_CHECK_ARG(gdr_at16({saved, gq, gk, gv, workspace}), "sp_gdr_bwd: saved, gq, gk, gv and workspace must be 16-byte aligned");
    const GdrLayout lay = gdr_saved(T, B, H, dk, dv, true);
    const GdrBwdLayout ws = gdr_bwd_ws(T, B, H, dk, dv);
    if (saved_bytes < lay.end || workspace_bytes < ws.end)
        return fail(SP_EWORKSPACE, "sp_gdr_bwd: saved %zu < %zu or workspace %zu < %zu bytes", saved_bytes, lay.end, workspace_bytes, ws.end);
    GdrArgs a{};
    gdr_fill(a, q, k, v, g, beta, lengths, strides, T, B, Hk, H, dk, dv, scale, flags);
    char* base = (char*)saved;
    a.vec = (float*)(base + lay.vec); a.X = (float*)(base + lay.X); a.P = (float*)(base + lay.P); a.S0 = (float*)(base + lay.S0);
    a.go = go; a.gsT = gstate_out;
    for (int i = 0; i < 3; ++i) a.gos[i] = strides[15 + i];
    char* wb = (char*)workspace;
    a.dS = (float*)(wb + ws.dS); a.E = (uint32_t*)(wb + ws.E); a.zpart = (float*)(wb + ws.z); a.bpart = (float*)(wb + ws.b); a.apart = (float*)(wb + ws.a);
    a.gq = gq; a.gk = gk; a.gv = gv; a.gg = gg; a.gbeta = gbeta; a.gs0 = gstate;
    hipStream_t s = (hipStream_t)stream;
    const bool wide = dk > 64;
    if (dtype == SP_F32) return wide ? gdr_backward<float, 128>(a, s) : gdr_backward<float, 64>(a, s);
    if (dtype == SP_F16) return wide ? gdr_backward<__half, 128>(a, s) : gdr_backward<__half, 64>(a, s);
    return wide ? gdr_backward<__hip_bfloat16, 128>(a, s) : gdr_backward<__hip_bfloat16, 64>(a, s);
}
