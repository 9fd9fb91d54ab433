// Dropout with the mask from a counter-based generator: Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as
// 1, 2, 3", SC'11) over (index / 8, step, site) under a 64-bit seed.  No mask in memory: the backward call runs the same kernel on gy.
// Every element's draw depends on its index alone, not on the launch.
//
// Bound: HBM (2 or 3 passes over the tensor), closely followed by the vector ALU: ten rounds of two 32 x 32 -> 64 bit products serve
// eight elements with 16 bits each.  Sixteen bits, not 32: the product's issue rate is a quarter, and 32-bit draws would double its
// share beyond what the memory time hides; the rate is then honoured to 2^-17 (documented, the scale follows the honoured rate).
// A thread owns one counter (eight elements, 16 or 32 bytes) and, in the shared form, walks that counter's elements down the rows: the
// generator runs once for all of them.
// Measured at 24032 x 1024 bf16: with a residual 23.4 us (147 MB at 6.3 TB/s), without (the backward) 20.3 us (98 MB at 4.8 TB/s: here the
// products show).
#include "common.h"

namespace sp {

struct DropWords { uint32_t w[4]; };

__device__ __forceinline__ DropWords philox(uint64_t index, uint32_t step, uint32_t site, uint64_t seed) {
    uint32_t c0 = (uint32_t)index, c1 = (uint32_t)(index >> 32), c2 = step, c3 = site;
    uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int i = 0; i < 10; ++i) {
        const uint64_t a = (uint64_t)0xD2511F53u * c0, b = (uint64_t)0xCD9E8D57u * c2;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)b;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return {{c0, c1, c2, c3}};
}

// Eight consecutive elements at an address that is only element-aligned: global memory takes 16-byte accesses at any alignment here.
template <typename T> struct __attribute__((packed, aligned(sizeof(T)))) Drop8 { T e[8]; };

template <typename T, bool RES>
__global__ __launch_bounds__(256) void dropout_kernel(const T* x, const T* res, int64_t rows, int64_t period, uint32_t thr,
                                                      float scale, const int64_t* __restrict__ rng, uint32_t site, T* y,
                                                      int64_t* __restrict__ used) {
    const uint64_t seed = (uint64_t)rng[0];
    const uint64_t step = (uint64_t)rng[1];
    if (used && blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x < 2) used[threadIdx.x] = (int64_t)(threadIdx.x ? step : seed);
    const int64_t j = (int64_t)blockIdx.x * 256 + threadIdx.x;     // counter
    if (j * 8 >= period) return;
    const DropWords d = philox((uint64_t)j, (uint32_t)step, site, seed);
    float gain[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) gain[i] = ((d.w[i >> 1] >> (16 * (i & 1))) & 0xFFFFu) >= thr ? scale : 0.f;
    const int n = (int)(period - j * 8 < 8 ? period - j * 8 : 8);
    for (int64_t r = blockIdx.y; r < rows; r += gridDim.y) {
        const int64_t at = r * period + j * 8;
        if (n == 8) {
            Drop8<T> v = *reinterpret_cast<const Drop8<T>*>(x + at), z;
            if (RES) z = *reinterpret_cast<const Drop8<T>*>(res + at);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float o = gain[i] != 0.f ? Elem<T>::f(v.e[i]) * gain[i] : 0.f;      // a select: dropped infinities and NaN are 0
                if (RES) o += Elem<T>::f(z.e[i]);
                Elem<T>::st(&v.e[i], o);
            }
            *reinterpret_cast<Drop8<T>*>(y + at) = v;
        } else {
            for (int i = 0; i < n; ++i) {
                float o = gain[i] != 0.f ? Elem<T>::ld(x + at + i) * gain[i] : 0.f;
                if (RES) o += Elem<T>::ld(res + at + i);
                Elem<T>::st(y + at + i, o);
            }
        }
    }
}

}  // namespace sp

using namespace sp;

extern "C" int sp_dropout(const void* x, const void* residual, int64_t rows, int64_t period, double p, const int64_t* rng, int site,
                          int dtype, void* y, int64_t* used, void* stream) {
    SP_CHECK_ARG(rows >= 0 && period >= 0 && period < (1ll << 34) && (period == 0 || rows < (1ll << 60) / period),
                 "sp_dropout: bad shape rows=%lld period=%lld (period below 2^34)", (long long)rows, (long long)period);
    SP_CHECK_ARG(p >= 0.0 && p <= 1.0, "sp_dropout: p=%g outside [0, 1]", p);
    SP_CHECK_ARG(dtype == SP_F32 || dtype == SP_BF16 || dtype == SP_F16, "sp_dropout: dtype %d not supported (f32, bf16, f16)", dtype);
    SP_CHECK_ARG(rng, "sp_dropout: null rng");
    SP_CHECK_ARG((rows == 0 || period == 0) || (x && y), "sp_dropout: null pointer");
    const uint32_t thr = (uint32_t)nearbyint(p * 65536.0);
    const float scale = thr < 65536 ? (float)(65536.0 / (65536.0 - thr)) : 0.f;
    if (rows == 0) period = 0;
    const int64_t blocks = period > 0 ? (period + 2047) / 2048 : 1;      // period 0: one workgroup that records `used`
    // shared form: enough rows of workgroups to fill the chip, the rest of the rows walked
    int64_t gy = rows > 0 ? rows : 1;
    if (gy > 1 && blocks * gy > 4096) { gy = 4096 / blocks; if (gy < 1) gy = 1; }
    hipStream_t s = (hipStream_t)stream;
#define SP_DROP(T) { \
    if (residual) hipLaunchKernelGGL((dropout_kernel<T, true>), dim3((unsigned)blocks, (unsigned)gy), dim3(256), 0, s, (const T*)x, (const T*)residual, \
                                     rows, period, thr, scale, rng, (uint32_t)site, (T*)y, used); \
    else hipLaunchKernelGGL((dropout_kernel<T, false>), dim3((unsigned)blocks, (unsigned)gy), dim3(256), 0, s, (const T*)x, (const T*)nullptr, \
                            rows, period, thr, scale, rng, (uint32_t)site, (T*)y, used); }
    if (dtype == SP_F32) SP_DROP(float) else if (dtype == SP_F16) SP_DROP(__half) else SP_DROP(__hip_bfloat16)
#undef SP_DROP
    return check_launch("dropout_kernel");
}
