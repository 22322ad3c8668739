// Dropout whose mask is drawn again in the backward pass instead of kept: y = keep ? x / (1 - p) : 0, plus a residual.
//
// The mask is a function of (seed, offset, element): element i of the row-major tensor takes word i % 4 of Philox4x32 with seven
// rounds (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011; seven is the smallest number of
// rounds that they found to pass BigCrush) at counter (i / 4, offset) under the key `seed`, and is kept when the word is at least
// p 2^32.  Nothing is stored: 4 (16-bit) or 8 (fp32) bytes an element forward, 2 or 4 more with a residual, the same backward.
#include <cuda_fp16.h>

#include "common.cuh"

namespace {

struct DropoutArgs {
    const void *x, *residual;
    void* y;
    long long n;
    unsigned long long seed, offset;
    const long long* state;          // NULL, or one or two numbers on the device: the seed and what is added to the offset
    int state_len;
    long long* used;                 // NULL, or where the (seed, offset) of this call go
    uint32_t threshold;
    float scale;
};

template <typename T>
struct Vec {
    static constexpr int N = 16 / sizeof(T);
    alignas(16) T v[N];
};

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(bf16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ bf16 from_float<bf16>(float v) { return __float2bfloat16(v); }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half(v); }

__device__ __forceinline__ uint4 philox(unsigned long long counter, unsigned long long offset, unsigned long long seed) {
    uint32_t c0 = (uint32_t)counter, c1 = (uint32_t)(counter >> 32), c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
    uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int r = 0; r < 7; ++r) {
        const unsigned long long a = (unsigned long long)c0 * 0xD2511F53u, b = (unsigned long long)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)b;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return make_uint4(c0, c1, c2, c3);
}

constexpr int kThreads = 256;
constexpr int kUnroll = 2;           // 16-byte vectors of a thread, all loaded before the first is used

// VEC: 16-byte vectors; else (a base that is not at a 16-byte boundary) element by element.  A thread takes whole groups of four.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads) dropout_kernel(const DropoutArgs a) {
    constexpr int N = Vec<T>::N;
    pdl_trigger();
    pdl_wait();
    unsigned long long seed = a.seed, offset = a.offset;
    if (a.state != nullptr) {
        seed = (unsigned long long)a.state[0];
        if (a.state_len > 1) offset += (unsigned long long)a.state[1];
    }
    if (a.used != nullptr && blockIdx.x == 0 && threadIdx.x == 0) {
        a.used[0] = (long long)seed;
        a.used[1] = (long long)offset;
    }
    const T* x = reinterpret_cast<const T*>(a.x);
    const T* res = reinterpret_cast<const T*>(a.residual);
    T* y = reinterpret_cast<T*>(a.y);
    const long long first = (long long)blockIdx.x * (kThreads * kUnroll * N);
    Vec<T> in[kUnroll], add[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const long long i = first + (u * kThreads + threadIdx.x) * N;
        if (VEC && i + N <= a.n) {
            in[u] = *reinterpret_cast<const Vec<T>*>(x + i);
            if (res != nullptr) add[u] = *reinterpret_cast<const Vec<T>*>(res + i);
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e) {
                if (i + e < a.n) {
                    in[u].v[e] = x[i + e];
                    if (res != nullptr) add[u].v[e] = res[i + e];
                }
            }
        }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const long long i = first + (u * kThreads + threadIdx.x) * N;
        if (i >= a.n) break;
        Vec<T> out;
#pragma unroll
        for (int g = 0; g < N; g += 4) {
            const uint4 w = philox((unsigned long long)(i + g) >> 2, offset, seed);
            const uint32_t word[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                // one rounding at the end; a dropped NaN is gone
                const float r = res != nullptr ? to_float(add[u].v[g + e]) : 0.f;
                const float kept = res != nullptr ? fmaf(to_float(in[u].v[g + e]), a.scale, r) : to_float(in[u].v[g + e]) * a.scale;
                out.v[g + e] = from_float<T>(word[e] >= a.threshold ? kept : r);
            }
        }
        if (VEC && i + N <= a.n) {
            *reinterpret_cast<Vec<T>*>(y + i) = out;
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (i + e < a.n) y[i + e] = out.v[e];
        }
    }
}

template <typename T>
int launch(const DropoutArgs& a, cudaStream_t st) {
    const long long per = (long long)kThreads * kUnroll * Vec<T>::N, blocks = (a.n + per - 1) / per;
    NXD_REQUIRE(blocks < (1ll << 31), "dropout: %lld elements", a.n);
    if ((((uintptr_t)a.x | (uintptr_t)a.residual | (uintptr_t)a.y) & 15) == 0)
        NXD_CHECK_CUDA((nxd_launch_pdl(dropout_kernel<T, true>, dim3((unsigned)blocks), dim3(kThreads), 0, st, a)));
    else
        NXD_CHECK_CUDA((nxd_launch_pdl(dropout_kernel<T, false>, dim3((unsigned)blocks), dim3(kThreads), 0, st, a)));
    NXD_LAUNCH_CHECK();
    return 0;
}

}  // namespace

// x, residual (or NULL), y: n elements each, dtype 0 fp32, 1 bf16, 2 fp16; 0 < p < 1.  state: NULL, or one or two int64 on the device that
// replace `seed` and are added to `offset`; used: NULL, or two int64 that get what this call used.  The backward pass is the
// same call on the gradient, without a residual.
NXD_API int nxd_dropout(const void* x, const void* residual, void* y, long long n, int dtype, double p, unsigned long long seed,
                        unsigned long long offset, const long long* state, int state_len, long long* used, void* stream) {
    NXD_REQUIRE(p > 0.0 && p < 1.0 && n > 0, "dropout: p = %f of %lld elements", p, n);
    DropoutArgs a{x, residual, y, n, seed, offset, state, state_len, used, (uint32_t)(p * 4294967296.0), (float)(1.0 / (1.0 - p))};
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == 0) return launch<float>(a, st);
    if (dtype == 1) return launch<bf16>(a, st);
    NXD_REQUIRE(dtype == 2, "dropout: dtype %d", dtype);
    return launch<__half>(a, st);
}
