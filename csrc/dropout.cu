// Dropout whose mask is drawn again in the backward pass instead of kept: y = keep ? x / (1 - p) : 0, plus a residual.
//
// The mask is a function of (seed, offset, element): element i of the row-major tensor takes word i % 4 of Philox4x32 with seven
// rounds (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011; seven is the smallest number of
// rounds that they found to pass BigCrush) at counter (i / 4, offset) under the key `seed`, and is kept when the word is at least
// p 2^32.  Nothing is stored: 4 (16-bit) or 8 (fp32) bytes an element forward, 2 or 4 more with a residual, the same backward.
//
// fp32 is bound by memory (33.5M elements: 41 us, 6.5 TB/s; with a residual 59 us), 16-bit types by the words as well: seven rounds
// take 60 of the 100 issue slots that four elements cost, 23 us of those 33.5M's 27 (a copy takes 25; with a residual 31).
//   * a thread's four vectors go to shared memory by cp.async, so 64 bytes a thread are on their way without registers; the words of
//     a vector are drawn before its wait.  Vectors in registers (two a thread, 54 registers): 41 us, two and full occupancy 35;
//     blocks that stay and fetch ahead 32, and 55 instead of 41 in fp32.
//   * pairs of elements are converted by one instruction: 27 us instead of 30.
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

// two neighbours at a time: one conversion instruction for the pair
__device__ __forceinline__ float2 pair(const float* v) { return make_float2(v[0], v[1]); }
__device__ __forceinline__ float2 pair(const bf16* v) { return __bfloat1622float2(*reinterpret_cast<const bf162*>(v)); }
__device__ __forceinline__ float2 pair(const __half* v) { return __half22float2(*reinterpret_cast<const __half2*>(v)); }
__device__ __forceinline__ void put(float* v, float a, float b) { v[0] = a, v[1] = b; }
__device__ __forceinline__ void put(bf16* v, float a, float b) { *reinterpret_cast<bf162*>(v) = __floats2bfloat162_rn(a, b); }
__device__ __forceinline__ void put(__half* v, float a, float b) { *reinterpret_cast<__half2*>(v) = __floats2half2_rn(a, b); }

// Seven rounds on counter words (c0, c1, c2, c3) under round keys `k`.  c1, c2 and c3 are the same in a block, so the products of a
// round that meet only them are too, and stay off the lanes.
__device__ __forceinline__ uint4 philox(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3, const uint32_t (&k)[14]) {
#pragma unroll
    for (int r = 0; r < 7; ++r) {
        const unsigned long long a = (unsigned long long)c0 * 0xD2511F53u, b = (unsigned long long)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ k[2 * r];
        c1 = (uint32_t)b;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ k[2 * r + 1];
        c3 = (uint32_t)a;
    }
    return make_uint4(c0, c1, c2, c3);
}

constexpr int kThreads = 256;
constexpr int kBlocks = 4;           // of an SM
constexpr int kStages = 4;           // 16-byte vectors of a thread on their way

__device__ __forceinline__ void copy16(void* dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
}

__device__ __forceinline__ void wait_left(int n) {          // n is known when the loop is unrolled
    static_assert(kStages == 4, "one line for each");
    if (n == 0) asm volatile("cp.async.wait_group 0;" ::: "memory");
    if (n == 1) asm volatile("cp.async.wait_group 1;" ::: "memory");
    if (n == 2) asm volatile("cp.async.wait_group 2;" ::: "memory");
    if (n == 3) asm volatile("cp.async.wait_group 3;" ::: "memory");
}

// VEC: 16-byte vectors; else (a base that is not at a 16-byte boundary) element by element.  STATE: the seed comes from the device.
template <typename T, bool VEC, bool STATE, bool RES>
__global__ void __launch_bounds__(kThreads, kBlocks) dropout_kernel(const DropoutArgs a) {
    constexpr int N = Vec<T>::N;
    __shared__ Vec<T> ring[VEC ? kStages : 1][RES ? 2 : 1][VEC ? kThreads : 1];
    pdl_trigger();
    pdl_wait();
    unsigned long long seed = a.seed, offset = a.offset;
    if (STATE) {
        seed = (unsigned long long)a.state[0];
        if (a.state_len > 1) offset += (unsigned long long)a.state[1];
    }
    if (a.used != nullptr && blockIdx.x == 0 && threadIdx.x == 0) {
        a.used[0] = (long long)seed;
        a.used[1] = (long long)offset;
    }
    uint32_t keys[14];
#pragma unroll
    for (int r = 0; r < 7; ++r) {
        keys[2 * r] = (uint32_t)seed + r * 0x9E3779B9u;
        keys[2 * r + 1] = (uint32_t)(seed >> 32) + r * 0xBB67AE85u;
    }
    const T* x = reinterpret_cast<const T*>(a.x);
    const T* res = reinterpret_cast<const T*>(a.residual);
    T* y = reinterpret_cast<T*>(a.y);
    constexpr int step = kThreads * N;
    auto request = [&](long long i, int s) {
        if (VEC && i + N <= a.n) {
            copy16(&ring[s][0][threadIdx.x], x + i);
            if (RES) copy16(&ring[s][RES ? 1 : 0][threadIdx.x], res + i);
        }
        if (VEC) asm volatile("cp.async.commit_group;" ::: "memory");
    };
    // the upper word of a counter is the block's: its counters are an aligned power of two
    long long first = (long long)blockIdx.x * (kThreads * N * kStages);
#pragma unroll
    for (int s = 0; s < kStages; ++s) request(first + s * step + threadIdx.x * N, s);
#pragma unroll
    for (int s = 0; s < kStages; ++s, first += step) {
        if (first >= a.n) break;
        const long long i = first + threadIdx.x * N;
        uint4 w[N / 4];
#pragma unroll
        for (int g = 0; g < N / 4; ++g)
            w[g] = philox((uint32_t)(i >> 2) + g, (uint32_t)(first >> 34), (uint32_t)offset, (uint32_t)(offset >> 32), keys);
        Vec<T> in, add, out;
        if (VEC) wait_left(kStages - 1 - s);
        if (VEC && i + N <= a.n) {
            in = ring[s][0][threadIdx.x];
            if (RES) add = ring[s][RES ? 1 : 0][threadIdx.x];
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e) {
                if (i + e < a.n) {
                    in.v[e] = x[i + e];
                    if (RES) add.v[e] = res[i + e];
                }
            }
        }
#pragma unroll
        for (int e = 0; e < N; e += 2) {          // one rounding, at the end; a dropped NaN is gone
            const uint4 u = w[e / 4];
            const bool k0 = (e % 4 ? u.z : u.x) >= a.threshold, k1 = (e % 4 ? u.w : u.y) >= a.threshold;
            const float2 v = pair(in.v + e), r = RES ? pair(add.v + e) : make_float2(0.f, 0.f);
            put(out.v + e, k0 ? (RES ? fmaf(v.x, a.scale, r.x) : v.x * a.scale) : r.x, k1 ? (RES ? fmaf(v.y, a.scale, r.y) : v.y * a.scale) : r.y);
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

template <typename T, bool VEC, bool STATE>
int launch_as(const DropoutArgs& a, cudaStream_t st) {
    const long long per = (long long)kThreads * Vec<T>::N * kStages, blocks = (a.n + per - 1) / per;
    NXD_REQUIRE(blocks < (1ll << 31), "dropout: %lld elements", a.n);
    const dim3 grid((unsigned)blocks);
    if (a.residual != nullptr)
        NXD_CHECK_CUDA((nxd_launch_pdl(dropout_kernel<T, VEC, STATE, true>, grid, dim3(kThreads), 0, st, a)));
    else
        NXD_CHECK_CUDA((nxd_launch_pdl(dropout_kernel<T, VEC, STATE, false>, grid, dim3(kThreads), 0, st, a)));
    NXD_LAUNCH_CHECK();
    return 0;
}

template <typename T>
int launch(const DropoutArgs& a, cudaStream_t st) {
    if ((((uintptr_t)a.x | (uintptr_t)a.residual | (uintptr_t)a.y) & 15) == 0)
        return a.state ? launch_as<T, true, true>(a, st) : launch_as<T, true, false>(a, st);
    return a.state ? launch_as<T, false, true>(a, st) : launch_as<T, false, false>(a, st);
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
