// Load-balancing loss of a mixture's routers with its per-expert counts, and its gradient (reference:
// src/neuronx_distributed/modules/moe/loss_function.py:5-48).
//
//   p_r = softmax(x_r) over E experts, S_r = the k largest logits of row r (ties: the lowest expert; NaN counts as largest),
//   f_e = #{r : e in S_r} / n,  P_e = sum_r p_re / n,  loss = E / k sum_e f_e P_e     over the n rows that the mask leaves
//   d loss / d x_re = E / (k n) p_re (f_e - sum_j p_rj f_j)
//
// The rows are those of up to 128 tensors (the layers' routers), read where they are.  L lanes share a row and hold V neighbouring experts
// each, so a row is read in 16-byte pieces and the softmax is L-lane shuffles; a thread keeps its experts' sums and counts in
// registers over all its rows.  Sums of a block go to global memory in a fixed order and a second kernel adds the blocks' in
// double precision: no atomics, the loss does not depend on the schedule.
//
// Forward is bound by issue (half of the instructions are comparisons and selections, two clocks each): 240042 rows of 128 experts in
// fp32, 8 of each, 77 us (memory alone: 19), 524288 rows of 64 69 us; backward by memory: 43 us (38).  Exponentials and the division are
// the library's exact ones (5 % forward; backward in fp32 nothing), and a row's sums are trees: the fp32 gradients of 16 experts are off by
// 2.65e-7 by norm, torch's by 2.7e-7 (sums one after the other: 3.2e-7).
#include <cuda_fp16.h>

#include "common.cuh"

#include <type_traits>

namespace {

constexpr int kMaxLayers = 128;
constexpr int kThreads = 512;            // forward: few blocks, so that there is little to add up
constexpr int kWarps = kThreads / 32;
constexpr int kBwdThreads = 256;

struct Layers {
    const void* x[kMaxLayers];
    long long ld[kMaxLayers];            // elements between rows
    long long first[kMaxLayers + 1];     // rows of the layers before
};
struct RouterArgs {
    const unsigned char* mask;           // [rows of a layer] or NULL: 0 leaves the row out
    int E, k, vec;                       // vec: whole 16-byte pieces
};

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(bf16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ void from_float(float v, float& o) { o = v; }
__device__ __forceinline__ void from_float(float v, bf16& o) { o = __float2bfloat16(v); }
__device__ __forceinline__ void from_float(float v, __half& o) { o = __float2half(v); }

template <typename T, int V>
__device__ __forceinline__ void load_row(const T* row, int e0, int E, bool vec, float (&x)[V]) {
    constexpr int N = 16 / sizeof(T) < V ? 16 / sizeof(T) : V;
    if (vec && e0 + V <= E) {
#pragma unroll
        for (int i = 0; i < V; i += N) {
            struct alignas(N * sizeof(T)) Piece { T v[N]; };
            const Piece p = *reinterpret_cast<const Piece*>(row + e0 + i);
#pragma unroll
            for (int j = 0; j < N; ++j) x[i + j] = to_float(p.v[j]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = e0 + i < E ? to_float(row[e0 + i]) : -INFINITY;
    }
}

template <typename T, int V>
__device__ __forceinline__ void store_row(T* row, int e0, int E, bool vec, const float (&x)[V]) {
    constexpr int N = 16 / sizeof(T) < V ? 16 / sizeof(T) : V;
    if (vec && e0 + V <= E) {
#pragma unroll
        for (int i = 0; i < V; i += N) {
            struct alignas(N * sizeof(T)) Piece { T v[N]; } p;
#pragma unroll
            for (int j = 0; j < N; ++j) from_float(x[i + j], p.v[j]);
            *reinterpret_cast<Piece*>(row + e0 + i) = p;
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (e0 + i < E) from_float(x[i], row[e0 + i]);
    }
}

template <int L>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
    for (int o = 1; o < L; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
template <int L>
__device__ __forceinline__ float group_max(float v) {
#pragma unroll
    for (int o = 1; o < L; o <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// 2^x by the hardware instruction, within 2 units in the last place; the rounding of its argument (x - max) log2 e adds 2^-24 of that
// argument.  For gradients that are rounded to 16 bits, 2^-11 of them at best: a probability as small as 2^-126 is off by 2^-17
// of itself, of which a rounding in some hundred of fp16 takes notice.  expf costs 5 us more for 240042 rows of 128 experts in bf16 (33).
__device__ __forceinline__ float exp_near(float x) {
    float y;
    asm("ex2.approx.f32 %0, %1;" : "=f"(y) : "f"(x * 1.4426950408889634f));
    return y;
}

// pairs, pairs of pairs and so on: the rounding of a sum grows with the logarithm of V
template <int N>
__device__ __forceinline__ float tree_sum(float (&v)[N]) {
#pragma unroll
    for (int d = 1; d < N; d <<= 1)
#pragma unroll
        for (int i = 0; i + d < N; i += 2 * d) v[i] += v[i + d];
    return v[0];
}

// x <- exp(x - max) of the row; their sum.  A NaN, or a maximum that is infinite, makes all of it NaN.
template <int L, bool NEAR, int V>
__device__ __forceinline__ float exp_row(float (&x)[V]) {
    float m = x[0];
#pragma unroll
    for (int i = 1; i < V; ++i) m = fmaxf(m, x[i]);
    m = group_max<L>(m);
    float s[V];
#pragma unroll
    for (int i = 0; i < V; ++i) s[i] = x[i] = NEAR ? exp_near(x[i] - m) : expf(x[i] - m);
    return group_sum<L>(tree_sum(s));
}

// Larger numbers have larger keys, +0 and -0 the same one, NaN the largest; 0 is below every number's.  Numbers of 16 bits leave room
// for the expert, so that no two keys of a row are equal and the lower of two equal logits has the larger one.
template <typename T>
__device__ __forceinline__ uint32_t order_key(float v, int e) {
    v += 0.f;          // -0 becomes +0, and every NaN the one whose bits are 0x7fffffff
    uint32_t b = __float_as_uint(v);
    if (std::is_same<T, __half>::value) b = (uint32_t)__half_as_ushort(__float2half_rn(v)) << 16;          // the bits that were read
    const uint32_t k = b ^ (uint32_t)((int)b >> 31 | (int)0x80000000);
    return sizeof(T) == 4 ? k : (k & 0xffff0000u) | (uint32_t)(0xffff - e);
}

// the largest key of a row's lanes.  A reduction of the whole warp is one instruction (160000 rows of 512 experts, 8 of each: 209 us instead
// of 237); of a part of it shuffles are faster (240042 rows of 128 experts: 86 us instead of 96, 524288 of 64: 88 and 118).
template <int L>
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
    if (L == 32) return __reduce_max_sync(0xffffffffu, v);
#pragma unroll
    for (int o = 1; o < L; o <<= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// the eight largest of the keys, largest first
template <int N>
__device__ __forceinline__ void order2(uint32_t (&h)[N], int i, int j) {
    const uint32_t a = max(h[i], h[j]), b = min(h[i], h[j]);
    h[i] = a;
    h[j] = b;
}
// Batcher's odd-even merge sort of eight, 19 exchanges
__device__ __forceinline__ void sort8(uint32_t (&h)[8]) {
    order2(h, 0, 1), order2(h, 2, 3), order2(h, 4, 5), order2(h, 6, 7);
    order2(h, 0, 2), order2(h, 1, 3), order2(h, 4, 6), order2(h, 5, 7);
    order2(h, 1, 2), order2(h, 5, 6);
    order2(h, 0, 4), order2(h, 1, 5), order2(h, 2, 6), order2(h, 3, 7);
    order2(h, 2, 4), order2(h, 3, 5);
    order2(h, 1, 2), order2(h, 3, 4), order2(h, 5, 6);
}
template <int V>
__device__ __forceinline__ void top8(const uint32_t (&key)[V], uint32_t (&h)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = key[i];
    sort8(h);
#pragma unroll
    for (int g = 8; g < V; g += 8) {
        uint32_t o[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = key[g + i];
        sort8(o);
        // the larger halves of two sorted lists are a bitonic list
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] = max(h[i], o[7 - i]);
#pragma unroll
        for (int d = 4; d > 0; d >>= 1)
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (!(i & d)) order2(h, i, i + d);
    }
}

// grid (blocks of a layer, layers).  part_p / part_c: [blocks][E] sums of probabilities and counts.
template <typename T, int L, int V>
__global__ void __launch_bounds__(kThreads) balance_fwd_kernel(const __grid_constant__ Layers layers, const RouterArgs a,
                                                               float* __restrict__ part_p, int* __restrict__ part_c) {
    constexpr int R = kThreads / L;      // rows of a block at a time
    pdl_trigger();
    pdl_wait();
    const int layer = blockIdx.y, l = threadIdx.x % L, e0 = l * V;
    const T* x0 = reinterpret_cast<const T*>(layers.x[layer]);
    const long long ld = layers.ld[layer], rows = layers.first[layer + 1] - layers.first[layer];
    float sum[V];
    int count[V];
#pragma unroll
    for (int i = 0; i < V; ++i) sum[i] = 0.f, count[i] = 0;
    const int lane = threadIdx.x & 31;
    const unsigned lanes_below = ((1u << lane) - 1u) & (0xffffffffu << (lane & ~(L - 1)));          // of this row's lanes
    // all lanes of a warp go through the same iterations: the shuffles want every one
    for (long long r0 = (long long)blockIdx.x * R; r0 < rows; r0 += (long long)gridDim.x * R) {
        const long long r = r0 + threadIdx.x / L;
        const bool valid = r < rows && (a.mask == nullptr || a.mask[r] != 0);
        float x[V];
        if (valid) {
            load_row<T, V>(x0 + r * ld, e0, a.E, a.vec, x);
        } else {                             // a row like any other, which counts nothing
#pragma unroll
            for (int i = 0; i < V; ++i) x[i] = 0.f;
        }
        uint32_t key[V];
#pragma unroll
        for (int i = 0; i < V; ++i) key[i] = e0 + i < a.E ? order_key<T>(x[i], e0 + i) : 0u;
        const float total = exp_row<L, false>(x), inv = valid ? 1.f / total : 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i) sum[i] = fmaf(x[i], inv, sum[i]);
        // The k-th largest key: every lane's largest ones in order, and k times the largest first one of the row's lanes leaves its list.
        // Equal keys (fp32 only) would leave together: then more than k keys are as large as the last one, and the row's warp takes them
        // one by one, the lowest expert first.
        bool exact = a.k <= 8;
        if (exact) {
            uint32_t h[8], last = 0u;
            top8<V>(key, h);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (j == a.k) break;
                last = row_max<L>(h[0]);
                const bool pop = h[0] == last;
#pragma unroll
                for (int i = 0; i < 7 - j; ++i) h[i] = pop ? h[i + 1] : h[i];          // no more are asked for
            }
            int chosen = 0;
#pragma unroll
            for (int i = 0; i < V; ++i) chosen += key[i] >= last;
            if (sizeof(T) == 4) {
                int all = chosen;
#pragma unroll
                for (int o = 1; o < L; o <<= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
                exact = __all_sync(0xffffffffu, !valid || all == a.k);
            }
            if (exact) {
                if (!valid) last = 0xffffffffu;          // above a zero's key
#pragma unroll
                for (int i = 0; i < V; ++i) count[i] += key[i] >= last;
            }
        }
        if (!exact) {
            for (int j = 0; j < a.k; ++j) {
                uint32_t best = key[0];
#pragma unroll
                for (int i = 1; i < V; ++i) best = max(best, key[i]);
                uint32_t top = best;
#pragma unroll
                for (int o = 1; o < L; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
                bool mine = true;
                if (L > 1) mine = (__ballot_sync(0xffffffffu, best == top) & lanes_below) == 0u;
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const bool hit = mine && key[i] == top;
                    if (hit) key[i] = 0u;
                    mine = mine && !hit;
                }
            }
#pragma unroll
            for (int i = 0; i < V; ++i) count[i] += valid && key[i] == 0u;          // those past E too: they are not stored
        }
    }
    // lanes that hold the same experts, then the warps in a fixed order, in one array for sums and counts
    __shared__ uint32_t s_warp[kWarps / 2][L * V];
    const long long base = ((long long)blockIdx.y * gridDim.x + blockIdx.x) * a.E;
    const int warp = threadIdx.x >> 5, slot = warp % (kWarps / 2);
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
        for (int o = L; o < 32; o <<= 1) {
            sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], o);
            count[i] += __shfl_xor_sync(0xffffffffu, count[i], o);
        }
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        if (warp / (kWarps / 2) == half && lane < L) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                uint32_t* at = &s_warp[slot][e0 + i];
                *at = __float_as_uint(half ? __uint_as_float(*at) + sum[i] : sum[i]);
            }
        }
        __syncthreads();
    }
    for (int e = threadIdx.x; e < a.E; e += kThreads) {
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps / 2; ++w) s += __uint_as_float(s_warp[w][e]);
        part_p[base + e] = s;
    }
    __syncthreads();
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        if (warp / (kWarps / 2) == half && lane < L) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                uint32_t* at = &s_warp[slot][e0 + i];
                *at = half ? *at + (uint32_t)count[i] : (uint32_t)count[i];
            }
        }
        __syncthreads();
    }
    for (int e = threadIdx.x; e < a.E; e += kThreads) {
        int c = 0;
#pragma unroll
        for (int w = 0; w < kWarps / 2; ++w) c += (int)s_warp[w][e];
        part_c[base + e] = c;
    }
}

// One block: sums over the blocks of the first kernel, the loss, the counts, and for the gradient f_e E / (k n).
constexpr int kFinalThreads = 1024;
__global__ void __launch_bounds__(kFinalThreads) balance_final_kernel(const float* __restrict__ part_p, const int* __restrict__ part_c,
                                                                      int blocks, int E, int k, float* loss, long long* counts,
                                                                      float* share) {
    __shared__ double s_p[kFinalThreads];
    __shared__ long long s_c[kFinalThreads];
    pdl_trigger();
    pdl_wait();
    const int tid = threadIdx.x;
    int W = 1;                            // threads of one expert group
    while (W < E) W <<= 1;                // at most 1024
    const int e = tid % W, g = tid / W, G = kFinalThreads / W;
    double p = 0.0;
    long long c = 0;
    if (e < E)
#pragma unroll 8
        for (int b = g; b < blocks; b += G) {
            p += (double)part_p[(long long)b * E + e];
            c += part_c[(long long)b * E + e];
        }
    s_p[tid] = p;
    s_c[tid] = c;
    __syncthreads();
    for (int h = kFinalThreads / 2; h >= W; h >>= 1) {
        if (tid < h) s_p[tid] += s_p[tid + h], s_c[tid] += s_c[tid + h];
        __syncthreads();
    }
    if (tid < W) p = s_p[tid], c = s_c[tid];
    __syncthreads();
    // over the experts: sum of f_e P_e and of the counts, which are k for every row
    if (tid < W) s_p[tid] = (double)c * p;
    __syncthreads();
    for (int h = W / 2; h > 0; h >>= 1) {
        if (tid < h) s_p[tid] += s_p[tid + h], s_c[tid] += s_c[tid + h];
        __syncthreads();
    }
    const double n = (double)(s_c[0] / k), factor = n > 0.0 ? (double)E / ((double)k * n * n) : 0.0;
    if (tid == 0) *loss = n > 0.0 ? (float)(s_p[0] * factor) : 0.f;
    if (tid < E) {
        counts[tid] = c;
        share[tid] = (float)((double)c * factor);
    }
}

template <typename T, int L, int V>
__global__ void __launch_bounds__(kBwdThreads) balance_bwd_kernel(const __grid_constant__ Layers layers, const RouterArgs a,
                                                               const float* __restrict__ share, const float* __restrict__ grad,
                                                               T* __restrict__ dx) {
    constexpr int R = kBwdThreads / L;
    pdl_trigger();
    pdl_wait();
    const int layer = blockIdx.y, l = threadIdx.x % L, e0 = l * V;
    const T* x0 = reinterpret_cast<const T*>(layers.x[layer]);
    const long long ld = layers.ld[layer], first = layers.first[layer], rows = layers.first[layer + 1] - first;
    float f[V];
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = e0 + i < a.E ? share[e0 + i] : 0.f;
    const float g = *grad;
    for (long long r0 = (long long)blockIdx.x * R; r0 < rows; r0 += (long long)gridDim.x * R) {
        const long long r = r0 + threadIdx.x / L;
        const bool valid = r < rows && (a.mask == nullptr || a.mask[r] != 0);
        float x[V];
        load_row<T, V>(x0 + min(r, rows - 1) * ld, e0, a.E, a.vec, x);
        // p (f - sum p f) with p = x / total: the reciprocal's rounding, which all p share, stays out of the difference
        const float total = exp_row<L, sizeof(T) == 2>(x), inv = 1.f / total;
        float pairs[V / 2];
#pragma unroll
        for (int i = 0; i < V; i += 2) pairs[i / 2] = fmaf(x[i], f[i], x[i + 1] * f[i + 1]);
        const float s = group_sum<L>(tree_sum(pairs));
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = valid ? x[i] * inv * (fmaf(f[i], total, -s) * (inv * g)) : 0.f;
        if (r < rows) store_row<T, V>(dx + (first + r) * a.E, e0, a.E, a.vec, x);
    }
}

struct Plan {
    Layers layers;
    RouterArgs args;
    long long most;                      // rows of the largest layer
    int blocks_x, n;
    bool backward;
};

// Blocks of a layer: all layers' together are on the chip at once and no more than that (half of a second round costs as much as a
// whole one; with three blocks for each SM, whatever fits, 524288 rows of 64 experts took 88 us instead of 72, 160000 of 512 209
// instead of 170, 240042 of 128 86 instead of 82), and no more than there are rows for.
int blocks_of(long long most_rows, int layers, int lanes, int threads, int per_sm) {
    const long long want = (most_rows + threads / lanes - 1) / (threads / lanes);
    const long long fill = (long long)per_sm * nxd_num_sms() / layers, n = want < fill ? want : fill;
    return n < 1 ? 1 : (int)n;
}
int lanes_of(int E) {
    int l = 1;
    while (l < 32 && l * 8 < E) l <<= 1;
    return l;
}

int make_plan(Plan* p, bool backward, const void* const* x, const long long* ld, const long long* rows, int n, int elem, const void* mask,
              int E, int k, const void* dx) {
    NXD_REQUIRE(n > 0 && n <= kMaxLayers && E > 0 && E <= 1024 && k > 0 && k <= E, "balance_loss: %d tensors, %d of %d experts", n, k, E);
    long long most = 0, total = 0;
    bool vec = (long long)E * elem % 16 == 0 && ((uintptr_t)dx & 15) == 0;
    for (int i = 0; i < n; ++i) {
        NXD_REQUIRE(rows[i] >= 0, "balance_loss: %lld rows", rows[i]);
        p->layers.x[i] = x[i];
        p->layers.ld[i] = ld[i];
        p->layers.first[i] = total;
        total += rows[i];
        most = rows[i] > most ? rows[i] : most;
        vec = vec && ((uintptr_t)x[i] & 15) == 0 && ld[i] * elem % 16 == 0;
    }
    p->layers.first[n] = total;
    NXD_REQUIRE(total < (1ll << 31) && total * k < (1ll << 40), "balance_loss: %lld rows", total);
    p->args = RouterArgs{(const unsigned char*)mask, E, k, vec};
    NXD_REQUIRE(!backward || dx != nullptr || total == 0, "balance_loss: no gradients' memory for %lld rows", total);
    p->n = n;
    p->most = most;
    p->backward = backward;
    return 0;
}

template <auto Kernel>
int blocks_per_sm(int threads) {
    static const int n = [threads] {
        int m = 0;
        return cudaOccupancyMaxActiveBlocksPerMultiprocessor(&m, Kernel, threads, 0) == cudaSuccess && m > 0 ? m : 1;
    }();
    return n;
}

template <typename T, int L, int V>
int run(Plan& p, float* scratch, const float* share, const float* grad, void* dx, cudaStream_t st) {
    if (!p.backward) {
        constexpr auto kern = balance_fwd_kernel<T, L, V>;
        p.blocks_x = blocks_of(p.most, p.n, L, kThreads, blocks_per_sm<kern>(kThreads));
        int* part_c = (int*)(scratch + (long long)p.blocks_x * p.n * p.args.E);
        NXD_CHECK_CUDA((nxd_launch_pdl(kern, dim3(p.blocks_x, p.n), dim3(kThreads), 0, st, p.layers, p.args, scratch, part_c)));
    } else {
        constexpr auto kern = balance_bwd_kernel<T, L, V>;
        p.blocks_x = blocks_of(p.most, p.n, L, kBwdThreads, blocks_per_sm<kern>(kBwdThreads));
        NXD_CHECK_CUDA((nxd_launch_pdl(kern, dim3(p.blocks_x, p.n), dim3(kBwdThreads), 0, st, p.layers, p.args, share, grad, (T*)dx)));
    }
    NXD_LAUNCH_CHECK();
    return 0;
}

template <typename T>
int run_sized(Plan& p, float* scratch, const float* share, const float* grad, void* dx, cudaStream_t st) {
    const int E = p.args.E;
    if (E <= 8) return run<T, 1, 8>(p, scratch, share, grad, dx, st);
    if (E <= 16) return run<T, 2, 8>(p, scratch, share, grad, dx, st);
    if (E <= 32) return run<T, 4, 8>(p, scratch, share, grad, dx, st);
    if (E <= 64) return run<T, 8, 8>(p, scratch, share, grad, dx, st);
    if (E <= 128) return run<T, 16, 8>(p, scratch, share, grad, dx, st);
    if (E <= 256) return run<T, 32, 8>(p, scratch, share, grad, dx, st);
    if (E <= 512) return run<T, 32, 16>(p, scratch, share, grad, dx, st);
    return run<T, 32, 32>(p, scratch, share, grad, dx, st);
}

int run_typed(Plan& p, int dtype, float* scratch, const float* share, const float* grad, void* dx, cudaStream_t st) {
    if (dtype == 0) return run_sized<float>(p, scratch, share, grad, dx, st);
    if (dtype == 1) return run_sized<bf16>(p, scratch, share, grad, dx, st);
    return run_sized<__half>(p, scratch, share, grad, dx, st);
}

}  // namespace

// Blocks of the first kernel at most: its scratch is that many times E floats and as many ints.
NXD_API int nxd_balance_loss_num_blocks(long long most_rows, int layers, int E) {
    return blocks_of(most_rows, layers, lanes_of(E), kThreads, 2048 / kThreads) * layers;
}

// x, ld, rows: HOST arrays of `layers` device pointers, row strides (elements; unit stride along the experts) and row counts;
// dtype 0 fp32, 1 bf16, 2 fp16; mask: NULL, or a byte per row that every layer shares.  loss: 1 float, counts: E int64, share: E floats
// for the backward call, scratch: nxd_balance_loss_num_blocks * E * 8 bytes.
NXD_API int nxd_balance_loss_fwd(const void* const* x, const long long* ld, const long long* rows, int layers, int dtype,
                                 const void* mask, int E, int k, float* loss, long long* counts, float* share, void* scratch,
                                 void* stream) {
    NXD_REQUIRE(dtype >= 0 && dtype <= 2, "balance_loss: dtype %d", dtype);
    Plan p;
    int rc = make_plan(&p, false, x, ld, rows, layers, dtype == 0 ? 4 : 2, mask, E, k, nullptr);
    if (rc) return rc;
    cudaStream_t st = (cudaStream_t)stream;
    if ((rc = run_typed(p, dtype, (float*)scratch, nullptr, nullptr, nullptr, st))) return rc;
    const int blocks = p.blocks_x * layers;
    const float* part_p = (const float*)scratch;
    const int* part_c = (const int*)(part_p + (long long)blocks * E);
    NXD_CHECK_CUDA(nxd_launch_pdl(balance_final_kernel, dim3(1), dim3(kFinalThreads), 0, st, part_p, part_c, blocks, E, k, loss, counts, share));
    NXD_LAUNCH_CHECK();
    return 0;
}

// dx: [all rows, E] in x's type, the layers one after the other (NULL where there are no rows); grad: the loss's gradient, 1 float on the device.
NXD_API int nxd_balance_loss_bwd(const void* const* x, const long long* ld, const long long* rows, int layers, int dtype,
                                 const void* mask, int E, int k, const float* share, const float* grad, void* dx, void* stream) {
    NXD_REQUIRE(dtype >= 0 && dtype <= 2, "balance_loss: dtype %d", dtype);
    Plan p;
    int rc = make_plan(&p, true, x, ld, rows, layers, dtype == 0 ? 4 : 2, mask, E, k, dx);
    if (rc || p.most == 0) return rc;          // no rows, no gradients
    return run_typed(p, dtype, nullptr, share, grad, dx, (cudaStream_t)stream);
}
