// Beam search for sm_100a: the choice of a step's candidates, the books of the beams, and the sequences at the end.
//
// Choice.  Of group b's beams w with running scores s[w] and logits x[w, v] the n best of s[w] + x[w, v] - log sum_u exp x[w, u], of equal
// ones the lowest w * V + v.  One pass over the logits: a CTA takes a chunk of one row into registers (256 threads x E values), has its
// maximum and its sum of exponentials, and the chunk's n best in order.  A second kernel joins the chunks of a group's rows.
//   The n best of a chunk: the n-th largest of the 256 threads' maxima bounds the n-th largest value from below, so what is not below it is
// collected (little more than n values as a rule) and ranked by counting.  Equal values in numbers (masked ones) do not fit the buffer: the exact
// n-th key is then found bit by bit and its ties are taken in the order of their indices.
//   Scores are compared in 64 bits: sums of near size decide between rows.  Within a row the logits decide.
// Floor: the logits are read once, 65.7 MB (32 requests of 8 beams, 128256 tokens, bf16) are 10.0 us at 6555 GB/s.
#include <cuda_fp16.h>

#include "common.cuh"

namespace {

constexpr int kRowThreads = 256;
constexpr int kMaxN = 64;
constexpr int kMaxBeams = 32;
constexpr int kMaxLists = 4096;          // chunks of a group
constexpr int kCollect = kRowThreads;    // values that a chunk's short way ranks
constexpr unsigned kFull = 0xffffffffu;

// order-preserving keys; -0 and +0 are one value (the caller adds 0)
__device__ __forceinline__ uint32_t order_key(float f) {
    const uint32_t u = __float_as_uint(f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k); }
constexpr uint32_t kLowestKey = 0x00800000u;          // of the lowest finite number
// the upper half of the same for 64 bits: sign, exponent and 20 bits of the fraction
__device__ __forceinline__ uint32_t order_key_hi(double d) {
    const uint32_t u = (uint32_t)((unsigned long long)__double_as_longlong(d + 0.0) >> 32);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
constexpr uint32_t kLowestKeyHi = 0x00100000u;

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
constexpr float kLog2e = 1.4426950408889634f;

template <typename T> __device__ __forceinline__ float to_float(T x);
template <> __device__ __forceinline__ float to_float<float>(float x) { return x; }
template <> __device__ __forceinline__ float to_float<bf16>(bf16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float to_float<__half>(__half x) { return __half2float(x); }

// Sum over the block's threads; red: 32 ints.
__device__ __forceinline__ int block_count(int v, int* red) {
    v = __reduce_add_sync(kFull, v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    int t = 0;
    for (int i = 0; i < (int)(blockDim.x >> 5); ++i) t += red[i];
    return t;
}

// What a call leaves for the second kernel: per chunk its maximum, the sum of exponentials behind it, and n (value, index) in order.
struct Lists {
    float* top;       // [rows, splits]
    float* sum;       // [rows, splits]
    float* value;     // [rows, splits, n], -inf behind the last
    int* index;       // [rows, splits, n]
};

__host__ __device__ inline Lists lists_of(float* scratch, long long lists, int n) {
    return {scratch, scratch + lists, scratch + 2 * lists, reinterpret_cast<int*>(scratch + 2 * lists + lists * n)};
}

template <typename T, int E>
__global__ void __launch_bounds__(kRowThreads) beam_rows_kernel(const T* __restrict__ logits, int V, long long stride, int splits, int n, Lists out) {
    constexpr int VE = 16 / sizeof(T), NV = E / VE;
    __shared__ uint32_t keys[kRowThreads];
    __shared__ float cand_v[kCollect];
    __shared__ int cand_i[kCollect];
    __shared__ uint32_t warp_key[kRowThreads / 32];
    __shared__ float warp_part[kRowThreads / 32];
    __shared__ int red[32];
    __shared__ uint32_t s_floor;
    __shared__ int s_count;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const long long list = blockIdx.x;
    const int split = (int)(list % splits);
    const T* row = logits + (list / splits) * stride;
    // vectors start on 16 bytes: the row's first element is element `mis` of the first one
    const int mis = (int)((reinterpret_cast<uintptr_t>(row) / sizeof(T)) % VE);
    const int first = split * (kRowThreads * E) + tid * VE - mis;          // index of this thread's first element

    float f[E];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int at = first + i * kRowThreads * VE;
        if (at >= 0 && at + VE <= V) {
            const uint4 raw = __ldg(reinterpret_cast<const uint4*>(row + at));
            const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
            for (int j = 0; j < VE; ++j) f[i * VE + j] = to_float<T>(e[j]);
        } else {
#pragma unroll
            for (int j = 0; j < VE; ++j) f[i * VE + j] = (at + j >= 0 && at + j < V) ? to_float<T>(row[at + j]) : -INFINITY;
        }
    }
    float m = f[0];
#pragma unroll
    for (int j = 1; j < E; ++j) m = fmaxf(m, f[j]);          // passes NaN by
    m = m == m ? m + 0.f : -INFINITY;
    // the differences first: a product of the maximum would lose their last bits.  A NaN, or an infinity, makes the sum NaN and takes the row out
    const float base = m == -INFINITY ? 0.f : m;
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < E; ++j) sum += exp2_approx((f[j] - base) * kLog2e);
    const uint32_t key = order_key(m);
    keys[tid] = key;
    const uint32_t wk = __reduce_max_sync(kFull, key);
    if (lane == 0) warp_key[warp] = wk;
    if (tid == 0) s_count = 0;
    __syncthreads();
    uint32_t block_key = 0;
#pragma unroll
    for (int i = 0; i < kRowThreads / 32; ++i) block_key = max(block_key, warp_key[i]);
    const float top = key_value(block_key);
    sum *= m == -INFINITY ? (sum == sum ? 0.f : 1.f) : exp2_approx((m - top) * kLog2e);
    sum = warp_sum(sum);
    if (lane == 0) warp_part[warp] = sum;
    if (warp == 0) {
        // the n-th largest of the threads' maxima, its upper 16 bits (all that bf16 has): 8 keys a lane
        uint32_t k[kRowThreads / 32];
#pragma unroll
        for (int i = 0; i < kRowThreads / 32; ++i) k[i] = keys[i * 32 + lane];
        uint32_t t = 0;
        for (int bit = 31; bit >= 16; --bit) {
            const uint32_t c = t | (1u << bit);
            int mine = 0;
#pragma unroll
            for (int i = 0; i < kRowThreads / 32; ++i) mine += k[i] >= c;
            if (__reduce_add_sync(kFull, mine) >= n) t = c;
        }
        if (lane == 0) s_floor = max(t, kLowestKey);
    }
    __syncthreads();
    if (tid == 0) {
        float total = 0.f;
#pragma unroll
        for (int i = 0; i < kRowThreads / 32; ++i) total += warp_part[i];
        out.top[list] = top;
        out.sum[list] = total;
    }
    if (key >= s_floor) {
        const float floor = key_value(s_floor);
#pragma unroll
        for (int j = 0; j < E; ++j) {
            if (f[j] >= floor) {
                const int at = atomicAdd(&s_count, 1);
                if (at < kCollect) {
                    cand_v[at] = f[j];
                    cand_i[at] = first + (j / VE) * kRowThreads * VE + j % VE;
                }
            }
        }
    }
    __syncthreads();
    int count = s_count;
    if (count > kCollect) {
        // many equal values: the n-th key bit by bit, then what is above it, then its ties in the order of their indices
        uint32_t t = 0;
        for (int bit = 31; bit >= 0; --bit) {
            const uint32_t c = t | (1u << bit);
            int mine = 0;
#pragma unroll
            for (int j = 0; j < E; ++j) mine += f[j] == f[j] && order_key(f[j] + 0.f) >= c;
            if (block_count(mine, red) >= n) t = c;
        }
        const float tie = key_value(t);
        if (tid == 0) s_count = 0;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < E; ++j) {
            if (f[j] > tie) {                // fewer than n
                const int at = atomicAdd(&s_count, 1);
                cand_v[at] = f[j];
                cand_i[at] = first + (j / VE) * kRowThreads * VE + j % VE;
            }
        }
        __syncthreads();
        int have = s_count;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            int mine = 0;
#pragma unroll
            for (int j = 0; j < VE; ++j) mine += f[i * VE + j] == tie;
            int before = mine;               // of this thread and the ones before it
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(kFull, before, o);
                if (lane >= o) before += x;
            }
            __syncthreads();
            if (lane == 31) red[warp] = before;
            __syncthreads();
            int at = have + before - mine;
            for (int w = 0; w < kRowThreads / 32; ++w) {
                if (w < warp) at += red[w];
                have += red[w];
            }
#pragma unroll
            for (int j = 0; j < VE; ++j) {
                if (f[i * VE + j] == tie) {
                    if (at < n) {
                        cand_v[at] = tie;
                        cand_i[at] = first + i * kRowThreads * VE + j;
                    }
                    ++at;
                }
            }
        }
        __syncthreads();
        count = min(have, n);
    }
    if (tid < count) {
        const float v = cand_v[tid];
        const int idx = cand_i[tid];
        int rank = 0;
        for (int j = 0; j < count; ++j) rank += cand_v[j] > v || (cand_v[j] == v && cand_i[j] < idx);
        if (rank < n) {
            out.value[list * n + rank] = v;
            out.index[list * n + rank] = idx;
        }
    }
    if (tid >= count && tid < n) out.value[list * n + tid] = -INFINITY;
}

// The rank of (score, order) among `count` of them: greater scores first, of equal ones the lower order.
__device__ __forceinline__ int rank_of(const double* score, const int* order, int count, int i) {
    const double s = score[i];
    const int o = order[i];
    int rank = 0;
    for (int j = 0; j < count; ++j) rank += score[j] > s || (score[j] == s && order[j] < o);
    return rank;
}

// One CTA joins the lists of one group's rows.  Every list is in order, so its head is its best: the n lists with the best heads hold
// the n best values, and none of those is below the n-th head.
__global__ void __launch_bounds__(1024) beam_join_kernel(const float* __restrict__ scores, int W, int V, int splits, int n, Lists in, float* __restrict__ out_scores,
                                 long long* __restrict__ out_beams, long long* __restrict__ out_tokens) {
    extern __shared__ double smem[];
    __shared__ double so_far[kMaxBeams], lse[kMaxBeams];
    __shared__ int sel[kMaxN];
    __shared__ int red[32];
    __shared__ uint32_t s_floor;
    __shared__ int s_count;
    __shared__ unsigned char used[2 * kMaxN];
    const int lists = W * splits, room = max(lists, n * min(n, lists));
    double* head = smem;                                     // [lists]
    double* cand = head + lists;                             // [room]
    int* cand_i = reinterpret_cast<int*>(cand + room);       // [room]
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nth = blockDim.x, warps = nth >> 5;
    const long long g = blockIdx.x, l0 = g * lists;
    pdl_wait();
    for (int w = warp; w < W; w += warps) {
        const long long at = l0 + (long long)w * splits;
        float top = -INFINITY;
        for (int i = lane; i < splits; i += 32) top = fmaxf(top, in.top[at + i]);
        top = warp_max(top);
        double sum = 0.0;
        for (int i = lane; i < splits; i += 32) {
            const float t = in.top[at + i];
            sum += (double)in.sum[at + i] * (t == -INFINITY ? 1.0 : exp((double)t - (double)top));
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(kFull, sum, o);
        const float own = scores[g * W + w];
        // a row with NaN, with +inf or without a finite logit has no candidates
        if (lane == 0) {
            so_far[w] = sum > 0.0 && own > -INFINITY ? (double)own : -INFINITY;
            lse[w] = sum > 0.0 ? (double)top + log(sum) : 0.0;
        }
    }
    if (tid == 0) s_count = 0;
    if (tid < 2 * kMaxN) used[tid] = 0;
    __syncthreads();
    for (int l = tid; l < lists; l += nth) {
        const float v = in.value[(l0 + l) * n];
        const int w = l / splits;
        head[l] = v > -INFINITY && so_far[w] > -INFINITY ? so_far[w] + ((double)v - lse[w]) : -INFINITY;
    }
    __syncthreads();
    if (warp == 0) {
        uint32_t t = 0;
        for (int bit = 31; bit >= 0; --bit) {
            const uint32_t c = t | (1u << bit);
            int mine = 0;
            for (int l = lane; l < lists; l += 32) mine += order_key_hi(head[l]) >= c;
            if (__reduce_add_sync(kFull, mine) >= n) t = c;
        }
        if (lane == 0) s_floor = max(t, kLowestKeyHi);
    }
    __syncthreads();
    for (int l = tid; l < lists; l += nth) {
        if (order_key_hi(head[l]) >= s_floor) {
            const int at = atomicAdd(&s_count, 1);
            cand[at] = head[l];
            cand_i[at] = l;          // heads of a row are in the order of their lists
        }
    }
    __syncthreads();
    const int heads = s_count;
    for (int i = tid; i < heads; i += nth) {
        const int r = rank_of(cand, cand_i, heads, i);
        if (r < n) sel[r] = cand_i[i];
    }
    __syncthreads();
    const int picked = min(heads, n);
    const double least = heads >= n ? head[sel[n - 1]] : -INFINITY;
    if (tid == 0) s_count = 0;
    __syncthreads();
    for (int e = tid; e < picked * n; e += nth) {
        const int l = sel[e / n], w = l / splits;
        const float v = in.value[(l0 + l) * n + e % n];
        const double s = so_far[w] + ((double)v - lse[w]);
        if (v > -INFINITY && so_far[w] > -INFINITY && s >= least) {
            const int at = atomicAdd(&s_count, 1);
            cand[at] = s;
            cand_i[at] = w * V + in.index[(l0 + l) * n + e % n];
        }
    }
    __syncthreads();
    int count = s_count;
    if (count > 4 * n && count > 128) {
        // few lists hold much that is not below the least head: the n-th score's upper half bit by bit, and what is not below that
        uint32_t t = 0;
        for (int bit = 31; bit >= 0; --bit) {
            const uint32_t c = t | (1u << bit);
            int mine = 0;
            for (int i = tid; i < count; i += nth) mine += order_key_hi(cand[i]) >= c;
            if (block_count(mine, red) >= n) t = c;
        }
        // moved to the front in rounds, each read before any of it is written
        if (tid == 0) s_count = 0;
        __syncthreads();
        for (int at = 0; at < count; at += nth) {
            const int i = at + tid;
            const double s = i < count ? cand[i] : 0.0;
            const int o = i < count ? cand_i[i] : 0;
            const bool keep = i < count && order_key_hi(s) >= t;
            __syncthreads();
            if (keep) {
                const int to = atomicAdd(&s_count, 1);
                cand[to] = s;
                cand_i[to] = o;
            }
            __syncthreads();
        }
        count = s_count;
    }
    for (int i = tid; i < count; i += nth) {
        const int r = rank_of(cand, cand_i, count, i), o = cand_i[i];
        if (r < n) {
            out_scores[g * n + r] = (float)cand[i];
            out_beams[g * n + r] = o / V;
            out_tokens[g * n + r] = o % V;
        }
        if (count < n && o < 2 * kMaxN) used[o] = 1;
    }
    __syncthreads();
    if (tid == 0 && count < n) {             // the rest are -inf, from the lowest index on
        int o = 0;
        for (int r = count; r < n; ++r, ++o) {
            while (used[o]) ++o;
            out_scores[g * n + r] = -INFINITY;
            out_beams[g * n + r] = o / V;
            out_tokens[g * n + r] = o % V;
        }
    }
}

// ---- the books --------------------------------------------------------------------------------------------------------

struct Books {
    const float* running;                            // [B, W]
    const float* pool_score;                         // [B, W]
    const int* pool_length;                          // [B, W]
    const int* pool_slot;                            // [B, W]
    const unsigned char* done;                       // [B]
};

// One entry of two rows of up to 32 in one order: the better first, of equal ones the first row's, then the lower place.
__device__ __forceinline__ void merge_ranks(float a, float b, int count, int lane, int& ra, int& rb) {
    ra = rb = 0;
    for (int j = 0; j < count; ++j) {
        const float aj = __shfl_sync(kFull, a, j), bj = __shfl_sync(kFull, b, j);
        ra += (aj > a || (aj == a && j < lane)) + (bj > a);
        rb += (aj >= b) + (bj > b || (bj == b && j < lane));
    }
}

// A warp per group: lane r has candidates r and 32 + r, lane w line w and place w of the pool.
__global__ void __launch_bounds__(128) beam_advance_kernel(const float* __restrict__ cand_s, const long long* __restrict__ cand_b, const long long* __restrict__ cand_t,
                                    int B, int W, int N, Books in, float norm, long long eos, long long pad, int early, float* __restrict__ running,
                                    long long* __restrict__ tokens, long long* __restrict__ parents, float* __restrict__ pool_score,
                                    int* __restrict__ pool_length, int* __restrict__ pool_slot, unsigned char* __restrict__ done,
                                    int* __restrict__ hist_token, int* __restrict__ hist_parent, int length) {
    constexpr int kWarps = 4;
    __shared__ int pick_of[kWarps][kMaxBeams], free_of[kWarps][kMaxBeams];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long b = (long long)blockIdx.x * kWarps + warp;
    if (b >= B) return;
    const long long at = b * W + lane;
    const bool mine = lane < W;
    const unsigned lines = W == 32 ? kFull : (1u << W) - 1u, below = (1u << lane) - 1u;
    const float old_running = mine ? in.running[at] : -INFINITY;
    const float old_score = mine ? in.pool_score[at] : -INFINITY;
    const int old_length = mine ? in.pool_length[at] : 0, old_slot = mine ? in.pool_slot[at] : 0;
    if (in.done[b]) {                                // a request that is over stays as it is
        if (mine) {
            running[at] = old_running;
            tokens[at] = pad;
            parents[at] = lane;
            pool_score[at] = old_score;
            pool_length[at] = old_length;
            pool_slot[at] = old_slot;
            hist_token[at] = (int)pad;
            hist_parent[at] = lane;
        }
        if (lane == 0) done[b] = 1;
        return;
    }
    const float s0 = lane < N ? cand_s[b * N + lane] : -INFINITY;
    const long long t0 = lane < N ? cand_t[b * N + lane] : eos;
    const bool on0 = lane < N && t0 != eos, on1 = 32 + lane < N && cand_t[b * N + 32 + lane] != eos;
    const unsigned g0 = __ballot_sync(kFull, on0), g1 = __ballot_sync(kFull, on1);
    // the best W that go on
    const int p0 = __popc(g0 & below), p1 = __popc(g0) + __popc(g1 & below);
    if (on0 && p0 < W) pick_of[warp][p0] = lane;
    if (on1 && p1 < W) pick_of[warp][p1] = 32 + lane;
    __syncwarp();
    const bool valid = mine && lane < __popc(g0) + __popc(g1);
    const int r = valid ? pick_of[warp][lane] : 0;
    const float score = valid ? cand_s[b * N + r] : -INFINITY;
    const long long token = valid ? cand_t[b * N + r] : pad;
    const long long parent = valid ? cand_b[b * N + r] : -1 - lane;
    // the best child of a beam stays in its line, the others go to the lines that nobody continues, in order
    const unsigned same = __match_any_sync(kFull, parent);
    const bool stays = valid && parent >= 0 && parent < W && (same & below) == 0;
    const unsigned taken = __reduce_or_sync(kFull, stays ? 1u << parent : 0u);
    const unsigned open = lines & ~taken;
    if (open >> lane & 1) free_of[warp][__popc(open & below)] = lane;
    const unsigned movers = __ballot_sync(kFull, mine && !stays);
    __syncwarp();
    const int slot = !mine ? 0 : stays ? (int)parent : free_of[warp][__popc(movers & below)];
    if (mine) {
        running[b * W + slot] = score;
        tokens[b * W + slot] = token;
        parents[b * W + slot] = valid ? parent : slot;
        hist_token[b * W + slot] = (int)token;
        hist_parent[b * W + slot] = valid ? (int)parent : slot;
    }
    // what has ended among the best W joins the pool
    const bool ends = mine && lane < N && t0 == eos && s0 > -INFINITY;
    const float ended = ends ? __fdiv_rn(s0, norm) : -INFINITY;
    int ra, rb;
    merge_ranks(old_score, ended, W, lane, ra, rb);
    if (mine && ra < W) {
        pool_score[b * W + ra] = old_score;
        pool_length[b * W + ra] = old_score > -INFINITY ? old_length : 0;
        pool_slot[b * W + ra] = old_score > -INFINITY ? old_slot : 0;
    }
    if (mine && rb < W) {
        pool_score[b * W + rb] = ended;
        pool_length[b * W + rb] = ends ? length : 0;
        pool_slot[b * W + rb] = ends ? (int)cand_b[b * N + lane] : 0;
    }
    const float last = warp_max(ra == W - 1 ? old_score : rb == W - 1 ? ended : -INFINITY);
    const float best = __fdiv_rn(warp_max(score), norm);
    if (lane == 0) done[b] = last > -INFINITY && (early || last >= best);
}

constexpr int kTraceSteps = 16;          // steps that a warp writes at a time

// The beams of requests that are not over join the pool, and every place's tokens are found from the last one back.  A line's history is
// a chain of parents; a warp walks a section of it for all lines at once (lane w starts in line w at the section's end), so the
// sections are walked side by side, joined, and walked once more for the tokens.
__global__ void __launch_bounds__(1024) beam_finish_kernel(Books in, int W, int B, int step, float norm, long long eos, long long pad, const int* __restrict__ hist_token,
                                   const int* __restrict__ hist_parent, long long* __restrict__ tokens, long long* __restrict__ lengths,
                                   float* __restrict__ scores) {
    extern __shared__ int stage[];                                       // [warps][W][kTraceSteps + 1]
    __shared__ int enter_at[kMaxBeams], enter_slot[kMaxBeams], len[kMaxBeams], ended[kMaxBeams];
    __shared__ unsigned char through[32][32], part[32][32], entry[32][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const long long b = blockIdx.x;
    const int section = (step + warps - 1) / warps;
    if (warp == 0) {
        const bool mine = lane < W;
        const long long at = b * W + lane;
        const float a = mine ? in.pool_score[at] : -INFINITY;
        const float r = mine && !in.done[b] ? __fdiv_rn(in.running[at], norm) : -INFINITY;
        const float c = r == r ? r : -INFINITY;
        int ra, rb;
        merge_ranks(a, c, W, lane, ra, rb);
        if (mine && ra < W) {
            const int n = a > -INFINITY ? min(max(in.pool_length[at], 0), step) : 0;
            scores[b * W + ra] = a;
            len[ra] = n;
            ended[ra] = 1;
            enter_at[ra] = n - 2;            // the last token is the one that ends
            enter_slot[ra] = min(max(in.pool_slot[at], 0), W - 1);
        }
        if (mine && rb < W) {
            const int n = c > -INFINITY ? step : 0;
            scores[b * W + rb] = c;
            len[rb] = n;
            ended[rb] = 0;
            enter_at[rb] = n - 1;
            enter_slot[rb] = lane;
        }
    }
    __syncthreads();
    const int mine = min(lane, W - 1);
    const int lo = warp * section, hi = min(step, lo + section);
    const int t_in = enter_at[mine];
    {
        int line = mine, cur = enter_slot[mine];
        for (int t1 = hi; t1 > lo; t1 -= kTraceSteps) {
            const int t0 = max(lo, t1 - kTraceSteps);
            int p[kTraceSteps];
#pragma unroll
            for (int i = 0; i < kTraceSteps; ++i) p[i] = t1 - 1 - i >= t0 ? min(max(hist_parent[((long long)(t1 - 1 - i) * B + b) * W + mine], 0), W - 1) : 0;
#pragma unroll
            for (int i = 0; i < kTraceSteps; ++i) {
                if (t1 - 1 - i < t0) break;
                line = __shfl_sync(kFull, p[i], line);
                const int next = __shfl_sync(kFull, p[i], cur);
                if (t1 - 1 - i <= t_in) cur = next;
            }
        }
        through[warp][lane] = (unsigned char)line;
        part[warp][lane] = (unsigned char)cur;
    }
    __syncthreads();
    if (warp == 0) {
        int cur = enter_slot[mine];
        for (int k = warps - 1; k >= 0; --k) {
            entry[k][lane] = (unsigned char)cur;
            const int k0 = k * section;
            if (t_in >= k0 + section) cur = through[k][cur];             // entered above this section
            else if (t_in >= k0) cur = part[k][lane];
        }
    }
    __syncthreads();
    int cur = entry[warp][lane];
    int* own = stage + warp * W * (kTraceSteps + 1);
    const int n = len[mine], ends = ended[mine];
    for (int t1 = hi; t1 > lo; t1 -= kTraceSteps) {
        const int t0 = max(lo, t1 - kTraceSteps), steps = t1 - t0;
        int p[kTraceSteps], k[kTraceSteps];
#pragma unroll
        for (int i = 0; i < kTraceSteps; ++i) {
            const long long at = ((long long)(t1 - 1 - i) * B + b) * W + mine;
            p[i] = i < steps ? min(max(hist_parent[at], 0), W - 1) : 0;
            k[i] = i < steps ? hist_token[at] : 0;
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < kTraceSteps; ++i) {
            if (i >= steps) break;
            const int t = t1 - 1 - i;
            const int token = __shfl_sync(kFull, k[i], cur), next = __shfl_sync(kFull, p[i], cur);
            const bool inside = t <= t_in;
            if (lane < W) own[lane * (kTraceSteps + 1) + t - t0] = inside ? token : (int)(ends && t == n - 1 ? eos : pad);
            if (inside) cur = next;
        }
        __syncwarp();
        for (int i = lane; i < W * kTraceSteps; i += 32) {
            const int h = i / kTraceSteps, t = i % kTraceSteps;
            if (t < steps) tokens[(b * W + h) * step + t0 + t] = own[h * (kTraceSteps + 1) + t];
        }
        __syncwarp();
    }
    if (warp == 0 && lane < W) lengths[b * W + lane] = n;
}

// Values a thread of the first kernel takes: 32, or 8 where the rows are so few that longer chunks leave SMs idle.
int values_per_thread(long long rows, int W, int V) {
    const bool few = rows * ((V + 8191) / 8192) < 2LL * nxd_num_sms();
    return few && (long long)W * ((V + 7 + 2047) / 2048) <= kMaxLists ? 8 : 32;
}

int splits_of(int V, int elem, int E) { return (V + 16 / elem - 1 + kRowThreads * E - 1) / (kRowThreads * E); }

template <typename T>
void launch_rows(int E, long long ctas, cudaStream_t s, const void* logits, int V, long long stride, int splits, int n, Lists out) {
    if (E == 8) beam_rows_kernel<T, 8><<<(unsigned)ctas, kRowThreads, 0, s>>>((const T*)logits, V, stride, splits, n, out);
    else beam_rows_kernel<T, 32><<<(unsigned)ctas, kRowThreads, 0, s>>>((const T*)logits, V, stride, splits, n, out);
}

}  // namespace

// Scratch of a call in floats, or 0 where the sizes are outside what is compiled.
NXD_API long long nxd_beam_select_scratch(int dtype, int B, int W, int V, int n) {
    if (dtype < 0 || dtype > 2 || B < 1 || W < 1 || W > kMaxBeams || V < 1 || n < 1 || n > kMaxN || (long long)W * V >= (1LL << 31) - 16 || n > (long long)W * V)
        return 0;
    const long long rows = (long long)B * W;
    const int splits = splits_of(V, dtype == 0 ? 4 : 2, values_per_thread(rows, W, V));
    if ((long long)W * splits > kMaxLists || rows * splits >= (1LL << 31)) return 0;
    return rows * splits * (2 + 2LL * n);
}

// logits [B * W, V] (0 fp32, 1 bf16, 2 fp16; rows `stride` elements apart), scores [B, W] -> the n best candidates of every group.
NXD_API int nxd_beam_select(int dtype, const void* logits, long long stride, const float* scores, int B, int W, int V, int n, float* scratch,
                            float* out_scores, long long* out_beams, long long* out_tokens, void* stream) {
    if (B == 0) return 0;
    NXD_REQUIRE(nxd_beam_select_scratch(dtype, B, W, V, n) > 0, "beam_select: %d beams of %d tokens, %d candidates are outside what is compiled", W, V, n);
    cudaStream_t s = (cudaStream_t)stream;
    const long long rows = (long long)B * W;
    const int E = values_per_thread(rows, W, V), splits = splits_of(V, dtype == 0 ? 4 : 2, E), lists = W * splits;
    const Lists l = lists_of(scratch, rows * splits, n);
    if (dtype == 0) launch_rows<float>(E, rows * splits, s, logits, V, stride, splits, n, l);
    else if (dtype == 1) launch_rows<bf16>(E, rows * splits, s, logits, V, stride, splits, n, l);
    else launch_rows<__half>(E, rows * splits, s, logits, V, stride, splits, n, l);
    NXD_LAUNCH_CHECK();
    const int room = lists > n * (n < lists ? n : lists) ? lists : n * (n < lists ? n : lists);
    const int smem = lists * 8 + room * 12;
    NXD_CHECK_CUDA(nxd_allow_smem<beam_join_kernel>(kMaxLists * 20));
    const int threads = lists > 256 || n > 16 ? 1024 : 256;
    beam_join_kernel<<<B, threads, smem, s>>>(scores, W, V, splits, n, l, out_scores, out_beams, out_tokens);
    NXD_LAUNCH_CHECK();
    return 0;
}

// One step of the books (the header has the arrays).
NXD_API int nxd_beam_advance(const float* cand_scores, const long long* cand_beams, const long long* cand_tokens, int B, int W, int N,
                             const float* running, const float* pool_scores, const int* pool_lengths, const int* pool_slots,
                             const unsigned char* done, float norm, long long eos, long long pad, int early_stopping, int length,
                             float* out_running, long long* out_tokens, long long* out_parents, float* out_pool_scores, int* out_pool_lengths,
                             int* out_pool_slots, unsigned char* out_done, int* hist_tokens, int* hist_parents, void* stream) {
    NXD_REQUIRE(W >= 1 && W <= kMaxBeams && N >= 1 && N <= kMaxN, "beam_advance: %d beams, %d candidates are outside what is compiled", W, N);
    if (B == 0) return 0;
    const Books in = {running, pool_scores, pool_lengths, pool_slots, done};
    beam_advance_kernel<<<(B + 3) / 4, 128, 0, (cudaStream_t)stream>>>(cand_scores, cand_beams, cand_tokens, B, W, N, in, norm, eos, pad, early_stopping,
                                                                      out_running, out_tokens, out_parents, out_pool_scores, out_pool_lengths,
                                                                      out_pool_slots, out_done, hist_tokens, hist_parents, length);
    NXD_LAUNCH_CHECK();
    return 0;
}

// The sequences of every group's best W hypotheses (the header has the arrays).
NXD_API int nxd_beam_finish(const float* running, const float* pool_scores, const int* pool_lengths, const int* pool_slots, const unsigned char* done,
                            int B, int W, int step, float norm, long long eos, long long pad, const int* hist_tokens, const int* hist_parents,
                            long long* tokens, long long* lengths, float* scores, void* stream) {
    NXD_REQUIRE(W >= 1 && W <= kMaxBeams && step >= 0, "beam_finish: %d beams, %d steps", W, step);
    if (B == 0) return 0;
    const Books in = {running, pool_scores, pool_lengths, pool_slots, done};
    const int warps = step <= kTraceSteps ? 1 : step >= 32 * kTraceSteps ? 32 : (step + kTraceSteps - 1) / kTraceSteps;
    const int smem = warps * W * (kTraceSteps + 1) * 4;
    NXD_CHECK_CUDA(nxd_allow_smem<beam_finish_kernel>(32 * kMaxBeams * (kTraceSteps + 1) * 4));
    beam_finish_kernel<<<B, warps * 32, smem, (cudaStream_t)stream>>>(in, W, B, step, norm, eos, pad, hist_tokens, hist_parents, tokens, lengths, scores);
    NXD_LAUNCH_CHECK();
    return 0;
}
