// Beam search for sm_100a: the choice of a step's candidates, the books of the beams, and the sequences at the end.
//
// Choice.  Of group b's beams w with running scores s[w] and logits x[w, v] the n best of s[w] + x[w, v] - log sum_u exp x[w, u], of equal
// ones the lowest w * V + v.  One pass over the logits: a CTA goes through a chunk of one row in rounds (512 threads x 4 vectors, 256 x 2 where
// rows are few), with its running maximum and sum of exponentials, and ends with the chunk's n best in order.  A second kernel joins the
// chunks of a group's rows.
//   The n best of a chunk: the n-th largest of a few maxima of every warp bounds the n-th largest value from below, so what is not below it is
// collected (about 1.3 n values of a round as a rule) and ranked by counting; later rounds look only at what is above the n-th so far.  Where that
// is too much (equal values in numbers, values that rise along the row, masks that leave a stretch of it) the rounds are gone through once more with
// the n-th largest of the threads' best, ties by their indices.
//   Scores are compared in 64 bits: sums of near size decide between rows.  Within a row the logits decide.  Threads have the same elements of every
// row, wherever it starts, so equal rows have equal sums and the lower of two equal beams comes first.
// Floor: the logits are read once, 65.7 MB (32 requests of 8 beams, 128256 tokens, bf16) are 10.0 us at 6555 GB/s.  Measured: 20.6 us for the rows and 4.1 for
// the join (rows of 128257, which start anywhere: 4 us more; rows in rising order, every round of which has too many: 181 in all).  Nothing is
// saturated in the rows: instructions are issued in 60 % of the cycles, DRAM stands at 35 %.  A warp waits 10.7 cycles an instruction: 2.1 for fixed
// latencies, 2.0 for shared memory, 1.7 at barriers (all CTAs put their candidates in order in the same rounds), 1.4 for its turn, 0.9 for memory; and 256
// rows on 148 SMs leave 14 % of them idle.  One request of 4 rows takes 3.8 and 5.0 us of latency.
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"

namespace {

constexpr int kMaxN = 64;
constexpr int kMaxBeams = 32;
constexpr int kMaxLists = 4096;          // chunks of a group
constexpr int kOwn = 2;                  // entries of a thread of the join where that is all (32 groups of 8 lists of 16: 4.4 us, by their heads 5.9; with four
                                         // entries, one group of 128 lists of 8: 5.6, by their heads 4.9)
constexpr int kStages = 2;               // rounds under way (3 leave one CTA an SM: 29 instead of 23 us for 256 rows of 128256 in all)
constexpr int kMany = 384;               // candidates that are all compared with each other (2048 rows of 500, 64 of them wanted: 158 us, with the search 84)
constexpr int kEasy = 512;               // candidates that are ranked without more ado
constexpr int kCollect = kMaxN + kMaxN * 32;          // that a CTA holds: those it keeps, and all values of n threads
constexpr unsigned kFull = 0xffffffffu;

// order-preserving keys; -0 and +0 are one value (the caller adds 0)
__device__ __forceinline__ uint32_t order_key(float f) {
    const uint32_t u = __float_as_uint(f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k); }
constexpr uint32_t kLowestKey = 0x00800000u;          // of the lowest finite number
// a value with its index, greater for greater values and of equal ones for lower indices
__device__ __forceinline__ unsigned long long entry_key(float f, int index) {
    return (unsigned long long)order_key(f + 0.f) << 32 | (uint32_t)~index;
}
// the same for 64 bits
__device__ __forceinline__ unsigned long long order_key(double d) {
    const unsigned long long u = (unsigned long long)__double_as_longlong(d + 0.0);
    return (u >> 63) ? ~u : (u | 1ull << 63);
}
__device__ __forceinline__ double key_value(unsigned long long k) { return __longlong_as_double((long long)((k >> 63) ? (k & ~(1ull << 63)) : ~k)); }
constexpr uint32_t kLowestKeyHi = 0x00100000u;          // the upper half of the lowest finite number's

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

// What a call leaves for the second kernel: per chunk its maximum, the sum of exponentials behind it, and n entries in order, 0 behind the last.
struct Lists {
    unsigned long long* entry;       // [rows, splits, n]
    float2* sum;                     // [rows, splits]: maximum, sum
};

__host__ __device__ inline Lists lists_of(void* scratch, long long lists, int n) {
    unsigned long long* entry = reinterpret_cast<unsigned long long*>(scratch);
    return {entry, reinterpret_cast<float2*>(entry + lists * n)};
}

// 16 bytes of logits
template <typename T> struct Vec { static constexpr int n = 16 / sizeof(T); };

template <typename T> __device__ __forceinline__ uint32_t bits_of(T x);
template <> __device__ __forceinline__ uint32_t bits_of<float>(float x) { return __float_as_uint(x); }
template <> __device__ __forceinline__ uint32_t bits_of<bf16>(bf16 x) { return __bfloat16_as_ushort(x); }
template <> __device__ __forceinline__ uint32_t bits_of<__half>(__half x) { return __half_as_ushort(x); }

template <typename T>
__device__ __forceinline__ uint4 load_vec(const T* row, int at, int V) {
    if (at >= 0 && at + Vec<T>::n <= V) return __ldg(reinterpret_cast<const uint4*>(row + at));
    // over an end of the row: its elements one by one, -inf outside
    constexpr uint32_t kOut = sizeof(T) == 4 ? 0xff800000u : std::is_same_v<T, bf16> ? 0xff80u : 0xfc00u, kAll = sizeof(T) == 4 ? kOut : kOut << 16 | kOut;
    if (at >= V) return make_uint4(kAll, kAll, kAll, kAll);
    constexpr int kBits = 8 * sizeof(T);
    unsigned long long lo = 0, hi = 0;
#pragma unroll 1
    for (int j = Vec<T>::n - 1; j >= 0; --j) {
        const int k = at + j;
        hi = hi << kBits | lo >> (64 - kBits);
        lo = lo << kBits | (k >= 0 && k < V ? bits_of<T>(row[k]) : kOut);
    }
    return make_uint4((uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32));
}

// Rows start anywhere, threads have the same elements of every row all the same, so that equal rows come to equal sums.  In memory a thread's vector
// then lies in two of the 16-byte ones, `mis` elements behind the start of the first.
template <typename T>
__device__ __forceinline__ uint4 join_vecs(const uint4& a, const uint4& b, int mis) {
    const int bytes = mis * (int)sizeof(T), bits = bytes % 4 * 8;          // the same for the whole block
    switch (bytes / 4) {
        case 0: return make_uint4(__funnelshift_r(a.x, a.y, bits), __funnelshift_r(a.y, a.z, bits), __funnelshift_r(a.z, a.w, bits), __funnelshift_r(a.w, b.x, bits));
        case 1: return make_uint4(__funnelshift_r(a.y, a.z, bits), __funnelshift_r(a.z, a.w, bits), __funnelshift_r(a.w, b.x, bits), __funnelshift_r(b.x, b.y, bits));
        case 2: return make_uint4(__funnelshift_r(a.z, a.w, bits), __funnelshift_r(a.w, b.x, bits), __funnelshift_r(b.x, b.y, bits), __funnelshift_r(b.y, b.z, bits));
        default: return make_uint4(__funnelshift_r(a.w, b.x, bits), __funnelshift_r(b.x, b.y, bits), __funnelshift_r(b.y, b.z, bits), __funnelshift_r(b.z, b.w, bits));
    }
}
template <typename T>
__device__ __forceinline__ uint4 load_elements(const T* row, int at, int V, int mis) {
    const uint4 a = load_vec<T>(row, at - mis, V);
    return mis == 0 ? a : join_vecs<T>(a, load_vec<T>(row, at - mis + Vec<T>::n, V), mis);
}

__device__ __forceinline__ void fetch_vec(uint4* to, const void* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from) : "memory");
}

// A round in shared memory: 33 vectors a warp and vector of its threads, of which the last is the next warp's first.
constexpr int kStagePitch = 33;

// A thread's vectors of a round on their way there (one group of copies; the ends of a row are stored at once).  Whether a round lies
// inside the row the block decides at once.  Of a row that starts on 16 bytes nobody reads the 33rd ones.
template <typename T, int NT, int NV>
__device__ __forceinline__ void fetch_round(uint4* stage, const T* row, int first, int V, int mis) {
    constexpr int VE = Vec<T>::n, kWarps = NT / 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, more = mis != 0 ? VE : 0;
    stage += warp * kStagePitch + lane;
    first -= mis;
    const int begin = first - (int)threadIdx.x * VE;
    if (begin >= 0 && begin + NT * NV * VE + more <= V) {
#pragma unroll
        for (int i = 0; i < NV; ++i) fetch_vec(stage + i * kWarps * kStagePitch, row + first + i * NT * VE);
        if (mis != 0 && lane == 31) {
#pragma unroll
            for (int i = 0; i < NV; ++i) fetch_vec(stage + i * kWarps * kStagePitch + 1, row + first + i * NT * VE + VE);
        }
        return;
    }
    auto fetch = [&](uint4* to, int at) {
        if (at >= 0 && at + VE <= V) fetch_vec(to, row + at);
        else *to = load_vec<T>(row, at, V);
    };
#pragma unroll 1
    for (int i = 0; i < NV; ++i, first += NT * VE, stage += kWarps * kStagePitch) {
        fetch(stage, first);
        if (mis != 0 && lane == 31) fetch(stage + 1, first + VE);
    }
}
__device__ __forceinline__ void fetch_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void fetch_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// A 32-bit word's one or two values.
template <typename T>
__device__ __forceinline__ void unpack_word(uint32_t w, float* f) {
    if constexpr (sizeof(T) == 4) {
        f[0] = __uint_as_float(w);
    } else if constexpr (std::is_same_v<T, bf16>) {
        f[0] = __uint_as_float(w << 16);
        f[1] = __uint_as_float(w & 0xffff0000u);
    } else {
        f[0] = __half2float(__ushort_as_half((unsigned short)(w & 0xffffu)));
        f[1] = __half2float(__ushort_as_half((unsigned short)(w >> 16)));
    }
}

template <typename T>
__device__ __forceinline__ void unpack_vec(const uint4& raw, float* f) {
    constexpr int per = Vec<T>::n / 4;
    unpack_word<T>(raw.x, f);
    unpack_word<T>(raw.y, f + per);
    unpack_word<T>(raw.z, f + 2 * per);
    unpack_word<T>(raw.w, f + 3 * per);
}

// What a word's values are above `base`: one instruction a 16-bit value, conversion and difference.
template <typename T>
__device__ __forceinline__ void above_word(uint32_t w, float base, float* d) {
    if constexpr (sizeof(T) == 4)
        d[0] = __uint_as_float(w) - base;
    else if constexpr (std::is_same_v<T, bf16>)
        asm("{.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tsub.f32.bf16 %0, lo, %3;\n\tsub.f32.bf16 %1, hi, %3;}" : "=f"(d[0]), "=f"(d[1]) : "r"(w), "f"(base));
    else
        asm("{.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tsub.f32.f16 %0, lo, %3;\n\tsub.f32.f16 %1, hi, %3;}" : "=f"(d[0]), "=f"(d[1]) : "r"(w), "f"(base));
}

template <typename T>
__device__ __forceinline__ uint32_t max_word(uint32_t a, uint32_t b) {
    uint32_t r;
    if constexpr (sizeof(T) == 4) r = __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
    else if constexpr (std::is_same_v<T, bf16>) asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// The largest of a thread's values, of NaN and a number the number.
template <typename T, int NV>
__device__ __forceinline__ float max_of(const uint4 (&raw)[NV]) {
    uint32_t m = max_word<T>(max_word<T>(raw[0].x, raw[0].y), max_word<T>(raw[0].z, raw[0].w));
#pragma unroll
    for (int i = 1; i < NV; ++i) m = max_word<T>(m, max_word<T>(max_word<T>(raw[i].x, raw[i].y), max_word<T>(raw[i].z, raw[i].w)));
    float f[2] = {-INFINITY, -INFINITY};
    unpack_word<T>(m, f);
    return fmaxf(fmaxf(f[0], f[1]), -INFINITY);
}

// The k-th largest key of a warp (0 where fewer threads have one).
__device__ __forceinline__ uint32_t kth_of_warp(uint32_t key, int k, int lane) {
    uint32_t v = 0;
    for (int i = 0; i < k; ++i) {
        v = __reduce_max_sync(kFull, key);
        if (lane == __ffs(__ballot_sync(kFull, key == v)) - 1) key = 0;
    }
    return v;
}

// A round that has more values above the bound than are ranked easily: equal ones, or many in few threads.  The n-th largest of the threads' best
// entries, found bit by bit (entries differ, so it is one thread's), has n entries that are not below it, all of them in n threads: what is collected
// behind the `have` candidates fits.  Reads the round's values once more.
template <typename T, int NT, int NV>
__device__ __noinline__ int collect_carefully(const T* row, int first, int V, int mis, int n, int have, float floor, unsigned long long* cand, int* s_count) {
    constexpr int VE = Vec<T>::n;
    uint4 raw[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) raw[i] = load_elements<T>(row, first + i * NT * VE, V, mis);
    unsigned long long best = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        float f[VE];
        unpack_vec<T>(raw[i], f);
#pragma unroll
        for (int j = 0; j < VE; ++j)
            if (f[j] > floor) best = max(best, entry_key(f[j], first + i * NT * VE + j));
    }
    if (threadIdx.x == 0) *s_count = have;
    unsigned long long least = 0;
    int count = __syncthreads_count(best > 0);
    for (int bit = 63; bit >= 0 && count > n; --bit) {
        const unsigned long long c = least | 1ull << bit;
        const int above = __syncthreads_count(best >= c);
        if (above >= n) least = c, count = above;
    }
    least = max(least, 1ull);
    if (best >= least) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float f[VE];
            unpack_vec<T>(raw[i], f);
#pragma unroll
            for (int j = 0; j < VE; ++j) {
                const unsigned long long e = entry_key(f[j], first + i * NT * VE + j);
                if (f[j] > floor && e >= least) cand[atomicAdd(s_count, 1)] = e;
            }
        }
    }
    __syncthreads();
    return *s_count;
}

// A CTA takes `rounds` rounds of NT threads x NV vectors of one row.  It keeps candidates, at least the n best so far; only values above the n-th of
// those, when they were last put in order, are looked at further.
template <typename T, int NT, int NV>
__global__ void __launch_bounds__(NT, 1024 / NT) beam_rows_kernel(const T* __restrict__ logits, int V, long long stride, int splits, int rounds, int n,
                                                                   Lists out) {
    constexpr int VE = Vec<T>::n, E = NV * VE, kWarps = NT / 32;
    __shared__ unsigned long long cand[kCollect];
    constexpr int kStage = NV * kWarps * kStagePitch;
    extern __shared__ uint4 ring[];            // [kStages][NV][kWarps][kStagePitch]
    __shared__ unsigned char looker[kWarps][32];
    __shared__ uint32_t warp_top[kWarps], bound_keys[2 * kMaxN];
    __shared__ float warp_sum_of[kWarps];
    __shared__ unsigned long long best[kMaxN];
    __shared__ int s_count;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const long long list = blockIdx.x;
    const int split = (int)(list % splits);
    const T* row = logits + (list / splits) * stride;
    // loads start on 16 bytes: the row's first element is element `mis` of the first vector
    const int mis = (int)((reinterpret_cast<uintptr_t>(row) / sizeof(T)) % VE);
    int first = split * rounds * (NT * E) + tid * VE;          // index of this thread's first element of the round

    if (tid == 0) s_count = 0;
#pragma unroll
    for (int q = 0; q < kStages - 1; ++q) {
        if (q < rounds) fetch_round<T, NT, NV>(ring + q * kStage, row, first + q * (NT * E), V, mis);
        fetch_commit();
    }
    float top = -INFINITY, sum = 0.f;          // this thread's
    float floor = -INFINITY;                   // only what is above it counts
    int until = 1;                             // the next round that puts the candidates in order
    int since = 0, kept = 0;                   // the first round since, and what was kept then
    float kept_floor = -INFINITY;
    // the n best candidates in order; eight lanes compare one with all, of many only the n best, found bit by bit
    auto keep_best = [&](int count) {
        if (count > kMany && count > 2 * n) {
            unsigned long long least = 0;
            int above = count;
            for (int bit = 63; bit >= 0 && above > n; --bit) {
                const unsigned long long c = least | 1ull << bit;
                int now = 0;
                for (int i = tid; i - tid < count; i += NT) now += __syncthreads_count(i < count && cand[i] >= c);
                if (now >= n) least = c, above = now;
            }
            if (tid == 0) s_count = 0;
            __syncthreads();
            for (int i = tid; i < count; i += NT) {
                const unsigned long long e = cand[i];
                if (e >= least) best[atomicAdd(&s_count, 1)] = e;
            }
            __syncthreads();
            if (tid < n) cand[tid] = best[tid];
            count = n;
            __syncthreads();
        }
        for (int i0 = warp * 4; i0 < count; i0 += NT / 8) {
            const int i = i0 + lane / 8;
            const unsigned long long own = i < count ? cand[i] : ~0ull;
            int before = 0;
#pragma unroll 4
            for (int j = tid % 8; j < count; j += 8) before += cand[j] > own;
            before += __shfl_xor_sync(kFull, before, 1);
            before += __shfl_xor_sync(kFull, before, 2);
            before += __shfl_xor_sync(kFull, before, 4);
            if (i < count && before < n && tid % 8 == 0) best[before] = own;
        }
        count = min(count, n);
        __syncthreads();
        if (tid < count) cand[tid] = best[tid];
        if (tid == 0) s_count = count;
        __syncthreads();
        kept = count;
        floor = kept_floor = count == n ? key_value((uint32_t)(best[n - 1] >> 32)) : -INFINITY;
    };
    for (int r = 0; r < rounds; ++r) {
        const uint4* stage = ring + r % kStages * kStage + warp * kStagePitch;          // this warp's
        fetch_wait<kStages - 2>();
        uint4 raw[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) raw[i] = stage[i * kWarps * kStagePitch + lane];
        if (mis != 0) {
            __syncwarp();
#pragma unroll
            for (int i = 0; i < NV; ++i) raw[i] = join_vecs<T>(raw[i], stage[i * kWarps * kStagePitch + lane + 1], mis);
        }
        // into the round before, which the warp is done with; not with the first ones, which would arrive later for it
        if (r + kStages - 1 < rounds)
            fetch_round<T, NT, NV>(ring + (r + kStages - 1) % kStages * kStage, row, first + (kStages - 1) * (NT * E), V, mis);
        fetch_commit();
        float m = max_of<T, NV>(raw) + 0.f;          // no -0; passes NaN by
        {
            // the differences first: a product of the maximum would lose their last bits.  A NaN, or an infinity, makes the sum NaN
            const float big = fmaxf(top, m), base = big == -INFINITY ? 0.f : big;
            if (top != -INFINITY) sum *= exp2_approx((top - base) * kLog2e);
            top = big;
            const uint64_t one = f2_pack(1.f, 1.f), log2e = f2_pack(kLog2e, kLog2e);
            uint64_t part[2] = {0, 0};
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                constexpr int per = VE / 4;
                float f[VE];
                above_word<T>(raw[i].x, base, f);
                above_word<T>(raw[i].y, base, f + per);
                above_word<T>(raw[i].z, base, f + 2 * per);
                above_word<T>(raw[i].w, base, f + 3 * per);
#pragma unroll
                for (int j = 0; j < VE; j += 2) {
                    const uint64_t d = f2_mul(f2_pack(f[j], f[j + 1]), log2e);
                    part[j / 2 % 2] = f2_fma(f2_pack(exp2_approx(f2_lo(d)), exp2_approx(f2_hi(d))), one, part[j / 2 % 2]);
                }
            }
            sum += (f2_lo(part[0]) + f2_hi(part[0])) + (f2_lo(part[1]) + f2_hi(part[1]));
        }
        if (r == 0) {
            // the largest maxima of each warp that has values, 2 n of them: the n-th of those (of more than 32 its upper 16 bits) has n values that are not
            // below it.  One warp has 32 at most: where more candidates are wanted nothing is known
            const int vecs = (V - split * rounds * (NT * E) + VE - 1) / VE, filled = min(max((vecs + 31) / 32, 1), kWarps);
            const int per = min((2 * n + filled - 1) / filled, min(2 * kMaxN / filled, 32)), keys = filled * per;
            uint32_t key = order_key(m);
            for (int i = 0; i < per; ++i) {
                const uint32_t v = __reduce_max_sync(kFull, key);
                if (lane == __ffs(__ballot_sync(kFull, key == v)) - 1) key = 0;
                if (lane == 0 && warp < filled) bound_keys[warp * per + i] = v;
            }
            __syncthreads();
            uint32_t least = 0;
            if (keys <= 32) {
                const uint32_t own = lane < keys ? bound_keys[lane] : 0;
                int before = 0;
#pragma unroll
                for (int j = 0; j < 32; ++j) before += __shfl_sync(kFull, own, j) > own;
                if (n <= keys) least = __reduce_min_sync(kFull, before < n ? own : kFull);
            } else {
                uint32_t own[2 * kMaxN / 32];
#pragma unroll
                for (int q = 0; q < 2 * kMaxN / 32; ++q) own[q] = q * 32 + lane < keys ? bound_keys[q * 32 + lane] : 0;
                for (int bit = 31; bit >= 16; --bit) {
                    const uint32_t c = least | 1u << bit;
                    int mine = 0;
#pragma unroll
                    for (int q = 0; q < 2 * kMaxN / 32; ++q) mine += own[q] >= c;
                    if (__reduce_add_sync(kFull, mine) >= n) least = c;
                }
            }
            // the number below that bound (below zero one that is not equal to it), so that what is above it is looked at in every round
            least = max(least, kLowestKey) - 1;
            floor = key_value(least == 0x7fffffffu ? least - 1 : least);
        }
        // the values of the threads that have some are looked at by their warp
        const bool look = m > floor;
        const unsigned lookers = __ballot_sync(kFull, look);
        if (lookers != 0) {
            if (look) looker[warp][__popc(lookers & ((1u << lane) - 1u))] = (unsigned char)lane;
            __syncwarp();
            for (int e = lane; e < __popc(lookers) * E; e += 32) {
                const int who = looker[warp][e / E], i = e % E / VE, j = e % VE;
                const float f = to_float<T>(reinterpret_cast<const T*>(stage + i * kWarps * kStagePitch + who)[mis + j]);
                if (f > floor) {
                    const int to = atomicAdd(&s_count, 1);
                    if (to < kCollect) cand[to] = entry_key(f, first + (who - lane) * VE + i * NT * VE + j);
                }
            }
            __syncwarp();
        }
        if (r == until || r + 1 == rounds) {
            __syncthreads();
            const int count = s_count;
            if (count <= kEasy) {
                keep_best(count);
            } else {          // the rounds since the last time once more, one by one
                __syncthreads();
                floor = kept_floor;
                for (int q = since; q <= r; ++q) keep_best(collect_carefully<T, NT, NV>(row, first - (r - q) * (NT * E), V, mis, n, kept, floor, cand, &s_count));
            }
            since = r + 1;
            until = 4 * r + 3;          // 1, 7, 31: at most 3 n or so pass the bound between these
        }
        first += NT * E;
    }
    pdl_trigger();
    const uint32_t block_key = __reduce_max_sync(kFull, order_key(top));
    if (lane == 0) warp_top[warp] = block_key;
    __syncthreads();
    uint32_t most = warp_top[0];
#pragma unroll
    for (int i = 1; i < kWarps; ++i) most = max(most, warp_top[i]);
    const float all = key_value(most);
    if (top != -INFINITY) sum *= exp2_approx((top - all) * kLog2e);
    sum = warp_sum(sum);
    if (lane == 0) warp_sum_of[warp] = sum;
    __syncthreads();
    if (tid == 0) {
        float total = 0.f;
#pragma unroll
        for (int i = 0; i < kWarps; ++i) total += warp_sum_of[i];
        out.sum[list] = make_float2(all, total);
    }
    if (tid < n) out.entry[list * n + tid] = tid < s_count ? cand[tid] : 0;
}

// The rank of an entry among `count` of them, by the eight lanes around it: greater scores (as keys) first, of equal ones the lower order.
__device__ __forceinline__ int rank_by_eight(const unsigned long long* score, const int* order, int count, unsigned long long s, int o) {
    int before = 0;
#pragma unroll 4
    for (int j = threadIdx.x % 8; j < count; j += 8) before += (int)(score[j] > s) | ((int)(score[j] == s) & (int)(order[j] < o));
    before += __shfl_xor_sync(kFull, before, 1);
    before += __shfl_xor_sync(kFull, before, 2);
    before += __shfl_xor_sync(kFull, before, 4);
    return before;
}

// One CTA joins the lists of one group's rows: up to two entries a thread are all looked at.  Of more, every list being in order, its head is
// its best: the n lists with the best heads hold the n best values, and none of those is below the n-th head.
__global__ void __launch_bounds__(1024, 1) beam_join_kernel(const float* __restrict__ scores, int W, int V, int splits, int n, int room, Lists in,
                                                            float* __restrict__ out_scores, long long* __restrict__ out_beams,
                                                            long long* __restrict__ out_tokens) {
    extern __shared__ unsigned long long smem[];
    __shared__ double so_far[kMaxBeams], lse[kMaxBeams];
    __shared__ uint32_t kth_of[2][32];
    __shared__ int sel[kMaxN];
    __shared__ int s_count, s_heads;
    __shared__ unsigned char used[2 * kMaxN];
    const int lists = W * splits;
    unsigned long long* cand = smem;                         // [room], keys of scores
    unsigned long long* head = cand + room;                  // [lists]
    int* cand_i = reinterpret_cast<int*>(head + lists);      // [room]
    int* list_of = cand_i + room;                            // [lists]
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nth = blockDim.x, warps = nth >> 5;
    const long long g = blockIdx.x, l0 = g * lists;
    if (tid == 0) s_count = s_heads = 0;
    if (tid < 2 * kMaxN) used[tid] = 0;
    pdl_wait();
    // what a thread reads first: up to kOwn entries around the warps if that is all of them, else the head of its first list
    const bool all = lists * n <= kOwn * nth;
    auto place = [&](int q) { return q * nth + lane * warps + (warp + lane & warps - 1); };          // every warp has heads of lists
    unsigned long long first[kOwn];
#pragma unroll
    for (int q = 0; q < kOwn; ++q) {
        const int e = all ? place(q) : lane * warps + warp;
        first[q] = all ? (e < lists * n ? in.entry[l0 * n + e] : 0) : q == 0 && e < lists ? in.entry[(l0 + e) * n] : 0;
    }
    for (int w = warp; w < W; w += warps) {
        const float2* part = in.sum + l0 + (long long)w * splits;
        const float own = scores[g * W + w];
        const float2 mine = lane < splits ? part[lane] : make_float2(-INFINITY, 0.f);
        float top = mine.x;
        for (int i = lane + 32; i < splits; i += 32) top = fmaxf(top, part[i].x);
        top = warp_max(top);
        double sum = mine.x == -INFINITY ? (double)mine.y : (double)mine.y * exp((double)mine.x - (double)top);
        for (int i = lane + 32; i < splits; i += 32) {
            const float2 p = part[i];
            sum += p.x == -INFINITY ? (double)p.y : (double)p.y * exp((double)p.x - (double)top);
        }
        for (int o = splits > 16 ? 16 : splits > 1 ? 8 : 0; o > 0; o >>= 1) sum += __shfl_xor_sync(kFull, sum, o);
        // a row with NaN, with +inf or without a finite logit has no candidates
        if (lane == 0) {
            so_far[w] = sum > 0.0 && own > -INFINITY ? (double)own : -INFINITY;
            lse[w] = sum > 0.0 ? (double)top + log(sum) : 0.0;
        }
    }
    __syncthreads();
    auto score_of = [&](unsigned long long entry, int w) -> unsigned long long {          // as a key, that of -inf where there is none
        return order_key(entry != 0 && so_far[w] > -INFINITY ? so_far[w] + ((double)key_value((uint32_t)(entry >> 32)) - lse[w]) : -INFINITY);
    };
    // of its threads' best each warp has a k-th largest, warps * k >= n: the least of those has n scores that are not below it
    const int k = (n + warps - 1) / warps;
    auto bound = [&](uint32_t own, uint32_t* kth_of) {
        const uint32_t kth = kth_of_warp(own, k, lane);
        if (lane == 0) kth_of[warp] = kth;
        __syncthreads();
        return max(__reduce_min_sync(kFull, lane < warps ? kth_of[lane] : kFull), kLowestKeyHi);
    };
    int count;
    if (all) {
        uint32_t own = 0;
#pragma unroll
        for (int q = 0; q < kOwn; ++q) {
            const int e = place(q);
            if (e < lists * n) own = max(own, (uint32_t)(score_of(first[q], e / n / splits) >> 32));
        }
        const uint32_t floor = bound(own, kth_of[0]);
#pragma unroll
        for (int q = 0; q < kOwn; ++q) {
            const int e = place(q);
            if (e < lists * n) {
                const unsigned long long s = score_of(first[q], e / n / splits);
                if ((uint32_t)(s >> 32) >= floor) {
                    const int at = atomicAdd(&s_count, 1);
                    cand[at] = s;
                    cand_i[at] = e / n / splits * V + (int)~(uint32_t)first[q];
                }
            }
        }
        __syncthreads();
        count = s_count;
    } else {
        uint32_t own = 0;
        for (int l = lane * warps + warp; l < lists; l += nth) {
            const unsigned long long h = score_of(l < nth ? first[0] : in.entry[(l0 + l) * n], l / splits);
            head[l] = h;
            own = max(own, (uint32_t)(h >> 32));
        }
        uint32_t floor = bound(own, kth_of[0]);
        for (int l = tid; l < lists; l += nth)
            if ((uint32_t)(head[l] >> 32) >= floor) list_of[atomicAdd(&s_heads, 1)] = l;
        __syncthreads();
        const int heads = s_heads;
        // what these lists hold, around the warps again, bounds the n-th score once more
        own = 0;
        for (int e = lane * warps + warp; e < heads * n; e += nth) {
            const int l = list_of[e / n];
            own = max(own, (uint32_t)(score_of(in.entry[(l0 + l) * n + e % n], l / splits) >> 32));
        }
        floor = max(floor, bound(own, kth_of[1]));
        auto take = [&](int l, int e, unsigned long long least) {
            const unsigned long long entry = in.entry[(l0 + l) * n + e], s = score_of(entry, l / splits);
            if (s >= least) {
                const int at = atomicAdd(&s_count, 1);
                if (at < room) {
                    cand[at] = s;
                    cand_i[at] = l / splits * V + (int)~(uint32_t)entry;
                }
            }
        };
        for (int e = lane * warps + warp; e < heads * n; e += nth) take(list_of[e / n], e % n, (unsigned long long)floor << 32);
        __syncthreads();
        count = s_count;
        if (count > room) {
            // equal scores in numbers: of the lists only the n with the best heads (those of a row are in the order of the lists), and nothing below
            // the n-th head
            for (int i0 = 0; i0 < heads; i0 += nth) {
                if (i0 + tid < heads) cand[i0 + tid] = head[list_of[i0 + tid]];
            }
            __syncthreads();
            for (int i0 = 0; i0 < heads; i0 += nth / 8) {
                const int i = i0 + tid / 8;
                const int r = rank_by_eight(cand, list_of, heads, i < heads ? cand[i] : 0, i < heads ? list_of[i] : 0);
                if (i < heads && r < n && tid % 8 == 0) sel[r] = list_of[i];
            }
            if (tid == 0) s_count = 0;
            __syncthreads();
            const int picked = min(heads, n);
            const unsigned long long least = max(heads >= n ? head[sel[n - 1]] : 0ull, (unsigned long long)kLowestKeyHi << 32);
            for (int e = tid; e < picked * n; e += nth) take(sel[e / n], e % n, least);
            __syncthreads();
            count = s_count;
        }
    }
    for (int i0 = 0; i0 < count; i0 += nth / 8) {
        const int i = i0 + tid / 8;
        const unsigned long long s = i < count ? cand[i] : 0;
        const int o = i < count ? cand_i[i] : 0;
        const int r = rank_by_eight(cand, cand_i, count, s, o);
        if (i < count && tid % 8 == 0) {
            if (r < n) {
                const int w = o / V;
                out_scores[g * n + r] = (float)key_value(s);
                out_beams[g * n + r] = w;
                out_tokens[g * n + r] = o - w * V;
            }
            if (count < n && o < 2 * kMaxN) used[o] = 1;
        }
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

constexpr int kBatch = 8;                    // reads under way
constexpr int kSections = 32;                // of a CTA
constexpr int kFinishThreads = 512;
constexpr int kFinishCluster = 8;            // CTAs of a group at most
constexpr int kFinishBytes = 100 * 1024;     // of shared memory: a byte a step and line, and where they fit their tokens

__host__ __device__ inline int token_pitch(int W) { return W | 1; }          // words a step: lanes of consecutive steps in different banks

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

__device__ __forceinline__ void store_of_rank(unsigned char* p, int rank, int v) {          // to the same place in a CTA of the cluster
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    asm volatile("st.shared::cluster.u8 [%0], %1;" ::"r"(at), "r"(v) : "memory");
}

// The beams of requests that are not over join the pool, and every place's tokens are found from the last one back.  A line's history is a
// chain of parents.  A cluster of CTAs has a group, each a span of its steps: the parents are brought into shared memory as bytes, with the tokens
// on their way behind them; a section of the span is walked for all lines at once (lane w starts in line w at the section's end; a warp has as many
// sections as it has room for lines); the sections are joined within a CTA, the spans across the cluster; then they are walked once
// more, which leaves the line of every place at every step where the parents were.
//   Latency bounds it, of the chain and of rows that are a few bytes each: 2000 steps of 8 lines in 64 groups 181 ms with an operation a step, 21 us with
// one CTA a group, 12 us with four (16 MB: 2.5 us at 6555 GB/s).
__global__ void __launch_bounds__(kFinishThreads) beam_finish_kernel(Books in, int W, int B, int step, int span, float norm, long long eos, long long pad,
                                                                     const int* __restrict__ hist_token, const int* __restrict__ hist_parent,
                                                                     long long* __restrict__ tokens, long long* __restrict__ lengths,
                                                                     float* __restrict__ scores, unsigned char* __restrict__ scratch, int staged) {
    extern __shared__ int finish_smem[];          // tokens [span][token_pitch] if staged, then the path [span][W] unless scratch is there
    __shared__ int enter_at[kMaxBeams], enter_slot[kMaxBeams], len[kMaxBeams], ended[kMaxBeams];
    __shared__ unsigned char through[kSections][32], part[kSections][32], entry[kSections][32];
    __shared__ unsigned char span_through[kFinishCluster][32], span_part[kFinishCluster][32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nth = blockDim.x;
    const int rank = blockIdx.x, ranks = gridDim.x;          // the cluster is a row of the grid
    // here a CTA says that it runs; the wait for the others' word stands before the first store into their shared memory
    if (ranks > 1) cluster_arrive();
    const long long b = blockIdx.y;
    const int pitch = token_pitch(W), first = rank * span, steps = max(min(span, step - first), 0);          // t counts from `first`
    unsigned char* path = scratch != nullptr ? scratch + (b * step + first) * W : reinterpret_cast<unsigned char*>(finish_smem + (staged ? span * pitch : 0));
    // a line in 2^shift lanes: lane w of them has line w
    const int shift = W <= 1 ? 0 : 32 - __clz(W - 1), wide = 1 << shift, w = lane & (wide - 1);
    const bool used = w < W;
    float old_score = -INFINITY, own_score = -INFINITY;
    int old_length = 0, old_slot = 0;
    bool over = false;
    if (warp == 0 && lane < W) {
        const long long at = b * W + lane;
        old_score = in.pool_score[at], own_score = in.running[at], old_length = in.pool_length[at], old_slot = in.pool_slot[at];
        over = in.done[b];
    }
    {
        const int apart = nth >> shift;
        for (int t0 = tid >> shift; t0 < steps; t0 += kBatch * apart) {
            int p[kBatch];
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                const int t = t0 + k * apart;
                const long long at = ((long long)(first + t) * B + b) * W + w;
                p[k] = used && t < steps ? hist_parent[at] : 0;
                if (staged && used && t < steps)
                    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"((uint32_t)__cvta_generic_to_shared(finish_smem + t * pitch + w)),
                                 "l"(hist_token + at) : "memory");
            }
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                const int t = t0 + k * apart;
                if (used && t < steps) path[t * W + w] = (unsigned char)min(max(p[k], 0), W - 1);
            }
        }
        fetch_commit();
    }
    if (warp == 0) {
        const float r = over ? -INFINITY : __fdiv_rn(own_score, norm), c = r == r ? r : -INFINITY;
        int ra, rb;
        merge_ranks(old_score, c, W, lane, ra, rb);
        if (lane < W && ra < W) {
            const int n = old_score > -INFINITY ? min(max(old_length, 0), step) : 0;
            len[ra] = n;
            ended[ra] = 1;
            enter_at[ra] = n - 2;            // the last token is the one that ends
            enter_slot[ra] = min(max(old_slot, 0), W - 1);
            if (rank == 0) scores[b * W + ra] = old_score, lengths[b * W + ra] = n;
        }
        if (lane < W && rb < W) {
            const int n = c > -INFINITY ? step : 0;
            len[rb] = n;
            ended[rb] = 0;
            enter_at[rb] = n - 1;
            enter_slot[rb] = lane;
            if (rank == 0) scores[b * W + rb] = c, lengths[b * W + rb] = n;
        }
    }
    __syncthreads();
    const int sections = max(min(min(kSections, (steps + 15) / 16), (nth >> 5) << (5 - shift)), 1), section = (steps + sections - 1) / sections;
    const int mine = used ? w : 0, sec = (warp << (5 - shift)) + (lane >> shift), t_in = enter_at[mine] - first;
    const bool walks = warp << (5 - shift) < sections;
    const int lo = sec * section;
    // the parents of steps that a section has not are its lanes' own lines
    auto fetch = [&](int (&p)[kBatch], int at) {
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            const int t = lo + section - 1 - at - k;
            p[k] = used && t >= lo && t < steps ? path[t * W + w] : w;
        }
    };
    if (walks) {
        int line = w, cur = enter_slot[mine];
        for (int at = 0; at < section; at += kBatch) {
            int p[kBatch];
            fetch(p, at);
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                line = __shfl_sync(kFull, p[k], line, wide);
                const int next = __shfl_sync(kFull, p[k], cur, wide);
                if (lo + section - 1 - at - k <= t_in) cur = next;
            }
        }
        if (sec < sections) through[sec][w] = (unsigned char)line, part[sec][w] = (unsigned char)cur;
    }
    __syncthreads();
    // of lane w: where line w of the span's end comes from, and place w if it enters the span
    auto join = [&](int t, int cur, bool keep) {
        for (int k = sections - 1; k >= 0; --k) {
            if (keep) entry[k][lane] = (unsigned char)cur;
            if (t >= min((k + 1) * section, steps)) cur = through[k][cur];             // entered above this section
            else if (t >= k * section) cur = part[k][lane];
        }
        return cur;
    };
    const int own_in = lane < W ? enter_at[lane] : -1;
    int cur = lane < W ? enter_slot[lane] : 0;
    if (ranks > 1) {
        cluster_wait();
        if (warp == 0 && lane < W) {
            int line = lane;
            for (int k = sections - 1; k >= 0; --k) line = through[k][line];
            const int place = join(own_in - first, cur, false);
            for (int r = 0; r < ranks; ++r) {
                store_of_rank(&span_through[rank][lane], r, line);
                store_of_rank(&span_part[rank][lane], r, place);
            }
        }
        __syncwarp();
        cluster_arrive();
        cluster_wait();
        if (warp == 0 && lane < W) {
            for (int r = ranks - 1; r > rank; --r) {
                if (own_in >= (r + 1) * span) cur = span_through[r][cur];
                else if (own_in >= r * span) cur = span_part[r][lane];
            }
        }
    }
    if (warp == 0 && lane < W) join(own_in - first, cur, true);
    __syncthreads();
    if (walks) {
        cur = sec < sections ? entry[sec][mine] : 0;
        for (int at = 0; at < section; at += kBatch) {
            int p[kBatch];
            fetch(p, at);
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                const int t = lo + section - 1 - at - k;
                const int next = __shfl_sync(kFull, p[k], cur, wide);
                if (used && t >= lo && t < steps) path[t * W + w] = (unsigned char)cur;
                if (t <= t_in) cur = next;
            }
        }
    }
    fetch_wait<0>();
    __syncthreads();
    for (int t = tid; t < steps; t += nth) {
        for (int h0 = 0; h0 < W; h0 += kBatch) {
            int token[kBatch];
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                token[k] = 0;
                if (h0 + k < W && first + t <= enter_at[h0 + k]) {
                    const int line = path[t * W + h0 + k];
                    token[k] = staged ? finish_smem[t * pitch + line] : hist_token[((long long)(first + t) * B + b) * W + line];
                }
            }
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                const int h = h0 + k;
                if (h < W)
                    tokens[(b * W + h) * step + first + t] = first + t <= enter_at[h] ? (long long)token[k] : ended[h] && first + t == len[h] - 1 ? eos : pad;
            }
        }
    }
}

// Steps of a CTA: a cluster of up to eight has a group, as long as two CTAs an SM are not exceeded and each has 64 steps.
int finish_span(int B, int step, int* ranks) {
    int r = 1;
    while (r < kFinishCluster && (long long)B * r * 2 <= 2LL * nxd_num_sms() && step >= 128 * r) r *= 2;
    *ranks = r;
    return (step + r - 1) / r;
}

// How rows are split: threads and vectors a thread of a round, rounds of a CTA, CTAs of a row.
struct Split {
    int threads, vecs, rounds, splits;
};

// Rounds of 512 threads x 4 vectors where that leaves no SM without a CTA, as many of them per CTA as leave one wave (two CTAs an SM): every CTA pays
// for its first bound and for putting candidates in order (256 rows of 128256, rows and join: 23 us, by 256 threads x 2 vectors 29).  Rounds of 256 x 2
// where rows are few (one row of 128256 6.6 us instead of 7.0, though four 8.0 instead of 7.4) or no longer than two of them (512 rows of 2000: 9 us
// instead of 16, of 5000 10 instead of 16; of 16000, which are longer, 15 instead of 16, but 256 rows of 16000 12 instead of 10).
Split split_of(long long rows, int W, int V, int elem) {
    const int per_vec = 16 / elem;
    const long long sms = nxd_num_sms(), span = V, large = 512LL * 4 * per_vec;
    Split s;
    const bool few = rows * ((span + large - 1) / large) < sms || span <= 2 * 512LL * per_vec;
    s.threads = few ? 256 : 512;
    s.vecs = few ? 2 : 4;
    const long long round = (long long)s.threads * s.vecs * per_vec, chunks = (span + round - 1) / round;
    long long beside = (few ? 4 : 2) * sms / rows;
    if (beside < 1) beside = 1;
    if (beside > kMaxLists / W) beside = kMaxLists / W;
    s.rounds = (int)((chunks + beside - 1) / beside);
    s.splits = (int)((chunks + s.rounds - 1) / s.rounds);
    return s;
}

template <typename T>
cudaError_t launch_rows(const Split& p, long long ctas, cudaStream_t s, const void* logits, int V, long long stride, int n, Lists out) {
    const int smem = (p.rounds < kStages ? p.rounds : kStages) * p.vecs * (p.threads / 32) * kStagePitch * 16;
    if (p.threads == 256) {
        beam_rows_kernel<T, 256, 2><<<(unsigned)ctas, 256, smem, s>>>((const T*)logits, V, stride, p.splits, p.rounds, n, out);
    } else {
        const cudaError_t e = nxd_allow_smem<beam_rows_kernel<T, 512, 4>>(kStages * 4 * 16 * kStagePitch * 16);
        if (e != cudaSuccess) return e;
        beam_rows_kernel<T, 512, 4><<<(unsigned)ctas, 512, smem, s>>>((const T*)logits, V, stride, p.splits, p.rounds, n, out);
    }
    return cudaSuccess;
}

}  // namespace

// Scratch of a call in bytes, or 0 where the sizes are outside what is compiled.
NXD_API long long nxd_beam_select_scratch(int dtype, int B, int W, int V, int n) {
    if (dtype < 0 || dtype > 2 || B < 1 || W < 1 || W > kMaxBeams || V < 1 || V > 1 << 30 || n < 1 || n > kMaxN || (long long)W * V >= (1LL << 31) - 16 || n > (long long)W * V)
        return 0;
    const long long rows = (long long)B * W, lists = rows * split_of(rows, W, V, dtype == 0 ? 4 : 2).splits;
    return lists < (1LL << 31) ? lists * (8 + 8LL * n) : 0;
}

// logits [B * W, V] (0 fp32, 1 bf16, 2 fp16; rows `stride` elements apart), scores [B, W] -> the n best candidates of every group.
NXD_API int nxd_beam_select(int dtype, const void* logits, long long stride, const float* scores, int B, int W, int V, int n, void* scratch,
                            float* out_scores, long long* out_beams, long long* out_tokens, void* stream) {
    if (B == 0) return 0;
    NXD_REQUIRE(nxd_beam_select_scratch(dtype, B, W, V, n) > 0, "beam_select: %d beams of %d tokens, %d candidates are outside what is compiled", W, V, n);
    cudaStream_t s = (cudaStream_t)stream;
    const long long rows = (long long)B * W;
    const Split p = split_of(rows, W, V, dtype == 0 ? 4 : 2);
    const int splits = p.splits, lists = W * splits;
    const Lists l = lists_of(scratch, rows * splits, n);
    if (dtype == 0) NXD_CHECK_CUDA(launch_rows<float>(p, rows * splits, s, logits, V, stride, n, l));
    else if (dtype == 1) NXD_CHECK_CUDA(launch_rows<bf16>(p, rows * splits, s, logits, V, stride, n, l));
    else NXD_CHECK_CUDA(launch_rows<__half>(p, rows * splits, s, logits, V, stride, n, l));
    NXD_LAUNCH_CHECK();
    const int threads = lists * n > 1024 ? 1024 : 256, picked = n * (n < lists ? n : lists);
    const int room = lists * n <= kOwn * threads ? lists * n : lists > picked ? lists : picked, smem = (lists + room) * 12;
    NXD_CHECK_CUDA(nxd_allow_smem<beam_join_kernel>(kMaxLists * 24));
    NXD_CHECK_CUDA(nxd_launch_pdl(beam_join_kernel, dim3(B), dim3(threads), smem, s, scores, W, V, splits, n, room, l, out_scores, out_beams, out_tokens));
    NXD_LAUNCH_CHECK();
    return 0;
}

// One step of the books (the header has the arrays).  3 us, latency: a warp a group.
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

// Bytes of scratch that a call needs, 0: none.
NXD_API long long nxd_beam_finish_scratch(int B, int W, int step) {
    int ranks;
    return (long long)W * finish_span(B, step, &ranks) > kFinishBytes ? (long long)B * W * step : 0;
}

// The sequences of every group's best W hypotheses (the header has the arrays).
NXD_API int nxd_beam_finish(const float* running, const float* pool_scores, const int* pool_lengths, const int* pool_slots, const unsigned char* done,
                            int B, int W, int step, float norm, long long eos, long long pad, const int* hist_tokens, const int* hist_parents,
                            long long* tokens, long long* lengths, float* scores, void* scratch, void* stream) {
    NXD_REQUIRE(W >= 1 && W <= kMaxBeams && step >= 1 && (long long)W * step < (1LL << 30) && B <= 65535, "beam_finish: %d requests of %d beams, %d steps", B, W, step);
    if (B == 0) return 0;
    const bool large = nxd_beam_finish_scratch(B, W, step) > 0;
    NXD_REQUIRE(!large || scratch != nullptr, "beam_finish: %d beams of %d steps need scratch", W, step);
    int ranks;
    const int span = finish_span(B, step, &ranks);
    const Books in = {running, pool_scores, pool_lengths, pool_slots, done};
    const long long token_bytes = 4LL * span * token_pitch(W), path_bytes = (long long)W * span;
    const bool staged = !large && token_bytes + path_bytes <= kFinishBytes;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ranks, B);
    cfg.blockDim = dim3(path_bytes >= kFinishThreads ? kFinishThreads : path_bytes <= 128 ? 128 : (unsigned)((path_bytes + 31) / 32 * 32));
    cfg.dynamicSmemBytes = (large ? 0 : path_bytes) + (staged ? token_bytes : 0);
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ranks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    NXD_CHECK_CUDA(nxd_allow_smem<beam_finish_kernel>(kFinishBytes));
    NXD_CHECK_CUDA(cudaLaunchKernelEx(&cfg, beam_finish_kernel, in, W, B, step, span, norm, eos, pad, hist_tokens, hist_parents, tokens, lengths, scores,
                                      large ? (unsigned char*)scratch : (unsigned char*)nullptr, (int)staged));
    NXD_LAUNCH_CHECK();
    return 0;
}
