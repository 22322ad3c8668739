// The tile list of a packed batch: sequences of different lengths laid end to end in `T` rows, bounded by cu[0 .. N], for the
// attention kernels, which work by tiles of 128 (packed_attention.cu, packed_attention_bwd.cu) or 256 rows (the former) of one sequence.
//
// The lengths stay on the device, so that a step needs no copy to the host and can be captured: the list has room for
// T / 128 + N + 2 tiles whatever the lengths are, and entries without a tile cost nothing.  Boundaries that fall or leave [0, T] are
// brought back (running maximum, clamped), so no list can lead a kernel out of its tensors.
//
// Order: longest first.  A query tile t of a causal sequence meets t + 1 tiles of keys, so with c(w) = the number of sequences of
// at least w tiles the list holds c(w) tiles of weight w, heaviest first (without a mask a tile weighs its whole sequence's tiles): a
// counting sort by weight in shared memory.  Tiles of one weight come in no fixed order; no result depends on it.
//
// One block: the boundaries are 4 bytes each and the list 16 bytes per 128 rows.  Bound by latency, two passes over the
// sequences (running maximum and padded offsets, then places); a thread places a sequence's first tiles, a warp those of a long one.
#include "attn_tc_common.cuh"

namespace {
using nxd_attn::PackedTile;

constexpr int kThreads = 1024;
constexpr int kBins = 4096;          // weights above (half a million rows) share the last bin
constexpr int kOwn = 2;              // tiles of a sequence that its thread places itself

struct ScanMax {
    __device__ static int op(int a, int b) { return max(a, b); }
};
struct ScanSum {
    __device__ static int op(int a, int b) { return a + b; }
};

// inclusive scan over the block (0 is the neutral element: maxima are of numbers >= 0); `total` is the last value
template <class Op>
__device__ int block_scan(int v, int* warps, int& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v = Op::op(v, u);
    }
    if (lane == 31) warps[warp] = v;
    __syncthreads();
    if (warp == 0) {
        int w = warps[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w = Op::op(w, u);
        }
        warps[lane] = w;
    }
    __syncthreads();
    if (warp > 0) v = Op::op(v, warps[warp - 1]);
    total = warps[31];
    __syncthreads();
    return v;
}

template <typename Index>
__global__ void __launch_bounds__(kThreads) packed_plan_kernel(const Index* __restrict__ cu, int N, int T, int causal, int rows, PackedTile* tiles,
                                                              int entries, int4* seqs, int* which) {
    __shared__ int bins[kBins + 2], warps[32];
    const int tid = threadIdx.x, lane = tid & 31;
    pdl_trigger();
    pdl_wait();
    for (int i = tid; i < kBins + 2; i += kThreads) bins[i] = 0;
    __syncthreads();
    const auto bound = [&](int i) {
        const long long c = (long long)cu[i];
        return (int)(c < 0 ? 0 : c > T ? T : c);
    };
    const int first = bound(0);
    int high = first, pad = 0, n_tiles = 0;          // running over the chunks, the same in every thread
    for (int base = 0; base < N; base += kThreads) {
        const int i = base + tid;
        int total;
        const int end = max(high, block_scan<ScanMax>(i < N ? bound(i + 1) : 0, warps, total));
        const int next_high = max(high, total);
        // the row where it starts is the maximum up to its left neighbour
        int start = __shfl_up_sync(0xffffffffu, end, 1);
        if (lane == 31) warps[tid >> 5] = end;
        __syncthreads();
        if (lane == 0) start = tid ? warps[(tid >> 5) - 1] : high;
        __syncthreads();
        const int len = i < N ? end - start : 0, n = (len + rows - 1) / rows;
        const int before = block_scan<ScanSum>((len + 3) & ~3, warps, total) - ((len + 3) & ~3);
        if (i < N) seqs[i] = make_int4(start, len, pad + before, n);
        pad += total;
        block_scan<ScanSum>(n, warps, total);
        n_tiles += total;
        high = next_high;
        if (n > 0) {
            if (causal) {            // differences of c(w): one tile of every weight up to n
                atomicAdd(&bins[1], 1);
                atomicSub(&bins[min(n, kBins) + 1], 1);
                if (n > kBins) atomicAdd(&bins[0], n - kBins);          // what the last bin gets besides
            } else {
                atomicAdd(&bins[min(n, kBins)], n);
            }
        }
    }
    __syncthreads();
    // bins[w] <- the place of the first tile of weight w: the number of heavier ones
    {
        constexpr int P = kBins / kThreads;
        const int extra = causal ? bins[0] : 0;
        int c[P], sum = 0, total;
#pragma unroll
        for (int j = 0; j < P; ++j) sum += c[j] = bins[1 + tid * P + j];
        if (causal) {                // counts from their differences
            int at = block_scan<ScanSum>(sum, warps, total) - sum;
            sum = 0;
#pragma unroll
            for (int j = 0; j < P; ++j) {
                at += c[j];
                c[j] = at;
                if (tid * P + j + 1 == kBins) c[j] += extra;
                sum += c[j];
            }
        }
        int lighter = block_scan<ScanSum>(sum, warps, total) - sum;
#pragma unroll
        for (int j = 0; j < P; ++j) {
            lighter += c[j];
            bins[1 + tid * P + j] = n_tiles - lighter;
        }
    }
    __syncthreads();
    const auto place = [&](const int4& s, int t, int sequence) {
        const int at = atomicAdd(&bins[min(causal ? t + 1 : s.w, kBins)], 1);
        if (at >= entries) return;
        reinterpret_cast<int4*>(tiles)[at] = make_int4(s.x, s.y, t, s.z);
        which[at] = sequence;
    };
    for (int base = 0; base < N; base += kThreads) {
        const int i = base + tid;
        const int4 s = i < N ? seqs[i] : make_int4(0, 0, 0, 0);
        for (int t = 0; t < min(s.w, kOwn); ++t) place(s, t, i);
        for (unsigned more = __ballot_sync(0xffffffffu, s.w > kOwn); more; more &= more - 1) {
            const int from = __ffs(more) - 1;
            const int4 q = make_int4(__shfl_sync(0xffffffffu, s.x, from), __shfl_sync(0xffffffffu, s.y, from),
                                     __shfl_sync(0xffffffffu, s.z, from), __shfl_sync(0xffffffffu, s.w, from));
            for (int t = kOwn + lane; t < q.w; t += 32) place(q, t, base + (tid & ~31) + from);
        }
    }
    // rows before the first and behind the last sequence, then entries without work
    const int gap0 = (first + rows - 1) / rows, gap1 = (T - high + rows - 1) / rows;
    for (int i = n_tiles + tid; i < entries; i += kThreads) {
        const int j = i - n_tiles;
        int from = 0, here = 0;
        if (j < gap0) from = j * rows, here = min(rows, first - from);
        else if (j < gap0 + gap1) from = high + (j - gap0) * rows, here = min(rows, T - from);
        reinterpret_cast<int4*>(tiles)[i] = make_int4(from, 0, here, 0);
    }
}

}  // namespace

// Tiles that the list has room for.
NXD_API int nxd_packed_plan_entries(long long T, int N, int rows) {
    const long long n = T / rows + (N < T ? N : T) + 2;
    return n < (1ll << 31) ? (int)n : -1;
}

// Columns of a row of the per-row scratch (log-sum-exp, Delta, dQ accumulator): sequences are padded to four columns, and a tile may
// reach 64 columns behind the last one.
NXD_API long long nxd_packed_plan_columns(long long T, int N) {
    return ((T + 3 * (N < T ? (long long)N : T) + 3) & ~3ll) + 64;
}

// cu: N + 1 boundaries, int32 or (wide) int64; rows of a tile: 128 or 256; tiles: nxd_packed_plan_entries entries of 16 bytes; seqs: 16 bytes of scratch
// per sequence, afterwards {first row, rows, first padded column, tiles} of each; which: an int per entry, the number of the tile's sequence.
NXD_API int nxd_packed_plan(const void* cu, int wide, int N, long long T, int causal, int rows, void* tiles, void* seqs, int* which, void* stream) {
    NXD_REQUIRE(rows == 128 || rows == 256, "packed_plan: tiles of %d rows", rows);
    const int entries = nxd_packed_plan_entries(T, N, rows);
    NXD_REQUIRE(N >= 0 && T > 0 && T < (1ll << 31) - 256 && entries > 0, "packed_plan: %d sequences in %lld rows", N, T);
    NXD_REQUIRE(cu && tiles && which && (seqs || N == 0), "packed_plan: %s", "a list is missing");
    NXD_REQUIRE((((uintptr_t)tiles | (uintptr_t)seqs) & 15) == 0, "packed_plan: the lists must be %s", "16-byte aligned");
    cudaStream_t st = (cudaStream_t)stream;
    if (wide)
        NXD_CHECK_CUDA((nxd_launch_pdl(packed_plan_kernel<long long>, dim3(1), dim3(kThreads), 0, st, (const long long*)cu, N, (int)T, causal, rows,
            (PackedTile*)tiles, entries, (int4*)seqs, which)));
    else
        NXD_CHECK_CUDA((nxd_launch_pdl(packed_plan_kernel<int>, dim3(1), dim3(kThreads), 0, st, (const int*)cu, N, (int)T, causal, rows,
            (PackedTile*)tiles, entries, (int4*)seqs, which)));
    NXD_LAUNCH_CHECK();
    return 0;
}
