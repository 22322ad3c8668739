// Whole lines and pages of a key/value cache, in every layer at once: lines that continue other lines (beam search), and pages that are copied
// (a line forks, a shared page is about to be written, a pool is compacted).
//
// Both only move bytes, so HBM bounds them: 699 MB (16 layers, 32 lines of up to 900 rows, recurrent states) are 107 us at 6555 GB/s and take 119, through a
// block table 139 (its entries are read for every unit and move); 1007 MB of pages are 154 us and take 156.  All tensors of one shape share a launch; their addresses travel as kernel parameters.
#include "common.cuh"
#include "nxd_b200.h"

namespace {

constexpr int kThreads = 256;
constexpr int kMaxTensors = 256;          // of a launch of page copies: 2 KB of parameters
constexpr int kJobTensors = 128;          // of one of the two shapes of a launch of lines
constexpr int kMaxBeams = 32;
constexpr int kDeep = 4;                  // units of a thread

struct Tensors {
    char* base[kMaxTensors];
    int n;
};

// What all tensors of a launch have in common, in units of U bytes (per_row) and in bytes (strides).
struct Shape {
    int heads, rows, per_row;
    long long line_stride, head_stride;
};

// The order in which a group's lines can be written in place: no line is written before those that continue it have read it.  Where
// lines continue each other in a circle, one of them is set aside first.  Entries (to, from); from = kAside: what was set aside, to = kAside: it.
constexpr int kAside = -1, kMaxMoves = kMaxBeams + kMaxBeams / 2;
struct Moves {
    signed char to[kMaxMoves], from[kMaxMoves];
    int n;
    bool circles;
};

// By one warp, lane w for line w; from[w] = w: it stays.
__device__ __forceinline__ void order_moves(int from, int lane, Moves& m) {
    unsigned left = __ballot_sync(0xffffffffu, from != lane);          // lines to be written
    int n = 0;
    bool circles = false;
    while (left != 0) {
        // lines that a line still to be written reads
        const unsigned read = __reduce_or_sync(0xffffffffu, left >> lane & 1 ? 1u << from : 0u);
        const unsigned ready = left & ~read;
        if (ready != 0) {
            if (ready >> lane & 1) {
                const int at = n + __popc(ready & ((1u << lane) - 1u));
                m.to[at] = (signed char)lane;
                m.from[at] = (signed char)from;
            }
            n += __popc(ready);
            left &= ~ready;
        } else {          // circles only: the first one, around
            circles = true;
            const int first = __ffs(left) - 1;
            if (lane == 0) m.to[n] = kAside, m.from[n] = (signed char)first;
            ++n;
            int at = first;
            do {
                const int next = __shfl_sync(0xffffffffu, from, at);
                if (lane == 0) m.to[n] = (signed char)at, m.from[n] = next == first ? (signed char)kAside : (signed char)next;
                ++n;
                left &= ~(1u << at);
                at = next;
            } while (at != first);
        }
    }
    if (lane == 0) m.n = n, m.circles = circles;
}

// Lines g * W + w of a group continue its lines g * W + parent[w], rows [start, end) of every head.  A thread takes kDeep units, a block's width
// apart, of all the group's lines in an order that works in place, so there is no scratch and each line that is wanted is read once from memory
// however many continue it.  Two moves of four units are read before the first of them is written (one unit: 147 us instead of 111 for the case
// above without its states, 98 of bytes).  Circles go one unit at a time, at 0.7 of that rate; no step of a search makes one.
//   With a table the lines are pages: PAGED.  Two shapes share a launch (keys and values, and a recurrent state): the first blocks are one's, the
// others the other's (the case above: 119 us instead of 124).
struct Job {
    char* base[kJobTensors];
    int n, num_pages;
    bool whole;                           // all rows, whatever start and end are
    unsigned first, blocks;
    Shape s;
};
struct Jobs {
    Job job[2];
};

template <typename U, bool PAGED>
__global__ void __launch_bounds__(kThreads, PAGED ? 3 : 4) reorder_lines_kernel(const __grid_constant__ Jobs jobs, int W, const long long* __restrict__ parents,
                                                                                const long long* __restrict__ start, const long long* __restrict__ end,
                                                                                const int* __restrict__ table, int page_size, int max_pages) {
    __shared__ Moves moves;
    const int g = blockIdx.y;
    const Job& t = jobs.job[blockIdx.x >= jobs.job[1].first];
    const Shape s = t.s;
    const unsigned block = blockIdx.x - t.first;
    const int num_pages = t.num_pages;
    const long long line0 = (long long)g * W;
    if (threadIdx.x < 32) {
        const int w = threadIdx.x;
        long long p = w < W ? parents[line0 + w] : w;
        if (p < 0 || p >= W) p = w;          // a line whose parent is none of the group's stays as it is
        order_moves((int)p, w, moves);
    }
    __syncthreads();
    const int n = moves.n;
    const long long lo = !t.whole && start != nullptr ? max(start[g], 0LL) : 0, hi = !t.whole && end != nullptr ? min(end[g], (long long)s.rows) : s.rows;
    if (n == 0 || hi <= lo) return;
    const unsigned per_head = (unsigned)(hi - lo) * (unsigned)s.per_row, per_tensor = per_head * (unsigned)s.heads;
    const unsigned total = per_tensor * (unsigned)t.n;          // the host keeps it below 2^31
    for (unsigned i0 = block * (kThreads * kDeep) + threadIdx.x; i0 < total; i0 += t.blocks * (kThreads * kDeep)) {
        char* base[kDeep];          // of a unit in the group's first line, or in page 0
        int page[PAGED ? kDeep : 1];
#pragma unroll
        for (int q = 0; q < kDeep; ++q) {
            const unsigned i = min(i0 + q * kThreads, total - 1);
            const unsigned tensor = i / per_tensor, in_tensor = i - tensor * per_tensor;
            const unsigned head = in_tensor / per_head, unit = in_tensor - head * per_head;
            char* at = t.base[tensor] + (long long)head * s.head_stride;
            if constexpr (PAGED) {
                const unsigned r = unit / (unsigned)s.per_row, row = (unsigned)lo + r;
                page[q] = (int)(row / (unsigned)page_size);
                at += ((long long)(row - (unsigned)page[q] * (unsigned)page_size) * s.per_row + (unit - r * (unsigned)s.per_row)) * (long long)sizeof(U);
            } else {
                at += line0 * s.line_stride + (lo * s.per_row + unit) * (long long)sizeof(U);
            }
            base[q] = at;
        }
        // of line w, or nothing where the table names no page
        auto place = [&](int q, int w) -> U* {
            if constexpr (PAGED) {
                const int p = table[(line0 + w) * max_pages + page[q]];
                return p < 0 || p >= num_pages ? nullptr : reinterpret_cast<U*>(base[q] + p * s.line_stride);
            } else {
                return reinterpret_cast<U*>(base[q] + w * s.line_stride);
            }
        };
        const unsigned left = (total - i0 + kThreads - 1) / kThreads;          // units that are this thread's
        if (moves.circles) {
#pragma unroll
            for (int q = 0; q < kDeep; ++q) {
                if (q >= left) break;
                U aside{};
                bool held = false;
#pragma unroll 1
                for (int k = 0; k < n; ++k) {
                    const int d = moves.to[k], f = moves.from[k];
                    const U* src = f == kAside ? nullptr : place(q, f);
                    U* dst = d == kAside ? nullptr : place(q, d);
                    if (d == kAside) {
                        held = src != nullptr;
                        if (held) aside = *src;
                    } else if (f == kAside) {
                        if (held && dst != nullptr) *dst = aside;
                    } else if (src != nullptr && dst != nullptr) {
                        *dst = *src;
                    }
                }
            }
            continue;
        }
        for (int k0 = 0; k0 < n; k0 += 2) {
            U v[2][kDeep];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                if (k0 + k < n) {
#pragma unroll
                    for (int q = 0; q < kDeep; ++q) {
                        const U* src = place(q, moves.from[k0 + k]);
                        if (q < left && (!PAGED || src != nullptr)) v[k][q] = *src;
                    }
                }
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                if (k0 + k < n) {
#pragma unroll
                    for (int q = 0; q < kDeep; ++q) {
                        U* dst = place(q, moves.to[k0 + k]);
                        if (q < left && (!PAGED || (dst != nullptr && place(q, moves.from[k0 + k]) != nullptr))) *dst = v[k][q];
                    }
                }
            }
        }
    }
}

// Page dst[i] becomes page src[i], its first rows[i] rows of every head.  No page that is read is written by the same call.
template <typename U>
__global__ void __launch_bounds__(kThreads) copy_pages_kernel(const __grid_constant__ Tensors t, Shape s, int pages, int pairs, const long long* __restrict__ src,
                                                              const long long* __restrict__ dst, const long long* __restrict__ rows) {
    for (int pair = blockIdx.y; pair < pairs; pair += gridDim.y) {
        const long long from = src[pair], to = dst[pair];
        if (from < 0 || to < 0 || from >= pages || to >= pages || from == to) continue;
        const int n = rows != nullptr ? (int)min(max(rows[pair], 0LL), (long long)s.rows) : s.rows;
        const unsigned per_head = (unsigned)n * (unsigned)s.per_row, per_tensor = per_head * (unsigned)s.heads;
        const unsigned total = per_tensor * (unsigned)t.n;
        for (unsigned i0 = blockIdx.x * (kThreads * kDeep) + threadIdx.x; i0 < total; i0 += gridDim.x * (kThreads * kDeep)) {
            U v[kDeep];
            U* at[kDeep];
#pragma unroll
            for (int k = 0; k < kDeep; ++k) {
                const unsigned i = i0 + k * kThreads;
                at[k] = nullptr;
                if (i < total) {
                    const unsigned tensor = i / per_tensor, in_tensor = i - tensor * per_tensor;
                    const unsigned head = in_tensor / per_head, unit = in_tensor - head * per_head;
                    char* base = t.base[tensor] + head * s.head_stride + (long long)unit * (long long)sizeof(U);
                    v[k] = *reinterpret_cast<const U*>(base + from * s.line_stride);
                    at[k] = reinterpret_cast<U*>(base + to * s.line_stride);
                }
            }
#pragma unroll
            for (int k = 0; k < kDeep; ++k)
                if (at[k] != nullptr) *at[k] = v[k];
        }
    }
}

// The widest unit that rows, strides and addresses allow.
int unit_of(void* const* base, int n, long long row_bytes, long long line_stride, long long head_stride) {
    unsigned long long all = (unsigned long long)row_bytes | (unsigned long long)line_stride | (unsigned long long)head_stride;
    for (int i = 0; i < n; ++i) all |= (unsigned long long)(uintptr_t)base[i];
    return (all & 15) == 0 ? 16 : (all & 3) == 0 ? 4 : (all & 1) == 0 ? 2 : 1;
}

// Blocks beside each other for one group or pair: what its units can use, up to four waves.  (16 layers, 32 lines of 900 rows: one wave 136 us, two 130,
// four 124, sixteen 121; but a block without work costs its start, and the host does not know the ranges.)
unsigned blocks_for(long long units, long long per_block, long long beside) {
    const long long want = (units + per_block - 1) / per_block, room = (16LL * nxd_num_sms() + beside - 1) / beside;
    const long long least = nxd_num_sms();
    return (unsigned)(want < room ? want : room < least ? (want < least ? want : least) : room);
}

constexpr long long kMaxUnits = (1LL << 31) - (1LL << 22);          // of a group or pair in a launch: the strides of the loops stay below 2^32

}  // namespace

// The header has the arrays.  Shapes whose widest unit is the same go two to a launch.
NXD_API int nxd_reorder_lines(const nxd_lines* kinds, int n_kinds, int groups, int W, const long long* parents, const long long* start, const long long* end,
                              const int* table, int page_size, int max_pages, void* stream) {
    NXD_REQUIRE(W >= 1 && W <= kMaxBeams, "reorder_lines: %d lines of a group are not between 1 and %d", W, kMaxBeams);
    NXD_REQUIRE(groups >= 0 && groups <= 65535, "reorder_lines: %d groups are more than 65535", groups);
    if (groups == 0) return 0;
    Jobs jobs;
    int held = 0, held_unit = 0;
    bool held_paged = false;
    cudaStream_t st = (cudaStream_t)stream;
    auto launch = [&]() -> cudaError_t {
        if (held == 0) return cudaSuccess;
        jobs.job[0].first = 0;
        jobs.job[1].first = jobs.job[0].blocks;          // of one job: behind the last block
        const dim3 grid(jobs.job[0].blocks + (held > 1 ? jobs.job[1].blocks : 0), groups);
        held = 0;
#define NXD_REORDER(U)                                                                                                                          \
    (held_paged ? reorder_lines_kernel<U, true><<<grid, kThreads, 0, st>>>(jobs, W, parents, start, end, table, page_size, max_pages)           \
                : reorder_lines_kernel<U, false><<<grid, kThreads, 0, st>>>(jobs, W, parents, start, end, nullptr, 0, 0))
        if (held_unit == 16) NXD_REORDER(uint4);
        else if (held_unit == 4) NXD_REORDER(uint32_t);
        else if (held_unit == 2) NXD_REORDER(uint16_t);
        else NXD_REORDER(uint8_t);
#undef NXD_REORDER
        nxd_count_launches(1);
        return cudaGetLastError();
    };
    for (int k = 0; k < n_kinds; ++k) {
        const nxd_lines& d = kinds[k];
        const bool paged = table != nullptr && !d.whole;
        const long long rows = paged ? (long long)page_size * max_pages : d.rows;
        if (d.n == 0 || rows == 0 || d.row_bytes == 0 || d.heads == 0) continue;
        const int unit = unit_of(d.base, d.n, d.row_bytes, d.line_stride, d.head_stride);
        const long long per_row = d.row_bytes / unit, per_tensor = rows * per_row * d.heads;
        NXD_REQUIRE(per_tensor <= kMaxUnits, "reorder_lines: a line of %lld rows of %lld bytes in %d heads is too long", rows, d.row_bytes, d.heads);
        const int most = (int)(kMaxUnits / per_tensor < kJobTensors ? kMaxUnits / per_tensor : kJobTensors);
        for (int at = 0; at < d.n; at += most) {
            if (held == 2 || (held == 1 && (held_unit != unit || held_paged != paged))) NXD_CHECK_CUDA(launch());
            Job& j = jobs.job[held++];
            held_unit = unit, held_paged = paged;
            j.n = d.n - at < most ? d.n - at : most;
            for (int i = 0; i < j.n; ++i) j.base[i] = (char*)d.base[at + i];
            j.num_pages = d.pages;
            j.whole = d.whole != 0;
            j.s = {d.heads, (int)rows, (int)per_row, d.line_stride, d.head_stride};
            j.blocks = blocks_for(per_tensor * j.n, kThreads * kDeep, groups);
        }
    }
    NXD_CHECK_CUDA(launch());
    return 0;
}

// n tensors of one shape [pages, heads, rows, row_bytes] at `base` (host array of device addresses).
NXD_API int nxd_copy_pages(void* const* base, int n, int pages, int heads, long long rows, long long row_bytes, long long page_stride,
                           long long head_stride, int pairs, const long long* src, const long long* dst, const long long* used, void* stream) {
    if (n == 0 || pairs == 0 || rows == 0 || row_bytes == 0 || heads == 0) return 0;
    const int unit = unit_of(base, n, row_bytes, page_stride, head_stride);
    const long long per_row = row_bytes / unit, per_tensor = rows * per_row * heads;
    NXD_REQUIRE(per_tensor <= kMaxUnits, "copy_pages: a page of %lld rows of %lld bytes in %d heads is too large", rows, row_bytes, heads);
    const int most = (int)(kMaxUnits / per_tensor < kMaxTensors ? kMaxUnits / per_tensor : kMaxTensors);
    for (int at = 0; at < n; at += most) {
        Tensors t;
        t.n = n - at < most ? n - at : most;
        for (int i = 0; i < kMaxTensors; ++i) t.base[i] = i < t.n ? (char*)base[at + i] : nullptr;
        const Shape s = {heads, (int)rows, (int)per_row, page_stride, head_stride};
        const dim3 grid(blocks_for(per_tensor * t.n, kThreads * 4, pairs), pairs < 65535 ? pairs : 65535);
        cudaStream_t st = (cudaStream_t)stream;
        if (unit == 16) copy_pages_kernel<uint4><<<grid, kThreads, 0, st>>>(t, s, pages, pairs, src, dst, used);
        else if (unit == 4) copy_pages_kernel<uint32_t><<<grid, kThreads, 0, st>>>(t, s, pages, pairs, src, dst, used);
        else if (unit == 2) copy_pages_kernel<uint16_t><<<grid, kThreads, 0, st>>>(t, s, pages, pairs, src, dst, used);
        else copy_pages_kernel<uint8_t><<<grid, kThreads, 0, st>>>(t, s, pages, pairs, src, dst, used);
        NXD_LAUNCH_CHECK();
    }
    return 0;
}
