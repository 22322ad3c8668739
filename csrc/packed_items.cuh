// What the packed attention kernels share (packed_attention.cu, packed_attention_bwd.cu): one CTA per SM stays for the whole call and
// walks over items of the batch's tile list.
#pragma once
#include "attn_tc_common.cuh"

namespace nxd_packed {

// A try of a wait lasts 3900 clocks, so a wait ends after two seconds; the results of a CTA that gave up are NaN.
constexpr int kTries = 1 << 20;

// A wait with an end: after kTries the CTA is marked, and no wait of its lasts any more.  The end costs the threads that wait 3 to 6 % of the
// backward pass (D = 128, 16384 tokens: 2980 us against 2800 without it; 3100 with two predicated tries ahead of the loop, 3290 with
// the counting in one condition with the try).
__device__ __forceinline__ void wait_for(uint64_t* bar, uint32_t parity, volatile int* dead) {
    if (ptx::mbar_try_wait(bar, parity)) return;
    for (int i = 0; !ptx::mbar_try_wait(bar, parity); ++i) {
        if (i == kTries) *dead = 1;
        if (*dead) break;
    }
}

// copies that were started may still be on their way into the memory of a CTA that gave up
__device__ __forceinline__ void let_copies_land() {
    const long long start = clock64();
    while (clock64() - start < 40000000) {          // 20 ms
    }
}

// The items of a CTA: every gridDim.x-th of the list, which is sorted by weight, forwards and backwards in turn so that nobody gets the
// longest of every round.  The TMA warp, which is ahead of the others, reads them and hands them on through a ring in shared memory.
constexpr int kItems = 4;
constexpr int kRowsOfNone = 1;           // added to the rows of an entry of no sequence, to tell its kind from an item's
__device__ __forceinline__ unsigned item_of_round(int round) {          // below 2^31 + gridDim.x
    return round * gridDim.x + (round & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
}

// hands an item on; all lanes of the warp take part
template <class Item>
__device__ __forceinline__ void publish_item(const Item& x, Item* ring, uint64_t* full, uint64_t* empty, int& count, volatile int* dead) {
    const int i = count % kItems;
    wait_for(&empty[i], ((uint32_t)(count / kItems) & 1u) ^ 1u, dead);
    ++count;
    if ((threadIdx.x & 31) == 0) {
        const int4* src = reinterpret_cast<const int4*>(&x);
        int4* dst = reinterpret_cast<int4*>(&ring[i]);
#pragma unroll
        for (int w = 0; w < 3; ++w) dst[w] = src[w];
        ptx::mbar_arrive(&full[i]);
    }
}

// the next item of the ring, for a whole warp or (WARP = false) one thread
template <bool WARP, class Item>
__device__ __forceinline__ Item next_item(const Item* ring, uint64_t* full, uint64_t* empty, int& count, volatile int* dead) {
    const int i = count % kItems;
    wait_for(&full[i], (uint32_t)(count / kItems) & 1u, dead);
    ++count;
    Item it{};
    if (!*dead) {
        const int4* src = reinterpret_cast<const int4*>(&ring[i]);
        int4* dst = reinterpret_cast<int4*>(&it);
#pragma unroll
        for (int w = 0; w < 3; ++w) dst[w] = src[w];
    }
    if (WARP) __syncwarp();
    if (!WARP || (threadIdx.x & 31) == 0) ptx::mbar_arrive(&empty[i]);
    return it;
}

}  // namespace nxd_packed
