// What the packed attention kernels share (packed_attention.cu, packed_attention_bwd.cu): one CTA per SM stays for the whole call and
// walks over items of the batch's tile list.
#pragma once
#include "attn_tc_common.cuh"

namespace nxd_packed {

// A try of a wait lasts 3900 clocks, so a wait ends after two seconds.  A CTA that gave one up loads no more and leaves NaN: forward in the
// results of all its items, backward in all gradients of the call.  It sets a word of pinned host memory, and the next call fails.
constexpr int kTries = 1 << 20;
constexpr int kGaveUp = -kTries;         // the CTA's mark; below that many tries a wait starts with their number less kTries
__device__ __forceinline__ bool gave_up(const volatile int* dead) { return *dead == kGaveUp; }

// Sets *word to the word above; fails where a call before this one has set it, and clears it.
int begin_call(int** word);

// A wait with an end: after kTries the CTA is marked, and no wait of its lasts any more (the mark leaves one try).  In one piece, because
// the loop's shape counts: of the backward pass of 4 documents in 16384 tokens, 32 heads of 128 over 8, it takes 2050 us (one of 16384
// tokens, 16 heads of 64 over 4: 1967) as here, 2090 (2057) as a loop in C++, 2106 (2166) as a call behind the first try, 2124 (2156)
// with the first try counted too.
__device__ __forceinline__ void wait_for(uint64_t* bar, uint32_t parity, volatile int* dead) {
    asm volatile(
        "{\n\t"
        ".reg .pred P, Q;\n\t"
        ".reg .s32 left;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 P, [%0], %1;\n\t"
        "@P bra DONE;\n\t"
        "ld.volatile.shared.s32 left, [%2];\n\t"          // 0, or kGaveUp, or (a smaller limit) between the two
        "add.s32 left, left, %3;\n"
        "TRY:\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 P, [%0], %1;\n\t"
        "@P bra DONE;\n\t"
        "sub.s32 left, left, 1;\n\t"
        "setp.gt.s32 Q, left, 0;\n\t"
        "@Q bra TRY;\n\t"
        "st.volatile.shared.s32 [%2], %4;\n"
        "DONE:\n\t"
        "}"
        ::"r"(ptx::smem_u32(bar)), "r"(parity), "r"(ptx::smem_u32(const_cast<const int*>(dead))), "n"(kTries), "n"(kGaveUp)
        : "memory");
}

// copies that were started may still be on their way into the memory of a CTA that gave up
__device__ __forceinline__ void let_copies_land() {
    const long long start = clock64();
    while (clock64() - start < 40000000) {          // 20 ms
    }
}

// The items of a CTA.  The list is sorted by weight, and the first item of a CTA is the one of its number.  Backward, whoever is done
// claims the next from a counter; forward, every gridDim.x-th is its own, forwards and backwards in turn so that nobody gets the longest
// of every round.  The counter needs a launch that clears it, which the backward pass has, and its items differ more (a key block's
// walk covers all heads of the group: 24 samples in 8192 tokens, 32 heads of 64 over 8, worst CTA 26 % above the mean in turn, 5 % by
// claims; 204 us and 181).  Forward the worst is 9 % above (claims: 3 %).  The TMA warp, which is ahead of the others, gets the
// items and hands them on through a ring in shared memory.
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
    if (!gave_up(dead)) {
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
