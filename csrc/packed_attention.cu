// Attention over packed sequences, forward, on 5th-gen tensor cores (tcgen05 + TMEM + TMA), sm_100a.
//
// q [T, Hq, D], k and v [T, Hkv, D]: the sequences of a batch laid end to end, each attending to itself (tile list: packed_plan.cu).
//   S = scale Q K^T, P = exp2(S - m), O = P V / sum P over the keys of the row's sequence (up to the row itself if causal)
//
// One CTA per SM stays for the whole call and walks over items of two query tiles of 128 rows that read the same keys and values: two
// heads of one key head, or (where the heads of a key head are odd in number) two neighbouring tiles of one head.  Sequences of
// fine-tuning are a few hundred tokens, so an item is a few key tiles long: with a CTA per item its start (barriers, tensor memory,
// the first loads) and end were most of its time.  Here the loads of the next item and its first scores run under the last softmax and
// the stores of this one.
//   warps 0-3, 4-7   softmax of query tile 0 / 1, a thread per row; the accumulator stays in tensor memory and is rescaled where a row's
//                    maximum has moved by more than 2^8; at the end of an item they divide and store their rows
//   warps 8, 11      MMA: S_s = Q_s K^T (128 x 128), O_s += P_s V with P_s from tensor memory
//   warp 9           TMA: Q_s of an item, key and value tiles of 128 rows in the order of their use through one ring
//   warp 10          zeros behind the end of a sequence in its last value tile
// D = 128: two accumulators and two score tiles fill the tensor memory, so P_s lies in the columns of S_s, and S_s of the next tile follows
// P_s V (the tensor core works in issue order).  One thread issues for both query tiles, which so fall half a tile apart: the scores of one
// are computed while the other's softmax runs (documents of 16384 tokens: 482 us against 523 with a thread for
// each).  D = 64: P_s has columns of its own, and S_s of the next tile is computed as soon as the scores are in registers, by a
// thread of each query tile, so the softmax warps, which bound this size (128 exponentials a row for half the products), never wait.
//
// Measured, 32 heads over 8: 7 prompts in 32768 tokens, heads of 128: bound by the tensor core at the power limit, 3.1 ms, 1140 TFLOP/s;
// 4 documents in 16384 tokens: 0.50 ms, 1160 (tensor cores busy 66 % of the cycles, exponentials 65 %); 24 samples in 8192 tokens, heads of 64: 67 us, 346, as tiles of 128 x 128 are a half full
// and an item is a few tiles.  120 sentences in 24576 tokens, 16 heads of 64, no mask: 102 us, 301 (by the length of an item too).
#include "attn_tc_common.cuh"
#include "gemm_tcgen05.cuh"
#include "packed_items.cuh"
#include "ptx.cuh"

namespace {
using namespace nxd_attn;
using namespace nxd_packed;

constexpr int kBM = 128, kBN = 128;
constexpr int kThreads = 384;                     // 8 softmax warps, MMA, TMA, ends of sequences, MMA (registers move by groups of four warps)
constexpr float kRescale = 8.0f;                  // log2 units

struct FwdParams {
    const PackedTile* tiles;
    float* lse;
    uint8_t* rest;                                // what rounding to bf16 took from o (attn_tc_common.cuh), NULL: not wanted
    const int* which;                             // sequence of an entry; NULL: the rows of `rest` are the padded columns
    long long rest_row;
    bf16* o;
    int* gave_up;                                 // host memory (packed_items.cuh)
    long long lse_row, o_head, o_row;
    int entries, group, pairs;                    // pairs: items of one tile-list entry
    int tries;                                    // of a wait
    int pos_q[3], pos_k[3], pos_v[3], pos_o[3];
    float scale_log2;
};

template <int D>
struct FwdSmem {
    static constexpr int kTileBytes = 128 * D * 2;
    static constexpr int kSlots = D == 64 ? 6 : 4;
    static constexpr int kQOff = 0;
    static constexpr int kRingOff = 2 * kTileBytes;
    static constexpr int kOutOff = kRingOff + kSlots * kTileBytes;       // 32 rows x 64 columns of each softmax warp
    static constexpr int kBarOff = kOutOff + 8 * 4096;
    static constexpr int kNumBars = 4 + 3 * kSlots + 10 + 8;
    static constexpr int kBytes = kBarOff + kNumBars * 8 + 16 + 1024;
    // tensor memory: O_0 O_1 | S_0 S_1 | P_0 P_1 (D = 64; else P_s = the first columns of S_s)
    static constexpr bool kAlias = D == 128;
    static constexpr int kMmaThreads = kAlias ? 1 : 2;
    static constexpr uint32_t kColS = 2 * D, kColP = kAlias ? kColS : kColS + 256, kPStep = kAlias ? 128 : 64;
};
static_assert(FwdSmem<128>::kBytes <= 232448 && FwdSmem<64>::kBytes > 116 * 1024, "one CTA per SM");

struct alignas(16) Item {
    int kind, start, len, pad;           // kind: 0 end of the items (`start`: the CTA's round that comes next), 1 an item, above: that many (less
                                         // kRowsOfNone) rows from `start` are of no sequence
    int t0, t1, n0, n1;                  // query tiles and the key tiles that they meet (0: there is no second one)
    int h0, h1, hkv, rest;               // rest: row of `rest` of the sequence's first
    __device__ __forceinline__ int t(int s) const { return s ? t1 : t0; }
    __device__ __forceinline__ int n(int s) const { return s ? n1 : n0; }
    __device__ __forceinline__ int h(int s) const { return s ? h1 : h0; }
};

template <bool CAUSAL, bool HEADS>
__device__ __forceinline__ Item fetch_item(const FwdParams& p, int round) {
    const unsigned at = item_of_round(round);
    Item it{};
    if (at >= (unsigned)p.entries * p.pairs) return it;
    const unsigned e = at / (unsigned)p.pairs;
    const int pr = (int)(at - e * p.pairs);
    const PackedTile pt = packed_tile(p.tiles, (int)e);
    it.start = pt.start, it.len = pt.len, it.pad = it.rest = pt.pad;
    if (p.which != nullptr) it.rest = (int)((unsigned)p.which[e] * kBN);          // (of no use where the entry is no item)
    it.h0 = HEADS ? 2 * pr : pr;
    it.h1 = HEADS ? it.h0 + 1 : it.h0;
    if (pt.len == 0) {                   // behind all items; an entry without anything: all that follow are like it
        it.kind = pt.t > 0 ? pt.t + kRowsOfNone : 0;
        return it;
    }
    const int all = (pt.len + kBN - 1) / kBN;
    it.kind = 1;
    it.hkv = it.h0 / p.group;
    it.t0 = HEADS ? pt.t : 2 * pt.t;     // entries are of 128 rows, or of 256 where an item is two tiles of one head
    it.t1 = HEADS ? pt.t : 2 * pt.t + 1;
    it.n0 = CAUSAL ? it.t0 + 1 : all;
    it.n1 = it.t1 < all ? (CAUSAL ? it.t1 + 1 : all) : 0;
    return it;
}

constexpr int kItemReaders = 9;          // besides the MMA threads: a lane of each softmax warp and of the one that cuts value tiles

__device__ __forceinline__ float max3(float a, float b, float c) {          // NaN if one of them is
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float max2(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// What a CTA that gave up a wait leaves: NaN for all its items, those among them that were ready, and zeros for rows of no sequence.
template <int D, bool CAUSAL, bool HEADS>
__device__ __forceinline__ void leave_nan(const FwdParams& p) {
    for (int round = 0;; ++round) {
        const Item x = fetch_item<CAUSAL, HEADS>(p, round);
        if (x.kind == 0) break;
        for (int s = 0; s < 2; ++s) {
            if (x.kind > 1 ? s == 1 && !HEADS : x.n(s) == 0) continue;
            const int first = x.kind > 1 ? 0 : x.t(s) * kBM, rows = x.kind > 1 ? x.kind - kRowsOfNone : min(x.len - first, kBM);
            const uint32_t fill = x.kind > 1 ? 0u : 0x7fff7fffu;
            for (int i = threadIdx.x; i < rows * (D / 8); i += kThreads)
                *reinterpret_cast<uint4*>(p.o + x.h(s) * p.o_head + (long long)(x.start + first + i / (D / 8)) * p.o_row + (i % (D / 8)) * 8) =
                    make_uint4(fill, fill, fill, fill);
            if (x.kind == 1 && p.lse != nullptr)
                for (int i = threadIdx.x; i < rows; i += kThreads) p.lse[x.h(s) * p.lse_row + x.pad + first + i] = NAN;
        }
    }
    if (threadIdx.x == 0) *reinterpret_cast<volatile int*>(p.gave_up) = 1;
}

template <int D, bool CAUSAL, bool HEADS>
__global__ void __launch_bounds__(kThreads, 1)
packed_fwd_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                  const __grid_constant__ CUtensorMap tmap_v, const __grid_constant__ CUtensorMap tmap_o,
                  const __grid_constant__ FwdParams p) {
    using L = FwdSmem<D>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    __shared__ int dead_word;
    __shared__ Item item_ring[kItems];
    uint8_t* smem = ptx::align_smem_1024(smem_raw);
    uint8_t* sQ = smem + L::kQOff;
    uint8_t* sRing = smem + L::kRingOff;
    uint64_t* q_full = reinterpret_cast<uint64_t*>(smem + L::kBarOff);
    uint64_t* q_empty = q_full + 2;
    uint64_t* kv_full = q_empty + 2;
    uint64_t* kv_empty = kv_full + L::kSlots;
    uint64_t* kv_cut = kv_empty + L::kSlots;
    uint64_t* s_full = kv_cut + L::kSlots;
    uint64_t* s_empty = s_full + 2;
    uint64_t* p_half = s_empty + 2;
    uint64_t* p_full = p_half + 2;
    uint64_t* pv_done = p_full + 2;
    uint64_t* item_full = pv_done + 2;
    uint64_t* item_empty = item_full + kItems;
    uint32_t* tmem_ptr_smem = reinterpret_cast<uint32_t*>(item_empty + kItems);
    volatile int* dead = &dead_word;

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        dead_word = p.tries - kTries;
        for (int s = 0; s < 2; ++s) {
            ptx::mbar_init(&q_full[s], 1);
            ptx::mbar_init(&q_empty[s], 1);
            ptx::mbar_init(&s_full[s], 1);
            ptx::mbar_init(&s_empty[s], 128);
            ptx::mbar_init(&p_half[s], 128);
            ptx::mbar_init(&p_full[s], 128);
            ptx::mbar_init(&pv_done[s], 1);
        }
        for (int i = 0; i < L::kSlots; ++i) {
            ptx::mbar_init(&kv_full[i], 1);
            ptx::mbar_init(&kv_empty[i], L::kMmaThreads);
            ptx::mbar_init(&kv_cut[i], 1);
        }
        for (int i = 0; i < kItems; ++i) {
            ptx::mbar_init(&item_full[i], 1);
            ptx::mbar_init(&item_empty[i], kItemReaders + L::kMmaThreads);
        }
        ptx::fence_barrier_init();
    }
    if (warp == 9 && lane == 0) {
        ptx::prefetch_tensormap(&tmap_q);
        ptx::prefetch_tensormap(&tmap_k);
        ptx::prefetch_tensormap(&tmap_v);
        ptx::prefetch_tensormap(&tmap_o);
    }
    if (warp == 8) ptx::tmem_alloc<1>(tmem_ptr_smem, 512);
    pdl_wait();
    ptx::tcgen05_fence_before();
    __syncthreads();
    ptx::tcgen05_fence_after();
    pdl_trigger();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_ptr_smem, 0);

    // 168 registers a thread at launch: 208 for the scores of a row, 88 for the others (256 x 208 + 128 x 88 = 384 x 168)
    if (warp == 9) {
        // ============================ TMA ============================
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        int it = 0, loads[2] = {0, 0}, round = 0, published = 0;
        // the item whose keys come next and its next key tile; the same of the values, which are one tile behind at most
        Item ki{}, vi{}, ahead = fetch_item<CAUSAL, HEADS>(p, round++);
        int kj = 0, vj = 0;
        // Goes on to the next item, of which the last value tile of this one must not wait for more than one: the readers take one more
        // before they end this one.  Rows of no sequence are behind all items and do not go through the ring.
        auto publish = [&]() {
            ki = ahead;
            if (__shfl_sync(0xffffffffu, gave_up(dead), 0)) ki.kind = 0;
            if (ki.kind == 1) {              // the one behind it is read meanwhile
                ahead = fetch_item<CAUSAL, HEADS>(p, round++);
            } else {
                ki = Item{};
                ki.start = round - 1;
            }
            publish_item(ki, item_ring, item_full, item_empty, published, dead);
            kj = 0;
        };
        auto load = [&](const CUtensorMap* map, const int* pos, uint64_t* bar, uint8_t* dst, int row, int h) {
            if (gave_up(dead)) return;           // what was loaded there before may be on its way still
            ptx::mbar_arrive_expect_tx(bar, L::kTileBytes);
            int c[4];
#pragma unroll
            for (int g = 0; g < D / 64; ++g) {
                c[0] = g * 64;
                coords(pos, row, h, 0, c);
                tma_load_4d(map, bar, dst + g * (128 * 128), c[0], c[1], c[2], c[3]);
            }
        };
        auto key_tile = [&]() {
            if (kj == 0) {
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    if (ki.n(s) == 0) continue;
                    wait_for(&q_empty[s], ((uint32_t)loads[s] & 1u) ^ 1u, dead);
                    ++loads[s];
                    if (lane == 0) load(&tmap_q, p.pos_q, &q_full[s], sQ + s * L::kTileBytes, ki.start + ki.t(s) * kBM, ki.h(s));
                }
            }
            const int slot = it % L::kSlots;
            wait_for(&kv_empty[slot], ((uint32_t)(it / L::kSlots) & 1u) ^ 1u, dead);
            if (lane == 0) load(&tmap_k, p.pos_k, &kv_full[slot], sRing + slot * L::kTileBytes, ki.start + kj * kBN, ki.hkv);
            ++it;
            ++kj;
        };
        auto value_tile = [&]() {
            const int slot = it % L::kSlots;
            wait_for(&kv_empty[slot], ((uint32_t)(it / L::kSlots) & 1u) ^ 1u, dead);
            // the tile that crosses the sequence's end goes through warp 10
            if (lane == 0)
                load(&tmap_v, p.pos_v, vi.len - vj * kBN < kBN ? &kv_cut[slot] : &kv_full[slot], sRing + slot * L::kTileBytes,
                     vi.start + vj * kBN, vi.hkv);
            ++it;
            ++vj;
        };
        publish();
        if (ki.kind == 1) key_tile();
        while (ki.kind == 1) {                // the order in which the MMA warp uses them
            vi = ki;
            vj = 0;
            const int n = max(vi.n0, vi.n1);
            for (; vj + 1 < n;) {
                if (L::kAlias) value_tile(), key_tile();
                else key_tile(), value_tile();
            }
            publish();
            value_tile();
            if (ki.kind == 1) key_tile();
        }
    } else if (warp == 8 || warp == 11) {
        // ============================ MMA ============================
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        if (warp == 8 || L::kMmaThreads == 2) if (ptx::elect_one()) {
            constexpr uint32_t idesc_s = ptx::make_idesc_bf16(kBM, kBN, 0, 0);
            constexpr uint32_t idesc_o = ptx::make_idesc_bf16(kBM, D, 0, 1);
            constexpr int kMine = 2 / L::kMmaThreads;          // query tiles of this thread, from s0
            const int s0 = warp == 8 ? 0 : 1;
            const uint32_t ring = ptx::smem_u32(sRing);
            int it = 0, items = 0, loads[kMine] = {}, tiles[kMine] = {}, done[kMine] = {};
            int n[kMine] = {}, steps = 0;     // key tiles that the query tiles meet in the item whose scores come next, and those of the item
            auto next = [&]() {
                const Item x = next_item<false, Item>(item_ring, item_full, item_empty, items, dead);
#pragma unroll
                for (int i = 0; i < kMine; ++i) n[i] = x.n(s0 + i);
                steps = max(x.n0, x.n1);
            };
            auto slot = [&]() {
                const int at = it % L::kSlots;
                wait_for(&kv_full[at], (uint32_t)(it / L::kSlots) & 1u, dead);
                ++it;
                return at;
            };
            auto scores = [&](int i, int j, int at) {          // S_s = Q_s K^T of key tile j, if query tile s meets it
                const int s = s0 + i;
                if (j >= n[i]) return;
                if (j == 0) wait_for(&q_full[s], (uint32_t)(loads[i]++) & 1u, dead);
                if (!L::kAlias) wait_for(&s_empty[s], ((uint32_t)tiles[i] & 1u) ^ 1u, dead);
                ++tiles[i];
                ptx::tcgen05_fence_after();
                const uint32_t qb = ptx::smem_u32(sQ) + s * L::kTileBytes, kb = ring + at * L::kTileBytes;
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk) {
                    const uint32_t off = (kk >> 2) * (128 * 128) + (kk & 3) * 32;
                    ptx::umma_bf16<1>(tmem + L::kColS + s * 128, ptx::make_smem_desc(qb + off, 16, 1024),
                                      ptx::make_smem_desc(kb + off, 16, 1024), idesc_s, kk != 0 ? 1u : 0u);
                }
                ptx::umma_commit(&s_full[s]);
                if (j + 1 == n[i]) ptx::umma_commit(&q_empty[s]);
            };
            auto weigh = [&](int i, int j, int meets, int at) {          // O_s += P_s V of key tile j
                const int s = s0 + i;
                if (j >= meets) return;
                const uint32_t vb = ring + at * L::kTileBytes;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    wait_for(half ? &p_full[s] : &p_half[s], (uint32_t)done[i] & 1u, dead);
                    ptx::tcgen05_fence_after();
#pragma unroll
                    for (int kk = half * 4; kk < half * 4 + 4; ++kk)
                        ptx::umma_bf16_ts(tmem + s * D, tmem + L::kColP + s * L::kPStep + kk * 8,
                                          ptx::make_smem_desc(vb + kk * 2048, kBN * 128, 1024), idesc_o, (j | kk) != 0 ? 1u : 0u);
                }
                ++done[i];
                ptx::umma_commit(&pv_done[s]);
            };
            auto all_scores = [&](int j) {
                const int at = slot();
#pragma unroll
                for (int i = 0; i < kMine; ++i) scores(i, j, at);
                ptx::umma_commit(&kv_empty[at]);
            };
            next();
            if (steps) all_scores(0);
            while (steps) {
                int meets[kMine];
#pragma unroll
                for (int i = 0; i < kMine; ++i) meets[i] = n[i];
                const int last = steps - 1;
                for (int j = 0; j < last; ++j) {
                    if (L::kMmaThreads == 2) {
                        all_scores(j + 1);
                        const int at = slot();
                        weigh(0, j, meets[0], at);
                        ptx::umma_commit(&kv_empty[at]);
                    } else {                           // the scores of one query tile while the softmax of the other runs
                        const int at = slot();
                        weigh(0, j, meets[0], at);
                        const int key = slot();
                        scores(0, j + 1, key);
                        weigh(kMine - 1, j, meets[kMine - 1], at);
                        ptx::umma_commit(&kv_empty[at]);
                        scores(kMine - 1, j + 1, key);
                        ptx::umma_commit(&kv_empty[key]);
                    }
                }
                next();
                const int at = slot();
#pragma unroll
                for (int i = 0; i < kMine; ++i) weigh(i, last, meets[i], at);
                ptx::umma_commit(&kv_empty[at]);
                if (steps) all_scores(0);
            }
        }
    } else if (warp < 8) {
        // ============================ softmax and results ============================
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        const int s = warp >> 2, q = warp & 3;
        const int row = q * 32 + lane;                   // of the query tile == TMEM lane
        const uint32_t lanes = (uint32_t)(q * 32) << 16;
        const uint32_t t_o = tmem + s * D + lanes, t_s = tmem + L::kColS + s * 128 + lanes, t_p = tmem + L::kColP + s * L::kPStep + lanes;
        const float sc = p.scale_log2;
        const uint64_t sc2 = f2_pack(sc, sc);
        int tiles = 0, items = 0;
        float m = -INFINITY, l = 0.f;                    // running maximum in units of the raw score, and sum
        // rescales what has been summed so far where the maximum has moved far; the exponent's offset
        auto follow_max = [&](float mx, int j) {
            float alpha = 1.f;
            bool rescale = false;
            if (!(mx < INFINITY)) l = NAN;               // a score that is NaN, or infinite: the row has no softmax
            if ((mx - m) * sc > kRescale || m == -INFINITY) {
                const float now = fmaxf(m, mx);
                if (now != -INFINITY) {
                    alpha = ex2_approx((m - now) * sc);
                    rescale = j > 0 && m != -INFINITY;
                    m = now;
                    l *= alpha;
                }
            }
            if (__any_sync(0xffffffffu, rescale)) {
                if (!L::kAlias) {                        // O has the weights of the tile before
                    wait_for(&pv_done[s], (uint32_t)(tiles - 1) & 1u, dead);
                    ptx::tcgen05_fence_after();
                }
                const float f = rescale ? alpha : 1.f;
                const uint64_t f2 = f2_pack(f, f);
#pragma unroll 1
                for (int c = 0; c < D / 16; ++c) {
                    uint32_t o[16];
                    ptx::tmem_ld_32x32b_x16(t_o + c * 16, o);
                    ptx::tmem_ld_wait();
#pragma unroll
                    for (int e = 0; e < 16; e += 2) {
                        const uint64_t z = f2_mul(f2_pack(__uint_as_float(o[e]), __uint_as_float(o[e + 1])), f2);
                        o[e] = (uint32_t)z;
                        o[e + 1] = (uint32_t)(z >> 32);
                    }
                    tmem_st_32x32b_x16(t_o + c * 16, o);
                }
            }
            return m == -INFINITY ? 0.f : -m * sc;
        };
        auto weights_free = [&](int j) {                 // D = 64: the weights of the tile before have been used
            if (!L::kAlias && j > 0) {
                wait_for(&pv_done[s], (uint32_t)(tiles - 1) & 1u, dead);
                ptx::tcgen05_fence_after();
            }
        };
        auto scores_read = [&]() {
            ptx::tmem_ld_wait();
            if (!L::kAlias) {
                ptx::tcgen05_fence_before();
                ptx::mbar_arrive(&s_empty[s]);
            }
        };
        // One tile: weights of its 128 columns, the row's maximum and sum; `mine` columns count for this row, `seen` for any of the warp.
        // All of one path: a tile on the diagonal or at the end of a sequence takes the same instructions behind its mask (chunks of 32
        // columns that were left out by branches made such a tile a half longer than a whole one).
        auto tile_weights = [&](int j, int seen, int mine) {
            uint32_t x[kBN];
            uint64_t sum[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll
            for (int c = 0; c < 4; ++c) ptx::tmem_ld_32x32b_x32(t_s + c * 32, x + c * 32);
            scores_read();
            if (__any_sync(0xffffffffu, mine < kBN)) {
#pragma unroll
                for (int e = 0; e < kBN; ++e) x[e] = e < mine ? x[e] : 0xff800000u;          // -inf
            }
            float a[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) a[i] = max3(__uint_as_float(x[i]), __uint_as_float(x[8 + i]), __uint_as_float(x[16 + i]));
#pragma unroll
            for (int e = 24; e < 120; e += 16)
#pragma unroll
                for (int i = 0; i < 8; ++i) a[i] = max3(a[i], __uint_as_float(x[e + i]), __uint_as_float(x[e + 8 + i]));
#pragma unroll
            for (int i = 0; i < 8; ++i) a[i] = max2(a[i], __uint_as_float(x[120 + i]));
            const float neg = follow_max(max3(max3(a[0], a[1], a[2]), max3(a[3], a[4], a[5]), max2(a[6], a[7])), j);
            const uint64_t neg2 = f2_pack(neg, neg);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                if (half && seen <= 64) {                        // no row of the warp sees the second half
#pragma unroll
                    for (int e = 0; e < 32; ++e) x[32 + e] = 0u;
                } else {
#pragma unroll
                    for (int e = 0; e < 64; e += 2) {
                        const int i = half * 64 + e;
                        const uint64_t z = f2_fma(f2_pack(__uint_as_float(x[i]), __uint_as_float(x[i + 1])), sc2, neg2);
                        const float p0 = ex2_approx(f2_lo(z)), p1 = ex2_approx(f2_hi(z));
                        sum[(e >> 1) & 3] = f2_add(sum[(e >> 1) & 3], f2_pack(p0, p1));
                        x[i >> 1] = pack_bf16x2(p0, p1);
                    }
                }
                if (half == 0) weights_free(j);
                tmem_st_32x32b_x32(t_p + half * 32, x + half * 32);
                tmem_st_wait();
                ptx::tcgen05_fence_before();
                ptx::mbar_arrive(half ? &p_full[s] : &p_half[s]);
            }
            const uint64_t all = f2_add(f2_add(sum[0], sum[1]), f2_add(sum[2], sum[3]));
            l += f2_lo(all) + f2_hi(all);
        };
        Item it = next_item<true, Item>(item_ring, item_full, item_empty, items, dead);
        for (; it.kind != 0;) {
            const int head = it.h(s), n = it.n(s), t = it.t(s);
            if (n == 0) {
                it = next_item<true, Item>(item_ring, item_full, item_empty, items, dead);
                continue;
            }
            m = -INFINITY, l = 0.f;
            for (int j = 0; j < n; ++j, ++tiles) {
                int seen = min(it.len - j * kBN, kBN);
                const bool diagonal = CAUSAL && j == t;
                const int mine = diagonal ? min(seen, row + 1) : seen;
                if (diagonal) seen = min(seen, q * 32 + 32);
                wait_for(&s_full[s], (uint32_t)tiles & 1u, dead);
                ptx::tcgen05_fence_after();
                tile_weights(j, seen, mine);
            }
            const Item done = it;                        // the next one is read while the last products run
            it = next_item<true, Item>(item_ring, item_full, item_empty, items, dead);
            // O / l, one row a thread, nothing behind the sequence's end.  A row without a finite score has no softmax.
            wait_for(&pv_done[s], (uint32_t)(tiles - 1) & 1u, dead);
            ptx::tcgen05_fence_after();
            const int at = t * kBM + row;
            const bool real = at < done.len;
            if (m == -INFINITY) l = NAN;
            const float inv = 1.f / l;
            if (p.lse != nullptr && real) p.lse[head * p.lse_row + done.pad + at] = m * sc + log2f(l);
            // through shared memory, 32 rows x 64 columns at a time: stored by rows from the registers, a warp's 16-byte pieces fall into
            // 32 different lines, and the end of an item took 5000 clocks
            const int first = t * kBM + q * 32;              // row of the warp in its sequence
            uint8_t* stage = smem + L::kOutOff + warp * 4096;
#pragma unroll 1
            for (int g = 0; g < D / 64; ++g) {
                uint32_t o[64];
                ptx::tmem_ld_32x32b_x32(t_o + g * 64, o);
                ptx::tmem_ld_32x32b_x32(t_o + g * 64 + 32, o + 32);
                ptx::tmem_ld_wait();
                if (lane == 0) ptx::bulk_wait_read<0>();     // what was stored from here before
                __syncwarp();
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    uint32_t w[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        w[i] = pack_bf16x2(__uint_as_float(o[8 * c + 2 * i]) * inv, __uint_as_float(o[8 * c + 2 * i + 1]) * inv);
                    st_shared_v4(stage + lane * 128 + ((c ^ (lane & 7)) << 4), w[0], w[1], w[2], w[3]);
                }
                if (p.rest != nullptr && n == 1) {           // eight bits of what the rounding took, for Delta of the backward pass
                    uint32_t most = 0u;
#pragma unroll
                    for (int e = 0; e < 64; e += 2) {
                        o[e] = __float_as_uint(__uint_as_float(o[e]) * inv);
                        o[e + 1] = __float_as_uint(__uint_as_float(o[e + 1]) * inv);
                        most = __vmaxu2(most, pack_bf16x2(__uint_as_float(o[e]), __uint_as_float(o[e + 1])) & 0x7fff7fffu);
                    }
                    const float up = rest_up(most);
                    uint8_t* to = p.rest + rest_offset<D>(head * p.rest_row + done.rest + at, g * 4);
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        uint32_t w[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint32_t* x = o + 16 * c + 4 * i;
                            w[i] = rest_pack(__uint_as_float(x[0]), __uint_as_float(x[1]), __uint_as_float(x[2]), __uint_as_float(x[3]), up);
                        }
                        if (real) *reinterpret_cast<uint4*>(to + c * 64) = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
                if (first + 32 <= done.len) {
                    ptx::fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) {
                        int c[4];
                        c[0] = g * 64;
                        coords(p.pos_o, done.start + first, head, 0, c);
                        tma_store_4d(&tmap_o, stage, c[0], c[1], c[2], c[3]);
                        ptx::bulk_commit();
                    }
                } else {                                     // the rows behind the end are the next sequence's
                    __syncwarp();
                    bf16* to = p.o + head * p.o_head + (long long)(done.start + first) * p.o_row + g * 64;
                    for (int i = lane; i < 32 * 8; i += 32) {
                        const int r = i >> 3, ch = i & 7;
                        if (first + r < done.len)
                            *reinterpret_cast<uint4*>(to + r * p.o_row + ch * 8) =
                                *reinterpret_cast<const uint4*>(stage + r * 128 + ((ch ^ (r & 7)) << 4));
                    }
                    __syncwarp();
                }
            }
            ptx::tcgen05_fence_before();
        }
        // zeros for rows of no sequence, once a head
        for (int round = it.start;; ++round) {
            it = fetch_item<CAUSAL, HEADS>(p, round);
            if (it.kind <= 1) break;
            if (HEADS || s == 0)
                for (int i = threadIdx.x & 127; i < (it.kind - kRowsOfNone) * (D / 8); i += 128)
                    *reinterpret_cast<uint4*>(p.o + it.h(s) * p.o_head + (long long)(it.start + i / (D / 8)) * p.o_row + (i % (D / 8)) * 8) =
                        make_uint4(0u, 0u, 0u, 0u);
        }
        if (lane == 0) ptx::bulk_wait<0>();
    } else if (warp == 10) {
        // ============================ ends of sequences ============================
        // Behind the end of a sequence a value tile holds the next one, and 0 * NaN is NaN: those rows become zeros once the tile is there.
        // (Tiles that a warp copied with zeros instead were 4000 clocks late.)
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        int it = 0, items = 0;
        uint32_t phases = 0;
        for (;;) {
            const Item x = next_item<true, Item>(item_ring, item_full, item_empty, items, dead);
            if (x.kind == 0) break;
            const int n = max(x.n0, x.n1), left = x.len - (n - 1) * kBN;
            it += 2 * n;                       // keys and values of the item; its last values are the last of them
            if (left >= kBN) continue;
            const int slot = (it - 1) % L::kSlots;
            wait_for(&kv_cut[slot], (phases >> slot) & 1u, dead);
            phases ^= 1u << slot;
            uint8_t* tile = sRing + slot * L::kTileBytes;
            for (int i = lane; i < (kBN - left) * (D / 8); i += 32) {
                const int r = left + i / (D / 8), ch = i % (D / 8);
                st_shared_v4(tile + (ch >> 3) * (128 * 128) + r * 128 + ((ch & 7) << 4), 0u, 0u, 0u, 0u);
            }
            ptx::fence_proxy_async();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(&kv_full[slot]);
        }
    }
    ptx::tcgen05_fence_before();
    __syncthreads();
    if (gave_up(dead)) {
        let_copies_land();
        leave_nan<D, CAUSAL, HEADS>(p);
    }
    if (warp == 8) ptx::tmem_dealloc<1>(tmem, 512);
}

template <int D, bool CAUSAL, bool HEADS>
int launch(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const CUtensorMap& to, const FwdParams& p, cudaStream_t st) {
    using L = FwdSmem<D>;
    constexpr auto kern = packed_fwd_kernel<D, CAUSAL, HEADS>;
    NXD_CHECK_CUDA(nxd_allow_smem<kern>(L::kBytes));
    const long long items = (long long)p.entries * p.pairs;
    const unsigned grid = (unsigned)(items < nxd_num_sms() ? items : nxd_num_sms());
    NXD_CHECK_CUDA(nxd_launch_pdl(kern, dim3(grid), dim3(kThreads), L::kBytes, st, tq, tk, tv, to, p));
    NXD_LAUNCH_CHECK();
    return 0;
}

template <int D>
int launch_as(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const CUtensorMap& to, const FwdParams& p, int causal, cudaStream_t st) {
    if (p.group % 2 == 0) return causal ? launch<D, true, true>(tq, tk, tv, to, p, st) : launch<D, false, true>(tq, tk, tv, to, p, st);
    return causal ? launch<D, true, false>(tq, tk, tv, to, p, st) : launch<D, false, false>(tq, tk, tv, to, p, st);
}

}  // namespace

// The word is there as long as the process, for graphs that are replayed.
int nxd_packed::begin_call(int** word) {
    static int* const shared = [] {
        int* w = nullptr;
        cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;          // the first call may be a captured one
        cudaThreadExchangeStreamCaptureMode(&mode);
        if (cudaHostAlloc((void**)&w, sizeof(int), cudaHostAllocPortable | cudaHostAllocMapped) != cudaSuccess) w = nullptr;
        cudaThreadExchangeStreamCaptureMode(&mode);
        if (w != nullptr) *w = 0;
        return w;
    }();
    NXD_REQUIRE(shared != nullptr, "packed_attn: no host memory for %s", "the status word");
    *word = shared;
    NXD_REQUIRE(__atomic_exchange_n(shared, 0, __ATOMIC_RELAXED) == 0, "packed_attn: a call before this one gave up a wait; %s", "its results are NaN");
    return 0;
}

// *gave_up <- whether a call gave up a wait since the last one that failed or asked for it.  Waits for the stream.
NXD_API int nxd_packed_attn_status(int* gave_up, void* stream) {
    int* word;
    NXD_CHECK_CUDA(cudaStreamSynchronize((cudaStream_t)stream));
    *gave_up = nxd_packed::begin_call(&word) != 0;
    return 0;
}

// Attention inside each sequence of a packed batch: q [T, Hq, D], k and v [T, Hkv, D], o [T, Hq, D], strides {q_h, q_row, k_h,
// k_row, v_h, v_row, o_h, o_row} in elements (multiples of 8), 16-byte aligned bases; tiles: the `entries` tiles that
// nxd_packed_plan has made; lse NULL or [Hq, lse_row] floats, log2 units, written at the plan's padded columns; rest NULL or [Hq, rest_row,
// D] bytes, for the backward pass, where rest_row is 128 for each sequence and `which` the plan's, or NULL and rest_row is lse_row.  Rows outside every sequence get zeros.  wait_tries: after which a wait gives up, -1: two seconds.
NXD_API int nxd_packed_attn_fwd(const void* q, const void* k, const void* v, void* o, float* lse, void* rest, const long long* strides,
                                const void* tiles, const int* which, long long rest_row, int entries, long long lse_row, long long T, int Hq, int Hkv, int D, float scale,
                                int causal, int wait_tries, void* stream) {
    NXD_REQUIRE(D == 64 || D == 128, "packed_attn: head dim %d not supported (64 or 128)", D);
    NXD_REQUIRE(T > 0 && T < (1ll << 31) - 256 && Hq > 0 && Hkv > 0 && Hq % Hkv == 0 && entries > 0 && (long long)entries * Hq < (1ll << 31),
                "packed_attn: bad problem");
    NXD_REQUIRE(scale >= 1.17549435e-38f && scale <= 1.7014118e38f, "packed_attn: a scale of %g", scale);
    for (int i = 0; i < 8; ++i)
        NXD_REQUIRE(strides[i] % 8 == 0, "packed_attn: stride %d (=%lld) must be a multiple of 8 elements", i, strides[i]);
    NXD_REQUIRE(q && k && v && o && tiles && (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)o | (uintptr_t)rest | (uintptr_t)tiles) & 15) == 0 && lse_row % 4 == 0 && rest_row % 4 == 0,
                "packed_attn: tensors must be 16-byte aligned, rows of the scratch multiples of four");
    NXD_REQUIRE(rest == nullptr || rest_row >= (which ? kBN : lse_row), "packed_attn: %lld rows of what the rounding took", rest_row);
    FwdParams p{};
    int rc;
    if ((rc = begin_call(&p.gave_up))) return rc;
    p.tries = wait_tries < 0 || wait_tries > kTries ? kTries : wait_tries;
    p.tiles = (const PackedTile*)tiles;
    p.entries = entries;
    p.lse = lse; p.lse_row = lse_row;
    p.rest = (uint8_t*)rest; p.which = rest ? which : nullptr; p.rest_row = rest_row;
    p.group = Hq / Hkv;
    p.pairs = p.group % 2 == 0 ? Hq / 2 : Hq;
    p.scale_log2 = scale * 1.4426950408889634f;
    p.o = (bf16*)o; p.o_head = strides[6]; p.o_row = strides[7];
    CUtensorMap tq, tk, tv, to;
    if ((rc = make_tmap_bhsd(&tq, q, D, T, Hq, 1, strides[1], strides[0], 0, kBM, p.pos_q))) return rc;
    if ((rc = make_tmap_bhsd(&tk, k, D, T, Hkv, 1, strides[3], strides[2], 0, kBN, p.pos_k))) return rc;
    if ((rc = make_tmap_bhsd(&tv, v, D, T, Hkv, 1, strides[5], strides[4], 0, kBN, p.pos_v))) return rc;
    if ((rc = make_tmap_bhsd(&to, o, D, T, Hq, 1, strides[7], strides[6], 0, 32, p.pos_o))) return rc;
    cudaStream_t st = (cudaStream_t)stream;
    return D == 64 ? launch_as<64>(tq, tk, tv, to, p, causal, st) : launch_as<128>(tq, tk, tv, to, p, causal, st);
}
