// Attention over packed sequences, backward, on 5th-gen tensor cores (tcgen05 + TMEM + TMA), sm_100a.
//
//   P = exp2(S - L), dS = P (dP - Delta), dP = dO V^T, Delta = rowsum(O dO);  dV = P^T dO, dK = scale dS^T Q, dQ = scale dS K
//
// The products and their layouts are those of flash_attn_bwd_tc.cu: a block of 128 key rows of one key head against the query tiles (64
// rows) of its query heads, scores transposed so that a thread owns a key row; dK and dV stay in tensor memory over the walk, dQ is
// added tile by tile to a d-major fp32 accumulator by TMA, in an order that is not fixed.
//
// Here one CTA per SM stays for the whole call (items: packed_items.cuh; the list is sorted by the key tiles that a query tile meets, and
// mirrored for key blocks: the block as far from the end meets as many query rows).  A block of a short sequence meets a few
// query tiles, and with a CTA per block its start, its end and the copies of tiles that cross the sequence's end by a warp were
// more than half of the time (120 sentences in 24576 tokens, 16 heads of 64, no mask: 410 us against 210).  Tiles that cross the end
// are loaded whole and cleared behind it once they are there: 0 * NaN is NaN, and behind the end is the next sequence.
//
// Measured (the whole pass: Delta, this kernel, dQ): 4 documents in 16384 tokens, 32 heads of 128 over 8: 1.8 ms, 810 TFLOP/s, shared memory
// busy 82 % of the cycles, the tensor cores 60 %, under the power limit; one sequence of 16384 tokens, 16 heads of 128 over 4: 990 TFLOP/s,
// the dense kernel in turn 1011; 24 samples in 8192 tokens, heads of 64: 171 us, 338; the sentences above: 290 us, 265, where a block's end (dK, dV out of tensor memory, while
// nothing else may use it) and 69 us of passes over the fp32 accumulator weigh most.  Two pairs of accumulators for heads of 64, so that
// the warps of dQ write the results under the next block: 309 us instead of 297, since those warps then hold up dQ.
//   warp 0      claims items; TMA: K, V of an item, then Q_i, dO_i, L_i, Delta_i through a ring of three; zeros behind the end of a sequence
//   warp 1      MMA: S^T = K Q^T, dP^T = V dO^T, dV += P^T dO, dK += dS^T Q, dQ^T = K^T dS^T
//   warps 2-9   P^T and dS^T, two warps to a lane quadrant with 32 of the 64 queries each; then dV (one half) and dK (the other)
//   warps 10-13 dQ^T -> fp32 accumulator
#include "attn_tc_common.cuh"
#include "gemm_tcgen05.cuh"
#include "packed_items.cuh"
#include "ptx.cuh"

#include <type_traits>

namespace {
using namespace nxd_attn;
using namespace nxd_packed;

constexpr int kBN = 128;              // key rows of a block
constexpr int kBM = 64;               // query rows of a tile
constexpr int kThreads = 448;
constexpr int kMathThreads = 256;
constexpr int kDrainThreads = 128;
constexpr int kItemReaders = 1 + 8 + 4;
constexpr int kStages = 3;            // of Q_i, dO_i, L_i, Delta_i: a tile is asked for one iteration before its products

struct BwdParams {
    const PackedTile* tiles;
    const float *lse, *delta;
    int* claimed;                // items that were given out behind everybody's first; then whether a CTA gave up a wait
    int* gave_up;                // host memory (packed_items.cuh)
    int tries;                   // of a wait
    bf16 *dk, *dv;
    long long lse_row, dk_head, dk_row, dv_head, dv_row;
    int entries, Hkv, group, nsplit;          // nsplit: items that share a key block; each walks its part of the (head, query tile) list
    int pos_q[3], pos_do[3], pos_k[3], pos_v[3], pos_dq[3], pos_acc[3];
    float scale, scale_log2;
};

template <int D>
struct BwdSmem {
    static constexpr int kBufs = D == 64 ? 2 : 1;           // of K and of V: the next block's are loaded under this one's end
    static constexpr int kKvBytes = kBN * D * 2, kStageBytes = kBM * D * 2;
    static constexpr int kKOff = 0;
    static constexpr int kVOff = kKOff + kBufs * kKvBytes;
    static constexpr int kQOff = kVOff + kBufs * kKvBytes;
    static constexpr int kDOOff = kQOff + kStages * kStageBytes;
    static constexpr int kOutOff = kDOOff + kStages * kStageBytes;       // 1 KB of each math warp
    static constexpr int kDStOff = kOutOff + 8 * 1024;
    static constexpr int kDQOff = kDStOff + kBN * kBM * 2;
    static constexpr int kLOff = kDQOff + kBM * D * 4;
    static constexpr int kBarOff = kLOff + kStages * 2 * kBM * 4;
    static constexpr int kNumBars = 5 * 2 + 3 * kStages + 6 + 2 * kItems;
    static constexpr int kBytes = kBarOff + kNumBars * 8 + 16 + 1024;
    static constexpr int kTxPerStage = 2 * kStageBytes + 2 * kBM * 4;
};
static_assert(BwdSmem<128>::kBytes + 2048 <= 232448 && BwdSmem<64>::kBytes > 116 * 1024, "one CTA per SM");

struct alignas(16) Item {
    int kind, start, len, pad;           // kind: 0 end of the list, 1 an item, above: that many (less kRowsOfNone) rows from `start` are of no sequence
    int n0, first, per_head, total;      // first key row; first query tile and number of them per head; tiles of this item
    int th, head, hkv, unused;           // where the item's walk starts: query tile (from `first`) and query head
    __device__ __forceinline__ bool keys_cut() const { return n0 + kBN > len; }
};

template <bool CAUSAL>
__device__ __forceinline__ Item fetch_item(const BwdParams& p, unsigned at) {
    const unsigned per = (unsigned)(p.Hkv * p.nsplit);
    Item it{};
    if (at >= (unsigned)p.entries * per) return it;
    const unsigned e = at / per, r = at - e * per;
    const PackedTile pt = packed_tile(p.tiles, (int)e);
    it.start = pt.start, it.len = pt.len, it.pad = pt.pad;
    it.hkv = (int)r / p.nsplit;
    const int split = (int)r % p.nsplit;
    if (pt.len == 0) {                   // with splits dK and dV come from accumulators that start as zeros
        it.kind = pt.t > 0 ? (split == 0 && p.nsplit == 1 ? pt.t : 0) + kRowsOfNone + 1 : 0;
        return it;
    }
    it.kind = 1;
    it.n0 = ((pt.len + kBN - 1) / kBN - 1 - pt.t) * kBN;
    it.first = CAUSAL ? it.n0 / kBM : 0;
    it.per_head = (pt.len + kBM - 1) / kBM - it.first;
    const int all = it.per_head * p.group, from = (int)((long long)all * split / p.nsplit);
    it.total = (int)((long long)all * (split + 1) / p.nsplit) - from;
    it.th = from % it.per_head;
    it.head = it.hkv * p.group + from / it.per_head;
    if (it.total == 0) it.kind = kRowsOfNone + 1;          // nothing to do, as for no rows
    return it;
}

template <int D, bool CAUSAL>
__global__ void __launch_bounds__(kThreads, 1)
packed_bwd_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_do,
                  const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                  const __grid_constant__ CUtensorMap tmap_dq, const __grid_constant__ CUtensorMap tmap_dk_acc,
                  const __grid_constant__ CUtensorMap tmap_dv_acc, const __grid_constant__ BwdParams p) {
    using L = BwdSmem<D>;
    constexpr uint32_t kColDK = 0, kColDV = D, kColST = 2 * D, kColDPT = 2 * D + 64, kColDQT = 2 * D + 128;
    constexpr uint32_t kColPT = 2 * D + 192, kColDST = kColPT + 32;          // bf16 P^T and dS^T, 128 lanes x 64 queries
    static_assert(kColDST + 32 <= 512, "tensor memory budget");
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    __shared__ int dead_word;
    __shared__ Item item_ring[kItems];
    uint8_t* smem = ptx::align_smem_1024(smem_raw);
    uint8_t* sK = smem + L::kKOff;
    uint8_t* sV = smem + L::kVOff;
    uint8_t* sQ = smem + L::kQOff;
    uint8_t* sDO = smem + L::kDOOff;
    uint8_t* sDSt = smem + L::kDStOff;
    uint8_t* sDQ = smem + L::kDQOff;
    float* sLD = reinterpret_cast<float*>(smem + L::kLOff);  // [stage][0: L, 1: Delta][64]
    uint64_t* k_full = reinterpret_cast<uint64_t*>(smem + L::kBarOff);      // [2] each, of which kBufs are used
    uint64_t* k_cut = k_full + 2;
    uint64_t* k_empty = k_cut + 2;
    uint64_t* v_full = k_empty + 2;
    uint64_t* v_empty = v_full + 2;
    uint64_t* qdo_full = v_empty + 2;
    uint64_t* qdo_cut = qdo_full + kStages;
    uint64_t* qdo_empty = qdo_cut + kStages;
    uint64_t* st_full = qdo_empty + kStages;
    uint64_t* st_empty = st_full + 1;
    uint64_t* pds_full = st_full + 2;
    uint64_t* pds_empty = st_full + 3;
    uint64_t* dq_full = st_full + 4;
    uint64_t* dq_empty = st_full + 5;
    uint64_t* item_full = st_full + 6;
    uint64_t* item_empty = item_full + kItems;
    uint32_t* tmem_ptr_smem = reinterpret_cast<uint32_t*>(item_empty + kItems);
    volatile int* dead = &dead_word;

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        dead_word = p.tries - kTries;
        for (int i = 0; i < 2; ++i) {
            ptx::mbar_init(&k_full[i], 1);
            ptx::mbar_init(&k_cut[i], 1);
            ptx::mbar_init(&k_empty[i], 1);
            ptx::mbar_init(&v_full[i], 1);
            ptx::mbar_init(&v_empty[i], 1);
        }
        for (int i = 0; i < kStages; ++i) {
            ptx::mbar_init(&qdo_full[i], 1);
            ptx::mbar_init(&qdo_cut[i], 1);
            ptx::mbar_init(&qdo_empty[i], 1);
        }
        ptx::mbar_init(st_full, 1);
        ptx::mbar_init(st_empty, kMathThreads);
        ptx::mbar_init(pds_full, kMathThreads);
        ptx::mbar_init(pds_empty, 1);
        ptx::mbar_init(dq_full, 1);
        ptx::mbar_init(dq_empty, kDrainThreads);
        for (int i = 0; i < kItems; ++i) {
            ptx::mbar_init(&item_full[i], 1);
            ptx::mbar_init(&item_empty[i], kItemReaders);
        }
        ptx::fence_barrier_init();
    }
    if (warp == 0 && lane == 0) {
        ptx::prefetch_tensormap(&tmap_q);
        ptx::prefetch_tensormap(&tmap_do);
        ptx::prefetch_tensormap(&tmap_k);
        ptx::prefetch_tensormap(&tmap_v);
        ptx::prefetch_tensormap(&tmap_dq);
    }
    pdl_wait();         // ahead of the allocation: nothing that this grid waits for may be short of tensor memory
    if (warp == 1) ptx::tmem_alloc<1>(tmem_ptr_smem, 512);
    ptx::tcgen05_fence_before();
    __syncthreads();
    ptx::tcgen05_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_ptr_smem, 0);

    if (warp == 0) {
        // ============================ TMA ============================
        int published = 0, blocks = 0, gi = 0;
        uint32_t k_phases = 0, q_phases = 0;
        auto clear = [&](uint8_t* tile, int rows, int left) {
            for (int i = lane; i < (rows - left) * (D / 8); i += 32) {
                const int r = left + i / (D / 8), ch = i % (D / 8);
                st_shared_v4(tile + (ch >> 3) * (rows * 128) + r * 128 + ((ch & 7) << 4), 0u, 0u, 0u, 0u);
            }
        };
        auto cleared = [&](uint64_t* bar) {
            ptx::fence_proxy_async();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(bar);
        };
        auto claim = [&]() {
            unsigned at = 0;
            if (lane == 0) at = (unsigned)atomicAdd(p.claimed, 1);
            return fetch_item<CAUSAL>(p, gridDim.x + __shfl_sync(0xffffffffu, at, 0));
        };
        for (Item x = fetch_item<CAUSAL>(p, blockIdx.x);; x = claim()) {          // the last tiles are still worked on when the next item is asked for
            publish_item(x, item_ring, item_full, item_empty, published, dead);
            if (x.kind == 0 || __shfl_sync(0xffffffffu, gave_up(dead), 0)) break;
            if (x.kind > 1) continue;
            const int buf = blocks % L::kBufs;
            const uint32_t ph = ((uint32_t)(blocks / L::kBufs) & 1u) ^ 1u;
            ++blocks;
            int c[4];
            wait_for(&v_empty[buf], ph, dead);
            if (lane == 0 && !gave_up(dead)) {
                ptx::mbar_arrive_expect_tx(&v_full[buf], L::kKvBytes);
#pragma unroll
                for (int g = 0; g < D / 64; ++g) {
                    c[0] = g * 64;
                    coords(p.pos_v, x.start + x.n0, x.hkv, 0, c);
                    tma_load_4d(&tmap_v, &v_full[buf], sV + buf * L::kKvBytes + g * (kBN * 128), c[0], c[1], c[2], c[3]);
                }
            }
            wait_for(&k_empty[buf], ph, dead);
            if (lane == 0 && !gave_up(dead)) {
                uint64_t* bar = x.keys_cut() ? &k_cut[buf] : &k_full[buf];
                ptx::mbar_arrive_expect_tx(bar, L::kKvBytes);
#pragma unroll
                for (int g = 0; g < D / 64; ++g) {
                    c[0] = g * 64;
                    coords(p.pos_k, x.start + x.n0, x.hkv, 0, c);
                    tma_load_4d(&tmap_k, bar, sK + buf * L::kKvBytes + g * (kBN * 128), c[0], c[1], c[2], c[3]);
                }
            }
            int th = x.th, hq = x.head;
            for (int it = 0; it < x.total; ++it, ++gi) {
                const int st = gi % kStages, m0 = (x.first + th) * kBM;
                wait_for(&qdo_empty[st], ((uint32_t)(gi / kStages) & 1u) ^ 1u, dead);
                if (lane == 0 && !gave_up(dead)) {
                    uint64_t* bar = m0 + kBM > x.len ? &qdo_cut[st] : &qdo_full[st];
                    ptx::mbar_arrive_expect_tx(bar, L::kTxPerStage);
#pragma unroll
                    for (int g = 0; g < D / 64; ++g) {
                        c[0] = g * 64;
                        coords(p.pos_q, x.start + m0, hq, 0, c);
                        tma_load_4d(&tmap_q, bar, sQ + st * L::kStageBytes + g * (kBM * 128), c[0], c[1], c[2], c[3]);
                        coords(p.pos_do, x.start + m0, hq, 0, c);
                        tma_load_4d(&tmap_do, bar, sDO + st * L::kStageBytes + g * (kBM * 128), c[0], c[1], c[2], c[3]);
                    }
                    const long long row = hq * p.lse_row + x.pad + m0;
                    bulk_load_1d(sLD + st * 2 * kBM, p.lse + row, kBM * 4, bar);
                    bulk_load_1d(sLD + st * 2 * kBM + kBM, p.delta + row, kBM * 4, bar);
                }
                if (it == 0 && x.keys_cut()) {
                    wait_for(&k_cut[buf], (k_phases >> buf) & 1u, dead);
                    k_phases ^= 1u << buf;
                    clear(sK + buf * L::kKvBytes, kBN, x.len - x.n0);
                    cleared(&k_full[buf]);
                }
                if (m0 + kBM > x.len) {          // two more tiles are there or on their way meanwhile
                    wait_for(&qdo_cut[st], (q_phases >> st) & 1u, dead);
                    q_phases ^= 1u << st;
                    clear(sQ + st * L::kStageBytes, kBM, x.len - m0);
                    clear(sDO + st * L::kStageBytes, kBM, x.len - m0);
                    cleared(&qdo_full[st]);
                }
                if (++th == x.per_head) { th = 0; ++hq; }
            }
        }
    } else if (warp == 1) {
        // ============================ MMA ============================
        if (ptx::elect_one()) {
            constexpr uint32_t idesc_st = ptx::make_idesc_bf16(kBN, kBM, 0, 0);   // S^T, dP^T: 128 x 64, K-major A / B
            constexpr uint32_t idesc_kv = ptx::make_idesc_bf16(kBN, D, 0, 1);     // dV, dK: B MN-major
            constexpr uint32_t idesc_dq = ptx::make_idesc_bf16(128, kBM, 1, 1);   // dQ^T: A and B MN-major
            const uint32_t q_addr = ptx::smem_u32(sQ), do_addr = ptx::smem_u32(sDO), dst_addr = ptx::smem_u32(sDSt);
            int items = 0, blocks = 0, gs = 0, gi = 0;          // gs: tiles whose scores were issued, gi: that are done
            for (;;) {
                const Item x = next_item<false, Item>(item_ring, item_full, item_empty, items, dead);
                if (x.kind == 0) break;
                if (x.kind > 1) continue;
                const int buf = blocks % L::kBufs;
                const uint32_t ph = (uint32_t)(blocks / L::kBufs) & 1u;
                ++blocks;
                const uint32_t k_addr = ptx::smem_u32(sK + buf * L::kKvBytes), v_addr = ptx::smem_u32(sV + buf * L::kKvBytes);
                auto issue_scores = [&](int it) {
                    const int st = gs % kStages;
                    wait_for(&qdo_full[st], (uint32_t)(gs / kStages) & 1u, dead);
                    wait_for(st_empty, ((uint32_t)gs & 1u) ^ 1u, dead);          // S^T / dP^T of the tile before are in registers
                    ++gs;
                    ptx::tcgen05_fence_after();
                    const uint32_t qb = q_addr + st * L::kStageBytes, dob = do_addr + st * L::kStageBytes;
#pragma unroll
                    for (int kk = 0; kk < D / 16; ++kk) {
                        const uint32_t ko = (kk >> 2) * (kBN * 128) + (kk & 3) * 32, qo = (kk >> 2) * (kBM * 128) + (kk & 3) * 32;
                        ptx::umma_bf16<1>(tmem + kColST, ptx::make_smem_desc(k_addr + ko, 16, 1024), ptx::make_smem_desc(qb + qo, 16, 1024),
                                          idesc_st, kk != 0 ? 1u : 0u);
                    }
#pragma unroll
                    for (int kk = 0; kk < D / 16; ++kk) {
                        const uint32_t ko = (kk >> 2) * (kBN * 128) + (kk & 3) * 32, qo = (kk >> 2) * (kBM * 128) + (kk & 3) * 32;
                        ptx::umma_bf16<1>(tmem + kColDPT, ptx::make_smem_desc(v_addr + ko, 16, 1024), ptx::make_smem_desc(dob + qo, 16, 1024),
                                          idesc_st, kk != 0 ? 1u : 0u);
                    }
                    ptx::umma_commit(st_full);
                    if (it + 1 == x.total) ptx::umma_commit(&v_empty[buf]);
                };
                wait_for(&k_full[buf], ph, dead);
                wait_for(&v_full[buf], ph, dead);
                issue_scores(0);
                for (int it = 0; it < x.total; ++it, ++gi) {
                    if (it + 1 < x.total) issue_scores(it + 1);
                    const int st = gi % kStages;
                    const uint32_t qb = q_addr + st * L::kStageBytes, dob = do_addr + st * L::kStageBytes;
                    wait_for(pds_full, (uint32_t)gi & 1u, dead);
                    ptx::tcgen05_fence_after();
#pragma unroll
                    for (int kk = 0; kk < kBM / 16; ++kk)
                        ptx::umma_bf16_ts(tmem + kColDV, tmem + kColPT + kk * 8, ptx::make_smem_desc(dob + kk * 2048, kBM * 128, 1024), idesc_kv,
                                          (it | kk) != 0 ? 1u : 0u);
#pragma unroll
                    for (int kk = 0; kk < kBM / 16; ++kk)
                        ptx::umma_bf16_ts(tmem + kColDK, tmem + kColDST + kk * 8, ptx::make_smem_desc(qb + kk * 2048, kBM * 128, 1024), idesc_kv,
                                          (it | kk) != 0 ? 1u : 0u);
                    ptx::umma_commit(&qdo_empty[st]);
                    // contraction over the 128 key rows, once dQ^T of the tile before is in registers.  D = 64: M stays 128, and the
                    // descriptor walks 64 rows past the K tile into what follows; nobody reads those lanes of dQ^T.
                    wait_for(dq_empty, ((uint32_t)gi & 1u) ^ 1u, dead);
                    ptx::tcgen05_fence_after();
#pragma unroll
                    for (int kk = 0; kk < kBN / 16; ++kk)
                        ptx::umma_bf16<1>(tmem + kColDQT, ptx::make_smem_desc(k_addr + kk * 2048, kBN * 128, 1024),
                                          ptx::make_smem_desc(dst_addr + kk * 2048, kBN * 128, 1024), idesc_dq, kk != 0 ? 1u : 0u);
                    ptx::umma_commit(pds_empty);
                    ptx::umma_commit(dq_full);
                }
                ptx::umma_commit(&k_empty[buf]);
            }
        }
    } else if (warp >= 10) {
        // ============================ dQ drain ============================
        // dQ^T [d = TMEM lane][64 q] -> this warp's staging rows (the accumulator in global memory is d-major) -> TMA reduce-add, 32 q
        // columns per box.  Staging, bulk groups and the waits on them are private to the warp.
        const int q4 = warp & 3;                 // TMEM lane quadrant this warp may access
        const uint32_t lane_off = (uint32_t)(q4 * 32) << 16;
        const bool has_rows = q4 * 32 < D;       // D = 64: lanes 64..127 of dQ^T are padding
        uint8_t* stage = sDQ + q4 * 8192;        // two 32 x 32 fp32 boxes (4 KB each)
        int items = 0, gi = 0;
        for (;;) {
            const Item x = next_item<true, Item>(item_ring, item_full, item_empty, items, dead);
            if (x.kind == 0) break;
            if (x.kind > 1) continue;
            int th = x.th, hq = x.head;
            for (int it = 0; it < x.total; ++it, ++gi) {
                const int m0 = (x.first + th) * kBM;
                wait_for(dq_full, (uint32_t)gi & 1u, dead);
                ptx::tcgen05_fence_after();
                uint32_t v[64];
                if (has_rows) {
                    ptx::tmem_ld_32x32b_x32(tmem + kColDQT + lane_off, v);
                    ptx::tmem_ld_32x32b_x32(tmem + kColDQT + lane_off + 32, v + 32);
                    ptx::tmem_ld_wait();
                }
                ptx::tcgen05_fence_before();
                ptx::mbar_arrive(dq_empty);
                if (has_rows) {
                    if (m0 + kBM > x.len) {          // those columns are the next sequence's: K may hold what 0 does not silence
#pragma unroll
                        for (int e = 0; e < 64; ++e) v[e] = m0 + e < x.len ? v[e] : 0u;
                    }
                    if (lane == 0) ptx::bulk_wait_read<0>();     // the reduce-adds before have read the staging rows
                    __syncwarp();
#pragma unroll
                    for (int h2 = 0; h2 < 2; ++h2) {
                        uint8_t* dst = stage + h2 * 4096 + lane * 128;
#pragma unroll
                        for (int c = 0; c < 8; ++c)
                            st_shared_v4(dst + ((c ^ (lane & 7)) << 4), __float_as_uint(__uint_as_float(v[h2 * 32 + 4 * c]) * p.scale),
                                         __float_as_uint(__uint_as_float(v[h2 * 32 + 4 * c + 1]) * p.scale),
                                         __float_as_uint(__uint_as_float(v[h2 * 32 + 4 * c + 2]) * p.scale),
                                         __float_as_uint(__uint_as_float(v[h2 * 32 + 4 * c + 3]) * p.scale));
                    }
                    ptx::fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) {
                        int c[4];
                        coords(p.pos_dq, q4 * 32, hq, 0, c);
                        tma_reduce_add_4d(&tmap_dq, stage, x.pad + m0, c[1], c[2], c[3]);
                        if (m0 + 32 < x.len) tma_reduce_add_4d(&tmap_dq, stage + 4096, x.pad + m0 + 32, c[1], c[2], c[3]);
                        ptx::bulk_commit();
                    }
                }
                if (++th == x.per_head) { th = 0; ++hq; }
            }
        }
        if (lane == 0) ptx::bulk_wait<0>();
    } else {
        // ============================ P^T, dS^T and the results of a block ============================
        const int q4 = warp & 3;
        const int row = q4 * 32 + lane;          // key row inside the block == TMEM lane
        const uint32_t lane_off = (uint32_t)(q4 * 32) << 16;
        const int half = (warp - 2) >> 2;        // which 32 of the 64 queries this warp handles; afterwards dV (0) or dK (1)
        const int c0h = half * 32;
        uint8_t* out = smem + L::kOutOff + (warp - 2) * 1024;
        int items = 0, gi = 0;
        uint32_t q_phases = 0;
        Item x = next_item<true, Item>(item_ring, item_full, item_empty, items, dead);
        for (; x.kind != 0;) {
            if (x.kind > 1) {
                const int rows = x.kind - kRowsOfNone - 1;
                if (rows > 0) {
                    block_zero_rows<D>(p.dk + (long long)x.start * p.dk_row + x.hkv * p.dk_head, p.dk_row, rows, threadIdx.x - 64, kMathThreads);
                    block_zero_rows<D>(p.dv + (long long)x.start * p.dv_row + x.hkv * p.dv_head, p.dv_row, rows, threadIdx.x - 64, kMathThreads);
                }
                x = next_item<true, Item>(item_ring, item_full, item_empty, items, dead);
                continue;
            }
            const int krow = x.n0 + row;
            // P^T = exp2(S^T c - L), dS^T = P^T (dP^T - Delta) for this thread's key row and 32 queries.  MASK: tiles on the diagonal or
            // at the end of the sequence
            auto softmax_bwd = [&](auto mask_tag, const uint32_t* s, const uint32_t* dp, const float* Ls, const float* Ds, int m0, uint32_t* pk,
                                   uint32_t* dk_) {
                constexpr bool MASK = decltype(mask_tag)::value;
                int first_ok = 0, last_ok = 64;          // queries [first_ok, last_ok) of the 32 see this key
                if (MASK) {
                    first_ok = CAUSAL ? krow - m0 - c0h : 0;
                    if (krow >= x.len) first_ok = 64;
                    last_ok = x.len - m0 - c0h;
                }
#pragma unroll
                for (int c = 0; c < 32; c += 4) {
                    const float4 l4 = ld_shared_f4(Ls + c0h + c);
                    const float4 d4 = ld_shared_f4(Ds + c0h + c);
                    const float lv[4] = {l4.x, l4.y, l4.z, l4.w}, dv[4] = {d4.x, d4.y, d4.z, d4.w};
                    float pv[4], dsv[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        pv[e] = ex2_approx(fmaf(__uint_as_float(s[c + e]), p.scale_log2, -lv[e]));
                        dsv[e] = pv[e] * (__uint_as_float(dp[c + e]) - dv[e]);
                        if (MASK && (c + e < first_ok || c + e >= last_ok)) pv[e] = dsv[e] = 0.f;
                    }
                    pk[c >> 1] = pack_bf16x2(pv[0], pv[1]);
                    pk[(c >> 1) + 1] = pack_bf16x2(pv[2], pv[3]);
                    dk_[c >> 1] = pack_bf16x2(dsv[0], dsv[1]);
                    dk_[(c >> 1) + 1] = pack_bf16x2(dsv[2], dsv[3]);
                }
            };
            int th = x.th;
            for (int it = 0; it < x.total; ++it, ++gi) {
                const int st = gi % kStages;
                const int m0 = (x.first + th) * kBM;
                wait_for(st_full, (uint32_t)gi & 1u, dead);
                ptx::tcgen05_fence_after();
                uint32_t s[32], dp[32];
                ptx::tmem_ld_32x32b_x32(tmem + kColST + lane_off + c0h, s);
                ptx::tmem_ld_32x32b_x32(tmem + kColDPT + lane_off + c0h, dp);
                ptx::tmem_ld_wait();
                ptx::tcgen05_fence_before();
                ptx::mbar_arrive(st_empty);
                // L and Delta came with Q_i and dO_i: wait for those copies here too, so that their bytes are visible to this thread
                if (m0 + kBM > x.len) {
                    wait_for(&qdo_cut[st], (q_phases >> st) & 1u, dead);
                    q_phases ^= 1u << st;
                }
                wait_for(&qdo_full[st], (uint32_t)(gi / kStages) & 1u, dead);
                const float* Ls = sLD + st * 2 * kBM;
                const float* Ds = Ls + kBM;
                const bool need_mask = x.n0 + kBN > x.len || m0 + kBM > x.len || (CAUSAL && x.n0 + q4 * 32 + 31 > m0 + c0h);
                uint32_t pk[16], dk_[16];
                if (need_mask) softmax_bwd(std::true_type{}, s, dp, Ls, Ds, m0, pk, dk_);
                else softmax_bwd(std::false_type{}, s, dp, Ls, Ds, m0, pk, dk_);
                if (gi > 0) wait_for(pds_empty, ((uint32_t)(gi - 1)) & 1u, dead);  // products of the tile before have read dS^T
                tmem_st_32x32b_x16(tmem + kColPT + lane_off + half * 16, pk);
                tmem_st_32x32b_x16(tmem + kColDST + lane_off + half * 16, dk_);
                uint8_t* drow = sDSt + row * 128;
#pragma unroll
                for (int c = 0; c < 4; ++c) {                // this warp's 4 of the row's 8 sixteen-byte chunks
                    const int sw = ((half * 4 + c) ^ (row & 7)) << 4;
                    st_shared_v4(drow + sw, dk_[4 * c], dk_[4 * c + 1], dk_[4 * c + 2], dk_[4 * c + 3]);
                }
                tmem_st_wait();
                ptx::fence_proxy_async();
                ptx::tcgen05_fence_before();
                ptx::mbar_arrive(pds_full);
                if (++th == x.per_head) th = 0;
            }
            const Item done = x;                             // the next one is read while the last products run
            x = next_item<true, Item>(item_ring, item_full, item_empty, items, dead);
            wait_for(pds_empty, ((uint32_t)(gi - 1)) & 1u, dead);          // the commit behind the last product: dK and dV are final
            ptx::tcgen05_fence_after();
            const uint32_t col = half == 0 ? kColDV : kColDK;
            const float mul = half == 0 ? 1.f : p.scale;
            if (p.nsplit > 1) {
                // partial dV / dK -> fp32 -> TMA reduce-add into the accumulators, 8 rows x 32 columns at a time
#pragma unroll 1
                for (int g = 0; g < D / 32; ++g) {
                    uint32_t o[32];
                    ptx::tmem_ld_32x32b_x32(tmem + col + lane_off + g * 32, o);
                    ptx::tmem_ld_wait();
                    if (done.n0 + row >= done.len) {         // the next sequence's row
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = 0u;
                    }
#pragma unroll 1
                    for (int part = 0; part < 4; ++part) {
                        if (lane == 0) ptx::bulk_wait_read<0>();
                        __syncwarp();
                        if ((lane >> 3) == part) {
                            const int r = lane & 7;
#pragma unroll
                            for (int c = 0; c < 8; ++c)
                                st_shared_v4(out + r * 128 + ((c ^ (r & 7)) << 4), __float_as_uint(__uint_as_float(o[4 * c]) * mul),
                                             __float_as_uint(__uint_as_float(o[4 * c + 1]) * mul), __float_as_uint(__uint_as_float(o[4 * c + 2]) * mul),
                                             __float_as_uint(__uint_as_float(o[4 * c + 3]) * mul));
                        }
                        ptx::fence_proxy_async();
                        __syncwarp();
                        const int first = done.n0 + q4 * 32 + part * 8;
                        if (lane == 0 && first < done.len) {
                            int c[4];
                            c[0] = g * 32;
                            coords(p.pos_acc, done.start + first, done.hkv, 0, c);
                            tma_reduce_add_4d(half == 0 ? &tmap_dv_acc : &tmap_dk_acc, out, c[0], c[1], c[2], c[3]);
                            ptx::bulk_commit();
                        }
                    }
                }
            } else {
                // 32 rows x 16 columns through shared memory, so that a row's 32 bytes are stored by neighbouring lanes
                const long long ld = half == 0 ? p.dv_row : p.dk_row;
                bf16* to = (half == 0 ? p.dv + done.hkv * p.dv_head : p.dk + done.hkv * p.dk_head) + (long long)(done.start + done.n0 + q4 * 32) * ld;
                const int left = done.len - done.n0 - q4 * 32;
#pragma unroll 1
                for (int g = 0; g < D / 16; ++g) {
                    uint32_t o[16];
                    ptx::tmem_ld_32x32b_x16(tmem + col + lane_off + g * 16, o);
                    ptx::tmem_ld_wait();
                    __syncwarp();
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        uint32_t w[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            w[i] = pack_bf16x2(__uint_as_float(o[8 * c + 2 * i]) * mul, __uint_as_float(o[8 * c + 2 * i + 1]) * mul);
                        st_shared_v4(out + lane * 32 + ((c ^ ((lane >> 2) & 1)) << 4), w[0], w[1], w[2], w[3]);
                    }
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int r = i * 16 + (lane >> 1), ch = lane & 1;
                        if (r < left)
                            *reinterpret_cast<uint4*>(to + r * ld + g * 16 + ch * 8) =
                                *reinterpret_cast<const uint4*>(out + r * 32 + ((ch ^ ((r >> 2) & 1)) << 4));
                    }
                }
            }
            ptx::tcgen05_fence_before();
        }
        if (lane == 0) ptx::bulk_wait<0>();
    }
    ptx::tcgen05_fence_before();
    __syncthreads();
    if (gave_up(dead)) {
        let_copies_land();
        if (threadIdx.x == 0) {
            p.claimed[1] = 1;            // the last kernel of the call then writes NaN
            *reinterpret_cast<volatile int*>(p.gave_up) = 1;
        }
    }
    if (warp == 1) ptx::tmem_dealloc<1>(tmem, 512);
}

// Delta of one entry (up to 128 rows) of one head, at the plan's padded columns, and zeros into the dQ accumulator's columns of those rows
// (nobody reads the padding), the counter of claims and the mark behind it.  kD / 8 lanes own a row.  Bound by memory: 24576 rows of 16 heads of 64,
// 201 MB, 38 us.
template <int kD>
__global__ void __launch_bounds__(256, 4) packed_delta_kernel(const bf16* __restrict__ o, const uint8_t* __restrict__ rest, const bf16* __restrict__ dout,
                                                           const PackedTile* tiles, const int* which, long long rest_row, float* __restrict__ delta,
                                                           float* __restrict__ acc, int* claimed, long long o_head, long long o_row,
                                                           long long do_head, long long do_row, long long lse_row, int Hq, int causal) {
    pdl_wait();         // and no trigger: CTAs of the next kernel that come while the SMs are full of this one's blocks stay slower for good
                        // (4 documents in 16384 tokens, 32 heads of 128 over 8: 2060 us for the pass instead of 1750)
    constexpr int L = kD / 8, R = 256 / L;
    const PackedTile pt = packed_tile(tiles, blockIdx.x / Hq);
    const int h = blockIdx.x % Hq, l = threadIdx.x % L;
    const int first = pt.t * kBN, rows = min(pt.len - first, kBN);        // negative where the entry is no tile
    if (blockIdx.x == 0 && threadIdx.x == 0) claimed[0] = claimed[1] = 0;
    if (pt.len == 0) return;
    {
        const int quads = (rows + 3) >> 2;
        float* to = acc + (long long)h * kD * lse_row + pt.pad + first;
#pragma unroll 4
        for (int i = threadIdx.x; i < kD * 32; i += 256)
            if ((i & 31) < quads) *reinterpret_cast<float4*>(to + (i >> 5) * lse_row + (i & 31) * 4) = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    const long long col = h * lse_row + pt.pad + first;
    const bool one_tile = causal ? pt.t == 0 : pt.len <= kBN;          // of keys: these rows have what the rounding took
    const long long rest_at = h * rest_row + (which == nullptr ? pt.pad : (int)((unsigned)which[blockIdx.x / Hq] * kBN));
    constexpr int U = 4;                     // rows of a lane on their way
#pragma unroll 1
    for (int r0 = threadIdx.x / L; r0 < kBN; r0 += U * R) {
        bf16x8 a[U], g[U];
        uint2 less[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int r = r0 + u * R;
            const long long row = pt.start + first + r;
            if (r < rows) {
                a[u] = reinterpret_cast<const bf16x8*>(o + h * o_head + row * o_row)[l];
                g[u] = reinterpret_cast<const bf16x8*>(dout + h * do_head + row * do_row)[l];
                if (one_tile) less[u] = *reinterpret_cast<const uint2*>(rest + rest_offset<kD>(rest_at + r, l >> 1) + (l & 1) * 8);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int r = r0 + u * R;
            float acc = 0.f;
            uint32_t most = 0u;              // of the row's 64 neighbours
            if (one_tile && r < rows) {
                const uint4 w = *reinterpret_cast<const uint4*>(&a[u]);
                most = __vmaxu2(__vmaxu2(w.x & 0x7fff7fffu, w.y & 0x7fff7fffu), __vmaxu2(w.z & 0x7fff7fffu, w.w & 0x7fff7fffu));
            }
            if (one_tile) {
#pragma unroll
                for (int off = 4; off > 0; off >>= 1) most = __vmaxu2(most, __shfl_xor_sync(0xffffffffu, most, off));
            }
            if (r < rows) {
                float fa[8], fg[8];
                unpack8(a[u], fa);
                unpack8(g[u], fg);
                if (one_tile) {
                    const float down = rest_down(most);
#pragma unroll
                    for (int e = 0; e < 8; ++e) fa[e] = fmaf(rest_of(e < 4 ? less[u].x : less[u].y, e & 3), down, fa[e]);
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) acc = fmaf(fa[e], fg[e], acc);
            }
#pragma unroll
            for (int off = L / 2; off > 0; off >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, off);
            if (l == 0 && r < rows) delta[col + r] = acc;
        }
    }
}

// d-major fp32 accumulator [Hq, D, lse_row] -> dq, 64 of the D of an entry (128 rows) of one head per block; rows of no sequence get
// zeros.  Where a CTA of the kernel before gave up a wait, dQ, dK and dV become NaN: what it and others had added is a part.  Bound by memory: 24576 rows of 16 heads of 64, 151 MB, 31 us; 16384 rows of 32 heads of 128, 403 MB, 79 us (142 as half
// entries through padded rows of shared memory, which two to four lanes met at one bank).
template <int kD>
__global__ void __launch_bounds__(256) packed_dq_kernel(const float* __restrict__ acc, bf16* __restrict__ dq, const BwdParams p, long long head,
                                                        long long row, int Hq) {
    const long long lse_row = p.lse_row;
    pdl_trigger();
    pdl_wait();
    __shared__ float4 tile[64][32];          // four columns of row d at place (columns / 4) ^ (d / 8 % 8): no bank twice, either way
    constexpr int kParts = kD / 64;
    const unsigned at = blockIdx.x / kParts;
    const PackedTile pt = packed_tile(p.tiles, at / Hq);
    const int h = at % Hq, d0 = blockIdx.x % kParts * 64;
    if (pt.len == 0) {
        if (d0 != 0) return;
        block_zero_rows<kD>(dq + (long long)pt.start * row + h * head, row, pt.t, threadIdx.x, 256);
        if (p.claimed[1] && h % p.group == 0) {
            block_zero_rows<kD>(p.dk + (long long)pt.start * p.dk_row + h / p.group * p.dk_head, p.dk_row, pt.t, threadIdx.x, 256);
            block_zero_rows<kD>(p.dv + (long long)pt.start * p.dv_row + h / p.group * p.dv_head, p.dv_row, pt.t, threadIdx.x, 256);
        }
        return;
    }
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int q0 = pt.t * kBN, left = pt.len - q0;
    const float* src = acc + ((long long)h * kD + d0) * lse_row + pt.pad + q0;
    float4 v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j)              // columns in fours: those of a sequence are padded to a multiple of four
        v[j] = 4 * lane < left ? *reinterpret_cast<const float4*>(src + (w + 8 * j) * lse_row + 4 * lane) : make_float4(0.f, 0.f, 0.f, 0.f);
    if (p.claimed[1]) {                      // asked for behind the loads
        const int key_head = h / p.group;
        for (int i = threadIdx.x; i < min(left, kBN) * 8; i += 256) {
            const long long r = pt.start + q0 + (i >> 3);
            const int c = d0 + (i & 7) * 8;
            const uint4 nan = make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);
            *reinterpret_cast<uint4*>(dq + h * head + r * row + c) = nan;
            if (h % p.group) continue;
            *reinterpret_cast<uint4*>(p.dk + key_head * p.dk_head + r * p.dk_row + c) = nan;
            *reinterpret_cast<uint4*>(p.dv + key_head * p.dv_head + r * p.dv_row + c) = nan;
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) tile[w + 8 * j][lane ^ j] = v[j];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {            // eight lanes write 128 bytes of a row
        const int r = w * 16 + i * 4 + (lane >> 3), c = lane & 7;
        if (r < left) {
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = reinterpret_cast<const float*>(&tile[c * 8 + e][(r >> 2) ^ c])[r & 3];
            *reinterpret_cast<uint4*>(dq + h * head + (long long)(pt.start + q0 + r) * row + d0 + 8 * c) =
                make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
        }
    }
}

// fp32 accumulator [Hkv, T, D] -> bf16 rows
__global__ void packed_kv_convert_kernel(const float* __restrict__ acc, bf16* __restrict__ to, long long head, long long row, int Hkv, long long T,
                                         int D) {
    pdl_trigger();
    pdl_wait();
    const long long idx = (long long)blockIdx.x * blockDim.x + threadIdx.x;  // one thread = 8 elements
    const int per = D / 8;
    if (idx >= Hkv * T * per) return;
    const long long r = idx / per, t = r % T;
    const int c = (int)(idx % per), h = (int)(r / T);
    const float4 a0 = reinterpret_cast<const float4*>(acc)[2 * idx], a1 = reinterpret_cast<const float4*>(acc)[2 * idx + 1];
    float f[8] = {a0.x, a0.y, a0.z, a0.w, a1.x, a1.y, a1.z, a1.w};
    reinterpret_cast<bf16x8*>(to + h * head + t * row)[c] = pack8(f);
}

template <int D, bool CAUSAL>
int launch(cudaStream_t st, const CUtensorMap& tq, const CUtensorMap& tdo, const CUtensorMap& tk, const CUtensorMap& tv, const CUtensorMap& tdq,
           const CUtensorMap& tdka, const CUtensorMap& tdva, const BwdParams& p) {
    using L = BwdSmem<D>;
    constexpr auto kern = packed_bwd_kernel<D, CAUSAL>;
    NXD_CHECK_CUDA(nxd_allow_smem<kern>(L::kBytes));
    const long long items = (long long)p.entries * p.Hkv * p.nsplit;
    const unsigned grid = (unsigned)(items < nxd_num_sms() ? items : nxd_num_sms());
    NXD_CHECK_CUDA((nxd_launch_pdl(kern, dim3(grid), dim3(kThreads), L::kBytes, st, tq, tdo, tk, tv, tdq, tdka, tdva, p)));
    NXD_LAUNCH_CHECK();
    return 0;
}

}  // namespace

// CTAs that share one K/V block of a packed batch: as nxd_flash_attn_bwd_tc_num_splits, for N sequences of average length.
NXD_API int nxd_packed_attn_bwd_splits(long long T, int N, int Hq, int Hkv) {
    const long long avg = (T + (N > 0 ? N : 1) - 1) / (N > 0 ? N : 1);
    const long long blocks = (avg + kBN - 1) / kBN * (N > 0 ? N : 1);
    const int B = (int)(blocks < 65536 ? blocks : 65536);
    const int sms = nxd_num_sms();
    const long long ctas = (long long)B * Hkv;
    if (ctas >= 2LL * sms) return 1;
    const long long iters = (avg + kBM - 1) / kBM * (Hq / (Hkv > 0 ? Hkv : 1));
    long long n = (4LL * sms + ctas - 1) / ctas;
    if (n > iters / 8) n = iters / 8;
    if (n > 16) n = 16;
    return n < 1 ? 1 : (int)n;
}

// Backward of nxd_packed_attn_fwd.  strides: {head, row} in elements of q, k, v, o, dout, dq, dk, dv (16 values, multiples of 8);
// lse, rest: what the forward pass wrote (which, rest_row: as there); delta: Hq * lse_row + 4 floats of scratch; dq_accum: [Hq, D, lse_row] floats of scratch;
// dkv_accum: NULL, or ZEROED [2, Hkv, T, D] floats where nxd_packed_attn_bwd_splits says more than one.
// dQ (with splits dK and dV too) is summed in fp32 in an order that is not fixed.  wait_tries: as forward.
NXD_API int nxd_packed_attn_bwd(const void* q, const void* k, const void* v, const void* o, const void* rest, const void* dout, const float* lse,
                                float* delta, float* dq_accum, float* dkv_accum, void* dq, void* dk, void* dv,
                                const long long* strides, const void* tiles, const int* which, long long rest_row, int entries, long long lse_row, long long T, int N, int Hq,
                                int Hkv, int D, float scale, int causal, int wait_tries, void* stream) {
    NXD_REQUIRE(D == 64 || D == 128, "packed_attn_bwd: head dim %d not supported (64 or 128)", D);
    NXD_REQUIRE(T > 0 && T < (1ll << 31) - 256 && Hq > 0 && Hkv > 0 && Hq % Hkv == 0 && entries > 0 && lse_row % 4 == 0 && rest_row % 4 == 0 &&
                (long long)entries * Hq * 16 < (1ll << 31), "packed_attn_bwd: bad problem");
    NXD_REQUIRE(scale >= 1.17549435e-38f && scale <= 1.7014118e38f, "packed_attn_bwd: a scale of %g", scale);
    for (int i = 0; i < 16; ++i)
        NXD_REQUIRE(strides[i] % 8 == 0, "packed_attn_bwd: stride %d (=%lld) must be a multiple of 8 elements", i, strides[i]);
    const void* bases[] = {q, k, v, o, rest, dout, lse, delta, dq_accum, dkv_accum, dq, dk, dv, tiles};
    for (const void* x : bases)
        NXD_REQUIRE(((uintptr_t)x & 15) == 0 && (x != nullptr || x == dkv_accum), "packed_attn_bwd: tensors must be %s", "there and 16-byte aligned");
    NXD_REQUIRE(rest_row >= (which ? kBN : lse_row), "packed_attn_bwd: %lld rows of what the rounding took", rest_row);
    cudaStream_t st = (cudaStream_t)stream;
    const PackedTile* pt = (const PackedTile*)tiles;
    BwdParams p{};
    int rc;
    if ((rc = begin_call(&p.gave_up))) return rc;
    p.tries = wait_tries < 0 || wait_tries > kTries ? kTries : wait_tries;
    p.entries = entries; p.Hkv = Hkv; p.group = Hq / Hkv;
    p.lse = lse; p.delta = delta; p.lse_row = lse_row;
    p.scale = scale; p.scale_log2 = scale * 1.4426950408889634f;
    p.nsplit = dkv_accum ? nxd_packed_attn_bwd_splits(T, N, Hq, Hkv) : 1;
    p.tiles = pt;
    p.claimed = (int*)(delta + (long long)Hq * lse_row);
    p.dk = (bf16*)dk; p.dk_head = strides[12]; p.dk_row = strides[13];
    p.dv = (bf16*)dv; p.dv_head = strides[14]; p.dv_row = strides[15];
    const unsigned per_head = (unsigned)entries * Hq;
    if (D == 128)
        NXD_CHECK_CUDA((nxd_launch_pdl(packed_delta_kernel<128>, dim3(per_head), dim3(256), 0, st, (const bf16*)o, (const uint8_t*)rest, (const bf16*)dout, pt, which, rest_row,
            delta, dq_accum, p.claimed, strides[6], strides[7], strides[8], strides[9], lse_row, Hq, causal)));
    else
        NXD_CHECK_CUDA((nxd_launch_pdl(packed_delta_kernel<64>, dim3(per_head), dim3(256), 0, st, (const bf16*)o, (const uint8_t*)rest, (const bf16*)dout, pt, which, rest_row,
            delta, dq_accum, p.claimed, strides[6], strides[7], strides[8], strides[9], lse_row, Hq, causal)));
    NXD_LAUNCH_CHECK();
    CUtensorMap tq, tdo, tk, tv, tdq, tdka, tdva;
    if ((rc = make_tmap_bhsd(&tq, q, D, T, Hq, 1, strides[1], strides[0], 0, kBM, p.pos_q))) return rc;
    if ((rc = make_tmap_bhsd(&tk, k, D, T, Hkv, 1, strides[3], strides[2], 0, kBN, p.pos_k))) return rc;
    if ((rc = make_tmap_bhsd(&tv, v, D, T, Hkv, 1, strides[5], strides[4], 0, kBN, p.pos_v))) return rc;
    if ((rc = make_tmap_bhsd(&tdo, dout, D, T, Hq, 1, strides[9], strides[8], 0, kBM, p.pos_do))) return rc;
    if ((rc = make_tmap_bhsd(&tdq, dq_accum, (int)lse_row, D, Hq, 1, lse_row, (long long)D * lse_row, 0, 32, p.pos_dq, 4))) return rc;
    const long long kv_elems = (long long)Hkv * T * D;
    float* dk_acc = dkv_accum;
    float* dv_acc = dkv_accum + kv_elems;
    tdka = tdva = tdq;             // unused maps still have to be valid
    if (p.nsplit > 1) {
        if ((rc = make_tmap_bhsd(&tdka, dk_acc, D, T, Hkv, 1, D, T * D, 0, 8, p.pos_acc, 4))) return rc;
        if ((rc = make_tmap_bhsd(&tdva, dv_acc, D, T, Hkv, 1, D, T * D, 0, 8, p.pos_acc, 4))) return rc;
    }
    if (D == 128)
        rc = causal ? launch<128, true>(st, tq, tdo, tk, tv, tdq, tdka, tdva, p) : launch<128, false>(st, tq, tdo, tk, tv, tdq, tdka, tdva, p);
    else
        rc = causal ? launch<64, true>(st, tq, tdo, tk, tv, tdq, tdka, tdva, p) : launch<64, false>(st, tq, tdo, tk, tv, tdq, tdka, tdva, p);
    if (rc) return rc;
    if (p.nsplit > 1) {
        const long long n = kv_elems / 8;
        NXD_CHECK_CUDA((nxd_launch_pdl(packed_kv_convert_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, (const float*)dk_acc,
            (bf16*)dk, strides[12], strides[13], Hkv, T, D)));
        NXD_CHECK_CUDA((nxd_launch_pdl(packed_kv_convert_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, (const float*)dv_acc,
            (bf16*)dv, strides[14], strides[15], Hkv, T, D)));
        NXD_LAUNCH_CHECK_N(2);
    }
    if (D == 128)
        NXD_CHECK_CUDA((nxd_launch_pdl(packed_dq_kernel<128>, dim3(per_head * 2), dim3(256), 0, st, (const float*)dq_accum, (bf16*)dq, p,
            strides[10], strides[11], Hq)));
    else
        NXD_CHECK_CUDA((nxd_launch_pdl(packed_dq_kernel<64>, dim3(per_head), dim3(256), 0, st, (const float*)dq_accum, (bf16*)dq, p,
            strides[10], strides[11], Hq)));
    NXD_LAUNCH_CHECK();
    return 0;
}

