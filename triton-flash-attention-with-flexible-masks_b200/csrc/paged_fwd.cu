// Attention of new tokens over a paged cache: O = softmax(scores) V for a ragged batch of new tokens [T, H, D], whose sequences' keys and values
// lie in pages [pages, page size, Hk, D] that a table names. A token at position p of its sequence sees the keys up to p (and a prefix); what lies
// in the pages behind a sequence's length is never part of a result. The score of a pair is that of the forward kernel, with the changes of
// scores.cuh.
//
// The forward kernel's structure (fwd.cu): two chains of key tiles with a maximum, a sum and an accumulator each, an epilogue group that merges them
// while the chains are in the next item, K and V rings that run across items, S and P V issued by a warp each. What differs:
//  - all heads of a kv head's group share a tile of queries, row = token * G + head of the group, so that K and V are read once for the group: one decoded
//    token of 32 / 8 heads reads its keys once instead of four times;
//  - a tile of 128 keys is 128 / page size boxes, one a page, which land one behind the other in the tile (a page of 8 rows is one
//    swizzle atom); the producers' lanes read the page numbers of the next tile while this one is under way;
//  - P of a masked entry is 0, but 0 times a NaN that an earlier user left in the page, or that a later token of the chunk has, is not: rows of V behind the last that the item
//    sees are zeroed in shared memory by the softmax group before it gives its P away (not by the warp that issues P V: its code has to stay free of loops by
//    lanes, or the descriptors go through vector registers);
//  - items of at most 32 rows (a decoded token's heads) take the tile four times over, so that each of a group's four warps has 32 keys of every row instead of 32 rows of
//    which most are nobody's: the chain from the scores to P is a quarter as long. 64 single tokens, 32 / 8 heads of 128, capped, 251 -> 218 us;
//  - each block works on one stretch of a line of all items (paged_plan.cuh); a piece of an item that was cut leaves normalised fp32 rows and
//    their log-sum-exp to paged_combine_kernel.
//
// What bounds it. Single tokens: HBM. 64 tokens over 1288 MB of keys and values 212-215 us in replayed graphs (6.0-6.1 TB/s; the copy rate is 6.56) and up to 243 in long series of
// calls under the power cap (5.3), one token over 537 MB 98-107 us, of which
// the plan and the first item's place take 2.3, the last tile's drain 3, the second kernel up to 4 (the main loop streams at 7 TB/s); one token over 1.4 MB
// 16 us, all of it latency: start, plan, a chain of tiles, epilogue, the second kernel's start. Chunks: the forward's chain of tiles, and twice as many loads. One chunk of 2000
// tokens, 32 / 8 heads, pages of 128 | 16: 64 | 64 us; a chunk of 500 behind 7500 67 | 76 us, where dense keys take 55.
#include <type_traits>
#include "common.cuh"
#include "paged_plan.cuh"
#include "params.cuh"

namespace fa {

template <int D>
struct PagedSmem {
    static constexpr int NS = (D == 128) ? 2 : 4;  // depth of the K ring and of the V ring
    static constexpr int NQ = 2;                   // item slots
    // TMEM columns as in the forward kernel
    static constexpr bool POWN = D == 128;
    static constexpr int NP = POWN ? 2 : 3;
    static constexpr int tmem_o = POWN ? 256 : 384;
    static __device__ int tmem_s(int g) { return POWN ? 0 : g % 3 * 128; }
    static __device__ int tmem_p(int g) { return POWN ? 128 + (g & 1) * 64 : g % 3 * 128; }
    static constexpr int TILE = kBlk * D * 2;
    static constexpr int BOX = kBlk * 64 * 2;
    static constexpr int NBOX = D / 64;
    static constexpr int off_q = 0;  // NQ Q tiles
    static constexpr int off_k = NQ * TILE;
    static constexpr int off_v = off_k + NS * TILE;
    static constexpr int off_ml = off_v + NS * TILE;             // float [NQ][2 groups][m, l][128]
    static constexpr int off_info = off_ml + NQ * 4 * kBlk * 4;  // int32 [NQ][16]: see I_*
    static constexpr int off_plan = off_info + NQ * 64;
    static constexpr int off_bar = off_plan + int(sizeof(PagedPlan));
    // item_full[NQ] item_empty[NQ] q_full[NQ] ml_full[NQ] staged k_full[NS] k_empty[NS] v_full[NS] v_empty[NS]
    // s_full[4] s_free[2] p_full[NP] pv_done[NP] o_full[2] o_free[2]
    static constexpr int n_bar = 4 * NQ + 1 + 4 * NS + 6 + 2 * NP + 4;
    static constexpr int off_misc = off_bar + n_bar * 8;  // tmem slot, abort flag
    static constexpr int total = off_misc + 16;
    static_assert(off_plan % 8 == 0 && off_bar % 8 == 0, "alignment");
};
static_assert(PagedSmem<128>::total <= 232448 && PagedSmem<64>::total <= 232448, "shared memory budget");
static_assert(PagedSmem<128>::total > 116736 && PagedSmem<64>::total > 116736, "shares an SM");

// What an item's slot says: number of its key tiles, the first one, whether there is an item (1, or -1: no more), kv head, first row of its tokens in
// q and out, how many of them, position of the first one, the sequence's length, its prefix, the sequence, slot of the workspace (-1: straight to out)
enum : int { I_TILES = 0, I_LO, I_MORE, I_HEAD, I_ROW, I_TOKENS, I_POS, I_LEN, I_FRONT, I_SEQ, I_PART };

template <int D, bool BF16, int KIND>
__global__ void __launch_bounds__(kFwdThreads, 1)
paged_fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmN, const __grid_constant__ CUtensorMap tmK,
                 const __grid_constant__ CUtensorMap tmV, const PagedParams p) {
    using S = PagedSmem<D>;
    constexpr bool SCORED = score_changed(KIND);
    constexpr int NS = S::NS, NQ = S::NQ, NP = S::NP;
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t sbase = smem_u32(smem);
    const int tid = threadIdx.x, warp = uniform(tid >> 5), lane = tid & 31;

    volatile int* misc = reinterpret_cast<volatile int*>(smem + S::off_misc);  // [0] tmem, [1] abort
    volatile int* info = reinterpret_cast<volatile int*>(smem + S::off_info);
    PagedPlan& plan = *reinterpret_cast<PagedPlan*>(smem + S::off_plan);
    const uint32_t bar0 = sbase + S::off_bar;
    auto BAR = [&](int i) { return bar0 + 8u * uint32_t(i); };
    constexpr int B_ITEMFULL = 0, B_ITEMEMPTY = NQ, B_QFULL = 2 * NQ, B_MLFULL = 3 * NQ, B_STAGED = 4 * NQ, B_KFULL = 4 * NQ + 1,
                  B_KEMPTY = B_KFULL + NS, B_VFULL = B_KEMPTY + NS, B_VEMPTY = B_VFULL + NS, B_SFULL = B_VEMPTY + NS,
                  B_SFREE = B_SFULL + 4, B_PFULL = B_SFREE + 2, B_PVDONE = B_PFULL + NP, B_OFULL = B_PVDONE + NP, B_OFREE = B_OFULL + 2;
    static_assert(B_OFREE + 2 == S::n_bar, "barriers");
    Abort ab{misc + 1, p.status, p.wait_limit};

    if (tid == 0) {
        for (int s = 0; s < NQ; ++s) {
            mbar_init(BAR(B_ITEMFULL + s), 1);
            mbar_init(BAR(B_ITEMEMPTY + s), 15);  // V producer, two MMA issuers, eight softmax warps, four epilogue warps
            mbar_init(BAR(B_QFULL + s), 1);
            mbar_init(BAR(B_MLFULL + s), 8);
        }
        for (int s = 0; s < NS; ++s) {
            mbar_init(BAR(B_KFULL + s), 1);
            mbar_init(BAR(B_KEMPTY + s), 1);
            mbar_init(BAR(B_VFULL + s), 1);
            mbar_init(BAR(B_VEMPTY + s), 1);
        }
        mbar_init(BAR(B_STAGED), 4);
        for (int s = 0; s < 4; ++s) mbar_init(BAR(B_SFULL + s), 1);
        for (int s = 0; s < NP; ++s) {
            mbar_init(BAR(B_PFULL + s), 4);  // here and below: one arrival a warp
            mbar_init(BAR(B_PVDONE + s), 1);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(BAR(B_SFREE + s), 4);
            mbar_init(BAR(B_OFULL + s), 1);
            mbar_init(BAR(B_OFREE + s), 4);
        }
        fence_mbar_init();
    }
    // Rows without a query are multiplied all the same: as zeros, until another item's rows have been there
    for (int i = tid; i < NQ * S::TILE / 16; i += kFwdThreads) reinterpret_cast<uint4*>(smem + S::off_q)[i] = make_uint4(0, 0, 0, 0);
    fence_proxy_async();
    wait_prerequisites();
    if (warp == 13) {
        take_tensor_memory(sbase + S::off_misc);
    }
    if (tid == 0) misc[1] = (status_is_fatal(*reinterpret_cast<volatile int*>(p.status)) || (sbase & 1023u) != 0) ? 1 : 0;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    launch_dependents();
    const uint32_t tmem = uint32_t(misc[0]);
    const bool aborted = misc[1] != 0;
    uint16_t* const out = static_cast<uint16_t*>(p.out);
    // (aborted: an earlier launch ran into a time-out that the host has not yet cleared. The second kernel fills the output.)
    if (aborted) {
        if (tid == 0) p.merge[blockIdx.x] = make_int4(-1, 0, 0, 0);
    } else if (p.B > kPagedWarpPlan) {
        paged_plan<kFwdThreads>(p, plan, int(gridDim.x));
    }
    const int worker = int(blockIdx.x);

    auto sQ = [&](int s) { return sbase + S::off_q + uint32_t(s) * S::TILE; };
    auto sK = [&](int s) { return sbase + S::off_k + uint32_t(s) * S::TILE; };
    auto sV = [&](int s) { return sbase + S::off_v + uint32_t(s) * S::TILE; };
    if (warp >= 12) {
        setmaxnreg_dec<kFwdServiceRegs>();
        // K and V are loaded by a warp each. (By one, 16 to 32 loads a tile with small pages, and the step from one tile's to the next, took longer than a
        // tile: one chunk of 500 tokens behind 7500, 32 / 8 heads of 128, pages of 128 | 16: 105 | 116 us.)
        const int rows = p.page < kBlk ? p.page : kBlk, log2_rows = p.page < kBlk ? p.log2_page : 7;  // of a box
        const int boxes = kBlk >> log2_rows;                                                          // of a tile, 16 at most
        // Lane i: the page that box i of a tile comes from. (Nothing is done with it here: the warp would wait for the load.)
        auto pages_of = [&](const int32_t* row_of_table, int tile, int len) {
            const int at = (tile << 7) + (lane << log2_rows);
            return lane < boxes && at < len ? row_of_table[at >> p.log2_page] : 0;
        };
        auto load = [&](const CUtensorMap* m, uint32_t dst, uint32_t bar, int pages, int tile, int hk, int len) {
            const int left = len - (tile << 7), n = left >= kBlk ? boxes : (left + rows - 1) >> log2_rows;
            pages = int(min(uint32_t(pages), uint32_t(p.n_pages)));  // (a page that there is not reads as zeros; the epilogue group reports it)
            mbar_expect_tx_elect(bar, uint32_t(n) << (log2_rows + 7) << (S::NBOX - 1));
            const int row = (tile << 7) & (p.page - 1) & ~(rows - 1);
#pragma unroll 1
            for (int i = 0; i < n; ++i) {
                const int page = __shfl_sync(0xffffffffu, pages, i);
#pragma unroll
                for (int x = 0; x < S::NBOX; ++x) tma_load_4d_elect(dst + uint32_t(x) * S::BOX, m, bar, x * 64, hk, row, page);
                dst += uint32_t(rows) * 128u;
            }
        };
        static_assert(S::NBOX == 1 || S::NBOX == 2, "bytes of a tile");
        if (aborted) {
        } else if (warp == 14) {
            // ------------------------------ item scheduler, and loads of Q and K ------------------------------
            tma_prefetch_desc(&tmQ);
            tma_prefetch_desc(&tmN);
            tma_prefetch_desc(&tmK);
            bool ok = true, first = true;
            int k = 0, gk = 0;
            int4 merge = make_int4(0, 0, 0, 0);
            if (p.B <= kPagedWarpPlan) paged_plan_warp(p, plan, int(gridDim.x));
            if (worker < plan.workers) {
                paged_stretch(p, plan, worker, [&](const PagedWalk& walk, int, int lo, int hi, int part) {
                    const int s = k % NQ, use = k / NQ;
                    const int T = uniform(hi - lo), tile0 = uniform(lo), hk = uniform(walk.hk), len = uniform(walk.s.len), tok0 = uniform(walk.s.start + walk.tile * p.tokens);
                    const int tokens = uniform(min(p.tokens, walk.s.n - walk.tile * p.tokens));
                    const int32_t* const row_of_table = p.table + walk.b * p.table_stride;
                    int pages = T > 0 ? pages_of(row_of_table, tile0, len) : 0;
                    if (use > 0) ok = mbar_wait_warp(BAR(B_ITEMEMPTY + s), (use - 1) & 1, ab, ST_WAIT_TIMEOUT + 11);
                    if (!ok) return false;
                    if (lane == 0) {
                        volatile int* it = info + 16 * s;
                        it[I_TILES] = T;
                        it[I_LO] = tile0;
                        it[I_MORE] = 1;
                        it[I_HEAD] = hk;
                        it[I_ROW] = tok0;
                        it[I_TOKENS] = tokens;
                        it[I_POS] = walk.s.base + walk.tile * p.tokens;
                        it[I_LEN] = len;
                        it[I_FRONT] = walk.s.front;
                        it[I_SEQ] = walk.b;
                        it[I_PART] = part;
                        mbar_arrive(BAR(B_ITEMFULL + s));
                    }
                    __syncwarp();
                    // (an item's slot is given away when its O has left, so that Q has been read, too)
                    if (tokens <= p.narrow) {  // four times the same rows
                        mbar_expect_tx_elect(BAR(B_QFULL + s), uint32_t(p.narrow * p.G) * 512u * S::NBOX);
                        for (int i = 0; i < 4 * S::NBOX; ++i)
                            tma_load_4d_elect(sQ(s) + (i >> 2) * S::BOX + (i & 3) * 4096, &tmN, BAR(B_QFULL + s), (i >> 2) * 64, 0, hk, tok0);
                    } else {
                        mbar_expect_tx_elect(BAR(B_QFULL + s), uint32_t(p.tokens * p.G) * 128u * S::NBOX);
                        for (int x = 0; x < S::NBOX; ++x) tma_load_4d_elect(sQ(s) + x * S::BOX, &tmQ, BAR(B_QFULL + s), x * 64, 0, hk, tok0);
                    }
                    for (int t = 0; t < T; ++t, ++gk) {
                        const int st = gk % NS, ug = gk / NS, own = pages;
                        if (t + 1 < T) pages = pages_of(row_of_table, tile0 + t + 1, len);
                        if (ug > 0) ok = mbar_wait_warp(BAR(B_KEMPTY + st), (ug - 1) & 1, ab, ST_WAIT_TIMEOUT + 1);
                        if (!ok) return false;
                        load(&tmK, sK(st), BAR(B_KFULL + st), own, tile0 + t, hk, len);
                    }
                    ++k;
                    if (first && paged_first_cut(plan, worker, walk)) {
                        // the item that this worker's stretch begins within is merged from its pieces by the second kernel
                        int from;
                        const int pieces = paged_pieces(p, plan, worker, walk, from);
                        merge = make_int4(pieces, tok0, tokens | hk << 8, from);
                    }
                    first = false;
                    return true;
                });
            }
            if (lane == 0) p.merge[worker] = merge;
            if (ok) {  // end marker
                const int s = k % NQ, use = k / NQ;
                if (use > 0) ok = mbar_wait_warp(BAR(B_ITEMEMPTY + s), (use - 1) & 1, ab, ST_WAIT_TIMEOUT + 11);
                if (ok && lane == 0) {
                    info[16 * s + I_MORE] = -1;
                    mbar_arrive(BAR(B_ITEMFULL + s));
                }
            }
        } else if (warp == 12) {
            // ------------------------------ loads of V ------------------------------
            tma_prefetch_desc(&tmV);
            bool ok = true;
            int gv = 0;
            for (int k = 0; ok; ++k) {
                const int s = k % NQ, use = k / NQ;
                ok = mbar_wait_warp(BAR(B_ITEMFULL + s), use & 1, ab, ST_WAIT_TIMEOUT + 12);
                if (!ok) break;
                volatile int* it = info + 16 * s;
                const int T = uniform(it[I_TILES]), lo = uniform(it[I_LO]), hk = uniform(it[I_HEAD]), len = uniform(it[I_LEN]), seq = uniform(it[I_SEQ]);
                if (uniform(it[I_MORE]) < 0) break;
                const int32_t* const row_of_table = p.table + seq * p.table_stride;
                int pages = T > 0 ? pages_of(row_of_table, lo, len) : 0;
                for (int t = 0; t < T; ++t, ++gv) {
                    const int st = gv % NS, ug = gv / NS, own = pages;
                    if (t + 1 < T) pages = pages_of(row_of_table, lo + t + 1, len);
                    if (ug > 0) ok = mbar_wait_warp(BAR(B_VEMPTY + st), (ug - 1) & 1, ab, ST_WAIT_TIMEOUT + 2);
                    if (!ok) break;
                    load(&tmV, sV(st), BAR(B_VFULL + st), own, lo + t, hk, len);
                }
                if (!ok) break;
                __syncwarp();
                if (lane == 0) mbar_arrive(BAR(B_ITEMEMPTY + s));
                __syncwarp();
            }
        } else {
            // ------------------------------ MMA issuers ------------------------------
            //   warp 13: P*V(g) when P(g) is there; warp 15: S(g) when its buffer is free
            const uint32_t utmem = uniform(int(tmem));
            constexpr uint32_t idesc_s = make_idesc(BF16, 128, 128, false, false);
            constexpr uint32_t idesc_pv = make_idesc(BF16, 128, D, false, true);
            constexpr uint64_t desc_v = desc_mn_major(S::BOX);
            bool ok = true;
            int G = 0;           // tiles of all earlier items
            int n0 = 0, n1 = 0;  // items in which the chains had tiles
            for (int k = 0;; ++k) {
                const int s = k % NQ, use = k / NQ;
                ok = mbar_wait_warp(BAR(B_ITEMFULL + s), use & 1, ab, ST_WAIT_TIMEOUT + 12);
                if (!ok) break;
                const int T = uniform(info[16 * s + I_TILES]);
                if (uniform(info[16 * s + I_MORE]) < 0) break;
                if (warp == 15) {
                    if (T > 0) ok = mbar_wait_warp(BAR(B_QFULL + s), use & 1, ab, ST_WAIT_TIMEOUT + 3);
                    for (int g = G; g < G + T && ok; ++g) {
                        const int st = g % NS;
                        ok = mbar_wait_warp(BAR(B_KFULL + st), (g / NS) & 1, ab, ST_WAIT_TIMEOUT + 4);
                        // the buffer: its scores have been read, or the P that took their place
                        if (S::POWN && ok && g > 0) ok = mbar_wait_warp(BAR(B_SFREE + ((g - 1) & 1)), ((g - 1) >> 1) & 1, ab, ST_WAIT_TIMEOUT + 15);
                        if (!S::POWN && ok && g >= NP) ok = mbar_wait_warp(BAR(B_PVDONE + g % NP), (g / NP - 1) & 1, ab, ST_WAIT_TIMEOUT + 15);
                        if (!ok) break;
                        tc_fence_after();
                        const uint32_t tS = utmem + uint32_t(S::tmem_s(g)), q_tile = sQ(s), k_tile = sK(st);
#pragma unroll
                        for (int kk = 0; kk < D / 16; ++kk) {
                            const uint32_t off = uint32_t(kk >> 2) * S::BOX + uint32_t(kk & 3) * 32u;
                            umma_ss(tS, smem_desc_at(kDescKMajor, q_tile + off), smem_desc_at(kDescKMajor, k_tile + off), idesc_s, kk > 0);
                        }
                        umma_commit(BAR(B_KEMPTY + st));
                        umma_commit(BAR(B_SFULL + (g & 3)));
                    }
                } else {
                    for (int t = 0; t < T; ++t) {
                        const int g = G + t, st = g % NS, w = g & 1;
                        const uint32_t tO = utmem + uint32_t(S::tmem_o + w * D), tP = utmem + uint32_t(S::tmem_p(g)), v_tile = sV(st);
                        ok = mbar_wait_warp(BAR(B_VFULL + st), (g / NS) & 1, ab, ST_WAIT_TIMEOUT + 5);
                        // The first P*V of a chain in an item overwrites its O: the epilogue of the last item that used it must have
                        // read it. (o_full and o_free count the items in which the chain had tiles, on both sides.)
                        const int n = w ? n1 : n0;
                        if (ok && t < 2 && n > 0) ok = mbar_wait_warp(BAR(B_OFREE + w), (n - 1) & 1, ab, ST_WAIT_TIMEOUT + 14);
                        if (ok) ok = mbar_wait_warp(BAR(B_PFULL + g % NP), (g / NP) & 1, ab, ST_WAIT_TIMEOUT + 6);
                        if (!ok) break;
                        tc_fence_after();
#pragma unroll
                        for (int kk = 0; kk < 8; ++kk)
                            umma_ts(tO, tP + uint32_t(kk) * 8u, smem_desc_at(desc_v, v_tile + uint32_t(kk) * 2048u), idesc_pv,
                                    (t > 1 || kk > 0) ? 1u : 0u);
                        umma_commit(BAR(B_VEMPTY + st));
                        umma_commit(BAR(B_PVDONE + g % NP));
                        if (t + 2 >= T) {  // the chain's last tile
                            umma_commit(BAR(B_OFULL + w));
                            if (w) ++n1; else ++n0;
                        }
                    }
                }
                if (!ok) break;
                G += T;
                if (lane == 0) mbar_arrive(BAR(B_ITEMEMPTY + s));
                __syncwarp();
            }
        }
        __syncwarp();
    } else if (warp >= 8) {
        // ------------------------------ epilogue group ------------------------------
        setmaxnreg_dec<kFwdEpilogueRegs>();
        const int r = tid & 127;
        const uint32_t lane_base = uint32_t((warp & 3) * 32) << 16;
        const float c = SCORED ? 1.f : p.scale_log2;
        const int tok_wide = r / p.G, tok_narrow = lane / p.G;
        // of a narrow item's sums: this thread adds up four columns of row r / 4
        const int row_sum = r >> 2, tok_sum = row_sum / p.G;
        int staged = 0;  // passes through the staging barrier
        bool alive = !aborted;
        if (alive && p.fill && p.starts) {
            // rows in front of the first sequence and behind the last one
            const int front = min(max(p.starts[0], 0), p.T), behind = max(min(p.starts[p.B], p.T), front);
            const int rows = front + p.T - behind;
            for (int64_t i = int64_t(blockIdx.x) * 4 + (warp & 3); i < int64_t(rows) * p.H; i += int64_t(gridDim.x) * 4) {
                const int t = int(i / p.H), h = int(i % p.H);
                for (int d = lane; d < p.D; d += 32) out[int64_t(t < front ? t : t - front + behind) * p.out_t + h * p.out_h + d] = 0;
            }
        }
        int G = 0;           // tiles of all earlier items
        int n0 = 0, n1 = 0;  // items in which the chains of group 0 and 1 had tiles
        for (int k = 0; alive; ++k) {
            const int s = k % NQ, use = k / NQ;
            alive = mbar_wait_warp(BAR(B_ITEMFULL + s), use & 1, ab, ST_WAIT_TIMEOUT + 12);
            if (!alive) break;
            volatile int* it = info + 16 * s;
            const int T = it[I_TILES], part = it[I_PART], hk = it[I_HEAD], tokens = it[I_TOKENS];
            if (it[I_MORE] < 0) break;
            const bool narrow = tokens <= p.narrow;
            const int tok = narrow ? tok_narrow : tok_wide, g_row = narrow ? lane - tok * p.G : r - tok * p.G, row = it[I_ROW] + tok;
            const bool valid = tok < tokens;
            {
                const int64_t row_of_table = it[I_SEQ] * p.table_stride;
                const int last = min((it[I_LO] + T) * kBlk, it[I_LEN]) - 1;
                for (int i = (it[I_LO] * kBlk >> p.log2_page) + r; i <= last >> p.log2_page && T > 0; i += kBlk)
                    if (uint32_t(p.table[row_of_table + i]) >= uint32_t(p.n_pages)) atomicCAS(p.status, 0, ST_PAGED_PAGE);
            }
            // the only wait here that lasts as long as an item: it allows each of the tiles what another wait may last
            const Abort item{ab.flag, ab.status, ab.limit * (T + 1)};
            alive = mbar_wait_warp(BAR(B_MLFULL + s), use & 1, item, ST_WAIT_TIMEOUT + 16);
            // an item without tiles: nobody has waited for its Q load yet, and its slot is about to be given away
            if (alive && T == 0) alive = mbar_wait_warp(BAR(B_QFULL + s), use & 1, ab, ST_WAIT_TIMEOUT + 17);
            const int we = G & 1;  // the chain that had the item's even tiles: index 0 below, 1 the other one
            const int i0 = we ? n1 : n0, i1 = we ? n0 : n1;
            if (alive && T > 0) alive = mbar_wait_warp(BAR(B_OFULL + we), i0 & 1, ab, ST_WAIT_TIMEOUT + 9);
            if (alive && T > 1) alive = mbar_wait_warp(BAR(B_OFULL + (we ^ 1)), i1 & 1, ab, ST_WAIT_TIMEOUT + 9);
            if (!alive) break;
            tc_fence_after();
            const float* ml = reinterpret_cast<const float*>(smem + S::off_ml) + s * (4 * kBlk);  // [2 groups][m, l][128]
            const int even = we * (2 * kBlk), odd = 2 * kBlk - even;
            const float m0 = ml[even + r], l0 = ml[even + kBlk + r], m1 = ml[odd + r], l1 = ml[odd + kBlk + r];
            float mt = fmaxf(m0, m1);
            if (narrow) {  // over the four warps' chains of the row
                for (int q = 0; q < 4; ++q) mt = fmaxf(mt, fmaxf(ml[even + 32 * q + lane], ml[odd + 32 * q + lane]));
            }
            const float a0 = (m0 == -INFINITY) ? 0.f : fast_exp2((m0 - mt) * c);
            const float a1 = (m1 == -INFINITY) ? 0.f : fast_exp2((m1 - mt) * c);
            float lt = l0 * a0 + l1 * a1;
            if (narrow) {
                lt = 0.f;
                for (int q = 0; q < 4; ++q) {
                    const float me = ml[even + 32 * q + lane], mo = ml[odd + 32 * q + lane];
                    lt += ml[even + kBlk + 32 * q + lane] * (me == -INFINITY ? 0.f : fast_exp2((me - mt) * c)) +
                          ml[odd + kBlk + 32 * q + lane] * (mo == -INFINITY ? 0.f : fast_exp2((mo - mt) * c));
                }
            }
            const float inv = (lt > 0.f) ? 1.0f / lt : lt == lt ? 0.f : lt;  // a NaN among a row's scores makes it NaN
            const float f0 = a0 * inv, f1 = a1 * inv;
            // a chain in which the row had no key takes no part, whatever the values behind its mask are
            const bool use0 = (T > 0) && (f0 != 0.f), use1 = (T > 1) && (f1 != 0.f);
            const bool both = __all_sync(0xffffffffu, !valid || (use0 && use1));
            const bool store = valid && misc[1] == 0;
            if (part >= 0 && store && (!narrow || warp == 8))  // (a piece that went NaN says so: -inf would pass for a piece without keys)
                p.part_lse[int64_t(part) * kBlk + r] = lt > 0.f ? fmaf(mt, c, log2f(lt)) : lt == lt ? -INFINITY : lt;
            float* const rows_of_part = p.part_o + (int64_t(part) * kBlk + (narrow ? row_sum : r)) * D;
            uint16_t* const row_out = narrow ? out + int64_t(it[I_ROW] + tok_sum) * p.out_t + int64_t(hk * p.G + row_sum - tok_sum * p.G) * p.out_h
                                             : out + int64_t(row) * p.out_t + int64_t(hk * p.G + g_row) * p.out_h;
            const bool store_sum = tok_sum < tokens && misc[1] == 0;
            float* const stage = reinterpret_cast<float*>(smem + S::off_q + s * S::TILE);  // (Q has been read) [2][4 warps][32 rows][16]
            const uint32_t tO0 = tmem + lane_base + uint32_t(S::tmem_o + we * D), tO1 = tmem + lane_base + uint32_t(S::tmem_o + (we ^ 1) * D);
#pragma unroll 1
            for (int q = 0; q < D / 16; ++q) {
                uint32_t x0[16], x1[16];
                // tcgen05.ld is warp-collective: always executed, the values are ignored when unused
                tmem_ld16(tO0 + uint32_t(q) * 16u, x0);
                tmem_ld16(tO1 + uint32_t(q) * 16u, x1);
                tc_wait_ld();
                if (q == D / 16 - 1) {  // O has been read: the MMA issuers may start another item's P*V
                    tc_fence_before();
                    if (T > 0) mbar_arrive_warp(BAR(B_OFREE + we), lane);
                    if (T > 1) mbar_arrive_warp(BAR(B_OFREE + (we ^ 1)), lane);
                }
                if (both) {
#pragma unroll
                    for (int y = 0; y < 16; ++y) x0[y] = __float_as_uint(fmaf(__uint_as_float(x1[y]), f1, __uint_as_float(x0[y]) * f0));
                } else {
#pragma unroll
                    for (int y = 0; y < 16; ++y) {
                        float v = 0.f;
                        if (use0) v = __uint_as_float(x0[y]) * f0;
                        if (use1) v = fmaf(__uint_as_float(x1[y]), f1, v);
                        x0[y] = __float_as_uint(v);
                    }
                }
                if (narrow) {
                    // the warps' sums of a row, 16 columns at a time, through one of two buffers
                    float* const buf = stage + (q & 1) * 2048;
#pragma unroll
                    for (int y = 0; y < 4; ++y)
                        *reinterpret_cast<uint4*>(buf + (warp & 3) * 512 + lane * 16 + 4 * ((y + (lane >> 1)) & 3)) = make_uint4(x0[4 * y], x0[4 * y + 1], x0[4 * y + 2], x0[4 * y + 3]);
                    mbar_arrive_warp(BAR(B_STAGED), lane);
                    alive = mbar_wait_warp(BAR(B_STAGED), staged++ & 1, ab, ST_WAIT_TIMEOUT + 18);
                    if (!alive) break;
                    if (store_sum && 16 * q < p.D) {
                        const int y = r & 3;
                        float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int u = 0; u < 4; ++u) {
                            const float4 x = *reinterpret_cast<const float4*>(buf + u * 512 + row_sum * 16 + 4 * ((y + (row_sum >> 1)) & 3));
                            v[0] += x.x; v[1] += x.y; v[2] += x.z; v[3] += x.w;
                        }
                        if (part >= 0) *reinterpret_cast<float4*>(rows_of_part + 16 * q + 4 * y) = make_float4(v[0], v[1], v[2], v[3]);
                        else *reinterpret_cast<uint2*>(row_out + 16 * q + 4 * y) = make_uint2(pack2<BF16>(v[0], v[1]), pack2<BF16>(v[2], v[3]));
                    }
                } else if (store && 16 * q < p.D) {
                    if (part >= 0) {
#pragma unroll
                        for (int y = 0; y < 4; ++y)
                            *reinterpret_cast<uint4*>(rows_of_part + 16 * q + 4 * y) = make_uint4(x0[4 * y], x0[4 * y + 1], x0[4 * y + 2], x0[4 * y + 3]);
                    } else {
                        auto two = [&](int y) { return pack2<BF16>(__uint_as_float(x0[y]), __uint_as_float(x0[y + 1])); };
                        uint4* dst = reinterpret_cast<uint4*>(row_out + 16 * q);
                        dst[0] = make_uint4(two(0), two(2), two(4), two(6));
                        dst[1] = make_uint4(two(8), two(10), two(12), two(14));
                    }
                }
            }
            if (!alive) break;
            if (narrow) fence_proxy_async();  // the slot may take another item's Q
            G += T;
            n0 += (we ? T > 1 : T > 0) ? 1 : 0;
            n1 += (we ? T > 0 : T > 1) ? 1 : 0;
            __syncwarp();
            if (lane == 0) mbar_arrive(BAR(B_ITEMEMPTY + s));
        }
    } else {
        setmaxnreg_inc<kFwdSoftmaxRegs>();
        // ------------------------------ softmax groups ------------------------------
        const int w = warp >> 2;  // group
        const int r = tid & 127;  // row inside the tile
        const uint32_t lane_base = uint32_t((warp & 3) * 32) << 16;
        const float c = SCORED ? 1.f : p.scale_log2;
        const uint32_t tO = tmem + lane_base + uint32_t(S::tmem_o + w * D);
        const int tok_wide = r / p.G, tok_narrow = lane / p.G;
        bool alive = !aborted;
        // Rows of V behind the keys that the item sees hold what was in the page, or in the stage: zeros, before P*V(g) is issued. A quarter of them a warp.
        auto zero_behind = [&](int g, int real) {
            const int st = g % NS;
            if (!mbar_wait_warp(BAR(B_VFULL + st), (g / NS) & 1, ab, ST_WAIT_TIMEOUT + 19)) return false;
            // (not unrolled: it stands twice in the code of the softmax warps, a batch of chunks and tokens with a bias 224 us for 237)
#pragma unroll 1
            for (int x = 0; x < S::NBOX; ++x)
#pragma unroll 1
                for (int i = real * 8 + r; i < kBlk * 8; i += kBlk) reinterpret_cast<uint4*>(smem + S::off_v + st * S::TILE + x * S::BOX)[i] = make_uint4(0, 0, 0, 0);
            fence_proxy_async();
            return true;
        };
        auto rescale = [&](float alpha) {
#pragma unroll 1
            for (int q = 0; q < D / 16; ++q) {
                uint32_t orr[16];
                tmem_ld16(tO + uint32_t(q) * 16u, orr);
                tc_wait_ld();
#pragma unroll
                for (int x = 0; x < 16; ++x) orr[x] = __float_as_uint(__uint_as_float(orr[x]) * alpha);
                tmem_st16(tO + uint32_t(q) * 16u, orr);
            }
            tc_wait_st();
        };
        int G = 0;  // tiles of all earlier items
        for (int k = 0; alive; ++k) {
            const int s = k % NQ, use = k / NQ;
            alive = mbar_wait_warp(BAR(B_ITEMFULL + s), use & 1, ab, ST_WAIT_TIMEOUT + 12);
            if (!alive) break;
            volatile int* it = info + 16 * s;
            const int T = it[I_TILES], lo = it[I_LO];
            if (it[I_MORE] < 0) break;
            const int pos0 = it[I_POS], len = it[I_LEN], front = it[I_FRONT];
            const int tokens = it[I_TOKENS];
            const bool narrow = tokens <= p.narrow;
            const int tok = narrow ? tok_narrow : tok_wide, g_row = narrow ? lane - tok * p.G : r - tok * p.G;
            const bool valid = tok < tokens;
            const bool active = __any_sync(0xffffffffu, valid);  // does this warp hold a query at all?
            const int pos = pos0 + tok;
            const int last = pos < 0 ? -1 : min(max(pos, front - 1), len - 1);  // the last key that this row sees (a token in front of the sequence sees no prefix, either)
            const int all_see = pos0 < 0 ? -1 : min(max(pos0, front - 1), len - 1);  // and that all rows of the tile see
            const int seen = min(max(pos0 + tokens, front), len);              // keys that any row sees
            float slope = 0.f;
            if constexpr (SCORED) {
                if (p.score.slopes) slope = p.score.slopes[int64_t(it[I_HEAD]) * p.G + g_row] * kScoreLog2e;
            }
            const int t0 = (G ^ w) & 1;  // this group's first tile of the item
            float m_run = -INFINITY, l_run = 0.f;

            for (int t = t0; t < T && alive; t += 2) {
                const int k0 = (lo + t) * kBlk;
                const int g = G + t;
                const uint32_t tS = tmem + lane_base + uint32_t(S::tmem_s(g)), tP = tmem + lane_base + uint32_t(S::tmem_p(g));
                // P*V of the group's tile before: it has read its P and added to O
                auto pv_before = [&] { return g < 2 || mbar_wait_warp(BAR(B_PVDONE + (g - 2) % NP), ((g - 2) / NP) & 1, ab, ST_WAIT_TIMEOUT + 8); };
                alive = mbar_wait_warp(BAR(B_SFULL + (g & 3)), (g >> 2) & 1, ab, ST_WAIT_TIMEOUT + 7);
                if (!alive) break;
                tc_fence_after();
                if (!active) {  // no row of this warp is a query: its lanes of P and O are never stored
                    if (S::POWN) {
                        mbar_arrive_warp(BAR(B_SFREE + w), lane);
                        alive = pv_before();
                        if (!alive) break;
                    }
                    if (seen - k0 < kBlk) alive = zero_behind(g, seen - k0);
                    if (!alive) break;
                    mbar_arrive_warp(BAR(B_PFULL + g % NP), lane);
                    continue;
                }
                if (narrow) {
                    // The tile's rows are the same 32 four times over, and this warp has 32 keys of each (its P of the others is 0): a chain of its own,
                    // which the epilogue merges with those of the other warps.
                    const int quarter = warp & 3, kq = k0 + 32 * quarter;
                    uint32_t sq[32];
                    tmem_ld32(tS + uint32_t(quarter) * 32u, sq);
                    tc_wait_ld();
                    if (S::POWN) {
                        tc_fence_before();
                        mbar_arrive_warp(BAR(B_SFREE + w), lane);
                    }
                    float* v = reinterpret_cast<float*>(sq);
                    if constexpr (SCORED) {
                        if (seen - kq < 32) {
#pragma unroll
                            for (int x = 0; x < 32; ++x) v[x] = x < seen - kq ? v[x] : 0.f;
                        }
                        const Bias bias(slope, front == 0, pos0 - (kq + 31), pos0 + 31 - kq);
                        score_row<KIND, 32>(v, p.score, bias, p.scale_log2, pos - kq, valid, m_run == -INFINITY ? 0.f : m_run);
                    }
                    if (kq + 31 > all_see) {
                        const uint32_t keep = first_bits(last - kq + 1);
#pragma unroll
                        for (int x = 0; x < 32; ++x) v[x] = (keep & (1u << x)) ? v[x] : -INFINITY;
                    }
                    float mx[4];
#pragma unroll
                    for (int a = 0; a < 4; ++a) mx[a] = max3(v[a], v[4 + a], v[8 + a]);
#pragma unroll
                    for (int x = 12; x < 28; x += 8) {
#pragma unroll
                        for (int a = 0; a < 4; ++a) mx[a] = max3(mx[a], v[x + a], v[x + 4 + a]);
                    }
#pragma unroll
                    for (int a = 0; a < 4; ++a) mx[a] = fmaxf(mx[a], v[28 + a]);
                    const float top = fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]);
                    float m_new = fmaxf(m_run, top);
                    bool need = (m_new - m_run) * c > 8.0f;
                    if constexpr (SCORED) {
                        const bool fresh = m_run == -INFINITY;
                        need = fresh ? top != -INFINITY : top > 8.0f;
                        m_new = (fresh ? 0.f : m_run) + top;
                    }
                    if (!need) m_new = m_run;
                    const bool scale_o = __any_sync(0xffffffffu, need) && t > t0;
                    if (S::POWN || scale_o) {  // P*V of the group's tile before has read its P and added to O
                        alive = pv_before();
                        if (!alive) break;
                        tc_fence_after();
                    }
                    const float alpha = need ? fast_exp2((m_run - m_new) * c) : 1.0f;
                    l_run *= alpha;
                    if (scale_o) rescale(alpha);
                    m_run = m_new;
                    // (SCORED: what is left to be subtracted)
                    const float mneg = SCORED ? (need ? -top : 0.f) : (m_run == -INFINITY) ? 0.f : -m_run * c;
                    float l4[4] = {0.f, 0.f, 0.f, 0.f};
                    uint32_t pk[16];
#pragma unroll
                    for (int x = 0; x < 32; x += 2) {
                        const float p0 = fast_exp2(fmaf(v[x], c, mneg)), p1 = fast_exp2(fmaf(v[x + 1], c, mneg));
                        l4[x & 2] += p0;
                        l4[(x & 2) + 1] += p1;
                        pk[x / 2] = pack2<BF16>(p0, p1);
                    }
                    uint32_t zero[16] = {};
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        if (q != quarter) tmem_st16(tP + uint32_t(q) * 16u, zero);
                    tmem_st16(tP + uint32_t(quarter) * 16u, pk);
                    tc_wait_st();
                    if (seen - k0 < kBlk) alive = zero_behind(g, seen - k0);
                    tc_fence_before();
                    mbar_arrive_warp(BAR(B_PFULL + g % NP), lane);
                    if (!alive) break;
                    l_run += (l4[0] + l4[1]) + (l4[2] + l4[3]);
                    continue;
                }
                uint32_t sr[128];
#pragma unroll
                for (int q = 0; q < 4; ++q) tmem_ld32(tS + uint32_t(q) * 32u, sr + q * 32);
                tc_wait_ld();
                if (S::POWN) {
                    tc_fence_before();
                    mbar_arrive_warp(BAR(B_SFREE + w), lane);  // the next tile's scores may overwrite these
                }
                float* sc = reinterpret_cast<float*>(sr);
                const int real = seen - k0;  // keys of the tile that some row sees
                // A capped tile without a mask is not capped before its exponentials: the greatest score tells the greatest capped one, and the polynomial
                // runs beside the special-function unit. (With a bias the greatest one has to be looked for behind it.)
                bool late = false;
                if constexpr (SCORED) {
                    // (what the others' scores are must not tell the warp which form of the cap to take)
                    if (real < kBlk) {
#pragma unroll
                        for (int x = 0; x < kBlk; ++x) sc[x] = x < real ? sc[x] : 0.f;
                    }
                    const Bias bias(slope, front == 0, pos0 - (k0 + kBlk - 1), pos0 + kBlk - 1 - k0);
                    if constexpr (KIND == SCORE_CAPPED) late = k0 + kBlk - 1 <= all_see && !any_beyond<kBlk>(sc, valid ? p.score.most : INFINITY);
                    if (!late) score_row<KIND, kBlk>(sc, p.score, bias, p.scale_log2, pos - k0, valid, m_run == -INFINITY ? 0.f : m_run);
                }
                if (k0 + kBlk - 1 > all_see) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const uint32_t keep = first_bits(last - k0 + 1 - 32 * q);
                        if (__any_sync(0xffffffffu, keep != ~0u)) {
#pragma unroll
                            for (int x = 0; x < 32; ++x) sc[32 * q + x] = (keep & (1u << x)) ? sc[32 * q + x] : -INFINITY;
                        }
                    }
                }
                float mxa[8];
#pragma unroll
                for (int a = 0; a < 8; ++a) mxa[a] = max3(sc[a], sc[8 + a], sc[16 + a]);
#pragma unroll
                for (int x = 24; x < 120; x += 16) {
#pragma unroll
                    for (int a = 0; a < 8; ++a) mxa[a] = max3(mxa[a], sc[x + a], sc[x + 8 + a]);
                }
#pragma unroll
                for (int a = 0; a < 8; ++a) mxa[a] = fmaxf(mxa[a], sc[120 + a]);
                float mx = fmaxf(max3(mxa[0], mxa[1], mxa[2]), max3(max3(mxa[3], mxa[4], mxa[5]), mxa[6], mxa[7]));
                float m_new = fmaxf(m_run, mx);
                // lazy rescale: keep the old reference point while the new maximum is within 2^8 of it
                bool need = (m_new - m_run) * c > 8.0f;
                if constexpr (SCORED) {  // (the scores, and mx, are relative to the old reference point, or to 0 in front of a row's first key)
                    const bool fresh = m_run == -INFINITY;
                    if (late) mx = cap_one(mx, p.score) - (fresh ? 0.f : m_run);
                    need = fresh ? mx != -INFINITY : mx > 8.0f;
                    m_new = (fresh ? 0.f : m_run) + mx;
                }
                if (!need) m_new = m_run;
                if (S::POWN) {  // this tile's P overwrites that one's
                    alive = pv_before();
                    if (!alive) break;
                    tc_fence_after();
                }
                if (__any_sync(0xffffffffu, need)) {
                    if (SCORED && !late) {
                        const float less = need ? -mx : 0.f;
#pragma unroll
                        for (int x = 0; x < 128; x += 2) unpack_f2(add_f2(pack_f2(sc[x], sc[x + 1]), pack_f2(less, less)), sc[x], sc[x + 1]);
                    }
                    const float alpha = need ? fast_exp2((m_run - m_new) * c) : 1.0f;
                    l_run *= alpha;
                    if (t > t0) {
                        if (!S::POWN) {
                            alive = pv_before();
                            if (!alive) break;
                            tc_fence_after();
                        }
                        rescale(alpha);
                    }
                }
                m_run = m_new;
                const float mneg = (m_run == -INFINITY) ? 0.f : -m_run * c;
                // exp2(s*c - m*c) on packed pairs
                const uint64_t c2 = pack_f2(c, c), mneg2 = pack_f2(mneg, mneg);
                uint64_t lacc0 = pack_f2(0.f, 0.f), lacc1 = lacc0;
                auto exponentials = [&](auto exponent) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        uint32_t pk[16];
#pragma unroll
                        for (int x = 0; x < 16; ++x) {
                            float x0, x1;
                            unpack_f2(exponent(pack_f2(sc[32 * q + 2 * x], sc[32 * q + 2 * x + 1])), x0, x1);
                            const float p0 = fast_exp2(x0), p1 = fast_exp2(x1);
                            if (x & 1) lacc1 = add_f2(lacc1, pack_f2(p0, p1)); else lacc0 = add_f2(lacc0, pack_f2(p0, p1));
                            pk[x] = pack2<BF16>(p0, p1);
                        }
                        tmem_st16(tP + uint32_t(q) * 16u, pk);
                    }
                };
                if constexpr (!SCORED) exponentials([&](uint64_t s2) { return fma_f2(s2, c2, mneg2); });
                else if (KIND == SCORE_CAPPED && late) exponentials([&](uint64_t s2) { return fma_f2(s2, cap_poly(s2, p.score), mneg2); });
                else exponentials([&](uint64_t s2) { return s2; });
                tc_wait_st();
                if (real < kBlk) alive = zero_behind(g, real);
                tc_fence_before();
                mbar_arrive_warp(BAR(B_PFULL + g % NP), lane);
                if (!alive) break;
                {
                    float a0, a1, b0, b1;
                    unpack_f2(lacc0, a0, a1);
                    unpack_f2(lacc1, b0, b1);
                    l_run += (a0 + a1) + (b0 + b1);
                }
            }
            if (!alive) break;
            float* ml = reinterpret_cast<float*>(smem + S::off_ml) + s * (4 * kBlk) + w * (2 * kBlk) + r;
            ml[0] = m_run;
            ml[kBlk] = l_run;
            mbar_arrive_warp(BAR(B_MLFULL + s), lane);
            G += T;
            __syncwarp();
            if (lane == 0) mbar_arrive(BAR(B_ITEMEMPTY + s));
        }
    }

    // ------------------------------ tear-down ------------------------------
    tc_fence_before();
    __syncthreads();
    if (warp == 13) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// Merges the pieces of the items that a cut went through: O = sum_s w_s O_s with w_s = 2^(lse_s - lse). The blocks (w, 0 .. 3) look after the item that
// the cut before worker w goes through first, each after 32 of its rows; the attention kernel has left word of its pieces. A piece whose lse is NaN or +inf makes the row its own, as in fwd_combine_kernel. All sums in fp32, in an order that the number of rows
// and pieces gives. Bound by latency: a warp has four rows, whose loads are in flight together, and where there are few rows (a decoded token's
// heads) several warps share the pieces.
constexpr int kCombineThreads = 256, kCombineRows = 4;

template <int D, bool BF16>
__global__ void __launch_bounds__(kCombineThreads, 2) paged_combine_kernel(const PagedParams p) {
    constexpr int kOwn = D / 32, kBatch = 4, kWarps = kCombineThreads / 32;  // columns of a lane; pieces in flight
    __shared__ float sums[kWarps][kCombineRows][D + 2];
    follow_stream();
    const int w = int(blockIdx.x), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // (both loads in flight together: one behind the other cost a call of one token a microsecond)
    const int status = *reinterpret_cast<volatile int*>(p.status);
    const int4 merge = p.merge[w];
    const bool failed = status_is_fatal(status) | (merge.x < 0);  // (the host may have cleared the word since)
    const int row0 = int(blockIdx.y) * kWarps * kCombineRows, pieces = merge.x, rows = (merge.z & 255) * p.G - row0, hk = merge.z >> 8;
    auto slot = [&](int s) { return 2 * (merge.w + s) + (s == 0 ? 1 : 0); };
    if (!failed && (pieces < 2 || rows <= 0)) return;
    if (failed) {
        // A time-out, of an earlier launch, of one on another stream meanwhile, or in the attention kernel: some of its blocks, or all, have left their rows as they
        // were, and which is not known. All rows become NaN, or those of the sequences in an output of the caller's.
        const bool all = p.fill || !p.starts;
        const int front = all ? 0 : min(max(p.starts[0], 0), p.T), behind = all ? p.T : max(min(p.starts[p.B], p.T), front);
        const int64_t first = int64_t(front) * p.H, end = int64_t(behind) * p.H;
        for (int64_t i = first + (int64_t(blockIdx.y) * gridDim.x + w) * kWarps + warp; i < end; i += int64_t(gridDim.x) * gridDim.y * kWarps)
            for (int d = lane; d < p.D; d += 32) static_cast<uint16_t*>(p.out)[i / p.H * p.out_t + i % p.H * p.out_h + d] = 0xffffu;
        return;
    }
    const int groups = min(cdiv(rows, kCombineRows), kWarps), subs = kWarps / groups;
    const int sub = warp / groups, r0 = (warp - sub * groups) * kCombineRows;  // (of this block's rows)
    // A warp's own pieces first: their greatest lse, and the sums relative to it. (An empty piece has an lse of -inf.)
    float top[kCombineRows], acc[kCombineRows][kOwn] = {}, total[kCombineRows] = {};
#pragma unroll
    for (int i = 0; i < kCombineRows; ++i) top[i] = -INFINITY;
    // A spoilt row's "greatest" is +inf: of such pieces each counts once, and all others not at all.
    auto weight = [](float lse, float most) { return lse < INFINITY ? (lse == -INFINITY ? 0.f : fast_exp2(lse - most)) : 1.f; };
    if (sub < subs) {
#pragma unroll 1
        for (int s0 = sub; s0 < pieces; s0 += subs * kBatch) {
            float v[kBatch][kCombineRows][kOwn], lse[kBatch][kCombineRows];
#pragma unroll
            for (int s = 0; s < kBatch; ++s) {
                const int64_t at = int64_t(slot(min(s0 + s * subs, pieces - 1))) * kBlk;
#pragma unroll
                for (int i = 0; i < kCombineRows; ++i) {
                    const int64_t row = at + row0 + min(r0 + i, rows - 1);
                    lse[s][i] = p.part_lse[row];
                    if constexpr (kOwn == 4) {
                        const float4 x = *reinterpret_cast<const float4*>(p.part_o + row * D + 4 * lane);
                        v[s][i][0] = x.x; v[s][i][1] = x.y; v[s][i][2] = x.z; v[s][i][3] = x.w;
                    } else {
                        // (columns beyond a head dim of 16 or 32 have not been written, and go nowhere)
                        const float2 x = *reinterpret_cast<const float2*>(p.part_o + row * D + 2 * lane);
                        v[s][i][0] = x.x; v[s][i][1] = x.y;
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < kCombineRows; ++i) {
                float most = top[i];
#pragma unroll
                for (int s = 0; s < kBatch; ++s) {
                    if (s0 + s * subs >= pieces) lse[s][i] = -INFINITY;
                    most = lse[s][i] < INFINITY ? fmaxf(most, lse[s][i]) : INFINITY;
                }
                const float keep = top[i] == most ? 1.f : weight(top[i], most);  // (0 if nothing was there, or the row is spoilt from here on)
                total[i] *= keep;
#pragma unroll
                for (int c = 0; c < kOwn; ++c) acc[i][c] = keep == 0.f ? 0.f : acc[i][c] * keep;
                top[i] = most;
#pragma unroll
                for (int s = 0; s < kBatch; ++s) {
                    const float wgt = weight(lse[s][i], most);
                    if (wgt == 0.f) continue;
                    total[i] += wgt;
#pragma unroll
                    for (int c = 0; c < kOwn; ++c) acc[i][c] = fmaf(wgt, v[s][i][c], acc[i][c]);
                }
            }
        }
    }
    if (subs > 1) {  // (the same for all threads)
        float (*mine)[D + 2] = sums[warp];
        if (sub > 0 && sub < subs) {
#pragma unroll
            for (int i = 0; i < kCombineRows; ++i) {
#pragma unroll
                for (int c = 0; c < kOwn; ++c) mine[i][lane * kOwn + c] = acc[i][c];
                if (lane == 0) {
                    mine[i][D] = total[i];
                    mine[i][D + 1] = top[i];
                }
            }
        }
        __syncthreads();
        if (sub == 0) {
#pragma unroll
            for (int i = 0; i < kCombineRows; ++i) {
                float most = top[i];
                for (int u = 1; u < subs; ++u) most = fmaxf(most, sums[warp + u * groups][i][D + 1]);
                for (int u = 0; u < subs; ++u) {
                    const float* other = sums[warp + u * groups][i];
                    const float t = u == 0 ? top[i] : other[D + 1], wgt = t == most && t != -INFINITY ? 1.f : t < INFINITY ? weight(t, most) : 0.f;
                    const float tt = u == 0 ? total[i] : other[D];
                    total[i] = (u == 0 ? 0.f : total[i]) + (wgt == 0.f ? 0.f : tt * wgt);
#pragma unroll
                    for (int c = 0; c < kOwn; ++c) {
                        const float x = u == 0 ? acc[i][c] : other[lane * kOwn + c];
                        acc[i][c] = (u == 0 ? 0.f : acc[i][c]) + (wgt == 0.f ? 0.f : x * wgt);
                    }
                }
            }
        }
    }
    if (sub > 0 || lane * kOwn >= p.D) return;
#pragma unroll
    for (int i = 0; i < kCombineRows; ++i) {
        if (r0 + i >= rows) return;
        const int r = row0 + r0 + i, tok = r / p.G, g = r - tok * p.G;
        const float inv = total[i] > 0.f ? 1.f / total[i] : 0.f;
        uint16_t* out = static_cast<uint16_t*>(p.out) + int64_t(merge.y + tok) * p.out_t + int64_t(hk * p.G + g) * p.out_h + lane * kOwn;
        if constexpr (kOwn == 4)
            *reinterpret_cast<uint2*>(out) = make_uint2(pack2<BF16>(acc[i][0] * inv, acc[i][1] * inv), pack2<BF16>(acc[i][2] * inv, acc[i][3] * inv));
        else
            *reinterpret_cast<uint32_t*>(out) = pack2<BF16>(acc[i][0] * inv, acc[i][1] * inv);
    }
}

// ---- host launchers (called from paged.cu) ----------------------------------------------
template <int D, bool BF16, int KIND>
static cudaError_t launch_paged_t(const CUtensorMap& tq, const CUtensorMap& tn, const CUtensorMap& tk, const CUtensorMap& tv, const PagedParams& p, int workers, cudaStream_t stream) {
    auto kern = paged_fwd_kernel<D, BF16, KIND>;
    constexpr int smem = PagedSmem<D>::total;
    static SmemAllowed allowed;
    cudaError_t e = allow_smem(kern, smem, allowed);
    if (e != cudaSuccess) return e;
    e = launch_overlapping(kern, dim3(workers), kFwdThreads, smem, stream, tq, tn, tk, tv, p);
    if (e != cudaSuccess) return e;
    return launch_overlapping(paged_combine_kernel<D, BF16>, dim3(workers, kBlk / (kCombineThreads / 32 * kCombineRows)), kCombineThreads, 0, stream, p);
}

cudaError_t launch_paged_fwd(bool bf16, const CUtensorMap& tq, const CUtensorMap& tn, const CUtensorMap& tk, const CUtensorMap& tv, const PagedParams& p, int workers, cudaStream_t stream) {
    auto pick = [&](auto d, auto kind) {
        constexpr int kD = decltype(d)::value, kKind = decltype(kind)::value;
        return bf16 ? launch_paged_t<kD, true, kKind>(tq, tn, tk, tv, p, workers, stream) : launch_paged_t<kD, false, kKind>(tq, tn, tk, tv, p, workers, stream);
    };
    using std::integral_constant;
    auto of = [&](auto d) {
        if (p.score.kind == SCORE_CAPPED_BIAS) return pick(d, integral_constant<int, SCORE_CAPPED_BIAS>{});
        if (p.score.kind == SCORE_CAPPED) return pick(d, integral_constant<int, SCORE_CAPPED>{});
        if (p.score.slopes) return pick(d, integral_constant<int, SCORE_BIAS>{});
        return pick(d, integral_constant<int, SCORE_PLAIN>{});  // (a prefix alone is part of the mask)
    };
    return p.D == 128 ? of(integral_constant<int, 128>{}) : of(integral_constant<int, 64>{});
}

}  // namespace fa
