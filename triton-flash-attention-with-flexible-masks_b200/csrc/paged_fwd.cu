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
#include <cstddef>
#include <type_traits>
#include "common.cuh"
#include "paged_plan.cuh"
#include "params.cuh"

namespace fa {

// Instances. FORM_MASKED: perhaps a window, perhaps drafted tokens whose parents are given. A tile of keys that the window hides from all of an item's tokens is not among its
// tiles, and what lies in such keys of the others is as far from the results as what lies behind the sequence: V's rows are zeroed, scores masked. A drafted token's branch is
// walked once an item, by the thread of each of its rows, and left as bits in shared memory: a load for each step, each behind the one before (with a window twice, first for the depth), which
// the first keys' way here hides of shallow trees alone. 16 sequences, 32 / 8 heads of 128, 60 new tokens behind 4000, us, a star | a chain 123 | 125; 256 new tokens 344 | 422, with a window of 512
// 168 | 284; one sequence, 256 behind 1200, 28 | 39 and 27 | 56.
// FORM_E4M3: the cache is of 8 bits. The rows of K and V land as they are in rings of their own, with their scales; each tile is turned
// into the fp16 tile that the products read (a row is e4m3 times a power of two from 2^-15 to 2^7, all of whose numbers are fp16's: nothing is rounded), with hidden rows as zeros: K's by the epilogue
// group, which has nothing to do while an item lasts, V's by the softmax group that owns the tile. The products are fp16's also where q is bf16: q's rows are brought to fp16, by a power of two where their greatest entry asks for it (their scores take it back in fp32),
// and P is 2^7 times as large as elsewhere, which brings what fp16 cannot tell from 0 from 2^-25 down to 2^-32 of a row's reference (l and O have the factor alike).
// FORM_DIRECT: of 8 bits and single tokens of few heads, as the host can tell: all items are multiplied by warps from the rings, and these have nearly all of shared memory. (The tiles of the tensor cores leave 3 and
// 2 places of 16 KB.)
enum : int { FORM_PLAIN = 0, FORM_MASKED = 1, FORM_E4M3 = 2, FORM_DIRECT = 4 };

// E4M3: rows of an item up to which warps multiply it directly. us, 32 single tokens over 349 MB, 8 kv heads of 128, 8 | 16 heads a kv head: by the tensor cores - | 148, directly 88 | 114, in
// the instance of single tokens 79 | 117.
constexpr int kDirectRows = 16;

template <int D, int FORM>
struct PagedSmem {
    static constexpr bool E4M3 = (FORM & FORM_E4M3) != 0, DIRECT = (FORM & FORM_DIRECT) != 0;
    static constexpr int NS = DIRECT ? 0 : E4M3 ? (D == 128 ? 1 : 2) : (D == 128) ? 2 : 4;  // depth of the K ring and of the V ring
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
    static constexpr int QBOX = DIRECT ? 32 * 128 : BOX, QTILE = QBOX * NBOX;
    static constexpr int off_q = 0;  // NQ Q tiles
    static constexpr int off_k = NQ * QTILE;
    static constexpr int off_v = off_k + NS * TILE;
    // E4M3: rings of rows as they are, and of their scales; the factor of each row's scores
    static constexpr int RAW = E4M3 ? kBlk * D : 0;
    static constexpr int NRK = !E4M3 ? 0 : DIRECT ? (D == 128 ? 4 : 8) : D == 128 ? 3 : 5, NRV = !E4M3 ? 0 : DIRECT ? NRK : D == 128 ? 2 : 5;
    // Barriers of those rings, and of V's places that have been read. A wait goes by a phase's parity, so that whoever waits must have seen the phase before: the groups take tiles in turn, and with
    // an odd number of places, which both groups come to, there are two barriers a place, one for each group's tiles. (A tile that lands before the one in front of it would let a group through a phase early.)
    static constexpr int NBK = NRK % 2 ? 2 * NRK : NRK, NBV = NRV % 2 ? 2 * NRV : NRV, NVE = E4M3 && NS % 2 ? 2 * NS : NS;
    static_assert(!E4M3 || (NBK % 2 == 0 && NBV % 2 == 0 && NVE % 2 == 0), "a group comes to the same barriers again");
    static constexpr int SUMS = 8 * kDirectRows * D * 4, off_sums = off_k;  // E4M3: what the warps leave of O; K's and V's tiles have the place, or nobody else
    static_assert(DIRECT || !E4M3 || SUMS <= 2 * NS * TILE, "room for the sums");
    static constexpr int off_raw_k = DIRECT ? off_sums + SUMS : off_v + NS * TILE, off_raw_v = off_raw_k + NRK * RAW;
    static constexpr int off_ml = off_raw_v + NRV * RAW;         // float [NQ][2 groups][m, l][128]
    static constexpr int off_info = off_ml + NQ * 4 * kBlk * 4;  // int32 [NQ][16]: see I_*
    static constexpr int off_scale_k = off_info + NQ * 64, off_scale_v = off_scale_k + NRK * kBlk;
    static constexpr int off_factor = off_scale_v + NRV * kBlk;  // float [NQ][128]
    static constexpr int off_plan = off_factor + (E4M3 ? NQ * kBlk * 4 : 0);
    static constexpr int off_bar = off_plan + int(sizeof(PagedPlan));
    // item_full[NQ] item_empty[NQ] q_full[NQ] ml_full[NQ] staged k_full[NS] k_empty[NS] v_full[NS] v_empty[NVE]
    // s_full[4] s_free[2] p_full[NP] pv_done[NP] o_full[2] o_free[2]; E4M3: raw_k_full[NBK] raw_k_empty[NBK] raw_v_full[NBV] raw_v_empty[NBV] q_ready[NQ] sums_free
    static constexpr int n_common = 4 * NQ + 1 + 3 * NS + NVE + 6 + 2 * NP + 4, n_bar = n_common + 2 * NBK + 2 * NBV + (E4M3 ? NQ + 1 : 0);
    static constexpr int off_misc = off_bar + n_bar * 8;  // tmem slot, abort flag
    static constexpr int total = off_misc + 16;
    static_assert(off_plan % 8 == 0 && off_bar % 8 == 0, "alignment");
    // FORM_MASKED: bits [2 groups][kPagedTree / 32][128 rows] of the new tokens that a drafted one sees, in the place of the plan's sums, which nobody needs when the
    // first item is there
    static constexpr int off_masks = off_plan + int(offsetof(PagedPlan, sums)), kMaskWords = kPagedTree / 32;
    static_assert(2 * kMaskWords * kBlk * 4 <= int(sizeof(PagedPlan::sums)), "room for the masks");
};
template <int D, int FORM>
constexpr bool kPagedFits = PagedSmem<D, FORM>::total <= 232448 && PagedSmem<D, FORM>::total > 116736;  // the budget, and no other block beside it on the SM
static_assert(kPagedFits<128, FORM_PLAIN> && kPagedFits<64, FORM_PLAIN> && kPagedFits<128, FORM_E4M3> && kPagedFits<64, FORM_E4M3> &&
              kPagedFits<128, FORM_E4M3 | FORM_DIRECT> && kPagedFits<64, FORM_E4M3 | FORM_DIRECT>, "shared memory");

// What an item's slot says: number of its key tiles, the first one, whether there is an item (1, or -1: no more), kv head, first row of its tokens in
// q and out, how many of them, position of the first one, the sequence's length, its prefix, the sequence, slot of the workspace (-1: straight to out)
// FORM_MASKED: key blocks from I_BORDER on lie I_SKIP further (I_TILES and I_LO count without those in between); place of a tree's first new token (else the
// length); first row of the sequence
enum : int { I_TILES = 0, I_LO, I_MORE, I_HEAD, I_ROW, I_TOKENS, I_POS, I_LEN, I_FRONT, I_SEQ, I_PART, I_BORDER, I_SKIP, I_BASE, I_FIRST };

// E4M3: where 16 numbers of a row lie in a tile of a ring (the 128- or 64-byte swizzle of the copy: lanes of neighbouring rows and of every other row find different banks)
template <int D>
__device__ __forceinline__ int raw_place(int row, int part) { return row * D + ((part ^ (D == 128 ? row & 7 : row >> 1 & 3)) << 4); }
// Where four columns of a row of a warp's O lie, so that those who write together, and who read together, have eight different 16-byte places
template <int D>
__device__ __forceinline__ int sums_place(int row, int four) { return four ^ (D == 128 ? row >> 1 & 3 : (row >> 1 & 1) | (row >> 2 & 1) << 2); }
// A row's scale, from its exponent biased by 127, as two numbers of fp16 and in fp32
__device__ __forceinline__ uint32_t scale_to_h2(uint32_t biased) {
    const int e = min(max(int(biased), kScaleLeast), kScaleMost) - kScaleLeast;
    const uint32_t one = e > 0 ? uint32_t(e) << 10 : 0x200u;  // 2^(e - 15)
    return one | one << 16;
}
__device__ __forceinline__ float scale_to_float(uint32_t biased) { return __uint_as_float(uint32_t(min(max(int(biased), kScaleLeast), kScaleMost)) << 23); }
// The power of two that a row of bf16 is divided by on its way to fp16; `most`: the bits of its greatest entry without the sign. (0, infinities and NaN go as they are.)
__device__ __forceinline__ int query_shift(uint32_t most) {
    const int exponent = int(most >> 7) - 127;
    return most == 0 || most >= 0x7f80u || (exponent >= -8 && exponent < 15) ? 0 : min(max(exponent, -120), 120);
}

template <int D, bool BF16, int KIND, int FORM>
__global__ void __launch_bounds__(kFwdThreads, 1)
paged_fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmN, const __grid_constant__ CUtensorMap tmK,
                 const __grid_constant__ CUtensorMap tmV, const PagedParams p) {
    using S = PagedSmem<D, FORM>;
    constexpr bool SCORED = score_changed(KIND), MASKED = (FORM & FORM_MASKED) != 0, E4M3 = S::E4M3, DIRECT = S::DIRECT;
    constexpr bool PBF16 = BF16 && !E4M3;           // the products' type
    constexpr bool BIASED = MASKED && (KIND & SCORE_BIAS) != 0;  // a tile's biases may be far from those before (tile_reference); without a window the keys of a piece lie side by side
    // (spilled registers come back from L2 here: shared memory leaves L1 nothing)
    constexpr int kSoftmaxRegs = DIRECT ? 192 : E4M3 ? 176 : kFwdSoftmaxRegs, kEpilogueRegs = DIRECT ? 64 : E4M3 ? 104 : kFwdEpilogueRegs, kServiceRegs = DIRECT ? 64 : E4M3 ? 56 : kFwdServiceRegs;
    static_assert(256 * kSoftmaxRegs + 128 * (kEpilogueRegs + kServiceRegs) <= kFwdThreads * 128, "registers at launch");
    constexpr float kRaised = E4M3 ? 7.f : 0.f;     // log2 of what P is multiplied by
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
                  B_KEMPTY = B_KFULL + NS, B_VFULL = B_KEMPTY + NS, B_VEMPTY = B_VFULL + NS, B_SFULL = B_VEMPTY + S::NVE,
                  B_SFREE = B_SFULL + 4, B_PFULL = B_SFREE + 2, B_PVDONE = B_PFULL + NP, B_OFULL = B_PVDONE + NP, B_OFREE = B_OFULL + 2;
    static_assert(B_OFREE + 2 == S::n_common, "barriers");
    constexpr int B_RAWK = S::n_common, B_RAWKEMPTY = B_RAWK + S::NBK, B_RAWV = B_RAWKEMPTY + S::NBK, B_RAWVEMPTY = B_RAWV + S::NBV, B_QREADY = B_RAWVEMPTY + S::NBV, B_SUMSFREE = B_QREADY + NQ;
    Abort ab{misc + 1, p.status, p.wait_limit};

    if (tid == 0) {
        for (int s = 0; s < NQ; ++s) {
            mbar_init(BAR(B_ITEMFULL + s), 1);
            mbar_init(BAR(B_ITEMEMPTY + s), DIRECT ? 13 : 15);  // V producer, two MMA issuers (where there are), eight softmax warps, four epilogue warps
            mbar_init(BAR(B_QFULL + s), 1);
            mbar_init(BAR(B_MLFULL + s), 8);
        }
        for (int s = 0; s < NS; ++s) {
            mbar_init(BAR(B_KFULL + s), E4M3 ? 4 : 1);  // (the warps that make the tile)
            mbar_init(BAR(B_KEMPTY + s), 1);
            mbar_init(BAR(B_VFULL + s), E4M3 ? 4 : 1);
        }
        for (int s = 0; s < S::NVE; ++s) mbar_init(BAR(B_VEMPTY + s), 1);
        if constexpr (E4M3) {
            for (int s = 0; s < S::NBK; ++s) {
                mbar_init(BAR(B_RAWK + s), 1);
                mbar_init(BAR(B_RAWKEMPTY + s), 4);
            }
            for (int s = 0; s < S::NBV; ++s) {
                mbar_init(BAR(B_RAWV + s), 1);
                mbar_init(BAR(B_RAWVEMPTY + s), 4);
            }
            for (int s = 0; s < NQ; ++s) mbar_init(BAR(B_QREADY + s), 4);
            mbar_init(BAR(B_SUMSFREE), 4);
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
    for (int i = tid; i < NQ * S::QTILE / 16; i += kFwdThreads) reinterpret_cast<uint4*>(smem + S::off_q)[i] = make_uint4(0, 0, 0, 0);
    fence_proxy_async();
    wait_prerequisites();
    if (!DIRECT && warp == 13) {
        take_tensor_memory(sbase + S::off_misc);
    }
    if (tid == 0) misc[1] = (status_is_fatal(*reinterpret_cast<volatile int*>(p.status)) || (sbase & 1023u) != 0) ? 1 : 0;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    launch_dependents();
    const uint32_t tmem = DIRECT ? 0u : uint32_t(misc[0]);
    const bool aborted = misc[1] != 0;
    uint16_t* const out = static_cast<uint16_t*>(p.out);
    // (aborted: an earlier launch ran into a time-out that the host has not yet cleared. The second kernel fills the output.)
    if (aborted) {
        if (tid == 0) p.merge[blockIdx.x] = make_int4(-1, 0, 0, 0);
    } else if (p.B > kPagedWarpPlan) {
        paged_plan<kFwdThreads, MASKED>(p, plan, int(gridDim.x));
    }
    const int worker = int(blockIdx.x);
    // E4M3: items of so few rows that warps multiply them with what they read of the rings
    auto is_direct = [&](int tokens) { return DIRECT || (E4M3 && tokens * p.G <= kDirectRows); };
    // what a row's scores are multiplied by (a factor must bring it neither to 0 nor beyond fp32: a maximum of minus infinity is multiplied, too)
    auto scale_of = [&](float factor) { return SCORED ? 1.f : E4M3 && BF16 ? fminf(fmaxf(p.scale_log2 * factor, 1.2e-38f), 3e38f) : p.scale_log2; };
    // the key block that is an item's x-th
    auto key_block = [](int x, int border, int skip) { return MASKED && x >= border ? x + skip : x; };

    auto sQ = [&](int s) { return sbase + S::off_q + uint32_t(s) * S::QTILE; };
    auto sK = [&](int s) { return sbase + S::off_k + uint32_t(s) * S::TILE; };
    auto sV = [&](int s) { return sbase + S::off_v + uint32_t(s) * S::TILE; };
    // E4M3: the g-th tile of K or V (the rings' raw_g-th), rows of D numbers in e4m3 to 64-column boxes of fp16 with the swizzle that the products read, by four warps. A thread takes 16
    // numbers at a time. In a loop, and in one place of the code for K and one for V: with the loop unrolled and V's in three places, whose code the softmax groups fetch beside their own, warps
    // stood without an instruction more than anything else. Three chunks of up to 500 and five tokens over 131 MB, 32 / 8 heads of 128: 333 us, capped 466, where 16 bits take 211 and 294: each item
    // converts all its keys for itself, a chunk of 500 tokens with four heads a kv head 16 times.
    auto unpack_tile = [&](auto values, int g, int raw_g, int k0, int seen, int early, int low) {
        constexpr bool V = decltype(values)::value;
        const int r = tid & 127;
        constexpr int R = V ? S::NRV : S::NRK, RB = V ? S::NBV : S::NBK, NE = V ? S::NVE : NS, kThreadsARow = D / 16, kRows = kBlk / kThreadsARow;  // kRows: that the group takes together
        const int raw = raw_g % R, st = g % NS;
        if (!mbar_wait_warp(BAR((V ? B_RAWV : B_RAWK) + raw_g % RB), (raw_g / RB) & 1, ab, ST_WAIT_TIMEOUT + 20)) return false;
        if (g >= NS && !mbar_wait_warp(BAR((V ? B_VEMPTY : B_KEMPTY) + (g - NS) % NE), ((g - NS) / NE) & 1, ab, ST_WAIT_TIMEOUT + 21)) return false;
        const int part = r % kThreadsARow, row0 = r / kThreadsARow;
        const uint8_t* from = smem + (V ? S::off_raw_v : S::off_raw_k) + raw * S::RAW + raw_place<D>(row0, part);  // (the rows that a thread takes have one swizzle)
        const uint8_t* scales = smem + (V ? S::off_scale_v : S::off_scale_k) + raw * kBlk + row0;
        uint8_t* to = smem + (V ? S::off_v : S::off_k) + st * S::TILE + (part >> 2) * S::BOX + row0 * 128;
        const int c0 = ((2 * (part & 3)) ^ (row0 & 7)) << 4, c1 = c0 ^ 16;
        static_assert(kRows % 8 == 0, "one swizzle");
        const bool all = k0 + kBlk <= seen && (k0 + kBlk <= early || k0 >= low);
        int key = k0 + row0;
#pragma unroll 1
        for (int i = 0; i < kBlk / (2 * kRows); ++i) {
            uint4 x[2];
            uint32_t scale[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                x[j] = *reinterpret_cast<const uint4*>(from + j * kRows * D);
                scale[j] = scales[j * kRows];
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const uint32_t two = scale_to_h2(scale[j]);
                uint32_t y[8];
                unpack_e4m3x4(x[j].x, y[0], y[1]);
                unpack_e4m3x4(x[j].y, y[2], y[3]);
                unpack_e4m3x4(x[j].z, y[4], y[5]);
                unpack_e4m3x4(x[j].w, y[6], y[7]);
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] = mul_h2(y[e], two);
                if (!all) {
                    const int at = key + j * kRows;
                    const uint32_t real = at < seen && (at < early || at >= low) ? ~0u : 0u;
#pragma unroll
                    for (int e = 0; e < 8; ++e) y[e] &= real;
                }
                *reinterpret_cast<uint4*>(to + j * kRows * 128 + c0) = make_uint4(y[0], y[1], y[2], y[3]);
                *reinterpret_cast<uint4*>(to + j * kRows * 128 + c1) = make_uint4(y[4], y[5], y[6], y[7]);
            }
            from += 2 * kRows * D;
            scales += 2 * kRows;
            to += 2 * kRows * 128;
            key += 2 * kRows;
        }
        mbar_arrive_warp(BAR((V ? B_RAWVEMPTY : B_RAWKEMPTY) + raw_g % RB), lane);
        fence_proxy_async();
        mbar_arrive_warp(BAR((V ? B_VFULL : B_KFULL) + st), lane);
        return true;
    };
    if (warp >= 12) {
        setmaxnreg_dec<kServiceRegs>();
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
        // E4M3: rows of D bytes, and a byte for each
        auto load_raw = [&](const CUtensorMap* m, uint32_t dst, const uint8_t* scales, int64_t scale_p, uint32_t dst_scale, uint32_t bar, int pages, int tile, int hk, int len) {
            const int left = len - (tile << 7), n = left >= kBlk ? boxes : (left + rows - 1) >> log2_rows;
            mbar_expect_tx_elect(bar, (uint32_t(n) << log2_rows) * uint32_t(D + 1));
            const int row = (tile << 7) & (p.page - 1) & ~(rows - 1);
#pragma unroll 1
            for (int i = 0; i < n; ++i) {
                const uint32_t page = uint32_t(__shfl_sync(0xffffffffu, pages, i));
                tma_load_4d_elect(dst, m, bar, 0, hk, row, int(min(page, uint32_t(p.n_pages))));
                bulk_load_1d_elect(dst_scale, scales + min(page, uint32_t(p.n_pages - 1)) * scale_p + row, uint32_t(rows), bar);
                dst += uint32_t(rows) * D;
                dst_scale += uint32_t(rows);
            }
        };
        if (aborted) {
        } else if (warp == 14) {
            // ------------------------------ item scheduler, and loads of Q and K ------------------------------
            tma_prefetch_desc(&tmQ);
            tma_prefetch_desc(&tmN);
            tma_prefetch_desc(&tmK);
            bool ok = true, first = true;
            int k = 0, gk = 0;
            int4 merge = make_int4(0, 0, 0, 0);
            if (p.B <= kPagedWarpPlan) paged_plan_warp<MASKED>(p, plan, int(gridDim.x));
            if (worker < plan.workers) {
                paged_stretch<MASKED>(p, plan, worker, [&](const PagedWalk<MASKED>& walk, int, int lo, int hi, int part) {
                    const int s = k % NQ, use = k / NQ;
                    const int T = uniform(hi - lo), tile0 = uniform(lo), hk = uniform(walk.hk), len = uniform(walk.s.len), tok0 = uniform(walk.s.start + walk.tile * p.tokens);
                    const int tokens = uniform(min(p.tokens, walk.s.n - walk.tile * p.tokens));
                    const int32_t* const row_of_table = p.table + walk.b * p.table_stride;
                    const int border = MASKED ? uniform(cdiv(walk.s.early, kBlk)) : 0, skip = MASKED ? uniform(paged_skip(p, walk.s, walk.tile)) : 0;
                    int pages = T > 0 ? pages_of(row_of_table, key_block(tile0, border, skip), len) : 0;
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
                        if constexpr (MASKED) {
                            it[I_BORDER] = border;
                            it[I_SKIP] = skip;
                            it[I_BASE] = walk.s.tree ? walk.s.base : len;
                            it[I_FIRST] = walk.s.start;
                        }
                        mbar_arrive(BAR(B_ITEMFULL + s));
                    }
                    __syncwarp();
                    // (an item's slot is given away when its O has left, so that Q has been read, too)
                    if (is_direct(tokens)) {
                        mbar_expect_tx_elect(BAR(B_QFULL + s), uint32_t(p.narrow * p.G) * 128u * S::NBOX);
                        for (int x = 0; x < S::NBOX; ++x) tma_load_4d_elect(sQ(s) + x * S::QBOX, &tmN, BAR(B_QFULL + s), x * 64, 0, hk, tok0);
                    } else if (tokens <= p.narrow) {  // four times the same rows
                        mbar_expect_tx_elect(BAR(B_QFULL + s), uint32_t(p.narrow * p.G) * 512u * S::NBOX);
                        for (int i = 0; i < 4 * S::NBOX; ++i)
                            tma_load_4d_elect(sQ(s) + (i >> 2) * S::BOX + (i & 3) * 4096, &tmN, BAR(B_QFULL + s), (i >> 2) * 64, 0, hk, tok0);
                    } else {
                        mbar_expect_tx_elect(BAR(B_QFULL + s), uint32_t(p.tokens * p.G) * 128u * S::NBOX);
                        for (int x = 0; x < S::NBOX; ++x) tma_load_4d_elect(sQ(s) + x * S::BOX, &tmQ, BAR(B_QFULL + s), x * 64, 0, hk, tok0);
                    }
                    for (int t = 0; t < T; ++t, ++gk) {
                        constexpr int R = E4M3 ? S::NRK : NS, RB = E4M3 ? S::NBK : NS;
                        const int st = gk % R, own = pages;
                        if (t + 1 < T) pages = pages_of(row_of_table, key_block(tile0 + t + 1, border, skip), len);
                        if (gk >= R) ok = mbar_wait_warp(BAR((E4M3 ? B_RAWKEMPTY : B_KEMPTY) + (gk - R) % RB), ((gk - R) / RB) & 1, ab, ST_WAIT_TIMEOUT + 1);
                        if (!ok) return false;
                        if constexpr (E4M3)
                            load_raw(&tmK, sbase + S::off_raw_k + uint32_t(st) * S::RAW, p.k_scales + hk * p.k_scale_h, p.k_scale_p, sbase + S::off_scale_k + uint32_t(st) * kBlk,
                                     BAR(B_RAWK + gk % RB), own, key_block(tile0 + t, border, skip), hk, len);
                        else
                            load(&tmK, sK(st), BAR(B_KFULL + st), own, key_block(tile0 + t, border, skip), hk, len);
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
                const int border = MASKED ? uniform(it[I_BORDER]) : 0, skip = MASKED ? uniform(it[I_SKIP]) : 0;
                const int32_t* const row_of_table = p.table + seq * p.table_stride;
                int pages = T > 0 ? pages_of(row_of_table, key_block(lo, border, skip), len) : 0;
                for (int t = 0; t < T; ++t, ++gv) {
                    constexpr int R = E4M3 ? S::NRV : NS, RB = E4M3 ? S::NBV : NS;
                    const int st = gv % R, own = pages;
                    if (t + 1 < T) pages = pages_of(row_of_table, key_block(lo + t + 1, border, skip), len);
                    if (gv >= R) ok = mbar_wait_warp(BAR((E4M3 ? B_RAWVEMPTY : B_VEMPTY) + (gv - R) % RB), ((gv - R) / RB) & 1, ab, ST_WAIT_TIMEOUT + 2);
                    if (!ok) break;
                    if constexpr (E4M3)
                        load_raw(&tmV, sbase + S::off_raw_v + uint32_t(st) * S::RAW, p.v_scales + hk * p.v_scale_h, p.v_scale_p, sbase + S::off_scale_v + uint32_t(st) * kBlk,
                                 BAR(B_RAWV + gv % RB), own, key_block(lo + t, border, skip), hk, len);
                    else
                        load(&tmV, sV(st), BAR(B_VFULL + st), own, key_block(lo + t, border, skip), hk, len);
                }
                if (!ok) break;
                __syncwarp();
                if (lane == 0) mbar_arrive(BAR(B_ITEMEMPTY + s));
                __syncwarp();
            }
        } else if constexpr (!DIRECT) {
            // ------------------------------ MMA issuers ------------------------------
            //   warp 13: P*V(g) when P(g) is there; warp 15: S(g) when its buffer is free
            const uint32_t utmem = uniform(int(tmem));
            constexpr uint32_t idesc_s = make_idesc(PBF16, 128, 128, false, false);
            constexpr uint32_t idesc_pv = make_idesc(PBF16, 128, D, false, true);
            constexpr uint64_t desc_v = desc_mn_major(S::BOX);
            bool ok = true;
            int G = 0;           // tiles of all earlier items
            int n0 = 0, n1 = 0;  // items in which the chains had tiles
            for (int k = 0;; ++k) {
                const int s = k % NQ, use = k / NQ;
                ok = mbar_wait_warp(BAR(B_ITEMFULL + s), use & 1, ab, ST_WAIT_TIMEOUT + 12);
                if (!ok) break;
                const int T = is_direct(uniform(info[16 * s + I_TOKENS])) ? 0 : uniform(info[16 * s + I_TILES]);
                if (uniform(info[16 * s + I_MORE]) < 0) break;
                if (warp == 15) {
                    if (T > 0) ok = mbar_wait_warp(BAR((E4M3 && BF16 ? B_QREADY : B_QFULL) + s), use & 1, ab, ST_WAIT_TIMEOUT + 3);
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
                        umma_commit(BAR(B_VEMPTY + g % S::NVE));
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
        setmaxnreg_dec<kEpilogueRegs>();
        const int r = tid & 127;
        const uint32_t lane_base = uint32_t((warp & 3) * 32) << 16;
        const int tok_wide = r / p.G, tok_narrow = lane / p.G;
        // E4M3 of bf16: this thread's row of Q to fp16 in place, times a power of two where its greatest entry is beyond fp16 or so small that the others would lose bits; what the
        // row's scores are to be multiplied by.
        auto query_to_fp16 = [&](int s) {
            uint8_t* const row = smem + S::off_q + s * S::QTILE + r * 128;
            auto at = [&](int i) { return reinterpret_cast<uint4*>(row + (i >> 3) * S::BOX + (((i + r) & 7) << 4)); };  // (any order will do: eight lanes at eight places)
            uint32_t most = 0;  // bf16 numbers without their sign go by size
#pragma unroll 4
            for (int i = 0; i < D / 8; ++i) {
                const uint4 x = *at(i);
                const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) most = max(most, max(w[j] & 0x7fffu, w[j] >> 16 & 0x7fffu));
            }
            const int shift = query_shift(most);
            const float back = __uint_as_float(uint32_t(127 + shift) << 23), there = __uint_as_float(uint32_t(127 - shift) << 23);
#pragma unroll 4
            for (int i = 0; i < D / 8; ++i) {
                uint4* const x = at(i);
                const uint4 v = *x;
                auto two = [&](uint32_t y) { return pack2<false>(__uint_as_float(y << 16) * there, __uint_as_float(y & 0xffff0000u) * there); };
                *x = make_uint4(two(v.x), two(v.y), two(v.z), two(v.w));
            }
            return back;
        };
        // E4M3: the output of an item that eight warps have multiplied directly, or a piece of it. Each has left its maximum and sum of the rows in `ml` and its O, [16 rows][D] in fp32; this
        // thread has D / 8 neighbouring columns of one row.
        auto sum_warps = [&](int s, int T, int part, int row0, int hk, int tokens) {
            constexpr int kTiles = D / 8;
            const int row = 2 * (r >> 1 & 3) + (r >> 5 & 1) + 8 * (r >> 6), n = 2 * (r >> 3 & 3) + (r & 1), tok = row / p.G;
            if (row >= tokens * p.G || misc[1] != 0) return;
            const float* const ml = reinterpret_cast<const float*>(smem + S::off_ml) + s * (4 * kBlk) + row;
            auto at = [](int q) { return (q >> 2) * (2 * kBlk) + (q & 3) * 32; };
            float mt = -INFINITY, lt = 0.f, acc[kTiles] = {};
#pragma unroll
            for (int q = 0; q < 8; ++q) mt = fmaxf(mt, ml[at(q)]);
#pragma unroll 1
            for (int q = 0; q < 8; ++q) {
                const float m = ml[at(q)], a = m == -INFINITY ? 0.f : fast_exp2(m - mt);
                lt += ml[at(q) + kBlk] * (m == -INFINITY ? 1.f : a);  // (a NaN that a row without a maximum has is not lost)
                if (a == 0.f) continue;
                const float4* const o = reinterpret_cast<const float4*>(smem + S::off_sums) + (q * kDirectRows + row) * (D / 4);
#pragma unroll
                for (int j = 0; j < kTiles; j += 4) {
                    const float4 x = o[sums_place<D>(row, (n * kTiles + j) / 4)];
                    acc[j] = fmaf(a, x.x, acc[j]);
                    acc[j + 1] = fmaf(a, x.y, acc[j + 1]);
                    acc[j + 2] = fmaf(a, x.z, acc[j + 2]);
                    acc[j + 3] = fmaf(a, x.w, acc[j + 3]);
                }
            }
            const float inv = lt > 0.f ? 1.0f / lt : lt == lt ? 0.f : lt;
            if (part >= 0) {
                if (n == 0) p.part_lse[int64_t(part) * kBlk + row] = lt > 0.f ? mt + log2f(lt) : lt == lt ? -INFINITY : lt;
                float4* const to = reinterpret_cast<float4*>(p.part_o + (int64_t(part) * kBlk + row) * D + n * kTiles);
#pragma unroll
                for (int j = 0; j < kTiles; j += 4) to[j / 4] = make_float4(acc[j] * inv, acc[j + 1] * inv, acc[j + 2] * inv, acc[j + 3] * inv);
            } else if (n * kTiles < p.D) {
                uint4* const to = reinterpret_cast<uint4*>(out + int64_t(row0 + tok) * p.out_t + int64_t(hk * p.G + row - tok * p.G) * p.out_h + n * kTiles);
#pragma unroll
                for (int j = 0; j < kTiles; j += 8)
                    to[j / 8] = make_uint4(pack2<BF16>(acc[j] * inv, acc[j + 1] * inv), pack2<BF16>(acc[j + 2] * inv, acc[j + 3] * inv),
                                           pack2<BF16>(acc[j + 4] * inv, acc[j + 5] * inv), pack2<BF16>(acc[j + 6] * inv, acc[j + 7] * inv));
            }
        };
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
        int raw_g = 0;       // E4M3: tiles of all earlier items, those counted that are multiplied directly
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
                auto check_pages = [&](int from, int end) {  // of the keys in between
                    for (int i = (from >> p.log2_page) + r; i <= (end - 1) >> p.log2_page && end > from; i += kBlk)
                        if (uint32_t(p.table[row_of_table + i]) >= uint32_t(p.n_pages)) atomicCAS(p.status, 0, ST_PAGED_PAGE);
                };
                if constexpr (MASKED) {
                    // (a window's server may have given the pages behind it away: nothing is asked of their entries)
                    const int lo = it[I_LO], border = it[I_BORDER], skip = it[I_SKIP], len = it[I_LEN], tree = it[I_BASE] < len;
                    const int early = p.window > 0 ? max(it[I_FRONT], p.sinks) : len, low = p.window > 0 ? (tree ? it[I_BASE] : it[I_POS]) - p.window + 1 : 0;
                    const int from = key_block(lo, border, skip) * kBlk, end = T > 0 ? min((key_block(lo + T - 1, border, skip) + 1) * kBlk, len) : 0;
                    check_pages(from, min(end, early));
                    if (p.window > 0) check_pages(max(from, low), end);
                } else {
                    if (T > 0) check_pages(it[I_LO] * kBlk, min((it[I_LO] + T) * kBlk, it[I_LEN]));
                }
            }
            float factor = 1.f;  // E4M3 of bf16: of this row's scores
            if constexpr (E4M3) {
                if (is_direct(tokens)) {
                    // the products are none of this group's: it adds up what the eight warps have (sum_warps)
                    if constexpr (BF16) mbar_arrive_warp(BAR(B_QREADY + s), lane);
                    mbar_arrive_warp(BAR(B_SUMSFREE), lane);  // (what K's and V's tiles are made in serves for that, and this group is done with the item before)
                    const Abort item{ab.flag, ab.status, ab.limit * (T + 1)};
                    alive = mbar_wait_warp(BAR(B_MLFULL + s), use & 1, item, ST_WAIT_TIMEOUT + 16);
                    if (!alive) break;
                    sum_warps(s, T, part, it[I_ROW], hk, tokens);
                    raw_g += T;
                    // (all of the group before any of it may make a tile there)
                    mbar_arrive_warp(BAR(B_STAGED), lane);
                    alive = mbar_wait_warp(BAR(B_STAGED), staged++ & 1, ab, ST_WAIT_TIMEOUT + 18);
                    if (!alive) break;
                    if (lane == 0) mbar_arrive(BAR(B_ITEMEMPTY + s));
                    continue;
                }
                if constexpr (BF16) {
                    // (not of an item without tiles: there no product waits until all four warps have done so, and the first of them would stage its zeros where the others' rows of Q are)
                    if (T > 0) {
                        alive = mbar_wait_warp(BAR(B_QFULL + s), use & 1, ab, ST_WAIT_TIMEOUT + 17);
                        if (!alive) break;
                        factor = fminf(query_to_fp16(s) * p.lift, 3e38f);
                        reinterpret_cast<float*>(smem + S::off_factor)[s * kBlk + r] = factor;
                        fence_proxy_async();
                    }
                    mbar_arrive_warp(BAR(B_QREADY + s), lane);
                }
                const int pos0 = it[I_POS], len = it[I_LEN], front = it[I_FRONT], lo = it[I_LO], border = it[I_BORDER], skip = it[I_SKIP];
                const int seen = min(max(pos0 + tokens, front), len), early = p.window > 0 ? max(front, p.sinks) : len;
                const int low = p.window > 0 ? (it[I_BASE] < len ? it[I_BASE] : pos0) - p.window + 1 : 0;
                for (int t = 0; t < T && alive; ++t) alive = unpack_tile(std::false_type{}, G + t, raw_g + t, key_block(lo + t, border, skip) * kBlk, seen, early, low);
                raw_g += T;
                if (!alive) break;
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
            const float c = scale_of(factor);
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
            float* const stage = reinterpret_cast<float*>(smem + S::off_q + s * S::QTILE);  // (Q has been read) [2][4 warps][32 rows][16]
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
        setmaxnreg_inc<kSoftmaxRegs>();
        // ------------------------------ softmax groups ------------------------------
        const int w = warp >> 2;  // group
        const int r = tid & 127;  // row inside the tile
        const uint32_t lane_base = uint32_t((warp & 3) * 32) << 16;
        const uint32_t tO = tmem + lane_base + uint32_t(S::tmem_o + w * D);
        const int tok_wide = r / p.G, tok_narrow = lane / p.G;
        bool alive = !aborted;
        // Rows of V behind the keys that the item sees hold what was in the page, or in the stage: zeros, before P*V(g) is issued. A quarter of them a warp. (MASKED: and the
        // rows from `from` to `end`, between the early keys and the window.)
        auto zero_behind = [&](int g, int real, int from, int end) {
            const int st = g % NS;
            if (!mbar_wait_warp(BAR(B_VFULL + st), (g / NS) & 1, ab, ST_WAIT_TIMEOUT + 19)) return false;
            // (not unrolled: it stands twice in the code of the softmax warps, a batch of chunks and tokens with a bias 224 us for 237)
#pragma unroll 1
            for (int x = 0; x < S::NBOX; ++x)
#pragma unroll 1
                for (int i = real * 8 + r; i < kBlk * 8; i += kBlk) reinterpret_cast<uint4*>(smem + S::off_v + st * S::TILE + x * S::BOX)[i] = make_uint4(0, 0, 0, 0);
            if constexpr (MASKED) {
#pragma unroll 1
                for (int x = 0; x < S::NBOX; ++x)
#pragma unroll 1
                    for (int i = from * 8 + r; i < end * 8; i += kBlk) reinterpret_cast<uint4*>(smem + S::off_v + st * S::TILE + x * S::BOX)[i] = make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async();
            return true;
        };
        // Which of the 32 keys from x0 on a row sees.
        auto keys_seen = [&](int x0, int last, int low, int early, int base, bool tree, const uint32_t* masks) {
            uint32_t keep = first_bits(last - x0 + 1);
            if constexpr (MASKED) {
                if (p.window > 0) keep &= ~hidden_bits(low - x0, early - x0);
                if (tree && x0 + 31 >= base) {
                    const int i = x0 - base, word = i >> 5;  // (below 0 where the cached text ends among the 32)
                    const uint32_t lo_bits = word >= 0 && word < S::kMaskWords ? masks[word * kBlk] : 0u;
                    const uint32_t hi_bits = word + 1 >= 0 && word + 1 < S::kMaskWords ? masks[(word + 1) * kBlk] : 0u;
                    const uint32_t text = first_bits(base - x0);
                    keep = (keep & text) | (__funnelshift_r(lo_bits, hi_bits, i) & ~text);
                }
            }
            return keep;
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
        int G = 0;      // tiles of all earlier items
        int raw_g = 0;  // E4M3: those counted that are multiplied directly
        int direct = 0; // E4M3: items of that kind
        bool was_direct = false;  // the item before
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
            int all_see = pos0 < 0 ? -1 : min(max(pos0, front - 1), len - 1);  // and that all rows of the tile see
            const int seen = min(max(pos0 + tokens, front), len);              // keys that any row sees
            // MASKED: keys below `low` are not in the row's window (below low_first in none's, low_last in some row's) and hidden but for the first `early`; of those
            // from `base` on, a tree's, the row sees those that its mask says
            const int border = MASKED ? it[I_BORDER] : 0, skip = MASKED ? it[I_SKIP] : 0, base = MASKED ? it[I_BASE] : 0;
            int low = 0, low_first = 0, low_last = 0, early = 0;
            bool tree = false;
            uint32_t* const masks = reinterpret_cast<uint32_t*>(smem + S::off_masks) + w * (S::kMaskWords * kBlk) + r;
            if constexpr (MASKED) {
                tree = base < len;
                int depth = 0;  // of the row's token in its tree, or its place behind the tile's first token
                if (tree) {
                    all_see = min(all_see, base - 1);
#pragma unroll
                    for (int i = 0; i < S::kMaskWords; ++i) masks[i * kBlk] = 0u;
                    if (valid && pos >= 0) {
                        const int32_t* const parents = p.parents + it[I_FIRST];
                        const int own = it[I_ROW] - it[I_FIRST] + tok;
                        auto parent = [&](int a) {  // one that does not lie before its token would be no tree's: the token continues the cached text
                            const int x = parents[a];
                            return x < a ? max(x, -1) : -1;
                        };
                        if (parents[own] < -1 || parents[own] >= own) atomicCAS(p.status, 0, ST_PAGED_PARENT);
                        if (p.window > 0) {
#pragma unroll 1
                            for (int a = own; (a = parent(a)) >= 0;) ++depth;
                        }
                        int up = 0;  // steps above the token
#pragma unroll 1
                        for (int a = own; a >= 0; a = parent(a), ++up)
                            if (p.window == 0 || up < p.window || base + depth - up < p.sinks) masks[(a >> 5) * kBlk] |= 1u << (a & 31);
                    }
                } else {
                    depth = tok;
                }
                if (p.window > 0) {
                    early = max(front, p.sinks);
                    low_first = (tree ? base : pos0) - p.window + 1;
                    low = low_first + depth;
                    low_last = pos0 + tokens - p.window;
                }
            }
            auto sees = [&](int x0) { return keys_seen(x0, last, low, early, base, tree, masks); };
            float slope = 0.f;
            if constexpr (SCORED) {
                if (p.score.slopes) slope = p.score.slopes[int64_t(it[I_HEAD]) * p.G + g_row] * kScoreLog2e;
            }
            if constexpr (E4M3 && !DIRECT) {
                // Which group has a ring's even tiles can change with the kind of the items: all of the tiles before have to be done with.
                if (k > 0 && is_direct(tokens) != was_direct) alive = mbar_wait_warp(BAR(B_MLFULL + (k - 1) % NQ), ((k - 1) / NQ) & 1, ab, ST_WAIT_TIMEOUT + 23);
                if (!alive) break;
                was_direct = is_direct(tokens);
            }
            const int item_raw = raw_g;
            raw_g += T;
            // E4M3: V's tile of a group's own tile of keys
            auto unpack_values = [&](int t) {
                if constexpr (E4M3 && !DIRECT)
                    return unpack_tile(std::true_type{}, G + t, item_raw + t, key_block(lo + t, border, skip) * kBlk, seen, p.window > 0 ? early : len, low_first);
                return true;
            };
            if constexpr (E4M3) {
                if (is_direct(tokens)) {
                    // ------------------------------ few rows: by warps, from the rings ------------------------------
                    // A tile belongs to one group, and each of its four warps has 32 of the keys, with a maximum, sums and an O of its own. mma.sync, with what there is much of as M: S^T = K Q^T, 16
                    // keys by 8 rows, and O^T = V^T P^T, 16 columns by 8 rows. What a thread multiplies in a step along the head dim, and which columns of V its tiles have, is a matter of order
                    // alone, so that it takes neighbouring bytes: of K's rows 4 a step, of V's the D / 8 of each of its keys. K's scales go to the scores, V's to the numbers, which fp16 holds exactly.
                    // A warp has a tile's bytes in registers before it begins, and has given the rings' places back; nothing else waits. Clocks a tile of 128 keys of 128: HBM's share of an SM 1400,
                    // conversions 450 of the ALU, products 256. 64 tokens, 32 / 8 heads of 128, over 650 MB, us: by the tensor memory's way 345; rows as M, 16 keys a warp of every tile 187; rows as
                    // N 154; 32 keys of every other tile 150; rings of 128 KB, and no spilled registers, 136.
                    alive = mbar_wait_warp(BAR(B_QFULL + s), use & 1, ab, ST_WAIT_TIMEOUT + 3);
                    if (!alive) break;
                    __syncwarp();  // (a row's mask is its lane's)
                    const int row0 = valid ? last : -1;
                    auto multiply = [&](auto tiles) {
                        constexpr int NT = decltype(tiles)::value;          // of 8 rows
                        constexpr int U = NT == 1 ? 2 : 1;                  // times 16 keys at once (the registers do not do for two of both)
                        constexpr int kSteps = D / 16, kCols = D / 16;      // along the head dim for S^T; of 16 columns of O
                        const int g8 = lane >> 2, c4 = lane & 3, own_keys = 32 * (warp & 3);  // own_keys: the first of the warp's in a tile
                        uint32_t qb[NT][kSteps][2];
                        float scale[NT][2], back[NT][2];  // of the scores of rows 8 n + 2 c4, + 1: to the log2 domain, and to what they are
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            float most = 0.f, own = 1.f;
                            const int row = g8 + 8 * n;
#pragma unroll
                            for (int i = 0; i < kSteps; ++i) {
                                const int d0 = c4 * (D / 4) + 4 * i;
                                const uint2 x = *reinterpret_cast<const uint2*>(smem + S::off_q + s * S::QTILE + (d0 >> 6) * S::QBOX + row * 128 + ((((d0 & 63) >> 3) ^ (row & 7)) << 4) + (d0 & 7) * 2);
                                qb[n][i][0] = x.x;
                                qb[n][i][1] = x.y;
                                if constexpr (BF16) {
#pragma unroll
                                    for (int e = 0; e < 2; ++e)
                                        most = fmaxf(most, fmaxf(fabsf(__uint_as_float(qb[n][i][e] << 16)), fabsf(__uint_as_float(qb[n][i][e] & 0xffff0000u))));
                                }
                            }
                            if constexpr (BF16) {
                                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
                                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
                                const int shift = query_shift(__float_as_uint(most) >> 16);
                                const float there = __uint_as_float(uint32_t(127 - shift) << 23);
                                own = fminf(__uint_as_float(uint32_t(127 + shift) << 23) * p.lift, 3e38f);
#pragma unroll
                                for (int i = 0; i < kSteps; ++i) {
#pragma unroll
                                    for (int e = 0; e < 2; ++e)
                                        qb[n][i][e] = pack2<false>(__uint_as_float(qb[n][i][e] << 16) * there, __uint_as_float(qb[n][i][e] & 0xffff0000u) * there);
                                }
                            }
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                back[n][e] = __shfl_sync(0xffffffffu, own, 4 * (2 * c4 + e));
                                scale[n][e] = scale_of(back[n][e]);
                            }
                        }
                        // (what an item's rows are lies one a lane)
                        int row_pos[NT][2];
                        float row_slope[NT][2];
                        if constexpr ((KIND & SCORE_BIAS) != 0) {
#pragma unroll
                            for (int n = 0; n < NT; ++n) {
#pragma unroll
                                for (int e = 0; e < 2; ++e) {
                                    row_pos[n][e] = __shfl_sync(0xffffffffu, pos, 8 * n + 2 * c4 + e);
                                    row_slope[n][e] = __shfl_sync(0xffffffffu, slope, 8 * n + 2 * c4 + e);
                                }
                            }
                        }
                        const uint32_t* const warp_masks = reinterpret_cast<const uint32_t*>(smem + S::off_masks) + w * (S::kMaskWords * kBlk) + (warp & 3) * 32;
                        float o[kCols][NT][4] = {}, m[NT][2], l[NT][2];
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            m[n][0] = m[n][1] = -INFINITY;
                            l[n][0] = l[n][1] = 0.f;
                        }
#pragma unroll 1
                        for (int step = ((item_raw ^ w) & 1) * (2 / U); step < T * (2 / U); step += U == 2 || (step & 1) ? 1 + 2 / U : 1) {
                            const int t = step / (2 / U), half = U == 2 ? 0 : step & 1, mine = own_keys + 16 * half;
                            const int k0 = key_block(lo + t, border, skip) * kBlk + mine, gr = item_raw + t;
                            const int rk = gr % S::NRK, rv = gr % S::NRV;
                            const bool give_back = U == 2 || half == 1;
                            // does some row not see all of these keys?
                            const bool masked = k0 + 16 * U - 1 > all_see || (p.window > 0 && k0 < low_last && k0 + 16 * U > early);
                            uint4 xk[U][2][D / 64];  // keys 16 u + 8 j + g8
                            float k_scale[U][2];
                            uint32_t xv[U][4][D / 32], v_scale[U][2];  // keys 16 u + 2 c4, + 1, + 8, + 9; columns from g8 * D / 8 on
                            auto take_values = [&] {
                                if (!mbar_wait_warp(BAR(B_RAWV + gr % S::NBV), (gr / S::NBV) & 1, ab, ST_WAIT_TIMEOUT + 20)) return false;
                                const uint8_t* const from = smem + S::off_raw_v + rv * S::RAW;
#pragma unroll
                                for (int u = 0; u < U; ++u) {
#pragma unroll
                                    for (int i = 0; i < 4; ++i) {
                                        const int row = mine + 16 * u + 2 * c4 + (i & 1) + 8 * (i >> 1);
                                        if constexpr (D == 128) {
                                            const uint4 y = *reinterpret_cast<const uint4*>(from + raw_place<D>(row, g8));
                                            xv[u][i][0] = y.x; xv[u][i][1] = y.y; xv[u][i][2] = y.z; xv[u][i][3] = y.w;
                                        } else {
                                            const uint2 y = *reinterpret_cast<const uint2*>(from + raw_place<D>(row, g8 >> 1) + (g8 & 1) * 8);
                                            xv[u][i][0] = y.x; xv[u][i][1] = y.y;
                                        }
                                    }
#pragma unroll
                                    for (int i = 0; i < 2; ++i) v_scale[u][i] = *reinterpret_cast<const uint16_t*>(smem + S::off_scale_v + rv * kBlk + mine + 16 * u + 2 * c4 + 8 * i);
                                }
                                if (give_back) mbar_arrive_warp(BAR(B_RAWVEMPTY + gr % S::NBV), lane);
                                return true;
                            };
                            if (!mbar_wait_warp(BAR(B_RAWK + gr % S::NBK), (gr / S::NBK) & 1, ab, ST_WAIT_TIMEOUT + 20)) return false;
                            {
                                const uint8_t* const from = smem + S::off_raw_k + rk * S::RAW;
#pragma unroll
                                for (int u = 0; u < U; ++u) {
#pragma unroll
                                    for (int j = 0; j < 2; ++j) {
#pragma unroll
                                        for (int i = 0; i < D / 64; ++i)
                                            xk[u][j][i] = *reinterpret_cast<const uint4*>(from + raw_place<D>(mine + 16 * u + 8 * j + g8, c4 * (D / 64) + i));
                                        k_scale[u][j] = scale_to_float(smem[S::off_scale_k + rk * kBlk + mine + 16 * u + 8 * j + g8]);
                                    }
                                }
                                if (give_back) mbar_arrive_warp(BAR(B_RAWKEMPTY + gr % S::NBK), lane);
                            }
                            if (NT == 1 && !take_values()) return false;
                            float sc[NT][U][4] = {};
#pragma unroll
                            for (int i = 0; i < kSteps; ++i) {
                                auto word = [&](const uint4& y) { return (i & 3) == 0 ? y.x : (i & 3) == 1 ? y.y : (i & 3) == 2 ? y.z : y.w; };
#pragma unroll
                                for (int u = 0; u < U; ++u) {
                                    uint32_t ka[4];
                                    unpack_e4m3x4(word(xk[u][0][i >> 2]), ka[0], ka[2]);
                                    unpack_e4m3x4(word(xk[u][1][i >> 2]), ka[1], ka[3]);
#pragma unroll
                                    for (int n = 0; n < NT; ++n) mma_16816(sc[n][u], ka, qb[n][i][0], qb[n][i][1]);
                                }
                            }
                            uint32_t pb[NT][U][2];
#pragma unroll
                            for (int n = 0; n < NT; ++n) {
                                float y[U][4];  // keys 16 u + g8, + 8 by rows 2 c4, 2 c4 + 1, in the log2 domain
#pragma unroll
                                for (int u = 0; u < U; ++u) {
#pragma unroll
                                    for (int j = 0; j < 2; ++j) {
                                        const float* const f = SCORED ? back[n] : scale[n];
                                        uint64_t y2 = mul_f2(pack_f2(sc[n][u][2 * j], sc[n][u][2 * j + 1]), pack_f2(k_scale[u][j] * f[0], k_scale[u][j] * f[1]));
                                        if constexpr (SCORED) {
                                            uint64_t b2 = 0;
                                            if constexpr ((KIND & SCORE_BIAS) != 0) {
                                                const int key = k0 + 16 * u + 8 * j + g8;
                                                b2 = pack_f2(-row_slope[n][0] * fabsf(float(row_pos[n][0] - key)), -row_slope[n][1] * fabsf(float(row_pos[n][1] - key)));
                                            }
                                            if constexpr ((KIND & SCORE_CAPPED) != 0) y2 = cap_any(y2, b2, p.score);
                                            else y2 = fma_f2(y2, pack_f2(p.scale_log2, p.scale_log2), b2);
                                        }
                                        unpack_f2(y2, y[u][2 * j], y[u][2 * j + 1]);
                                    }
                                }
                                if (masked) {
#pragma unroll
                                    for (int e = 0; e < 2; ++e) {
                                        const int row = 8 * n + 2 * c4 + e;
                                        const uint32_t keep = keys_seen(k0, __shfl_sync(0xffffffffu, row0, row), __shfl_sync(0xffffffffu, low, row), early, base, tree, warp_masks + row) >> g8;
#pragma unroll
                                        for (int u = 0; u < U; ++u) {
                                            y[u][e] = (keep >> (16 * u) & 1u) ? y[u][e] : -INFINITY;
                                            y[u][2 + e] = (keep >> (16 * u) & 256u) ? y[u][2 + e] : -INFINITY;
                                        }
                                    }
                                }
                                float top[2];
#pragma unroll
                                for (int e = 0; e < 2; ++e) {
                                    top[e] = fmaxf(y[0][e], y[0][2 + e]);
                                    if constexpr (U == 2) top[e] = fmaxf(top[e], fmaxf(y[U - 1][e], y[U - 1][2 + e]));
                                    top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 4));
                                    top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 8));
                                    top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 16));
                                }
                                // lazy: the old reference point stays while the new maximum is within 2^8 of it
                                const bool need0 = top[0] - m[n][0] > 8.f, need1 = top[1] - m[n][1] > 8.f;
                                if (__any_sync(0xffffffffu, need0 || need1)) {
                                    const float a0 = need0 ? fast_exp2(m[n][0] - top[0]) : 1.f, a1 = need1 ? fast_exp2(m[n][1] - top[1]) : 1.f;
                                    if (need0) m[n][0] = top[0];
                                    if (need1) m[n][1] = top[1];
                                    l[n][0] *= a0;
                                    l[n][1] *= a1;
#pragma unroll
                                    for (int i = 0; i < kCols; ++i) {
                                        o[i][n][0] *= a0;
                                        o[i][n][1] *= a1;
                                        o[i][n][2] *= a0;
                                        o[i][n][3] *= a1;
                                    }
                                }
#pragma unroll
                                for (int e = 0; e < 2; ++e) {
                                    const float ref = (m[n][e] == -INFINITY ? 0.f : m[n][e]) - kRaised;
#pragma unroll
                                    for (int u = 0; u < U; ++u) {
                                        y[u][e] = fast_exp2(y[u][e] - ref);
                                        y[u][2 + e] = fast_exp2(y[u][2 + e] - ref);
                                    }
                                    l[n][e] += U == 2 ? (y[0][e] + y[0][2 + e]) + (y[U - 1][e] + y[U - 1][2 + e]) : y[0][e] + y[0][2 + e];
                                }
#pragma unroll
                                for (int u = 0; u < U; ++u) {
                                    pb[n][u][0] = transpose_8x8(pack2<false>(y[u][0], y[u][1]));
                                    pb[n][u][1] = transpose_8x8(pack2<false>(y[u][2], y[u][3]));
                                }
                            }
                            if (NT != 1 && !take_values()) return false;
                            if (k0 + 16 * U > seen || (p.window > 0 && k0 + 16 * U > early && k0 < low_first)) {  // keys that no row sees
#pragma unroll
                                for (int u = 0; u < U; ++u) {
#pragma unroll
                                    for (int i = 0; i < 4; ++i) {
                                        const int key = k0 + 16 * u + 2 * c4 + (i & 1) + 8 * (i >> 1);
                                        const bool real = key < seen && !(p.window > 0 && key >= early && key < low_first);
#pragma unroll
                                        for (int j = 0; j < D / 32; ++j) xv[u][i][j] = real ? xv[u][i][j] : 0u;
                                    }
                                }
                            }
#pragma unroll
                            for (int u = 0; u < U; ++u) {
                                uint32_t two[2];
#pragma unroll
                                for (int i = 0; i < 2; ++i) two[i] = (scale_to_h2(v_scale[u][i] & 255u) & 0xffffu) | (scale_to_h2(v_scale[u][i] >> 8) & 0xffff0000u);
#pragma unroll
                                for (int i = 0; i < kCols; ++i) {
                                    // bytes 2 i and 2 i + 1 of the first key, each beside the second one's
                                    const uint32_t pick = (i & 1) ? 0x7362u : 0x5140u;
                                    uint32_t va[4];
                                    unpack_e4m3x4(__byte_perm(xv[u][0][i >> 1], xv[u][1][i >> 1], pick), va[0], va[1]);
                                    unpack_e4m3x4(__byte_perm(xv[u][2][i >> 1], xv[u][3][i >> 1], pick), va[2], va[3]);
#pragma unroll
                                    for (int e = 0; e < 4; ++e) va[e] = mul_h2(va[e], two[e >> 1]);
#pragma unroll
                                    for (int n = 0; n < NT; ++n) mma_16816(o[i][n], va, pb[n][u][0], pb[n][u][1]);
                                }
                            }
                        }
                        if (!mbar_wait_warp(BAR(B_SUMSFREE), direct & 1, ab, ST_WAIT_TIMEOUT + 22)) return false;
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const int row = 8 * n + 2 * c4 + e;
#pragma unroll
                                for (int d = 4; d < 32; d <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], d);
                                if (g8 == 0) {
                                    float* const ml = reinterpret_cast<float*>(smem + S::off_ml) + s * (4 * kBlk) + w * (2 * kBlk) + (warp & 3) * 32 + row;
                                    ml[0] = m[n][e];
                                    ml[kBlk] = l[n][e];
                                }
                                float4* const to = reinterpret_cast<float4*>(smem + S::off_sums) + (warp * kDirectRows + row) * (D / 4);
#pragma unroll
                                for (int i = 0; i < kCols; i += 2)
                                    to[sums_place<D>(row, g8 * (D / 32) + i / 2)] = make_float4(o[i][n][e], o[i][n][2 + e], o[i + 1][n][e], o[i + 1][n][2 + e]);
                            }
                        }
                        return true;
                    };
                    alive = tokens * p.G <= 8 ? multiply(std::integral_constant<int, 1>{}) : multiply(std::integral_constant<int, 2>{});
                    ++direct;
                    if (!alive) break;
                    mbar_arrive_warp(BAR(B_MLFULL + s), lane);
                    if (lane == 0) mbar_arrive(BAR(B_ITEMEMPTY + s));
                    continue;
                }
            }
            const int t0 = (G ^ w) & 1;  // this group's first tile of the item
            float m_run = -INFINITY, l_run = 0.f;
            float factor = 1.f;  // E4M3 of bf16: of the row's scores

            for (int t = t0; t < T && alive; alive = alive && unpack_values(t), t += 2) {
                const int k0 = key_block(lo + t, border, skip) * kBlk;
                // MASKED: rows of the tile that no row of the item sees although they lie before its last key
                const int none_from = MASKED ? max(early - k0, 0) : 0, none_end = MASKED ? min(low_first - k0, kBlk) : 0;
                const bool none = MASKED && none_end > none_from;
                // does some row not see all of the tile?
                auto masked = [&] { return k0 + kBlk - 1 > all_see || (MASKED && p.window > 0 && k0 < low_last && k0 + kBlk > early); };
                const int g = G + t;
                const uint32_t tS = tmem + lane_base + uint32_t(S::tmem_s(g)), tP = tmem + lane_base + uint32_t(S::tmem_p(g));
                // P*V of the group's tile before: it has read its P and added to O
                auto pv_before = [&] { return g < 2 || mbar_wait_warp(BAR(B_PVDONE + (g - 2) % NP), ((g - 2) / NP) & 1, ab, ST_WAIT_TIMEOUT + 8); };
                alive = mbar_wait_warp(BAR(B_SFULL + (g & 3)), (g >> 2) & 1, ab, ST_WAIT_TIMEOUT + 7);
                if (!alive) break;
                tc_fence_after();
                if constexpr (E4M3 && BF16) factor = reinterpret_cast<volatile float*>(smem + S::off_factor)[s * kBlk + r];  // (written before Q was given to the product)
                const float c = scale_of(factor);
                if (!active) {  // no row of this warp is a query: its lanes of P and O are never stored
                    if (S::POWN) {
                        mbar_arrive_warp(BAR(B_SFREE + w), lane);
                        alive = pv_before();
                        if (!alive) break;
                    }
                    if (!E4M3 && (seen - k0 < kBlk || none)) alive = zero_behind(g, MASKED ? min(seen - k0, kBlk) : seen - k0, none_from, none_end);
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
                    float ref = m_run == -INFINITY ? 0.f : m_run;  // SCORED: as below
                    if constexpr (SCORED) {
                        if (E4M3 && BF16 && __any_sync(0xffffffffu, factor != 1.f)) {
#pragma unroll
                            for (int x = 0; x < 32; ++x) v[x] *= factor;
                        }
                        if (!E4M3 && seen - kq < 32) {
#pragma unroll
                            for (int x = 0; x < 32; ++x) v[x] = x < seen - kq ? v[x] : 0.f;
                        }
                        if (!E4M3 && none) {
#pragma unroll
                            for (int x = 0; x < 32; ++x) v[x] = x + 32 * quarter >= none_from && x + 32 * quarter < none_end ? 0.f : v[x];
                        }
                        const Bias bias(slope, front == 0, pos0 - (kq + 31), pos0 + 31 - kq);
                        if constexpr (BIASED) ref = tile_reference(bias, ref, pos - kq - 16);
                        score_row<KIND, 32>(v, p.score, bias, p.scale_log2, pos - kq, valid, ref - kRaised);
                    }
                    if (MASKED ? masked() : kq + 31 > all_see) {
                        const uint32_t keep = sees(kq);
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
                    float top = fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]);
                    if constexpr (E4M3 && SCORED) top -= kRaised;
                    float m_new = fmaxf(m_run, top);
                    bool need = (m_new - m_run) * c > 8.0f;
                    float move = 0.f;
                    if constexpr (SCORED) {
                        const bool fresh = m_run == -INFINITY;
                        if (BIASED && !fresh) move = ref - m_run;
                        need = fresh ? top != -INFINITY : top + move > 8.0f;
                        m_new = ref + top;
                        if (need) move = BIASED ? ref - m_new : -top;
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
                    // (SCORED: what is left to be added)
                    const float mneg = SCORED ? move : (m_run == -INFINITY) ? 0.f : E4M3 ? kRaised - m_run * c : -m_run * c;
                    float l4[4] = {0.f, 0.f, 0.f, 0.f};
                    uint32_t pk[16];
#pragma unroll
                    for (int x = 0; x < 32; x += 2) {
                        const float p0 = fast_exp2(fmaf(v[x], c, mneg)), p1 = fast_exp2(fmaf(v[x + 1], c, mneg));
                        l4[x & 2] += p0;
                        l4[(x & 2) + 1] += p1;
                        pk[x / 2] = pack2<PBF16>(p0, p1);
                    }
                    uint32_t zero[16] = {};
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        if (q != quarter) tmem_st16(tP + uint32_t(q) * 16u, zero);
                    tmem_st16(tP + uint32_t(quarter) * 16u, pk);
                    tc_wait_st();
                    if (!E4M3 && (seen - k0 < kBlk || none)) alive = zero_behind(g, MASKED ? min(seen - k0, kBlk) : seen - k0, none_from, none_end);
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
                float ref = m_run == -INFINITY ? 0.f : m_run;  // SCORED: what the scores are relative to
                if constexpr (SCORED) {
                    if (E4M3 && BF16 && __any_sync(0xffffffffu, factor != 1.f)) {
#pragma unroll
                        for (int x = 0; x < kBlk; ++x) sc[x] *= factor;
                    }
                    // (what the others' scores are must not tell the warp which form of the cap to take. E4M3: they are 0)
                    if (!E4M3 && real < kBlk) {
#pragma unroll
                        for (int x = 0; x < kBlk; ++x) sc[x] = x < real ? sc[x] : 0.f;
                    }
                    if (!E4M3 && none) {
#pragma unroll
                        for (int x = 0; x < kBlk; ++x) sc[x] = x >= none_from && x < none_end ? 0.f : sc[x];
                    }
                    const Bias bias(slope, front == 0, pos0 - (k0 + kBlk - 1), pos0 + kBlk - 1 - k0);
                    if constexpr (KIND == SCORE_CAPPED) late = !masked() && !any_beyond<kBlk>(sc, valid ? p.score.most : INFINITY);
                    if constexpr (BIASED) ref = tile_reference(bias, ref, pos - k0 - kBlk / 2);
                    if (!late) score_row<KIND, kBlk>(sc, p.score, bias, p.scale_log2, pos - k0, valid, ref - kRaised);
                }
                if (masked()) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const uint32_t keep = sees(k0 + 32 * q);
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
                float move = 0.f;  // SCORED: from `ref` to the reference point
                if constexpr (SCORED) {  // (the scores, and mx, are relative to `ref`: the old reference point, or 0 in front of a row's first key, or BIASED perhaps the tile's own)
                    const bool fresh = m_run == -INFINITY;
                    if (late) mx = cap_one(mx, p.score) - ref;
                    else if constexpr (E4M3) mx -= kRaised;
                    if (BIASED && !fresh) move = ref - m_run;
                    need = fresh ? mx != -INFINITY : mx + move > 8.0f;
                    m_new = ref + mx;
                    if (need) move = BIASED ? ref - m_new : -mx;
                }
                if (!need) m_new = m_run;
                if (S::POWN) {  // this tile's P overwrites that one's
                    alive = pv_before();
                    if (!alive) break;
                    tc_fence_after();
                }
                if (__any_sync(0xffffffffu, need || (BIASED && move != 0.f))) {
                    if (SCORED && !late) {
#pragma unroll
                        for (int x = 0; x < 128; x += 2) unpack_f2(add_f2(pack_f2(sc[x], sc[x + 1]), pack_f2(move, move)), sc[x], sc[x + 1]);
                    }
                    const float alpha = need ? fast_exp2((m_run - m_new) * c) : 1.0f;
                    l_run *= alpha;
                    if (t > t0 && (!BIASED || __any_sync(0xffffffffu, need))) {
                        if (!S::POWN) {
                            alive = pv_before();
                            if (!alive) break;
                            tc_fence_after();
                        }
                        rescale(alpha);
                    }
                }
                m_run = m_new;
                const float mneg = (m_run == -INFINITY) ? 0.f : E4M3 ? kRaised - m_run * c : -m_run * c;
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
                            pk[x] = pack2<PBF16>(p0, p1);
                        }
                        tmem_st16(tP + uint32_t(q) * 16u, pk);
                    }
                };
                if constexpr (!SCORED) exponentials([&](uint64_t s2) { return fma_f2(s2, c2, mneg2); });
                else if (KIND == SCORE_CAPPED && late) exponentials([&](uint64_t s2) { return fma_f2(s2, cap_poly(s2, p.score), mneg2); });
                else exponentials([&](uint64_t s2) { return s2; });
                tc_wait_st();
                if (!E4M3 && (real < kBlk || none)) alive = zero_behind(g, MASKED ? min(real, kBlk) : real, none_from, none_end);
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
    if (!DIRECT && warp == 13) {
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
template <int D, bool BF16, int KIND, int FORM>
static cudaError_t launch_paged_t(const CUtensorMap& tq, const CUtensorMap& tn, const CUtensorMap& tk, const CUtensorMap& tv, const PagedParams& p, int workers, cudaStream_t stream) {
    auto kern = paged_fwd_kernel<D, BF16, KIND, FORM>;
    constexpr int smem = PagedSmem<D, FORM>::total;
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
        if (p.k_scales && !p.starts && p.G <= kDirectRows)
            return bf16 ? launch_paged_t<kD, true, kKind, FORM_MASKED | FORM_E4M3 | FORM_DIRECT>(tq, tn, tk, tv, p, workers, stream)
                        : launch_paged_t<kD, false, kKind, FORM_MASKED | FORM_E4M3 | FORM_DIRECT>(tq, tn, tk, tv, p, workers, stream);
        if (p.k_scales)
            return bf16 ? launch_paged_t<kD, true, kKind, FORM_MASKED | FORM_E4M3>(tq, tn, tk, tv, p, workers, stream)
                        : launch_paged_t<kD, false, kKind, FORM_MASKED | FORM_E4M3>(tq, tn, tk, tv, p, workers, stream);
        if (p.window > 0 || p.parents)
            return bf16 ? launch_paged_t<kD, true, kKind, FORM_MASKED>(tq, tn, tk, tv, p, workers, stream)
                        : launch_paged_t<kD, false, kKind, FORM_MASKED>(tq, tn, tk, tv, p, workers, stream);
        return bf16 ? launch_paged_t<kD, true, kKind, FORM_PLAIN>(tq, tn, tk, tv, p, workers, stream)
                    : launch_paged_t<kD, false, kKind, FORM_PLAIN>(tq, tn, tk, tv, p, workers, stream);
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
