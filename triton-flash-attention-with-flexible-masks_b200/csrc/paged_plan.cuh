// How the attention over a paged cache is shared out, worked out by every block for itself from the lengths in device memory (the host does not
// know them, and a captured call has to follow them).
//
// An item is a tile of queries (tokens_per_tile new tokens of a sequence, all heads of a kv head's group) of one kv head. Its weight is the
// number of keys that its last token sees (with a window, less those that lie between the first keys and it), and a constant for what an item costs besides its tiles. The items, in the order sequence, kv head,
// tile, lie behind one another on a line of length `total`, and each of n workers gets an equal stretch of it, whatever the lengths, with at most
// n - 1 cuts. An item that a cut goes through is computed in pieces, whose fp32 rows the second kernel merges.
// Where there are no more items than workers and whole items, one a worker, are done as soon, nothing is cut (`keyed` false: all weights are 1):
// merging costs what some tiles cost. Whole | cut, us, 32 / 8 heads of 128 but for the first: one token behind 699 of 8 heads of 64 15.9 | 20.7, eight behind 300
// each 16.6 | 33.0, one behind 1500 22.6 | 25.7, one behind 3000 28.9 | 26.3, one behind 131071 879 | 99.
#pragma once
#include "common.cuh"
#include "params.cuh"

namespace fa {

// New tokens of a sequence up to which its parents are looked at; more are a chunk, each behind the one before it.
constexpr int kPagedTree = 256;
constexpr int kPagedGroups = 1024;   // entries of the table of sums: a sequence each, or several
// Sequences up to which one warp makes the plan, beside which the others go on. One warp | all, us: single tokens of 1 sequence 15.9 | 16.6, of 128 101.0 | 102.0,
// of 256 179.6 | 179.9, of 512 322 | 318.
constexpr int kPagedWarpPlan = 128;
// Entries of the table of a batch, and its sequences an entry.
__host__ __device__ __forceinline__ int paged_entries(int B) { return B <= kPagedWarpPlan ? 32 : kPagedGroups; }
__host__ __device__ __forceinline__ int paged_group(int B) { return cdiv(B, paged_entries(B)); }
// Of an item besides its tiles, in keys. With 64 | 256 | 640 | 1500, us: 256 single tokens behind up to 1000 189 | 177 | 165 | 167, two chunks of 500 behind 1500
// 67 | 53 | 43 | 45, twelve sequences with four chunks of 1000 186 | 183 | 174 | 175, one token behind 3000 26.9 | 26.1 | 24.5 | 29.7 (pieces of 2048 there).
constexpr int kPagedItemCost = 640;
// A worker's stretch is at least 2 to this long. With 10 | 11 | 12, us: one token behind 3000 26.1 | 30.8 | 29.4, two chunks of 500 behind 1500 53 | 53 | 65.
constexpr int kPagedLog2Piece = 10;
// What the second kernel costs, in tiles of 128 keys. With 2 | 6 | 12, us: eight tokens behind 1500 each 30.9 | 24.5 | 24.8.
constexpr int kPagedMergeTiles = 6;

struct PagedPlan {
    long long total;
    long long stretch;  // of a worker: no less than total / workers
    int workers;
    int keyed;
    int group;  // sequences an entry of `sums`
    int pad;
    long long warp_sums[32], warp_items[32];
    int warp_max[32];
    long long sums[kPagedGroups];  // of what lies before an entry's sequences
};

__host__ __device__ __forceinline__ int paged_clamp(int x, int lo, int hi) { return x < lo ? lo : x > hi ? hi : x; }

// One sequence of the batch. Every number is taken into its range: whatever the caller's tensors hold, nothing outside of them is touched.
struct PagedSeq {
    int start, n;  // first row and number of new tokens
    int len;       // cached tokens, the new ones among them
    int base;      // position of the first new one (below 0: those see nothing)
    int front;     // leading keys that all see
    int tiles;     // of queries
    // MASKED (a call with a window or with parents, or of an 8-bit cache)
    int early;     // leading keys that the window hides from none
    int tree;      // the tokens' parents count
};

template <bool MASKED>
__host__ __device__ __forceinline__ PagedSeq paged_seq(const PagedParams& p, int b) {
    PagedSeq s;
    int end;
    if (p.starts) {
        s.start = paged_clamp(p.starts[b], 0, p.T);
        end = paged_clamp(p.starts[b + 1], s.start, p.T);
    } else {
        s.start = b;
        end = b + 1;
    }
    s.n = end - s.start;
    s.len = paged_clamp(p.lens[b], 0, p.capacity);
    s.base = s.len - s.n;
    s.front = p.prefix ? paged_clamp(p.prefix[b], 0, s.len) : 0;
    s.tiles = cdiv(s.n, p.tokens);
    if constexpr (MASKED) {
        s.early = s.front > p.sinks ? s.front : p.sinks;
        s.tree = p.parents && s.n <= kPagedTree;
    }
    return s;
}

// The end of the keys that tile i's last token sees.
__host__ __device__ __forceinline__ int paged_seen(const PagedParams& p, const PagedSeq& s, int i) {
    const long long end = s.base + (long long)(i + 1) * p.tokens;
    const int seen = end < s.len ? int(end) : s.len;
    return seen > s.front ? seen : s.front;
}
// With a window: the first key that is in the window of a token of tile i (a tree's tokens may all continue the cached text).
__host__ __device__ __forceinline__ int paged_low(const PagedParams& p, const PagedSeq& s, int i) {
    const long long low = s.base + (s.tree ? 0 : (long long)i * p.tokens) - p.window + 1;
    return low > 0 ? int(low) : 0;
}
// Key blocks that lie between tile i's early keys and its window.
__host__ __device__ __forceinline__ int paged_skip(const PagedParams& p, const PagedSeq& s, int i) {
    if (p.window == 0) return 0;
    const int skip = paged_low(p, s, i) / kBlk - cdiv(s.early, kBlk);
    return skip > 0 ? skip : 0;
}
// What tile i counts for: the keys that its last token sees, less those between the early ones and the window (so no more than its blocks hold).
template <bool MASKED>
__host__ __device__ __forceinline__ int paged_keys(const PagedParams& p, const PagedSeq& s, int i) {
    int keys = paged_seen(p, s, i);
    if constexpr (MASKED) {
        const int hidden = p.window > 0 ? paged_low(p, s, i) - s.early : 0;
        if (hidden > 0) keys -= hidden;
    }
    return keys;
}

// The weights of the first m tiles of one head together.
template <bool MASKED>
__host__ __device__ __forceinline__ long long paged_weight(const PagedParams& p, const PagedSeq& s, int m, bool keyed) {
    if (!keyed) return m;
    // the tiles but the last end at base + (i + 1) tokens < len; those below `front` see that many keys
    const int inner = m < s.tiles ? m : s.tiles - 1;
    long long sum = (long long)m * kPagedItemCost;
    if (inner > 0) {
        const long long ahead = (long long)s.front - s.base;
        const long long fewer = ahead > 0 ? (ahead + p.tokens - 1) / p.tokens - 1 : 0, below = fewer < inner ? fewer : inner;
        const long long rest = inner - below;
        sum += below * s.front + rest * s.base + (long long)p.tokens * (rest * (below + 1) + rest * (rest - 1) / 2);
    }
    if constexpr (MASKED) {
        if (p.window > 0) {  // the hidden keys of tile i: first + i tokens of them where that is above 0; of a tree's tiles all the same
            const long long first = (long long)s.base - p.window + 1 - s.early;
            if (s.tree) {
                if (first > 0) sum -= m * first;
            } else {
                const long long none = first >= 0 ? 0 : (-first + p.tokens - 1) / p.tokens, some = m > none ? m - none : 0;
                sum -= some * first + (long long)p.tokens * (some * none + some * (some - 1) / 2);
            }
        }
    }
    return m == s.tiles && m > 0 ? sum + s.len : sum;
}

// a / b for 0 <= a, 0 < b: the short division where it will do
__host__ __device__ __forceinline__ long long paged_divide(long long a, long long b) {
    return ((a | b) >> 32) == 0 ? (long long)(uint32_t(a) / uint32_t(b)) : a / b;
}

// Weights of all items together, their number and the longest sequence's length, to the plan's numbers.
__host__ __device__ __forceinline__ void paged_share_out(PagedPlan& plan, long long weight, long long items, int longest, int most_workers) {
    long long workers = weight >> kPagedLog2Piece;
    workers = workers < 1 ? 1 : workers > most_workers ? most_workers : workers;
    plan.keyed = items > most_workers || (long long)(cdiv(longest, kBlk) - kPagedMergeTiles) * kBlk * workers > weight;
    plan.workers = int(plan.keyed ? workers : items);
    plan.total = plan.keyed ? weight : items;
    // (a hair more than total / workers: a division in fp32 takes a fraction of one of 64 bits)
    plan.stretch = plan.keyed ? (long long)(float(weight) / float(workers) * 1.00001f) + 1 : 1;
}

// The plan of up to kPagedWarpPlan sequences, by one warp, the one that needs it: 32 entries of `sums`. (By all warps it costs a microsecond more, of which with
// many sequences nothing is left.)
template <bool MASKED>
__device__ __forceinline__ void paged_plan_warp(const PagedParams& p, PagedPlan& plan, int most_workers) {
    const int lane = threadIdx.x & 31, group = paged_group(p.B);
    long long w = 0, n = 0;
    int longest = 0;
#pragma unroll 1
    for (int b = lane * group; b < min(p.B, (lane + 1) * group); ++b) {
        const int len = p.lens[b];
        const PagedSeq s = paged_seq<MASKED>(p, b);
        if (len > p.capacity || len < 0) atomicCAS(p.status, 0, ST_PAGED_LENGTH);
        w += p.Hk * paged_weight<MASKED>(p, s, s.tiles, true);
        n += (long long)p.Hk * s.tiles;
        longest = max(longest, s.tiles > 0 ? MASKED ? paged_keys<MASKED>(p, s, s.tiles - 1) : s.len : 0);
    }
    __syncwarp();
    longest = __reduce_max_sync(0xffffffffu, longest);
    long long w_sum = w, n_sum = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, w_sum, o), y = __shfl_up_sync(0xffffffffu, n_sum, o);
        if (lane >= o) {
            w_sum += x;
            n_sum += y;
        }
    }
    PagedPlan own;
    paged_share_out(own, __shfl_sync(0xffffffffu, w_sum, 31), __shfl_sync(0xffffffffu, n_sum, 31), longest, most_workers);
    plan.sums[lane] = own.keyed ? w_sum - w : n_sum - n;
    if (lane == 0) {
        plan.total = own.total;
        plan.stretch = own.stretch;
        plan.workers = own.workers;
        plan.keyed = own.keyed;
        plan.group = group;
    }
    __syncwarp();
}

// All threads of the block (a multiple of 32, at most 1024, that divides 2 * kPagedGroups). Ends with a barrier.
template <int kThreads, bool MASKED>
__device__ __forceinline__ void paged_plan(const PagedParams& p, PagedPlan& plan, int most_workers) {
    constexpr int kOwn = kPagedGroups / kThreads, kWarps = kThreads / 32;
    static_assert(kOwn * kThreads == kPagedGroups && kOwn >= 1, "groups of a thread");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int group = paged_group(p.B), first = threadIdx.x * kOwn;
    long long weight[kOwn], items[kOwn], w = 0, n = 0;
    int longest = 0;
#pragma unroll
    for (int o = 0; o < kOwn; ++o) {
        weight[o] = items[o] = 0;
        for (int b = (first + o) * group; b < min(p.B, (first + o + 1) * group); ++b) {
            const PagedSeq s = paged_seq<MASKED>(p, b);
            if (p.lens[b] > p.capacity || p.lens[b] < 0) atomicCAS(p.status, 0, ST_PAGED_LENGTH);
            weight[o] += p.Hk * paged_weight<MASKED>(p, s, s.tiles, true);
            items[o] += (long long)p.Hk * s.tiles;
            if (s.tiles > 0) longest = max(longest, MASKED ? paged_keys<MASKED>(p, s, s.tiles - 1) : s.len);
        }
        w += weight[o];
        n += items[o];
    }
    // inclusive sums over the warp, then over the warps
    longest = __reduce_max_sync(0xffffffffu, longest);
    long long w_before = w, n_before = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, w_before, o), y = __shfl_up_sync(0xffffffffu, n_before, o);
        if (lane >= o) {
            w_before += x;
            n_before += y;
        }
    }
    if (lane == 31) {
        plan.warp_sums[warp] = w_before;
        plan.warp_items[warp] = n_before;
        plan.warp_max[warp] = longest;
    }
    __syncthreads();
    w_before -= w;
    n_before -= n;
    w = n = 0;
    longest = 0;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
        const long long x = plan.warp_sums[i], y = plan.warp_items[i];
        w += x;
        n += y;
        if (i < warp) {
            w_before += x;
            n_before += y;
        }
        longest = max(longest, plan.warp_max[i]);
    }
    PagedPlan own;
    paged_share_out(own, w, n, longest, most_workers);
    const bool keyed = own.keyed;
    long long before = keyed ? w_before : n_before;
#pragma unroll
    for (int o = 0; o < kOwn; ++o) {
        plan.sums[first + o] = before;
        before += keyed ? weight[o] : items[o];
    }
    if (threadIdx.x == 0) {
        plan.total = own.total;
        plan.stretch = own.stretch;
        plan.workers = own.workers;
        plan.keyed = own.keyed;
        plan.group = group;
    }
    __syncthreads();
}

// Where worker w's stretch begins; the last ones' may be empty.
__host__ __device__ __forceinline__ long long paged_cut(const PagedPlan& plan, int w) {
    const long long x = plan.stretch * w;
    return x < plan.total ? x : plan.total;
}

// A walk over the items from a point of the line on.
template <bool MASKED>
struct PagedWalk {
    PagedSeq s;
    int b, hk, tile;
    long long at;  // where the item begins

    // The item that covers x, 0 <= x < total.
    __host__ __device__ __forceinline__ void find(const PagedParams& p, const PagedPlan& plan, long long x) {
        int lo = 0;  // the last entry with sums[lo] <= x
#ifdef __CUDA_ARCH__
        static_assert(kPagedGroups == 32 * 32, "two steps of a warp");  // (whose lanes all ask for the same x)
        if (p.B > kPagedWarpPlan) lo = 32 * (31 - __clz(__ballot_sync(0xffffffffu, plan.sums[32 * (threadIdx.x & 31)] <= x)));
        lo += 31 - __clz(__ballot_sync(0xffffffffu, plan.sums[lo + (threadIdx.x & 31)] <= x));
#else
        while (lo + 1 < paged_entries(p.B) && plan.sums[lo + 1] <= x) ++lo;
#endif
        long long rem = x - plan.sums[lo];
        b = lo * plan.group;
        long long head;
        for (;; ++b) {
            if (b >= p.B) {  // (somebody writes the lengths while the kernel reads them)
                s = PagedSeq{};
                hk = tile = 0;
                at = x;
                return;
            }
            s = paged_seq<MASKED>(p, b);
            head = paged_weight<MASKED>(p, s, s.tiles, plan.keyed);
            if (rem < head * p.Hk) break;
            rem -= head * p.Hk;
        }
        hk = int(paged_divide(rem, head));
        rem -= hk * head;
        int t0 = 0, t1 = s.tiles;  // weight(t0) <= rem < weight(t1)
        while (t1 - t0 > 1) {
            const int mid = (t0 + t1) >> 1;
            if (paged_weight<MASKED>(p, s, mid, plan.keyed) <= rem) t0 = mid; else t1 = mid;
        }
        tile = t0;
        at = x - rem + paged_weight<MASKED>(p, s, t0, plan.keyed);
    }
    __host__ __device__ __forceinline__ long long end(const PagedParams& p, const PagedPlan& plan) const {
        return at + (plan.keyed ? paged_keys<MASKED>(p, s, tile) + kPagedItemCost : 1);
    }
    // The next item; there is one.
    __host__ __device__ __forceinline__ void next(const PagedParams& p, const PagedPlan& plan) {
        at = end(p, plan);
        if (++tile < s.tiles) return;
        tile = 0;
        if (++hk < p.Hk) return;
        hk = 0;
        do s = ++b < p.B ? paged_seq<MASKED>(p, b) : PagedSeq{}; while (s.tiles == 0 && b < p.B);
    }
    __host__ __device__ __forceinline__ int key_tiles(const PagedParams& p) const { return cdiv(paged_seen(p, s, tile), kBlk) - (MASKED ? paged_skip(p, s, tile) : 0); }
    // The item's key tile at point x of the line: the pieces on both sides of a cut at x meet there.
    __host__ __device__ __forceinline__ int key_tile_at(const PagedParams& p, const PagedPlan& plan, long long x) const {
        const int n = key_tiles(p);
        if (x <= at) return 0;
        if (x >= end(p, plan)) return n;
        const long long t = x - at - kPagedItemCost;
        static_assert(kBlk == 1 << 7, "shift");
        return t < 0 ? 0 : (t >> 7) > n ? n : int(t >> 7);
    }
};

// The pieces of worker w's stretch, in their order: emit(walk, key tiles of the item, first and last + 1 of the piece, slot of the workspace or -1 for a
// piece that is the whole item) until one says false. A piece without tiles is left out, but for the one that begins an item without any,
// whose rows are zeros.
template <bool MASKED, class Emit>
__host__ __device__ __forceinline__ void paged_stretch(const PagedParams& p, const PagedPlan& plan, int w, Emit emit) {
    PagedWalk<MASKED> walk;
    const long long x0 = paged_cut(plan, w), x1 = paged_cut(plan, w + 1);
    if (x0 >= x1) return;
    walk.find(p, plan, x0);
    for (long long from = x0;;) {
        const int n = walk.key_tiles(p), lo = walk.key_tile_at(p, plan, from), hi = walk.key_tile_at(p, plan, x1);
        if (walk.s.tiles > 0 && (hi > lo || (n == 0 && from <= walk.at)) && !emit(walk, n, lo, hi, hi - lo == n ? -1 : 2 * w + (lo == 0 ? 1 : 0))) return;
        if (walk.end(p, plan) >= x1 || walk.b >= p.B) return;
        walk.next(p, plan);
        from = walk.at;
    }
}

// Is the cut before worker w the first one through the item at `walk`, which it falls into?
template <bool MASKED>
__host__ __device__ __forceinline__ bool paged_first_cut(const PagedPlan& plan, int w, const PagedWalk<MASKED>& walk) {
    return w > 0 && walk.s.tiles > 0 && walk.at < paged_cut(plan, w) && (w == 1 || walk.at >= paged_cut(plan, w - 1));
}

// How many pieces the item at `walk` has, which the cut before worker w goes through first: one each of the workers from `from` on. (Where that cut falls into the item's fixed
// cost or into its first tile, the worker in front of it has none: a cut inside a tile gives the tile to the worker behind the cut, who thus has the last one at least; and a stretch
// that lies within the item has tiles, for it is longer than the cost and a tile.) The first piece's slot is 2 * from + 1, the others' are 2 * (from + i).
template <bool MASKED>
__host__ __device__ __forceinline__ int paged_pieces(const PagedParams& p, const PagedPlan& plan, int w, const PagedWalk<MASKED>& walk, int& from) {
    static_assert((1 << kPagedLog2Piece) > kPagedItemCost + 2 * kBlk, "every stretch within an item has tiles");
    from = walk.key_tile_at(p, plan, paged_cut(plan, w)) > 0 ? w - 1 : w;
    // the last worker: the cuts lie a stretch apart, and its own is the last one before the item's end
    const int v = w + int(paged_divide(walk.end(p, plan) - 1 - paged_cut(plan, w), plan.stretch));
    return (v < plan.workers ? v : plan.workers - 1) - from + 1;  // (somebody writes the lengths while the kernel reads them)
}

}  // namespace fa
