// New tokens' keys and values into the pages of a cache: token t of a sequence with n new tokens and `len` cached ones (the new ones among
// them) goes to position len - n + t, slot position % page size of the page that the sequence's row of the table names.
//
// Moves 8 bytes for each element of K (2 read and 2 written, of K and of V each). One warp per token: it asks for its rows' first 4 KB before it looks for the token's
// sequence (a search over the batch's first rows, then the length, then the table: a chain of three or four loads, which is what a step of
// single tokens is bound by).
//
// Measured: 8 prompts of 3500 tokens, 8 heads of 128, pages of 16, 198 MB in 33-35 us, 5.7-6.1 TB/s (the copy rate is 6.56); one token each of 64 sequences 4 us.
#include "common.cuh"
#include "params.cuh"

namespace fa {

struct AppendRows {
    const uint4* k;
    const uint4* v;
    int64_t k_t, k_h, v_t, v_h;  // strides in 16 bytes
};
struct AppendPages {
    uint4* k;
    uint4* v;
    int64_t k_p, k_s, k_h, v_p, v_s, v_h;  // page, slot, head
};

constexpr int kAppendThreads = 128;

// kLog2Row: log2 of 16-byte words of a head's row
template <int kLog2Row>
__global__ void __launch_bounds__(kAppendThreads) paged_append_kernel(const PagedParams p, const AppendRows in, const AppendPages to) {
    follow_stream();
    const int t = int(blockIdx.x) * (kAppendThreads / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (t >= p.T) return;
    const int words = p.Hk << kLog2Row;
    constexpr int kAhead = 4, kMask = (1 << kLog2Row) - 1;
    const uint4* k_row = in.k + t * in.k_t;
    const uint4* v_row = in.v + t * in.v_t;
    uint4 k[kAhead], v[kAhead];
    auto fetch = [&](int w0) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int w = w0 + 32 * i + lane;
            if (w >= words) continue;
            k[i] = k_row[(w >> kLog2Row) * in.k_h + (w & kMask)];
            v[i] = v_row[(w >> kLog2Row) * in.v_h + (w & kMask)];
        }
    };
    fetch(0);
    // the last sequence that begins at or before t: starts[b] <= t < starts[b + 1]
    int b = t, first = t, n = 1;
    if (p.starts) {
        int lo = 0, hi = p.B;  // of the sequences in [lo, hi); a step looks at 32 of them
        if (t < p.starts[0] || t >= p.starts[p.B]) return;  // of no sequence
        while (hi - lo > 1) {
            const int step = (hi - lo + 31) >> 5, at = lo + lane * step;
            const uint32_t before = __ballot_sync(0xffffffffu, at < hi && p.starts[at] <= t);
            lo += (31 - __clz(before | 1u)) * step;
            hi = min(hi, lo + step);
        }
        b = lo;
        first = p.starts[b];
        n = p.starts[b + 1] - first;
    }
    const int len = p.lens[b];
    const long long pos = (long long)len - n + (t - first);
    if (len < 0 || len > p.capacity || pos >= len) {
        if (lane == 0) atomicCAS(p.status, 0, ST_PAGED_LENGTH);
        return;
    }
    if (pos < 0) return;  // more new tokens than cached ones: the cache begins behind these
    const int page = p.table[b * p.table_stride + (pos >> p.log2_page)];
    if (uint32_t(page) >= uint32_t(p.n_pages)) {
        if (lane == 0) atomicCAS(p.status, 0, ST_PAGED_PAGE);
        return;
    }
    const int slot = int(pos) & (p.page - 1);
    uint4* k_to = to.k + page * to.k_p + slot * to.k_s;
    uint4* v_to = to.v + page * to.v_p + slot * to.v_s;
    for (int w0 = 0;;) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int w = w0 + 32 * i + lane;
            if (w >= words) continue;
            k_to[(w >> kLog2Row) * to.k_h + (w & kMask)] = k[i];
            v_to[(w >> kLog2Row) * to.v_h + (w & kMask)] = v[i];
        }
        w0 += 32 * kAhead;
        if (w0 >= words) break;
        fetch(w0);
    }
}

// strides[10]: k rows (token, head), v rows, k pages (page, slot, head), v pages, in 16 bytes (called from paged.cu)
cudaError_t launch_paged_append(const PagedParams& p, const void* k, const void* v, void* k_pages, void* v_pages, const int64_t* strides, cudaStream_t stream) {
    const AppendRows in{static_cast<const uint4*>(k), static_cast<const uint4*>(v), strides[0], strides[1], strides[2], strides[3]};
    const AppendPages to{static_cast<uint4*>(k_pages), static_cast<uint4*>(v_pages), strides[4], strides[5], strides[6], strides[7], strides[8], strides[9]};
    const dim3 grid(cdiv(p.T, kAppendThreads / 32));
    switch (p.D) {
        case 16: return launch_overlapping(paged_append_kernel<1>, grid, kAppendThreads, 0, stream, p, in, to);
        case 32: return launch_overlapping(paged_append_kernel<2>, grid, kAppendThreads, 0, stream, p, in, to);
        case 64: return launch_overlapping(paged_append_kernel<3>, grid, kAppendThreads, 0, stream, p, in, to);
        case 128: return launch_overlapping(paged_append_kernel<4>, grid, kAppendThreads, 0, stream, p, in, to);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace fa
