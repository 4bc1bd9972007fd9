// New tokens' keys and values into the pages of a cache: token t of a sequence with n new tokens and `len` cached ones (the new ones among
// them) goes to position len - n + t, slot position % page size of the page that the sequence's row of the table names.
//
// Moves 8 bytes for each element of K (2 read and 2 written, of K and of V each). One warp per token: it asks for its rows' first 4 KB before it looks for the token's
// sequence (a search over the batch's first rows, then the length, then the table: a chain of three or four loads, which is what a step of
// single tokens is bound by).
//
// Measured: 8 prompts of 3500 tokens, 8 heads of 128, pages of 16, 198 MB in 33-35 us, 5.7-6.1 TB/s (the copy rate is 6.56); one token each of 64 sequences 4 us.
#include <type_traits>
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

// of 8 bits: bytes
struct AppendPages8 {
    uint8_t *k, *v, *k_scales, *v_scales;
    int64_t k_p, k_s, k_h, v_p, v_s, v_h;
};

constexpr int kAppendThreads = 128;

// Where token t goes; false where it goes nowhere. By all lanes of a warp.
__device__ __forceinline__ bool place_of(const PagedParams& p, int t, int lane, int& page, int& slot) {
    // the last sequence that begins at or before t: starts[b] <= t < starts[b + 1]
    int b = t, first = t, n = 1;
    if (p.starts) {
        int lo = 0, hi = p.B;  // of the sequences in [lo, hi); a step looks at 32 of them
        if (t < p.starts[0] || t >= p.starts[p.B]) return false;  // of no sequence
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
        return false;
    }
    if (pos < 0) return false;  // more new tokens than cached ones: the cache begins behind these
    page = p.table[b * p.table_stride + (pos >> p.log2_page)];
    if (uint32_t(page) >= uint32_t(p.n_pages)) {
        if (lane == 0) atomicCAS(p.status, 0, ST_PAGED_PAGE);
        return false;
    }
    slot = int(pos) & (p.page - 1);
    return true;
}

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
    int page, slot;
    if (!place_of(p, t, lane, page, slot)) return;
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

// The same into a cache of 8 bits: each head's row of a token becomes e4m3 times a power of two, the least that brings its largest finite number to 448 or below, from 2^-15 to 2^7. (A
// power of two costs a floating format no precision, and dividing by it nothing and no rounding: the rows are what the definition says to the bit.) What is not finite becomes a NaN;
// numbers beyond 448 * 2^7 = 57344 become that.
//
// Moves 6 bytes for each element of K (2 read and 1 written, of K and of V each) and a byte for each row. The lanes that hold a head's row (16 at a head dim of 128) find its largest
// number among them by shuffles, in registers. 8 prompts of 3500 tokens, 8 heads of 128, pages of 16: 149 MB in 32 us, 4.7 TB/s, which is the time that a 16-bit append of a third more bytes takes. No
// unit is full: 62 % of the ALU, 61 % of the issue slots; what is left is a warp's chain from the starts to its stores. (Each number in fp32 by itself, with its own look at whether it is
// finite, takes as long.)
template <int kLog2Row, bool BF16>
__global__ void __launch_bounds__(kAppendThreads) paged_append_e4m3_kernel(const PagedParams p, const AppendRows in, const AppendPages8 to) {
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
            k[i] = v[i] = make_uint4(0, 0, 0, 0);
            if (w >= words) continue;
            k[i] = k_row[(w >> kLog2Row) * in.k_h + (w & kMask)];
            v[i] = v_row[(w >> kLog2Row) * in.v_h + (w & kMask)];
        }
    };
    fetch(0);
    int page, slot;
    if (!place_of(p, t, lane, page, slot)) return;
    constexpr uint32_t kInf = BF16 ? 0x7f80u : 0x7c00u;
    auto put = [&](uint4 row, uint8_t* data, uint8_t* scale, bool real, bool first) {
        uint32_t w[4] = {row.x, row.y, row.z, row.w}, most = 0;
        // (numbers of 16 bits without their sign go by size)
#pragma unroll
        for (int i = 0; i < 4; ++i) most = __vmaxu2(most, w[i] & 0x7fff7fffu);
        most = max(most & 0xffffu, most >> 16);
        if (__any_sync(0xffffffffu, most >= kInf)) {  // not finite: NaN, which have no say
            most = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t lo = w[i] & 0x7fffu, hi = w[i] >> 16 & 0x7fffu;
                if (lo >= kInf) w[i] |= 0x7fffu; else most = max(most, lo);
                if (hi >= kInf) w[i] |= 0x7fff0000u; else most = max(most, hi);
            }
        }
#pragma unroll
        for (int o = 1; o <= kMask; o <<= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
        float largest, none;
        unpack2<BF16>(most, largest, none);
        const uint32_t bits = __float_as_uint(largest);  // 448 = 1.75 * 2^8
        const int biased = min(max(int(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0), kScaleLeast), kScaleMost);
        if (!real) return;
        const float inverse = __uint_as_float(uint32_t(254 - biased) << 23);
        uint32_t e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float lo, hi;
            unpack2<BF16>(w[i], lo, hi);
            e[i] = pack_e4m3x2(lo * inverse, hi * inverse);
        }
        *reinterpret_cast<uint2*>(data) = make_uint2(__byte_perm(e[0], e[1], 0x5410), __byte_perm(e[2], e[3], 0x5410));
        if (first) *scale = uint8_t(biased);
    };
    uint8_t* const k_to = to.k + page * to.k_p + slot * to.k_s;
    uint8_t* const v_to = to.v + page * to.v_p + slot * to.v_s;
    uint8_t* const k_scale = to.k_scales + page * p.k_scale_p + slot;
    uint8_t* const v_scale = to.v_scales + page * p.v_scale_p + slot;
    for (int w0 = 0;;) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int w = w0 + 32 * i + lane, h = w >> kLog2Row, at = w & kMask;
            if (w0 + 32 * i >= words) break;  // (the same for all lanes)
            put(k[i], k_to + h * to.k_h + at * 8, k_scale + h * p.k_scale_h, w < words, at == 0);
            put(v[i], v_to + h * to.v_h + at * 8, v_scale + h * p.v_scale_h, w < words, at == 0);
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

// strides[10]: k rows (token, head), v rows, in 16 bytes; k pages (page, slot, head), v pages, in bytes
cudaError_t launch_paged_append_e4m3(bool bf16, const PagedParams& p, const void* k, const void* v, void* k_pages, void* v_pages, uint8_t* k_scales, uint8_t* v_scales,
                                     const int64_t* strides, cudaStream_t stream) {
    const AppendRows in{static_cast<const uint4*>(k), static_cast<const uint4*>(v), strides[0], strides[1], strides[2], strides[3]};
    const AppendPages8 to{static_cast<uint8_t*>(k_pages), static_cast<uint8_t*>(v_pages), k_scales, v_scales, strides[4], strides[5], strides[6], strides[7], strides[8], strides[9]};
    const dim3 grid(cdiv(p.T, kAppendThreads / 32));
    auto launch = [&](auto log2_row) {
        constexpr int kLog2Row = decltype(log2_row)::value;
        return launch_overlapping(bf16 ? paged_append_e4m3_kernel<kLog2Row, true> : paged_append_e4m3_kernel<kLog2Row, false>, grid, kAppendThreads, 0, stream, p, in, to);
    };
    using std::integral_constant;
    switch (p.D) {
        case 16: return launch(integral_constant<int, 1>{});
        case 32: return launch(integral_constant<int, 2>{});
        case 64: return launch(integral_constant<int, 3>{});
        case 128: return launch(integral_constant<int, 4>{});
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace fa
