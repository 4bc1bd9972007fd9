// extern "C" surface of the paged cache (declared in include/fa_b200.h): argument checks, tensor maps, launches. Nothing here allocates,
// synchronises or throws.
#include <algorithm>
#include <cmath>
#include "../../include/fa_b200.h"
#include "common.cuh"
#include "host_shared.cuh"
#include "paged_plan.cuh"
#include "params.cuh"

namespace fa {
cudaError_t launch_paged_append(const PagedParams&, const void*, const void*, void*, void*, const int64_t*, cudaStream_t);
cudaError_t launch_paged_append_e4m3(bool, const PagedParams&, const void*, const void*, void*, void*, uint8_t*, uint8_t*, const int64_t*, cudaStream_t);
cudaError_t launch_paged_fwd(bool, const CUtensorMap&, const CUtensorMap&, const CUtensorMap&, const CUtensorMap&, const PagedParams&, int, cudaStream_t);
}  // namespace fa

namespace {

constexpr int kMostTokens = 1 << 22;  // of a sequence, and of a call
// The line of all items (paged_plan.cuh), whose points are 64-bit numbers: (kMostTokens + 65535) tiles of queries of 1024 heads, each weighing kMostTokens keys and its cost.
static_assert(double(kMostTokens + 65535) * 1024 * (kMostTokens + fa::kPagedItemCost) < 9.2e18, "64 bits");

bool aligned(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// base and strides (in elements) of a tensor whose last stride is 1, `n` extents before it
int check_strides(const void* ptr, const int64_t* stride, const int* extent, int n) {
    if (!ptr) return FA_ERR_BAD_ARG;
    if (!aligned(ptr, 16)) return FA_ERR_ALIGNMENT;
    for (int i = 0; i < n; ++i)
        if (extent[i] > 1 && (stride[i] <= 0 || stride[i] % 8 != 0)) return FA_ERR_ALIGNMENT;
    return FA_OK;
}

int check_cache(const fa_paged_cache* c) {
    if (!c) return FA_ERR_BAD_ARG;
    if (c->B <= 0 || c->Hk <= 0 || c->pages <= 0 || c->page_size <= 0 || c->table_pages <= 0) return FA_ERR_BAD_ARG;
    if (c->D != 16 && c->D != 32 && c->D != 64 && c->D != 128) return FA_ERR_UNSUPPORTED;
    if (c->dtype != FA_BF16 && c->dtype != FA_FP16) return FA_ERR_UNSUPPORTED;
    if (c->page_size < 8 || (c->page_size & (c->page_size - 1)) != 0) return FA_ERR_PAGED;
    if (int64_t(c->table_pages) * c->page_size > kMostTokens || c->B > 65535 || c->Hk > 1024) return FA_ERR_PAGED;
    if (!c->table || !c->lens) return FA_ERR_BAD_ARG;
    if (!aligned(c->table, 4) || !aligned(c->lens, 4)) return FA_ERR_ALIGNMENT;
    if (c->B > 1 && c->table_stride < c->table_pages) return FA_ERR_BAD_ARG;
    const int extent[3] = {c->pages, c->page_size, c->Hk};
    int rc = check_strides(c->k, c->k_stride, extent, 3);
    return rc ? rc : check_strides(c->v, c->v_stride, extent, 3);
}

// The scales of a cache of 8 bits, and what such a cache asks for besides; without any, nothing.
int check_scales(const fa_paged_cache* c, const fa_paged_more* more) {
    if (!more->k_scales && !more->v_scales) return FA_OK;
    if (!more->k_scales || !more->v_scales) return FA_ERR_BAD_ARG;
    if (c->page_size < 16) return FA_ERR_PAGED;
    const int extent[3] = {c->pages, c->page_size, c->Hk};
    for (int i = 0; i < 3; ++i)
        if (extent[i] > 1 && (c->k_stride[i] % 16 != 0 || c->v_stride[i] % 16 != 0)) return FA_ERR_ALIGNMENT;
    const int64_t strides[4] = {more->k_scale_stride[0], more->k_scale_stride[1], more->v_scale_stride[0], more->v_scale_stride[1]};
    for (int i = 0; i < 4; ++i)
        if ((i % 2 ? c->Hk : c->pages) > 1 && (strides[i] <= 0 || strides[i] % 16 != 0)) return FA_ERR_ALIGNMENT;
    return aligned(more->k_scales, 16) && aligned(more->v_scales, 16) ? FA_OK : FA_ERR_ALIGNMENT;
}

void fill_scales(fa::PagedParams* p, const fa_paged_cache* c, const fa_paged_more* more) {
    p->k_scales = more->k_scales;
    p->v_scales = more->v_scales;
    p->k_scale_p = c->pages > 1 ? more->k_scale_stride[0] : 0;
    p->k_scale_h = c->Hk > 1 ? more->k_scale_stride[1] : 0;
    p->v_scale_p = c->pages > 1 ? more->v_scale_stride[0] : 0;
    p->v_scale_h = c->Hk > 1 ? more->v_scale_stride[1] : 0;
}

int check_rows(const fa_rows* r, int T, int H) {
    if (!r) return FA_ERR_BAD_ARG;
    const int extent[2] = {T, H};
    return check_strides(r->ptr, r->stride, extent, 2);
}

int fill_params(fa::PagedParams* p, const fa_paged_cache* c, int T, const int32_t* starts, int32_t* status) {
    if (T <= 0 || T > kMostTokens || !status || (!starts && T != c->B)) return FA_ERR_BAD_ARG;
    if (!aligned(starts, 4)) return FA_ERR_ALIGNMENT;
    p->table = c->table;
    p->table_stride = c->B > 1 ? c->table_stride : 0;
    p->lens = c->lens;
    p->starts = starts;
    p->B = c->B;
    p->T = T;
    p->Hk = c->Hk;
    p->D = c->D;
    p->page = c->page_size;
    while ((1 << p->log2_page) < c->page_size) ++p->log2_page;
    p->n_pages = c->pages;
    p->capacity = c->table_pages * c->page_size;
    p->status = status;
    p->wait_limit = fa::wait_limit_clocks();
    return FA_OK;
}

// 4-D map with 64 columns a box and a 128-byte swizzle; extents, strides (elements, of the last three) and box, innermost first
int map4(CUtensorMap* out, int dtype, const void* ptr, int D, const int (&extent)[3], const int64_t (&stride)[3], const int (&box)[3]) {
    const fa::EncodeFn fn = fa::encode_fn();
    if (!fn) return FA_ERR_NO_DRIVER;
    const cuuint64_t dims[4] = {cuuint64_t(D), cuuint64_t(extent[0]), cuuint64_t(extent[1]), cuuint64_t(extent[2])};
    cuuint64_t bytes[3];
    for (int i = 0; i < 3; ++i) bytes[i] = cuuint64_t(extent[i] > 1 ? stride[i] : D < 8 ? 8 : D) * 2;  // an extent of 1 may carry any stride
    const cuuint32_t b[4] = {64, cuuint32_t(box[0]), cuuint32_t(box[1]), cuuint32_t(box[2])}, step[4] = {1, 1, 1, 1};
    const CUresult r = fn(out, dtype == FA_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(ptr), dims, bytes,
                          b, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? FA_OK : FA_ERR_TENSORMAP;
}

// The same over a cache of 8 bits: whole rows of 64 or 128 bytes, with that swizzle
int map_bytes(CUtensorMap* out, const void* ptr, int D, const int (&extent)[3], const int64_t (&stride)[3], int rows) {
    const fa::EncodeFn fn = fa::encode_fn();
    if (!fn) return FA_ERR_NO_DRIVER;
    const cuuint64_t dims[4] = {cuuint64_t(D), cuuint64_t(extent[0]), cuuint64_t(extent[1]), cuuint64_t(extent[2])};
    cuuint64_t bytes[3];
    for (int i = 0; i < 3; ++i) bytes[i] = cuuint64_t(extent[i] > 1 ? stride[i] : D);  // an extent of 1 may carry any stride
    const cuuint32_t b[4] = {D > 64 ? 128u : 64u, 1, cuuint32_t(rows), 1}, step[4] = {1, 1, 1, 1};
    const CUresult r = fn(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void*>(ptr), dims, bytes, b, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          D > 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? FA_OK : FA_ERR_TENSORMAP;
}

// fp32 rows and log-sum-exps of two pieces for each worker, and what is merged from which
size_t workspace_bytes(int D, int workers) {
    return size_t(2) * workers * fa::kBlk * ((D > 64 ? 128 : 64) + 1) * sizeof(float) + workers * sizeof(int4);
}

// fa_debug_paged_pieces and fa_debug_paged_pieces_more
template <bool MASKED>
int debug_pieces(int32_t B, int32_t T, int32_t Hk, int32_t G, int32_t capacity, const int32_t* lens, const int32_t* starts, const int32_t* prefix,
                 fa_window window, const int32_t* parents, int32_t most_workers, int32_t* rows, int32_t most_rows) {
    if (B <= 0 || T < 0 || Hk <= 0 || G <= 0 || G > fa::kBlk || capacity <= 0 || !lens || most_workers <= 0 || !rows) return -1;
    fa::PagedParams p{};
    p.lens = lens;
    p.starts = starts;
    p.prefix = prefix;
    p.B = B;
    p.T = T;
    p.Hk = Hk;
    p.G = G;
    p.tokens = fa::kBlk / G;
    p.capacity = capacity;
    p.window = window.keys;
    p.sinks = window.sinks;
    p.parents = parents;
    fa::PagedPlan plan;
    plan.group = fa::paged_group(B);
    const int entries = fa::paged_entries(B);
    long long weight = 0, items = 0;
    int longest = 0;
    auto each = [&](int g, auto add) {
        for (int b = g * plan.group; b < B && b < (g + 1) * plan.group; ++b) add(fa::paged_seq<MASKED>(p, b));
    };
    for (int g = 0; g < entries; ++g)
        each(g, [&](const fa::PagedSeq& s) {
            weight += Hk * fa::paged_weight<MASKED>(p, s, s.tiles, true);
            items += (long long)Hk * s.tiles;
            if (s.tiles > 0) longest = std::max(longest, MASKED ? fa::paged_keys<MASKED>(p, s, s.tiles - 1) : s.len);
        });
    fa::paged_share_out(plan, weight, items, longest, most_workers);
    if (plan.workers > 1023) return -1;
    long long before = 0;
    for (int g = 0; g < entries; ++g) {
        plan.sums[g] = before;
        each(g, [&](const fa::PagedSeq& s) { before += Hk * fa::paged_weight<MASKED>(p, s, s.tiles, plan.keyed); });
    }
    int n = 0;
    auto put = [&](int a, int b, int c, int d, int e, int f, int g, int h) {
        const int32_t row[8] = {a, b, c, d, e, f, g, h};
        if (n < most_rows)
            for (int i = 0; i < 8; ++i) rows[8 * n + i] = row[i];
        ++n;
    };
    for (int w = 0; w < plan.workers; ++w) {
        bool first = true;
        fa::paged_stretch<MASKED>(p, plan, w, [&](const fa::PagedWalk<MASKED>& k, int tiles, int lo, int hi, int part) {
            put(w, k.b, k.hk, k.tile, lo, hi, tiles, part);
            if (first && fa::paged_first_cut(plan, w, k)) {
                int from;
                const int pieces = fa::paged_pieces(p, plan, w, k, from);
                for (int i = 0; pieces > 1 && i < pieces; ++i) put(-1, k.b, k.hk, k.tile, 0, 0, 0, 2 * (from + i) + (i == 0));
            }
            first = false;
            return true;
        });
    }
    return n;
}

}  // namespace

extern "C" {

int fa_paged_append(const fa_paged_cache* cache, int32_t T, const int32_t* starts, const fa_rows* k, const fa_rows* v, int32_t* status, void* stream) {
    return fa_paged_append_more(cache, nullptr, T, starts, k, v, status, stream);
}

int fa_paged_append_more(const fa_paged_cache* cache, const fa_paged_more* more, int32_t T, const int32_t* starts, const fa_rows* k, const fa_rows* v, int32_t* status,
                         void* stream) {
    int rc = check_cache(cache);
    if (!rc && more) rc = check_scales(cache, more);
    if (rc) return rc;
    if ((rc = check_rows(k, T, cache->Hk)) || (rc = check_rows(v, T, cache->Hk))) return rc;
    fa::PagedParams p{};
    if ((rc = fill_params(&p, cache, T, starts, status))) return rc;
    if (more && more->k_scales) {
        fill_scales(&p, cache, more);
        const int64_t strides[10] = {k->stride[0] / 8, k->stride[1] / 8, v->stride[0] / 8, v->stride[1] / 8, cache->k_stride[0], cache->k_stride[1], cache->k_stride[2],
                                     cache->v_stride[0], cache->v_stride[1], cache->v_stride[2]};
        return fa::launch_paged_append_e4m3(cache->dtype == FA_BF16, p, k->ptr, v->ptr, cache->k, cache->v, more->k_scales, more->v_scales, strides,
                                            static_cast<cudaStream_t>(stream)) == cudaSuccess ? FA_OK : FA_ERR_LAUNCH;
    }
    const int64_t strides[10] = {k->stride[0] / 8, k->stride[1] / 8, v->stride[0] / 8, v->stride[1] / 8,
                                 cache->k_stride[0] / 8, cache->k_stride[1] / 8, cache->k_stride[2] / 8,
                                 cache->v_stride[0] / 8, cache->v_stride[1] / 8, cache->v_stride[2] / 8};
    return fa::launch_paged_append(p, k->ptr, v->ptr, cache->k, cache->v, strides, static_cast<cudaStream_t>(stream)) == cudaSuccess ? FA_OK : FA_ERR_LAUNCH;
}

int fa_paged_workspace_bytes(const fa_paged_cache* cache, size_t* bytes) {
    if (!bytes) return FA_ERR_BAD_ARG;
    const int rc = check_cache(cache);
    if (rc) return rc;
    const int sms = fa::sm_count();
    if (sms <= 0) return FA_ERR_LAUNCH;
    *bytes = workspace_bytes(cache->D, sms);
    return FA_OK;
}

int fa_paged_fwd_more(const fa_paged_cache* cache, const fa_paged_more* more, int32_t T, int32_t H, const int32_t* starts, float sm_scale,
                      const fa_scores* scores, const fa_rows* q, const fa_rows* o, int32_t fill, void* workspace, size_t bytes, int32_t* status, void* stream) {
    int rc = check_cache(cache);
    if (rc) return rc;
    if (H <= 0 || H % cache->Hk != 0) return FA_ERR_BAD_ARG;
    const int G = H / cache->Hk;
    if (G > fa::kBlk || !(sm_scale > 0.f)) return FA_ERR_UNSUPPORTED;
    if ((rc = check_rows(q, T, H)) || (rc = check_rows(o, T, H))) return rc;
    const fa_scores none{};
    const fa_scores* sc = scores ? scores : &none;
    if (sc->softcap != 0.f && !(sc->softcap >= 1e-6f && sc->softcap <= 1e6f)) return FA_ERR_SCORES;
    const fa_paged_more nothing{};
    if (!more) more = &nothing;
    const fa_window window = more->window;
    if (window.keys < 0 || window.sinks < 0 || (window.keys == 0 && window.sinks > 0) || (more->parents && (sc->slopes || sc->prefix))) return FA_ERR_SCORES;
    if (!aligned(more->parents, 4)) return FA_ERR_ALIGNMENT;
    if ((rc = check_scales(cache, more))) return rc;
    if (!aligned(sc->slopes, 4) || !aligned(sc->prefix, 4) || !aligned(workspace, 16)) return FA_ERR_ALIGNMENT;
    fa::PagedParams p{};
    if ((rc = fill_params(&p, cache, T, starts, status))) return rc;
    const int sms = fa::sm_count();
    if (sms <= 0) return FA_ERR_LAUNCH;
    if (!workspace || bytes < workspace_bytes(cache->D, sms)) return FA_ERR_PLAN_SIZE;
    p.prefix = sc->prefix;
    p.window = std::min(window.keys, kMostTokens + 1);  // (no token is further away)
    p.sinks = std::min(window.sinks, kMostTokens + 1);
    p.parents = more->parents;
    fill_scales(&p, cache, more);
    p.out = o->ptr;
    p.out_t = o->stride[0];
    p.out_h = o->stride[1];
    p.part_o = static_cast<float*>(workspace);
    p.part_lse = p.part_o + size_t(2) * sms * fa::kBlk * (cache->D > 64 ? 128 : 64);
    p.merge = reinterpret_cast<int4*>(p.part_lse + size_t(2) * sms * fa::kBlk);
    p.H = H;
    p.G = G;
    p.tokens = fa::kBlk / G;
    p.narrow = 32 / G;
    p.fill = fill ? 1 : 0;
    p.lift = 1.f;
    if (p.k_scales && cache->dtype == FA_BF16) {  // (the squares of the scores that a cap takes stay in fp32's range, however large q and small the scale)
        int n = 0;
        frexpf(sm_scale, &n);
        n = n > 120 ? 120 : n < -120 ? -120 : n < 20 && n > -20 ? 0 : n;
        p.lift = ldexpf(1.f, n);
        sm_scale = ldexpf(sm_scale, -n);
    }
    p.scale_log2 = sm_scale * fa::kScoreLog2e;
    p.score = fa::make_score_args(sc->softcap, sc->slopes, sc->prefix != nullptr, sm_scale);
    const int box_rows = cache->page_size < fa::kBlk ? cache->page_size : fa::kBlk;
    CUtensorMap tq, tk, tv;
    if ((rc = map4(&tq, cache->dtype, q->ptr, cache->D, {G, cache->Hk, T}, {q->stride[1], q->stride[1] * G, q->stride[0]}, {G, 1, p.tokens}))) return rc;
    CUtensorMap tn;  // of the rows of 32 / G tokens
    if ((rc = map4(&tn, cache->dtype, q->ptr, cache->D, {G, cache->Hk, T}, {q->stride[1], q->stride[1] * G, q->stride[0]}, {G, 1, p.narrow > 0 ? p.narrow : p.tokens}))) return rc;
    if (p.k_scales) {
        if ((rc = map_bytes(&tk, cache->k, cache->D, {cache->Hk, cache->page_size, cache->pages}, {cache->k_stride[2], cache->k_stride[1], cache->k_stride[0]}, box_rows))) return rc;
        if ((rc = map_bytes(&tv, cache->v, cache->D, {cache->Hk, cache->page_size, cache->pages}, {cache->v_stride[2], cache->v_stride[1], cache->v_stride[0]}, box_rows))) return rc;
        return fa::launch_paged_fwd(cache->dtype == FA_BF16, tq, tn, tk, tv, p, sms, static_cast<cudaStream_t>(stream)) == cudaSuccess ? FA_OK : FA_ERR_LAUNCH;
    }
    if ((rc = map4(&tk, cache->dtype, cache->k, cache->D, {cache->Hk, cache->page_size, cache->pages},
                   {cache->k_stride[2], cache->k_stride[1], cache->k_stride[0]}, {1, box_rows, 1}))) return rc;
    if ((rc = map4(&tv, cache->dtype, cache->v, cache->D, {cache->Hk, cache->page_size, cache->pages},
                   {cache->v_stride[2], cache->v_stride[1], cache->v_stride[0]}, {1, box_rows, 1}))) return rc;
    return fa::launch_paged_fwd(cache->dtype == FA_BF16, tq, tn, tk, tv, p, sms, static_cast<cudaStream_t>(stream)) == cudaSuccess ? FA_OK : FA_ERR_LAUNCH;
}

int fa_paged_fwd(const fa_paged_cache* cache, int32_t T, int32_t H, const int32_t* starts, float sm_scale, const fa_scores* scores, const fa_rows* q,
                 const fa_rows* o, int32_t fill, void* workspace, size_t bytes, int32_t* status, void* stream) {
    return fa_paged_fwd_more(cache, nullptr, T, H, starts, sm_scale, scores, q, o, fill, workspace, bytes, status, stream);
}

int fa_debug_paged_pieces(int32_t B, int32_t T, int32_t Hk, int32_t G, int32_t capacity, const int32_t* lens, const int32_t* starts, const int32_t* prefix,
                          int32_t most_workers, int32_t* rows, int32_t most_rows) {
    return debug_pieces<false>(B, T, Hk, G, capacity, lens, starts, prefix, fa_window{}, nullptr, most_workers, rows, most_rows);
}

int fa_debug_paged_pieces_more(int32_t B, int32_t T, int32_t Hk, int32_t G, int32_t capacity, const int32_t* lens, const int32_t* starts, const int32_t* prefix,
                               const fa_window* window, const int32_t* parents, int32_t most_workers, int32_t* rows, int32_t most_rows) {
    return debug_pieces<true>(B, T, Hk, G, capacity, lens, starts, prefix, window ? *window : fa_window{}, parents, most_workers, rows, most_rows);
}

}  // extern "C"
