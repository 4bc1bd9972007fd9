/*
 * C ABI of the B200 (sm_100a) document-masked flash-attention library.
 *
 * The library replaces the four Triton launches of the reference operator
 * (flash_triton.py:541 `_fwd_kernel`, :585 `_bwd_preprocess`, :596 `_bwd_kv_kernel`,
 * :617 `_bwd_q_kernel`) and adds the mask plan (per-block id ranges, no counterpart in the
 * reference: README.md:18 lists block sparsity as not implemented).
 *
 * Conventions
 *  - every pointer is a device pointer of the current CUDA device unless stated otherwise;
 *  - tensors are [B, H, L, D] with ELEMENT strides; the last stride must be 1, the other
 *    strides multiples of 8 elements and the base 16-byte aligned (TMA rules);
 *  - lse, delta and plan buffers must be 16-byte aligned (the kernels read them with bulk copies
 *    and 16-byte loads); a misaligned buffer is refused with FA_ERR_ALIGNMENT;
 *  - the caller owns every buffer;
 *  - every function enqueues on `stream` and returns without synchronising;
 *  - return value 0 = ok, otherwise an FA_ERR_* code (fa_error_string() describes it);
 *  - `status` is one int32 in device memory, zeroed by the caller. Kernels write a non-zero
 *    code there when a bounded wait ran out (100..199), an id was out of range (200), or a page or
 *    a length of a paged cache or the parent of a drafted token was (201, 202, 203). The first code stays, but a time-out takes the place
 *    of the others. A time-out code is sticky: while the word holds one, every later
 *    fa_fwd / fa_bwd_dkdv / fa_bwd_dq / fa_paged_fwd launch given that word computes nothing and fills its
 *    outputs (o; dk, dv; dq) with NaN, until the host has read the word and set it back to 0.
 *    The outputs of the launch in which the wait ran out are undefined. Codes from 200 on only concern
 *    the call that they come from (with 200, its result may mask that query wrongly); later calls run.
 *  - one bounded wait lasts at most 5e8 SM clocks (about 0.25 s); the environment variable
 *    FA_B200_WAIT_LIMIT_CLOCKS (>= 10000), read when the library is first used, replaces the limit,
 *    e.g. on hosts where several contexts time-share the GPU. The scheduler of a kernel waits for as
 *    long as one of its work items takes (up to 1024 tiles of 128 x 128, in fa_bwd_dkdv for each head
 *    of a group, some 3000 clocks each): a limit below that can end valid calls.
 */
#ifndef FA_B200_H_
#define FA_B200_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define FA_VERSION 1

/* Head dims 16, 32, 64 and 128 (flash_triton.py:512). FA_BF16 / FA_FP16 run on tensor-core kernels built for 64
 * and 128 columns; with head dims 16 and 32 the 64-wide kernels read the tensors through TMA maps of the real
 * head dim, which fill the missing columns with zeros and never write them (no padded copies anywhere).
 * FA_FP32 tensors (4-byte aligned base, last stride 1, any positive other strides) take fp32 FMA kernels
 * (testing.py:158): exact to fp32 rounding, not fast. */
enum fa_dtype { FA_BF16 = 0, FA_FP16 = 1, FA_FP32 = 2 };
enum fa_id_dtype { FA_ID_NONE = 0, FA_ID_INT32 = 1, FA_ID_INT64 = 2 };
/* score_func_mode of the reference (flash_triton.py:20-22) */
enum fa_mode { FA_MODE0_NOPE = 0, FA_MODE1_DOC = 1 };

enum fa_error {
    FA_OK = 0,
    FA_ERR_BAD_ARG = 1,      /* null pointer, non-positive size, unknown enum */
    FA_ERR_UNSUPPORTED = 2,  /* head dim not in {16,32,64,128}, unknown dtype, sm_scale <= 0 */
    FA_ERR_ALIGNMENT = 3,    /* a base address or stride breaks the TMA 16-byte rules */
    FA_ERR_TENSORMAP = 4,    /* the driver refused to encode a tensor map */
    FA_ERR_LAUNCH = 5,       /* kernel launch failed (cudaGetLastError) */
    FA_ERR_PLAN_SIZE = 6,    /* plan buffer too small / missing for FA_MODE1_DOC, or workspace of a split forward */
    FA_ERR_NO_DRIVER = 7,    /* cuTensorMapEncodeTiled could not be resolved */
    FA_ERR_SCRATCH_LIMIT = 8, /* fa_fwd_static_plan: the plan does not fit in FA_STATIC_PLAN_BYTES */
    FA_ERR_SCORES = 9,       /* fa_scores: softcap neither 0 nor within 1e-6 .. 1e6, or a prefix or a window without a causal mask, or
                              sinks without a window */
    FA_ERR_PAGED = 10        /* fa_paged_cache: page size not a power of two from 8 on, or sizes beyond what the kernels count */
};

typedef struct fa_problem {
    int32_t B, H, Hk; /* batch, query heads, key/value heads (H % Hk == 0) */
    int32_t M, N, D;  /* query length, key length, head dim */
    int32_t dtype;    /* enum fa_dtype, of q/k/v/o and all gradients */
    int32_t causal;   /* bottom-right aligned: query i sees key j iff j <= i + max(0, N-M) */
    int32_t mode;     /* enum fa_mode */
    int32_t id_heads; /* head extent of the id tensors as stored in the plan: 1 (broadcast) or H */
    float sm_scale;   /* > 0 */
} fa_problem;

typedef struct fa_tensor {
    void* ptr;
    int64_t stride[4]; /* elements, order [B, H, L, D] */
} fa_tensor;

typedef struct fa_ids {
    const void* ptr;
    int64_t stride[3]; /* elements, order [B, H, L]; any value incl. 0 */
    int32_t dtype;     /* enum fa_id_dtype */
} fa_ids;

int fa_version(void);
const char* fa_error_string(int code);

/* Rows of the internal per-row fp32 buffers (log-sum-exp, delta): M rounded up to 128. */
int64_t fa_padded_rows(int32_t M);

/* Size in bytes of the mask plan for this problem (when mode == FA_MODE0_NOPE: 512 bytes, the work
 * counters of the attention kernels only; such a plan is optional). */
int fa_plan_bytes(const fa_problem* p, size_t* bytes);

/* 1 if a plan would gain the launches for this problem nothing: no ids, and no launch (with `backward` != 0, of the
 * backward too) has more items than the current device has SMs. The runs of a split forward are not counted: there are
 * at most two per SM if fa_fwd_splits set their number, all nearly as long, and dealing them out in a fixed order takes
 * no longer than through a plan's counters. Results are the same bits with and without a plan. */
int fa_plan_optional(const fa_problem* p, int32_t backward);

/* With ids fa_plan_build launches one kernel for at most this many blocks of 128 queries and of 128
 * keys together, else three. */
#define FA_PLAN_ONE_KERNEL_BLOCKS 64

/* Builds the mask plan from eq [B,H,M] / ek [B,H,N]: 32-bit id codes, per-128-block id
 * min/max, per-block ranges of blocks that hold at least one unmasked entry, and a few work
 * counters through which the CTAs of fa_fwd / fa_bwd_dkdv / fa_bwd_dq share out their work.
 * The attention kernels update those counters (although they take the plan as `const void*`) and
 * leave them zero, so a plan can be used any number of times, but only by one launch of each of
 * the three at a time.
 * Mask rule (flash_triton.py:114, README.md:16): keep = (eq >= 0) | (eq == ek). */
int fa_plan_build(const fa_problem* p, const fa_ids* eq, const fa_ids* ek, void* plan, size_t plan_bytes,
                  int32_t* status, void* stream);

/* Launches. The kernels are launched programmatically, but for the debug entry points' and that of a separate fa_bwd_dq: a kernel sets
 * itself up while the one before it in the stream ends, and waits for that one's end before it reads or writes memory. The one exception
 * is the dQ kernel of fa_bwd, which reads, takes work from the plan's counters and writes dq beside the dK/dV kernel and waits for it
 * only at its end (see fa_bwd for what may not share memory). What comes after a call in its stream finds the call's results complete; a
 * programmatic kernel of the caller's does so behind its own wait (griddepcontrol.wait). */

/* Forward (replaces flash_triton.py:541). o has q's shape; lse is [B, H, fa_padded_rows(M)] fp32,
 * log2-domain log-sum-exp of the scaled scores (flash_triton.py:133), -inf for a row with no
 * unmasked key (whose output row is 0). plan may be NULL when mode == FA_MODE0_NOPE (here and in
 * the backward entry points): the CTAs then share out their work in a fixed order instead of through
 * the plan's counters, which costs a few percent when the work per block is uneven. */
int fa_fwd(const fa_problem* p, const fa_tensor* q, const fa_tensor* k, const fa_tensor* v,
           const fa_tensor* o, float* lse, const void* plan, int32_t* status, void* stream);

/* The same forward for calls without ids (mode 0, 16-bit types) that are too few to fill the GPU, a decoded token or
 * a short block of queries against long keys: the keys of each query block are cut into `splits` runs that
 * different SMs work on, their fp32 results go to `workspace` (16-byte aligned, at least fa_fwd_workspace_bytes)
 * and a second kernel merges them. fa_fwd_splits returns the number that pays on the current device (1: call
 * fa_fwd, or pass splits = 1 and no workspace); more than one per 128 keys is refused, as is any splitting of other
 * calls (FA_ERR_UNSUPPORTED). The workspace is free again when the launches are done. */
int fa_fwd_splits(const fa_problem* p);
int fa_fwd_workspace_bytes(const fa_problem* p, int32_t splits, size_t* bytes);
int fa_fwd_split(const fa_problem* p, const fa_tensor* q, const fa_tensor* k, const fa_tensor* v, const fa_tensor* o,
                 float* lse, const void* plan, int32_t splits, void* workspace, size_t workspace_bytes, int32_t* status,
                 void* stream);

/* delta[b,h,i] = sum_d o*do in fp32 (replaces flash_triton.py:585); delta is
 * [B, H, fa_padded_rows(M)], padding rows are written as 0. */
int fa_bwd_delta(const fa_problem* p, const fa_tensor* o, const fa_tensor* d_o, float* delta, void* stream);

/* dK, dV [B, Hk, N, D] (replaces flash_triton.py:596 and the group sum at :635-637; the sum
 * over the query heads of a group is accumulated in fp32 inside the kernel). */
int fa_bwd_dkdv(const fa_problem* p, const fa_tensor* q, const fa_tensor* k, const fa_tensor* v,
                const fa_tensor* d_o, const float* lse, const float* delta, const fa_tensor* dk,
                const fa_tensor* dv, const void* plan, int32_t* status, void* stream);

/* dQ [B, H, M, D] (replaces flash_triton.py:617). */
int fa_bwd_dq(const fa_problem* p, const fa_tensor* q, const fa_tensor* k, const fa_tensor* v,
              const fa_tensor* d_o, const float* lse, const float* delta, const fa_tensor* dq,
              const void* plan, int32_t* status, void* stream);

/* fa_bwd_delta, fa_bwd_dkdv and fa_bwd_dq in this order; stops at the first that fails. The dQ kernel is launched so
 * that it may run on SMs that the dK/dV kernel has left, or (fp32) beside its blocks; it ends after it. So dq, dk and dv must share no
 * memory with one another, nor with q, k, v, d_o, lse, delta or the plan (the three calls one by one ask that of the
 * tensors of each call only). */
int fa_bwd(const fa_problem* p, const fa_tensor* q, const fa_tensor* k, const fa_tensor* v, const fa_tensor* o,
           const fa_tensor* d_o, const float* lse, float* delta, const fa_tensor* dq, const fa_tensor* dk,
           const fa_tensor* dv, const void* plan, int32_t* status, void* stream);

/* attention_scored: what is done to a scaled score s_ij = sm_scale q_i . k_j before the softmax (no counterpart in the reference):
 *   x_ij = softcap * tanh(s_ij / softcap) - slopes[h] * |i + gap - j|,   gap = max(0, N - M);
 * and, with a causal mask, prefix[b] leading keys that it leaves visible to every query of sequence b (values are taken into [0, N]; the
 * ids' rule holds for those keys as for the others). softcap 0, slopes NULL, prefix NULL: without that part. There are no gradients for
 * the three. */
typedef struct fa_scores {
    float softcap;         /* 0, or 1e-6 .. 1e6 */
    const float* slopes;   /* [H], device */
    const int32_t* prefix; /* [B], device; needs p->causal */
} fa_scores;

/* fa_plan_build, fa_fwd_split (splits = 1: fa_fwd) and fa_bwd of a call with such scores: the same arguments and rules. The plan of a call
 * with ids must have been built with the same prefix; without ids fa_plan_build's will do. With M <= 64 and no ids the heads of a group share
 * tiles and fa_fwd_splits says into how many runs the keys are best cut, as for fa_fwd_split.
 * rest: NULL, or (16-bit types, some change of the scores, splits = 1) a contiguous [B, H, M, D] buffer of the type, 16-byte aligned, that the forward fills with
 * what the rounding of o has left out and the backward adds to it: dq and dk are then as exact as their own rounding lets them also where a few
 * keys carry a row. */
int fa_plan_build_scored(const fa_problem* p, const fa_scores* scores, const fa_ids* eq, const fa_ids* ek, void* plan, size_t plan_bytes,
                         int32_t* status, void* stream);
int fa_fwd_scored(const fa_problem* p, const fa_scores* scores, const fa_tensor* q, const fa_tensor* k, const fa_tensor* v, const fa_tensor* o, void* rest,
                  float* lse, const void* plan, int32_t splits, void* workspace, size_t workspace_bytes, int32_t* status, void* stream);
/* The same rest of a forward that fa_fwd_scored has cut into splits > 1 runs, from the workspace that it has left, by a kernel of its own. */
int fa_fwd_rest(const fa_problem* p, int32_t splits, const void* workspace, size_t workspace_bytes, void* rest, int32_t* status, void* stream);
int fa_bwd_scored(const fa_problem* p, const fa_scores* scores, const fa_tensor* q, const fa_tensor* k, const fa_tensor* v, const fa_tensor* o,
                  const void* rest, const fa_tensor* d_o, const float* lse, float* delta, const fa_tensor* dq, const fa_tensor* dk, const fa_tensor* dv,
                  const void* plan, int32_t* status, void* stream);

/* A sliding window, and the first tokens that it leaves visible: with a causal mask, query i sees the keys j <= i + gap with i + gap - j < keys or
 * j < sinks, besides those that a prefix shows it; the ids' rule holds on top. keys 0: none. */
typedef struct fa_window {
    int32_t keys;
    int32_t sinks;
} fa_window;

/* The four of a call with a window (scores may be NULL, window NULL or of 0 keys is a call without one). The plan of a call with ids must have been built with the
 * same window; fa_fwd_splits_windowed says into how many runs the keys that are left are best cut (in a call with a prefix, which may
 * show any of the others, ask it with window NULL); fa_fwd_rest serves these forwards, too. */
int fa_plan_build_windowed(const fa_problem* p, const fa_scores* scores, const fa_window* window, const fa_ids* eq, const fa_ids* ek, void* plan,
                           size_t plan_bytes, int32_t* status, void* stream);
int fa_fwd_splits_windowed(const fa_problem* p, const fa_window* window);
int fa_fwd_windowed(const fa_problem* p, const fa_scores* scores, const fa_window* window, const fa_tensor* q, const fa_tensor* k, const fa_tensor* v,
                    const fa_tensor* o, void* rest, float* lse, const void* plan, int32_t splits, void* workspace, size_t workspace_bytes, int32_t* status,
                    void* stream);
int fa_bwd_windowed(const fa_problem* p, const fa_scores* scores, const fa_window* window, const fa_tensor* q, const fa_tensor* k, const fa_tensor* v,
                    const fa_tensor* o, const void* rest, const fa_tensor* d_o, const float* lse, float* delta, const fa_tensor* dq, const fa_tensor* dk,
                    const fa_tensor* dv, const void* plan, void* workspace, size_t workspace_bytes, int32_t* status, void* stream);
/* What fa_bwd_windowed needs as its workspace (16-byte aligned; 0: none, and NULL will do): with first keys that all queries see, fp32 sums of runs of queries. */
int fa_bwd_workspace_bytes(const fa_problem* p, const fa_window* window, size_t* bytes);

/* A cache of keys and values in pages, for serving (no counterpart in the reference). k and v are [pages, page_size, Hk, D], 16-bit, with 16-byte
 * aligned bases, last stride 1 and other strides multiples of 8 elements. Sequence b's tokens lie, page_size at a time, in the pages
 * table[b * table_stride + i], i = 0 .. ; lens[b] is how many tokens it has. table and lens are device memory, read when the kernels run.
 * Entries of the table behind a sequence's last page are not read. page_size: a power of two, at least 8; table_pages * page_size <= 2^22.
 *
 * New tokens: rows [T, heads, D]. starts [B + 1], non-decreasing: sequence b has the rows from starts[b] to starts[b + 1]; they are its last
 * ones, at the positions lens[b] - n .. lens[b] - 1, so that lens counts them. starts NULL: T == B and every sequence has one new token.
 * Rows before starts[0] and from starts[B] on belong to no sequence. A page number outside [0, pages) or a length outside
 * [0, table_pages * page_size] sets status 201 or 202; nothing outside the tensors is read or written, the results of that sequence are
 * undefined, and later calls run. */
typedef struct fa_paged_cache {
    int32_t B, Hk, D, dtype;          /* sequences; kv heads; head dim 16, 32, 64 or 128; FA_BF16 or FA_FP16 */
    int32_t pages, page_size, table_pages; /* table_pages: entries of a sequence's row of the table */
    const int32_t* table;
    int64_t table_stride;
    const int32_t* lens;
    void* k;
    void* v;
    int64_t k_stride[3], v_stride[3]; /* elements: page, slot, head */
} fa_paged_cache;

typedef struct fa_rows {
    void* ptr;
    int64_t stride[2]; /* elements: token, head */
} fa_rows;

/* Copies new tokens' k and v, [T, Hk, D], to their places in the pages. Rows of no sequence, and new tokens in front of position 0 (more new
 * ones than lens says there are), are left out. Two tokens at one place (a page that two sequences name): either's values may stay. */
int fa_paged_append(const fa_paged_cache* cache, int32_t T, const int32_t* starts, const fa_rows* k, const fa_rows* v, int32_t* status, void* stream);

/* o[t] = softmax(scores of row t with the keys it sees) V, for new tokens q [T, H, D] whose own keys are in the cache already. A token at position p
 * sees the keys j <= p and, with scores->prefix, j < prefix[b], of its sequence (scores may be NULL; i + gap in fa_scores is the position). H / Hk at most 128. A row that sees no key, or is at a position below 0, gets zeros. Rows of no
 * sequence are set to 0 where `fill` is not 0 and else left as they are. o may not overlap q or the cache. Two kernels; `workspace`: 16-byte
 * aligned, at least fa_paged_workspace_bytes, which goes by the head dim and the current device alone; free again when the launches are done.
 * How the work is cut depends on all lengths of the batch, so the last bits of a sequence's result can differ with what it is batched with. */
int fa_paged_workspace_bytes(const fa_paged_cache* cache, size_t* bytes);
int fa_paged_fwd(const fa_paged_cache* cache, int32_t T, int32_t H, const int32_t* starts, float sm_scale, const fa_scores* scores, const fa_rows* q,
                 const fa_rows* o, int32_t fill, void* workspace, size_t bytes, int32_t* status, void* stream);

/* What attention over a paged cache, and an append, may have besides; NULL, or all zeros: nothing.
 * window: a token at position p sees, of the keys j <= p, those with p - j < window.keys or j < window.sinks. Entries of the table whose pages no token of the call
 *   sees may hold anything.
 * parents [T], device: sequences of up to 256 new tokens have them drafted as a tree. parents[t] is the place, among its sequence's new tokens, of the one that token t
 *   continues, which lies before it, or -1: it continues the cached text. A token then sees the cached text, itself and those on its branch; its position is
 *   that of the text's end and its depth on the branch. Sequences of more new tokens are chunks, whose parents are not read. A parent that does not lie before its
 *   token sets status 203 and counts as -1. Not with slopes or a prefix (FA_ERR_SCORES).
 * k_scales, v_scales [pages, Hk, page_size], device: the cache's k and v are e4m3, a byte each, with strides that are multiples of 16 and a page size of 16 at least; a head's row of a token stands for
 *   its numbers times 2^(byte - 127), bytes from 112 to 134 (others are taken into that range by the attention). Rows and q are of cache->dtype, which the
 *   cache itself does not depend on. An append stores, of a row x, the nearest of e4m3's numbers to x 2^-e (ties to even, 448 at most) with the least e from -15 to 7
 *   for which the largest finite |x| is at most 448 2^e, and a NaN for what is not finite. Where two tokens go to one place their parts may mix.
 *   Scales: 16-byte aligned, last stride 1, other strides multiples of 16. An append takes nothing else from this struct. */
typedef struct fa_paged_more {
    fa_window window;
    const int32_t* parents;
    uint8_t* k_scales; /* an 8-bit cache's (below), or both NULL */
    uint8_t* v_scales;
    int64_t k_scale_stride[2], v_scale_stride[2]; /* bytes: page, head */
} fa_paged_more;
int fa_paged_append_more(const fa_paged_cache* cache, const fa_paged_more* more, int32_t T, const int32_t* starts, const fa_rows* k, const fa_rows* v, int32_t* status,
                         void* stream);
int fa_paged_fwd_more(const fa_paged_cache* cache, const fa_paged_more* more, int32_t T, int32_t H, const int32_t* starts, float sm_scale,
                      const fa_scores* scores, const fa_rows* q, const fa_rows* o, int32_t fill, void* workspace, size_t bytes, int32_t* status, void* stream);

/* Debug: materialise the kernels' decisions. keep is [B, id_heads, M, N] bytes (1 = unmasked),
 * produced by the same device predicate the attention kernels use; tile_class is
 * [B, id_heads, ceil(M/128), ceil(N/128)] bytes: bit0 visited, bit1 bound/causal check,
 * bit2 id check, bit3 query tail, bit4 / bit5 key / query codes of the block are monotone.
 * Either pointer may be NULL. */
int fa_debug_mask(const fa_problem* p, const void* plan, uint8_t* keep, uint8_t* tile_class, void* stream);

/* Size of the plan array built into the library for fa_fwd_static_plan (1 MiB per GPU). It holds
 * the plan of, e.g., one 32768-token sequence with head-broadcast ids (0.27 MB) or a batch of
 * 12 such 4096-token sequences; fa_plan_bytes() tells the size for any problem. */
#define FA_STATIC_PLAN_BYTES (1u << 20)

/* Forward for callers that cannot allocate device memory (no counterpart in the reference, whose
 * launcher allocates with torch, flash_triton.py:539-540). Same result as fa_plan_build + fa_fwd,
 * but the mask plan is built in a fixed FA_STATIC_PLAN_BYTES array inside the library instead of
 * a caller-allocated buffer, and the call allocates nothing. q, k, v, o, lse, eq, ek, status are
 * passed as for the other entry points (eq / ek may be NULL when mode == FA_MODE0_NOPE).
 * Returns FA_ERR_SCRATCH_LIMIT when the plan would not fit. The array is shared by all calls on a
 * GPU: it keeps the previous call's contents (every element read is overwritten first, nothing
 * needs clearing) and calls that overlap on the same GPU race. The first call on a device looks
 * up the array's address; make it before any stream capture on that device (with several contexts on
 * a device, so does a call in another context than the one before). */
int fa_fwd_static_plan(const fa_problem* p, const fa_tensor* q, const fa_tensor* k, const fa_tensor* v,
                       const fa_tensor* o, float* lse, const fa_ids* eq, const fa_ids* ek, int32_t* status,
                       void* stream);

/* Largest query length fa_group_rows sorts (the longer rows in the shared memory of one CTA each). */
#define FA_GROUP_MAX_ROWS 16384

/* Grouping of the queries by id for calls WITHOUT a causal mask, where the order of the query rows is
 * free (no counterpart in the reference, which evaluates every tile whatever the ids,
 * flash_triton.py:94-129). Sorts each id row of eq [B, id_heads, M] by the 32-bit code the mask plan
 * uses for it (ids >= 0 share one code, which sorts last), stable, so rows that are grouped already keep
 * their places. Writes three int32 arrays [B, id_heads, M], contiguous: `order` (grouped position ->
 * caller's position), `inverse` (caller's position -> grouped position) and `grouped_ids` (the ids in
 * grouped order; pass them as the eq of fa_plan_build). p->M <= FA_GROUP_MAX_ROWS, else
 * FA_ERR_UNSUPPORTED. An id below -2^31 sets status 200 as in fa_plan_build. One of the outputs may take the
 * place of a contiguous int32 eq (each row is read before its results are written); other overlaps are not supported. */
int fa_group_rows(const fa_problem* p, const fa_ids* eq, int32_t* order, int32_t* inverse, int32_t* grouped_ids,
                  int32_t* status, void* stream);

/* dst[b, h, i, :] = src[b, h, index[b, he, i], :] for [B, H, M, D] tensors of p->dtype (he = h, or 0 when
 * p->id_heads == 1); index is [B, id_heads, M] int32 with values in [0, M). With `order` it gathers q or dO
 * into the grouped order, with `inverse` it puts o or dQ back. src and dst must not overlap; both need a
 * 16-byte aligned base, last stride 1 and other strides that are whole 16-byte units. */
int fa_permute_rows(const fa_problem* p, const fa_tensor* src, const fa_tensor* dst, const int32_t* index,
                    void* stream);

/* Test hook for the failure path (no counterpart in the reference, which has no failure handling):
 * one warp waits on a barrier nobody arrives at, with the kernels' own bounded wait and a limit of
 * `limit_clocks` SM clocks. The wait gives up, the kernel returns normally and `*status` holds
 * 100 + role (role in 0..97). With a few thousand clocks this takes microseconds; nothing faults,
 * traps or hangs. */
int fa_debug_wait_timeout(int32_t* status, int64_t limit_clocks, int32_t role, void* stream);

/* Host-only helper, no GPU involved: the tile classification the kernels apply to tile
 * (qb, kb) given the id-code min/max of its query block and key block. Returns the tile_class
 * bits of fa_debug_mask. Exposed so that the block-skipping rule can be tested on a CPU
 * (no counterpart in the reference, which never skips a tile). */
uint32_t fa_classify_tile(int32_t M, int32_t N, int32_t causal, int32_t mode, int32_t qb, int32_t kb,
                          int32_t qmin, int32_t qmax, int32_t kmin, int32_t kmax);

/* Host-only helper, no GPU involved: how fa_paged_fwd cuts a batch among `most_workers` blocks, by the kernels' own code; lens, starts and prefix are
 * host memory here. Writes up to most_rows rows of 8 and returns how many there are, or -1: (worker, sequence, kv head, tile of queries, first key tile,
 * last + 1, key tiles of the item, slot of the workspace or -1 for a whole item) for each piece, and (-1, sequence, kv head, tile of queries, 0, 0, 0, slot) for each
 * piece that the second kernel merges. Exposed so that the cutting can be tested on a CPU. */
int fa_debug_paged_pieces(int32_t B, int32_t T, int32_t Hk, int32_t G, int32_t capacity, const int32_t* lens, const int32_t* starts, const int32_t* prefix,
                          int32_t most_workers, int32_t* rows, int32_t most_rows);
/* The same of fa_paged_fwd_more (parents: host memory that is not read, NULL for none); key tiles are counted without those that lie between the first keys and the window. */
int fa_debug_paged_pieces_more(int32_t B, int32_t T, int32_t Hk, int32_t G, int32_t capacity, const int32_t* lens, const int32_t* starts, const int32_t* prefix,
                               const fa_window* window, const int32_t* parents, int32_t most_workers, int32_t* rows, int32_t most_rows);

#ifdef __cplusplus
}
#endif
#endif /* FA_B200_H_ */
