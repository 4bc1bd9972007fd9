"""Serving from a cache of pages: new tokens' keys and values into it (`paged_append`), and the tokens' attention over it (`paged_attention`)."""
import ctypes
import math

import torch

from . import _lib, ops
from .ops import _count, _current, _same_device, _status_word, _stream, check_status
from .scored import _checked_softcap, _checked_slopes, _checked_window, _native, _pointer, _scores

_TYPES = {torch.bfloat16: _lib.FA_BF16, torch.float16: _lib.FA_FP16}
_workspace_bytes = {}  # (device, head dim) -> bytes


def _regular(x, multiple=8):
    """Does the library take the tensor as it is?"""
    return x.stride(-1) == 1 and x.data_ptr() % 16 == 0 and not x.is_neg() and all(
        n == 1 or (s > 0 and s % multiple == 0) for n, s in zip(x.shape[:-1], x.stride()[:-1]))


def _int32(x, shape, name, like):
    if not isinstance(x, torch.Tensor) or x.dtype != torch.int32 or tuple(x.shape) != shape:
        raise ValueError(f"flash_b200: {name} must be an int32 tensor of shape {list(shape)}")
    _same_device(like, **{name: x})
    return x if x.is_contiguous() else x.contiguous()


def _rows(x):
    return _lib.Rows(x.data_ptr(), x.stride()[:2])


def _no_tangents(*tensors):
    """No derivative goes through a cache, forward-mode ones no more than gradients: they are refused, not lost."""
    if ops._forward_ad._current_level >= 0 and any(isinstance(x, torch.Tensor) and ops._forward_ad.unpack_dual(x).tangent is not None for x in tensors):
        raise RuntimeError("flash_b200: there is no forward-mode derivative through a paged cache; call it with the primals")


def _checked(rows, name, k_pages, v_pages, page_table, kv_lens, q_starts, k_scales, v_scales):
    """The cache as the library takes it, what it has besides, its starts, and what has to live as long as they are used."""
    if rows.dim() != 3 or k_pages.dim() != 4 or v_pages.shape != k_pages.shape:
        raise ValueError(f"flash_b200: {name} must be [T, heads, D], k_pages and v_pages [pages, page size, Hk, D]")
    if not rows.is_cuda:
        raise RuntimeError("flash_b200 runs on CUDA tensors only (there is no CPU implementation)")
    if torch.is_grad_enabled() and (rows.requires_grad or k_pages.requires_grad or v_pages.requires_grad):
        raise RuntimeError("flash_b200: there is no gradient through a paged cache; call it under torch.no_grad()")
    pages, page_size, Hk, D = k_pages.shape
    if rows.shape[2] != D or D not in (16, 32, 64, 128):
        raise ValueError(f"flash_b200: the head dim must be 16, 32, 64 or 128 and the cache's, got {rows.shape[2]} and {D}")
    eight, more = k_scales is not None or v_scales is not None, _lib.PagedMore()
    if rows.dtype not in _TYPES or (not eight and (k_pages.dtype != rows.dtype or v_pages.dtype != rows.dtype)):
        raise ValueError(f"flash_b200: a paged cache and its rows are all bf16 or all fp16 (or the cache has scales and is float8_e4m3fn), got {rows.dtype}, {k_pages.dtype}, {v_pages.dtype}")
    _same_device(rows, k_pages=k_pages, v_pages=v_pages)
    for x, n in ((k_pages, "k_pages"), (v_pages, "v_pages")):
        if not _regular(x, 16 if eight else 8):
            raise ValueError(f"flash_b200: {n} needs a 16-byte aligned base, last stride 1 and other strides that are multiples of {16 if eight else 8}")
    if eight:
        if k_pages.dtype != torch.float8_e4m3fn or v_pages.dtype != torch.float8_e4m3fn:
            raise ValueError(f"flash_b200: a paged cache with scales is float8_e4m3fn, got {k_pages.dtype}, {v_pages.dtype}")
        if page_size < 16:
            raise ValueError(f"flash_b200: the page size of a cache with scales must be 16 at least, got {page_size}")
        for x, n in ((k_scales, "k_scales"), (v_scales, "v_scales")):
            if not isinstance(x, torch.Tensor) or x.dtype != torch.float8_e8m0fnu or tuple(x.shape) != (pages, Hk, page_size):
                raise ValueError(f"flash_b200: {n} must be a float8_e8m0fnu tensor of shape [pages, Hk, page size] = {[pages, Hk, page_size]}; k_scales and v_scales go together")
            if not _regular(x, 16):
                raise ValueError(f"flash_b200: {n} needs a 16-byte aligned base, last stride 1 and other strides that are multiples of 16")
        _same_device(rows, k_scales=k_scales, v_scales=v_scales)
        more = _lib.PagedMore(_lib.Window(), None, k_scales.data_ptr(), v_scales.data_ptr(), k_scales.stride()[:2], v_scales.stride()[:2])
    if page_size < 8 or page_size & (page_size - 1):
        raise ValueError(f"flash_b200: the page size must be a power of two from 8 on, got {page_size}")
    if not isinstance(page_table, torch.Tensor) or page_table.dim() != 2 or page_table.shape[1] == 0:
        raise ValueError("flash_b200: page_table must be [sequences, pages of a sequence]")
    B = page_table.shape[0]
    if page_table.dtype != torch.int32:
        raise ValueError("flash_b200: page_table must be int32")
    _same_device(rows, page_table=page_table)
    if page_table.stride(1) != 1 or (B > 1 and page_table.stride(0) < page_table.shape[1]):
        page_table = page_table.contiguous()
    kv_lens = _int32(kv_lens, (B,), "kv_lens", rows)
    if q_starts is None:
        if rows.shape[0] != B:
            raise ValueError(f"flash_b200: without q_starts every sequence has one new token, got {rows.shape[0]} rows for {B} sequences")
    else:
        q_starts = _int32(q_starts, (B + 1,), "q_starts", rows)
    cache = _lib.PagedCache(B, Hk, D, _TYPES[rows.dtype], pages, page_size, page_table.shape[1], page_table.data_ptr(), page_table.stride(0), kv_lens.data_ptr(),
                            k_pages.data_ptr(), v_pages.data_ptr(), k_pages.stride()[:3], v_pages.stride()[:3])
    return cache, more, None if q_starts is None else q_starts.data_ptr(), (page_table, kv_lens, q_starts)


def paged_append(k, v, k_pages, v_pages, page_table, kv_lens, q_starts=None, k_scales=None, v_scales=None):
    """Writes the keys and values of new tokens to their places in a cache of pages, in place.

    k, v: [T, Hk, D], bf16 or fp16. k_pages, v_pages: [pages, page size, Hk, D], page size a power of two from 8 on; token j of sequence b lies in slot
    j % page size of page page_table[b, j // page size] (int32 [B, pages of a sequence]; entries behind a sequence's last page may hold anything).
    kv_lens: int32 [B], how many tokens each sequence has, the new ones among them. q_starts: int32 [B + 1], non-decreasing: the rows q_starts[b] to
    q_starts[b + 1] are sequence b's last tokens; None: one row a sequence. Rows of no sequence are left out, and so are new tokens in
    front of a sequence's beginning (more rows than kv_lens). The places that are written share no memory with k and v, and where two rows go to one place either may
    stay.

    k_scales, v_scales: float8_e8m0fnu [pages, Hk, page size]; k_pages and v_pages are then float8_e4m3fn, with pages of 16 tokens at least, and a head's row x of a token is quantised as it
    is written: to the numbers of e4m3 nearest to x / s (ties to even, 448 at most), and the scale s = 2^e with the least e from -15 to 7 for which the largest finite |x| is at most
    448 s. A row stands for its numbers times its scale. What is not finite becomes a NaN, a number beyond 448 * 2^7 = 57344 becomes that. Where two rows go to one place their parts may mix.

    There is no derivative through the cache: under autograd, tensors that ask for a gradient are refused, and so are dual tensors of forward mode.

    All lengths and tables are read on the device, so that a captured call follows them. A page number or a length that the cache does not have
    writes nothing and is reported by `check_status`."""
    native = _native(k, v, k_pages, v_pages, page_table, kv_lens, q_starts, k_scales, v_scales)
    if native is not None and native[0].paged_append(k, v, k_pages, v_pages, page_table, kv_lens, q_starts, k_scales, v_scales, native[1]):
        return
    _no_tangents(k, v, k_pages, v_pages)
    if v.shape != k.shape or k.shape[1:2] != k_pages.shape[2:3]:
        raise ValueError("flash_b200: k and v must be [T, Hk, D] with the heads of the cache")
    if v.dtype != k.dtype:
        raise ValueError(f"flash_b200: k and v must share one dtype, got {k.dtype}, {v.dtype}")
    if torch.is_grad_enabled() and v.requires_grad:
        raise RuntimeError("flash_b200: there is no gradient through a paged cache; call it under torch.no_grad()")
    cache, more, starts, held = _checked(k, "k", k_pages, v_pages, page_table, kv_lens, q_starts, k_scales, v_scales)
    _same_device(k, v=v)
    T = k.shape[0]
    if T == 0 or cache.B == 0 or cache.pages == 0:
        return
    k, v = (x if _regular(x) else x.resolve_neg().clone(memory_format=torch.contiguous_format) for x in (k, v))
    with _current(k.device):
        _lib.check(_lib.load().fa_paged_append_more(cache, more, T, starts, _rows(k), _rows(v), _status_word(k.device).data_ptr(), _stream()), "fa_paged_append_more")
    _count(1)
    _bump(k_pages, v_pages, *(x for x in (k_scales, v_scales) if x is not None))
    if ops._SYNC_STATUS:
        check_status(k.device)


def _bump(*tensors):
    """They have been written to in place, which autograd's version counters tell (tensors made in inference mode have none)."""
    torch.autograd.graph.increment_version([x for x in tensors if not x.is_inference()])


def _overlap(a, b):
    """Do the two share memory, as far as their first and last elements tell?"""
    ends = [(x.data_ptr(), x.data_ptr() + x.element_size() * (1 + sum((n - 1) * s for n, s in zip(x.shape, x.stride())))) for x in (a, b)]
    return ends[0][0] < ends[1][1] and ends[1][0] < ends[0][1]


def paged_attention(q, k_pages, v_pages, page_table, kv_lens, q_starts=None, sm_scale=None, softcap=None, slopes=None, prefix=None, out=None, window=None, sinks=0, parents=None,
                    k_scales=None, v_scales=None):
    """Attention of new tokens over a cache of pages that holds their keys and values already (`paged_append`): chunks of prompts and single
    tokens in one ragged batch.

    q: [T, H, D], bf16 or fp16, H a multiple of the cache's Hk and at most 128 times that; the rest as in `paged_append`. The new token at position p of its sequence sees the
    tokens 0 to p. sm_scale: 1 / sqrt(D) if None. softcap, slopes, prefix: as in `attention_scored`, the token's position in the place of
    i + gap; prefix is int32 [B]. window, sinks: as in `attention_scored`; entries of page_table whose pages no token of the call sees may then hold anything.

    parents: int32 [T]; sequences of up to 256 new tokens then have them drafted as a tree. parents[t] is the place, among its sequence's new tokens, of the one that
    token t continues, which lies before it, or -1: t continues the cached text. t sees the text in front of the new tokens, itself and the tokens on its
    branch; its position, by which a window goes, is the text's length plus its depth on the branch (0 where it continues the text), theirs likewise. Sequences of more new tokens
    are chunks, whose parents are not read. A parent that does not lie before its token counts as -1 and is reported by `check_status`. Not together with slopes or a prefix.

    k_scales, v_scales: of a cache of 8 bits, as `paged_append` leaves them (scales outside 2^-15 to 2^7 are taken into that range). Its rows are read as the numbers that they stand for, exactly.

    A row that sees no token (a length of 0, a position below 0) gives zeros. No derivative, as in `paged_append`.

    Returns [T, H, D], zeros in the rows of no sequence; or `out`, whose rows of no sequence are left as they were. `out` shares no memory with q
    or the cache. What lies in the pages behind a sequence's length, or in pages that no sequence names, has no influence, also
    if it is not finite; a value that some row of a block sees (a block is the heads of a group and up to 128 / G neighbouring tokens of a sequence) may spread in it if it is
    not finite (a drafted token's in those that are drafted behind it, too). How the work is cut goes by all lengths of the batch, so that the last bits of a sequence's rows can differ with what
    it is batched with."""
    softcap, window = _checked_softcap(softcap), _checked_window(window, sinks)
    if parents is not None and (slopes is not None or prefix is not None):
        raise ValueError("flash_b200: drafted tokens have no bias by distance and no prefix: parents go without slopes and prefix")
    if sm_scale is None or type(sm_scale) is float:
        native = _native(q, k_pages, v_pages, page_table, kv_lens, q_starts, slopes, prefix, out, parents, k_scales, v_scales)
        if native is not None:
            done = native[0].paged_attention(q, k_pages, v_pages, page_table, kv_lens, q_starts, sm_scale, softcap, slopes, prefix, out, *window, parents, k_scales, v_scales, native[1])
            if done is not None:
                return done if out is None else out
    _no_tangents(q, k_pages, v_pages, slopes, out)
    cache, more, starts, held = _checked(q, "q", k_pages, v_pages, page_table, kv_lens, q_starts, k_scales, v_scales)
    T, H, D = q.shape
    if cache.Hk == 0 or H == 0 or H % cache.Hk or H // cache.Hk > 128:
        raise ValueError(f"flash_b200: the number of heads in q must be a multiple of that in the cache, at most 128 times it, got {H} and {cache.Hk}")
    if sm_scale is None:
        sm_scale = 1. / math.sqrt(D)
    if not 0 < sm_scale < math.inf:
        raise NotImplementedError("flash_b200 needs sm_scale > 0")
    slopes = _checked_slopes(slopes, H, q)
    if prefix is not None:
        prefix = _int32(prefix, (cache.B,), "prefix", q)
    if parents is not None:
        parents = _int32(parents, (T,), "parents", q)
    more.window, more.parents = _lib.Window(*window), _pointer(parents)
    fill = out is None
    if fill:
        out = torch.empty((T, H, D), dtype=q.dtype, device=q.device)
    else:
        if out.shape != q.shape or out.dtype != q.dtype or out.requires_grad or not _regular(out):
            raise ValueError("flash_b200: out must be like q, with a 16-byte aligned base, last stride 1 and other strides that are multiples of 8")
        _same_device(q, out=out)
        for x, name in ((q, "q"), (k_pages, "k_pages"), (v_pages, "v_pages"), (k_scales, "k_scales"), (v_scales, "v_scales")):
            if x is not None and _overlap(out, x):
                raise ValueError(f"flash_b200: out and {name} share memory")
    if T == 0 or cache.B == 0 or cache.pages == 0:
        return out.zero_() if fill else out
    if not _regular(q):
        q = q.resolve_neg().clone(memory_format=torch.contiguous_format)
    lib, device = _lib.load(), q.device
    with _current(device):
        size = _workspace_bytes.get((device.index, D))
        if size is None:
            size = ctypes.c_size_t(0)
            _lib.check(lib.fa_paged_workspace_bytes(cache, size), "fa_paged_workspace_bytes")
            size = _workspace_bytes[device.index, D] = size.value
        work = torch.empty(size // 4, dtype=torch.float32, device=device)
        with ops._timed("paged", 2):
            _lib.check(lib.fa_paged_fwd_more(cache, more, T, H, starts, sm_scale, _scores(softcap, slopes, prefix),
                                             _rows(q), _rows(out), fill, work.data_ptr(), size, _status_word(device).data_ptr(), _stream()), "fa_paged_fwd_more")
    if not fill:
        _bump(out)
    if ops._SYNC_STATUS:
        check_status(device)
    return out
