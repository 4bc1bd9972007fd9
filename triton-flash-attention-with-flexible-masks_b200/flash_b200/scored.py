"""Attention whose scores are capped, biased by distance, or masked up to a prefix.

`attention_scored` is `attention` with three more arguments, forward and backward on the same kernels; without any of the three
it is `attention` itself.
"""
import ctypes
import math

import torch
from . import _lib, ops
from .ops import (SCORE_FUNC_MODE0_NOPE, SCORE_FUNC_MODE1_DOC, _count, _current, _id_tensor, _ids, _plan_kernels, _PermuteRows, _problem,
                  _same_device, _status_word, _stream, _tensor, attention, check_status, group_rows, maybe_contiguous)

SOFTCAP_LEAST, SOFTCAP_MOST = 1e-6, 1e6


def _checked_softcap(softcap):
    """0.0 for none."""
    if softcap is None:
        return 0.0
    softcap = float(softcap)
    if softcap != 0.0 and not SOFTCAP_LEAST <= softcap <= SOFTCAP_MOST:
        raise ValueError(f"flash_b200: softcap must be None, 0 or from {SOFTCAP_LEAST:g} to {SOFTCAP_MOST:g}, got {softcap}")
    return softcap


def _checked_slopes(slopes, H, q):
    """One contiguous fp32 number a head, or None."""
    if slopes is None:
        return None
    if not isinstance(slopes, torch.Tensor) or slopes.dtype != torch.float32 or slopes.shape != (H,):
        raise ValueError(f"flash_b200: slopes must be a float32 tensor of shape [H] = [{H}]")
    if slopes.requires_grad and torch.is_grad_enabled():
        raise ValueError("flash_b200: slopes are constants of the operator (there is no gradient for them); pass slopes.detach()")
    _same_device(q, slopes=slopes)
    return slopes.resolve_neg().contiguous()


def _checked_prefix(prefix, B, N, q):
    """One contiguous int32 number a sequence, or None. The kernels take each into [0, N]; wider integers are brought there first."""
    if prefix is None:
        return None
    if not isinstance(prefix, torch.Tensor) or prefix.dtype not in (torch.int32, torch.int64) or prefix.shape != (B,):
        raise ValueError(f"flash_b200: prefix must be an int32 or int64 tensor of shape [bs] = [{B}]")
    _same_device(q, prefix=prefix)
    return (prefix if prefix.dtype == torch.int32 else prefix.clamp(0, N).to(torch.int32)).contiguous()


def _native(*tensors):
    """The native host calls, where a call of these tensors may take them (see `attention`): the module and the device's status word; else None."""
    first = tensors[0]
    if (all(x is None or type(x) in ops._PLAIN for x in tensors) and ops.PROFILE is None and not ops._SYNC_STATUS and ops._transforms() is None
            and ops._forward_ad._current_level < 0 and ops._tracing_state() is None and first.is_cuda):
        return ops._HOST or ops._host(), _status_word(first.device)
    return None


def _pointer(x):
    return None if x is None else x.data_ptr()


def _scores(softcap, slopes, prefix):
    return _lib.Scores(softcap, _pointer(slopes), _pointer(prefix))


def _once(grads, inputs):
    """Gradients that a graph is to be made of (create_graph=True): an error waits between them and the inputs, where there would be nothing."""
    if not torch.is_grad_enabled():
        return grads
    error = torch._C._functions.DelayedError(b"flash_b200: attention_scored has gradients once; these cannot be differentiated", 6)
    return error(*(g.detach().requires_grad_() for g in grads), *inputs)[:3]


class ScoredAttention(torch.autograd.Function):
    """The autograd node of `attention_scored`. Saves q, k, v, the output, its log-sum-exp, the slopes and prefix that there are, and what the rounding
    of the output has left out."""

    @staticmethod
    def forward(ctx, q, k, v, causal, sm_scale, eq, ek, score_func_mode, softcap, slopes, prefix):
        needs_grad = any(ctx.needs_input_grad[:3])
        B, H, M, D = q.shape
        Hk, N = k.shape[1:3]
        lib, device = _lib.load(), q.device
        q, k, v = maybe_contiguous(q), maybe_contiguous(k), maybe_contiguous(v)
        id_heads = 1
        if score_func_mode == SCORE_FUNC_MODE1_DOC:
            eq, ek = _id_tensor(eq, B, H, M, "eq"), _id_tensor(ek, B, H, N, "ek")
            id_heads = 1 if H == 1 or (eq.stride(1) == 0 and ek.stride(1) == 0) else H
        scores = _scores(softcap, slopes, prefix)
        with _current(device):
            prob = _problem(B, H, Hk, M, N, D, q.dtype, causal, score_func_mode, id_heads, sm_scale)
            status, stream, plan = _status_word(device), _stream(), None
            if score_func_mode == SCORE_FUNC_MODE1_DOC or not lib.fa_plan_optional(prob, needs_grad):
                size = ctypes.c_size_t(0)
                _lib.check(lib.fa_plan_bytes(prob, size), "fa_plan_bytes")
                plan = torch.empty(size.value // 4, dtype=torch.int32, device=device)
                ids = (_ids(eq), _ids(ek)) if eq is not None else (None, None)
                with ops._timed("plan", _plan_kernels(M, N) if eq is not None else 1):
                    _lib.check(lib.fa_plan_build_scored(prob, scores, *ids, plan.data_ptr(), size.value, status.data_ptr(), stream),
                               "fa_plan_build_scored")
            out = torch.empty_like(q)
            if maybe_contiguous(out) is not out:
                out = torch.empty((B, H, M, D), dtype=q.dtype, device=device)
            lse = torch.empty((B, H, lib.fa_padded_rows(M)), dtype=torch.float32, device=device)
            splits, work, size = lib.fa_fwd_splits(prob), None, ctypes.c_size_t(0)
            if splits > 1:
                _lib.check(lib.fa_fwd_workspace_bytes(prob, splits, size), "fa_fwd_workspace_bytes")
                work = torch.empty(size.value // 4, dtype=torch.float32, device=device)
            # what the rounding of the output leaves out, for the gradients
            rest = torch.empty((B, H, M, D), dtype=q.dtype, device=device) if needs_grad and q.dtype != torch.float32 else None
            with ops._timed("fwd", (2 if splits > 1 else 1) + (splits > 1 and rest is not None)):
                _lib.check(lib.fa_fwd_scored(prob, scores, _tensor(q), _tensor(k), _tensor(v), _tensor(out), _pointer(rest) if splits == 1 else None, lse.data_ptr(),
                                             _pointer(plan), splits, _pointer(work),
                                             size.value, status.data_ptr(), stream), "fa_fwd_scored")
                if splits > 1 and rest is not None:
                    _lib.check(lib.fa_fwd_rest(prob, splits, work.data_ptr(), size.value, rest.data_ptr(), status.data_ptr(), stream), "fa_fwd_rest")
            if ops._SYNC_STATUS:
                check_status(device)
        if needs_grad:
            extra = slopes, prefix, rest
            ctx.save_for_backward(q, k, v, out, lse, *(x for x in extra if x is not None))
            ctx.has = tuple(x is not None for x in extra)
            ctx.plan, ctx.prob, ctx.softcap = plan, prob, softcap
        return out

    @staticmethod
    def backward(ctx, do):
        q, k, v, out, lse, *extra = ctx.saved_tensors
        slopes, prefix, rest = (extra.pop(0) if has else None for has in ctx.has)
        lib, device, plan = _lib.load(), q.device, ctx.plan
        do = maybe_contiguous(do.detach().to(q.dtype))
        with _current(device):
            delta = torch.empty_like(lse)
            dq, dk, dv = (torch.empty(x.shape, dtype=x.dtype, device=device) for x in (q, k, v))
            _lib.check(lib.fa_bwd_scored(ctx.prob, _scores(ctx.softcap, slopes, prefix), *map(_tensor, (q, k, v, out)), _pointer(rest), _tensor(do),
                                         lse.data_ptr(), delta.data_ptr(), *map(_tensor, (dq, dk, dv)), _pointer(plan), _status_word(device).data_ptr(),
                                         _stream()), "fa_bwd_scored")
            _count(3)
            if ops._SYNC_STATUS:
                check_status(device)
        return (*_once((dq, dk, dv), (q, k, v)), *(None,) * 8)


def attention_scored(q, k, v, causal=False, sm_scale=None, eq=None, ek=None, score_func_mode=SCORE_FUNC_MODE0_NOPE, softcap=None, slopes=None,
                     prefix=None):
    """`attention(q, k, v, causal, sm_scale, eq, ek, score_func_mode)` with changed scores. With s = sm_scale q_i . k_j and gap = max(0, N - M),

        x_ij = softcap * tanh(s / softcap) - slopes[h] * |i + gap - j|

    takes the place of s before the softmax, and a key j < prefix[b] is visible to every query of sequence b whatever the causal mask says (the
    ids' rule holds for it as for the others).

    softcap: None or 0 for none, else from 1e-6 to 1e6. slopes: float32 [H], None for none. prefix: int32 or int64 [bs], None for none; it
    needs causal=True, values are taken into [0, N]. All else is as in `attention`: types (bf16, fp16, fp32), head dims, grouped heads, strides, a row
    that the masks leave no key gives zeros and takes no part in the gradients. There are gradients for q, k and v, once (with create_graph=True, to differentiate them raises); slopes and
    prefix are constants, and slopes that ask for a gradient are refused unless grad mode is off. As in `attention`, masked entries are products with an exact 0: a
    value that is not finite may spread from a key that some query of its block of 128 sees."""
    softcap = _checked_softcap(softcap)
    if softcap == 0.0 and slopes is None and prefix is None:
        return attention(q, k, v, causal, sm_scale, eq, ek, score_func_mode)
    grouped = ops.GROUP_QUERIES and eq is not None and not causal and slopes is None and q.dim() == 4 and 128 < q.shape[2] <= _lib.FA_GROUP_MAX_ROWS
    if not grouped and type(score_func_mode) is int and abs(score_func_mode) < 8 and (sm_scale is None or type(sm_scale) is float):
        native = _native(q, k, v, eq, ek, slopes, prefix)
        if native is not None:
            done = native[0].attend_scored(q, k, v, bool(causal), sm_scale, eq, ek, score_func_mode, softcap, slopes, prefix, native[1])
            if done is not None:
                return done
    D = q.shape[-1]
    assert k.shape[-1] == D and v.shape[-1] == D, "feature size of q, k, v should be equal"
    assert D in {16, 32, 64, 128}
    B, H, M, D = q.shape
    Hk, N = k.shape[1:3]
    assert k.shape == v.shape and k.shape[0] == B, "k and v should be [bs, Hk, N, D]"
    assert H % Hk == 0, "number of heads in q must be a multiple of that in k & v"
    assert N >= M or not causal, "KV length should be larger than M length in causal mode!"
    assert (eq is None) == (ek is None)
    assert score_func_mode in (SCORE_FUNC_MODE0_NOPE, SCORE_FUNC_MODE1_DOC)
    assert (eq is None) == (score_func_mode == SCORE_FUNC_MODE0_NOPE)
    if not q.is_cuda:
        raise RuntimeError("flash_b200 runs on CUDA tensors only (there is no CPU implementation)")
    _same_device(q, k=k, v=v, eq=eq, ek=ek)
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"flash_b200: q, k, v must share one dtype, got {q.dtype}, {k.dtype}, {v.dtype}")
    if sm_scale is None:
        sm_scale = 1. / math.sqrt(D)
    if not sm_scale > 0:
        raise NotImplementedError("flash_b200 needs sm_scale > 0")
    if prefix is not None and not causal:
        raise ValueError("flash_b200: a prefix is what a causal mask leaves visible; it needs causal=True")
    slopes, prefix = _checked_slopes(slopes, H, q), _checked_prefix(prefix, B, N, q)
    args = float(sm_scale), softcap, slopes, prefix
    # queries of scattered documents side by side, as in `attention`; a bias goes by the queries' places, which have to stay
    if grouped:
        order, inverse, ids, id_heads = group_rows(eq, B, H, M)
        o = ScoredAttention.apply(_PermuteRows.apply(q, order, inverse, id_heads), k, v, False, args[0], ids.expand(B, H, M), ek, score_func_mode, *args[1:])
        return _PermuteRows.apply(o, inverse, order, id_heads)
    return ScoredAttention.apply(q, k, v, bool(causal), args[0], eq, ek, int(score_func_mode), *args[1:])
