"""Sliding windows with sinks, trees of drafted tokens, and 8-bit caches: `flash_b200`'s attention over them, at the sizes their users call it with.

`attention_scored` with `window` and `sinks`: a query sees the last keys and a few first ones, forward alone or with its gradients.
`paged_append` with `k_scales` and `v_scales`: new tokens are quantised to e4m3 as they are put into the cache's pages.
`paged_attention` over such a cache, with a window and sinks, and for trees of drafted tokens (`parents`).

`listed()` names one call per kind of use and `draw()` gives other sizes of the same kinds. Where `own` is false `run` computes the plain form
in elementary torch operations in 32 bits, else by the package, which is taken from the working folder.
"""
import functools
import os
import sys

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
LEAST, MOST = -15, 7  # exponents of a row's scale


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def _scored(use, B, H, Hk, M, N, D, dtype, window, sinks, backward, cap=0.0, bias=False, docs=0, len_seed=0, std=1.5, layout="bhld"):
    """`docs`: most documents of a sequence (0: no ids); `len_seed` fixes their lengths. `std` of q and k. `layout`: "bhld" contiguous, "blhd" the
    views that a projection's output [B, L, H, D] is transposed to."""
    return dict(op="scored", use=use, B=B, H=H, Hk=Hk, M=M, N=N, D=D, dtype=dtype, window=window, sinks=sinks, backward=backward, cap=cap, bias=bias,
                docs=docs, len_seed=len_seed, std=std, layout=layout)


def _paged(use, op, B, H, Hk, D, dtype, page, longest, chunks, chunk, eight, window=0, sinks=0, tree=0, cap=0.0, bias=False, len_seed=0):
    """`B` sequences of at most `longest` cached tokens, the first `chunks` of them with about `chunk` new tokens and the others with one; `tree`: each has
    so many at most, drafted as a tree. `eight`: the cache is of 8 bits."""
    return dict(op=op, use=use, B=B, H=H, Hk=Hk, D=D, dtype=dtype, page=page, longest=longest, chunks=chunks, chunk=chunk, eight=eight, window=window, sinks=sinks,
                tree=tree, cap=cap, bias=bias, len_seed=len_seed)


def listed():
    cases = {
        # The smallest window call in use: one short prompt of a small model. Launches and host time are all there is.
        "window_prompt": _scored("prompt", 1, 8, 8, 300, 300, 64, "bf16", 128, 4, False),
        # fp32 step of a check-sized model.
        "window_fp32_step": _scored("fp32", 2, 4, 4, 512, 512, 64, "fp32", 100, 2, True),
        # Training step of a long-context model whose layers have a window: grouped-query heads, projection layout.
        "window_step": _scored("step", 2, 16, 4, 4000, 4000, 128, "bf16", 1024, 4, True, layout="blhd"),
        # Packed pretraining step with capped scores, documents and a window, ragged length.
        "window_packed_step": _scored("packed", 1, 16, 16, 8111, 8111, 64, "fp16", 2048, 0, True, cap=50.0, docs=4, len_seed=3),
        # One token for each of 64 conversations, of which a layer sees a window and the first tokens; 16-bit cache.
        "window_decode": _paged("decode", "attend", 64, 32, 8, 128, "bf16", 64, 16000, 0, 1, False, 4096, 4),
        # An 8-bit cache's side of a server's step: one new token each, and whole prompts.
        "eight_append_tokens": _paged("append", "append", 64, 32, 8, 128, "bf16", 64, 8192, 0, 1, True),
        "eight_append_prompts": _paged("append", "append", 8, 32, 8, 128, "bf16", 16, 4000, 8, 3500, True),
        # One token of one conversation over an 8-bit cache, small model, small pages: latency.
        "eight_decode_one": _paged("decode", "attend", 1, 8, 8, 64, "fp16", 16, 700, 0, 1, True),
        # One token for each of 64 conversations of ragged length over an 8-bit cache.
        "eight_decode_batch": _paged("decode", "attend", 64, 32, 8, 128, "bf16", 64, 8192, 0, 1, True),
        # A server's step over an 8-bit cache: chunks of prompts and single tokens, capped scores.
        "eight_mixed_batch": _paged("mixed", "attend", 8, 32, 8, 128, "bf16", 32, 8000, 3, 500, True, cap=30.0),
        # One conversation's drafted tokens, small model.
        "tree_one": _paged("tree", "attend", 1, 16, 4, 64, "bf16", 16, 1200, 0, 1, False, tree=24),
        # Drafted trees of 32 conversations in one step.
        "tree_batch": _paged("tree", "attend", 32, 32, 8, 128, "bf16", 64, 6000, 0, 1, False, tree=61, len_seed=5),
    }
    return [dict(c, name=n) for n, c in cases.items()]


def _log_int(rng, lo, hi):
    """An integer from [lo, hi], even over the logarithm."""
    return min(hi, int(lo * (hi / lo) ** rng.random() + 0.5))


def _draw_one(rng):
    use = rng.choice(("prompt", "fp32", "step", "packed", "decode", "decode", "mixed", "mixed", "append", "tree", "tree"))
    half = rng.choice(("bf16", "fp16"))
    gqa = rng.choice(((32, 8), (16, 4), (64, 8), (16, 16), (12, 2)))
    cap, bias, seed, sinks = rng.choice((0.0, 0.0, 30.0, 50.0)), rng.random() < 0.25, rng.randrange(1 << 20), rng.choice((0, 1, 4, 4, 130))
    if use == "prompt":
        h, m = rng.choice((4, 8, 12, 16)), _log_int(rng, 1, 2048)
        return _scored(use, rng.choice((1, 1, 2)), h, h, m, m + rng.choice((0, 0, 700)), rng.choice((64, 128)), half, _log_int(rng, 1, 1024), sinks, False, cap, bias)
    if use == "fp32":
        h, m = rng.choice((2, 4, 8)), _log_int(rng, 100, 1024)
        return _scored(use, rng.choice((1, 2, 4)), h, h, m, m, rng.choice((32, 64, 128)), "fp32", _log_int(rng, 1, 512), sinks, True, cap, bias, 4 * rng.randrange(2), seed)
    if use == "step":
        m = _log_int(rng, 256, 4000)
        return _scored(use, rng.choice((1, 2, 4)), gqa[0], gqa[1], m, m, rng.choice((32, 64, 128)), half, _log_int(rng, 64, 2048), sinks, True, cap, bias, layout="blhd")
    if use == "packed":
        h, m = rng.choice((8, 16)), _log_int(rng, 1000, 8111)
        return _scored(use, rng.choice((1, 2)), h, h, m, m, rng.choice((64, 128)), half, _log_int(rng, 64, 4096), sinks, True, cap, bias, rng.choice((4, 16)), seed)
    page, eight = rng.choice((16, 32, 64, 128)), rng.random() < 0.6
    window, sinks = (_log_int(rng, 16, 8192), sinks) if not eight or rng.random() < 0.4 else (0, 0)
    if use == "decode":
        b = _log_int(rng, 1, 64)
        return _paged(use, "attend", b, gqa[0], gqa[1], rng.choice((64, 128)), half, page, _log_int(rng, 300, min(131072, (1 << 19) // b)), 0, 1, eight, window, sinks,
                      0, cap, bias, seed)
    if use == "tree":
        b = _log_int(rng, 1, 32)
        return _paged(use, "attend", b, gqa[0], gqa[1], rng.choice((64, 128)), half, page, _log_int(rng, 300, min(32768, (1 << 18) // b)), 0, 1, eight, window, sinks,
                      _log_int(rng, 2, 200), cap, False, seed)
    b = _log_int(rng, 1, 16)
    chunk = _log_int(rng, 17, 2048)
    longest = chunk + _log_int(rng, 100, 8000)
    if use == "append":
        return _paged(use, "append", b, gqa[0], gqa[1], rng.choice((64, 128)), half, page, longest, rng.randrange(1, b + 1), chunk, True, len_seed=seed)
    return _paged(use, "attend", b, gqa[0], gqa[1], rng.choice((64, 128)), half, page, longest, rng.randrange(1, b + 1), chunk, eight, window, sinks, 0, cap, bias, seed)


def draw(rng):
    while True:
        c = _draw_one(rng)
        w = work(c)
        if w["flops"] <= 2.1e11 and w["bytes"] <= 1.0e9 and _scores(c) <= 1.06e9:
            return c


def _scores(c):
    """Entries of the plain form's score matrix."""
    if c["op"] == "scored":
        return c["B"] * c["H"] * c["M"] * c["N"]
    if c["op"] == "append":
        return 0
    new, total = _ragged(c)
    return c["B"] * c["H"] * int(new.max()) * (int(total.max()) + c["page"])


def _ragged(c):
    """(new tokens, cached tokens with the new ones) of each sequence."""
    rng = np.random.default_rng(c["len_seed"])
    new = np.ones(c["B"], dtype=np.int64)
    if c["tree"]:
        new = rng.integers(c["tree"] // 2 + 1, c["tree"] + 1, c["B"])
    new[: c["chunks"]] = np.maximum(1, (c["chunk"] * rng.uniform(0.7, 1.0, c["chunks"])).astype(np.int64))
    if c["chunks"]:
        new[0] = c["chunk"]
    total = np.maximum(new, (c["longest"] * rng.uniform(0.2, 1.0, c["B"])).astype(np.int64))
    total[0] = max(c["longest"], new[0])
    return new, total


def _trees(c):
    """Of each sequence's new tokens the one that each continues, -1: the cached text. A token joins one of the last few drafted before it."""
    rng, new = np.random.default_rng(c["len_seed"] + 2), _ragged(c)[0]
    return [np.array([-1] + [int(rng.integers(max(-1, t - 12), t)) for t in range(1, n)], dtype=np.int32) for n in new]


def _documents(c):
    """Document lengths of each sequence: 1 to `docs` documents of Dirichlet(1) weights."""
    rng, out = np.random.default_rng(c["len_seed"]), []
    for _ in range(c["B"]):
        w = rng.dirichlet(np.ones(int(rng.integers(1, c["docs"] + 1))))
        ends = np.round(np.cumsum(w) / w.sum() * c["N"]).astype(np.int64)
        out.append(np.diff(np.concatenate([[0], ends])))
    return out


def _seen(at, first, window, sinks):
    """How many keys from `first` on a causal query at position `at` sees."""
    if not window:
        return (at + 1 - first).clip(0)
    low = (at - window + 1).clip(0)
    return (at + 1 - np.maximum(low, first)).clip(0) + (np.minimum(sinks, low) - first).clip(0)


def _depths(parents):
    d = np.zeros(len(parents), dtype=np.int64)
    for t, a in enumerate(parents):
        d[t] = d[a] + 1 if a >= 0 else 0
    return d


def _visible(c):
    """Unmasked entries of the scores over all sequences and heads."""
    if c["op"] != "scored":
        new, total = _ragged(c)
        if c["tree"]:
            at = [t - n + _depths(p) for n, t, p in zip(new, total, _trees(c))]
        else:
            at = [np.arange(t - n, t) for n, t in zip(new, total)]
        return c["H"] * float(sum(_seen(a, 0, c["window"], c["sinks"]).sum() for a in at))
    count, at = 0.0, np.arange(c["N"] - c["M"], c["N"])
    for lengths in _documents(c) if c["docs"] else [np.array([c["N"]])] * c["B"]:
        first = np.repeat(np.cumsum(lengths) - lengths, lengths)[at]
        count += float(_seen(at, first, c["window"], c["sinks"]).sum())
    return c["H"] * count


def work(case):
    """Flops of the unmasked entries alone (2 products forward, 5 backward); each input read and each output written once."""
    c = case
    if c["op"] == "scored":
        size = 4 if c["dtype"] == "fp32" else 2
        q, kv = c["B"] * c["H"] * c["M"] * c["D"] * size, c["B"] * c["Hk"] * c["N"] * c["D"] * size
        tensors = (2 * q + 2 * kv) * (2 if c["backward"] else 1)  # q, k, v, o and dO, dq, dk, dv
        return {"bytes": tensors + (8 * c["B"] * c["N"] if c["docs"] else 0), "flops": (14 if c["backward"] else 4) * c["D"] * _visible(c)}
    new, total = _ragged(c)
    row = 2 * c["Hk"] * (c["D"] + 1 if c["eight"] else 2 * c["D"])  # of the cache, K and V
    if c["op"] == "append":
        return {"bytes": int(new.sum()) * (4 * c["Hk"] * c["D"] + row) + 4 * int((-(-total // c["page"])).sum()), "flops": 0}
    low = (total - new - c["window"] + 1).clip(0) if c["window"] else 0 * total  # the window's first key of a sequence's first token
    keys = int((total - low + np.minimum(low, c["sinks"])).sum())
    return {"bytes": 4 * int(new.sum()) * c["H"] * c["D"] + keys * row + 4 * (keys // c["page"]) + (4 * int(new.sum()) if c["tree"] else 0),
            "flops": 4 * c["D"] * _visible(c)}


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _package():
    path = os.path.abspath("triton-flash-attention-with-flexible-masks_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import flash_b200
    return flash_b200


def _slopes(H):
    """A geometric series from head to head, as models with a linear bias take."""
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], dtype=torch.float32, device="cuda")


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[c["dtype"]]

    def values(*shape, std=1.0):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).mul_(std).to(dtype)

    s = {"case": c, "cap": c["cap"] or None, "slopes": _slopes(c["H"]) if c["bias"] else None, "window": c["window"] or None}
    if c["op"] == "scored":
        def tensor(heads, length, std):
            return values(c["B"], heads, length, c["D"], std=std) if c["layout"] == "bhld" else values(c["B"], length, heads, c["D"], std=std).transpose(1, 2)
        s |= {"q": tensor(c["H"], c["M"], c["std"]), "k": tensor(c["Hk"], c["N"], c["std"]), "v": tensor(c["Hk"], c["N"], 1.0), "do": None, "ids": None}
        if c["backward"]:
            s["do"] = tensor(c["H"], c["M"], 1.0)
            for n in ("q", "k", "v"):
                s[n].requires_grad_()
        if c["docs"]:
            row = np.stack([np.repeat(-(np.arange(len(x), dtype=np.int64) + 1), x) for x in _documents(c)])
            s["ids"] = torch.from_numpy(row).cuda()[:, None, :].expand(c["B"], c["H"], c["N"])
        return s
    new, total = _ragged(c)
    pages = -(-total // c["page"])
    n_pages = int(pages.sum()) + 8  # some that belong to nobody
    order = np.random.default_rng(seed).permutation(n_pages)
    table = np.zeros((c["B"], int(pages.max())), dtype=np.int32)
    for b, first in enumerate(np.cumsum(pages) - pages):
        table[b, : pages[b]] = order[first: first + pages[b]]
    T, Hk, D = int(new.sum()), c["Hk"], c["D"]
    s |= {"table": torch.from_numpy(table).cuda(), "kv_lens": torch.from_numpy(total.astype(np.int32)).cuda(), "most": int(new.max()), "k_scales": None, "v_scales": None,
          "starts": torch.from_numpy(np.concatenate([[0], np.cumsum(new)]).astype(np.int32)).cuda() if c["chunks"] or c["tree"] else None,
          "parents": torch.from_numpy(np.concatenate(_trees(c))).cuda() if c["tree"] else None}
    if c["eight"]:
        # rows whose largest entry is from 224 to 448, as quantising leaves them, and scales that bring them to a deviation around 1
        def page_values():
            x = torch.randn((n_pages, c["page"], Hk, D), generator=gen, device="cuda")
            return x.mul_(torch.rand((n_pages, c["page"], Hk, 1), generator=gen, device="cuda").add_(1).mul_(224 / x.abs().amax(-1, keepdim=True))).to(torch.float8_e4m3fn)

        def page_scales():
            return torch.randint(119, 121, (n_pages, Hk, c["page"]), generator=gen, device="cuda", dtype=torch.uint8).view(torch.float8_e8m0fnu)
        s |= {"k_pages": page_values(), "v_pages": page_values(), "k_scales": page_scales(), "v_scales": page_scales()}
    else:
        s |= {"k_pages": values(n_pages, c["page"], Hk, D), "v_pages": values(n_pages, c["page"], Hk, D)}
    if c["op"] == "append":
        s |= {"k": values(T, Hk, D, std=2.0), "v": values(T, Hk, D)}
    else:
        s["q"] = values(T, c["H"], D, std=2.0)
    return s


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def _softmax(x, keep):
    """Over the kept entries of the last axis; a row without any gives zeros."""
    x = x.masked_fill_(~keep, -torch.inf)
    x = x.sub_(x.amax(-1, keepdim=True).clamp_(min=-1e38)).exp_()
    return x.div_(x.sum(-1, keepdim=True).clamp_(min=1e-38))


def _plain_scored(s):
    c = s["case"]
    M, N, G, scale = c["M"], c["N"], c["H"] // c["Hk"], c["D"] ** -0.5
    q, k, v = s["q"].detach().float(), s["k"].detach().float().repeat_interleave(G, 1), s["v"].detach().float().repeat_interleave(G, 1)
    keys = torch.arange(N, device="cuda")
    far = torch.arange(M, device="cuda")[:, None] + (N - M) - keys  # how far the key lies behind
    x = (q @ k.mT).mul_(scale)
    t = None
    if s["cap"]:
        t = x.div_(s["cap"]).tanh_()
        x = t * s["cap"]
    if s["slopes"] is not None:
        x = x - s["slopes"][:, None, None] * far.abs()
    keep = ((far >= 0) & ((far < s["window"]) | (keys < c["sinks"])))[None, None]
    if s["ids"] is not None:
        eq = s["ids"][:, :1, N - M:, None]
        keep = keep & ((eq >= 0) | (eq == s["ids"][:, :1, None, :]))
    p = _softmax(x, keep)
    o = p @ v
    if not c["backward"]:
        return o.to(s["q"].dtype)
    do = s["do"].float()
    dv = p.mT @ do
    ds = (do @ v.mT).sub_((do * o).sum(-1, keepdim=True)).mul_(p)
    if t is not None:
        ds = ds.mul_(1 - t * t)
    dq, dk = (ds @ k).mul_(scale), (ds.mT @ q).mul_(scale)
    dk, dv = (g.reshape(c["B"], c["Hk"], G, N, c["D"]).sum(2) for g in (dk, dv))
    return tuple(g.to(s["q"].dtype) for g in (o, dq, dk, dv))


def _token_rows(s):
    """Of each sequence and new token: the token's row, whether there is such a token, and its place in the cache."""
    B = s["kv_lens"].shape[0]
    starts = s["starts"].long() if s["starts"] is not None else torch.arange(B + 1, device="cuda")
    at = torch.arange(s["most"], device="cuda")
    new = starts[1:] - starts[:-1]
    return starts[:-1, None] + at, at < new[:, None], (s["kv_lens"] - new)[:, None] + at


def _quantised(x):
    """Rows of e4m3 and the exponents of their scales, which are the least that bring the largest finite entry to 448 or below."""
    x = x.float()
    finite = x.isfinite()
    most = torch.where(finite, x.abs(), 0.0).amax(-1)
    part, exponent = torch.frexp(most / 448)
    exponent = torch.where(most > 0, exponent - (part == 0.5).int(), LEAST).clamp_(LEAST, MOST)
    q = torch.ldexp(x, -exponent[..., None]).clamp_(-448, 448)
    return torch.where(finite, q, torch.nan).to(torch.float8_e4m3fn), exponent


def _plain_append(s):
    row, real, at = _token_rows(s)
    page = s["table"].long().gather(1, (at // s["case"]["page"]).clamp(max=s["table"].shape[1] - 1))
    row, page, slot = row[real], page[real], (at % s["case"]["page"])[real]
    (k, k_exponent), (v, v_exponent) = _quantised(s["k"][row]), _quantised(s["v"][row])
    s["k_pages"].view(torch.uint8)[page, slot] = k.view(torch.uint8)
    s["v_pages"].view(torch.uint8)[page, slot] = v.view(torch.uint8)
    s["k_scales"].view(torch.uint8)[page, :, slot] = (k_exponent + 127).to(torch.uint8)
    s["v_scales"].view(torch.uint8)[page, :, slot] = (v_exponent + 127).to(torch.uint8)
    return _cache(s)


def _cache(s):
    """The cache after an append: its values, and the exponents of their scales (biased by 127)."""
    return s["k_pages"], s["v_pages"], s["k_scales"].view(torch.uint8), s["v_scales"].view(torch.uint8)


def _pages_of(s, pages, scales):
    """[B, Hk, N, D] in 32 bits."""
    x = pages[s["table"].long()] if scales is None else pages.view(torch.uint8)[s["table"].long()].view(torch.float8_e4m3fn)
    x = x.float()
    if scales is not None:
        x = torch.ldexp(x, (scales.view(torch.uint8)[s["table"].long()].int() - 127).permute(0, 1, 3, 2)[..., None])
    B, n, page, Hk, D = x.shape
    return x.reshape(B, n * page, Hk, D).permute(0, 2, 1, 3)


def _plain_keep(s, row, at, N):
    """[B, m, N]: which places of the cache each new token sees; and the tokens' positions."""
    c, keys = s["case"], torch.arange(N, device="cuda")
    base, m = at[:, :1], at.shape[1]
    position, place = at, keys.expand(c["B"], N)
    mine = keys <= at[..., None]
    if c["tree"]:
        parents = s["parents"].long()[row.clamp(max=s["parents"].shape[0] - 1)]
        reach = torch.eye(m, device="cuda") + (parents[..., None] == torch.arange(m, device="cuda")).float()
        reach = functools.reduce(lambda a, _: (a @ a).clamp_(max=1), range(max(1, m.bit_length())), reach)  # [B, m, m] own and all tokens before it on its branch
        depth = reach.sum(-1).long() - 1
        position = base + depth
        i = keys - base  # [B, N] place among the new tokens
        new, i = (i >= 0) & (i < m), i.clamp(0, m - 1)
        place = torch.where(new, base + depth.gather(1, i), place)
        mine = (~new[:, None] & (keys < base)[:, None]) | (new[:, None] & (reach.gather(2, i[:, None].expand(-1, m, -1)) > 0))
    if s["window"]:
        mine = mine & ((position[..., None] - place[:, None] < s["window"]) | (place[:, None] < c["sinks"]))
    return mine, position


def _plain_attend(s):
    c = s["case"]
    B, H, Hk, D, m = c["B"], c["H"], c["Hk"], c["D"], s["most"]
    row, real, at = _token_rows(s)
    k, v = _pages_of(s, s["k_pages"], s["k_scales"]), _pages_of(s, s["v_pages"], s["v_scales"])
    N = k.shape[2]
    q = s["q"][row.clamp(max=s["q"].shape[0] - 1)].float()  # [B, m, H, D]
    q = q.reshape(B, m, Hk, H // Hk, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, H // Hk * m, D)
    x = (q @ k.mT).mul_(D ** -0.5).reshape(B, H, m, N)
    if s["cap"]:
        x = x.div_(s["cap"]).tanh_().mul_(s["cap"])
    keep, position = _plain_keep(s, row, at, N)
    if s["slopes"] is not None:
        x = x - s["slopes"][:, None, None] * (position[:, None, :, None] - torch.arange(N, device="cuda")).abs()
    p = _softmax(x, keep[:, None])
    o = (p.reshape(B, Hk, H // Hk * m, N) @ v).reshape(B, H, m, D).permute(0, 2, 1, 3)
    return o[real].to(s["q"].dtype)


def run(state):
    s = state
    c = s["case"]
    if not own:
        with torch.no_grad():
            return {"scored": _plain_scored, "append": _plain_append, "attend": _plain_attend}[c["op"]](s)
    fb = _package()
    if c["op"] == "append":
        fb.paged_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["kv_lens"], s["starts"], k_scales=s["k_scales"], v_scales=s["v_scales"])
        return _cache(s)
    if c["op"] == "attend":
        return fb.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["kv_lens"], s["starts"], softcap=s["cap"], slopes=s["slopes"],
                                  window=s["window"], sinks=c["sinks"], parents=s["parents"], k_scales=s["k_scales"], v_scales=s["v_scales"])
    mode = fb.SCORE_FUNC_MODE0_NOPE if s["ids"] is None else fb.SCORE_FUNC_MODE1_DOC
    eq = None if s["ids"] is None else s["ids"][:, :, c["N"] - c["M"]:]
    o = fb.attention_scored(s["q"], s["k"], s["v"], True, None, eq, s["ids"], mode, softcap=s["cap"], slopes=s["slopes"], window=s["window"], sinks=c["sinks"])
    if not c["backward"]:
        return o
    return (o.detach(), *torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"]))


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    with torch.no_grad():
        s = prepare(case, seed)
        return {"scored": _exact_scored, "append": _exact_append, "attend": _exact_attend}[case["op"]](case, s)


def _exact_scored(c, s):
    """Whole rows of the score matrix, as many at a time as fit in 1 GB."""
    B, H, M, N, D = c["B"], c["H"], c["M"], c["N"], c["D"]
    gap, scale, new = N - M, 1.0 / D ** 0.5, {"device": "cuda", "dtype": torch.float64}
    o = torch.zeros(B, H, M, D, **new)
    dq, dk, dv = (torch.zeros(B, h, n, D, **new) if c["backward"] else None for h, n in ((H, M), (c["Hk"], N), (c["Hk"], N)))
    keys = torch.arange(N, device="cuda")[None]
    step = max(1, min(M, (1 << 27) // N))
    for b in range(B):
        for h in range(H):
            hk = h * c["Hk"] // H
            k, v = s["k"][b, hk].double(), s["v"][b, hk].double()
            for i in range(0, M, step):
                rows = slice(i, min(i + step, M))
                at = torch.arange(rows.start, rows.stop, device="cuda")[:, None] + gap
                q = s["q"][b, h, rows].double()
                x, slope = q @ k.T * scale, 1.0
                if c["cap"]:
                    th = torch.tanh(x / c["cap"])
                    x, slope = c["cap"] * th, 1 - th ** 2
                if c["bias"]:
                    x = x - s["slopes"][h].double() * (at - keys).abs()
                hidden = (keys > at) | ((keys <= at - c["window"]) & (keys >= c["sinks"]))
                if c["docs"]:
                    ids = s["ids"][b, h]
                    mine = ids[gap:][rows, None]
                    hidden = hidden | ((mine < 0) & (mine != ids[None]))
                x = torch.where(hidden, -torch.inf, x)
                p = torch.exp(x - x.amax(1, keepdim=True).clamp(min=-1e300))
                p = p / p.sum(1, keepdim=True).clamp(min=1e-300)
                o[b, h, rows] = p @ v
                if c["backward"]:
                    do = s["do"][b, h, rows].double()
                    dv[b, hk] += p.T @ do
                    ds = (do @ v.T - (do * o[b, h, rows]).sum(1, keepdim=True)) * p * slope
                    dq[b, h, rows] = ds @ k * scale
                    dk[b, hk] += ds.T @ q * scale
    return (o, dq, dk, dv) if c["backward"] else o


def _sequences(c):
    """(sequence, its first row, new tokens, cached tokens) of each."""
    new, total = _ragged(c)
    first = np.cumsum(new) - new
    return [(b, int(first[b]), int(new[b]), int(total[b])) for b in range(c["B"])]


#: The numbers from 0 to 448 that e4m3 has.
_E4M3 = [m / 512 for m in range(8)] + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8) if (e, m) != (15, 7)]


def _nearest(x):
    """The number that e4m3 has nearest to each of x (of two the one with an even last bit), by search in the list of all."""
    all_of = torch.tensor(_E4M3, dtype=torch.float64, device=x.device)
    size = x.abs().clamp(max=448.0)
    above = torch.searchsorted(all_of, size).clamp(1, len(_E4M3) - 1)
    low, high = size - all_of[above - 1], all_of[above] - size
    up = (high < low) | ((high == low) & (above % 2 == 0))
    return torch.copysign(all_of[torch.where(up, above, above - 1)], x)


def _exact_append(c, s):
    table, out = s["table"].long(), []
    for rows, pages, scales in ((s["k"], s["k_pages"], s["k_scales"]), (s["v"], s["v_pages"], s["v_scales"])):
        pages, scales = pages.double(), scales.view(torch.uint8).clone()
        x = rows.double()
        most = 448 * 2.0 ** torch.arange(LEAST, MOST, device="cuda", dtype=torch.float64)  # what a row of each exponent holds
        exponent = LEAST + (x.abs().amax(-1, keepdim=True) > most).sum(-1)
        x = _nearest(torch.ldexp(x, -exponent[..., None]))
        for b, first, new, total in _sequences(c):
            at = torch.arange(total - new, total, device="cuda")
            page, slot = table[b, at // c["page"]], at % c["page"]
            pages[page, slot] = x[first: first + new]
            scales[page, :, slot] = (exponent[first: first + new] + 127).to(torch.uint8)
        out.append((pages, scales))
    return out[0][0], out[1][0], out[0][1], out[1][1]


def _exact_attend(c, s):
    H, Hk, D = c["H"], c["Hk"], c["D"]
    o = torch.zeros(s["q"].shape, device="cuda", dtype=torch.float64)
    trees = _trees(c) if c["tree"] else None
    for b, first, new, total in _sequences(c):
        table = s["table"][b, : -(-total // c["page"])].long()
        base = total - new
        at, keys = np.arange(base, total)[:, None], np.arange(total)[None]
        sees, position, place = keys <= at, at, keys
        if trees:
            sees = np.tile(keys < base, (new, 1))
            depth = _depths(trees[b])
            for t in range(new):
                a = t
                while a >= 0:
                    sees[t, base + a] = True
                    a = int(trees[b][a])
            position, place = base + depth[:, None], np.concatenate([np.arange(base), base + depth])[None]
        if c["window"]:
            sees = sees & ((position - place < c["window"]) | (place < c["sinks"]))
        sees = torch.from_numpy(sees).cuda()
        far = torch.from_numpy(np.abs(position - keys)).cuda()

        def cached(pages, scales, hk):
            if scales is None:
                return pages[table, :, hk].double().flatten(0, 1)[:total]
            x = pages.view(torch.uint8)[table, :, hk].view(torch.float8_e4m3fn).double()
            return (x * 2.0 ** (scales.view(torch.uint8)[table, hk].double() - 127)[..., None]).flatten(0, 1)[:total]
        for hk in range(Hk):
            k, v = cached(s["k_pages"], s["k_scales"], hk), cached(s["v_pages"], s["v_scales"], hk)
            for h in range(hk * (H // Hk), (hk + 1) * (H // Hk)):
                x = s["q"][first: first + new, h].double() @ k.T / D ** 0.5
                if c["cap"]:
                    x = c["cap"] * torch.tanh(x / c["cap"])
                if c["bias"]:
                    x = x - s["slopes"][h].double() * far
                o[first: first + new, h] = torch.softmax(torch.where(sees, x, -torch.inf), 1) @ v
    return o
