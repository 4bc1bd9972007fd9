"""The operators around `flash_b200.attention` that change its scores or read and write a paged cache, over the sizes their users call them with.

`attention_scored`: scores capped by a tanh, a bias that falls with distance, document and prefix masks, forward alone or with its gradients.
`paged_append` and `paged_attention`: new tokens of a ragged batch put into a cache of pages, and their attention over it.

`listed()` names one call per kind of use and `draw()` gives other sizes of the same kinds. Where `own` is false `run` computes the plain form
in elementary torch operations in 32 bits, else by the package, which is taken from the working folder.
"""
import os
import sys

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def _scored(use, B, H, Hk, M, N, D, dtype, causal, backward, cap=0.0, bias=False, prefix=False, docs=0, len_seed=0, std=2.0, layout="bhld"):
    """`docs`: most documents of a sequence (0: no ids); `len_seed` fixes their lengths and the prefixes'. `std` of q and k: 2 gives scores of
    deviation 4. `layout`: "bhld" contiguous, "blhd" the views that a projection's output [B, L, H, D] is transposed to."""
    return dict(op="scored", use=use, B=B, H=H, Hk=Hk, M=M, N=N, D=D, dtype=dtype, causal=causal, backward=backward, cap=cap, bias=bias, prefix=prefix,
                docs=docs, len_seed=len_seed, std=std, layout=layout)


def _paged(use, op, B, H, Hk, D, dtype, page, longest, chunks, chunk, cap=0.0, bias=False, len_seed=0):
    """`B` sequences, the first `chunks` of them with about `chunk` new tokens and the others with one; `longest` cached tokens at most."""
    return dict(op=op, use=use, B=B, H=H, Hk=Hk, D=D, dtype=dtype, page=page, longest=longest, chunks=chunks, chunk=chunk, cap=cap, bias=bias, len_seed=len_seed)


def listed():
    cases = {
        # The smallest call in use: one short prompt of a small model with capped scores. Launches and host time are all there is.
        "capped_prompt": _scored("prompt", 1, 8, 8, 200, 200, 64, "bf16", True, False, cap=30.0),
        # fp32 step of a check-sized model: distance bias, documents.
        "biased_fp32_step": _scored("fp32", 2, 4, 4, 512, 512, 64, "fp32", True, True, cap=20.0, bias=True, docs=4, len_seed=1),
        # Encoder step with a bias that falls with the distance on both sides, narrow heads, odd length.
        "biased_encoder_step": _scored("encoder", 16, 8, 8, 577, 577, 32, "fp16", False, True, bias=True, std=1.0),
        # Training step of a prefix language model: the prompt sees itself in both directions. Grouped-query heads, projection layout.
        "prefix_step": _scored("prefix", 4, 16, 4, 1500, 1500, 64, "bf16", True, True, prefix=True, len_seed=2, std=1.0, layout="blhd"),
        # Packed pretraining step with capped scores and a distance bias, ragged length.
        "capped_packed_step": _scored("packed", 1, 16, 16, 8111, 8111, 128, "bf16", True, True, cap=50.0, bias=True, docs=4, len_seed=3),
        # Prefill of a long prompt with capped scores and grouped-query heads, the largest call.
        "capped_prefill": _scored("prefill", 1, 32, 8, 5801, 5801, 128, "fp16", True, False, cap=50.0),
        # One token of one conversation, small model, small pages: latency.
        "decode_one": _paged("decode", "attend", 1, 8, 8, 64, "bf16", 16, 700, 0, 1),
        # One token for each of 64 conversations of ragged length, capped scores.
        "decode_batch": _paged("decode", "attend", 64, 32, 8, 128, "bf16", 64, 8192, 0, 1, cap=30.0),
        # One token against a very long cache, eight query heads a kv head: split over the keys.
        "decode_long": _paged("decode", "attend", 1, 64, 8, 128, "fp16", 32, 131072, 0, 1),
        # A server's step: chunks of prompts and single tokens in one ragged batch, distance bias.
        "mixed_batch": _paged("mixed", "attend", 8, 32, 8, 128, "bf16", 16, 8000, 3, 500, bias=True),
        # The cache's side of the same two steps: one new token each, and whole prompts.
        "append_tokens": _paged("append", "append", 64, 32, 8, 128, "bf16", 64, 8192, 0, 1),
        "append_prompts": _paged("append", "append", 8, 32, 8, 128, "bf16", 16, 4000, 8, 3500),
    }
    return [dict(c, name=n) for n, c in cases.items()]


def _log_int(rng, lo, hi):
    """An integer from [lo, hi], even over the logarithm."""
    return min(hi, int(lo * (hi / lo) ** rng.random() + 0.5))


def _draw_one(rng):
    use = rng.choice(("prompt", "fp32", "encoder", "prefix", "packed", "prefill", "decode", "decode", "mixed", "mixed", "append"))
    half = rng.choice(("bf16", "fp16"))
    gqa = rng.choice(((32, 8), (16, 4), (64, 8), (16, 16), (12, 2)))
    cap, bias, seed = rng.choice((0.0, 20.0, 30.0, 50.0)), rng.random() < 0.5, rng.randrange(1 << 20)
    if use == "prompt":
        h, m = rng.choice((4, 8, 12, 16)), _log_int(rng, 1, 1024)
        return _scored(use, rng.choice((1, 1, 2)), h, h, m, m + rng.choice((0, 0, 300)), rng.choice((64, 128)), half, True, False, cap or 30.0, bias)
    if use == "fp32":
        h, m = rng.choice((2, 4, 8)), _log_int(rng, 100, 1024)
        return _scored(use, rng.choice((1, 2, 4)), h, h, m, m, rng.choice((32, 64, 128)), "fp32", True, True, cap, True, rng.random() < 0.3, 4, seed)
    if use == "encoder":
        h, m = rng.choice((6, 8, 16)), _log_int(rng, 196, 1600)
        return _scored(use, rng.choice((8, 16)), h, h, m, m, rng.choice((16, 32, 64)), half, False, True, cap, True, std=1.0)
    if use == "prefix":
        m = _log_int(rng, 256, 4000)
        return _scored(use, rng.choice((1, 2, 4)), gqa[0], gqa[1], m, m, rng.choice((64, 128)), half, True, True, cap, bias, True, 0, seed, 1.0, "blhd")
    if use == "packed":
        h, m = rng.choice((8, 16)), _log_int(rng, 1000, 8111)
        return _scored(use, rng.choice((1, 2)), h, h, m, m, rng.choice((64, 128)), half, True, True, cap or 50.0, bias, False, rng.choice((4, 16)), seed)
    if use == "prefill":
        m = _log_int(rng, 500, 5801)
        return _scored(use, rng.choice((1, 2)), gqa[0], gqa[1], m, m, 128, half, True, False, cap or 50.0, bias)
    page = rng.choice((16, 32, 64, 128))
    if use == "decode":
        b = _log_int(rng, 1, 64)
        return _paged(use, "attend", b, gqa[0], gqa[1], rng.choice((64, 128)), half, page, _log_int(rng, 300, min(131072, (1 << 19) // b)), 0, 1, cap, bias, seed)
    b = _log_int(rng, 1, 16)
    chunk = _log_int(rng, 17, 2048)
    longest = chunk + _log_int(rng, 100, 8000)
    return _paged(use, "attend" if use == "mixed" else "append", b, gqa[0], gqa[1], rng.choice((64, 128)), half, page, longest, rng.randrange(1, b + 1), chunk,
                  cap, bias, seed)


def draw(rng):
    while True:
        c = _draw_one(rng)
        w = work(c)
        if w["flops"] <= 2.7e11 and w["bytes"] <= 1.2e9 and _scores(c) <= 1.05e9:
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
    new[: c["chunks"]] = np.maximum(1, (c["chunk"] * rng.uniform(0.7, 1.0, c["chunks"])).astype(np.int64))
    if c["chunks"]:
        new[0] = c["chunk"]
    total = np.maximum(new, (c["longest"] * rng.uniform(0.2, 1.0, c["B"])).astype(np.int64))
    total[0] = c["longest"]
    return new, total


def _documents(c):
    """Document lengths of each sequence: 1 to `docs` documents of Dirichlet(1) weights."""
    rng, out = np.random.default_rng(c["len_seed"]), []
    for _ in range(c["B"]):
        w = rng.dirichlet(np.ones(int(rng.integers(1, c["docs"] + 1))))
        ends = np.round(np.cumsum(w) / w.sum() * c["N"]).astype(np.int64)
        out.append(np.diff(np.concatenate([[0], ends])))
    return out


def _prefixes(c):
    return np.random.default_rng(c["len_seed"] + 1).integers(c["N"] // 10, c["N"] // 2 + 1, c["B"])


def _visible(c):
    """Unmasked entries of the scores over all sequences and heads."""
    if c["op"] != "scored":
        new, total = _ragged(c)
        return c["H"] * float((new * total - new * (new - 1) // 2).sum())
    M, N = c["M"], c["N"]
    if not c["causal"]:
        return c["B"] * c["H"] * float(M * N)
    total, gap = 0.0, N - M
    for b in range(c["B"]):
        if c["docs"]:
            ends = np.cumsum(_documents(c)[b])
            first = np.repeat(ends - _documents(c)[b], _documents(c)[b])
        else:
            ends, first = np.array([N]), np.zeros(N, dtype=np.int64)
        i = np.arange(N - M, N)
        last = i + 1
        if c["prefix"]:
            end = np.repeat(ends, np.diff(np.concatenate([[0], ends])))[gap:]
            last = np.maximum(last, np.minimum(end, _prefixes(c)[b]))
        total += float((last - first[gap:]).clip(0).sum())
    return c["H"] * total


def work(case):
    """Flops of the unmasked entries alone (2 products forward, 5 backward); each input read and each output written once."""
    c = case
    if c["op"] == "scored":
        size = 4 if c["dtype"] == "fp32" else 2
        q, kv = c["B"] * c["H"] * c["M"] * c["D"] * size, c["B"] * c["Hk"] * c["N"] * c["D"] * size
        tensors = (2 * q + 2 * kv) * (2 if c["backward"] else 1)  # q, k, v, o and dO, dq, dk, dv
        return {"bytes": tensors + (8 * c["B"] * c["N"] if c["docs"] else 0), "flops": (14 if c["backward"] else 4) * c["D"] * _visible(c)}
    new, total = _ragged(c)
    pages = 4 * int((-(-total // c["page"])).sum())
    if c["op"] == "append":
        return {"bytes": 8 * int(new.sum()) * c["Hk"] * c["D"] + pages, "flops": 0}
    return {"bytes": 4 * int(new.sum()) * c["H"] * c["D"] + 4 * int(total.sum()) * c["Hk"] * c["D"] + pages, "flops": 4 * c["D"] * _visible(c)}


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

    s = {"case": c, "cap": c["cap"] or None, "slopes": _slopes(c["H"]) if c["bias"] else None}
    if c["op"] == "scored":
        def tensor(heads, length, std):
            x = values(c["B"], heads, length, c["D"], std=std) if c["layout"] == "bhld" else values(c["B"], length, heads, c["D"], std=std).transpose(1, 2)
            return x
        s |= {"q": tensor(c["H"], c["M"], c["std"]), "k": tensor(c["Hk"], c["N"], c["std"]), "v": tensor(c["Hk"], c["N"], 1.0), "do": None, "ids": None, "prefix": None}
        if c["backward"]:
            s["do"] = tensor(c["H"], c["M"], 1.0)
            for n in ("q", "k", "v"):
                s[n].requires_grad_()
        if c["docs"]:
            row = np.stack([np.repeat(-(np.arange(len(x), dtype=np.int64) + 1), x) for x in _documents(c)])
            s["ids"] = torch.from_numpy(row).cuda()[:, None, :].expand(c["B"], c["H"], c["N"])
        if c["prefix"]:
            s["prefix"] = torch.from_numpy(_prefixes(c).astype(np.int32)).cuda()
        return s
    new, total = _ragged(c)
    pages = -(-total // c["page"])
    n_pages = int(pages.sum()) + 8  # some that belong to nobody
    order = np.random.default_rng(seed).permutation(n_pages)
    table = np.zeros((c["B"], int(pages.max())), dtype=np.int32)
    for b, first in enumerate(np.cumsum(pages) - pages):
        table[b, : pages[b]] = order[first: first + pages[b]]
    T, Hk, D = int(new.sum()), c["Hk"], c["D"]
    s |= {"k_pages": values(n_pages, c["page"], Hk, D), "v_pages": values(n_pages, c["page"], Hk, D), "table": torch.from_numpy(table).cuda(),
          "kv_lens": torch.from_numpy(total.astype(np.int32)).cuda(), "most": int(new.max()),
          "starts": torch.from_numpy(np.concatenate([[0], np.cumsum(new)]).astype(np.int32)).cuda() if c["chunks"] else None}
    if c["op"] == "append":
        s |= {"k": values(T, Hk, D), "v": values(T, Hk, D)}
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
    far = torch.arange(M, device="cuda")[:, None] + max(0, N - M) - torch.arange(N, device="cuda")  # how far the key lies behind
    x = (q @ k.mT).mul_(scale)
    t = None
    if s["cap"]:
        t = x.div_(s["cap"]).tanh_()
        x = t * s["cap"]
    if s["slopes"] is not None:
        x = x - s["slopes"][:, None, None] * far.abs()
    keep = torch.ones(1, 1, M, N, dtype=torch.bool, device="cuda")
    if c["causal"]:
        keep = (far >= 0)[None, None]
        if s["prefix"] is not None:
            keep = keep | (torch.arange(N, device="cuda") < s["prefix"][:, None, None, None])
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
    """Of each sequence and new token: the token's row, whether there is such a token, and its position."""
    B = s["kv_lens"].shape[0]
    starts = s["starts"].long() if s["starts"] is not None else torch.arange(B + 1, device="cuda")
    at = torch.arange(s["most"], device="cuda")
    new = starts[1:] - starts[:-1]
    return starts[:-1, None] + at, at < new[:, None], (s["kv_lens"] - new)[:, None] + at


def _plain_append(s):
    row, real, at = _token_rows(s)
    page = s["table"].long().gather(1, (at // s["case"]["page"]).clamp(max=s["table"].shape[1] - 1))
    row, page, slot = row[real], page[real], (at % s["case"]["page"])[real]
    s["k_pages"][page, slot] = s["k"][row]
    s["v_pages"][page, slot] = s["v"][row]
    return s["k_pages"], s["v_pages"]


def _plain_attend(s):
    c = s["case"]
    B, H, Hk, D, m = c["B"], c["H"], c["Hk"], c["D"], s["most"]
    row, real, at = _token_rows(s)
    k, v = (x[s["table"].long()].reshape(B, -1, Hk, D).permute(0, 2, 1, 3).float() for x in (s["k_pages"], s["v_pages"]))
    N = k.shape[2]
    q = s["q"][row.clamp(max=s["q"].shape[0] - 1)].float()  # [B, m, H, D]
    q = q.reshape(B, m, Hk, H // Hk, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, H // Hk * m, D)
    x = (q @ k.mT).mul_(D ** -0.5).reshape(B, H, m, N)
    if s["cap"]:
        x = x.div_(s["cap"]).tanh_().mul_(s["cap"])
    far = at[:, None, :, None] - torch.arange(N, device="cuda")
    if s["slopes"] is not None:
        x = x - s["slopes"][:, None, None] * far.abs()
    p = _softmax(x, far >= 0)
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
        fb.paged_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["kv_lens"], s["starts"])
        return s["k_pages"], s["v_pages"]
    if c["op"] == "attend":
        return fb.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["kv_lens"], s["starts"], softcap=s["cap"], slopes=s["slopes"])
    mode = fb.SCORE_FUNC_MODE0_NOPE if s["ids"] is None else fb.SCORE_FUNC_MODE1_DOC
    eq = None if s["ids"] is None else s["ids"][:, :, c["N"] - c["M"]:]
    o = fb.attention_scored(s["q"], s["k"], s["v"], c["causal"], None, eq, s["ids"], mode, softcap=s["cap"], slopes=s["slopes"], prefix=s["prefix"])
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
    gap, scale, new = max(0, N - M), 1.0 / D ** 0.5, {"device": "cuda", "dtype": torch.float64}
    o = torch.zeros(B, H, M, D, **new)
    dq, dk, dv = (torch.zeros(B, h, n, D, **new) if c["backward"] else None for h, n in ((H, M), (c["Hk"], N), (c["Hk"], N)))
    keys = torch.arange(N, device="cuda")[None]
    step = max(1, min(M, (1 << 27) // N))
    for b in range(B):
        front = int(s["prefix"][b]) if s["prefix"] is not None else 0
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
                hidden = torch.zeros(at.shape[0], N, dtype=torch.bool, device="cuda")
                if c["causal"]:
                    hidden = (keys > at) & (keys >= front)
                if c["docs"]:
                    ids = s["ids"][b, h]
                    mine = ids[N - M:][rows, None]
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


def _sequences(c, s):
    """(sequence, its first row, new tokens, cached tokens) of each."""
    new, total = _ragged(c)
    first = np.cumsum(new) - new
    return [(b, int(first[b]), int(new[b]), int(total[b])) for b in range(c["B"])]


def _exact_append(c, s):
    k, v, table = s["k_pages"].double(), s["v_pages"].double(), s["table"].long()
    for b, first, new, total in _sequences(c, s):
        at = torch.arange(total - new, total, device="cuda")
        place = table[b, at // c["page"]] * c["page"] + at % c["page"]
        k.flatten(0, 1)[place] = s["k"][first: first + new].double()
        v.flatten(0, 1)[place] = s["v"][first: first + new].double()
    return k, v


def _exact_attend(c, s):
    H, Hk, D = c["H"], c["Hk"], c["D"]
    o = torch.zeros(s["q"].shape, device="cuda", dtype=torch.float64)
    for b, first, new, total in _sequences(c, s):
        pages = s["table"][b, : -(-total // c["page"])].long()
        k, v = (x[pages].flatten(0, 1)[:total] for x in (s["k_pages"], s["v_pages"]))
        at, keys = torch.arange(total - new, total, device="cuda")[:, None], torch.arange(total, device="cuda")[None]
        for h in range(H):
            x = s["q"][first: first + new, h].double() @ k[:, h * Hk // H].double().T / D ** 0.5
            if c["cap"]:
                x = c["cap"] * torch.tanh(x / c["cap"])
            if c["bias"]:
                x = x - s["slopes"][h].double() * (at - keys).abs()
            p = torch.softmax(torch.where(keys > at, -torch.inf, x), 1)
            o[first: first + new, h] = p @ v[:, h * Hk // H].double()
    return o
