"""attention_scored against the plain computation in 64 bits, element by element within bounds derived from the roundings (scored_reference.py)."""
import contextlib
import itertools
import math

import pytest
import torch

from scored_reference import attention_64

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def _inputs(B, H, Hk, M, N, D, dtype, seed, std=1.5, layout="bhld"):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def tensor(h, n, s):
        x = torch.randn((B, h, n, D) if layout == "bhld" else (B, n, h, D), generator=gen, device="cuda") * s
        return (x if layout == "bhld" else x.transpose(1, 2)).to(dtype)

    return tensor(H, M, std), tensor(Hk, N, std), tensor(Hk, N, 1.0), tensor(H, M, 1.0)


def _slopes(H, kind):
    if kind is None:
        return None
    if kind == "series":
        return torch.tensor([2.0 ** (-8 * (h + 1) / H) for h in range(H)], device="cuda")
    if kind == "mixed":  # zero, negative and steep ones
        return torch.tensor([(0.0, -0.01, 3.0, 0.2)[h % 4] for h in range(H)], device="cuda")
    return torch.full((H,), float(kind), device="cuda")


def _docs(B, H, L, seed, per_head=False):
    gen = torch.Generator().manual_seed(seed)
    rows = []
    for _ in range(B * (H if per_head else 1)):
        cuts = torch.sort(torch.randint(1, max(2, L), (3,), generator=gen)).values
        ids = -1 - torch.searchsorted(cuts, torch.arange(L), right=True)
        ids[torch.rand(L, generator=gen) < 0.03] = 5
        rows.append(ids)
    ids = torch.stack(rows).reshape(B, -1, L).cuda()
    return ids.expand(B, H, L)


def _check(got, want, what):
    value, bound = want
    off = (got.double() - value).abs()
    assert torch.isfinite(got).all(), what
    worst = (off / bound).max().item()
    assert worst <= 1, f"{what}: {worst:.2f} times its bound, at most {off.max().item():.3g} off"


def _run(fb, q, k, v, do, causal, eq=None, ek=None, cap=None, slopes=None, prefix=None, sm_scale=None):
    a, b, c = (x.detach().requires_grad_() for x in (q, k, v))
    o = fb.attention_scored(a, b, c, causal, sm_scale, eq, ek, 0 if eq is None else 1, softcap=cap, slopes=slopes, prefix=prefix)
    grads = torch.autograd.grad(o, (a, b, c), do)
    with torch.no_grad():
        assert torch.equal(o, fb.attention_scored(q, k, v, causal, sm_scale, eq, ek, 0 if eq is None else 1, softcap=cap, slopes=slopes, prefix=prefix))
    fb.check_status()
    return dict(zip(("o", "dq", "dk", "dv"), (o.detach(), *grads)))


def _compare(q, k, v, do, causal, **kw):
    import flash_b200 as fb
    got = _run(fb, q, k, v, do, causal, **kw)
    want = attention_64(q, k, v, do, causal, kw.get("sm_scale"), kw.get("eq"), kw.get("ek"), kw.get("cap"), kw.get("slopes"), kw.get("prefix"))
    for name in ("o", "dq", "dk", "dv"):
        _check(got[name], want[name], name)
    return got, want


# (B, H, Hk, M, N, D): one token, tiles that end inside, more keys than queries, grouped heads, few queries (packed heads, runs of keys)
SHAPES = [(1, 1, 1, 1, 1, 64), (2, 2, 1, 129, 129, 128), (1, 4, 2, 200, 333, 64), (2, 8, 2, 1, 700, 128), (1, 4, 1, 30, 2500, 64), (1, 3, 1, 100, 1300, 128),
          (1, 2, 2, 257, 300, 32), (2, 4, 4, 96, 96, 16), (1, 2, 1, 640, 640, 128)]
CHANGES = [dict(cap=20.0), dict(slopes="series"), dict(cap=5.0, slopes="mixed")]


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("change", CHANGES, ids=["cap", "bias", "both"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_shapes(shape, change, causal, dtype):
    B, H, Hk, M, N, D = shape
    q, k, v, do = _inputs(*shape, dtype, 7)
    _compare(q, k, v, do, causal, cap=change.get("cap"), slopes=_slopes(H, change.get("slopes")))


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("prefix,kind", [((0, 300), torch.int32), ((-5, 1000), torch.int32), ((130, 1 << 40), torch.int64), ((1, 127), torch.int64)])
@pytest.mark.parametrize("D,M,N", [(64, 300, 300), (128, 140, 420), (32, 5, 300)])
def test_prefix(D, M, N, prefix, kind, dtype):
    q, k, v, do = _inputs(2, 4, 2, M, N, D, dtype, 8)
    p = torch.tensor(prefix, dtype=kind, device="cuda")
    _compare(q, k, v, do, True, prefix=p)
    _compare(q, k, v, do, True, prefix=p, cap=10.0, slopes=_slopes(4, "mixed"))


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("per_head", [False, True])
@pytest.mark.parametrize("causal,prefix", [(True, None), (False, None), (True, (90, 300))])
def test_documents(causal, prefix, per_head, dtype):
    B, H, Hk, L, D = 2, 4, 2, 390, 64
    q, k, v, do = _inputs(B, H, Hk, L, L, D, dtype, 9)
    ids = _docs(B, H, L, 10, per_head)
    prefix = None if prefix is None else torch.tensor(prefix, dtype=torch.int32, device="cuda")
    for cap, slopes in ((15.0, None), (None, "series"), (6.0, "mixed")):
        _compare(q, k, v, do, causal, eq=ids, ek=ids, cap=cap, slopes=_slopes(H, slopes), prefix=prefix)


def test_documents_over_many_blocks():
    """The plan of long id rows, built by three kernels, and queries of scattered documents without a causal mask."""
    B, H, L, D = 1, 2, 4700, 64
    q, k, v, do = _inputs(B, H, 1, L, L, D, BF16, 11)
    ids = _docs(B, H, L, 12)
    _compare(q, k, v, do, True, eq=ids, ek=ids, cap=20.0, slopes=_slopes(H, "series"), prefix=torch.tensor([1500], dtype=torch.int32, device="cuda"))
    scattered = ids[:, :1, torch.randperm(L, device="cuda")].expand(B, H, L)
    _compare(q, k, v, do, False, eq=scattered, ek=ids, cap=20.0)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("causal", [True, False])
def test_rows_without_a_key(causal, dtype):
    import flash_b200 as fb
    q, k, v, do = _inputs(2, 2, 2, 260, 260, 64, dtype, 13)
    eq = torch.full((2, 1, 260), -1, device="cuda")
    ek = torch.full((2, 1, 260), -1, device="cuda")
    eq[0, 0, 100:180] = -9  # nobody's
    ek[1] = -2              # a whole sequence without keys
    eq, ek = eq.expand(2, 2, 260), ek.expand(2, 2, 260)
    got, want = _compare(q, k, v, do, causal, eq=eq, ek=ek, cap=10.0, slopes=_slopes(2, "series"))
    empty = ~want["keep"].any(-1)[:, 0]
    assert empty[0, 100:180].all() and empty[1].all()
    for b in range(2):
        assert (got["o"][b][:, empty[b]] == 0).all() and (got["dq"][b][:, empty[b]] == 0).all()
    assert (got["dk"][1] == 0).all() and (got["dv"][1] == 0).all()


@pytest.mark.parametrize("cap", [1e-6, 0.5, 1.0, 300.0, 1e6])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_caps_of_every_size(cap, dtype):
    """Scores on both sides of the cap, within one call: both forms of the tanh, also next to each other."""
    q, k, v, do = _inputs(1, 2, 2, 200, 200, 64, dtype, 14)
    q[:, :, 50:60] *= 8
    q[:, :, 100:150] *= 0.01
    _compare(q, k, v, do, True, cap=cap)


def test_scores_that_are_not_finite_in_the_type_of_the_inputs():
    """fp16 products beyond 65504, capped."""
    q, k, v, do = _inputs(1, 2, 2, 150, 150, 64, FP16, 15, std=60.0)
    _compare(q, k, v, do, True, cap=30.0)


def test_strides_and_scale():
    q, k, v, do = _inputs(2, 4, 2, 190, 190, 64, BF16, 16, layout="blhd")
    _compare(q, k, v, do, True, cap=8.0, slopes=_slopes(4, "series"), sm_scale=0.3)
    wide = torch.randn(2, 190, 4, 3, 67, device="cuda", dtype=BF16)[..., 1:65]  # nothing that a tensor map takes
    a, b, c = (wide[:, :, :, i].transpose(1, 2) for i in range(3))
    _compare(a, b, c, do[:, :, :, torch.arange(64, device="cuda").flip(0)].transpose(2, 3).contiguous().transpose(2, 3), True, cap=8.0)
    slopes = torch.rand(8, device="cuda")[::2]
    prefix = torch.tensor([[7, 0], [100, 0]], dtype=torch.int32, device="cuda")[:, 0]
    _compare(q, k, v, do, True, slopes=slopes, prefix=prefix)
    _compare(q, k, v, do[:, :, :1].expand(2, 4, 190, 64), True, slopes=slopes)  # a broadcast gradient


def test_without_changes_it_is_attention():
    import flash_b200 as fb
    q, k, v, do = _inputs(1, 4, 2, 300, 300, 64, BF16, 17)
    for softcap in (None, 0, 0.0):
        assert torch.equal(fb.attention_scored(q, k, v, True, softcap=softcap), fb.attention(q, k, v, True))
    # nothing but zeros in the changes: the same function by the other instances
    zero = fb.attention_scored(q, k, v, True, slopes=torch.zeros(4, device="cuda"), prefix=torch.zeros(1, dtype=torch.int32, device="cuda"))
    want = attention_64(q, k, v, do, True, None, None, None, None, None, None)
    _check(zero, want["o"], "o")


def test_gradients_against_differences():
    """A directional derivative of sum(o * do) by central differences of the fp32 kernels' forward. With a step of h the difference is off by h^2 / 6 of
    the third derivative and by the forward's rounding over h: with h = 2^-6 some 1e-3 and 1e-4 of the derivative's size here; 5e-3 is asked for."""
    import flash_b200 as fb
    q, k, v, do = _inputs(1, 2, 1, 70, 90, 32, FP32, 18, std=0.7)
    kw = dict(cap=2.0, slopes=_slopes(2, "series"), prefix=torch.tensor([40], dtype=torch.int32, device="cuda"))
    got = _run(fb, q, k, v, do, True, **kw)
    for i, name in enumerate(("dq", "dk", "dv")):
        x = [q, k, v]
        way = got[name] / got[name].norm()  # the steepest one
        h = 2.0 ** -6
        ends = []
        for sign in (1, -1):
            y = list(x)
            y[i] = x[i] + sign * h * way
            ends.append((fb.attention_scored(*y, True, softcap=2.0, slopes=kw["slopes"], prefix=kw["prefix"]).double() * do.double()).sum())
        assert abs((ends[0] - ends[1]) / (2 * h) / got[name].double().norm() - 1) < 5e-3, name


def test_captured_forward_and_backward_on_new_values():
    import flash_b200 as fb
    q, k, v, do = _inputs(2, 4, 2, 300, 300, 128, BF16, 19)
    ids = _docs(2, 4, 300, 20)
    slopes, prefix = _slopes(4, "series"), torch.tensor([20, 200], dtype=torch.int32, device="cuda")
    call = dict(eq=ids, ek=ids, cap=10.0, slopes=slopes, prefix=prefix)
    _run(fb, q, k, v, do, True, **call)
    a, b, c = (x.detach().clone().requires_grad_() for x in (q, k, v))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        o = fb.attention_scored(a, b, c, True, None, ids, ids, 1, softcap=10.0, slopes=slopes, prefix=prefix)
        grads = torch.autograd.grad(o, (a, b, c), do)
    q2, k2, v2, do2 = _inputs(2, 4, 2, 300, 300, 128, BF16, 21)
    with torch.no_grad():
        for x, y in ((a, q2), (b, k2), (c, v2)):
            x.copy_(y)
    do.copy_(do2)
    prefix.copy_(torch.tensor([150, 3]))
    slopes.mul_(0.5)
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    want = _run(fb, q2, k2, v2, do2, True, **call)
    for got, name in zip((o, *grads), ("o", "dq", "dk", "dv")):
        assert torch.equal(got, want[name]), name


def test_two_streams_at_once():
    import flash_b200 as fb
    sets = [_inputs(1, 8, 8, 900, 900, 64, BF16, 30 + i) for i in range(2)]
    want = [_run(fb, *s, True, cap=10.0 + i) for i, s in enumerate(sets)]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for i, (s, st) in enumerate(zip(sets, streams)):
            with torch.cuda.stream(st):
                a, b, c = (x.detach().requires_grad_() for x in s[:3])
                o = fb.attention_scored(a, b, c, True, softcap=10.0 + i)
                got.append((i, (o.detach(), *torch.autograd.grad(o, (a, b, c), s[3]))))
    torch.cuda.synchronize()
    for i, outs in got:
        for x, name in zip(outs, ("o", "dq", "dk", "dv")):
            assert torch.equal(x, want[i][name])


def test_tiles_skipped_or_not_give_the_same(monkeypatch):
    """The environment's switches walk every tile and evaluate every mask entry by entry."""
    import flash_b200 as fb
    q, k, v, do = _inputs(1, 2, 1, 520, 520, 64, BF16, 22)
    ids = _docs(1, 2, 520, 23)
    kw = dict(eq=ids, ek=ids, cap=10.0, slopes=_slopes(2, "series"), prefix=torch.tensor([140], dtype=torch.int32, device="cuda"))
    want = _run(fb, q, k, v, do, True, **kw)
    monkeypatch.setenv("FA_B200_ALL_PARTIAL", "1")
    for name, x in _run(fb, q, k, v, do, True, **kw).items():
        assert torch.equal(x, want[name]), name
    monkeypatch.setenv("FA_B200_NO_SKIP", "1")
    exact = attention_64(q, k, v, do, True, None, ids, ids, 10.0, kw["slopes"], kw["prefix"])
    for name, x in _run(fb, q, k, v, do, True, **kw).items():
        _check(x, exact[name], name)


def test_refusals():
    import flash_b200 as fb
    q, k, v, _ = _inputs(2, 4, 2, 32, 32, 64, BF16, 24)
    for bad in (-1.0, 1e-7, 2e6, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="softcap"):
            fb.attention_scored(q, k, v, True, softcap=bad)
    for bad in (torch.ones(2, device="cuda"), torch.ones(4, device="cuda", dtype=torch.float64), torch.ones(4), [1.0] * 4,
                torch.ones(4, device="cuda", requires_grad=True)):
        with pytest.raises(ValueError):
            fb.attention_scored(q, k, v, True, slopes=bad)
    for bad in (torch.ones(2), torch.ones(2, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda"), 5):
        with pytest.raises(ValueError):
            fb.attention_scored(q, k, v, True, prefix=bad)
    with pytest.raises(ValueError, match="causal"):
        fb.attention_scored(q, k, v, False, prefix=torch.ones(2, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError, match="dtype"):
        fb.attention_scored(q, k.half(), v, True, softcap=5.0)
    with pytest.raises(AssertionError):
        fb.attention_scored(q, k[:, :, :8], v[:, :, :8], True, softcap=5.0)
    with pytest.raises(AssertionError):
        fb.attention_scored(q, k, v, True, eq=torch.zeros(2, 4, 32, device="cuda", dtype=torch.int64), softcap=5.0)
    a = q.detach().requires_grad_()
    g, = torch.autograd.grad(fb.attention_scored(a, k, v, True, softcap=5.0).sum(), a, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_both_ways_through_the_host_give_the_same(monkeypatch):
    """The native host call and its autograd node, and the ones in Python: a call that the kernels do not take as it is, and hooks on saved tensors, go that way."""
    import flash_b200 as fb
    from flash_b200 import ops
    q, k, v, do = _inputs(2, 4, 2, 260, 260, 64, BF16, 40)
    ids, slopes, prefix = _docs(2, 4, 260, 41), _slopes(4, "series"), torch.tensor([100, 9], dtype=torch.int32, device="cuda")
    for kw in (dict(cap=9.0), dict(slopes=slopes, prefix=prefix), dict(cap=9.0, eq=ids, ek=ids, prefix=prefix)):
        want = _run(fb, q, k, v, do, True, **kw)
        with monkeypatch.context() as m:
            m.setattr(ops, "PROFILE", [])
            other = _run(fb, q, k, v, do, True, **kw)
        with torch.autograd.graph.saved_tensors_hooks(lambda x: x, lambda x: x):
            hooked = _run(fb, q, k, v, do, True, **kw)
        for name in want:
            assert torch.equal(want[name], other[name]) and torch.equal(want[name], hooked[name]), name


def test_saved_tensors_that_change_are_noticed():
    import flash_b200 as fb
    q, k, v, do = _inputs(1, 4, 4, 40, 40, 64, BF16, 42)
    for victim in ("slopes", "prefix"):
        kw = dict(slopes=_slopes(4, "series"), prefix=torch.tensor([10], dtype=torch.int32, device="cuda"))
        a = q.detach().requires_grad_()
        o = fb.attention_scored(a, k, v, True, **kw)
        kw[victim].add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            o.backward(do)


def _with_a_time_out_on_record():
    """The status word as a bounded wait that ran out leaves it (nothing waits, faults or hangs here)."""
    from flash_b200 import ops
    ops._status_word(torch.device("cuda", torch.cuda.current_device())).fill_(142)


def test_after_a_time_out_results_are_nan_until_it_has_been_read():
    import flash_b200 as fb
    q, k, v, do = _inputs(1, 4, 2, 300, 300, 64, BF16, 43)
    for kw in (dict(softcap=9.0), dict(slopes=_slopes(4, "series")), dict(prefix=torch.tensor([70], dtype=torch.int32, device="cuda"))):
        a, b, c = (x.detach().requires_grad_() for x in (q, k, v))
        o = fb.attention_scored(a, b, c, True, **kw)
        want = torch.autograd.grad(o, (a, b, c), do, retain_graph=True)
        _with_a_time_out_on_record()
        lost = fb.attention_scored(q, k, v, True, **kw)
        grads = torch.autograd.grad(o, (a, b, c), do, retain_graph=True)
        assert all(torch.isnan(x).all() for x in (lost, *grads))
        with pytest.raises(RuntimeError, match="role 42"):
            fb.check_status()
        assert torch.equal(fb.attention_scored(q, k, v, True, **kw), o)
        assert all(torch.equal(x, y) for x, y in zip(torch.autograd.grad(o, (a, b, c), do), want))


def test_gradients_where_a_few_keys_carry_a_row():
    """Scores of deviation 9. Each of dQ's and dK's two roundings (of dS and of the result) is off by u / sqrt(3) at most in the mean square, u = 2^-8; delta adds what
    the rounding of P puts into O, as much again at most: 1.75 u / sqrt(3) = 3.9e-3 of the whole, where a delta from the rounded O alone had 4.5e-3."""
    import flash_b200 as fb
    q, k, v, do = _inputs(1, 4, 4, 1024, 1024, 128, BF16, 44, std=3.0)
    got = _run(fb, q, k, v, do, True, cap=50.0)
    want = attention_64(q, k, v, do, True, None, None, None, 50.0, None, None)
    for name in ("dq", "dk"):
        value = want[name][0]
        assert ((got[name].double() - value).norm() / value.norm()).item() < 3.9e-3, name


def test_what_the_node_saves_is_freed_with_its_gradients():
    """Between the call and the end of this test the output and the gradient of q stay; the LSE and what the rounding of the output has left out do not."""
    import flash_b200 as fb
    q, k, v, do = _inputs(1, 8, 8, 1024, 1024, 128, BF16, 61)
    size = q.numel() * q.element_size()
    for hooked in (False, True):  # the native node, and the one in Python
        a = q.detach().requires_grad_()
        before = torch.cuda.memory_allocated()
        with (torch.autograd.graph.saved_tensors_hooks(lambda x: x, lambda x: x) if hooked else contextlib.nullcontext()):
            o = fb.attention_scored(a, k, v, True, softcap=20.0)
        o.backward(do)
        torch.cuda.synchronize()
        assert 2 * size <= torch.cuda.memory_allocated() - before < 2 * size + size // 2
        del o, a


@pytest.mark.parametrize("slopes", [None, "series"])
@pytest.mark.parametrize("times", [0.6, 1.5, 3.9, 12.0])
@pytest.mark.parametrize("D, dtype", [(64, FP16), (128, BF16)])
def test_scores_up_to_so_many_caps(times, slopes, D, dtype):
    """Each form of the tanh by itself, in whole tiles and masked ones."""
    q, k, v, do = _inputs(1, 2, 2, 300, 300, D, dtype, 62)
    cap = (q.double() @ k.double().mT).abs().max().item() / D ** 0.5 / times
    _compare(q, k, v, do, True, cap=cap, slopes=_slopes(2, slopes))


@pytest.mark.parametrize("slopes", [None, "series"])
@pytest.mark.parametrize("cap", [100.0, 3.0, 0.2])
def test_a_key_that_is_not_a_number_behind_the_mask(cap, slopes):
    """Rows in front of it have the bits that they have with a key of zeros there, also beside it in a pair of scores."""
    import flash_b200 as fb
    for N, at in ((300, 101), (300, 290), (40, 30)):
        q, k, v, _ = _inputs(1, 2, 1, N, N, 64, BF16, 63)
        k[:, :, at] = 0
        with torch.no_grad():
            want = fb.attention_scored(q, k, v, True, softcap=cap, slopes=_slopes(2, slopes))
            k[:, :, at] = float("nan")
            got = fb.attention_scored(q, k, v, True, softcap=cap, slopes=_slopes(2, slopes))
        assert torch.equal(got[:, :, :at], want[:, :, :at]) and torch.isnan(got[:, :, at:]).all()


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("M, N, slopes, splits", [(600, 600, None, 1), (600, 600, "series", 1), (40, 2500, None, 1), (16, 4000, "series", 5)])
def test_a_prefix_that_the_kernel_directly_before_writes(M, N, slopes, splits, captured):
    """The build of a plan lets its dependents begin before it has written anything: its first query's code (the largest int32 for an id that is not negative, else the
    id) is the prefix of the forward behind it, all keys visible or the causal mask alone, in turn. The bits of forwards that the host has waited in front of."""
    import ctypes
    from flash_b200 import _lib, ops
    lib, H, D, L, n = _lib.load(), 8, 64, 4096, 8
    q, k, v, _ = _inputs(1, H, H, M, N, D, BF16, 64)
    slopes = _slopes(H, slopes)
    prob, build = ops._problem(1, H, H, M, N, D, BF16, True, 0, 1, D ** -0.5), ops._problem(1, 1, 1, L, L, D, BF16, True, 1, 1, 1.0)
    status, size = torch.zeros(1, dtype=torch.int32, device="cuda"), ctypes.c_size_t()
    _lib.check(lib.fa_plan_bytes(build, size), "fa_plan_bytes")
    plan = torch.zeros(size.value // 4, dtype=torch.int32, device="cuda")
    ids = [torch.full((1, 1, L), x, dtype=torch.int32, device="cuda") for x in (-1, 5)]
    lse, work = torch.empty(1, H, lib.fa_padded_rows(M), device="cuda"), None
    if splits > 1:
        need = ctypes.c_size_t()
        _lib.check(lib.fa_fwd_workspace_bytes(prob, splits, need), "fa_fwd_workspace_bytes")
        work = torch.empty(need.value, dtype=torch.uint8, device="cuda")
    scores = _lib.Scores(0.0, None if slopes is None else slopes.data_ptr(), plan.data_ptr())
    t = [ops._tensor(x) for x in (q, k, v)]

    def run(outs, wait):
        s = ops._stream()
        for i, o in enumerate(outs):
            e = ops._ids(ids[i % 2])
            _lib.check(lib.fa_plan_build(build, e, e, plan.data_ptr(), size.value, status.data_ptr(), s), "fa_plan_build")
            if wait:
                torch.cuda.synchronize()
            _lib.check(lib.fa_fwd_scored(prob, scores, *t, ops._tensor(o), None, lse.data_ptr(), None, splits, None if work is None else work.data_ptr(),
                                         0 if work is None else work.numel(), status.data_ptr(), s), "fa_fwd_scored")

    want, got = ([torch.empty_like(q) for _ in range(n)] for _ in range(2))
    run(want, True)
    torch.cuda.synchronize()
    assert not torch.equal(want[0], want[1])
    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run(got, False)
    for _ in range(5):
        if captured:
            graph.replay()
        else:
            torch.cuda._sleep(3_000_000)
            run(got, False)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want, strict=True))
    assert int(status.item()) == 0


def _outliers(M, N, D, dtype, seed, q_rows, key, times):
    """Ordinary inputs, and the same with some queries and a key so many times as large; the last query and `q_rows` have no gradient."""
    q, k, v, do = _inputs(1, 4, 2, M, N, D, dtype, seed)
    do[:, :, [*q_rows, M - 1]] = 0
    big_q, big_k = q.clone(), k.clone()
    big_q[:, :, q_rows] *= times
    big_k[:, :, key] *= times
    return q, k, v, do, big_q, big_k


@pytest.mark.parametrize("slopes", [None, "series"])
@pytest.mark.parametrize("dtype, D, M, N, cap", [(FP16, 64, 300, 300, 1e4), (FP16, 128, 280, 400, 1e4), (FP16, 64, 20, 700, 1e4), (BF16, 128, 700, 700, 1e5), (BF16, 64, 300, 300, 1e6)])
def test_a_score_beyond_a_large_cap_among_ordinary_ones(dtype, D, M, N, cap, slopes):
    """Queries of which all scores, and a last key of which the last query's score, are beyond the cap: all other rows, and the gradients of all keys (those queries have
    none), are those of ordinary inputs, within the bounds of these."""
    import flash_b200 as fb
    rows, slopes = [i for i in (5, 70, 150) if i < M - 1], _slopes(4, slopes)
    q, k, v, do, big_q, big_k = _outliers(M, N, D, dtype, 65, rows, N - 1, 0.8 * cap if dtype == FP16 else 4 * cap)
    want = attention_64(q, k, v, do, True, None, None, None, cap, slopes, None)
    got = _run(fb, big_q, big_k, v, do, True, cap=cap, slopes=slopes)
    plain = torch.ones(M, dtype=torch.bool, device="cuda")
    plain[[*rows, M - 1]] = False
    for name in ("o", "dq"):
        _check(got[name][:, :, plain], tuple(x[:, :, plain] for x in want[name]), name)
    for name in ("dk", "dv"):
        _check(got[name], want[name], name)


@pytest.mark.parametrize("cap", [3.0, 30.0, 1e4])
@pytest.mark.parametrize("slopes", [None, "mixed"])
@pytest.mark.parametrize("dtype, D, M, N", [(BF16, 64, 300, 300), (FP16, 128, 500, 500), (BF16, 128, 140, 333), (FP16, 64, 25, 700)])
@pytest.mark.parametrize("hidden", ["ahead", "other document"])
def test_a_hidden_key_beyond_the_cap_leaves_all_bits(hidden, dtype, D, M, N, slopes, cap):
    """One that only the last query sees, which has no gradient, or one of a document that no query is of, in tiles with others."""
    import flash_b200 as fb
    key, kw = N - 1, dict(cap=cap, slopes=_slopes(4, slopes))
    if hidden != "ahead":
        key = N - 30
        ids = torch.full((1, 1, N), -1, dtype=torch.int32, device="cuda")
        ids[..., N // 2:] = -2
        kw["eq"] = ids[..., N - M:].clone().expand(1, 4, M)
        ids[..., key] = -9
        kw["ek"] = ids.expand(1, 4, N)
    q, k, v, do, _, big_k = _outliers(M, N, D, dtype, 66, [], key, 10 * cap)
    if dtype == FP16:
        big_k = big_k.clamp(-6e4, 6e4)
    for causal in (True, False) if hidden != "ahead" else (True,):
        want, got = (_run(fb, q, x, v, do, causal, **kw) for x in (k, big_k))
        rows = M - 1 if hidden == "ahead" else M
        for name in ("o", "dq", "dk", "dv"):
            n = rows if name in ("o", "dq") else N
            assert torch.equal(got[name][:, :, :n], want[name][:, :, :n]), (name, causal)


def _capped_scores(dtype, cap, s, N, slopes=None):
    """What the kernels make of scores s (fp32, of up to 24 bits), one a row, each for N keys alike: the logarithm of the sum of N equal exponentials, less log N."""
    from flash_b200 import _lib, ops
    import ctypes
    M, D = s.numel(), 16
    q, rest = torch.zeros(1, 1, M, D, dtype=dtype, device="cuda"), s.clone()
    for i in range(3):  # parts whose sum, in fp32, is the score
        q[0, 0, :, i] = rest.to(dtype)
        rest -= q[0, 0, :, i].float()
    assert (rest == 0).all()
    k = torch.zeros(1, 1, N, D, dtype=dtype, device="cuda")
    k[..., :3] = 1
    o, lib, status = torch.empty_like(q), _lib.load(), torch.zeros(1, dtype=torch.int32, device="cuda")
    prob = ops._problem(1, 1, 1, M, N, D, dtype, False, 0, 1, 1.0)
    lse = torch.empty(1, 1, lib.fa_padded_rows(M), device="cuda")
    t = [ops._tensor(x) for x in (q, k, k, o)]
    scores = _lib.Scores(cap, None if slopes is None else slopes.data_ptr(), None)
    _lib.check(lib.fa_fwd_scored(prob, scores, *t, None, lse.data_ptr(), None, 1, None, 0, status.data_ptr(), ops._stream()), "fa_fwd_scored")
    assert int(status.item()) == 0
    return lse[0, 0, :M].double() * math.log(2) - math.log(N)


@pytest.mark.parametrize("slopes", [False, True])
@pytest.mark.parametrize("N", [128, 1])  # without a mask, and with one
@pytest.mark.parametrize("cap", [1e-3, 1.0, 30.0, 64.0, 65.0, 320.0, 330.0, 2000.0, 6000.0, 5e4, 1e6])
def test_how_exact_a_capped_score_is(cap, N, slopes):
    """Scores from 1e-4 to 3 caps of both signs, mixed over the rows, so that the warps have both forms of the tanh side by side.
    The polynomial: its fit, 3.0e-6 up to a cap of 64, 6e-7 up to one of 320 and 8e-8 beyond, and 4e-7 for its coefficients' rounding and four FMAs. The other form, a - 2 a r with
    r = 1 / (1 + e): an exp2 and a reciprocal to 2^-22 and 2^-23, the argument, the sum and the product to 2^-24, at most 5e-7 of the cap; it begins at 0.9 caps, 0.75, 0.6, or
    (where a coefficient leaves fp32's range) 0.24 or 0.125. The sum's logarithm 2^-22 of its value and 2e-6."""
    gen = torch.Generator(device="cuda").manual_seed(67)
    t = torch.logspace(-4, 0.5, 1024, device="cuda", dtype=torch.float64)[torch.randperm(1024, generator=gen, device="cuda")]
    s = (t * cap * (1 - 2 * torch.randint(0, 2, t.shape, generator=gen, device="cuda"))).float()
    got = _capped_scores(BF16, cap, s, N, torch.zeros(1, device="cuda") if slopes else None)
    want = cap * torch.tanh(s.double() / cap)
    bound = (4e-6 if cap <= 64 else 1e-6 if cap <= 320 else 5e-7) * want.abs()
    if cap > 64:
        bound = torch.where(s.abs() > cap / 8, torch.full_like(bound, 5.5e-7 * cap), bound)
    bound = bound + 2.0 ** -22 * want.abs() + 2e-6
    off = (got - want).abs()
    assert (off <= bound).all(), (off / bound).max().item()


def test_tangents_are_refused():
    import flash_b200 as fb
    import torch.autograd.forward_ad as fwad
    q, k, v, _ = _inputs(1, 4, 2, 40, 40, 64, BF16, 68)
    with fwad.dual_level():
        dual = lambda x: fwad.make_dual(x, torch.ones_like(x))  # noqa: E731
        for args, slopes in (((dual(q), k, v), None), ((q, k, dual(v)), None), ((q, k, v), dual(_slopes(4, "series")))):
            with pytest.raises((RuntimeError, NotImplementedError)):
                fb.attention_scored(*args, True, softcap=9.0, slopes=slopes)
        plain = fb.attention_scored(q, k, v, True, softcap=9.0)
    assert torch.equal(plain, fb.attention_scored(q, k, v, True, softcap=9.0))


def test_slopes_that_are_a_parameter_without_grad_mode(monkeypatch):
    """As other inputs that would ask for a gradient: refused under grad mode, taken without, by either way through the host."""
    import flash_b200 as fb
    from flash_b200 import ops
    q, k, v, _ = _inputs(1, 4, 2, 40, 40, 64, BF16, 69)
    slopes = torch.nn.Parameter(_slopes(4, "series"))
    pages, table, lens = k.transpose(1, 2)[:, :32].reshape(2, 16, 2, 64).contiguous(), torch.tensor([[0, 1]], dtype=torch.int32, device="cuda"), torch.tensor([32], dtype=torch.int32, device="cuda")
    calls = (lambda s: fb.attention_scored(q, k, v, True, slopes=s), lambda s: fb.paged_attention(q[0, :, :1].transpose(0, 1), pages, pages, table, lens, slopes=s))
    for profile in (None, []):
        monkeypatch.setattr(ops, "PROFILE", profile)
        for call in calls:
            with pytest.raises(ValueError, match="gradient"):
                call(slopes)
            want = call(slopes.detach())
            for off in (torch.no_grad, torch.inference_mode):
                with off():
                    got = call(slopes)
                assert torch.equal(got, want) and not got.requires_grad


@pytest.mark.parametrize("dtype, D", [(BF16, 128), (FP16, 64), (BF16, 32)])
def test_what_the_rounding_of_a_forward_in_runs_has_left_out(dtype, D):
    """Against the runs' own rows, merged here in 64 bits: o and the rest together have them to 2^-21 (the kernel's sums in fp32) and the rounding of the rest."""
    import ctypes
    from flash_b200 import _lib, ops
    B, H, M, N, splits = 2, 4, 21, 1500, 5
    q, k, v, _ = _inputs(B, H, 2, M, N, D, dtype, 70)
    lib, status, size, dk = _lib.load(), torch.zeros(1, dtype=torch.int32, device="cuda"), ctypes.c_size_t(), 128 if D > 64 else 64
    prob, o, rest = ops._problem(B, H, 2, M, N, D, dtype, True, 0, 1, D ** -0.5), torch.empty_like(q), torch.empty_like(q)
    _lib.check(lib.fa_fwd_workspace_bytes(prob, splits, size), "fa_fwd_workspace_bytes")
    work, lse = torch.empty(size.value // 4, device="cuda"), torch.empty(B, H, lib.fa_padded_rows(M), device="cuda")
    _lib.check(lib.fa_fwd_scored(prob, _lib.Scores(9.0, None, None), *(ops._tensor(x) for x in (q, k, v, o)), None, lse.data_ptr(), None, splits, work.data_ptr(),
                                 size.value, status.data_ptr(), ops._stream()), "fa_fwd_scored")
    _lib.check(lib.fa_fwd_rest(prob, splits, work.data_ptr(), size.value, rest.data_ptr(), status.data_ptr(), ops._stream()), "fa_fwd_rest")
    assert int(status.item()) == 0
    parts = work[: splits * B * H * M * dk].reshape(splits, B, H, M, dk)[..., :D].double()
    weight = torch.softmax(work[splits * B * H * M * dk:][: B * H * M * splits].reshape(B, H, M, splits).double() * math.log(2), -1)
    value = torch.einsum("bhms,sbhmd->bhmd", weight, parts)
    off = (o.double() + rest.double() - value).abs()
    u = torch.finfo(dtype).eps / 2
    size_of = torch.einsum("bhms,sbhmd->bhmd", weight, parts.abs())
    assert (off <= 2.0 ** -21 * size_of + u * (u * value.abs()) + torch.finfo(dtype).smallest_normal).all()
    assert ((o.double() - value).abs() > 2.0 ** -18 * size_of).any()


@pytest.mark.parametrize("hooked", [False, True])  # the native node, and the one in Python
def test_gradients_of_few_queries_where_a_few_keys_carry_a_row(hooked):
    """As of many, in test_gradients_where_a_few_keys_carry_a_row: 3.9e-3 of dQ and dK, also where the forward is cut into runs of keys (4.7e-3 with a delta from the rounded O alone)."""
    import flash_b200 as fb
    B, H, M, N, D = 1, 4, 64, 2048, 128
    assert fb.forward_splits(B, H, H, M, N, D, BF16, True, 0) > 1
    q, k, v, do = _inputs(B, H, H, M, N, D, BF16, 71, std=4.0)
    with (torch.autograd.graph.saved_tensors_hooks(lambda x: x, lambda x: x) if hooked else contextlib.nullcontext()):
        got = _run(fb, q, k, v, do, True, cap=100.0)
    want = attention_64(q, k, v, do, True, None, None, None, 100.0, None, None)
    for name in ("dq", "dk"):
        value = want[name][0]
        assert ((got[name].double() - value).norm() / value.norm()).item() < 3.9e-3, name


@pytest.mark.parametrize("hooked", [False, True])  # the native node, and the one in Python
def test_second_gradients_are_refused_beside_others(hooked):
    """A penalty on the gradients, added to a loss that has gradients of its own, raises: nothing of it is lost. The first gradients are what they are without a graph."""
    import flash_b200 as fb
    q, k, v, do = _inputs(1, 4, 2, 40, 40, 64, BF16, 72)
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]

    def forward():
        with (torch.autograd.graph.saved_tensors_hooks(lambda x: x, lambda x: x) if hooked else contextlib.nullcontext()):
            return fb.attention_scored(*leaves, True, softcap=5.0)

    want = torch.autograd.grad(forward(), leaves, do)
    for asks in (False, True):
        o = forward()
        grads = torch.autograd.grad(o, leaves, do.detach().requires_grad_(asks), create_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(grads, want))
        with pytest.raises(RuntimeError, match="once"):
            torch.autograd.grad(o.sum() + grads[0].square().sum(), leaves)
    o = forward()
    o.backward(do, create_graph=True)
    assert all(torch.equal(x.grad, g) for x, g in zip(leaves, want))
