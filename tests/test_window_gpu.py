"""attention_scored with a sliding window and sinks against the plain computation in 64 bits, element by element within bounds derived from the roundings
(masked_reference.py)."""
import pytest
import torch

from masked_reference import attention_64, check, windowed

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
NAMES = ("o", "dq", "dk", "dv")


def _inputs(B, H, Hk, M, N, D, dtype, seed, std=1.5, layout="bhld"):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def tensor(h, n, s):
        x = torch.randn((B, h, n, D) if layout == "bhld" else (B, n, h, D), generator=gen, device="cuda") * s
        return (x if layout == "bhld" else x.transpose(1, 2)).to(dtype)

    return tensor(H, M, std), tensor(Hk, N, std), tensor(Hk, N, 1.0), tensor(H, M, 1.0)


def _slopes(H, steep=True):
    return torch.tensor([(0.0, -0.01, 3.0 if steep else 0.05, 0.2)[h % 4] for h in range(H)], device="cuda")


def _run(q, k, v, do, window, sinks, **kw):
    import flash_b200 as fb
    mode = 0 if kw.get("eq") is None else 1
    a, b, c = (x.detach().requires_grad_() for x in (q, k, v))
    o = fb.attention_scored(a, b, c, True, score_func_mode=mode, window=window, sinks=sinks, **kw)
    grads = torch.autograd.grad(o, (a, b, c), do)
    with torch.no_grad():
        assert torch.equal(o, fb.attention_scored(q, k, v, True, score_func_mode=mode, window=window, sinks=sinks, **kw))
    fb.check_status()
    return dict(zip(NAMES, (o.detach(), *grads)))


def _compare(q, k, v, do, window, sinks, **kw):
    M, N = q.shape[2], k.shape[2]
    keep = windowed(M, N, window, sinks, kw.get("prefix"))
    if kw.get("eq") is not None:
        keep = keep & ((kw["eq"][..., None] >= 0) | (kw["eq"][..., None] == kw["ek"][:, :, None, :]))
    got = _run(q, k, v, do, window, sinks, **kw)
    want = attention_64(q, k, v, do, keep, kw.get("sm_scale"), kw.get("softcap"), kw.get("slopes"))
    for n in NAMES:
        check(got[n], want[n], n)
    return got, keep


# one token, tiles that end inside, more keys than queries, grouped heads, few queries (packed heads, runs of keys), several blocks between sinks and window
SHAPES = [(1, 1, 1, 1, 1, 64), (2, 2, 1, 129, 129, 128), (1, 4, 2, 200, 333, 64), (2, 8, 2, 1, 700, 128), (1, 4, 1, 30, 2500, 64), (1, 3, 1, 100, 1300, 128),
          (1, 2, 2, 257, 300, 32), (2, 4, 4, 96, 96, 16), (1, 2, 1, 900, 900, 128)]
WINDOWS = [(1, 0), (1, 3), (64, 0), (128, 4), (129, 128), (200, 130), (5000, 0)]


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("window,sinks", WINDOWS)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_shapes(shape, window, sinks, dtype):
    _compare(*_inputs(*shape, dtype, 7), window, sinks)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("window,sinks", [(1, 0), (100, 2), (256, 1)])
@pytest.mark.parametrize("change", ["cap", "bias", "both"])
def test_changed_scores(change, window, sinks, dtype):
    q, k, v, do = _inputs(2, 4, 2, 390, 520, 64 if change == "cap" else 128, dtype, 8)
    _compare(q, k, v, do, window, sinks, softcap=10.0 if change != "bias" else None, slopes=_slopes(4) if change != "cap" else None)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("prefix", [(0, 300), (130, 1000), (1, 127)])
@pytest.mark.parametrize("D,M,N,window,sinks", [(64, 500, 500, 100, 0), (128, 140, 720, 90, 3), (32, 5, 600, 30, 140)])
def test_prefix(D, M, N, window, sinks, prefix, dtype):
    q, k, v, do = _inputs(2, 4, 2, M, N, D, dtype, 9)
    p = torch.tensor(prefix, dtype=torch.int32, device="cuda")
    _compare(q, k, v, do, window, sinks, prefix=p)
    _compare(q, k, v, do, window, sinks, prefix=p, softcap=10.0, slopes=_slopes(4))


def _documents(B, H, L, seed, per_head=False):
    gen = torch.Generator().manual_seed(seed)
    rows = []
    for _ in range(B * (H if per_head else 1)):
        cuts = torch.sort(torch.randint(1, max(2, L), (3,), generator=gen)).values
        ids = -1 - torch.searchsorted(cuts, torch.arange(L), right=True)
        ids[torch.rand(L, generator=gen) < 0.03] = 5
        rows.append(ids)
    return torch.stack(rows).reshape(B, -1, L).cuda().expand(B, H, L)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("per_head", [False, True])
@pytest.mark.parametrize("L,window,sinks", [(390, 60, 3), (1000, 200, 0), (1000, 140, 129)])
def test_documents(L, window, sinks, per_head, dtype):
    B, H = 2, 4
    q, k, v, do = _inputs(B, H, 2, L, L, 64, dtype, 10)
    ids = _documents(B, H, L, 11, per_head)
    _compare(q, k, v, do, window, sinks, eq=ids, ek=ids)
    _compare(q, k, v, do, window, sinks, eq=ids, ek=ids, softcap=8.0, slopes=_slopes(H), prefix=torch.tensor([70, 300], dtype=torch.int32, device="cuda"))


def test_documents_over_many_blocks():
    """The plan of long id rows, which three kernels build."""
    L = 4700
    q, k, v, do = _inputs(1, 2, 1, L, L, 64, BF16, 12)
    ids = _documents(1, 2, L, 13)
    _compare(q, k, v, do, 700, 4, eq=ids, ek=ids, softcap=20.0)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_rows_that_the_masks_leave_nothing(dtype):
    """A query of a document whose keys all lie before the window, and one of a document without keys."""
    L = 600
    q, k, v, do = _inputs(1, 2, 2, L, L, 64, dtype, 14)
    ek = torch.full((1, 2, L), -1, device="cuda")
    eq = ek.clone()
    ek[..., 300:] = -2
    eq[..., 500:] = -7  # nobody's
    got, keep = _compare(q, k, v, do, 50, 0, eq=eq, ek=ek)
    empty = ~keep.any(-1)[0, 0]
    assert empty[380:].all() and not empty[:340].any()
    assert (got["o"][:, :, empty] == 0).all() and (got["dq"][:, :, empty] == 0).all()


def test_strides_and_scales():
    q, k, v, do = _inputs(2, 4, 2, 333, 400, 64, BF16, 15, layout="blhd")
    _compare(q, k, v, do, 77, 2, sm_scale=0.3)
    wide = torch.randn(2, 4, 333, 3 * 64, device="cuda").to(BF16)
    _compare(wide[..., 64:128], k, v, do, 77, 2)
    _compare(q[..., :33, :], k, v, do[..., :33, :], 30, 2)  # few queries of many


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_long_sequences_keep_to_their_window(dtype):
    """More keys than a query block's list may have between sinks and window; a row block at a time against 64 bits."""
    N, M, window, sinks = 70000, 300, 1000, 7
    q, k, v, do = _inputs(1, 2, 1, M, N, 64, dtype, 16)
    _compare(q, k, v, do, window, sinks)


def test_window_of_all_keys_is_none():
    import flash_b200 as fb
    q, k, v, _ = _inputs(1, 2, 2, 300, 300, 64, BF16, 17)
    p = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert torch.equal(fb.attention_scored(q, k, v, True, prefix=p), fb.attention_scored(q, k, v, True, window=1 << 40, sinks=0))
    assert torch.equal(fb.attention_scored(q, k, v, True, prefix=p), fb.attention_scored(q, k, v, True, window=300, sinks=9))


@pytest.mark.parametrize("flag", ["FA_B200_NO_SKIP", "FA_B200_ALL_PARTIAL"])
@pytest.mark.parametrize("docs", [False, True])
def test_skipped_blocks_change_nothing(flag, docs, monkeypatch):
    q, k, v, do = _inputs(1, 4, 2, 700, 900, 64, BF16, 18)
    kw = {}
    if docs:
        ek = _documents(1, 4, 900, 19)
        kw = dict(eq=ek[..., 200:].contiguous(), ek=ek)
    got = _run(q, k, v, do, 130, 5, **kw)
    monkeypatch.setenv(flag, "1")
    again = _run(q, k, v, do, 130, 5, **kw)
    for n in NAMES:
        if flag == "FA_B200_ALL_PARTIAL":
            assert torch.equal(got[n], again[n]), n
        else:  # (tiles go to the two chains by their place in the walk)
            assert (got[n].double() - again[n].double()).abs().max() <= 2.0 ** -6 * got[n].double().abs().max(), n


def test_gradients_against_differences():
    """fp32. A directional derivative against the central difference of the kernel's own loss: off by the loss's rounding over the step, and by the difference's
    own error, which 64 bits tell."""
    import flash_b200 as fb
    M, N, window, sinks, h = 150, 210, 40, 3, 2.0 ** -6
    q, k, v, do = _inputs(1, 2, 1, M, N, 32, FP32, 20)
    keep, slopes = windowed(M, N, window, sinks), _slopes(2, False)
    got = _run(q, k, v, do, window, sinks, softcap=6.0, slopes=slopes)

    def loss(x):
        o = fb.attention_scored(*x, True, window=window, sinks=sinks, softcap=6.0, slopes=slopes)
        ref, bound = attention_64(*x, None, keep, cap=6.0, slopes=slopes)["o"]
        return (o.double() * do.double()).sum().item(), (ref * do.double()).sum().item(), (bound * do.double().abs()).sum().item()

    gen = torch.Generator(device="cuda").manual_seed(21)
    exact = attention_64(q, k, v, do, keep, cap=6.0, slopes=slopes)
    for n, name in enumerate(("dq", "dk", "dv")):
        x = [q, k, v]
        way = torch.randint(0, 2, x[n].shape, generator=gen, device="cuda").float() * 2 - 1
        ahead, behind = (loss([y + s * h * way if i == n else y for i, y in enumerate(x)]) for s in (1, -1))
        step = ((x[n] + h * way) - (x[n] - h * way)).double()  # as rounding left it
        slope = (got[name].double() * step).sum().item()
        own = abs((ahead[1] - behind[1]) - (exact[name][0] * step).sum().item())
        tolerance = ahead[2] + behind[2] + own + (exact[name][1] * step.abs()).sum().item()
        assert abs((ahead[0] - behind[0]) - slope) <= tolerance, name


def test_other_streams_and_graphs():
    import flash_b200 as fb
    q, k, v, do = _inputs(1, 8, 2, 700, 700, 64, BF16, 22)
    want = _run(q, k, v, do, 150, 4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _run(q, k, v, do, 150, 4)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(got[n], want[n]) for n in NAMES)

    a, b, c = (x.clone().requires_grad_() for x in (q, k, v))
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(fb.attention_scored(a, b, c, True, window=150, sinks=4), (a, b, c), do)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        o = fb.attention_scored(a, b, c, True, window=150, sinks=4)
        grads = torch.autograd.grad(o, (a, b, c), do)
    q2, k2, v2, _ = _inputs(1, 8, 2, 700, 700, 64, BF16, 23)
    with torch.no_grad():
        for x, y in ((a, q2), (b, k2), (c, v2)):
            x.copy_(y)
    graph.replay()
    want = _run(q2, k2, v2, do, 150, 4)
    for x, n in zip((o, *grads), NAMES):
        assert torch.equal(x, want[n]), n


def test_python_path_gives_the_same(monkeypatch):
    """With saved-tensor hooks, or with launches being timed, the node in Python takes the call."""
    q, k, v, do = _inputs(1, 4, 2, 500, 700, 128, FP16, 24)
    want = _run(q, k, v, do, 333, 3, softcap=20.0, slopes=_slopes(4, False))
    with torch.autograd.graph.saved_tensors_hooks(lambda x: x, lambda x: x):
        got = _run(q, k, v, do, 333, 3, softcap=20.0, slopes=_slopes(4, False))
    assert all(torch.equal(got[n], want[n]) for n in NAMES)
    from flash_b200 import scored
    monkeypatch.setattr(scored, "_native", lambda *tensors: None)
    got = _run(q, k, v, do, 333, 3, softcap=20.0, slopes=_slopes(4, False))
    assert all(torch.equal(got[n], want[n]) for n in NAMES)


def test_one_gradient_only_and_twice_refused():
    import flash_b200 as fb
    q, k, v, do = _inputs(1, 2, 2, 200, 200, 64, BF16, 25)
    k.requires_grad_()
    o = fb.attention_scored(q, k, v, True, window=20)
    (dk,) = torch.autograd.grad(o, k, do, create_graph=True)
    check(dk.detach(), attention_64(q, k.detach(), v, do, windowed(200, 200, 20, 0))["dk"], "dk")
    with pytest.raises(RuntimeError, match="once"):
        dk.sum().backward()


def test_after_a_time_out_results_are_nan_until_it_has_been_read():
    """The kernel that adds up the runs of queries of the first keys' blocks among the others."""
    import flash_b200 as fb
    from flash_b200 import ops
    q, k, v, do = _inputs(1, 4, 2, 1000, 1000, 64, BF16, 26)
    want = _run(q, k, v, do, 100, 4)
    a, b, c = (x.detach().requires_grad_() for x in (q, k, v))
    o = fb.attention_scored(a, b, c, True, window=100, sinks=4)
    ops._status_word(q.device).fill_(142)  # as a bounded wait that ran out leaves it
    for g in torch.autograd.grad(o, (a, b, c), do):
        assert g.isnan().all()
    assert fb.attention_scored(q, k, v, True, window=100, sinks=4).isnan().all()
    with pytest.raises(RuntimeError, match="role 42"):
        fb.check_status()
    got = _run(q, k, v, do, 100, 4)
    assert all(torch.equal(got[n], want[n]) for n in NAMES)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("B,H,Hk,L,D,window,sinks", [(1, 4, 1, 3000, 64, 128, 1), (2, 2, 2, 1300, 128, 200, 200), (1, 8, 2, 2000, 32, 64, 128), (1, 2, 1, 5000, 128, 1, 3)])
def test_first_keys_that_all_queries_see(B, H, Hk, L, D, window, sinks, dtype):
    """Their dK and dV come from many runs of queries."""
    _compare(*_inputs(B, H, Hk, L, L, D, dtype, 27), window, sinks)


def test_the_same_bits_again():
    q, k, v, do = _inputs(1, 8, 2, 3000, 3000, 64, BF16, 28)
    want = _run(q, k, v, do, 200, 4)
    for _ in range(3):
        got = _run(q, k, v, do, 200, 4)
        assert all(torch.equal(got[n], want[n]) for n in NAMES)


@pytest.mark.parametrize("B,H,Hk,L,D,window,sinks", [(1, 4, 1, 1500, 64, 60, 1), (2, 2, 2, 700, 128, 100, 200), (1, 8, 2, 900, 32, 64, 33), (3, 2, 1, 1000, 16, 1, 3), (8, 8, 8, 400, 32, 20, 40)])
def test_first_keys_that_all_queries_see_in_fp32(B, H, Hk, L, D, window, sinks):
    """Blocks of 16 and of 32 keys."""
    _compare(*_inputs(B, H, Hk, L, L, D, FP32, 29), window, sinks)
    _compare(*_inputs(B, H, Hk, L - 90, L, D, FP32, 30), window, sinks, softcap=7.0, slopes=_slopes(H))


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("B,Hk,L,D,window,sinks", [(1, 1, 131072, 128, 1, 131072), (1, 1, 131072, 128, 1000, 60000), (4, 8, 20000, 64, 64, 5000), (1, 1, 8000, 128, 1, 300), (64, 32, 4000, 128, 4, 4)])
def test_runs_of_queries_stay_few(B, Hk, L, D, window, sinks, dtype):
    """Where there are many first keys they are work enough by themselves: the workspace holds some blocks' sums for each SM, not 32 times all of dK and dV."""
    import ctypes
    from flash_b200 import _lib
    problem, size = _lib.Problem(), ctypes.c_size_t(0)
    for name, value in dict(B=B, H=Hk, Hk=Hk, M=L, N=L, D=D, dtype=dtype, causal=1, mode=0, id_heads=1, sm_scale=0.1).items():
        setattr(problem, name, value)
    _lib.check(_lib.load().fa_bwd_workspace_bytes(problem, _lib.Window(window, sinks), size), "fa_bwd_workspace_bytes")
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    # S = 2 SMs (fp32: 8, of blocks of 32 keys). All the work is W >= blocks * walk, a run is at least floor(W / S), which is at least W / 2S if it is 1, and walk / run + 1 bounds the runs: those of
    # all blocks are at most 2 S + blocks; where there are two runs floor(W / S) < walk, so that blocks < S. (fp32 gives a block of 32 keys at most the room of 128.)
    most = (3 * 8 if dtype == 2 else 3 * 2) * sms
    assert size.value <= most * 2 * 128 * max(D, 64) * 4



def test_many_first_keys_in_fp32():
    """As many blocks, times 32 runs of queries, would be more than a launch can have. A window of one key with all keys first ones, and one of all keys, see the same."""
    L = 70000
    q, k, v, do = _inputs(1, 1, 1, L, L, 16, FP32, 33)
    a, b = _run(q, k, v, do, 1, L), _run(q, k, v, do, L, 0)
    for n in NAMES:
        assert torch.equal(a[n], b[n]), n
