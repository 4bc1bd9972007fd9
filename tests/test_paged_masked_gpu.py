"""paged_attention with a window and sinks, and of drafted trees, against the plain computation in 64 bits, within the bounds of masked_reference.py."""
import pytest
import torch

from masked_reference import attention_64, check, paged_keep
from test_paged_gpu import BF16, FP16, Cache, _starts

pytestmark = pytest.mark.gpu


def _slopes(H):
    return torch.tensor([2.0 ** (-8 * (h + 1) / H) for h in range(H)], device="cuda")


def _tree(n, seed, reach=12):
    """A token continues one of the last few drafted before it, or the text."""
    gen = torch.Generator().manual_seed(seed)
    return [-1] + [int(torch.randint(max(-1, t - reach), t, (1,), generator=gen)) for t in range(1, n)]


def _parents(trees):
    return torch.tensor([x for t in trees for x in t], dtype=torch.int32, device="cuda")


def _give_away(cache, keeps):
    """Pages that no token sees hold what another sequence left there, if they are named at all."""
    for b, keep in enumerate(keeps):
        seen = keep.any(0)
        for i in range(-(-seen.shape[0] // cache.page)):
            if not seen[i * cache.page: (i + 1) * cache.page].any():
                page = int(cache.table[b, i])
                cache.k_pages[page], cache.v_pages[page] = float("nan"), float("inf")
                if i % 2:
                    cache.table[b, i] = (-3, 1 << 29)[i // 2 % 2]


def _attend(cache, H, new, dtype, window=None, sinks=0, trees=None, prefix=None, softcap=None, slopes=None, give_away=True, seed=1, **kw):
    import flash_b200 as fb
    gen = torch.Generator(device="cuda").manual_seed(seed)
    q = (torch.randn(sum(new), H, cache.k.shape[2], generator=gen, device="cuda") * 1.5).to(dtype)
    keeps = [paged_keep(length, n, window, sinks, None if trees is None or n > 256 else trees[b], 0 if prefix is None else int(prefix[b]))
             for b, (length, n) in enumerate(zip(cache.lens, new))]
    if give_away:
        _give_away(cache, keeps)
    got = fb.paged_attention(q, cache.k_pages, cache.v_pages, cache.table, cache.kv_lens, _starts(new), window=window, sinks=sinks,
                             parents=None if trees is None else _parents(trees), prefix=prefix, softcap=softcap, slopes=slopes, **kw)
    fb.check_status()
    compare(got, cache, q, new, keeps, softcap, slopes)
    return q, got


def compare(got, cache, q, new, keeps, softcap=None, slopes=None):
    row = 0
    for b, (n, keep) in enumerate(zip(new, keeps)):
        x, lost = got[row: row + n], max(0, n - cache.lens[b])
        assert (x[:lost] == 0).all()
        if n > lost:
            rows = slice(cache.first[b], cache.first[b] + cache.lens[b])
            Q, K, V = (t.transpose(0, 1)[None] for t in (q[row + lost: row + n], cache.k[rows], cache.v[rows]))
            check(x[lost:].transpose(0, 1)[None], attention_64(Q, K, V, None, keep[lost:], None, softcap, slopes)["o"], f"sequence {b}")
        row += n


BATCHES = [([1], [1]), ([128], [1]), ([700, 1, 129], [1, 1, 1]), ([300, 77, 1000, 128], [300, 20, 1, 5]), ([0, 40, 0], [0, 3, 2]), ([10, 600], [25, 600]),
           ([5000, 9, 2200], [1, 9, 150])]
WINDOWS = [(1, 0), (17, 1), (128, 4), (300, 130), (1 << 40, 0)]
SHAPES = [(2, 4, 128, 16), (1, 1, 64, 64), (3, 2, 64, 8), (2, 5, 32, 128), (1, 8, 128, 256), (2, 3, 16, 32)]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("window,sinks", WINDOWS)
@pytest.mark.parametrize("Hk,G,D,page", SHAPES)
@pytest.mark.parametrize("lens,new", BATCHES, ids=lambda x: "-".join(map(str, x)))
def test_windows(lens, new, Hk, G, D, page, window, sinks, dtype):
    _attend(Cache(lens, Hk, D, page, dtype, 3).fill(), Hk * G, new, dtype, window, sinks)


@pytest.mark.parametrize("changes", [dict(softcap=4.0), dict(slopes=True), dict(softcap=10.0, slopes=True)], ids=["cap", "bias", "both"])
@pytest.mark.parametrize("prefix", [None, (0, 50, 300, 2000), (400, 77, 1, 128)])
@pytest.mark.parametrize("Hk,G,D,page,window,sinks", [(2, 4, 128, 16, 100, 3), (1, 12, 64, 64, 200, 0), (1, 48, 32, 16, 60, 140)])
def test_windows_with_changed_scores_and_prefixes(Hk, G, D, page, window, sinks, prefix, changes):
    lens, new = [900, 77, 1000, 128], [300, 20, 1, 5]
    prefix = None if prefix is None else torch.tensor(prefix, dtype=torch.int32, device="cuda")
    slopes = _slopes(Hk * G) if changes.get("slopes") else None
    _attend(Cache(lens, Hk, D, page, BF16, 4).fill(), Hk * G, new, BF16, window, sinks, prefix=prefix, softcap=changes.get("softcap"), slopes=slopes)


@pytest.mark.parametrize("window,sinks", [(500, 4), (4096, 0), (3000, 700)])
def test_long_caches_are_cut_by_what_their_window_shows(window, sinks):
    """Few items of many keys, and of few seen ones: pieces that meet between the first keys and the window."""
    for lens, new, Hk, G in (([60000], [1], 2, 8), ([20000, 70, 33333], [1, 70, 200], 1, 4), ([9000] * 40, [1] * 40, 4, 4)):
        _attend(Cache(lens, Hk, 128, 64, BF16, 5).fill(), Hk * G, new, BF16, window, sinks)


def test_many_sequences():
    """More than a warp's plan takes."""
    lens = [(37 * i) % 900 + 1 for i in range(300)]
    new = [1 if i % 7 else min(lens[i], 9) for i in range(300)]
    _attend(Cache(lens, 2, 64, 16, FP16, 6).fill(), 8, new, FP16, 120, 2)
    _attend(Cache(lens, 2, 64, 16, FP16, 7).fill(), 8, new, FP16, trees=[_tree(n, i) for i, n in enumerate(new)])


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("window,sinks", [(None, 0), (3, 0), (40, 2), (300, 400)])
@pytest.mark.parametrize("Hk,G,D,page", SHAPES)
@pytest.mark.parametrize("lens,new", [([1], [1]), ([300], [24]), ([256, 300, 7, 1000], [256, 33, 7, 64]), ([130, 3, 900], [12, 9, 200]), ([2000, 500], [1, 100])],
                         ids=lambda x: "-".join(map(str, x)))
def test_trees(lens, new, Hk, G, D, page, window, sinks, dtype):
    trees = [_tree(n, 10 + b) for b, n in enumerate(new)]
    _attend(Cache(lens, Hk, D, page, dtype, 8).fill(), Hk * G, new, dtype, window, sinks, trees)


@pytest.mark.parametrize("G", [1, 8, 40, 128])
def test_trees_of_all_shapes(G):
    """A chain, a star, a comb, two chains side by side; a chunk beside them; capped scores."""
    n = 100
    trees = [list(range(-1, n - 1)), [-1] * n, [max(-1, t // 2 * 2 - 2) if t % 2 == 0 else t - 1 for t in range(n)], [t - 2 if t >= 2 else -1 for t in range(n)],
             list(range(-1, 299)), [-1]]
    new = [len(t) for t in trees]
    lens = [n, 1000, 531, 128 + n, 700, 1]
    _attend(Cache(lens, 2, 64, 16, BF16, 9).fill(), 2 * G, new, BF16, trees=trees, softcap=10.0)
    _attend(Cache(lens, 2, 64, 16, BF16, 9).fill(), 2 * G, new, BF16, 60, 5, trees=trees, softcap=10.0)


def test_a_chain_is_what_it_is_without_parents():
    import flash_b200 as fb
    lens, new = [700, 90, 300], [60, 90, 1]
    cache = Cache(lens, 2, 64, 32, BF16, 11).fill()
    q, got = _attend(cache, 8, new, BF16, trees=[list(range(-1, n - 1)) for n in new])
    assert torch.equal(got, fb.paged_attention(q, cache.k_pages, cache.v_pages, cache.table, cache.kv_lens, _starts(new)))


def test_long_texts_with_trees_are_cut():
    lens, new = [30000, 200], [40, 9]
    trees = [_tree(n, 30 + b) for b, n in enumerate(new)]
    _attend(Cache(lens, 1, 128, 64, FP16, 12).fill(), 8, new, FP16, trees=trees)
    _attend(Cache(lens, 1, 128, 64, FP16, 12).fill(), 8, new, FP16, 2000, 3, trees=trees)


def test_parents_that_are_none_are_reported():
    import flash_b200 as fb
    cache = Cache([50, 300], 1, 64, 16, BF16, 13).fill()
    q = torch.randn(9, 4, 64, device="cuda").to(BF16)
    for bad in ([-1, 1, 0, 0, -1, 0, 1, 2, 3], [-1, 0, 0, 0, -1, 0, 1, 2, 2000000000], [-7, 0, 0, 0, -1, 0, 1, 2, 3]):
        got = fb.paged_attention(q, cache.k_pages, cache.v_pages, cache.table, cache.kv_lens, _starts([4, 5]),
                                 parents=torch.tensor(bad, dtype=torch.int32, device="cuda"))
        with pytest.raises(RuntimeError, match="parent"):
            fb.check_status()
        first = [x if -1 <= x < t else -1 for t, x in enumerate(bad[:4])]
        second = [x if -1 <= x < t else -1 for t, x in enumerate(bad[4:])]
        compare(got, cache, q, [4, 5], [paged_keep(50, 4, parents=first), paged_keep(300, 5, parents=second)])


def test_rows_of_no_sequence_and_an_output_of_the_callers():
    import flash_b200 as fb
    cache = Cache([50, 300], 2, 64, 16, BF16, 14).fill()
    trees = [_tree(6, 1), _tree(5, 2)]
    q = torch.randn(20, 8, 64, device="cuda").to(BF16)
    parents = torch.full((20,), 9, dtype=torch.int32, device="cuda")  # (of no sequence: not read)
    parents[4:15] = _parents(trees)
    starts = _starts([6, 5], front=4)
    got = fb.paged_attention(q, cache.k_pages, cache.v_pages, cache.table, cache.kv_lens, starts, parents=parents, window=70, sinks=2)
    fb.check_status()
    assert (got[:4] == 0).all() and (got[15:] == 0).all()
    out = torch.full_like(q, 7.0)
    same = fb.paged_attention(q, cache.k_pages, cache.v_pages, cache.table, cache.kv_lens, starts, parents=parents, window=70, sinks=2, out=out)
    assert same is out and (out[:4] == 7).all() and (out[15:] == 7).all() and torch.equal(out[4:15], got[4:15])
    compare(got[4:15], cache, q[4:15], [6, 5], [paged_keep(50, 6, 70, 2, trees[0]), paged_keep(300, 5, 70, 2, trees[1])])


def test_captured_calls_follow_lengths_and_parents(monkeypatch):
    import flash_b200 as fb
    cache = Cache([400, 90], 2, 64, 16, BF16, 15).fill()
    trees = [_tree(20, 3), _tree(20, 4)]
    q, parents = torch.randn(40, 8, 64, device="cuda").to(BF16), _parents(trees)
    call = lambda: fb.paged_attention(q, cache.k_pages, cache.v_pages, cache.table, cache.kv_lens, _START, parents=parents, window=100, sinks=1)  # noqa: E731
    _START = _starts([20, 20])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for lens, seed in (([400, 90], 3), ([333, 41], 5)):
        trees = [_tree(20, seed), _tree(20, seed + 1)]
        parents.copy_(_parents(trees))
        cache.kv_lens.copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        whole, cache.lens = cache.lens, lens
        compare(got, cache, q, [20, 20], [paged_keep(n, 20, 100, 1, t) for n, t in zip(lens, trees)])
        cache.lens = whole
        from flash_b200 import paged
        monkeypatch.setattr(paged, "_native", lambda *tensors: None)  # the general way through the host gives the same
        assert torch.equal(call(), got)
        monkeypatch.undo()


def test_after_a_time_out_results_are_nan_until_it_has_been_read():
    import flash_b200 as fb
    from flash_b200 import ops
    cache = Cache([700, 400], 2, 64, 16, BF16, 16).fill()
    q, parents = torch.randn(25, 4, 64, device="cuda").to(BF16), _parents([_tree(20, 1), _tree(5, 2)])
    call = lambda: fb.paged_attention(q, cache.k_pages, cache.v_pages, cache.table, cache.kv_lens, _starts([20, 5]), window=300, sinks=1, parents=parents)  # noqa: E731
    want = call()
    ops._status_word(q.device).fill_(142)  # as a bounded wait that ran out leaves it
    assert call().isnan().all()
    with pytest.raises(RuntimeError, match="role 42"):
        fb.check_status()
    assert torch.equal(call(), want)


@pytest.mark.parametrize("cap", [None, 3.0])
def test_a_drafted_token_that_is_not_finite_reaches_those_that_see_it(cap):
    """A key that is not a number makes the tokens on its branch NaN and leaves the others' scores as they were; a value behind all tokens of a tile stays out."""
    import flash_b200 as fb
    n, length = 40, 300
    tree = [-1] + [0] * 19 + [19] * 20  # two levels: 1 .. 19 continue 0, 20 .. 39 continue 19
    cache = Cache([length], 1, 64, 16, BF16, 17).fill()
    q = torch.randn(n, 2, 64, device="cuda").to(BF16)
    call = lambda: fb.paged_attention(q, cache.k_pages, cache.v_pages, cache.table, cache.kv_lens, _starts([n]), parents=_parents([tree]), softcap=cap)  # noqa: E731
    want = call()
    page, slot = cache.places(0, length - n + 5, length - n + 6)
    cache.k_pages[page, slot] = float("nan")
    got = call()
    assert got[5].isnan().all() and torch.equal(got[:5], want[:5]) and torch.equal(got[6:], want[6:])
