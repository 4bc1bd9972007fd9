"""A paged cache of 8 bits: what paged_append writes, to the bit, and paged_attention over it against the plain computation in 64 bits of the numbers that it stands
for, within the bounds of masked_reference.py."""
import pytest
import torch

from eight_bit_cache import LEAST, MOST, Cache8, quantised, times_power
from masked_reference import attention_64, check, paged_keep
from test_paged_masked_gpu import BATCHES, _parents, _slopes, _tree

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16
# P is fp16, raised by 2^7, whatever q is: an entry below 2^-14 / 2^7 of the row's reference may lack half of fp16's last step, 2^-25 / 2^7, of a row whose sum is 1 at least
SUB = 2.0 ** -32


def _starts(new, front=0):
    return torch.tensor([front + sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32, device="cuda")


def compare(got, cache, q, new, keeps, softcap=None, slopes=None, sm_scale=None):
    row = 0
    for b, (n, keep) in enumerate(zip(new, keeps)):
        x, lost = got[row: row + n], max(0, n - cache.lens[b])
        assert (x[:lost] == 0).all()
        if n > lost:
            rows = slice(cache.first[b], cache.first[b] + cache.lens[b])
            Q, K, V = (t.transpose(0, 1)[None] for t in (q[row + lost: row + n], cache.k[rows], cache.v[rows]))
            check(x[lost:].transpose(0, 1)[None], attention_64(Q, K, V, None, keep[lost:], sm_scale, softcap, slopes, SUB)["o"], f"sequence {b}")
        row += n


def _attend(cache, H, new, dtype, window=None, sinks=0, trees=None, prefix=None, softcap=None, slopes=None, seed=1, q=None, **kw):
    import flash_b200 as fb
    if q is None:
        gen = torch.Generator(device="cuda").manual_seed(seed)
        q = (torch.randn(sum(new), H, cache.k.shape[2], generator=gen, device="cuda") * 1.5).to(dtype)
    keeps = [paged_keep(length, n, window, sinks, None if trees is None or n > 256 else trees[b], 0 if prefix is None else int(prefix[b]))
             for b, (length, n) in enumerate(zip(cache.lens, new))]
    got = fb.paged_attention(q, *cache.args(), _starts(new), window=window, sinks=sinks, parents=None if trees is None else _parents(trees), prefix=prefix, softcap=softcap,
                             slopes=slopes, **cache.scales(), **kw)
    fb.check_status()
    compare(got, cache, q, new, keeps, softcap, slopes, kw.get("sm_scale"))
    return q, got


SHAPES = [(2, 4, 128, 16), (1, 1, 64, 64), (3, 2, 64, 32), (2, 5, 32, 128), (1, 8, 128, 256), (2, 3, 16, 32), (1, 48, 64, 16)]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("changes", [{}, dict(softcap=4.0), dict(slopes=True), dict(softcap=10.0, slopes=True)], ids=["plain", "cap", "bias", "both"])
@pytest.mark.parametrize("Hk,G,D,page", SHAPES)
@pytest.mark.parametrize("lens,new", BATCHES, ids=lambda x: "-".join(map(str, x)))
def test_batches(lens, new, Hk, G, D, page, changes, dtype):
    slopes = _slopes(Hk * G) if changes.get("slopes") else None
    _attend(Cache8(lens, Hk, D, page, dtype, 3).fill(), Hk * G, new, dtype, softcap=changes.get("softcap"), slopes=slopes)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("window,sinks,softcap", [(17, 1, None), (300, 130, 6.0), (1 << 40, 0, None)])
@pytest.mark.parametrize("Hk,G,D,page", SHAPES)
def test_windows_and_trees(Hk, G, D, page, window, sinks, softcap, dtype):
    lens, new = [900, 77, 1000, 130, 256], [300, 20, 1, 5, 256]
    cache = Cache8(lens, Hk, D, page, dtype, 4).fill()
    _attend(cache, Hk * G, new, dtype, window, sinks, softcap=softcap)
    trees = [_tree(n, 10 + b) for b, n in enumerate(new)]
    _attend(cache, Hk * G, new, dtype, window, sinks, trees, softcap=softcap)
    _attend(cache, Hk * G, new, dtype, trees=trees, softcap=softcap)


@pytest.mark.parametrize("order", ["phd", "hpd"])
@pytest.mark.parametrize("prefix", [None, (0, 50, 300, 2000)])
def test_orders_and_prefixes(order, prefix):
    cache = Cache8([900, 77, 1000, 128], 2, 128, 32, BF16, 5, order).fill()
    prefix = None if prefix is None else torch.tensor(prefix, dtype=torch.int32, device="cuda")
    _attend(cache, 8, [300, 20, 1, 5], BF16, prefix=prefix, slopes=_slopes(8))
    _attend(cache, 8, [300, 20, 1, 5], BF16, 200, 3, prefix=prefix)


def test_long_caches_and_many_sequences():
    for lens, new, Hk, G, D in (([60000], [1], 2, 8, 128), ([20000, 70, 33333], [1, 70, 200], 1, 4, 64), ([9000] * 40, [1] * 40, 4, 4, 128)):
        _attend(Cache8(lens, Hk, D, 64, BF16, 6).fill(), Hk * G, new, BF16)
    lens = [(37 * i) % 900 + 1 for i in range(300)]
    new = [1 if i % 7 else min(lens[i], 9) for i in range(300)]
    _attend(Cache8(lens, 2, 64, 16, FP16, 7).fill(), 8, new, FP16)
    _attend(Cache8(lens, 2, 64, 16, FP16, 7).fill(), 8, new, FP16, trees=[_tree(n, i) for i, n in enumerate(new)])


@pytest.mark.parametrize("cap", [None, 50.0])
def test_queries_of_all_sizes(cap):
    """bf16's range is wider than that of the products' type: each row comes to it by a factor of its own."""
    lens, new = [200, 300], [40, 1]
    cache = Cache8(lens, 2, 128, 16, BF16, 8, std=0.25).fill()
    gen = torch.Generator(device="cuda").manual_seed(9)
    size = torch.tensor([1.0, 3e4, 1e6, 1e-6, 1e30, 1e-30, 0.0, 2e-3], device="cuda")[torch.arange(41 * 8, device="cuda") % 8].reshape(41, 8, 1)
    q = torch.randn(41, 8, 128, generator=gen, device="cuda")
    for scale, rows in ((1.0, size <= 1), (1e-6, size <= 1e6), (1e-30, size <= 1e30)):
        _attend(cache, 8, new, BF16, q=(q * torch.where(rows, size, 0.0)).to(BF16), sm_scale=scale, softcap=cap)


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_many_small_weights_beside_a_large_one(dtype):
    """One key far above 100000 others, each below what fp16 holds beside it unless P is raised: together they are a third of the row."""
    import flash_b200 as fb
    N, D = 100000, 64
    cache = Cache8([N], 1, D, 64, dtype, 10)
    x = torch.zeros(N, 1, D, device="cuda", dtype=torch.float64)
    x[:, :, 0] = 1.0
    x[777, :, 0] = 1.0 + 12.25  # the others at exp(-12.25) = 2^-17.7 of it
    cache.k_rows, cache.v_rows = x.to(dtype), cache.v_rows
    (k, ke), (v, ve) = quantised(cache.k_rows), quantised(cache.v_rows)
    cache.k, cache.v, cache.parts = times_power(k, ke[..., None]), times_power(v, ve[..., None]), (k, ke, v, ve)
    cache.fill()
    q = torch.zeros(1, 4, D, device="cuda", dtype=dtype)
    q[:, :, 0] = 1
    got = fb.paged_attention(q, *cache.args(), sm_scale=1.0, **cache.scales())
    compare(got, cache, q, [1], [paged_keep(N, 1)], sm_scale=1.0)


# ---- append ----------------------------------------------------------------------------------------------------------------------------------------------------
def _bits(x):
    return x.view(torch.uint8)


def _appended(cache, new, k, v, starts, before):
    """The pages and scales that an append of rows k and v leaves, plainly."""
    pages = [x.clone() for x in before]
    (kq, ke), (vq, ve) = quantised(k), quantised(v)
    row = 0 if starts is None else int(starts[0])
    for b, n in enumerate(new):
        lost = max(0, n - cache.lens[b])
        page, slot = cache.places(b, cache.lens[b] - n + lost, cache.lens[b])
        rows = slice(row + lost, row + n)
        for data, scales, x, e in ((pages[0], pages[2], kq, ke), (pages[1], pages[3], vq, ve)):
            data[page, slot] = _bits(x[rows].float().to(torch.float8_e4m3fn))
            scales[page, :, slot] = (e[rows] + 127).to(torch.uint8)
        row += n
    return pages


def _append_and_compare(cache, new, k, v, starts):
    import flash_b200 as fb
    state = lambda: [_bits(x) for x in (cache.k_pages, cache.v_pages, cache.k_scales, cache.v_scales)]  # noqa: E731
    want = _appended(cache, new, k, v, starts, state())
    versions = [x._version for x in (cache.k_pages, cache.v_pages, cache.k_scales, cache.v_scales)]
    fb.paged_append(k, v, *cache.args(), starts, **cache.scales())
    fb.check_status()
    for x, y, what in zip(state(), want, ("k", "v", "k scales", "v scales")):
        if what in ("k", "v"):  # (of a NaN the sign may be either)
            x, y = (torch.where((t & 127) == 127, 127, t) for t in (x, y))
        assert torch.equal(x, y), what
    assert [x._version for x in (cache.k_pages, cache.v_pages, cache.k_scales, cache.v_scales)] == [n + 1 for n in versions]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("order", ["phd", "hpd"])
@pytest.mark.parametrize("Hk,D,page", [(8, 128, 16), (1, 64, 64), (3, 32, 128), (24, 128, 32), (5, 16, 256), (9, 64, 16)])
@pytest.mark.parametrize("lens,new", [([1], [1]), ([700, 16, 129], [700, 1, 30]), ([0, 40], [3, 50]), ([33] * 40, [1] * 40)], ids=lambda x: "-".join(map(str, x[:3])))
def test_append(lens, new, Hk, D, page, order, dtype):
    cache = Cache8(lens, Hk, D, page, dtype, 11, order)
    gen = torch.Generator(device="cuda").manual_seed(12)
    T = sum(new)
    size = torch.ldexp(torch.ones(T + 5, Hk, 1, device="cuda"), torch.randint(-24, 14, (T + 5, Hk, 1), generator=gen, device="cuda"))
    k, v = ((torch.randn(T + 5, Hk, D, generator=gen, device="cuda") * size).to(dtype) for _ in range(2))
    _append_and_compare(cache, new, k, v, _starts(new, 2))
    _append_and_compare(cache, new, k[:, :, :].transpose(0, 1).contiguous().transpose(0, 1), v, _starts(new, 1))
    if all(n == 1 for n in new):
        _append_and_compare(cache, new, k[:T], v[:T], None)


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_append_of_special_rows(dtype):
    D = 64
    info = torch.finfo(dtype)
    halfway = torch.tensor([17.0, 19.0, 33 / 1024, 1.5 / 512, 0.5 / 512, 2.5 / 512, 216.0, 232.0])  # between two of e4m3's numbers (with a scale of 1)
    rows = [torch.zeros(D), torch.full((D,), info.max), torch.full((D,), info.smallest_normal), torch.full((D,), -info.smallest_normal * info.eps),
            torch.full((D,), float("inf")), torch.full((D,), float("nan")), torch.full((D,), -0.0)]
    for top in (448.0, 449.0, 450.0, 7.0, 7.03125, 3.5, 2.0 ** -15 * 448, 2.0 ** -16 * 448, 57344.0, 60000.0):
        x = torch.linspace(-top, top, D)
        x[:8] = halfway * (top / 448)
        x[-1] = top
        rows.append(x)
    mixed = torch.randn(D)
    mixed[3], mixed[9], mixed[11] = float("inf"), float("-inf"), float("nan")
    rows.append(mixed)
    k = torch.stack(rows).to(dtype).cuda()[:, None, :]
    v = (-k.flip(0)).contiguous()
    n = len(rows)
    cache = Cache8([n], 1, D, 16, dtype, 13)
    _append_and_compare(cache, [n], k, v, _starts([n]))
    assert LEAST == -15 and MOST == 7


def test_append_reports_pages_that_there_are_not():
    import flash_b200 as fb
    cache = Cache8([40, 40], 1, 64, 16, BF16, 14)
    k = torch.randn(80, 1, 64, device="cuda").to(BF16)
    cache.table[1, 1] = 1000
    before = cache.k_pages.view(torch.uint8).clone()
    fb.paged_append(k, k, *cache.args(), _starts([0, 80]), **cache.scales())
    with pytest.raises(RuntimeError, match="page"):
        fb.check_status()
    page, slot = cache.places(0, 0, 40)
    assert torch.equal(cache.k_pages.view(torch.uint8)[page, slot], before[page, slot])
    cache.kv_lens[0] = 5000
    fb.paged_append(k, k, *cache.args(), _starts([40, 40]), **cache.scales())
    with pytest.raises(RuntimeError, match="length|page"):
        fb.check_status()


def test_a_step_of_serving():
    """A prompt in chunks, drafted tokens and the ones that are kept, with a window, over one cache, by captured calls on a side stream: the cache's own numbers tell what each call
    has to give."""
    import flash_b200 as fb
    Hk, G, D, page, window, sinks = 2, 4, 128, 16, 200, 4
    H = Hk * G
    gen = torch.Generator(device="cuda").manual_seed(15)
    cache = Cache8([640, 480], Hk, D, page, BF16, 16)
    lens = [0, 0]
    k_all, v_all = cache.k_rows, cache.v_rows
    steps = [([300, 5], None), ([100, 301], None), ([24, 1], None), ([20, 33], [_tree(20, 1), _tree(33, 2)]), ([1, 1], None)]
    side = torch.cuda.Stream()
    for new, trees in steps:
        lens = [a + n for a, n in zip(lens, new)]
        rows = torch.cat([torch.arange(cache.first[b] + lens[b] - new[b], cache.first[b] + lens[b]) for b in range(2)]).cuda()
        q = torch.randn(sum(new), H, D, generator=gen, device="cuda").to(BF16)
        kv_lens, starts, k, v = torch.tensor(lens, dtype=torch.int32, device="cuda"), _starts(new), k_all[rows], v_all[rows]
        parents = None if trees is None else _parents(trees)

        def step():
            fb.paged_append(k, v, cache.k_pages, cache.v_pages, cache.table, kv_lens, starts, **cache.scales())
            return fb.paged_attention(q, cache.k_pages, cache.v_pages, cache.table, kv_lens, starts, window=window, sinks=sinks, parents=parents, **cache.scales())

        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            first = step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        graph.replay()
        fb.check_status()
        assert torch.equal(first, got)
        whole, cache.lens = cache.lens, lens
        compare(got, cache, q, new, [paged_keep(lens[b], new[b], window, sinks, trees and trees[b]) for b in range(2)])
        cache.lens = whole


def test_the_general_way_through_the_host_gives_the_same(monkeypatch):
    import flash_b200 as fb
    from flash_b200 import paged
    lens, new = [300, 77], [40, 5]
    cache = Cache8(lens, 2, 64, 32, FP16, 17).fill()
    q, got = _attend(cache, 8, new, FP16, 100, 2, [_tree(40, 5), _tree(5, 6)])
    k = torch.randn(45, 2, 64, device="cuda").to(FP16)
    other = Cache8(lens, 2, 64, 32, FP16, 17).fill()
    fb.paged_append(k, -k, *cache.args(), _starts(new), **cache.scales())
    monkeypatch.setattr(paged, "_native", lambda *tensors: None)
    _attend(other, 8, new, FP16, 100, 2, [_tree(40, 5), _tree(5, 6)], q=q)
    fb.paged_append(k, -k, *other.args(), _starts(new), **other.scales())
    for x, y in zip((*cache.args()[:2], *cache.scales().values()), (*other.args()[:2], *other.scales().values())):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    out = torch.full_like(q, 3.0)
    fb.paged_attention(q, *other.args(), _starts(new), window=100, sinks=2, parents=_parents([_tree(40, 5), _tree(5, 6)]), out=out, **other.scales())
    monkeypatch.undo()
    assert torch.equal(out, fb.paged_attention(q, *cache.args(), _starts(new), window=100, sinks=2, parents=_parents([_tree(40, 5), _tree(5, 6)]), **cache.scales()))


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("changes", [{}, dict(softcap=4.0), dict(slopes=True), dict(softcap=10.0, slopes=True)], ids=["plain", "cap", "bias", "both"])
@pytest.mark.parametrize("Hk,G,D,page", [(2, 4, 128, 16), (1, 1, 64, 64), (2, 8, 64, 32), (1, 12, 128, 128), (2, 16, 32, 16), (1, 17, 64, 16), (3, 9, 16, 32), (1, 48, 128, 16)])
def test_single_tokens(Hk, G, D, page, changes, dtype):
    """Without starts; up to 16 heads a group an instance of its own."""
    import flash_b200 as fb
    lens = [1, 700, 0, 128, 129, 5000, 31, 16, 2500]
    cache = Cache8(lens, Hk, D, page, dtype, 20).fill()
    gen = torch.Generator(device="cuda").manual_seed(21)
    q = (torch.randn(len(lens), Hk * G, D, generator=gen, device="cuda") * 1.5).to(dtype)
    slopes = _slopes(Hk * G) if changes.get("slopes") else None
    for window, sinks, prefix in ((None, 0, None), (100, 3, None), (1, 0, None), (40, 200, None), (300, 2, (0, 50, 9, 300, 100, 4000, 1, 0, 1000))):
        keeps = [paged_keep(n, 1, window, sinks, prefix=0 if prefix is None else prefix[b]) for b, n in enumerate(lens)]
        p = None if prefix is None else torch.tensor(prefix, dtype=torch.int32, device="cuda")
        got = fb.paged_attention(q, *cache.args(), window=window, sinks=sinks, prefix=p, softcap=changes.get("softcap"), slopes=slopes, **cache.scales())
        fb.check_status()
        compare(got, cache, q, [1] * len(lens), keeps, changes.get("softcap"), slopes)


@pytest.mark.parametrize("tree", [False, True])
def test_single_tokens_of_many_sequences_and_as_trees(tree):
    import flash_b200 as fb
    lens = [(37 * i) % 900 for i in range(300)]
    cache = Cache8(lens, 2, 64, 16, BF16, 22).fill()
    q = torch.randn(300, 8, 64, device="cuda").to(BF16)
    got = fb.paged_attention(q, *cache.args(), parents=torch.full((300,), -1, dtype=torch.int32, device="cuda") if tree else None, **cache.scales())
    fb.check_status()
    compare(got, cache, q, [1] * 300, [paged_keep(n, 1) for n in lens])


def test_single_tokens_of_all_sizes_and_not_finite():
    """Rows of bf16 at their own factors in the instance of single tokens, too; a row that sees a key that is not a number is NaN, and its neighbours are not."""
    import flash_b200 as fb
    cache = Cache8([300, 200], 1, 128, 16, BF16, 23, std=0.25)
    size = torch.tensor([1.0, 3e4, 1e6, 1e-6, 1e30, 1e-30, 0.0, 2e-3], device="cuda").reshape(1, 8, 1)
    gen = torch.Generator(device="cuda").manual_seed(24)
    q = torch.randn(2, 8, 128, generator=gen, device="cuda")
    for scale, most in ((1.0, 1), (1e-6, 1e6), (1e-30, 1e30)):
        x = (q * torch.where(size <= most, size, 0.0)).to(BF16)
        for cap in (None, 50.0):
            got = fb.paged_attention(x, *cache.fill().args(), sm_scale=scale, softcap=cap, **cache.scales())
            compare(got, cache, x, [1, 1], [paged_keep(300, 1), paged_keep(200, 1)], cap, sm_scale=scale)
    page, slot = cache.places(0, 100, 101)
    cache.k_pages.view(torch.uint8)[page, slot, 0, 5] = 127
    got = fb.paged_attention(x, *cache.args(), **cache.scales())
    assert got[0].isnan().all() and got[1].isfinite().all()


@pytest.mark.parametrize("single", [False, True])
def test_after_a_time_out_results_are_nan_until_it_has_been_read(single):
    import flash_b200 as fb
    from flash_b200 import ops
    cache = Cache8([700, 400], 2, 64, 16, BF16, 25).fill()
    new = [1, 1] if single else [90, 5]
    q = torch.randn(sum(new), 4, 64, device="cuda").to(BF16)
    call = lambda: fb.paged_attention(q, *cache.args(), None if single else _starts(new), window=300, sinks=1, **cache.scales())  # noqa: E731
    want = call()
    ops._status_word(q.device).fill_(142)  # as a bounded wait that ran out leaves it
    assert call().isnan().all()
    with pytest.raises(RuntimeError, match="role 42"):
        fb.check_status()
    assert torch.equal(call(), want)


def test_pages_and_lengths_that_there_are_not():
    import flash_b200 as fb
    cache = Cache8([300, 200], 2, 64, 16, BF16, 26).fill()
    q = torch.randn(2, 8, 64, device="cuda").to(BF16)
    want = fb.paged_attention(q, *cache.args(), **cache.scales())
    table = cache.table.clone()
    for bad in (-1, 1 << 29, cache.k_pages.shape[0]):
        cache.table[1, 2] = bad
        for starts in (None, _starts([1, 1])):
            got = fb.paged_attention(q, *cache.args(), starts, **cache.scales())
            with pytest.raises(RuntimeError, match="page"):
                fb.check_status()
            assert torch.equal(got[0], want[0])
    cache.table.copy_(table)
    cache.kv_lens[1] = 1 << 28
    got = fb.paged_attention(q, *cache.args(), **cache.scales())
    with pytest.raises(RuntimeError, match="length|page"):
        fb.check_status()
    assert torch.equal(got[0], want[0])


def test_two_streams_at_once():
    import flash_b200 as fb
    caches = [Cache8([3000, 5000, 20], 2, 128, 64, BF16, 27 + i).fill() for i in range(2)]
    q = [torch.randn(203, 8, 128, device="cuda").to(BF16) for _ in range(2)]
    starts, streams = _starts([200, 1, 2]), [torch.cuda.Stream() for _ in range(2)]
    call = lambda i: fb.paged_attention(q[i], *caches[i].args(), starts, window=1000, sinks=2, **caches[i].scales())  # noqa: E731
    want = [call(i) for i in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(call(i))
    torch.cuda.synchronize()
    fb.check_status()
    assert all(torch.equal(x, want[i]) for i in range(2) for x in got[i])


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D,page", [(128, 16), (64, 16), (128, 64), (64, 256)])
def test_items_of_both_kinds_in_turn(D, page, dtype):
    """Single tokens, which warps multiply as they read the rings, between chunks, which the tensor cores do, with odd and even numbers of tiles; the rings' places go to both groups of
    warps then, and loads of small pages land in any order. The same bits each time."""
    import flash_b200 as fb
    lens = [1 + (977 * b * b + 613 * b) % 2500 for b in range(36)]
    new = [1 if b % 3 else min(lens[b], 40 + 5 * b) for b in range(36)]
    cache = Cache8(lens, 2, D, page, dtype, 41).fill()
    q, first = _attend(cache, 8, new, dtype)
    for _ in range(40):
        assert torch.equal(fb.paged_attention(q, *cache.args(), _starts(new), **cache.scales()), first)
    single = q[:36].contiguous()
    once = fb.paged_attention(single, *cache.args(), torch.arange(37, dtype=torch.int32, device="cuda"), **cache.scales())
    for _ in range(20):
        assert torch.equal(fb.paged_attention(single, *cache.args(), torch.arange(37, dtype=torch.int32, device="cuda"), **cache.scales()), once)
    fb.check_status()
