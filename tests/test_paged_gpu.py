"""paged_append and paged_attention against the plain computation in 64 bits, within the bounds of scored_reference.py."""
import pytest
import torch

from scored_reference import attention_64

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


class Cache:
    """Pages of a batch with what a long-running server leaves in them: NaN and infinities in every slot that holds no token of a sequence, page
    numbers that do not exist behind a sequence's last page."""

    def __init__(self, lens, Hk, D, page, dtype, seed, order="phd", spare=3):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.lens, self.page = lens, page
        need = [-(-n // page) for n in lens]
        pages = sum(need) + spare
        perm = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
        self.table = torch.full((len(lens), max(max(need), 1) + 1), -7, dtype=torch.int32)
        self.table[:, -1] = 1 << 30
        self.k, self.v = (torch.randn(sum(lens), Hk, D, generator=gen, device="cuda").to(dtype) for _ in range(2))
        self.first = [sum(lens[:b]) for b in range(len(lens))]
        shape = {"phd": (pages, page, Hk, D), "hpd": (pages, Hk, page, D), "both": (pages, 2, page, Hk, D)}[order]
        if order == "both":  # keys and values of a page side by side
            whole = torch.full(shape, float("nan"), device="cuda", dtype=dtype)
            self.k_pages, self.v_pages = whole[:, 0], whole[:, 1]
        else:
            self.k_pages, self.v_pages = (torch.full(shape, x, device="cuda", dtype=dtype) for x in (float("nan"), float("inf")))
            if order == "hpd":
                self.k_pages, self.v_pages = self.k_pages.transpose(1, 2), self.v_pages.transpose(1, 2)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = torch.tensor(perm[at: at + n])
            at += n
        self.table = self.table.cuda()
        self.kv_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")

    def places(self, b, lo, hi):
        at = torch.arange(lo, hi, device="cuda")
        return self.table[b].long()[at // self.page], at % self.page

    def fill(self):
        for b, n in enumerate(self.lens):
            place, rows = self.places(b, 0, n), slice(self.first[b], self.first[b] + n)
            self.k_pages[place], self.v_pages[place] = self.k[rows], self.v[rows]
        return self


def _starts(new, front=0):
    return torch.tensor([front + sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32, device="cuda")


def _slopes(H, on):
    return torch.tensor([2.0 ** (-8 * (h + 1) / H) for h in range(H)], device="cuda") if on else None


def _check(got, cache, q, new, cap=None, slopes=None, prefix=None, sm_scale=None, front=0):
    row = front
    for b, n in enumerate(new):
        length, x = cache.lens[b], got[row: row + n]
        lost = max(0, n - length)  # tokens in front of the sequence's beginning
        assert (x[:lost] == 0).all()
        if n > lost:
            rows = slice(cache.first[b], cache.first[b] + length)
            Q, K, V = (t.transpose(0, 1)[None] for t in (q[row + lost: row + n], cache.k[rows], cache.v[rows]))
            p = None if prefix is None else prefix[b: b + 1]
            value, bound = attention_64(Q, K, V, torch.zeros_like(Q), True, sm_scale, None, None, cap, slopes, p)["o"]
            off = (x[lost:].transpose(0, 1)[None].double() - value).abs()
            assert torch.isfinite(x).all(), f"sequence {b}"
            assert (off <= bound).all(), f"sequence {b}: {(off / bound).max().item():.2f} times its bound, {off.max().item():.3g} off"
        row += n


def _attend(cache, H, new, dtype, seed=1, q_std=1.5, prefix=None, decode=False, **kw):
    import flash_b200 as fb
    gen = torch.Generator(device="cuda").manual_seed(seed)
    q = (torch.randn(sum(new), H, cache.k.shape[2], generator=gen, device="cuda") * q_std).to(dtype)
    starts = None if decode else _starts(new)
    got = fb.paged_attention(q, cache.k_pages, cache.v_pages, cache.table, cache.kv_lens, starts, prefix=prefix, softcap=kw.get("cap"), slopes=kw.get("slopes"),
                             sm_scale=kw.get("sm_scale"))
    fb.check_status()
    _check(got, cache, q, new, prefix=prefix, **kw)
    return got


BATCHES = [([1], [1]), ([128], [1]), ([700, 1, 129], [1, 1, 1]), ([300, 77, 1000, 128], [300, 20, 1, 5]), ([0, 40, 0], [0, 3, 2]), ([10, 600], [25, 600]),
           ([5000, 9, 2200], [1, 9, 150])]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("changes", [{}, dict(cap=4.0), dict(slopes=True), dict(cap=10.0, slopes=True)], ids=["plain", "cap", "bias", "both"])
@pytest.mark.parametrize("Hk,G,D,page", [(2, 4, 128, 16), (1, 1, 64, 64), (3, 2, 64, 8), (2, 5, 32, 128), (1, 8, 128, 256), (2, 3, 16, 32)])
@pytest.mark.parametrize("lens,new", BATCHES, ids=lambda x: "-".join(map(str, x)))
def test_batches(lens, new, Hk, G, D, page, changes, dtype):
    cache = Cache(lens, Hk, D, page, dtype, 3).fill()
    _attend(cache, Hk * G, new, dtype, cap=changes.get("cap"), slopes=_slopes(Hk * G, changes.get("slopes")))


@pytest.mark.parametrize("order", ["phd", "hpd", "both"])
@pytest.mark.parametrize("G", [1, 12, 128])
def test_orders_of_the_pages_and_groups(order, G):
    lens, new = [333, 64, 1500], [1, 64, 40]
    _attend(Cache(lens, 2, 64, 32, BF16, 4, order).fill(), 2 * G, new, BF16, cap=8.0)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("decode", [True, False])
def test_single_tokens(decode, dtype):
    """Few and many sequences, short and long: whole items, cut ones, several pieces of an item."""
    for B, longest, Hk, G, D in ((1, 20000, 2, 4, 128), (3, 9000, 1, 8, 64), (40, 1500, 8, 4, 128), (200, 300, 2, 2, 64), (1100, 40, 1, 1, 64)):
        lens = [1 + (longest * (b * 7 + 1)) % longest for b in range(B - 1)] + [longest]
        _attend(Cache(lens, Hk, D, 16, dtype, 5).fill(), Hk * G, [1] * B, dtype, decode=decode)


@pytest.mark.parametrize("D", [64, 128])
def test_prefix(D):
    prefix = torch.tensor([100, 0, 5000, -3], dtype=torch.int32, device="cuda")
    cache = Cache([400, 200, 310, 64], 2, D, 16, BF16, 6).fill()
    for cap, slopes in ((None, False), (5.0, True)):
        _attend(cache, 4, [400, 30, 310, 1], BF16, prefix=prefix, cap=cap, slopes=_slopes(4, slopes))


def test_long_sequence_in_pieces_with_many_rows():
    cache = Cache([30000, 50], 1, 128, 64, FP16, 7).fill()
    _attend(cache, 16, [13, 2], FP16, cap=6.0, slopes=_slopes(16, True), sm_scale=0.2)


def test_rows_of_no_sequence():
    import flash_b200 as fb
    cache = Cache([100, 30], 2, 64, 16, BF16, 8).fill()
    new, front = [4, 30], 3
    q = torch.randn(60, 4, 64, device="cuda").to(BF16)
    args = (cache.k_pages, cache.v_pages, cache.table, cache.kv_lens, _starts(new, front))
    for poison in (1, 2):  # what a new tensor's memory holds
        torch.full((60, 4, 64), 7.0, device="cuda", dtype=BF16)
        got = fb.paged_attention(q, *args)
        _check(got, cache, q, new, front=front)
        assert (got[:front] == 0).all() and (got[front + 34:] == 0).all()
    wide = torch.full((60, 6, 72), 7.0, device="cuda", dtype=BF16)
    out = wide[:, 1:5, :64]
    version = out._version
    assert fb.paged_attention(q, *args, out=out) is out and out._version > version
    _check(out, cache, q, new, front=front)
    assert torch.equal(out[front: front + 34], got[front: front + 34])
    out[front: front + 34] = 7.0
    assert (wide == 7.0).all()


def test_queries_in_any_layout():
    import flash_b200 as fb
    cache = Cache([70, 300], 2, 64, 16, BF16, 9).fill()
    new = [5, 1]
    base = torch.randn(6, 3, 4, 65, device="cuda").to(BF16)
    whole = torch.randn(6, 3, 4, 64, device="cuda").to(BF16)
    for q in (whole[:, 1], base[:, 0, :, 1:], whole[:, 2].flip(2).transpose(1, 2).contiguous().transpose(1, 2), whole[:1, 0].expand(6, 4, 64)):
        args = (cache.k_pages, cache.v_pages, cache.table[:, : cache.table.shape[1]], cache.kv_lens, _starts(new))
        _check(fb.paged_attention(q, *args), cache, q, new)
    table = torch.stack([cache.table, cache.table], 2)[:, :, 0]  # strided
    lens = torch.stack([cache.kv_lens] * 2, 1)[:, 1]
    _check(fb.paged_attention(q, cache.k_pages, cache.v_pages, table, lens, _starts(new)), cache, q, new)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("order", ["phd", "hpd", "both"])
@pytest.mark.parametrize("lens,new", BATCHES + [([90] * 300, [1] * 300), ([1000] * 70, [3, 0] * 35)], ids=lambda x: "-".join(map(str, x[:4])))
@pytest.mark.parametrize("Hk,D,page", [(2, 64, 16), (8, 128, 64), (5, 32, 8), (1, 16, 256)])
def test_append(lens, new, Hk, D, page, order, dtype):
    import flash_b200 as fb
    cache = Cache(lens, Hk, D, page, dtype, 10, order)
    new = [min(n, m) if i % 2 else n for i, (n, m) in enumerate(zip(new, lens))]  # every other one may be longer than its sequence
    T, front = sum(new) + 5, 2
    k, v = (torch.randn(T, Hk, D, device="cuda").to(dtype) for _ in range(2))
    want_k, want_v = cache.k_pages.clone(), cache.v_pages.clone()
    row = front
    for b, n in enumerate(new):
        real = min(n, lens[b])
        place, rows = cache.places(b, lens[b] - real, lens[b]), slice(row + n - real, row + n)
        want_k[place], want_v[place] = k[rows], v[rows]
        row += n
    version = cache.k_pages._version
    fb.paged_append(k, v, cache.k_pages, cache.v_pages, cache.table, cache.kv_lens, _starts(new, front))
    assert cache.k_pages._version > version
    fb.check_status()
    assert torch.equal(cache.k_pages.view(torch.int16), want_k.view(torch.int16)) and torch.equal(cache.v_pages.view(torch.int16), want_v.view(torch.int16))


def test_append_of_strided_rows_and_single_tokens():
    import flash_b200 as fb
    cache = Cache([17, 64, 1], 2, 64, 16, BF16, 11)
    whole = torch.randn(3, 4, 64, device="cuda").to(BF16)
    odd = torch.randn(3, 2, 65, device="cuda").to(BF16)
    for k, v in ((whole[:, :2], whole[:, 2:]), (odd[..., 1:], whole[:, 1:3])):
        fb.paged_append(k, v, cache.k_pages, cache.v_pages, cache.table, cache.kv_lens)
        for b, n in enumerate(cache.lens):
            place = cache.places(b, n - 1, n)
            assert torch.equal(cache.k_pages[place][0], k[b]) and torch.equal(cache.v_pages[place][0], v[b])


def test_bad_pages_and_lengths_are_reported_and_harmless():
    import flash_b200 as fb
    lens, new = [100, 50, 300], [1, 50, 2]
    cache = Cache(lens, 2, 64, 16, BF16, 12).fill()
    q, k, v = torch.randn(53, 4, 64, device="cuda").to(BF16), torch.randn(53, 2, 64, device="cuda").to(BF16), torch.randn(53, 2, 64, device="cuda").to(BF16)
    good = cache.table.clone(), cache.kv_lens.clone()
    want = fb.paged_attention(q, cache.k_pages, cache.v_pages, *good, _starts(new))
    for page, length, what in ((-1, 100, "page"), (2 ** 31 - 1, 100, "page"), (None, -5, "length"), (None, 1 << 20, "length")):
        table, kv_lens = good[0].clone(), good[1].clone()
        if page is not None:
            table[0, 6] = page
        kv_lens[0] = length
        before = cache.k_pages.clone(), cache.v_pages.clone()
        got = fb.paged_attention(q, cache.k_pages, cache.v_pages, table, kv_lens, _starts(new))
        with pytest.raises(RuntimeError, match=what):
            fb.check_status()
        assert torch.allclose(got[1:].float(), want[1:].float(), atol=2 ** -6)  # the other sequences (cut elsewhere, perhaps)
        fb.paged_append(k[:1], v[:1], cache.k_pages, cache.v_pages, table[:1], kv_lens[:1])
        with pytest.raises(RuntimeError, match=what):
            fb.check_status()
        for x, y in zip((cache.k_pages, cache.v_pages), before):
            assert torch.equal(x.view(torch.int16), y.view(torch.int16))
    fb.check_status()
    assert torch.equal(fb.paged_attention(q, cache.k_pages, cache.v_pages, *good, _starts(new)), want)


def test_cache_beyond_two_to_the_31_elements():
    import flash_b200 as fb
    pages, page, Hk, D = 33000, 64, 8, 128  # 2.16e9 elements each
    k_pages, v_pages = (torch.empty(pages, page, Hk, D, device="cuda", dtype=BF16) for _ in range(2))
    lens, new = [200, 70], [3, 70]
    cache = Cache(lens, Hk, D, page, BF16, 13)
    cache.table[0, :4] = torch.tensor([32999, 0, 32800, 5], dtype=torch.int32)
    cache.table[1, :2] = torch.tensor([32900, 32790], dtype=torch.int32)
    cache.k_pages, cache.v_pages = k_pages, v_pages
    k, v = cache.k, cache.v
    fb.paged_append(k, v, k_pages, v_pages, cache.table, cache.kv_lens, _starts(lens))
    for b, n in enumerate(lens):
        rows = slice(cache.first[b], cache.first[b] + n)
        assert torch.equal(k_pages[cache.places(b, 0, n)], k[rows]) and torch.equal(v_pages[cache.places(b, 0, n)], v[rows])
    _attend(cache, 16, new, BF16)


def test_a_conversation_gives_what_dense_attention_gives():
    """A prompt in chunks, then token by token, two sequences of different lengths side by side, with capped and biased scores: each step appends and
    attends. The same as attention_scored over the whole sequence, to the roundings."""
    import flash_b200 as fb
    Hk, H, D, page, total = 2, 8, 64, 16, [213, 150]
    cache = Cache(total, Hk, D, page, BF16, 14)
    slopes = _slopes(H, True)
    q = [torch.randn(n, H, D, device="cuda").to(BF16) for n in total]
    out = [torch.empty_like(x) for x in q]
    done = [0, 0]
    steps = [[100, 60], [60, 1], [1, 60]] + [[1, 1]] * 29 + [[23, 0]]
    for new in steps:
        done = [d + n for d, n in zip(done, new)]
        kv_lens, rows = torch.tensor(done, dtype=torch.int32, device="cuda"), [slice(d - n, d) for d, n in zip(done, new)]
        k, v = (torch.cat([x[cache.first[b] + r.start: cache.first[b] + r.stop] for b, r in enumerate(rows)]) for x in (cache.k, cache.v))
        starts = None if new == [1, 1] else _starts(new)
        fb.paged_append(k, v, cache.k_pages, cache.v_pages, cache.table, kv_lens, starts)
        o = fb.paged_attention(torch.cat([x[r] for x, r in zip(q, rows)]), cache.k_pages, cache.v_pages, cache.table, kv_lens, starts, softcap=10.0, slopes=slopes)
        for x, r, part in zip(out, rows, o.split(new)):
            x[r] = part
    assert [d for d in done] == [213, 150]
    fb.check_status()
    for b, n in enumerate(total):
        r = slice(cache.first[b], cache.first[b] + n)
        Q, K, V = (x.transpose(0, 1)[None] for x in (q[b], cache.k[r], cache.v[r]))
        value, bound = attention_64(Q, K, V, torch.zeros_like(Q), True, None, None, None, 10.0, slopes, None)["o"]
        dense = fb.attention_scored(Q, K, V, True, softcap=10.0, slopes=slopes)
        for x in (dense, out[b].transpose(0, 1)[None]):
            assert ((x.double() - value).abs() <= bound).all()


def test_captured_step_follows_lengths_and_tables():
    import flash_b200 as fb
    lens, new = [900, 64, 300], [1, 1, 1]
    cache = Cache(lens, 2, 128, 16, BF16, 15).fill()
    q, k, v = torch.randn(3, 8, 128, device="cuda").to(BF16), torch.randn(3, 2, 128, device="cuda").to(BF16), torch.randn(3, 2, 128, device="cuda").to(BF16)
    table, kv_lens = cache.table.clone(), cache.kv_lens.clone()
    for _ in range(2):
        fb.paged_attention(q, cache.k_pages, cache.v_pages, table, kv_lens)
    graphs, outs = [], []
    torch.cuda.synchronize()
    for _ in range(2):  # two graphs, each with a workspace of its own
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            fb.paged_append(k, v, cache.k_pages, cache.v_pages, table, kv_lens)
            outs.append(fb.paged_attention(q, cache.k_pages, cache.v_pages, table, kv_lens))
        graphs.append(g)
    for lens in ([900, 64, 300], [10, 1, 300], [899, 33, 1]):
        kv_lens.copy_(torch.tensor(lens))
        cache.lens = lens
        table.copy_(cache.table)
        for x in (q, k, v):
            x.copy_(torch.randn_like(x, dtype=torch.float32))
        for b, n in enumerate(lens):
            cache.k[cache.first[b] + n - 1], cache.v[cache.first[b] + n - 1] = k[b], v[b]
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for got in outs:
            _check(got, cache, q, new)
    fb.check_status()


def test_streams_and_the_same_call_twice():
    import flash_b200 as fb
    caches = [Cache([4000 + 500 * i, 20, 700], 2, 64, 32, FP16, 16 + i).fill() for i in range(2)]
    new = [1, 20, 130]
    qs = [torch.randn(151, 8, 64, device="cuda").to(FP16) for _ in caches]
    call = lambda c, q: fb.paged_attention(q, c.k_pages, c.v_pages, c.table, c.kv_lens, _starts(new), softcap=7.0)  # noqa: E731
    want = [call(c, q) for c, q in zip(caches, qs)]
    streams = [torch.cuda.Stream() for _ in caches]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append((i, call(caches[i], qs[i])))
    torch.cuda.synchronize()
    for i, x in got:
        assert torch.equal(x, want[i])
        _check(x, caches[i], qs[i], new, cap=7.0)


def test_nothing_to_do():
    import flash_b200 as fb
    cache = Cache([5], 2, 64, 16, BF16, 18).fill()
    none = torch.empty(0, 4, 64, device="cuda", dtype=BF16)
    starts = torch.zeros(2, dtype=torch.int32, device="cuda")
    assert fb.paged_attention(none, cache.k_pages, cache.v_pages, cache.table, cache.kv_lens, starts).shape == (0, 4, 64)
    fb.paged_append(none[:, :2], none[:, :2], cache.k_pages, cache.v_pages, cache.table, cache.kv_lens, starts)
    q = torch.randn(3, 4, 64, device="cuda").to(BF16)
    nobody = fb.paged_attention(q, cache.k_pages, cache.v_pages, cache.table[:0], cache.kv_lens[:0], starts[:1])
    assert nobody.shape == q.shape and (nobody == 0).all()
    assert (fb.paged_attention(q, cache.k_pages, cache.v_pages, cache.table, cache.kv_lens, starts) == 0).all()  # sequences without new tokens
    fb.check_status()


def test_refusals():
    import flash_b200 as fb
    c = Cache([50, 60], 2, 64, 16, BF16, 19).fill()
    q, kv = torch.randn(2, 4, 64, device="cuda").to(BF16), torch.randn(2, 2, 64, device="cuda").to(BF16)
    good = dict(q=q, k_pages=c.k_pages, v_pages=c.v_pages, page_table=c.table, kv_lens=c.kv_lens)
    bad = [dict(q=q.half()), dict(q=q[:1]), dict(q=q[..., :32]), dict(q=q[:, :3]), dict(q=q[0]), dict(v_pages=c.v_pages[:1]), dict(k_pages=c.k_pages[:, :12], v_pages=c.v_pages[:, :12]),
           dict(page_table=c.table.long()), dict(page_table=c.table[0]), dict(page_table=c.table[:, :0]), dict(page_table=c.table.cpu()), dict(kv_lens=c.kv_lens.long()), dict(kv_lens=c.kv_lens[:1]),
           dict(kv_lens=c.kv_lens.cpu()), dict(q_starts=c.kv_lens), dict(softcap=-1.0), dict(slopes=torch.ones(2, device="cuda")), dict(prefix=c.kv_lens.long()),
           dict(prefix=c.kv_lens[:1]), dict(out=q), dict(out=torch.empty(2, 4, 64, device="cuda")), dict(out=torch.empty_like(q)[:1]), dict(out=torch.empty(2, 4, 65, device="cuda", dtype=BF16)[..., 1:]),
           dict(k_pages=torch.empty(5, 16, 2, 65, device="cuda", dtype=BF16)[..., :64], v_pages=torch.empty(5, 16, 2, 64, device="cuda", dtype=BF16))]
    for change in bad:
        with pytest.raises(ValueError):
            fb.paged_attention(**{**good, **change})
    with pytest.raises(NotImplementedError):
        fb.paged_attention(**good, sm_scale=0.0)
    for change in (dict(k=kv.half(), v=kv.half()), dict(v=kv[:1]), dict(k=kv[:, :1], v=kv[:, :1]), dict(v=kv.half()), dict(kv_lens=c.kv_lens.long())):
        with pytest.raises(ValueError):
            fb.paged_append(**{**dict(k=kv, v=kv, k_pages=c.k_pages, v_pages=c.v_pages, page_table=c.table, kv_lens=c.kv_lens), **change})
    asks = q.detach().requires_grad_()
    with pytest.raises(RuntimeError, match="gradient"):
        fb.paged_attention(**{**good, "q": asks})
    with torch.no_grad():
        fb.paged_attention(**{**good, "q": asks})
    fb.check_status()


def test_inference_mode_and_both_ways_through_the_host(monkeypatch):
    """Tensors made in inference mode have no version counters. The same bits by the native host call and by the Python one."""
    import flash_b200 as fb
    from flash_b200 import ops
    with torch.inference_mode():
        cache = Cache([100, 30], 2, 64, 16, BF16, 20)
        k, v, q = (torch.randn(2, h, 64, device="cuda").to(BF16) for h in (2, 2, 4))
        results = []
        for profile in (None, []):
            monkeypatch.setattr(ops, "PROFILE", profile)
            cache.fill()
            fb.paged_append(k, v, cache.k_pages, cache.v_pages, cache.table, cache.kv_lens)
            out = torch.empty_like(q)
            fb.paged_attention(q, cache.k_pages, cache.v_pages, cache.table, cache.kv_lens, out=out)
            results.append((cache.k_pages.clone(), cache.v_pages.clone(), out, fb.paged_attention(q, cache.k_pages, cache.v_pages, cache.table, cache.kv_lens)))
        for a, b in zip(*results):
            assert torch.equal(a.view(torch.int16), b.view(torch.int16))
        assert torch.equal(results[0][2], results[0][3])


def test_after_a_time_out_results_are_nan_until_it_has_been_read():
    import flash_b200 as fb
    from flash_b200 import ops
    cache = Cache([700, 40], 2, 64, 16, BF16, 21).fill()
    q, new = torch.randn(8, 4, 64, device="cuda").to(BF16), [1, 5]
    args = (cache.k_pages, cache.v_pages, cache.table, cache.kv_lens, _starts(new))
    want = fb.paged_attention(q, *args)
    ops._status_word(q.device).fill_(142)  # as a bounded wait that ran out leaves it
    assert torch.isnan(fb.paged_attention(q, *args)).all()
    rows = torch.randn(6, 2, 64, device="cuda").to(BF16)
    fb.paged_append(rows, rows, *args)  # waits for nothing that can run out
    place = cache.places(1, 35, 40)
    assert torch.equal(cache.k_pages[place], rows[1:]) and torch.equal(cache.v_pages[place], rows[1:])
    with pytest.raises(RuntimeError, match="role 42"):
        fb.check_status()
    cache.fill()
    assert torch.equal(fb.paged_attention(q, *args), want)


def test_neighbours_in_a_batch_do_not_reach_a_sequence():
    """Rows of another sequence in the same tile of queries, NaN among them, and what an earlier call left in shared memory."""
    import flash_b200 as fb
    cache = Cache([130, 130, 130], 2, 64, 16, BF16, 22).fill()
    new = [40, 3, 40]
    q = torch.randn(83, 4, 64, device="cuda").to(BF16)
    call = lambda: fb.paged_attention(q, cache.k_pages, cache.v_pages, cache.table, cache.kv_lens, _starts(new), softcap=3.0)  # noqa: E731
    want = call()
    q[:40] = float("nan")
    q[43:] *= 1e4
    for _ in range(3):
        assert torch.equal(call()[40:43], want[40:43])
    bad = cache.places(2, 0, 130)
    cache.k_pages[bad], cache.v_pages[bad] = float("nan"), float("nan")
    assert torch.equal(call()[40:43], want[40:43])


@pytest.mark.parametrize("cap", [None, 3.0])
@pytest.mark.parametrize("length, at, new", [(97, 96, 1), (97, 0, 1), (300, 130, 1), (20000, 7, 1), (20000, 19999, 1), (500, 400, 150), (20000, 19900, 200)])
def test_a_row_that_sees_a_key_that_is_not_a_number(length, at, new, cap):
    """It is NaN, whether the key is the only one of its warp, in a piece of an item, or in a tile of many rows; the rows in front of the key keep their bits."""
    import flash_b200 as fb
    cache = Cache([length, 140], 2, 64, 16, BF16, 23).fill()
    q = torch.randn(new + 1, 4, 64, device="cuda").to(BF16)
    place = cache.places(0, at, at + 1)
    call = lambda: fb.paged_attention(q, cache.k_pages, cache.v_pages, cache.table, cache.kv_lens, _starts([new, 1]), softcap=cap)  # noqa: E731
    cache.k_pages[place] = 0
    want = call()
    cache.k_pages[place] = float("nan")
    got = call()
    sees = torch.arange(length - new, length, device="cuda") >= at
    assert torch.equal(got[:new][~sees], want[:new][~sees]) and torch.equal(got[new:], want[new:])
    assert sees.any() and torch.isnan(got[:new][sees]).all()
    fb.check_status()


@pytest.mark.parametrize("cap", [3.0, 30.0, 1e4])
@pytest.mark.parametrize("slopes", [False, True])
@pytest.mark.parametrize("D, new", [(64, 3), (128, 3), (64, 40), (128, 90)])
def test_a_key_beyond_the_cap_leaves_the_bits_of_rows_in_front_of_it(D, new, slopes, cap):
    import flash_b200 as fb
    cache = Cache([333, 200], 2, D, 16, BF16, 24).fill()
    q = torch.randn(new + 1, 8, D, device="cuda").to(BF16)
    call = lambda: fb.paged_attention(q, cache.k_pages, cache.v_pages, cache.table, cache.kv_lens, _starts([new, 1]), softcap=cap, slopes=_slopes(8, slopes))  # noqa: E731
    want, place = call(), cache.places(0, 332, 333)
    cache.k_pages[place] *= 40 * cap
    got = call()
    assert torch.equal(got[:new - 1], want[:new - 1]) and torch.equal(got[new:], want[new:]) and not torch.equal(got, want)


@pytest.mark.parametrize("cap", [1e4, 1e6])
@pytest.mark.parametrize("slopes", [False, True])
@pytest.mark.parametrize("D, new", [(64, 3), (128, 3), (64, 40), (128, 90)])
def test_a_query_beyond_a_large_cap_among_ordinary_ones(D, new, slopes, cap):
    """Its neighbours are within their own bounds."""
    import flash_b200 as fb
    cache = Cache([333, 200], 2, D, 16, BF16, 25).fill()
    q = (torch.randn(new + 1, 8, D, device="cuda") * 1.5).to(BF16)
    args = (cache.k_pages, cache.v_pages, cache.table, cache.kv_lens, _starts([new, 1]))
    big = q.clone()
    big[1] *= 10 * cap
    got = fb.paged_attention(big, *args, softcap=cap, slopes=_slopes(8, slopes))
    got[1] = fb.paged_attention(q, *args, softcap=cap, slopes=_slopes(8, slopes))[1]
    _check(got, cache, q, [new, 1], cap=cap, slopes=_slopes(8, slopes))


@pytest.mark.parametrize("given", [False, True])
def test_a_time_out_on_record_while_the_call_runs(given):
    """The word is set by a copy beside the attention kernel, whose blocks have begun by then: no row keeps what was there, cut items' among them, but for rows of no
    sequence in `out`."""
    import time
    import flash_b200 as fb
    from flash_b200 import ops
    new, front, T = [4000, 1, 3, 2500], 2, 6510
    cache = Cache([60000, 30000, 700, 40000], 2, 128, 64, BF16, 26).fill()
    q = torch.randn(T, 32, 128, device="cuda").to(BF16)
    out = torch.full_like(q, 7.0)
    call = lambda **kw: fb.paged_attention(q, cache.k_pages, cache.v_pages, cache.table, cache.kv_lens, _starts(new, front), **kw)  # noqa: E731
    want = call()
    status, code, side = ops._status_word(q.device), torch.tensor([142], dtype=torch.int32).pin_memory(), torch.cuda.Stream()
    for _ in range(20):
        begin, middle, end = (torch.cuda.Event(enable_timing=True) for _ in range(3))
        torch.cuda.synchronize()
        begin.record()
        got = call(out=out.fill_(7.0)) if given else call()
        end.record()
        time.sleep(0.0005)
        with torch.cuda.stream(side):
            status.copy_(code, non_blocking=True)
            middle.record()
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="role 42"):
            fb.check_status()
        if begin.elapsed_time(middle) > 0.3 and middle.elapsed_time(end) > 0.3:  # (of some 5 ms; the copy has come too early or too late else)
            break
    else:
        pytest.skip("the copy has never come while the kernel ran")
    rows = slice(front, front + sum(new))
    assert torch.isnan(got[rows]).all()
    for x in (got[:front], got[front + sum(new):]):
        assert (x == 7.0).all() if given else torch.isnan(x).all()
    assert torch.equal(call(), want)


@pytest.mark.parametrize("cap", [None, 3.0])
@pytest.mark.parametrize("D, G, at", [(64, 4, 470), (128, 4, 470), (64, 1, 470), (128, 30, 425)])
def test_a_later_token_of_a_chunk_that_is_not_finite(D, G, at, cap):
    """100 tokens behind 400, keys and values from position `at` on NaN and infinite: they lie in the same 128 keys as what earlier blocks of 128 / G tokens see, none of whose
    rows sees them."""
    import flash_b200 as fb
    cache = Cache([500, 77], 2, D, 16, BF16, 27).fill()
    q = torch.randn(101, 2 * G, D, device="cuda").to(BF16)
    call = lambda: fb.paged_attention(q, cache.k_pages, cache.v_pages, cache.table, cache.kv_lens, _starts([100, 1]), softcap=cap)  # noqa: E731
    want, block = call(), 128 // G
    place = cache.places(0, at, 500)
    cache.k_pages[place], cache.v_pages[place] = float("nan"), float("inf")
    got, clean = call(), (at - 400) // block * block  # rows of blocks that end in front of it
    assert torch.equal(got[:clean], want[:clean]) and torch.equal(got[100:], want[100:])
    assert not torch.isfinite(got[at - 400: 100]).any()
    fb.check_status()


@pytest.mark.parametrize("code", [200, 201, 202])
def test_a_time_out_is_recorded_over_what_concerned_one_call(code):
    """A report that nobody has read yet lets later calls run; a wait that runs out in one of them (the test hook's here) has to stop those behind it."""
    import flash_b200 as fb
    from flash_b200 import _lib, ops
    cache = Cache([100, 30], 2, 64, 16, BF16, 28).fill()
    q = torch.randn(2, 4, 64, device="cuda").to(BF16)
    args = (q, cache.k_pages, cache.v_pages, cache.table, cache.kv_lens)
    want, status = fb.paged_attention(*args), ops._status_word(q.device)
    status.fill_(code)
    assert torch.equal(fb.paged_attention(*args), want) and int(status.item()) == code
    _lib.check(_lib.load().fa_debug_wait_timeout(status.data_ptr(), 20000, 42, ops._stream()), "fa_debug_wait_timeout")
    assert torch.isnan(fb.paged_attention(*args)).all() and torch.isnan(fb.attention(q[None].transpose(1, 2), q[None].transpose(1, 2), q[None].transpose(1, 2))).all()
    cache.kv_lens[0] = -1  # is reported, but not in the place of the time-out
    fb.paged_append(q[:, :2].contiguous(), q[:, :2].contiguous(), *args[1:])
    with pytest.raises(RuntimeError, match="role 42"):
        fb.check_status()


@pytest.mark.parametrize("cap, slopes", [(None, False), (5.0, False), (5.0, True)])
@pytest.mark.parametrize("G", [1, 4, 33])
def test_tokens_in_front_of_a_sequence_see_no_prefix(G, cap, slopes):
    """More new tokens than the sequence has: those at positions below 0 are nobody's (`paged_append` leaves them out) and give zeros, whatever the prefix."""
    lens, new = [1, 40, 0, 200], [24, 41, 3, 330]
    prefix = torch.tensor([28, 17, 5, 150], dtype=torch.int32, device="cuda")
    _attend(Cache(lens, 2, 64, 16, BF16, 29).fill(), 2 * G, new, BF16, prefix=prefix, cap=cap, slopes=_slopes(2 * G, slopes))
