"""paged_attention with a window or drafted trees where nothing that the masks hide from all of a sequence's tokens is a number: keys, values and scales in slots of pages that are seen in
part, whole pages that were given away, and the table's entries of these."""
import pytest
import torch

import test_paged_e4m3_gpu as eight
import test_paged_masked_gpu as sixteen
from eight_bit_cache import Cache8
from masked_reference import paged_keep
from test_paged_gpu import BF16, FP16, Cache, _starts
from test_paged_masked_gpu import _parents, _slopes, _tree

pytestmark = pytest.mark.gpu


def _hide(cache, keeps):
    """How many slots of pages that are seen in part, and how many pages, hold no numbers afterwards."""
    slots = pages = 0
    for b, keep in enumerate(keeps):
        seen = keep.any(0)
        at = (~seen).nonzero()[:, 0]
        page, slot = cache.table[b].long()[at // cache.page], at % cache.page
        if isinstance(cache, Cache8):
            for x in (cache.k_pages, cache.v_pages):
                x.view(torch.uint8)[page, slot] = 127
            for x in (cache.k_scales, cache.v_scales):
                x.view(torch.uint8)[page, :, slot] = 255
        else:
            cache.k_pages[page, slot], cache.v_pages[page, slot] = float("nan"), float("inf")
        slots += len(at)
        for i in range(-(-seen.shape[0] // cache.page)):
            own = seen[i * cache.page: (i + 1) * cache.page]
            if not own.any():
                slots -= len(own)
                pages += 1
                if i % 3:
                    cache.table[b, i] = (-3, 1 << 29)[i % 3 - 1]
    return slots, pages


def _attend(cache, G, new, dtype, window, sinks, trees=None, prefix=None, softcap=None, slopes=None, single=False):
    import flash_b200 as fb
    H = cache.k.shape[1] * G
    gen = torch.Generator(device="cuda").manual_seed(1)
    q = (torch.randn(sum(new), H, cache.k.shape[2], generator=gen, device="cuda") * 1.5).to(dtype)
    keeps = [paged_keep(length, n, window, sinks, None if trees is None or n > 256 else trees[b], 0 if prefix is None else prefix[b])
             for b, (length, n) in enumerate(zip(cache.lens, new))]
    slots, pages = _hide(cache, keeps)
    assert slots > 0 and pages > 0
    scales = cache.scales() if isinstance(cache, Cache8) else {}
    p = None if prefix is None else torch.tensor(prefix, dtype=torch.int32, device="cuda")
    got = fb.paged_attention(q, cache.k_pages, cache.v_pages, cache.table, cache.kv_lens, None if single else _starts(new), window=window, sinks=sinks,
                             parents=None if trees is None else _parents(trees), prefix=p, softcap=softcap, slopes=slopes, **scales)
    fb.check_status()
    (eight if scales else sixteen).compare(got, cache, q, new, keeps, softcap, slopes)


CHANGES = [{}, dict(softcap=6.0), dict(slopes=True), dict(softcap=6.0, slopes=True)]


@pytest.mark.parametrize("kind", [Cache8, Cache])
@pytest.mark.parametrize("changes", CHANGES, ids=["plain", "cap", "bias", "both"])
@pytest.mark.parametrize("window,sinks", [(17, 1), (70, 0), (300, 130)])
@pytest.mark.parametrize("Hk,G,D,page,dtype", [(2, 4, 128, 16, BF16), (1, 1, 64, 64, FP16), (1, 12, 128, 128, FP16), (1, 48, 64, 16, BF16), (2, 8, 32, 32, BF16)])
def test_chunks_and_single_tokens(Hk, G, D, page, dtype, window, sinks, changes, kind):
    """Items of many rows, of few, and of the fewest, which warps multiply by themselves over 8 bits."""
    lens, new = [900, 800, 1000, 700, 1300], [200, 20, 1, 5, 2]
    kw = dict(changes, slopes=_slopes(Hk * G) if changes.get("slopes") else None)
    _attend(kind(lens, Hk, D, page, dtype, 4).fill(), G, new, dtype, window, sinks, **kw)
    if not changes.get("slopes"):
        _attend(kind(lens, Hk, D, page, dtype, 4).fill(), G, new, dtype, window, sinks, trees=[_tree(n, 10 + b) for b, n in enumerate(new)], **kw)


@pytest.mark.parametrize("kind", [Cache8, Cache])
@pytest.mark.parametrize("window,sinks,prefix", [(1, 0, None), (100, 3, None), (129, 128, None), (300, 2, (0, 50, 9, 300, 100, 4000, 1, 0, 1000))])
@pytest.mark.parametrize("Hk,G,D,page,dtype", [(2, 4, 128, 16, BF16), (2, 8, 64, 32, FP16), (1, 12, 128, 128, BF16), (2, 16, 32, 16, FP16), (1, 17, 64, 16, BF16)])
def test_calls_of_single_tokens(Hk, G, D, page, dtype, window, sinks, prefix, kind):
    lens = [1, 700, 0, 128, 129, 5000, 31, 16, 2500]
    for changes in CHANGES:
        kw = dict(changes, slopes=_slopes(Hk * G) if changes.get("slopes") else None)
        _attend(kind(lens, Hk, D, page, dtype, 20).fill(), G, [1] * len(lens), dtype, window, sinks, prefix=prefix, single=True, **kw)


@pytest.mark.parametrize("kind", [Cache8, Cache])
@pytest.mark.parametrize("order", ["phd", "hpd"])
def test_prefixes_and_orders(order, kind):
    lens, new, prefix = [900, 77, 1000, 428], [300, 20, 1, 5], (0, 50, 300, 2000)
    _attend(kind(lens, 2, 128, 32, BF16, 5, order).fill(), 4, new, BF16, 200, 3, prefix=prefix)
    _attend(kind(lens, 2, 128, 32, BF16, 5, order).fill(), 4, new, BF16, 33, 0, prefix=prefix, softcap=6.0, slopes=_slopes(8))


@pytest.mark.parametrize("kind", [Cache8, Cache])
def test_long_caches_that_are_cut(kind):
    """Pieces that begin, end and meet between the first keys and the window."""
    for lens, new, Hk, G, D in (([60000], [1], 2, 8, 128), ([20000, 700, 33333], [1, 70, 200], 1, 4, 64)):
        for window, sinks in ((500, 4), (3000, 700)):
            _attend(kind(lens, Hk, D, 64, BF16, 6).fill(), G, new, BF16, window, sinks)
