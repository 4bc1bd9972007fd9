"""Windows, sinks and parents of paged_attention without a GPU: how the work is cut, and what is refused."""
import ctypes

import pytest
import torch

import flash_b200 as fb
from flash_b200 import _lib
from test_paged import _cache


def _cut(lens, new, Hk, G, workers, window, sinks, tree, prefix=None, capacity=1 << 20):
    lib, ints = _lib.load(), lambda v: (ctypes.c_int32 * len(v))(*v)  # noqa: E731
    first = [0]
    for n in new:
        first.append(first[-1] + n)
    args = (len(lens), first[-1], Hk, G, capacity, ints(lens), ints(first), None if prefix is None else ints(prefix), _lib.Window(window, sinks), 256 if tree else None, workers)
    rows = (ctypes.c_int32 * 8)()
    n = lib.fa_debug_paged_pieces_more(*args, rows, 1)
    rows = (ctypes.c_int32 * (8 * max(1, n)))()
    assert lib.fa_debug_paged_pieces_more(*args, rows, n) == n
    got = [tuple(rows[8 * i: 8 * i + 8]) for i in range(n)]
    return [r for r in got if r[0] >= 0], [r for r in got if r[0] < 0]


def _blocks(length, n, tile, tokens, window, sinks, tree, front):
    """Key blocks that the item has: those up to its last token's last key, less those that lie whole between the first keys and the window."""
    base = length - n
    end = max(min(base + (tile + 1) * tokens, length), front, 0)
    blocks = -(-end // 128)
    if window:
        early, low = -(-max(front, sinks) // 128), max(0, base + (0 if tree and n <= 256 else tile * tokens) - window + 1) // 128
        blocks -= max(0, low - early)
    return blocks


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (100, 4), (4096, 1000), (1 << 22, 0)])
@pytest.mark.parametrize("workers", [1, 7, 148])
@pytest.mark.parametrize("lens,new,Hk,G,prefix", [
    ([1], [1], 1, 1, None), ([131072], [1], 8, 8, None), ([9000] * 64, [1] * 64, 8, 4, None), ([700, 1, 129, 0], [300, 1, 64, 0], 3, 5, None),
    ([20000, 7500, 10], [500, 200, 25], 2, 4, None), ([5000, 3000], [2000, 40], 2, 4, [700, 2990]), ([333] * 200, [9] * 200, 1, 16, None),
])
def test_every_key_block_is_in_one_piece(lens, new, Hk, G, prefix, workers, window, sinks, tree):
    pieces, merges = _cut(lens, new, Hk, G, workers, window, sinks, tree, prefix)
    tokens, want = 128 // G, {}
    for b, (length, n) in enumerate(zip(lens, new)):
        for tile in range(-(-n // tokens)):
            for h in range(Hk):
                want[b, h, tile] = _blocks(length, n, tile, tokens, window, sinks, tree, 0 if prefix is None else min(prefix[b], length))
    got, slots, merged, loads = {}, set(), {}, {}
    for w, b, h, tile, lo, hi, n, part in pieces:
        assert n == want[b, h, tile] and 0 <= lo <= hi <= n and 0 <= w < workers
        got.setdefault((b, h, tile), []).append((lo, hi, part))
        loads[w] = loads.get(w, 0) + hi - lo
        assert (part < 0) == (hi - lo == n)
        if part >= 0:
            assert part not in slots and part < 2 * workers
            slots.add(part)
    for _, b, h, tile, _, _, _, slot in merges:
        merged.setdefault((b, h, tile), []).append(slot)
    assert set(got) == set(want)
    for key, parts in got.items():
        end = 0
        for lo, hi, _ in sorted(parts):
            assert lo == end
            end = hi
        assert end == want[key]
        assert (len(parts) == 1) == (parts[0][2] < 0) == (key not in merged)
        if len(parts) > 1:
            assert merged[key] == [p for _, _, p in sorted(parts)]


def test_a_windows_work_is_shared_out_by_what_it_shows():
    """Two sequences that see alike, one of them with a cache a hundred times as long: nobody has much more to do than the others."""
    pieces, _ = _cut([400000, 4500] * 200, [1, 1] * 200, 1, 4, 148, 4096, 4, False)
    loads = {}
    for w, _, _, _, lo, hi, _, _ in pieces:
        loads[w] = loads.get(w, 0) + hi - lo
    assert len(loads) == 148 and max(loads.values()) <= 1.2 * sum(loads.values()) / 148


def _attend(**kw):
    q, pages = torch.zeros(2, 4, 64, dtype=torch.bfloat16), torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16)
    ints = torch.zeros(2, 2, dtype=torch.int32)
    return fb.paged_attention(q, pages, pages, ints, ints[0], **kw)


@pytest.mark.parametrize("kw,match", [
    (dict(window=0), "at least 1"), (dict(window=1.5), "integer"), (dict(sinks=2), "need a window"), (dict(window=3, sinks=-2), "negative"),
    (dict(parents=torch.zeros(2, dtype=torch.int32), slopes=torch.zeros(4)), "without slopes and prefix"),
    (dict(parents=torch.zeros(2, dtype=torch.int32), prefix=torch.zeros(2, dtype=torch.int32)), "without slopes and prefix"),
])
def test_python_refuses(kw, match):
    with pytest.raises(ValueError, match=match):
        _attend(**kw)


def _code(more, scores=None):
    rows = _lib.Rows(256, (256, 64))
    return _lib.load().fa_paged_fwd_more(_cache(), more, 2, 4, None, 0.1, scores, rows, rows, 1, 256, 1 << 30, 256, None)


def test_c_entry_refuses():
    for window in ((-1, 0), (0, 1), (4, -1)):
        assert _code(_lib.PagedMore(_lib.Window(*window))) == 9
    assert _code(_lib.PagedMore(_lib.Window(0, 0), 256), _lib.Scores(0.0, 256, None)) == 9
    assert _code(_lib.PagedMore(_lib.Window(0, 0), 256), _lib.Scores(0.0, None, 256)) == 9
    assert _code(_lib.PagedMore(_lib.Window(4, 0), 258)) == 3
