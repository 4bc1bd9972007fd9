"""CPU tests of the paged cache: how a batch is cut among the blocks, by the kernels' own code on the host, and what the library and the Python calls
refuse before a device is touched."""
import ctypes
import random

import pytest
import torch

from flash_b200 import _lib, paged_append, paged_attention


def _cut(lens, new, Hk, G, workers, prefix=None, capacity=1 << 20, starts=True):
    lib = _lib.load()
    B, ints = len(lens), lambda v: (ctypes.c_int32 * len(v))(*v)  # noqa: E731
    first = [0]
    for n in new:
        first.append(first[-1] + n)
    args = (B, first[-1], Hk, G, capacity, ints(lens), ints(first) if starts else None, None if prefix is None else ints(prefix), workers)
    rows = (ctypes.c_int32 * 8)()
    n = lib.fa_debug_paged_pieces(*args, rows, 1)
    rows = (ctypes.c_int32 * (8 * max(1, n)))()
    assert lib.fa_debug_paged_pieces(*args, rows, n) == n
    got = [tuple(rows[8 * i: 8 * i + 8]) for i in range(n)]
    return [r for r in got if r[0] >= 0], [r for r in got if r[0] < 0]


def _check(lens, new, Hk, G, workers, prefix=None, capacity=1 << 20):
    """Every key tile of every item in one piece, every item's pieces either one that goes to the output or all of them merged, in order."""
    pieces, merges = _cut(lens, new, Hk, G, workers, prefix, capacity)
    tokens = 128 // G
    want = {}
    for b, (length, n) in enumerate(zip(lens, new)):
        length = min(max(length, 0), capacity)
        front = 0 if prefix is None else min(max(prefix[b], 0), length)
        for tile in range(-(-n // tokens)):
            last = length - n + min((tile + 1) * tokens, n) - 1
            keys = max(last + 1, front, 0)
            for h in range(Hk):
                want[b, h, tile] = -(-keys // 128)
    got, slots, loads = {}, set(), {}
    for w, b, h, tile, lo, hi, n, part in pieces:
        assert n == want[b, h, tile] and 0 <= lo <= hi <= n and 0 <= w < workers
        got.setdefault((b, h, tile), []).append((lo, hi, part))
        loads[w] = loads.get(w, 0) + hi - lo
        assert (part < 0) == (hi - lo == n)
        if part >= 0:
            assert part not in slots and part < 2 * workers
            slots.add(part)
    merged = {}
    for _, b, h, tile, _, _, _, slot in merges:
        merged.setdefault((b, h, tile), []).append(slot)
    assert set(got) == set(want)
    for key, parts in got.items():
        end = 0
        for lo, hi, _ in sorted(parts):
            assert lo == end, key
            end = hi
        assert end == want[key]
        whole = len(parts) == 1
        assert whole == (parts[0][2] < 0) and (key in merged) == (not whole)
        if not whole:
            assert merged[key] == [p for _, _, p in sorted(parts)]
    return loads


@pytest.mark.parametrize("workers", [1, 7, 148])
@pytest.mark.parametrize("lens,new,Hk,G", [
    ([700], [1], 8, 1), ([131072], [1], 8, 8), ([5], [5], 1, 128), ([0, 0], [1, 0], 2, 4), ([0], [0], 1, 1), ([1000] * 64, [1] * 64, 8, 4),
    ([8000, 1, 3000, 64], [500, 1, 3000, 0], 4, 6), ([100], [300], 2, 4), ([4096], [4096], 2, 1), ([17, 0, 129, 128, 127], [17, 0, 129, 1, 2], 3, 5),
])
def test_cuts(lens, new, Hk, G, workers):
    _check(lens, new, Hk, G, workers)
    _check(lens, new, Hk, G, workers, prefix=[n // 2 for n in lens])


def test_cuts_of_random_batches():
    rng = random.Random(0)
    for _ in range(150):
        B = rng.choice((1, 2, 5, 40))
        lens = [rng.choice((0, 1, 127, 128, 129, rng.randrange(1, 20000))) for _ in range(B)]
        new = [rng.choice((0, 1, 1, min(n, rng.randrange(0, 600)), n % 700, rng.randrange(0, 200))) for n in lens]
        prefix = None if rng.random() < 0.5 else [rng.randrange(-5, 3000) for _ in range(B)]
        _check(lens, new, rng.choice((1, 2, 8)), rng.choice((1, 2, 3, 4, 7, 8, 64, 128)), rng.choice((1, 2, 13, 148)), prefix, rng.choice((1 << 20, 4096)))


@pytest.mark.parametrize("B", [31, 32, 33, 63, 64, 65, 96, 97, 127, 128, 129, 200])
def test_sequences_that_share_an_entry_of_the_table_of_sums(B):
    """Up to 128 sequences the table has 32 entries, of one to four sequences each (the last ones perhaps of none), beyond it 1024."""
    rng = random.Random(B)
    for workers in (1, 7, 148):
        _check([500] * B, [1] * B, 2, 4, workers)
        for _ in range(6):
            lens = [rng.choice((0, 1, 127, 128, 129, rng.randrange(1, 9000))) for _ in range(B)]
            new = [rng.choice((0, 0, 1, 1, min(n, rng.randrange(0, 300)))) for n in lens]
            prefix = None if rng.random() < 0.5 else [rng.randrange(-5, 3000) for _ in range(B)]
            _check(lens, new, rng.choice((1, 2, 8)), rng.choice((1, 4, 7, 64)), workers, prefix)


def test_more_sequences_than_entries_of_the_table_of_sums():
    rng = random.Random(1)
    for B in (1024, 1025, 5000):
        lens = [rng.randrange(0, 300) for _ in range(B)]
        _check(lens, [rng.choice((0, 1, 1, 3)) for _ in range(B)], 2, 4, 148)


def test_work_is_even():
    """A worker's tiles: its share of all keys, one more for either end, and what its items' fixed costs are taken for."""
    rng = random.Random(2)
    lens = [rng.randrange(1500, 9000) for _ in range(64)]
    loads = _check(lens, [1] * 64, 8, 4, 148)
    assert len(loads) == 148 and max(loads.values()) <= 1.15 * sum(loads.values()) / 148 + 2
    loads = _check([131072], [1], 8, 8, 148)
    # stretches of equal length: a tile more or less at either end, and 640 / 128 = 5 tiles less where an item begins
    assert len(loads) == 148 and max(loads.values()) - min(loads.values()) <= 2 + 5


def test_lengths_beyond_everything_stay_inside():
    big = 2 ** 31 - 1
    _check([big, -big, 5000], [1, 1, 1], 2, 4, 148, prefix=[big, -big, big], capacity=4096)
    pieces, _ = _cut([300, 300], [1, 1], 2, 4, 148, starts=False)
    assert {p[1] for p in pieces} == {0, 1}
    # starts that fall or leave the rows: nothing outside [0, T)
    lib, ints = _lib.load(), lambda v: (ctypes.c_int32 * len(v))(*v)  # noqa: E731
    rows = (ctypes.c_int32 * 800)()
    n = lib.fa_debug_paged_pieces(3, 10, 1, 1, 4096, ints([50, 50, 50]), ints([-5, 8, 3, 1000]), None, 4, rows, 100)
    assert 0 < n <= 100


def test_a_wait_for_the_longest_item_fits_its_type():
    """The longest limit that a wait may be given, times the tiles of an item of the longest sequence and one."""
    import os
    import re
    csrc = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "triton-flash-attention-with-flexible-masks_b200", "csrc")
    read = lambda name: open(os.path.join(csrc, name)).read()  # noqa: E731
    most = int(re.search(r"kMost = 1LL << (\d+);", read("api.cu")).group(1))
    tokens = int(re.search(r"kMostTokens = 1 << (\d+);", read("paged.cu")).group(1))
    assert "ab.limit * (T + 1)" in read("paged_fwd.cu")
    assert (1 << most) * ((1 << tokens) // 128 + 1) < 1 << 63


def _cache(**kw):
    c = dict(B=2, Hk=2, D=64, dtype=0, pages=8, page_size=16, table_pages=4, table=256, table_stride=4, lens=256, k=256, v=256,
             k_stride=(16 * 2 * 64, 2 * 64, 64), v_stride=(16 * 2 * 64, 2 * 64, 64))
    c.update(kw)
    three = ctypes.c_int64 * 3
    c["k_stride"], c["v_stride"] = three(*c["k_stride"]), three(*c["v_stride"])
    return _lib.PagedCache(*c.values())


def _append(c, T=2, starts=None, k=None, v=None, status=256):
    rows = _lib.Rows(256, (128, 64))
    return _lib.load().fa_paged_append(c, T, starts, k or rows, v or rows, status, None)


def _attend(c, T=2, H=4, starts=None, q=None, o=None, scale=0.1, scores=None, work=256, size=1 << 30, status=256):
    rows = _lib.Rows(256, (256, 64))
    return _lib.load().fa_paged_fwd(c, T, H, starts, scale, scores, q or rows, o or rows, 1, work, size, status, None)


@pytest.mark.parametrize("kw,code", [
    (dict(B=0), 1), (dict(Hk=0), 1), (dict(pages=0), 1), (dict(D=48), 2), (dict(D=256), 2), (dict(dtype=2), 2), (dict(page_size=12), 10), (dict(page_size=4), 10),
    (dict(page_size=0), 1), (dict(table_pages=1 << 20, table_stride=1 << 20), 10), (dict(table_stride=3), 1), (dict(table=None), 1), (dict(lens=None), 1),
    (dict(table=258), 3), (dict(k=264), 3), (dict(v=None), 1), (dict(k_stride=(16 * 2 * 64, 2 * 64, 60)), 3), (dict(v_stride=(-2048, 128, 64)), 3), (dict(B=70000), 10),
])
def test_caches_that_the_library_refuses(kw, code):
    assert _append(_cache(**kw)) == code
    assert _attend(_cache(**kw)) == code
    assert _lib.load().fa_paged_workspace_bytes(_cache(**kw), ctypes.byref(ctypes.c_size_t(0))) == code


def test_calls_that_the_library_refuses():
    c = _cache()
    assert _append(None) == 1 and _attend(None) == 1
    for call in (_append, _attend):
        assert call(c, T=3) == 1               # without starts T is B
        assert call(c, T=0) == 1
        assert call(c, status=None) == 1
        assert call(c, starts=258) == 3
    assert _append(c, k=_lib.Rows(256, (100, 64))) == 3 and _append(c, v=_lib.Rows(None, (128, 64))) == 1
    assert _attend(c, H=3) == 1 and _attend(c, H=0) == 1 and _attend(c, H=516) == 2
    assert _attend(c, scale=0.0) == 2 and _attend(c, q=_lib.Rows(264, (256, 64))) == 3 and _attend(c, o=_lib.Rows(256, (256, 4))) == 3
    assert _attend(c, scores=_lib.Scores(-1.0, None, None)) == 9 and _attend(c, scores=_lib.Scores(1.0, 258, None)) == 3
    assert _attend(c, work=260) == 3
    assert b"page size" in _lib.load().fa_error_string(10)


def test_python_calls_refuse_before_a_launch():
    pages = torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16)
    rows, table, lens = torch.zeros(2, 2, 64, dtype=torch.bfloat16), torch.zeros(2, 2, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged_append(rows, rows, pages, pages, table, lens)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged_attention(rows, pages, pages, table, lens)
    with pytest.raises(ValueError):
        paged_append(rows, rows[:1], pages, pages, table, lens)
    with pytest.raises(ValueError):
        paged_attention(rows[0], pages, pages, table, lens)


def test_tangents_are_refused():
    """In front of all that asks for a device, so that it shows here."""
    import torch.autograd.forward_ad as fwad
    pages = torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16)
    rows, table, lens = torch.zeros(2, 2, 64, dtype=torch.bfloat16), torch.zeros(2, 2, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    slopes = torch.ones(2)
    with fwad.dual_level():
        dual = lambda x: fwad.make_dual(x, torch.ones_like(x))  # noqa: E731
        for args in ((dual(rows), rows, pages, pages), (rows, dual(rows), pages, pages), (rows, rows, dual(pages), pages), (rows, rows, pages, dual(pages))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                paged_append(*args, table, lens)
        for args, kw in (((dual(rows), pages, pages), {}), ((rows, dual(pages), pages), {}), ((rows, pages, dual(pages)), {}), ((rows, pages, pages), dict(slopes=dual(slopes)))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                paged_attention(*args, table, lens, **kw)
        with pytest.raises(RuntimeError, match="CUDA"):  # within a level, and none of them dual
            paged_append(rows, rows, pages, pages, table, lens)


def test_tensor_memory_is_taken_between_the_wait_and_the_next_launch():
    """The order that test_launch_order.py asks of the other kernels that allocate tensor memory."""
    import os
    import re
    csrc = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "triton-flash-attention-with-flexible-masks_b200", "csrc")
    for name in sorted(os.listdir(csrc)):
        with open(os.path.join(csrc, name)) as f:
            code = re.sub(r"//[^\n]*|/\*.*?\*/", "", f.read(), flags=re.S)
        if name == "paged_fwd.cu":
            assert code.count("take_tensor_memory(") == 1
            alloc = code.index("take_tensor_memory(")
            start, barrier = code.rindex("__global__", 0, alloc), code.index("__syncthreads();", alloc)
            go = code.index("launch_dependents();", start)
            assert start < code.index("wait_prerequisites();", start) < alloc < barrier < go
        elif name != "ptx.cuh":
            assert "take_tensor_memory(" not in code, name
