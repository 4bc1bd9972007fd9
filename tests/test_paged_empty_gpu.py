"""paged_attention of many new tokens whose sequences hold nothing: zeros, whatever else the batch has, call after call."""
import pytest
import torch

from eight_bit_cache import Cache8
from test_paged_gpu import BF16, FP16, Cache, _starts

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", [Cache8, Cache])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("G,D", [(4, 128), (20, 128), (24, 128), (32, 64), (40, 128)])
@pytest.mark.parametrize("single", [False, True])
def test_rows_of_empty_sequences_are_zeros(single, G, D, dtype, kind):
    """Items without tiles of few rows go through the staging of those with tiles; every twentieth sequence has some keys."""
    import flash_b200 as fb
    lens = [200 if b % 20 == 7 else 0 for b in range(1500)]
    new = [1] * len(lens)
    cache = kind(lens, 4, D, 16, dtype, 1).fill()
    scales = cache.scales() if kind is Cache8 else {}
    gen = torch.Generator(device="cuda").manual_seed(2)
    q = (torch.randn(len(lens), 4 * G, D, generator=gen, device="cuda") * 3e4).to(dtype)
    empty = torch.tensor([n == 0 for n in lens], device="cuda")
    starts = None if single else _starts(new)
    call = lambda: fb.paged_attention(q, cache.k_pages, cache.v_pages, cache.table, cache.kv_lens, starts, **scales)  # noqa: E731
    for _ in range(60):
        got = call()
        assert (got[empty] == 0).all() and (got[~empty] != 0).any()  # (3e4 times a normal number may be infinite in fp16, and rows that see keys NaN)
    fb.check_status()
