"""Biased scores where a row's keys lie far apart: the first tokens, a prefix or a document's beginning, and then the keys next to the query. The far ones have biases of thousands; the
others' weights must not take that size's rounding, forward and backward, of long sequences and of paged caches."""
import pytest
import torch

import test_paged_e4m3_gpu as eight
import test_paged_masked_gpu as sixteen
from eight_bit_cache import Cache8
from masked_reference import attention_64, check, windowed
from test_paged_gpu import BF16, FP16, Cache
from test_window_gpu import FP32, NAMES, _inputs, _run

pytestmark = pytest.mark.gpu


def _slopes(H):
    return torch.tensor([(0.5, 0.25, 0.84, -0.02)[h % 4] for h in range(H)], device="cuda")


def _check(q, k, v, do, keep, window=None, sinks=0, **kw):
    got = _run(q, k, v, do, window, sinks, **kw)
    want = attention_64(q, k, v, do, keep, None, kw.get("softcap"), kw.get("slopes"))
    for n in NAMES:
        check(got[n], want[n], n)


@pytest.mark.parametrize("dtype", [FP16, BF16, FP32])
@pytest.mark.parametrize("softcap", [None, 10.0])
@pytest.mark.parametrize("M,N,window,sinks,prefix", [(200, 24000, 100, 4, None), (1, 24000, 300, 130, None), (20, 9000, 64, 1, None), (700, 700, 17, 1, None), (200, 24000, 100, 0, 5),
                                                     (3000, 3000, 200, 2, None)])
def test_first_keys_and_a_window(M, N, window, sinks, prefix, softcap, dtype):
    q, k, v, do = _inputs(1, 4, 2, M, N, 64, dtype, 1)
    p = None if prefix is None else torch.tensor([prefix], dtype=torch.int32, device="cuda")
    _check(q, k, v, do, windowed(M, N, window, sinks, p), window, sinks, slopes=_slopes(4), softcap=softcap, prefix=p)


@pytest.mark.parametrize("dtype", [FP16, BF16, FP32])
@pytest.mark.parametrize("softcap", [None, 10.0])
@pytest.mark.parametrize("M,N", [(256, 24000), (1500, 1500)])
def test_documents_that_are_scattered(M, N, softcap, dtype):
    """A document that has a few keys at the beginning and the last ones."""
    q, k, v, do = _inputs(1, 4, 2, M, N, 64, dtype, 2)
    ids = torch.full((N,), -2, device="cuda")
    ids[:3], ids[-200:] = -1, -1
    ids = ids.expand(1, 4, N)
    keep = windowed(M, N, N, 0) & (ids[:, :, N - M:, None] == ids[:, :, None, :])
    _check(q, k, v, do, keep, slopes=_slopes(4), softcap=softcap, eq=ids[..., N - M:], ek=ids)


@pytest.mark.parametrize("kind", [Cache, Cache8])
@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("softcap", [None, 10.0])
@pytest.mark.parametrize("G", [4, 20, 40])
@pytest.mark.parametrize("new", [[1, 1, 1], [300, 40, 5]], ids=["tokens", "chunks"])
def test_paged(new, G, softcap, dtype, kind):
    module = eight if kind is Cache8 else sixteen
    lens = [30000, 5000, 1000]
    for window, sinks, prefix in ((100, 4, None), (33, 130, None), (100, 0, (7, 0, 200))):
        p = None if prefix is None else torch.tensor(prefix, dtype=torch.int32, device="cuda")
        module._attend(kind(lens, 1, 64, 64, dtype, 3).fill(), G, new, dtype, window, sinks, prefix=p, slopes=_slopes(G), softcap=softcap)
