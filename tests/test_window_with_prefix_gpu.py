"""Few queries of attention_scored with a window and a prefix: the prefix may show them any number of keys, so that the forward is cut into the runs that all keys would be cut into."""
import pytest
import torch

from test_window_gpu import BF16, FP16, _compare, _inputs

pytestmark = pytest.mark.gpu


def _launches(call):
    from flash_b200 import ops
    before = ops.LAUNCHES
    call()
    return ops.LAUNCHES - before


@pytest.mark.parametrize("general", [False, True])
@pytest.mark.parametrize("B,H,Hk,M,N,D", [(1, 32, 8, 1, 16384, 128), (1, 8, 8, 30, 9000, 64), (2, 4, 1, 200, 5000, 128)])
def test_the_forward_is_cut_as_without_the_window(B, H, Hk, M, N, D, general, monkeypatch):
    """A prefix of all keys, a window of few: the kernels that are launched are those of the prefix alone (the forward and the one that joins its runs)."""
    import flash_b200 as fb
    from flash_b200 import scored
    if general:
        monkeypatch.setattr(scored, "_native", lambda *tensors: None)
    q, k, v, _ = _inputs(B, H, Hk, M, N, D, BF16, 1)
    prefix = torch.full((B,), N, dtype=torch.int32, device="cuda")
    alone = _launches(lambda: fb.attention_scored(q, k, v, True, prefix=prefix))
    assert alone == 2
    assert _launches(lambda: fb.attention_scored(q, k, v, True, prefix=prefix, window=16)) == alone
    assert _launches(lambda: fb.attention_scored(q, k, v, True, prefix=prefix, window=16, sinks=4)) == alone
    assert _launches(lambda: fb.attention_scored(q, k, v, True, window=16)) == 1


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("prefix", [(0, 5000), (1, 128), (4999, 130), (2500, 3)])
@pytest.mark.parametrize("H,Hk,M,D,window,sinks", [(8, 2, 1, 128, 16, 0), (4, 4, 30, 64, 200, 3), (6, 2, 200, 128, 1, 0), (8, 1, 7, 32, 2600, 130)])
def test_prefixes_of_all_lengths(H, Hk, M, D, window, sinks, prefix, dtype):
    """Where the prefix is short most runs have no keys."""
    q, k, v, do = _inputs(2, H, Hk, M, 5000, D, dtype, 2)
    p = torch.tensor(prefix, dtype=torch.int32, device="cuda")
    _compare(q, k, v, do, window, sinks, prefix=p)
    _compare(q, k, v, do, window, sinks, prefix=p, softcap=10.0)
