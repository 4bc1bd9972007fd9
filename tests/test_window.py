"""What attention_scored and the C entries refuse of a window, without a GPU."""
import ctypes

import pytest
import torch

import flash_b200 as fb
from flash_b200 import _lib


def _call(**kw):
    q = torch.zeros(1, 2, 8, 64, dtype=torch.bfloat16)
    causal = kw.pop("causal", True)
    return fb.attention_scored(q, q, q, causal, **kw)


@pytest.mark.parametrize("kw,match", [
    (dict(window=0), "at least 1"), (dict(window=-5), "at least 1"), (dict(window=2.0), "integer"), (dict(window="4"), "integer"),
    (dict(window=4, sinks=-1), "negative"), (dict(window=4, sinks=1.5), "integer"), (dict(sinks=3), "need a window"),
])
def test_python_refuses(kw, match):
    with pytest.raises(ValueError, match=match):
        _call(**kw)


def test_a_window_needs_a_causal_mask_and_a_gpu():
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        _call(window=4, causal=False)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        _call(window=4, sinks=2)


def _problem(**kw):
    base = dict(B=1, H=2, Hk=2, M=256, N=256, D=64, dtype=0, causal=1, mode=0, id_heads=1, sm_scale=0.1)
    return _lib.Problem(**{**base, **kw})


def _codes(problem, window, scores=None):
    lib, t = _lib.load(), _lib.Tensor(256, (64 * 256 * 2, 64 * 256, 64, 1))
    w = None if window is None else _lib.Window(*window)
    plan = lib.fa_plan_build_windowed(problem, scores, w, None, None, 256, 512, 256, None)
    fwd = lib.fa_fwd_windowed(problem, scores, w, t, t, t, t, None, None, None, 1, None, 0, 256, None)
    bwd = lib.fa_bwd_windowed(problem, scores, w, t, t, t, t, None, t, None, None, t, t, t, None, None, 0, 256, None)
    return plan, fwd, bwd


@pytest.mark.parametrize("window", [(-1, 0), (0, 2), (5, -1)])
def test_c_entries_refuse_bad_windows(window):
    assert _codes(_problem(), window) == (9, 9, 9)


def test_c_entries_refuse_windows_without_a_causal_mask():
    assert _codes(_problem(causal=0), (5, 0)) == (9, 9, 9)
    assert _codes(_problem(causal=0), (5, 0), _lib.Scores(3.0, None, None)) == (9, 9, 9)


def test_runs_of_keys_go_by_the_window():
    """Without a GPU the number of SMs is not known and nothing is cut; arguments are looked at all the same."""
    lib = _lib.load()
    assert lib.fa_fwd_splits_windowed(_problem(M=1, N=100000), None) >= 1
    assert lib.fa_fwd_splits_windowed(_problem(M=1, N=100000), _lib.Window(2 ** 31 - 1, 2 ** 31 - 1)) >= 1
    assert lib.fa_fwd_splits_windowed(ctypes.POINTER(_lib.Problem)(), _lib.Window(4, 0)) == 1
