"""CPU tests of attention_scored: what the library and the Python call refuse before a device is touched, and the plain computation in 64 bits
that the GPU tests go by, against autograd."""
import ctypes
import os
import re

import pytest
import torch

from flash_b200 import _lib, attention_scored
from scored_reference import attention_64


def _problem(**kw):
    p = dict(B=1, H=2, Hk=2, M=64, N=64, D=64, dtype=0, causal=1, mode=0, id_heads=1, sm_scale=0.1)
    return _lib.Problem(*{**p, **kw}.values())


def _calls(prob, scores):
    lib = _lib.load()
    t = _lib.Tensor(256, (64 * 64 * 2, 64 * 64, 64, 1))
    return (lib.fa_fwd_scored(prob, scores, t, t, t, t, None, 256, None, 1, None, 0, 256, None),
            lib.fa_bwd_scored(prob, scores, t, t, t, t, None, t, 256, 256, t, t, t, None, 256, None),
            lib.fa_plan_build_scored(prob, scores, None, None, 256, 512, 256, None))


@pytest.mark.parametrize("cap", [-1.0, 1e-7, 2e6, float("nan"), float("inf")])
def test_softcaps_that_the_library_refuses(cap):
    assert _calls(_problem(), _lib.Scores(cap, None, None)) == (9, 9, 9)
    assert b"softcap" in _lib.load().fa_error_string(9)


def test_a_prefix_needs_a_causal_mask_and_scores_have_to_be_given():
    assert _calls(_problem(causal=0), _lib.Scores(1.0, None, 256)) == (9, 9, 9)
    assert _calls(_problem(), None) == (1, 1, 1)
    assert _calls(_problem(), _lib.Scores(1.0, 258, None)) == (3, 3, 3)
    assert _calls(_problem(), _lib.Scores(1.0, None, 258)) == (3, 3, 3)


def test_bad_problems_are_refused_as_elsewhere():
    s = _lib.Scores(1.0, None, None)
    assert _calls(_problem(D=48), s) == (2, 2, 2)
    assert _calls(_problem(M=128), s) == (1, 1, 1)
    prob = _problem(M=16, N=1024)
    t = _lib.Tensor(256, (64 * 64 * 2, 64 * 64, 64, 1))
    assert _lib.load().fa_fwd_scored(prob, s, t, t, t, t, None, 256, None, 2, None, 0, 256, None) == 6  # no workspace


def test_what_a_rounding_leaves_out_is_for_16_bit_calls_with_changed_scores_in_one_run():
    lib, s, t = _lib.load(), _lib.Scores(1.0, None, None), _lib.Tensor(256, (64 * 64 * 2, 64 * 64, 64, 1))
    fwd = lambda prob, scores, rest, splits=1: lib.fa_fwd_scored(prob, scores, t, t, t, t, rest, 256, None, splits, 256, 1 << 30, 256, None)  # noqa: E731
    assert fwd(_problem(dtype=2), s, 256) == 2
    assert fwd(_problem(M=16, N=1024), s, 256, 2) == 2
    assert fwd(_problem(), _lib.Scores(0.0, None, None), 256) == 2
    assert fwd(_problem(), s, 264) == 3
    assert lib.fa_bwd_scored(_problem(dtype=2), s, t, t, t, t, 256, t, 256, 256, t, t, t, None, 256, None) == 2


def test_cpu_tensors_and_bad_arguments_raise():
    q = torch.randn(1, 2, 8, 64)
    with pytest.raises(RuntimeError, match="CUDA"):
        attention_scored(q, q, q, True, softcap=5.0)
    with pytest.raises(ValueError, match="softcap"):
        attention_scored(q, q, q, True, softcap=-5.0)
    with pytest.raises(AssertionError):
        attention_scored(q, q[:, :, :4], q[:, :, :4], True, softcap=5.0)
    with pytest.raises(AssertionError):
        attention_scored(q, q[..., :32], q[..., :32], True, softcap=5.0)


@pytest.mark.parametrize("causal", [True, False])
def test_the_formulas_against_autograd(causal):
    gen = torch.Generator().manual_seed(0)
    q, do = (torch.randn(2, 4, 6, 16, generator=gen, dtype=torch.float64) for _ in range(2))
    k, v = (torch.randn(2, 2, 9, 16, generator=gen, dtype=torch.float64) for _ in range(2))
    ids = torch.tensor([-1, -1, -1, -2, -2, -2, 3, -2, -2]).expand(2, 4, 9)
    slopes, prefix = torch.tensor([0.5, 0.1, 0.0, 2.0]), torch.tensor([4, 0]) if causal else None
    a, b, c = (x.clone().requires_grad_() for x in (q, k, v))
    s = a @ b.repeat_interleave(2, 1).mT / 4
    i, j = torch.arange(6)[:, None] + 3, torch.arange(9)
    x = 2 * torch.tanh(s / 2) - slopes.double()[:, None, None] * (i - j).abs()
    keep = (ids[..., 3:, None] >= 0) | (ids[..., 3:, None] == ids[..., None, :])
    if causal:
        keep = keep & ((j <= i) | (j < prefix[:, None, None, None]))
    o = torch.softmax(x.masked_fill(~keep, -1e300), -1) @ c.repeat_interleave(2, 1)
    o.backward(do)
    got = attention_64(q, k, v, do, causal, None, ids[..., 3:], ids, 2.0, slopes, prefix)
    for name, want in (("o", o), ("dq", a.grad), ("dk", b.grad), ("dv", c.grad)):
        assert torch.allclose(got[name][0], want, rtol=1e-12, atol=1e-12), name


def test_the_forward_reads_no_prefix_before_the_kernel_before_it_is_complete():
    """Its first item's range of keys goes by the prefix, so that a call with one works that item out behind the wait. (In the sources, as the order in
    test_launch_order.py: a wrong one shows only now and then.)"""
    csrc = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "triton-flash-attention-with-flexible-masks_b200", "csrc")
    with open(os.path.join(csrc, "fwd.cu")) as f:
        code = re.sub(r"//[^\n]*", "", f.read())
    kernel = code[code.index("fwd_kernel(const"):]
    wait = kernel.index("wait_prerequisites();")
    before = kernel[kernel.index("fence_mbar_init();"): wait]
    assert re.search(r"early = mk\.mode == 0 && !\(PREFIX && mk\.prefix\);", before)
    assert re.findall(r"if \([^\n]*\bprepare\(|\bprepare\(", before) == ["if (warp == 14 && early) item = prepare("]
    assert not re.search(r"\b(front_keys|slopes|prefix\[)", before)
    assert "if ((k > 0 || !early) && j < n_items) item = prepare(j);" in kernel[wait:]


def test_what_the_library_refuses_of_a_rest_of_runs():
    lib = _lib.load()
    prob = _problem(M=16, N=1024)
    call = lambda p=prob, splits=2, work=256, size=1 << 30, rest=256, status=256: lib.fa_fwd_rest(p, splits, work, size, rest, status, None)  # noqa: E731
    assert call(_problem(D=48)) == 2 and call(_problem(M=16, N=1024, dtype=2)) == 2 and call(_problem(M=16, N=1024, mode=1)) == 2 and call(splits=9) == 2
    assert call(splits=1) == 1 and call(rest=None) == 1 and call(status=None) == 1
    assert call(work=None) == 6 and call(size=100) == 6
    assert call(work=264) == 3 and call(rest=264) == 3
