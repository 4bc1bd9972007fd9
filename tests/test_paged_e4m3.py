"""What a paged cache of 8 bits refuses, without a GPU."""
import ctypes

import pytest
import torch

from flash_b200 import _lib
from test_paged import _cache

E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
TWO = ctypes.c_int64 * 2


def _more(k=256, v=256, strides=(64, 32)):
    return _lib.PagedMore(_lib.Window(), None, k, v, TWO(*strides), TWO(*strides))


def _codes(more, **kw):
    c, lib = _cache(**{**dict(k_stride=(16 * 2 * 64, 2 * 64, 64), v_stride=(16 * 2 * 64, 2 * 64, 64)), **kw}), _lib.load()
    rows, heads = _lib.Rows(256, (128, 64)), _lib.Rows(256, (256, 64))
    return (lib.fa_paged_append_more(c, more, 2, None, rows, rows, 256, None),
            lib.fa_paged_fwd_more(c, more, 2, 4, None, 0.1, None, heads, heads, 1, 256, 1 << 30, 256, None))


@pytest.mark.parametrize("more,kw,code", [
    (dict(k=None), {}, 1), (dict(v=None), {}, 1), (dict(k=264), {}, 3), (dict(v=260), {}, 3), (dict(strides=(40, 32)), {}, 3), (dict(strides=(64, 8)), {}, 3),
    (dict(strides=(0, 32)), {}, 3), (dict(strides=(64, -32)), {}, 3), ({}, dict(page_size=8, table_pages=4), 10), ({}, dict(k_stride=(2056, 128, 64)), 3),
    ({}, dict(v_stride=(2048, 128, 72)), 3),
])
def test_c_entries_refuse(more, kw, code):
    assert _codes(_more(**more), **kw) == (code, code)


def _python(**kw):
    from flash_b200.paged import _checked
    a = dict(rows=torch.zeros(2, 2, 64, dtype=torch.bfloat16), k_pages=torch.zeros(4, 16, 2, 64).to(E4M3), v_pages=torch.zeros(4, 16, 2, 64).to(E4M3),
             k_scales=torch.zeros(4, 2, 16, dtype=torch.uint8).view(E8M0), v_scales=torch.zeros(4, 2, 16, dtype=torch.uint8).view(E8M0))
    a.update(kw)
    ints = torch.zeros(2, 2, dtype=torch.int32)

    class OnGpu(torch.Tensor):  # (the checks come in front of anything that needs a GPU)
        is_cuda = True

    return _checked(a["rows"].as_subclass(OnGpu), "k", a["k_pages"], a["v_pages"], ints, ints[0], None, a["k_scales"], a["v_scales"])


@pytest.mark.parametrize("kw,match", [
    (dict(k_pages=torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16)), "with scales is float8_e4m3fn"), (dict(k_scales=None), "go together"),
    (dict(v_scales=None), "go together"), (dict(k_scales=torch.zeros(4, 2, 16)), "float8_e8m0fnu"),
    (dict(v_scales=torch.zeros(4, 16, 2, dtype=torch.uint8).view(E8M0)), "shape"),
    (dict(k_scales=torch.zeros(4, 2, 24, dtype=torch.uint8).view(E8M0)[:, :, :16]), "multiples of 16"),
    (dict(k_scales=None, v_scales=None), "all bf16 or all fp16"),
    (dict(rows=torch.zeros(2, 2, 64)), "all bf16 or all fp16"),
    (dict(k_pages=torch.zeros(4, 8, 2, 64).to(E4M3), v_pages=torch.zeros(4, 8, 2, 64).to(E4M3), k_scales=torch.zeros(4, 2, 8, dtype=torch.uint8).view(E8M0),
          v_scales=torch.zeros(4, 2, 8, dtype=torch.uint8).view(E8M0)), "16 at least"),
    (dict(k_pages=torch.zeros(4, 16, 2, 72).to(E4M3)[..., :64]), "multiples of 16"),
])
def test_python_refuses(kw, match):
    with pytest.raises(ValueError, match=match):
        _python(**kw)


def test_what_is_taken():
    cache, more, starts, _ = _python()
    assert more.k_scales and list(more.k_scale_stride) == [32, 16] and starts is None and cache.page_size == 16
