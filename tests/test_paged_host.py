"""CPU tests of the serving operators' host side: the rotary frequencies
against their formulas, and calls that are refused before any device work."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from edgeexpert_b200 import _lib
from edgeexpert_b200.paged import PagedKV, rope_frequencies

# double arithmetic on both sides: a pow and a few products apart
TOL = 1e-13


def freqs(rot, **kw):
    f, m = rope_frequencies(rot, device="cpu", **kw)
    return f.numpy(), m


@pytest.mark.parametrize("rot", [2, 36, 64, 256])
def test_plain_linear_and_base(rot):
    i = np.arange(rot // 2)
    f, m = freqs(rot, theta=10000.0)
    np.testing.assert_allclose(f, 10000.0 ** (-2 * i / rot), rtol=TOL)
    assert m == 1.0
    f, m = freqs(rot, theta=500.0, scaling="linear", factor=4.0)
    np.testing.assert_allclose(f, 500.0 ** (-2 * i / rot) / 4, rtol=TOL)
    assert m == 1.0
    if rot > 2:
        f, m = freqs(rot, scaling="base", factor=8.0)
        np.testing.assert_allclose(f, (10000.0 * 8 ** (rot / (rot - 2))) ** (-2 * i / rot), rtol=TOL)
        # the slowest pair is slowed by the whole factor, the fastest not at all
        assert f[0] == 1.0 and math.isclose(f[-1] * 8, 10000.0 ** (-2 * i[-1] / rot), rel_tol=1e-12)


def test_ramp_keeps_fast_pairs_and_slows_slow_ones():
    rot, ctx, s = 128, 8192, 16.0
    plain, _ = freqs(rot)
    f, m = freqs(rot, scaling="ramp", factor=s, original_context=ctx, low=1.0, high=32.0)
    assert math.isclose(m, 0.1 * math.log(s) + 1, rel_tol=1e-15)
    lo = max(math.floor(rot * math.log(ctx / (32 * 2 * math.pi)) / (2 * math.log(10000))), 0)
    hi = min(math.ceil(rot * math.log(ctx / (2 * math.pi)) / (2 * math.log(10000))), rot - 1)
    share = np.clip((np.arange(rot // 2) - lo) / (hi - lo), 0, 1)
    np.testing.assert_allclose(f, plain / s * share + plain * (1 - share), rtol=TOL)
    assert (f[:lo + 1] == plain[:lo + 1]).all() and np.allclose(f[hi:], plain[hi:] / s, rtol=TOL)


def test_bands_by_turns():
    rot, ctx, s, low, high = 64, 8192, 8.0, 1.0, 4.0
    plain, _ = freqs(rot)
    f, m = freqs(rot, scaling="bands", factor=s, original_context=ctx, low=low, high=high)
    turns = ctx * plain / (2 * math.pi)
    keep = np.clip((turns - low) / (high - low), 0, 1)
    np.testing.assert_allclose(f, plain / s * (1 - keep) + plain * keep, rtol=1e-12)
    assert m == 1.0 and (f[turns >= high] == plain[turns >= high]).all()


@pytest.mark.parametrize("rot,kw", [(3, {}), (0, {}), (64, dict(theta=0.0)), (64, dict(scaling="linear", factor=0.0)),
                                    (64, dict(scaling="ramp", factor=2.0)),
                                    (64, dict(scaling="bands", factor=2.0, original_context=8.0, low=4.0, high=4.0)),
                                    (2, dict(scaling="base", factor=2.0)), (64, dict(scaling="spiral")),
                                    (64, dict(theta=float("nan")))])
def test_frequencies_refused(rot, kw):
    with pytest.raises(_lib.TFError):
        rope_frequencies(rot, device="cpu", **kw)


def test_entry_points_refuse_a_null_context():
    lib = _lib.lib()
    z = C.c_void_p(0)
    kv = _lib.PagedKVDesc()
    assert lib.tf_kv_pages_resize(z, z, z, 1, z, 1, z, 1, z, 1, 0, z, z, z, z, z, z, 0, z, 0, z) == _lib.TF_ERR_INVALID_ARG
    assert lib.tf_rope_kv_write(z, z, 0, z, 0, z, 0, z, 0, C.byref(kv), z, z, z, 0, 0, 1.0, 0, z, z, 0.0, 1, 1,
                                z) == _lib.TF_ERR_INVALID_ARG
    assert lib.tf_shared_prefix_attention(z, z, 0, C.byref(kv), z, 0, z, 1, z, z, 1, 1, 1, 1, 1.0, 0, z, 0, z, z, 0,
                                          z) == _lib.TF_ERR_INVALID_ARG
    assert lib.tf_shared_prefix_attention_workspace_bytes(z, C.byref(kv), 1, 1, 1, 1, 1) == 0
    assert lib.tf_kv_pages_workspace_bytes(3) >= 3 * 8


def test_paged_kv_describes_strides():
    k = torch.zeros(5, 16, 2, 64, dtype=torch.float16)
    kv = PagedKV(k, torch.zeros_like(k))
    assert (kv.desc.page_stride, kv.desc.position_stride, kv.desc.head_stride) == (16 * 128, 128, 64)
    both = torch.zeros(5, 2, 4, 16, 64, dtype=torch.bfloat16)  # [page][K or V][head][position][dim]
    kv = PagedKV(both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2))
    assert (kv.desc.page_stride, kv.desc.position_stride, kv.desc.head_stride) == (2 * 4 * 16 * 64, 64, 16 * 64)
    assert (kv.num_pages, kv.page_size, kv.num_kv_heads, kv.head_dim, kv.desc.dtype) == (5, 16, 4, 64, 1)
    for bad in ((k.float(), k.float()), (k, k.bfloat16()), (k[..., ::2], k[..., ::2]), (k[0], k[0])):
        with pytest.raises(_lib.TFError):
            PagedKV(*bad)
