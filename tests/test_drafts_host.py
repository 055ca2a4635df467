"""CPU tests of the drafted trees' host side: calls that are refused before any device work."""
import ctypes as C

import pytest
import torch

from edgeexpert_b200 import _lib
from edgeexpert_b200.paged import PagedKVLayers


def test_entry_points_refuse_a_null_context():
    lib, z = _lib.lib(), C.c_void_p(0)
    kv, rules = _lib.PagedKVDesc(), _lib.LogitRulesDesc()
    bad = _lib.TF_ERR_INVALID_ARG
    assert lib.tf_draft_tree_plan(z, z, z, z, 1, 1, 1, 0, z, z, 1, z) == bad
    assert lib.tf_tree_attention(z, z, 0, C.byref(kv), z, 0, z, 1, z, z, 1, z, 1, z, 1, 1, 1, 1.0, 0, z, 0, z, z, 0, z) == bad
    assert lib.tf_tree_attention_workspace_bytes(z, C.byref(kv), 1, 1, 1, 1, 1) == 0
    assert lib.tf_logit_rules_apply(z, z, 1, z, 1, 2, 1, 1, z, 1, 1, C.byref(rules), z, z, 0, z) == bad
    assert lib.tf_draft_accept(z, z, z, z, z, z, z, 1, 1, 1, z, z, z, z, C.byref(kv), 0, 0, z, 0, z) == bad
    assert lib.tf_logit_rules_workspace_bytes(3, 262144, 2, 100, 5) >= 3 * 8 + 16 * (2 * 100 + 5 + 3)


def test_layers_describe_strides():
    k = torch.zeros(3, 5, 16, 2, 64, dtype=torch.float16)
    layers = PagedKVLayers(k, torch.zeros_like(k))
    assert layers.layers == 3 and layers.layer_stride == 5 * 16 * 2 * 64 and len(layers.layer) == 3
    assert layers.layer[2].desc.k == k[2].data_ptr() and layers.layer[0].num_pages == 5
    for bad in ((k, k[:2]), (k[0], k[0]), (k.float(), k.float()), (k, k.transpose(2, 3).contiguous().transpose(2, 3))):
        with pytest.raises(_lib.TFError):
            PagedKVLayers(*bad)


def test_tensors_elsewhere_are_refused():
    t = torch.zeros(2)
    _lib.on_device("x", -1, t, None)  # (-1: host memory)
    with pytest.raises(_lib.TFError):
        _lib.on_device("x", 0, None, t)
    _lib.int32_on_device("x", -1, t.int())
    for bad in (t, t.long(), torch.zeros(2, 2, dtype=torch.int32).t()[:1]):
        with pytest.raises(_lib.TFError):
            _lib.int32_on_device("x", -1, bad)
