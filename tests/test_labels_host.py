"""The label operators' entry points without a GPU: what they refuse before they touch one."""

from __future__ import annotations

import ctypes

import pytest

import splat_b200 as sb
from splat_b200 import _lib


def test_null_handles_are_refused():
    lib = _lib.load()
    out = ctypes.c_void_p()
    assert lib.sp_embedding_create(None, 5, 8, 0, 4, ctypes.byref(out)) == _lib.SP_ERR_INVALID
    assert lib.sp_label_head_create(None, 5, 8, 0, 4, 1, ctypes.byref(out)) == _lib.SP_ERR_INVALID
    assert lib.sp_embedding_lookup(None, None, 8, None, 0, 1, 1.0, None, 8) == _lib.SP_ERR_INVALID
    assert lib.sp_embedding_gradient(None, None, 8, None, 0, 1, 1.0, None, 8) == _lib.SP_ERR_INVALID
    assert lib.sp_embedding_check(None) == _lib.SP_ERR_INVALID
    assert lib.sp_label_head_loss(None, None, 8, None, 8, None, 0, 1, 1.0, None, None, None) == _lib.SP_ERR_INVALID
    assert lib.sp_label_head_gradient(None, None, 8, None, 8, None, 0, 1, 1.0, None, None, None, 8, None,
                                      8) == _lib.SP_ERR_INVALID
    assert lib.sp_label_head_predict(None, None, 8, None, 8, 1, 1.0, None, None) == _lib.SP_ERR_INVALID
    assert lib.sp_label_head_check(None) == _lib.SP_ERR_INVALID
    lib.sp_embedding_destroy(None)
    lib.sp_label_head_destroy(None)


def test_the_public_names():
    for name in ("Embedding", "LabelHead", "LabelLoss"):
        assert hasattr(sb, name)


def test_other_element_types_are_refused_before_a_handle_is_made():
    import torch

    class NoContext:
        lib = None

    for handle in (lambda: sb.Embedding(NoContext(), 5, 8, torch.float16, 4),
                   lambda: sb.LabelHead(NoContext(), 5, 8, torch.int8, 4)):
        with pytest.raises(ValueError):
            handle()
