"""CPU checks of the training losses' boundary: argument refusals that need no device, and the
Python forms' checks of shapes and types, which come before any call into the library."""
import ctypes
from types import SimpleNamespace

import numpy as np
import pytest


@pytest.fixture(scope="module")
def rh():
    import rust_ppocrv6_b200 as rh

    rh.load()
    return rh


def test_null_context_is_refused_by_every_entry_point(rh):
    lib = rh.load()
    p = ctypes.c_void_p(16)  # never read: the context is looked at first
    calls = [
        lib.rh_head_cross_entropy(None, p, p, 1, 8, 0, p, p, p),
        lib.rh_head_distill(None, p, p, 1, 8, 0, p, p, 2, 1.0, p, p),
        lib.rh_head_cross_entropy_device(None, p, 0, p, 1, 0, p, p, p, p, 1 << 20, None),
        lib.rh_head_distill_device(None, p, 0, p, 1, 0, p, p, 2, 1.0, p, p, p, 1 << 20, None),
        lib.rh_head_cross_entropy_grad(None, p, 1, 8, 0, p, 4, p, p, p, p, p, p, p, p),
        lib.rh_head_distill_grad(None, p, 1, 8, 0, p, 4, p, p, p, 2, 1.0, p, p, p, p, p, p),
        lib.rh_head_cross_entropy_grad_device(None, 0, 0, p, 1, 8, 0, p, 4, p, p, p, p, p, p, p, p, p, 1 << 20, None),
        lib.rh_head_distill_grad_device(None, 0, 0, p, 1, 8, 0, p, 4, p, p, p, 2, 1.0, p, p, p, p, p, p, p, 1 << 20, None),
    ]
    assert calls == [rh.RH_ERR_INVALID_ARG] * len(calls)
    assert "context" in lib.rh_last_error().decode()
    assert lib.rh_head_score_workspace_bytes(None, p, 0, 1) == -1
    assert lib.rh_head_grad_workspace_bytes(None, 0, 0, 1, 8, 4, 0) == -1


@pytest.mark.parametrize("call", [
    lambda rh, qw, x: rh.head_cross_entropy(x, qw, np.zeros(4, np.int32)),             # one target too many
    lambda rh, qw, x: rh.head_cross_entropy(x, qw, np.zeros(3, np.float32)),           # not classes
    lambda rh, qw, x: rh.head_cross_entropy(x, qw, np.full(3, 2 ** 31)),               # beyond 32 bits
    lambda rh, qw, x: rh.head_cross_entropy(x[:, :7], qw, np.zeros(3, np.int32)),      # wrong K
    lambda rh, qw, x: rh.head_cross_entropy(x, qw, np.zeros(3, np.int32), kt=True),    # not [batch, k, T]
    lambda rh, qw, x: rh.head_distill(x, qw, np.zeros((3, 2), np.int32), np.zeros((3, 3), np.float32)),
    lambda rh, qw, x: rh.head_distill(x, qw, np.zeros(3, np.int32), np.zeros(3, np.float32)),
    lambda rh, qw, x: rh.head_cross_entropy_grad(x, np.zeros(8), np.zeros(3, np.int32)),
    lambda rh, qw, x: rh.head_cross_entropy_grad(x, np.zeros((5, 8)), np.zeros(3, np.int32), bias=np.zeros(4)),
    lambda rh, qw, x: rh.head_cross_entropy_grad(x, np.zeros((5, 8)), np.zeros(3, np.int32), row_grad=np.zeros(2)),
    lambda rh, qw, x: rh.head_cross_entropy_grad(x, np.zeros((5, 7)), np.zeros(3, np.int32)),
    lambda rh, qw, x: rh.head_distill_grad(x, np.zeros((5, 8)), np.zeros((2, 3), np.int32), np.zeros((2, 3))),
    lambda rh, qw, x: rh.head_grad_workspace_bytes(None, "fp8", 1, 8, 5),
])
def test_python_forms_refuse_wrong_shapes_and_types(rh, call):
    qw = SimpleNamespace(cols=8, rows=5, bias=None)  # a packed head's sizes are all that is looked at
    with pytest.raises(rh.RecHeadError) as e:
        call(rh, qw, np.zeros((3, 8), np.float32))
    assert e.value.code == rh.RH_ERR_INVALID_ARG


def test_every_form_is_public(rh):
    for op in ("head_cross_entropy", "head_distill"):
        for form in ("", "_device", "_grad", "_grad_device"):
            assert op + form in rh.__all__ and callable(getattr(rh, op + form))
