"""Edges of the dense operators that need no GPU: the layout of split sums, refusals."""
import ctypes

import pytest
import torch

import maba_v2_architecture_b200 as mb
from maba_v2_architecture_b200 import _native as N
from maba_v2_architecture_b200 import dense


@pytest.mark.parametrize("splits,pairs", [(2, 1), (16, 1), (10, 2)])
@pytest.mark.parametrize("rows", [1, 2, 33])
def test_split_sums_stay_in_their_buffer(rows, splits, pairs):
    """A split's sums start where the one before ends, rows of ``cols`` up to a multiple of four: the
    last element stored ends a row's padding before the end of what was reserved, whatever the size."""
    reserved, reached = ctypes.c_int64(), ctypes.c_int64()
    for cols in [*range(1, 41), 100, 650, 1003, 1251, 2048]:
        rc = N.lib().maba_selftest_split_layout(rows, cols, splits, pairs, ctypes.byref(reserved), ctypes.byref(reached))
        assert rc == N.OK
        padded = (cols + 3) // 4 * 4
        assert reserved.value == 4 * splits * pairs * rows * padded
        assert reached.value == reserved.value - 4 * (padded - cols), cols


def test_split_layout_refusals():
    v = ctypes.c_int64()
    for bad in ((0, 1, 1, 1), (1, 0, 1, 1), (1, 1, 0, 1), (1, 1, 1, 0)):
        assert N.lib().maba_selftest_split_layout(*bad, ctypes.byref(v), ctypes.byref(v)) == N.ERR_INVALID
    assert N.lib().maba_selftest_split_layout(1, 1, 1, 1, None, ctypes.byref(v)) == N.ERR_INVALID


# ---------------------------------------------------------------------------
# forward-mode derivatives
# ---------------------------------------------------------------------------
def test_dual_tensors_are_refused():
    """A tangent is not dropped in silence, whichever input carries it."""
    fw = torch.autograd.forward_ad
    t = {"x": torch.zeros(4, 16), "w": torch.zeros(8, 16), "wu": torch.zeros(8, 16), "bias": torch.zeros(8),
         "scale": torch.zeros(8), "residual": torch.zeros(4, 8), "g": torch.zeros(4, 8)}
    calls = {
        ("x", "w", "bias", "scale", "residual"): lambda a: mb.b200_linear(a["x"], a["w"], a["bias"], "silu", a["scale"],
                                                                          a["residual"]),
        ("x", "w", "bias", "scale", "g"): lambda a: mb.b200_linear_backward(a["g"], a["x"], a["w"], a["bias"], "silu",
                                                                            a["scale"]),
        ("x", "w", "wu"): lambda a: mb.b200_gated_ffn(a["x"], a["w"], a["wu"]),
        ("x", "w", "wu", "g"): lambda a: mb.b200_gated_ffn_backward(a["g"], a["x"], a["w"], a["wu"]),
    }
    with fw.dual_level():
        for names, call in calls.items():
            for name in names:
                for grad in (False, True):
                    dual = fw.make_dual(t[name].clone().requires_grad_(grad), torch.ones_like(t[name]))
                    with pytest.raises(NotImplementedError, match="forward-mode"):
                        call({**t, name: dual})
            with pytest.raises(RuntimeError, match="no CPU path"):  # a level without duals changes nothing
                call(t)


def test_out_counts_as_modified(monkeypatch):
    """With the launch left out: a write through out= raises the version that autograd checks."""
    monkeypatch.setattr(dense.N, "require_cuda", lambda *a, **k: None)
    monkeypatch.setattr(dense, "_linear", lambda *a: a[6])
    monkeypatch.setattr(dense, "_gated_ffn", lambda *a: a[4])
    x, w, out = torch.zeros(4, 16), torch.zeros(8, 16), torch.zeros(4, 8)
    for call in (lambda: mb.b200_linear(x, w, out=out), lambda: mb.b200_linear(x, w, residual=out, out=out),
                 lambda: mb.b200_gated_ffn(x, w, w, out=out)):
        y = torch.ones(8, requires_grad=True) * out
        assert call() is out
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()
