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


# ---------------------------------------------------------------------------
# the module
# ---------------------------------------------------------------------------
def recorded(monkeypatch):
    """The module's two calls replaced by ones that note their operands' types and compute with torch."""
    from maba_v2_architecture_b200 import layers

    calls = []

    def gated(x, wg, wu):
        calls.append((x.dtype, wg.dtype, wu.dtype))
        return torch.nn.functional.silu(x @ wg.t()) * (x @ wu.t())

    def linear(x, w, scale=None, residual=None, out_dtype=None):
        calls.append((x.dtype, w.dtype))
        y = x @ w.t()
        y = y if scale is None else y * scale
        return (y if residual is None else y + residual).to(out_dtype or x.dtype)

    monkeypatch.setattr(layers, "b200_gated_ffn", gated)
    monkeypatch.setattr(layers, "b200_linear", linear)
    return calls


class Adapter(torch.nn.Module):
    def __init__(self, base):
        super().__init__()
        self.base, self.weight, self.bias = base, base.weight, None

    def forward(self, x):
        return 2 * self.base(x)


class Scaled(torch.nn.Linear):
    def forward(self, x):
        return 2 * super().forward(x)


@pytest.mark.parametrize("name", ["w_gate", "w_up", "w_down"])
@pytest.mark.parametrize("change", ["wrapper", "subclass", "own forward", "bias", "forward hook", "pre-hook", "backward hook",
                                    "backward pre-hook"])
def test_projections_that_do_more_are_refused(monkeypatch, name, change):
    """The module reads its projections' weights; what a projection's module would do beside the product
    is not passed by in silence."""
    calls = recorded(monkeypatch)
    ffn = mb.SwiGLUFFN(dim=16, intermediate_size=24)
    lin = getattr(ffn, name)
    if change == "wrapper":
        setattr(ffn, name, Adapter(lin))
    elif change == "subclass":
        setattr(ffn, name, Scaled(lin.in_features, lin.out_features, bias=False))
    elif change == "own forward":
        lin.forward = lambda x: 2 * x
    elif change == "bias":
        setattr(ffn, name, torch.nn.Linear(lin.in_features, lin.out_features))
    else:
        add = {"forward hook": lin.register_forward_hook, "pre-hook": lin.register_forward_pre_hook,
               "backward hook": lin.register_full_backward_hook, "backward pre-hook": lin.register_full_backward_pre_hook}
        handle = add[change](lambda *a: None)
    with pytest.raises(RuntimeError, match=f"{name} must be a plain nn.Linear"):
        ffn(torch.zeros(3, 16))
    assert not calls
    if "hook" in change:
        handle.remove()
        assert ffn(torch.zeros(3, 16)).shape == (3, 16)


def test_a_parametrized_weight_is_read_as_it_is_computed(monkeypatch):
    recorded(monkeypatch)
    ffn = mb.SwiGLUFFN(dim=16, intermediate_size=24)
    x = torch.ones(3, 16)
    want = ffn(x)

    class Twice(torch.nn.Module):
        def forward(self, w):
            return 2 * w

    torch.nn.utils.parametrize.register_parametrization(ffn.w_down, "weight", Twice())
    assert torch.equal(ffn(x), 2 * want)


@pytest.mark.parametrize("x_dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_autocast_reaches_the_module(monkeypatch, x_dtype):
    """float32 weights under autocast, whatever x's type: the operators get autocast's, as nn.Linear does;
    outside, and for float64, types are left alone."""
    calls = recorded(monkeypatch)
    ffn = mb.SwiGLUFFN(dim=16, intermediate_size=24)
    x, r = torch.randn(3, 16).to(x_dtype), torch.zeros(3, 16)
    bf = torch.bfloat16
    with torch.autocast("cpu", dtype=bf):
        assert ffn(x).dtype is bf and ffn(x, residual=r).dtype is torch.float32
    assert calls == [(bf, bf, bf), (bf, bf)] * 2
    calls.clear()
    if x_dtype is torch.float32:
        ffn(x)
        with torch.autocast("cpu", dtype=bf):
            ffn.double()(x.double())
        f32, f64 = torch.float32, torch.float64
        assert calls == [(f32, f32, f32), (f32, f32), (f64, f64, f64), (f64, f64)]


# ---------------------------------------------------------------------------
# refusals of the C entries (nothing is launched: the workspace is missing)
# ---------------------------------------------------------------------------
def descriptor(shape, stride=None):
    t = N.MabaTensor(1 << 20, 0, len(shape))
    run = 1
    for i in reversed(range(len(shape))):
        t.shape[i], t.stride[i] = shape[i], run if stride is None else stride[i]
        run *= shape[i]
    return ctypes.byref(t)


def test_gradient_vectors_that_overlap_themselves_are_refused():
    d = descriptor
    x, w, g, v, same = d((4, 16)), d((8, 16)), d((4, 8)), d((8,)), d((8,), (0,))
    lib = N.lib()
    run = lambda *vec: lib.maba_linear_backward(g, x, w, v, 0, v, None, None, *vec, None, 0, None)
    assert run(v, v) == N.ERR_WORKSPACE  # accepted
    assert run(same, v) == N.ERR_INVALID and b"dbias" in lib.maba_last_error()
    assert run(v, same) == N.ERR_INVALID and b"dscale" in lib.maba_last_error()
    one = d((1,), (0,))  # (a single element does not)
    assert lib.maba_linear_backward(d((4, 1)), x, d((1, 16)), one, 0, None, None, None, one, None, None, 0, None) == N.ERR_WORKSPACE


def test_negative_sizes_are_refused():
    """Also where every tensor agrees on them."""
    d, lib = descriptor, N.lib()
    assert lib.maba_linear_backward(d((-4, 8)), d((-4, 16)), d((8, 16)), None, 1, None, d((-4, 16)), None, None, None, None, 0,
                                    None) == N.ERR_INVALID
    assert lib.maba_gated_ffn_workspace_size(d((-4, 16)), d((8, 16)), d((8, 16)), d((-4, 8))) == 0
    assert b"negative size" in lib.maba_last_error()
