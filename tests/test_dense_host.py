"""Refusals of the dense operators, without a GPU: shapes, types, devices, activations, out."""
import ctypes
import struct

import pytest
import torch

import maba_v2_architecture_b200 as mb
from maba_v2_architecture_b200 import _native as N
from maba_v2_architecture_b200 import dense

X, W = torch.zeros(4, 16), torch.zeros(8, 16)


def test_no_cpu_path():
    for call in (lambda: mb.b200_linear(X, W), lambda: mb.b200_gated_ffn(X, W, W),
                 lambda: mb.b200_linear_backward(torch.zeros(4, 8), X, W),
                 lambda: mb.b200_gated_ffn_backward(torch.zeros(4, 8), X, W, W)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


@pytest.mark.parametrize("kw,err,match", [
    (dict(activation="tanh"), ValueError, "Unknown activation"),
    (dict(bias=torch.zeros(7)), ValueError, "bias shape"),
    (dict(bias=torch.zeros(8, 1)), ValueError, "bias shape"),
    (dict(bias=torch.zeros(8, dtype=torch.float64)), TypeError, "bias must be"),
    (dict(scale=torch.zeros(16)), ValueError, "scale shape"),
    (dict(residual=torch.zeros(8)), ValueError, "residual shape"),
    (dict(residual=torch.zeros(4, 8, dtype=torch.float16)), TypeError, "residual must be"),
    (dict(out_dtype=torch.bfloat16), TypeError, "out_dtype"),
])
def test_linear_refusals(kw, err, match):
    with pytest.raises(err, match=match):
        mb.b200_linear(X, W, **kw)


def test_operand_refusals():
    with pytest.raises(TypeError, match="Unsupported dtype"):
        mb.b200_linear(X.double(), W.double())
    with pytest.raises(TypeError, match="must match"):
        mb.b200_linear(X, W.half())
    with pytest.raises(ValueError, match="weight shape"):
        mb.b200_linear(X, W[:, :15])
    with pytest.raises(ValueError, match="weight shape"):
        mb.b200_linear(X, W[0])
    with pytest.raises(ValueError, match="at least one dimension"):
        mb.b200_linear(X[0, 0], W)
    with pytest.raises(ValueError, match="no features"):
        mb.b200_linear(X, W[:0])
    with pytest.raises(ValueError, match="no features"):
        mb.b200_linear(X[:, :0], W[:, :0])
    with pytest.raises(ValueError, match="w_up shape"):
        mb.b200_gated_ffn(X, W, W[:7])
    with pytest.raises(ValueError, match="Unknown activation"):
        mb.b200_gated_ffn(X, W, W, activation="none")
    with pytest.raises(RuntimeError, match="same device"):
        mb.b200_linear(X, W.to("meta"))
    with pytest.raises(ValueError, match="grad_out shape"):
        mb.b200_linear_backward(torch.zeros(4, 7), X, W)
    with pytest.raises(TypeError, match="grad_out must be"):
        mb.b200_gated_ffn_backward(torch.zeros(4, 8), X.half(), W.half(), W.half())


def test_out_rules():
    buf = torch.zeros(64)
    x, w = buf[:32].view(4, 8), torch.zeros(8, 8)
    res = torch.zeros(40)
    for out, inputs, residual, match in [
        (buf[16:48].view(4, 8), (("x", x),), None, "shares memory with x"),
        (res[8:40].view(4, 8), (), res[:32].view(4, 8), "overlaps residual"),
        (torch.zeros(8, 4).t(), (), None, "contiguous rows"),
        (torch.zeros(1, 8).expand(4, 8), (), None, "contiguous rows"),
    ]:
        with pytest.raises(ValueError, match=match):
            dense._check_out(out, x, (4, 8), inputs, residual)
    dense._check_out(res[:32].view(4, 8), x, (4, 8), (("x", x), ("weight", w)), res[:32].view(4, 8))
    with pytest.raises(ValueError, match="out shape"):
        dense._check_out(torch.zeros(4, 7), x, (4, 8), (), None)


def test_c_entry_refusals():
    """The C entries check what they are given before anything is launched."""
    lib = N.lib()
    ptr = 1 << 20  # never read: every call below is refused on the host

    def d(shape, stride=None, dt=0):
        t = N.MabaTensor(ptr, dt, len(shape))
        run = 1
        for i in reversed(range(len(shape))):
            t.shape[i], t.stride[i] = shape[i], run if stride is None else stride[i]
            run *= shape[i]
        return ctypes.byref(t)

    def linear(x, w, bias=None, act=0, scale=None, res=None, out=None):
        return lib.maba_linear(x, w, bias, act, scale, res, out, None, 0, None)

    x, w, o = d((4, 16)), d((8, 16)), d((4, 8))
    assert linear(None, w, out=o) == N.ERR_INVALID
    assert linear(x, d((8, 15)), out=o) == N.ERR_INVALID
    assert linear(x, d((8, 16), dt=2), out=o) == N.ERR_DTYPE
    assert linear(d((4, 16), dt=3), w, out=o) == N.ERR_DTYPE
    assert linear(x, w, act=4, out=o) == N.ERR_INVALID
    assert linear(x, w, act=-1, out=o) == N.ERR_INVALID
    assert linear(x, w, bias=d((7,)), out=o) == N.ERR_INVALID
    assert linear(x, w, out=None) == N.ERR_INVALID
    assert linear(x, w, out=d((4, 8), (8, 2))) == N.ERR_INVALID
    assert linear(x, w, out=d((4, 8), (4, 1))) == N.ERR_INVALID
    assert linear(x, w, out=d((4, 8), (-8, 1))) == N.ERR_INVALID
    assert linear(d((1 << 31, 16)), w, out=d((1 << 31, 8))) == N.ERR_UNSUPPORTED
    assert lib.maba_gated_ffn(x, w, w, 0, o, None, 0, None) == N.ERR_INVALID
    assert lib.maba_gated_ffn_backward(d((4, 7)), x, w, w, 2, None, None, None, None, 0, None) == N.ERR_INVALID
    # a backward pass that needs scratch memory and has none
    rc = lib.maba_gated_ffn_backward(o, x, w, w, 2, d((4, 16)), None, None, None, 0, None)
    assert rc == N.ERR_WORKSPACE and b"workspace" in lib.maba_last_error()
    need = lib.maba_gated_ffn_backward_workspace_size(o, x, w, w, d((4, 16)), None, None)
    assert need >= 2 * 4 * 8 * 4
    assert lib.maba_linear_backward(o, x, w, None, 0, None, None, None, d((8,)), None, None, 0, None) == N.ERR_INVALID


# ---------------------------------------------------------------------------
# the module and its installation
# ---------------------------------------------------------------------------
def test_swiglu_module_parameters():
    from maba_v2_architecture_b200.config import get_101m_config
    from maba_v2_architecture_b200.engine import ModelShape, parameter_shapes

    m = mb.SwiGLUFFN(get_101m_config())
    want = {k[len("layers.0.ffn."):]: v for k, v in parameter_shapes(ModelShape.from_config(get_101m_config())).items()
            if k.startswith("layers.0.ffn.")}
    assert {k: tuple(v.shape) for k, v in m.state_dict().items()} == want
    with pytest.raises(RuntimeError, match="no CPU path"):
        m(torch.zeros(2, 640))


def test_install_patches_the_ffn_only_when_asked(monkeypatch):
    import sys
    import types

    names = ["maba_sparse", "maba_sparse.kernels", "maba_sparse.kernels.dispatcher", "maba_sparse.model"]
    mods = {n: types.ModuleType(n) for n in names}
    disp = mods["maba_sparse.kernels.dispatcher"]
    disp._KERNEL_REGISTRY = {}
    disp.register_kernel = lambda b, op: (lambda f: disp._KERNEL_REGISTRY.setdefault(b, {}).__setitem__(op, f))
    disp.clear_dispatcher_cache = lambda: None

    class SwiGLUFFN(torch.nn.Module):
        def forward(self, x):
            return x

    mods["maba_sparse.model"].SwiGLUFFN = SwiGLUFFN
    for n, m in mods.items():
        monkeypatch.setitem(sys.modules, n, m)
    monkeypatch.delenv("MABA_BACKEND", raising=False)
    monkeypatch.delenv("MABA_STRICT_BACKEND", raising=False)
    from maba_v2_architecture_b200.integration import install, uninstall

    before = SwiGLUFFN.forward
    h = install(mods["maba_sparse"], patch_layers=False)
    assert SwiGLUFFN.forward is before
    uninstall(h)
    h = install(mods["maba_sparse"], patch_layers=False, patch_ffn=True)
    assert SwiGLUFFN.forward is mb.SwiGLUFFN.forward
    uninstall(h)
    assert SwiGLUFFN.forward is before


def test_copies_of_inputs_are_held_until_the_launch(monkeypatch):
    """Inputs that no view turns into rows are copied: the copies are alive, so apart, at the launch."""
    launches = []
    monkeypatch.setattr(dense, "_call", lambda fn, size, x, head, size_args: launches.append(head))
    x, g = (torch.zeros(6, 5, 32).transpose(0, 1) for _ in range(2))
    w = torch.zeros(32, 32)
    dense._linear_backward(g, x, w, None, 0, None, (True, True, False, False))
    dense._gated_ffn_backward(g, x, w, w, 2, (True, True, True))
    for head in launches:
        places = [struct.unpack_from("Q", d)[0] for d in head if isinstance(d, bytes)]
        assert len(set(places)) == len(places) - (head[2] == head[3])  # (one weight is given twice)
