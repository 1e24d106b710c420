"""Edges of the dense operators: products of one row whose contraction is split, among others.
Values and bounds from tests/dense_oracle.py."""
import pytest
import torch

import dense_oracle as O
import maba_v2_architecture_b200 as mb
from maba_v2_architecture_b200 import _native as N
from test_gpu_dense import BF, DEV, F32, HF, gen, linear_case, no_device_error, randn  # noqa: F401

pytestmark = pytest.mark.gpu

# Products of one row (dx, dz and the projections of one row; dW of one output feature) with a split
# contraction, widths of 1 to 4 past a multiple of eight, and their neighbours
ONE = [(4096, 300, 1), (8192, 100, 1), (1, 300, 2048), (1, 100, 2048), (1, 650, 1251), (1, 4000, 100), (1, 4000, 25),
       (2, 4000, 100), (4096, 300, 2), (1, 104, 2048)]


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("m,k,n", ONE)
def test_split_sums_of_one_row(m, k, n, dt):
    for i, (act, bias, scale) in enumerate([("none", "none", "none"), ("none", "f32", "f32"), ("silu", "same", "f32")]):
        t = linear_case(m, k, n, dt, bias, scale, "none", seed=i, grad=dt)
        want = O.linear_backward(t["g"], t["x"], t["w"], t["bias"], act, t["scale"])
        for name, v in zip(("dx", "dw", "dbias", "dscale"),
                           mb.b200_linear_backward(t["g"], t["x"], t["w"], t["bias"], act, t["scale"])):
            if v is not None:
                O.assert_within(v, want[name], f"{name} {(m, k, n)} {act}")
    g = gen(6)
    x, wg, wu = randn(g, m, k, dt=dt), randn(g, n, k, dt=dt, std=k ** -0.5), randn(g, n, k, dt=dt, std=k ** -0.5)
    d = randn(g, m, n, dt=dt, std=0.3)
    want = O.gated_backward(d, x, wg, wu, "silu")
    for name, v in zip(("dx", "dw_gate", "dw_up"), mb.b200_gated_ffn_backward(d, x, wg, wu)):
        O.assert_within(v, want[name], f"{name} {(m, k, n)}")


@pytest.mark.parametrize("m,k,n", ONE)
def test_nothing_is_written_behind_the_workspace(m, k, n):
    """The C entries with a workspace of exactly the size they ask for, in a larger buffer whose other
    bytes keep their values."""
    t = linear_case(m, k, n, BF, "none", "none", "none", seed=3, grad=BF)
    wu = randn(gen(4), n, k, dt=BF, std=k ** -0.5)
    dx, dw, dwu = torch.empty_like(t["x"]), torch.empty_like(t["w"]), torch.empty_like(wu)
    pg, px, pw, pwu, pdx, pdw, pdwu = map(N.pack_matrix, (t["g"], t["x"], t["w"], wu, dx, dw, dwu))
    lib, stream = N.lib(), torch.cuda.current_stream().cuda_stream
    linear = (pg, px, pw, None, 2, None, pdx, pdw, None, None)
    ffn = (pg, px, pw, pwu, 2, pdx, pdw, pdwu)
    for fn, args, need in ((lib.maba_linear_backward, linear, lib.maba_linear_backward_workspace_size(*linear)),
                           (lib.maba_gated_ffn_backward, ffn, lib.maba_gated_ffn_backward_workspace_size(*ffn[:4], *ffn[5:]))):
        buf = torch.full((need + 8192,), 0x5a, dtype=torch.uint8, device=DEV)
        assert need and buf.data_ptr() % 256 == 0
        N.check(fn(*args, buf.data_ptr(), need, stream), fn.__name__)
        torch.cuda.synchronize()
        assert bool((buf[need:] == 0x5a).all())


@pytest.mark.parametrize("dt", [BF, HF, F32])
@pytest.mark.parametrize("m,k", [(70, 40), (200, 40), (1001, 700), (70, 4000)])
def test_an_infinite_scale_stays_in_its_column(m, k, dt):
    """dz = grad * scale is +inf in every row of that column, and so is its sum, however many rows the
    last block of 32 lacks.  The other columns are what they are without it."""
    n, col = 72, 5
    t = linear_case(m, k, n, dt, "f32", "f32", "none", seed=7, grad=dt)
    t["g"] = t["g"].abs() + 0.25
    clean = mb.b200_linear_backward(t["g"], t["x"], t["w"], t["bias"], "none", t["scale"], needs=(False, False, True, True))
    scale = t["scale"].clone()
    scale[col] = float("inf")
    db, ds = mb.b200_linear_backward(t["g"], t["x"], t["w"], t["bias"], "none", scale, needs=(False, False, True, True))[2:]
    assert float(db[col]) == float("inf")
    db[col] = clean[2][col]
    assert torch.equal(db, clean[2]) and torch.equal(ds, clean[3])


@pytest.mark.parametrize("dt", [BF, F32])
def test_column_sums_of_many_rows(dt):
    """More blocks of 128 rows than a grid's second dimension holds (65,535).  The gradient's elements
    are 0 and 1, so every partial sum is a whole number below 2^24 and the sums are exact."""
    m, k, n = 8_400_000, 8, 8
    rows = torch.arange(m, device=DEV)
    g = torch.stack([rows % 3 == c % 3 if c < 6 else rows >= 65535 * 128 + 40 * (c - 7) for c in range(n)], 1).to(dt)
    x, w, b = randn(gen(1), m, k, dt=dt), randn(gen(2), n, k, dt=dt), torch.zeros(n, device=DEV)
    dx, dw, db, _ = mb.b200_linear_backward(g, x, w, b)
    assert torch.equal(db, g.sum(0, dtype=torch.float64).float())
    want = O.linear_backward(g[-300:], x[-300:], w, b)
    O.assert_within(dx[-300:], want["dx"], "dx")
    assert dw.shape == w.shape and bool(dw.isfinite().all())


def test_a_dual_gradient_is_refused_in_the_backward_pass():
    x, w = randn(gen(1), 70, 40, dt=F32), randn(gen(2), 24, 40, dt=F32).requires_grad_(True)
    fw = torch.autograd.forward_ad
    for y in (mb.b200_linear(x, w), mb.b200_gated_ffn(x, w, w)):
        with fw.dual_level():
            g = fw.make_dual(torch.ones_like(y), torch.ones_like(y))
            with pytest.raises(RuntimeError):
                torch.autograd.grad(y, w, g)


@pytest.mark.parametrize("op", ["linear", "gated_ffn"])
def test_out_counts_as_modified(op):
    """A tensor that another operation saved for its backward pass and out= then overwrote is noticed."""
    x, w = randn(gen(1), 70, 40, dt=BF), randn(gen(2), 24, 40, dt=BF)
    stream, p = randn(gen(3), 70, 24, dt=BF), torch.ones(24, dtype=BF, device=DEV, requires_grad=True)
    y = p * stream
    version = stream._version
    if op == "linear":
        mb.b200_linear(x, w, residual=stream, out=stream)
    else:
        mb.b200_gated_ffn(x, w, w, out=stream)
    assert stream._version > version
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    with torch.inference_mode():  # (tensors without a version)
        out = torch.empty(70, 24, dtype=BF, device=DEV)
        O.assert_within(mb.b200_linear(x, w, out=out), O.linear(x, w), "inference mode")


@pytest.mark.parametrize("x_dtype", [F32, BF])
def test_module_under_autocast(x_dtype):
    """A training step in mixed precision: float32 weights, their gradients float32; values and gradients
    are those of the calls on operands cast to autocast's type."""
    torch.manual_seed(4)
    ffn = mb.SwiGLUFFN(dim=96, intermediate_size=200).to(DEV)
    x = randn(gen(1), 70, 96, dt=x_dtype).requires_grad_(True)
    d = randn(gen(2), 70, 96, dt=BF)
    with torch.autocast("cuda", dtype=BF):
        y = ffn(x)
    assert y.dtype is BF
    y.backward(d)
    xb, wg, wu, wd = (t.detach().to(BF) for t in (x, ffn.w_gate.weight, ffn.w_up.weight, ffn.w_down.weight))
    a = mb.b200_gated_ffn(xb, wg, wu)
    assert torch.equal(y, mb.b200_linear(a, wd))
    da, dwd, _, _ = mb.b200_linear_backward(d, a, wd)
    dx, dwg, dwu = mb.b200_gated_ffn_backward(da, xb, wg, wu)
    for p, want in ((ffn.w_down.weight, dwd), (ffn.w_gate.weight, dwg), (ffn.w_up.weight, dwu), (x, dx)):
        assert p.grad.dtype is p.dtype and torch.equal(p.grad, want.to(p.dtype))


@pytest.mark.parametrize("m,k", [(4, 300), (40, 300), (300, 300), (70, 4000)])
def test_silu_far_below_zero(m, k):
    """z in [-60, -5], exact (one nonzero product per sum), float32: silu and its slope keep their relative
    accuracy.  In units of 2^-23: exp 2, 1 + exp 0.5, the quotient 0.5: 3 for silu, and 1 more for the
    product with the up projection's value.  The slope s (1 + z (1 - s)): s 3, z (1 - s) 1, which the sum
    with 1 stretches by at most 5/4 and rounds by 0.5, the product 0.5: 5.25."""
    n = 240
    z = -torch.randint(20, 241, (m, n), generator=gen(1), device=DEV) / 4.0
    x, w = torch.zeros(m, k, device=DEV), torch.eye(n, k, device=DEV)
    x[:, :n] = z
    zd = z.double()
    s = torch.sigmoid(zd)
    unit = 2.0 ** -23
    off = lambda got, want: float(((got.double() - want) / want).abs().max()) / unit
    assert off(mb.b200_linear(x, w, activation="silu"), zd * s) <= 3
    assert off(mb.b200_gated_ffn(x, w, w), zd * s * zd) <= 4
    # w's columns 0..239 are a unit matrix, so dx there is dz, or dg and du added: grad z s' + grad silu
    one = torch.ones(m, n, device=DEV)
    slope = s * (1 + zd * (1 - s))
    assert off(mb.b200_linear_backward(one, x, w, None, "silu")[0][:, :n], slope) <= 5.25
    dx = mb.b200_gated_ffn_backward(one, x, w, 2 * w)[0][:, :n]  # up: 2 z
    assert off(dx, 2 * zd * slope + 2 * zd * s) <= 8


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("m", [40, 300])
def test_silu_far_below_zero_from_16_bit_operands(m, dt):
    """The same with 16-bit operands and a float32 result.  On the tensor cores' path, in units of 2^-23: the
    exponential's argument is rounded twice, |z|; the SFU's exponential 2, the sum 0.5, the SFU's
    reciprocal 1, the product 0.5."""
    k = n = 240
    z = -torch.randint(20, 241, (m, n), generator=gen(1), device=DEV) / 4.0
    zd = z.double()
    got = mb.b200_linear(z.to(dt), torch.eye(n, k, dtype=dt, device=DEV), activation="silu", out_dtype=F32).double()
    want = zd * torch.sigmoid(zd)
    assert bool(((got - want).abs() <= (4 + zd.abs()) * 2.0 ** -23 * want.abs()).all())
