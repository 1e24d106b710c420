"""b200_linear and b200_gated_ffn, forward and backward, against their definitions in 64 bits
(tests/dense_oracle.py: every element within a bound that is added up from the roundings)."""
import pytest
import torch

import dense_oracle as O
import maba_v2_architecture_b200 as mb
from maba_v2_architecture_b200 import _native as N

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def no_device_error():
    yield
    torch.cuda.synchronize()
    assert N.device_error() == 0, "a bounded wait ran out"


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(g, *shape, dt=F32, std=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * std).to(dt)


def linear_case(m, k, n, dt, bias, scale, residual, seed=0, grad=None):
    g = gen(seed)
    vec = {"none": None, "same": dt, "f32": F32}
    t = {"x": randn(g, m, k, dt=dt), "w": randn(g, n, k, dt=dt, std=k ** -0.5),
         "bias": None if bias == "none" else randn(g, n, dt=vec[bias], std=0.2),
         "scale": None if scale == "none" else torch.sigmoid(randn(g, n)).to(vec[scale]),
         "residual": None if residual == "none" else randn(g, m, n, dt=vec[residual])}
    if grad is not None:
        t["g"] = randn(g, m, n, dt=grad, std=0.3)
    return t


SHAPES = [(1, 1, 1), (1, 64, 64), (1, 1248, 640), (3, 7, 5), (8, 640, 1544), (16, 33, 100), (17, 640, 1544), (33, 72, 24),
          (64, 1248, 640), (65, 130, 72), (128, 64, 128), (129, 641, 257), (300, 640, 1003), (513, 96, 2000),
          (1000, 2048, 136)]
LARGE = [(2000, 264, 2056), (5003, 328, 520), (9001, 72, 250)]  # several tiles of a CTA pair per SM, ragged edges
EPILOGUES = [("none", "none", "none", "none", None), ("silu", "f32", "none", "none", None),
             ("gelu", "same", "f32", "same", None), ("relu", "none", "same", "f32", F32), ("none", "none", "f32", "f32", F32)]


LONG = [(100, 4000, 40), (24, 3776, 120), (257, 1300, 33)]  # few tiles, a long contraction: split sums


@pytest.mark.parametrize("dt", [BF, HF, F32])
@pytest.mark.parametrize("m,k,n", SHAPES + LARGE + LONG)
def test_linear(m, k, n, dt):
    for i, (act, bias, scale, residual, out_dtype) in enumerate(EPILOGUES):
        t = linear_case(m, k, n, dt, bias, scale, residual, seed=i)
        y = mb.b200_linear(t["x"], t["w"], t["bias"], act, t["scale"], t["residual"], out_dtype=out_dtype)
        assert y.dtype == (out_dtype or dt)
        O.assert_within(y, O.linear(t["x"], t["w"], t["bias"], act, t["scale"], t["residual"], out_dtype),
                        f"{(m, k, n)} {EPILOGUES[i]}")


@pytest.mark.parametrize("dt", [BF, HF, F32])
@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (1, 64, 64), (3, 7, 5), (40, 136, 72), (65, 130, 72), (129, 641, 257),
                                   (300, 96, 1003), (2100, 200, 136)] + LARGE + LONG)
def test_linear_backward(m, k, n, dt):
    for i, (act, bias, scale, _, out_dtype) in enumerate(EPILOGUES + [("none", "f32", "none", "none", F32)]):
        t = linear_case(m, k, n, dt, bias, scale, "none", seed=i, grad=out_dtype or dt)
        got = mb.b200_linear_backward(t["g"], t["x"], t["w"], t["bias"], act, t["scale"])
        want = O.linear_backward(t["g"], t["x"], t["w"], t["bias"], act, t["scale"])
        for name, v in zip(("dx", "dw", "dbias", "dscale"), got):
            assert (v is None) == (name not in want), name
            if v is not None:
                O.assert_within(v, want[name], f"{name} {(m, k, n)} {act}")


@pytest.mark.parametrize("dt", [BF, HF, F32])
@pytest.mark.parametrize("m,k,n", SHAPES + LARGE + LONG)
def test_gated_ffn(m, k, n, dt):
    g = gen(5)
    x, wg, wu = randn(g, m, k, dt=dt), randn(g, n, k, dt=dt, std=k ** -0.5), randn(g, n, k, dt=dt, std=k ** -0.5)
    for act in ("silu", "gelu", "relu"):
        O.assert_within(mb.b200_gated_ffn(x, wg, wu, act), O.gated(x, wg, wu, act), f"{(m, k, n)} {act}")


@pytest.mark.parametrize("dt", [BF, HF, F32])
@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (1, 64, 64), (3, 7, 5), (40, 136, 72), (65, 130, 72), (129, 641, 257),
                                   (300, 96, 1003), (2100, 200, 136)] + LARGE + LONG)
def test_gated_ffn_backward(m, k, n, dt):
    g = gen(6)
    x, wg, wu = randn(g, m, k, dt=dt), randn(g, n, k, dt=dt, std=k ** -0.5), randn(g, n, k, dt=dt, std=k ** -0.5)
    d = randn(g, m, n, dt=dt, std=0.3)
    for act in ("silu", "gelu", "relu"):
        got = mb.b200_gated_ffn_backward(d, x, wg, wu, act)
        want = O.gated_backward(d, x, wg, wu, act)
        for name, v in zip(("dx", "dw_gate", "dw_up"), got):
            O.assert_within(v, want[name], f"{name} {(m, k, n)} {act}")


# ---------------------------------------------------------------------------
# layouts
# ---------------------------------------------------------------------------
def layouts(t):
    """The values of the matrix t in other places: a column slice (aligned, unaligned), transposed
    storage, every other row, every other column."""
    r, c = t.shape
    big = torch.zeros(2 * r + 1, 2 * c + 16, dtype=t.dtype, device=t.device)
    for view in (big[:r, 8:8 + c], big[1:r + 1, 3:3 + c], big[:2 * r:2, :c], big[:r, :2 * c:2]):
        view.copy_(t)
        yield view
    yield t.t().contiguous().t()


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("m", [2, 100, 300])
def test_strides(dt, m):
    k, n = 136, 72
    t = linear_case(m, k, n, dt, "same", "f32", "same", seed=3, grad=dt)
    fwd = O.linear(t["x"], t["w"], t["bias"], "silu", t["scale"], t["residual"])
    bwd = O.linear_backward(t["g"], t["x"], t["w"], t["bias"], "silu", t["scale"])
    glu = O.gated(t["x"], t["w"], t["w"], "gelu")
    glub = O.gated_backward(t["g"], t["x"], t["w"], t["w"], "gelu")
    for name in ("x", "w", "residual", "g"):
        for v in layouts(t[name]):
            a = {**t, name: v}
            what = f"{name} strides {v.stride()} offset {v.storage_offset()}"
            O.assert_within(mb.b200_linear(a["x"], a["w"], a["bias"], "silu", a["scale"], a["residual"]), fwd, what)
            for key, got in zip(("dx", "dw", "dbias", "dscale"),
                                mb.b200_linear_backward(a["g"], a["x"], a["w"], a["bias"], "silu", a["scale"])):
                O.assert_within(got, bwd[key], key + " " + what)
            O.assert_within(mb.b200_gated_ffn(a["x"], a["w"], t["w"], "gelu"), glu, what)
            O.assert_within(mb.b200_gated_ffn(a["x"], t["w"], a["w"], "gelu"), glu, what)
            for key, got in zip(("dx", "dw_gate", "dw_up"),
                                mb.b200_gated_ffn_backward(a["g"], a["x"], a["w"], t["w"], "gelu")):
                O.assert_within(got, glub[key], key + " " + what)


@pytest.mark.parametrize("dt", [BF, F32])
def test_vectors_and_broadcast_inputs(dt):
    """Strided and stride-0 vectors, a broadcast residual, the gradient of a sum (all strides 0)."""
    m, k, n = 150, 72, 40
    t = linear_case(m, k, n, dt, "f32", "f32", "none", seed=8)
    bias2 = torch.stack([t["bias"], t["bias"]], 1)[:, 0]
    scale0 = torch.full((1,), 0.75, device=DEV).expand(n)
    res = randn(gen(2), 1, n, dt=dt).expand(m, n)
    O.assert_within(mb.b200_linear(t["x"], t["w"], bias2, "gelu", scale0, res),
                    O.linear(t["x"], t["w"], t["bias"], "gelu", scale0, res), "broadcast")
    one = torch.ones((), dtype=dt, device=DEV).expand(m, n)
    want = O.linear_backward(one, t["x"], t["w"], bias2, "gelu", scale0)
    for name, got in zip(("dx", "dw", "dbias", "dscale"),
                         mb.b200_linear_backward(one, t["x"], t["w"], bias2, "gelu", scale0)):
        O.assert_within(got, want[name], name)


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("m", [5, 200])
def test_out_and_in_place_residual(dt, m):
    k, n = 200, 96
    t = linear_case(m, k, n, dt, "none", "f32", "f32", seed=4)
    want = O.linear(t["x"], t["w"], None, "none", t["scale"], t["residual"], F32)
    stream = t["residual"].clone()
    got = mb.b200_linear(t["x"], t["w"], scale=t["scale"], residual=stream, out=stream)
    assert got is stream
    O.assert_within(stream, want, "in place")
    # rows of a wider buffer, and what lies beside them
    for lead in (0, 1, 3):
        wide = torch.full((m + 2, n + 13), 7.0, dtype=dt, device=DEV)
        view = wide[1:m + 1, lead:lead + n]
        mb.b200_linear(t["x"], t["w"], out=view)
        O.assert_within(view, O.linear(t["x"], t["w"]), "out slice")
        view2 = wide[1:m + 1, lead:lead + n]
        mb.b200_gated_ffn(t["x"], t["w"], t["w"], out=view2)
        O.assert_within(view2, O.gated(t["x"], t["w"], t["w"], "silu"), "out slice")
        wide[1:m + 1, lead:lead + n] = 7.0
        assert bool((wide == 7.0).all()), "memory around out was written"


def test_leading_dimensions_and_empty():
    x = randn(gen(0), 2, 3, 40, dt=BF)
    w = randn(gen(1), 24, 40, dt=BF)
    y = mb.b200_linear(x, w)
    assert y.shape == (2, 3, 24)
    O.assert_within(y.view(6, 24), O.linear(x.view(6, 40), w))
    assert mb.b200_linear(x[0, 0], w).shape == (24,)
    O.assert_within(mb.b200_linear(x[0, 0], w)[None], O.linear(x[0, :1], w))
    O.assert_within(mb.b200_gated_ffn(x.transpose(0, 1), w, w)[2, 1][None], O.gated(x[1, 2][None], w, w, "silu"))
    e = x[:0]
    assert mb.b200_linear(e, w).shape == (0, 3, 24) and mb.b200_gated_ffn(e, w, w).shape == (0, 3, 24)
    b = torch.ones(24, device=DEV)
    dx, dw, db, ds = mb.b200_linear_backward(torch.empty(0, 3, 24, dtype=BF, device=DEV), e, w, b, scale=b)
    assert dx.shape == e.shape and not dw.any() and not db.any() and not ds.any()
    dx, dg, du = mb.b200_gated_ffn_backward(torch.empty(0, 3, 24, dtype=BF, device=DEV), e, w, w)
    assert dx.shape == e.shape and not dg.any() and not du.any()


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("m", [5, 70, 200])
def test_rows_do_not_mix(dt, m):
    """NaN and infinity in one row of x stay in that row; the others keep their bits."""
    k, n = 200, 72
    t = linear_case(m, k, n, dt, "f32", "none", "none", seed=9)
    clean = mb.b200_linear(t["x"], t["w"], t["bias"], "silu")
    clean2 = mb.b200_gated_ffn(t["x"], t["w"], t["w"])
    bad = t["x"].clone()
    bad[1, 7], bad[3, 11] = float("nan"), float("inf")
    y, y2 = mb.b200_linear(bad, t["w"], t["bias"], "silu"), mb.b200_gated_ffn(bad, t["w"], t["w"])
    keep = torch.tensor([r not in (1, 3) for r in range(m)], device=DEV)
    assert torch.equal(y[keep], clean[keep]) and torch.equal(y2[keep], clean2[keep])
    assert bool(y[1].isnan().all()) and not bool(y[3].isfinite().any())


# ---------------------------------------------------------------------------
# gradients: needs, differences, autograd
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dt", [BF, F32])
def test_inputs_without_a_view_as_rows(dt):
    """Leading dimensions that only a copy makes rows of, for two inputs of the same size at once."""
    x, g = (randn(gen(i), 60, 50, 128, dt=dt).transpose(0, 1) for i in (5, 6))
    w, wu = (randn(gen(i), 128, 128, dt=dt, std=0.1) for i in (7, 8))
    r = randn(gen(9), 60, 50, 128, dt=dt).transpose(0, 1)
    xr, gr, rr = (t.reshape(-1, 128).clone() for t in (x, g, r))
    same = lambda a, b: torch.equal(a.reshape(-1, a.shape[-1]), b)
    assert same(mb.b200_linear(x, w, residual=r), mb.b200_linear(xr, w, residual=rr))
    assert same(mb.b200_gated_ffn(x, w, wu), mb.b200_gated_ffn(xr, w, wu))
    for got, want in ((mb.b200_linear_backward(g, x, w), mb.b200_linear_backward(gr, xr, w)),
                      (mb.b200_gated_ffn_backward(g, x, w, wu), mb.b200_gated_ffn_backward(gr, xr, w, wu))):
        for a, b in zip(got, want):
            assert (a is None and b is None) or same(a, b)


def test_needs_select_the_outputs():
    t = linear_case(70, 40, 24, BF, "f32", "f32", "none", seed=2, grad=BF)
    full = mb.b200_linear_backward(t["g"], t["x"], t["w"], t["bias"], "silu", t["scale"])
    for bits in range(16):
        needs = tuple(bool(bits >> i & 1) for i in range(4))
        got = mb.b200_linear_backward(t["g"], t["x"], t["w"], t["bias"], "silu", t["scale"], needs=needs)
        for n, a, b in zip(needs, got, full):
            assert (a is not None) == n and (a is None or torch.equal(a, b))
    w2 = randn(gen(3), 24, 40, dt=BF)
    full = mb.b200_gated_ffn_backward(t["g"], t["x"], t["w"], w2)
    want = O.gated_backward(t["g"], t["x"], t["w"], w2, "silu")
    for bits in range(8):
        needs = tuple(bool(bits >> i & 1) for i in range(3))
        got = mb.b200_gated_ffn_backward(t["g"], t["x"], t["w"], w2, needs=needs)
        for name, n, a in zip(("dx", "dw_gate", "dw_up"), needs, got):
            assert (a is not None) == n
            if n:
                O.assert_within(a, want[name], name)


def test_gradients_against_differences():
    """d/dh sum(g * f(x + h d)) at 0 by central differences of the float32 forward pass.  With
    |f| <= ~5 summed over 50 x 24 elements in float64, each off by ~1e-6: noise 1e-6 * 0.3 *
    sqrt(1200) / (2 h) = 5e-4 at h = 1e-2, curvature h^2 f''' / 6 of the order 1e-4 of a sum of
    order 10: 5e-3 of the largest directional derivative."""
    g = gen(11)
    t = linear_case(50, 40, 24, F32, "f32", "f32", "none", seed=12, grad=F32)
    wu = randn(g, 24, 40, std=40 ** -0.5)

    def lin(p):
        return mb.b200_linear(p["x"], p["w"], p["bias"], "gelu", p["scale"])

    def ffn(p):
        return mb.b200_gated_ffn(p["x"], p["w"], p["wu"])

    dl = dict(zip(("x", "w", "bias", "scale"),
                  mb.b200_linear_backward(t["g"], t["x"], t["w"], t["bias"], "gelu", t["scale"])))
    t["wu"] = wu
    df = dict(zip(("x", "w", "wu"), mb.b200_gated_ffn_backward(t["g"], t["x"], t["w"], wu)))
    for f, grads in ((lin, dl), (ffn, df)):
        for name, gr in grads.items():
            d = randn(g, *t[name].shape)
            d = d * (t[name].norm() / d.norm())
            h = 1e-2
            hi, lo = f({**t, name: t[name] + h * d}), f({**t, name: t[name] - h * d})
            num = float(((hi.double() - lo.double()) * t["g"].double()).sum() / (2 * h))
            ana = float((gr.double() * d.double()).sum())
            size = float(gr.double().norm() * d.double().norm()) / gr.numel() ** 0.5
            assert abs(num - ana) <= 5e-3 * max(abs(ana), size, 1.0), (f.__name__, name, num, ana)


@pytest.mark.parametrize("dt", [BF, F32])
def test_autograd_matches_the_backward_calls(dt):
    t = linear_case(90, 72, 40, dt, "same", "f32", "f32", seed=6, grad=F32)
    leaves = [t[k].clone().requires_grad_(True) for k in ("x", "w", "bias", "scale", "residual")]
    x, w, b, s, r = leaves
    y = mb.b200_linear(x, w, b, "silu", s, r, out_dtype=F32)
    grads = torch.autograd.grad(y, leaves, t["g"], retain_graph=True)
    want = mb.b200_linear_backward(t["g"], t["x"], t["w"], t["bias"], "silu", t["scale"])
    for a, e in zip(grads, want):
        assert torch.equal(a, e)
    assert torch.equal(grads[4], t["g"])
    # only what is asked for, and no graph without gradients
    assert torch.equal(torch.autograd.grad(y, w, t["g"])[0], want[1])
    with torch.no_grad():
        assert not mb.b200_linear(x, w).requires_grad
    d = randn(gen(3), 90, 40, dt=dt)
    wu = randn(gen(4), 40, 72, dt=dt).requires_grad_(True)
    z = mb.b200_gated_ffn(x, w, wu, "gelu")
    got = torch.autograd.grad(z, (x, w, wu), d)
    for a, e in zip(got, mb.b200_gated_ffn_backward(d, t["x"], t["w"], wu.detach(), "gelu")):
        assert torch.equal(a, e)
    # one weight for both projections: its gradient is the sum of the two
    z = mb.b200_gated_ffn(x, w, w)
    got = torch.autograd.grad(z, w, d)[0]
    _, dg, du = mb.b200_gated_ffn_backward(d, t["x"], t["w"], t["w"])
    assert torch.equal(got, dg + du)
    with pytest.raises(RuntimeError, match="once_differentiable"):  # no second derivatives
        y = mb.b200_linear(x, w)
        gx, = torch.autograd.grad(y.float().square().sum(), x, create_graph=True)
        gx.float().sum().backward()


# ---------------------------------------------------------------------------
# streams, graphs, repeats
# ---------------------------------------------------------------------------
def train_calls(t, wu):
    y = mb.b200_linear(t["x"], t["w"], t["bias"], "silu", t["scale"])
    a = mb.b200_gated_ffn(t["x"], t["w"], wu)
    return [y, a, *mb.b200_linear_backward(t["g"], t["x"], t["w"], t["bias"], "silu", t["scale"]),
            *mb.b200_gated_ffn_backward(t["g"], t["x"], t["w"], wu)]


@pytest.mark.parametrize("dt,m", [(BF, 4), (BF, 1500), (F32, 1500)])
def test_same_bits_again_on_another_stream_and_in_two_graphs(dt, m):
    """Results do not change from call to call, nor on a side stream, nor in captured graphs; two
    graphs of the same shapes, replayed at once on two streams, do not share scratch memory."""
    ts = [linear_case(m, 264, 200, dt, "f32", "f32", "none", seed=s, grad=dt) for s in (1, 2)]
    wu = randn(gen(9), 200, 264, dt=dt, std=0.06)
    want = [train_calls(t, wu) for t in ts]
    for t, e in zip(ts, want):
        for a, b in zip(train_calls(t, wu), e):
            assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = train_calls(ts[0], wu)
    side.synchronize()
    for a, b in zip(again, want[0]):
        assert torch.equal(a, b)
    graphs, outs = [], []
    for t in ts:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(train_calls(t, wu))
        graphs.append(gr)
    s2 = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(20):
        with torch.cuda.stream(side):
            graphs[0].replay()
        with torch.cuda.stream(s2):
            graphs[1].replay()
    torch.cuda.synchronize()
    for o, e in zip(outs, want):
        for a, b in zip(o, e):
            assert torch.equal(a, b)


# ---------------------------------------------------------------------------
# the run of them: a block's dense half
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dt,m", [(BF, 1), (BF, 333), (HF, 48), (F32, 130)])
def test_block_of_ffn_and_gated_residual(dt, m):
    """x += sigmoid(gate) * W_down ffn(h), as MabaBlock computes it (maba_sparse/model.py:107-108):
    the inner activation is rounded to the type between the two calls."""
    g = gen(21)
    D, inner = 640, 1248
    h, stream = randn(g, m, D, dt=dt), randn(g, m, D)
    wg, wu = (randn(g, inner, D, dt=dt, std=D ** -0.5) for _ in range(2))
    wd, gate = randn(g, D, inner, dt=dt, std=inner ** -0.5), torch.sigmoid(randn(g, D) + 2)
    a, ea = O.gated(h, wg, wu, "silu")
    y, ey = O.product(a, wd.double())
    y = y * gate.double() + stream.double()
    err = gate.double() * (ey + ea @ wd.double().abs().t()) + 3 * O.E23 * (y.abs() + stream.double().abs())
    mb.b200_linear(mb.b200_gated_ffn(h, wg, wu), wd, scale=gate, residual=stream, out=stream)
    O.assert_within(stream, (y, O.stored(y, err, F32)), "block")


def test_swiglu_module_trains():
    """The module under autograd: its gradients are those of the operators' backward calls, chained;
    and one optimizer step runs."""
    torch.manual_seed(3)
    ffn = mb.SwiGLUFFN(dim=96, intermediate_size=200).to(DEV, BF)
    gate = torch.full((96,), 2.0, device=DEV, requires_grad=True)
    x = randn(gen(1), 2, 35, 96, dt=BF).requires_grad_(True)
    r = randn(gen(2), 2, 35, 96).requires_grad_(True)
    y = ffn(x, residual=r, gate=torch.sigmoid(gate))
    assert y.dtype == F32 and y.shape == r.shape
    d = randn(gen(3), 2, 35, 96)
    y.backward(d)
    wg, wu, wd = (w.weight.detach() for w in (ffn.w_gate, ffn.w_up, ffn.w_down))
    a = mb.b200_gated_ffn(x.detach(), wg, wu)
    s = torch.sigmoid(gate.detach())
    da, dwd, _, ds = mb.b200_linear_backward(d, a, wd, scale=s)
    dx, dwg, dwu = mb.b200_gated_ffn_backward(da, x.detach(), wg, wu)
    for got, want in ((ffn.w_down.weight.grad, dwd), (ffn.w_gate.weight.grad, dwg), (ffn.w_up.weight.grad, dwu),
                      (x.grad, dx), (r.grad, d)):
        assert torch.equal(got, want)
    assert torch.allclose(gate.grad, ds * s * (1 - s), rtol=1e-6, atol=0)
    before = wg.clone()
    torch.optim.SGD(ffn.parameters(), lr=0.1).step()
    assert not torch.equal(ffn.w_gate.weight.detach(), before)


# ---------------------------------------------------------------------------
# extremes
# ---------------------------------------------------------------------------
def test_offsets_past_32_bits():
    """More than 2^31 elements of output and of gradient (4.5 GB): the last rows, and a gradient
    that sums over all of them."""
    m, k, n = 1_100_003, 64, 2048
    w = randn(gen(1), n, k, dt=BF, std=0.1)
    x = randn(gen(2), m, k, dt=BF)
    y = mb.b200_linear(x, w, activation="relu")
    assert y.numel() > 2 ** 31
    for rows in (slice(0, 40), slice(m - 300, m)):
        O.assert_within(y[rows], O.linear(x[rows], w, act="relu"), "rows")
    a = mb.b200_gated_ffn(x, w, w, out=y)
    O.assert_within(a[m - 300:], O.gated(x[m - 300:], w, w, "silu"), "last rows")
    # a gradient that is 1 in the last row and 0 before: dw is that row's outer product
    y.zero_()
    y[m - 1] = 1
    dx, dw, _, _ = mb.b200_linear_backward(y, x, w, activation="relu")
    want = O.linear_backward(y[m - 1:], x[m - 1:], w, act="relu")
    O.assert_within(dw, want["dw"], "dw")
    O.assert_within(dx[m - 1:], want["dx"], "dx")
    assert not dx[:m - 1].any()


@pytest.mark.parametrize("scale", [1e-36, 1e-30, 1e30, 3e38])
def test_float32_magnitudes(scale):
    """Float32 operands at the ends of their range, one nonzero w per sum: the product's rounding, half a
    step 2^-24, within 2^-22 of the value."""
    m, k, n = 70, 8, 40
    g = gen(3)
    x = (torch.rand(m, k, generator=g, device=DEV) * 0.5 + 0.5) * scale
    w = torch.eye(k, device=DEV).repeat(n // k, 1) * (1.0 / scale if scale < 1 else 1e-3)
    y = mb.b200_linear(x, w)
    want = x.double() @ w.double().t()
    tol = 2.0 ** -22 * want.abs()
    assert bool(((y.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("m", [5, 70])
def test_float16_subnormals(m):
    """Float16 values below 2^-14 are operands like any other."""
    x = torch.full((m, 64), 2.0 ** -20, dtype=HF, device=DEV)
    x[:, 32:] = 3 * 2.0 ** -24
    w = torch.full((40, 64), 512.0, dtype=HF, device=DEV)
    want = 32 * 512 * (2.0 ** -20 + 3 * 2.0 ** -24)
    assert bool((mb.b200_linear(x, w, out_dtype=F32) == want).all())


def test_float32_infinities_as_in_float32():
    """inf * w is the infinity of w's sign, inf * 0 and inf - inf are NaN."""
    x = torch.ones(70, 8, device=DEV)
    x[1, 2], x[2, 3], x[3, 0], x[3, 1] = float("inf"), float("-inf"), float("inf"), float("inf")
    w = torch.full((40, 8), 0.3, device=DEV)
    w[5, 2] = -0.7
    w[6, 2] = 0.0
    w[7, 0] = -1.0
    y, want = mb.b200_linear(x, w), x.cpu() @ w.cpu().t()
    assert torch.equal(y.isnan().cpu(), want.isnan()) and torch.equal(y.isinf().cpu(), want.isinf())
    assert torch.equal(y[y.isinf()].cpu(), want[want.isinf()])
    assert bool(y[10:].isfinite().all())


def test_first_call_of_a_process_inside_a_capture():
    """Nothing has to run before a call is captured: a fresh process captures its first calls."""
    import subprocess
    import sys
    import os

    code = """
import torch, maba_v2_architecture_b200 as mb
x = torch.randn(300, 96, device="cuda").bfloat16(); w = torch.randn(64, 96, device="cuda").bfloat16()
f = torch.randn(300, 96, device="cuda"); v = torch.randn(64, 96, device="cuda")
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    outs = [mb.b200_linear(x, w), mb.b200_linear(x[:3], w), mb.b200_gated_ffn(f, v, v), mb.b200_linear(f[:2], v)]
    outs += list(mb.b200_gated_ffn_backward(outs[0], x, w, w))
g.replay(); torch.cuda.synchronize()
again = [mb.b200_linear(x, w), mb.b200_linear(x[:3], w), mb.b200_gated_ffn(f, v, v), mb.b200_linear(f[:2], v)]
again += list(mb.b200_gated_ffn_backward(again[0], x, w, w))
assert all(torch.equal(a, b) for a, b in zip(outs, again))
print("captured")
"""
    repo = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=repo, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


def test_two_threads_at_once():
    """Calls from two host threads, each on its own stream."""
    import threading

    ts = [linear_case(m, 264, 200, BF, "f32", "f32", "none", seed=m, grad=BF) for m in (700, 1500)]
    wu = randn(gen(9), 200, 264, dt=BF, std=0.06)
    want = [train_calls(t, wu) for t in ts]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(20):
                got = train_calls(ts[i], wu)
                s.synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                    bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


@pytest.mark.parametrize("dt", [BF, HF, F32])
@pytest.mark.parametrize("m,k,n", [(900, 3000, 300), (64, 1500, 40)])
def test_float32_results_of_long_sums(m, k, n, dt):
    """What ends in float32 (a float32 result, the gradient of a float32 scale) does not lose what the
    tensor cores truncate over a long contraction.  An accumulation of 640 random products loses 6e-7
    of its own size; those of a sum add like its parts do, in quadrature, so the sum loses 6e-7 of its
    norm whatever its length, and the rounding of the additions (2^-24 each) stays below 1e-7.  One
    accumulation of 3,000 would lose 3e-6."""
    t = linear_case(m, k, n, dt, "f32", "f32", "none", seed=2, grad=dt)
    y = mb.b200_linear(t["x"], t["w"], t["bias"], "none", t["scale"], out_dtype=F32)
    want = (t["x"].double() @ t["w"].double().t() + t["bias"].double()) * t["scale"].double()
    assert float((y.double() - want).norm() / want.norm()) <= 1e-6
    ds = mb.b200_linear_backward(t["g"], t["x"], t["w"], t["bias"], "none", t["scale"])[3]
    z = t["x"].double() @ t["w"].double().t() + t["bias"].double()
    want = (t["g"].double() * z).sum(0)
    assert float((ds.double() - want).norm() / want.norm()) <= 1e-6
