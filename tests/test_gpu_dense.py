"""Dense operators (gated feed-forward block, projection with its epilogue) against plain float64 torch.

Tolerances.  A product of K terms on the tensor cores adds 16 terms per instruction to a float32 accumulator and may
truncate: every addition is off by at most one step (2^-23) of a running sum that is at most S = sum |a b|, so the sum is off by
at most T(K) S with T(K) = (K / 16 + 16) 2^-22 (twice that bound, which also covers the joins of a split sum).  The activations add 2^-18 relative, and
a result is rounded once, by at most eps / 2.  A gradient product reads operands that were rounded once more: S (eps / 2).  As S is
far above |result| for random signs, gradients are also bounded in the 2-norm: two independent roundings of at most
eps / 2 each stay below eps.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def eps(dt):
    return torch.finfo(dt).eps


def trunc(k):
    return (k / 16 + 16) * 2.0**-22


def rows(gen, m, k, dt, pad=0, scale=1.0):
    """Random rows as a view into longer ones whose padding is NaN: nothing may depend on it."""
    t = torch.full((m, k + pad), float("nan"), dtype=dt, device="cuda")
    t[:, :k] = (scale * torch.randn((m, k), device="cuda", generator=gen)).to(dt)
    return t[:, :k]


def within(got, want, tol, what):
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    bad = off > tol
    assert not bad.any(), f"{what}: {int(bad.sum())} values off, worst {float((off - tol).max()):.3g} beyond the tolerance"


def rel_fro(got, want):
    return float((got.double() - want).norm() / want.norm().clamp(min=1e-300))


def glu64(g, u, act):
    if act == "geglu":
        g, u = g.clamp(max=7.0), u.clamp(-7.0, 7.0) + 1.0
        return g * torch.sigmoid(1.702 * g) * u
    return g * torch.sigmoid(g) * u


def act64(z, act):
    if act == "relu":
        return torch.relu(z)  # no gradient at 0 (clamp has one there)
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu":
        return z * 0.5 * torch.erfc(-z * 0.5**0.5)
    return z


# tokens, k, n: one token, a few, every tile of the token side, several tiles; one to several tiles of k and n, odd n
SHAPES = [
    (1, 8, 1), (1, 4096, 640), (2, 64, 7), (7, 72, 129), (16, 520, 128), (17, 1000, 200), (33, 128, 64), (64, 2048, 127), (65, 192, 300),
    (128, 64, 256), (129, 1024, 1001), (300, 776, 520), (513, 1544, 260), (1030, 512, 777),
    # enough 256 x 256 tiles for the kernel of CTA pairs, forward and backward: fewer tiles than pairs, several rounds, odd edges
    (1300, 520, 2100), (130, 1544, 3001), (2049, 264, 1290), (2600, 72, 3100), (4096, 136, 2304),
]  # fmt: skip


@pytest.mark.parametrize("m,k,n", SHAPES)
@pytest.mark.parametrize("act,dt,pad", [("swiglu", BF16, 0), ("geglu", FP16, 24)])
def test_gated_ffn(m, k, n, act, dt, pad):
    import cudnn_frontend_b200 as cf

    gen = torch.Generator(device="cuda").manual_seed(m * 7 + k + n)
    size = (3.0 if act == "geglu" else 1.0) / k**0.5
    x, wg, wu = rows(gen, m, k, dt, pad), rows(gen, n, k, dt, pad, size), rows(gen, n, k, dt, pad, size)
    h, gate, up = cf.gated_ffn(x, wg, wu, act_func=act, return_preact=True)
    only = cf.gated_ffn(x, wg, wu, act_func=act)
    x, wg, wu = x.double(), wg.double(), wu.double()
    g, u = x @ wg.t(), x @ wu.t()
    sg, su = x.abs() @ wg.abs().t() * trunc(k), x.abs() @ wu.abs().t() * trunc(k)
    e = eps(dt) / 2
    tiny = torch.finfo(dt).tiny * eps(dt)  # half a step below the normal numbers
    within(gate, g, e * (g.abs() + sg) + sg + tiny, "gate")
    within(up, u, e * (u.abs() + su) + su + tiny, "up")
    want = glu64(g, u, act)
    # |d h / d gate| <= 1.2 (|u| + 1), |d h / d up| <= |gate|
    off = 1.2 * (u.abs() + 1) * sg + g.abs() * su + 2.0**-18 * want.abs()
    within(h, want, e * (want.abs() + off) + off + tiny, "h")
    assert torch.equal(h, only)


@pytest.mark.parametrize("m,k,n", SHAPES)
@pytest.mark.parametrize("act,dt,pad", [("swiglu", BF16, 8), ("geglu", FP16, 0)])
def test_gated_ffn_backward(m, k, n, act, dt, pad):
    import cudnn_frontend_b200 as cf

    gen = torch.Generator(device="cuda").manual_seed(m * 5 + k + n)
    x, wg, wu = rows(gen, m, k, dt, pad), rows(gen, n, k, dt, pad, k**-0.5), rows(gen, n, k, dt, pad, k**-0.5)
    dh = rows(gen, m, n, dt, pad)
    gate, up = rows(gen, m, n, dt, pad, 4.0), rows(gen, m, n, dt, 0, 4.0)
    dx, dwg, dwu = cf.gated_ffn_backward(dh, x, wg, wu, gate, up, act_func=act)
    g, u = gate.double().requires_grad_(), up.double().requires_grad_()
    dg, du = torch.autograd.grad(glu64(g, u, act), (g, u), dh.double())
    x, wg, wu = x.double(), wg.double(), wu.double()
    e = eps(dt) / 2
    for name, got, pairs, red in (("dx", dx, ((dg, wg), (du, wu)), 2 * n), ("dw_gate", dwg, ((dg.t(), x),), m), ("dw_up", dwu, ((du.t(), x),), m)):
        want = sum(a @ b for a, b in pairs)
        s = sum(a.abs() @ b.abs() for a, b in pairs)
        off = s * (e + 2.0**-18 + trunc(red)) + sum((a != 0).double() @ b.abs() for a, b in pairs) * torch.finfo(dt).tiny * eps(dt)
        within(got, want, e * (want.abs() + off) + off + torch.finfo(dt).tiny * eps(dt), name)
        if want.numel() > 1000:
            assert rel_fro(got, want) <= eps(dt), name


@pytest.mark.parametrize("m,k,n", SHAPES)
@pytest.mark.parametrize(
    "act,dt,pad,bias,res,out",
    [(None, BF16, 0, None, False, None), ("gelu", FP16, 24, "same", True, None), ("silu", BF16, 8, "f32", True, torch.float32), ("relu", FP16, 0, None, False, None),
     (None, BF16, 0, "same", False, torch.float32)],
)  # fmt: skip
def test_linear(m, k, n, act, dt, pad, bias, res, out):
    import cudnn_frontend_b200 as cf

    gen = torch.Generator(device="cuda").manual_seed(m * 3 + k + n)
    x, w = rows(gen, m, k, dt, pad), rows(gen, n, k, dt, pad, k**-0.5)
    b = None if bias is None else torch.randn((n,), device="cuda", generator=gen).to(dt if bias == "same" else torch.float32)
    r = rows(gen, m, n, dt, 3) if res else None
    y, z = cf.linear(x, w, bias=b, act_func=act, residual=r, out_dtype=out, return_preact=True)
    assert torch.equal(y, cf.linear(x, w, bias=b, act_func=act, residual=r, out_dtype=out))
    x, w = x.double(), w.double()
    z64 = x @ w.t() + (0 if b is None else b.double())
    s = x.abs() @ w.abs().t() * trunc(k if out is None else 512)  # float32 results: summed by segments of 512
    if out is not None:
        s = s + (x.abs() @ w.abs().t() + z64.abs()) * (k / 512 + 9) * 2.0**-24  # and the segments with round-to-nearest
    s = s + 2.0**-23 * z64.abs()  # the bias addition
    e, tiny = eps(dt) / 2, torch.finfo(dt).tiny * eps(dt)
    within(z, z64, e * (z64.abs() + s) + s + tiny, "preact")
    want = act64(z64, act)
    off = 1.2 * s + 2.0**-18 * want.abs()  # |act'| <= 1.2
    if res:
        want = want + r.double()
        off = off + 2.0**-23 * want.abs()
    if out is None:
        within(y, want, e * (want.abs() + off) + off + tiny, "y")
    else:
        assert y.dtype == torch.float32
        within(y, want, 2.0**-23 * want.abs() + off + 1e-30, "y")


def test_linear_float32_output_is_not_biased_by_the_accumulator():
    """Over a long reduction the truncating accumulator alone would leave 7e-6; in segments of 512 elements at most
    16 * 32 / 16 = 32 truncations of 2^-23 each, of which the mean is half: 2e-6 as a bound, and 2^-24 per segment's addition."""
    import cudnn_frontend_b200 as cf

    gen = torch.Generator(device="cuda").manual_seed(1)
    x, w = rows(gen, 300, 14336, BF16), rows(gen, 256, 14336, BF16, scale=14336**-0.5)
    for m in (300, 5):
        y = cf.linear(x[:m], w, out_dtype=torch.float32)
        assert rel_fro(y, x[:m].double() @ w.double().t()) <= 2e-6


@pytest.mark.parametrize("m,k,n", SHAPES)
@pytest.mark.parametrize(
    "act,dt,pad,bias,dy_f32",
    [(None, BF16, 0, True, False), ("gelu", FP16, 24, True, False), ("silu", BF16, 8, True, True), ("relu", FP16, 0, False, False), (None, BF16, 3, False, True)],
)
def test_linear_backward(m, k, n, act, dt, pad, bias, dy_f32):
    import cudnn_frontend_b200 as cf

    gen = torch.Generator(device="cuda").manual_seed(m * 11 + k + n)
    even = pad // 8 * 8
    x, w = rows(gen, m, k, dt, even), rows(gen, n, k, dt, even, k**-0.5)
    dy = rows(gen, m, n, torch.float32 if dy_f32 else dt, pad)
    z = rows(gen, m, n, dt, pad, 2.0) if act else None
    dx, dw, db = cf.linear_backward(dy, x, w, preact=z, act_func=act, bias_grad=bias)
    dz = dy.double()
    if act:
        z64 = z.double().requires_grad_()
        (dz,) = torch.autograd.grad(act64(z64, act), z64, dz)
    x, w = x.double(), w.double()
    e, tiny = eps(dt) / 2, torch.finfo(dt).tiny * eps(dt)
    near = 2.0**-18 * (dy.double().abs() if act else 0)  # the activation's derivative may cancel: an absolute error of 2^-18
    for name, got, a, b, red in (("dx", dx, dz, w, n), ("dw", dw, dz.t(), x, m)):
        want, s = a @ b, a.abs() @ b.abs()
        off = s * (e + trunc(red)) + torch.ones_like(a) @ b.abs() * tiny
        if act:
            off = off + (near if name == "dx" else near.t()) @ b.abs()
        within(got, want, e * (want.abs() + off) + off + tiny, name)
        if want.numel() > 1000:
            assert rel_fro(got, want) <= eps(dt), name
    assert (db is None) == (not bias)
    if bias:
        within(db, dz.sum(0), (dz.abs().sum(0) * (m + 8) * 2.0**-24) + (near.sum(0) if act else 0) + 1e-30, "dbias")


def test_broadcast_residual_and_single_row_views():
    import cudnn_frontend_b200 as cf

    gen = torch.Generator(device="cuda").manual_seed(3)
    x, w = rows(gen, 40, 64, BF16), rows(gen, 96, 64, BF16)
    r = torch.randn((1, 96), device="cuda", generator=gen).to(BF16)
    assert torch.equal(cf.linear(x, w, residual=r.expand(40, 96)), cf.linear(x, w, residual=r.repeat(40, 1)))
    assert torch.equal(cf.linear(x[5:6], w)[0], cf.linear(x, w)[5])
    # every other row, and a row whose pitch is odd
    assert torch.equal(cf.linear(x[::2], w), cf.linear(x, w)[::2])
    one = torch.randn((1, 71), device="cuda", generator=gen).to(BF16)[:, :64]
    assert torch.equal(cf.linear(one, w), cf.linear(one.contiguous(), w))


def test_gradients_that_are_not_asked_for():
    import cudnn_frontend_b200 as cf

    gen = torch.Generator(device="cuda").manual_seed(12)
    for m, k, n in ((40, 64, 96), (1500, 512, 2048)):
        x, w, u, dy = rows(gen, m, k, BF16), rows(gen, n, k, BF16), rows(gen, n, k, BF16), rows(gen, m, n, BF16)
        full = cf.linear_backward(dy, x, w, bias_grad=True)
        dx, none, _ = cf.linear_backward(dy, x, w, weight_grad=False)
        none2, dw, none3 = cf.linear_backward(dy, x, w, input_grad=False)
        assert none is none2 is none3 is None
        assert rel_fro(dx, full[0].double()) <= eps(BF16) and rel_fro(dw, full[1].double()) <= eps(BF16)
        only = cf.linear_backward(dy, x, w, bias_grad=True, input_grad=False, weight_grad=False)
        assert only[0] is only[1] is None and torch.equal(only[2], full[2])
        full = cf.gated_ffn_backward(dy, x, w, u, dy, dy)
        dx, *none = cf.gated_ffn_backward(dy, x, w, u, dy, dy, weight_grad=False)
        none4, *dws = cf.gated_ffn_backward(dy, x, w, u, dy, dy, input_grad=False)
        assert none == [None, None] and none4 is None
        for a, b in zip((dx, *dws), full):
            assert rel_fro(a, b.double()) <= eps(BF16)


def test_traced_calls_go_through_the_custom_ops():
    import cudnn_frontend_b200 as cf

    gen = torch.Generator(device="cuda").manual_seed(13)
    x, wg, wu, wd, wr = rows(gen, 30, 64, BF16), rows(gen, 96, 64, BF16), rows(gen, 96, 64, BF16), rows(gen, 64, 96, BF16), rows(gen, 8, 64, BF16)

    def layer(x):
        w, ids = cf.router_topk(cf.linear(x, wr, out_dtype=torch.float32), 2)
        h, gate, up = cf.gated_ffn(x, wg, wu, return_preact=True)
        return (*cf.linear(h, wd, act_func="silu", residual=x, return_preact=True), gate, up, w, ids)

    seen = []

    def backend(graph, _):
        seen.extend(str(n.target) for n in graph.graph.nodes if n.op == "call_function")
        return graph.forward

    got = torch.compile(layer, backend=backend, fullgraph=True)(x)
    assert all(torch.equal(a, b) for a, b in zip(got, layer(x)))
    assert sum("b200moe" in t for t in seen) == 4


def test_no_tokens():
    import cudnn_frontend_b200 as cf

    x, w = torch.empty((0, 64), dtype=BF16, device="cuda"), torch.randn((24, 64), device="cuda").to(BF16)
    e = torch.empty((0, 24), dtype=BF16, device="cuda")
    assert cf.gated_ffn(x, w, w).shape == (0, 24) and cf.linear(x, w, bias=w[:, 0].contiguous(), residual=e).shape == (0, 24)
    dx, dg, du = cf.gated_ffn_backward(e, x, w, w, e, e)
    assert dx.shape == (0, 64) and not dg.any() and not du.any() and dg.shape == du.shape == w.shape
    dx, dw, db = cf.linear_backward(e, x, w, bias_grad=True)
    assert dx.shape == (0, 64) and not dw.any() and not db.any()


def test_special_values_stay_in_their_rows():
    import cudnn_frontend_b200 as cf

    gen = torch.Generator(device="cuda").manual_seed(4)
    for m in (5, 300):
        x, w = rows(gen, m, 200, BF16), rows(gen, 136, 200, BF16, scale=0.07)
        clean = cf.gated_ffn(x, w, w), cf.linear(x, w, act_func="relu")
        x2 = x.clone()
        x2[3, 7], x2[4, 8] = float("nan"), float("inf")
        for got, want in zip((cf.gated_ffn(x2, w, w), cf.linear(x2, w, act_func="relu")), clean):
            assert torch.isnan(got[3]).all()
            keep = [i for i in range(m) if i not in (3, 4)]
            assert torch.equal(got[keep], want[keep])


def test_geglu_limits_have_no_gradient():
    import cudnn_frontend_b200 as cf

    one = torch.ones((4, 8), dtype=FP16, device="cuda")
    w = torch.eye(8, dtype=FP16, device="cuda")
    gate = torch.full((4, 8), 7.5, dtype=FP16, device="cuda")
    up = torch.full((4, 8), 2.0, dtype=FP16, device="cuda")
    _, dg, du = cf.gated_ffn_backward(one, one, w, w, gate, up, act_func="geglu")
    assert not dg.any() and du.all()
    _, dg, du = cf.gated_ffn_backward(one, one, w, w, up, -gate, act_func="geglu")
    assert dg.all() and not du.any()


def test_results_do_not_depend_on_timing_or_stream():
    import cudnn_frontend_b200 as cf

    gen = torch.Generator(device="cuda").manual_seed(5)
    for m, k, n in ((3, 2048, 512), (700, 512, 1024)):
        x, wg, wu = rows(gen, m, k, BF16), rows(gen, n, k, BF16, scale=k**-0.5), rows(gen, n, k, BF16, scale=k**-0.5)
        dh = rows(gen, m, n, BF16)
        h, g, u = cf.gated_ffn(x, wg, wu, return_preact=True)
        back = cf.gated_ffn_backward(dh, x, wg, wu, g, u)
        lin = cf.linear_backward(dh, x, wg, preact=g, act_func="gelu", bias_grad=True)
        torch.cuda.synchronize()
        side = [torch.cuda.Stream(), torch.cuda.Stream()]
        for s in side:
            s.wait_stream(torch.cuda.current_stream())
        runs = []
        for i in range(6):  # two streams at once, one named by its raw handle
            s = side[i % 2] if i < 4 else side[i % 2].cuda_stream
            runs.append((cf.gated_ffn(x, wg, wu, stream=s), cf.gated_ffn_backward(dh, x, wg, wu, g, u, stream=s),
                         cf.linear_backward(dh, x, wg, preact=g, act_func="gelu", bias_grad=True, stream=s)))  # fmt: skip
        torch.cuda.synchronize()
        for a, b, c in runs:
            assert torch.equal(a, h)
            assert all(torch.equal(p, q) for p, q in zip(b, back)) and all(torch.equal(p, q) for p, q in zip(c, lin))


def test_captured_graphs_replay_on_new_values():
    import cudnn_frontend_b200 as cf

    gen = torch.Generator(device="cuda").manual_seed(6)
    k, n = 512, 384
    wg, wu, wd = rows(gen, n, k, BF16, scale=k**-0.5), rows(gen, n, k, BF16, scale=k**-0.5), rows(gen, k, n, BF16, scale=n**-0.5)

    def step(x, dy):
        h, g, u = cf.gated_ffn(x, wg, wu, return_preact=True)
        y = cf.linear(h, wd, residual=x)
        dh, dwd, _ = cf.linear_backward(dy, h, wd)
        return (y, dwd, *cf.gated_ffn_backward(dh, x, wg, wu, g, u))

    graphs = []
    for m in (4, 150):  # two graphs, whose memory is their own, replayed at the same time
        x, dy = rows(gen, m, k, BF16).clone(), rows(gen, m, k, BF16).clone()
        step(x, dy)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(x, dy)
        graphs.append((graph, x, dy, out))
    for _ in range(3):
        for _, x, dy, _ in graphs:
            x.copy_(torch.randn(x.shape, device="cuda", generator=gen))
            dy.copy_(torch.randn(dy.shape, device="cuda", generator=gen))
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for (graph, *_), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for _, x, dy, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, step(x, dy)))


def test_gradients_against_differences():
    """The backward pass against central differences of the forward pass, which runs with float32 output on fp16 inputs, so that
    only the difference's own third-order error and the gradient's roundings (2^-11 of dz, of the result and of the saved
    pre-activation: below 2e-3 of the terms' sizes) count."""
    import cudnn_frontend_b200 as cf

    gen = torch.Generator(device="cuda").manual_seed(7)
    m, k, n = 24, 64, 40
    x, w = rows(gen, m, k, FP16, scale=0.5), rows(gen, n, k, FP16, scale=k**-0.5)
    b = torch.randn((n,), device="cuda", generator=gen)
    dy = torch.randn((m, n), device="cuda", generator=gen)
    for act in ("silu", "gelu"):
        z = (x.double() @ w.double().t() + b.double()).half()
        dx, dw, db = cf.linear_backward(dy, x, w, preact=z, act_func=act, bias_grad=True)

        def loss(x, w, b):
            y = cf.linear(x, w, bias=b, act_func=act, out_dtype=torch.float32)
            return float((y.double() * dy.double()).sum())

        # the bias: a central difference along the gradient's signs, off by third derivatives (below 1.2) times step^3 / 6
        # per value, and by the pre-activation's rounding in the derivative
        step = 2.0**-4
        v = step * torch.sign(db)
        got = (loss(x, w, b + v) - loss(x, w, b - v)) / 2
        size = float(dy.double().abs().sum())
        assert abs(got - float((db.double() * v.double()).sum())) <= size * (1.2 / 6 * step**3 + 1e-3 * step) + 1e-4
        # one coordinate at a time: third derivatives of both activations are below 1.2, so the difference is off by at most
        # (step |v|)^3 / 6 * 1.2 * sum |dy| of the row or column, and by the gradient's own rounding
        for _ in range(6):
            i, j, o = (int(torch.randint(0, q, (1,), generator=gen, device="cuda")) for q in (m, k, n))
            up, down = x.clone(), x.clone()
            up[i, j] += 0.25
            down[i, j] -= 0.25
            d = float(up[i, j].double() - down[i, j].double()) / 2
            got = (loss(up, w, b) - loss(down, w, b)) / 2
            third = 1.2 / 6 * float(((d * w[:, j].double()).abs() ** 3 * dy[i].double().abs()).sum())
            scale = float((w[:, j].double().abs() * dy[i].double().abs()).sum()) * abs(d)
            assert abs(got - float(dx[i, j]) * d) <= third + 2e-3 * scale + 1e-4
            up, down = w.clone(), w.clone()
            up[o, j] += 0.125
            down[o, j] -= 0.125
            d = float(up[o, j].double() - down[o, j].double()) / 2
            got = (loss(x, up, b) - loss(x, down, b)) / 2
            third = 1.2 / 6 * float(((d * x[:, j].double()).abs() ** 3 * dy[:, o].double().abs()).sum())
            scale = float((x[:, j].double().abs() * dy[:, o].double().abs()).sum()) * abs(d)
            assert abs(got - float(dw[o, j]) * d) <= third + 2e-3 * scale + 1e-4


def test_refusals():
    import cudnn_frontend_b200 as cf

    x, w = torch.randn((4, 64), device="cuda").to(BF16), torch.randn((24, 64), device="cuda").to(BF16)
    h = torch.randn((4, 24), device="cuda").to(BF16)
    with pytest.raises(NotImplementedError):
        cf.gated_ffn(x.float(), w, w)
    with pytest.raises(NotImplementedError):
        cf.linear(x, w, out_dtype=FP16)
    with pytest.raises(NotImplementedError):
        cf.linear(x, w, bias=torch.zeros(24, device="cuda", dtype=FP16))
    for call in (
        lambda: cf.gated_ffn(x, w, w.half()),
        lambda: cf.gated_ffn(x, w, w[:8]),
        lambda: cf.gated_ffn(x, w, w, act_func="relu"),
        lambda: cf.gated_ffn(x.cpu(), w, w),
        lambda: cf.gated_ffn(x, w.cpu(), w),
        lambda: cf.linear(x[0], w),
        lambda: cf.linear(x, w, act_func="swiglu"),
        lambda: cf.linear(x, w[:, :40]),
        lambda: cf.linear(x[:, :60], w[:, :60]),  # k not a multiple of 8
        lambda: cf.linear(x, torch.randn((24, 65), device="cuda").to(BF16)[:, 1:]),  # odd pitch and start
        lambda: cf.linear(torch.randn((4 * 64 + 1,), device="cuda").to(BF16)[1:].view(4, 64), w),  # not on a 16-byte boundary
        lambda: cf.linear(torch.randn((64, 4), device="cuda").to(BF16).t(), w),  # columns contiguous
        lambda: cf.linear(x[:1].expand(4, 64), w),  # rows on top of one another
        lambda: cf.linear(x, w, bias=torch.zeros(23, device="cuda")),
        lambda: cf.linear(x, w, residual=h.t()),
        lambda: cf.linear_backward(h, x, w, act_func="silu"),  # no pre-activation
        lambda: cf.linear_backward(h[:3], x, w),
        lambda: cf.gated_ffn_backward(h, x, w, w, h, h.float()),
    ):
        with pytest.raises(ValueError):
            call()
    torch.cuda.synchronize()


@pytest.mark.parametrize("m,n,kernel", [(3, 256, "tile"), (40, 300, "tile"), (2048, 2048, "pair")])
def test_bounded_waits_report_and_recover(m, n, kernel):
    """A launch whose operand B never arrives ends after its wait limit, says which wait gave up, and leaves the device
    usable: the next launch is right."""
    import ctypes

    import cudnn_frontend_b200 as cf
    from cudnn_frontend_b200 import _lib, ops

    gen = torch.Generator(device="cuda").manual_seed(8)
    k = 2048
    x, w = rows(gen, m, k, BF16), rows(gen, n, k, BF16, scale=k**-0.5)
    want = cf.linear(x, w)
    y = torch.zeros_like(want)
    args = dict(x=x.data_ptr(), w0=w.data_ptr(), y=y.data_ptr(), m=m, n=n, k=k, ld_x=k, ld_w0=k, ld_y=n, act=_lib.ACT_NONE, wait_limit_ms=20)
    torch.cuda.synchronize()
    assert ops.device_status(clear=True) == 0
    stream = torch.cuda.current_stream().cuda_stream
    assert _lib.load().b200moe_linear(ctypes.byref(_lib.DenseArgs(flags=_lib.FLAG_TEST_SKIP_B_LOADS, **args)), stream) == 0
    torch.cuda.synchronize()
    assert ops.device_status(clear=True) in ({"tile": (401, 402, 403), "pair": (411, 412, 413, 414)}[kernel])
    assert _lib.load().b200moe_linear(ctypes.byref(_lib.DenseArgs(**args)), stream) == 0
    torch.cuda.synchronize()
    assert ops.device_status(clear=True) == 0
    assert torch.equal(y, want)


def test_offsets_beyond_32_bits():
    """Inputs and outputs of more than 2^32 bytes and 2^31 elements: their last rows against the same rows alone."""
    import cudnn_frontend_b200 as cf

    gen = torch.Generator(device="cuda").manual_seed(14)
    m, k, n = 540_000, 4096, 16  # x: 2.2e9 elements
    x = torch.empty((m, k), dtype=BF16, device="cuda").normal_(generator=gen)
    w = rows(gen, n, k, BF16, scale=k**-0.5)
    for kw in ({}, {"out_dtype": torch.float32}):
        assert rel_fro(cf.linear(x, w, **kw)[-300:], x[-300:].double() @ w.double().t()) <= eps(BF16)
    dy = rows(gen, m, n, BF16)
    dx, dw, _ = cf.linear_backward(dy, x, w)
    assert rel_fro(dx[-300:], dy[-300:].double() @ w.double()) <= eps(BF16)
    want = sum(dy[i : i + 60_000].float().t() @ x[i : i + 60_000].float() for i in range(0, m, 60_000))
    assert rel_fro(dw, want.double()) <= eps(BF16)
    del x, dx
    m, k, n = 60_000, 64, 40_000  # results: 2.4e9 elements
    x, w = rows(gen, m, k, BF16), rows(gen, n, k, BF16, scale=k**-0.5)
    g = x[-300:].double() @ w.double().t()
    assert rel_fro(cf.linear(x, w)[-300:], g) <= eps(BF16)
    assert rel_fro(cf.gated_ffn(x, w, w)[-300:], g * torch.sigmoid(g) * g) <= eps(BF16)


def scaled_operand_tol(a):
    """What rounding dz (dg, du) to fp16 may cost beyond half a step of each value.  The call scales them by a power of two so that
    the largest lies in [2^14, 2^15); the smallest step of fp16, 2^-24, is then at most 2^-24 2^-14 of the largest, and a rounding
    half of that."""
    return 2.0**-39 * a.abs().max()


@pytest.mark.parametrize("m,k,n", [(1, 64, 8), (3, 64, 40), (65, 192, 300), (700, 512, 1024), (2049, 264, 1290), (1024, 2048, 256)])
@pytest.mark.parametrize("act,dy_f32", [(None, True), ("silu", True), ("gelu", False), ("relu", True)])
@pytest.mark.parametrize("size", [1e-7, 1.0, 1e5])
def test_float16_gradients_keep_their_range(m, k, n, act, dy_f32, size):
    """dz far below or above what fp16 holds, with gradients that it does hold: inputs and weights are large where dy is small
    (float32 values of 1e-7, far below fp16's normal numbers) and small where it is large."""
    import cudnn_frontend_b200 as cf

    if not dy_f32:
        size = min(size, 2e4)  # (3 standard deviations below 65504; times |act'| <= 1.13 it may leave the range)
    gen = torch.Generator(device="cuda").manual_seed(m + k + n)
    other = min(64.0, 3000.0 / size / (m + n) ** 0.5)  # gradients of a few thousand at most: no sum leaves fp16's range
    x, w = rows(gen, m, k, FP16, 8, other), rows(gen, n, k, FP16, 0, other)
    dy = rows(gen, m, n, torch.float32 if dy_f32 else FP16, 8, size)
    if not dy_f32:
        dy.clamp_(-65504, 65504)
    z = rows(gen, m, n, FP16, 0, 2.0) if act else None
    dx, dw, db = cf.linear_backward(dy, x, w, preact=z, act_func=act, bias_grad=True)
    dz = dy.double()
    if act:
        z64 = z.double().requires_grad_()
        (dz,) = torch.autograd.grad(act64(z64, act), z64, dz)
    x, w = x.double(), w.double()
    e, tiny = eps(FP16) / 2, torch.finfo(FP16).tiny * eps(FP16)
    near = 2.0**-18 * (dy.double().abs() if act else torch.zeros_like(dz))
    step = scaled_operand_tol(dz)
    for name, got, a, near_a, b, red in (("dx", dx, dz, near, w, n), ("dw", dw, dz.t(), near.t(), x, m)):
        want, s = a @ b, a.abs() @ b.abs()
        off = s * (e + trunc(red)) + (near_a + step) @ b.abs()
        within(got, want, e * (want.abs() + off) + off + tiny, name)
    within(db, dz.sum(0), dz.abs().sum(0) * (m + 8) * 2.0**-24 + near.sum(0) + 1e-30, "dbias")


@pytest.mark.parametrize("m,k,n", [(1, 64, 8), (3, 64, 40), (65, 192, 300), (700, 512, 1024), (2049, 264, 1290), (128, 2048, 512)])
@pytest.mark.parametrize("act", ["swiglu", "geglu"])
@pytest.mark.parametrize("dh_size,up_size", [(1e4, 30.0), (1e-4, 1e-3), (1.0, 1.0)])
def test_float16_gated_gradients_keep_their_range(m, k, n, act, dh_size, up_size):
    """dg = dh up act'(gate) beyond 65504, or far below fp16's normal numbers, with gradients that fp16 holds."""
    import cudnn_frontend_b200 as cf

    gen = torch.Generator(device="cuda").manual_seed(m + k + n)
    other = min(64.0, 1500.0 / (dh_size * max(up_size, 4.0)) / (m + n) ** 0.5)
    x, wg, wu = rows(gen, m, k, FP16, 8, other), rows(gen, n, k, FP16, 0, other), rows(gen, n, k, FP16, 8, other)
    dh, gate, up = rows(gen, m, n, FP16, 0, dh_size), rows(gen, m, n, FP16, 8, 4.0), rows(gen, m, n, FP16, 0, up_size)
    dx, dwg, dwu = cf.gated_ffn_backward(dh, x, wg, wu, gate, up, act_func=act)
    g, u = gate.double().requires_grad_(), up.double().requires_grad_()
    dg, du = torch.autograd.grad(glu64(g, u, act), (g, u), dh.double())
    x, wg, wu = x.double(), wg.double(), wu.double()
    e, tiny = eps(FP16) / 2, torch.finfo(FP16).tiny * eps(FP16)
    step = max(scaled_operand_tol(dg), scaled_operand_tol(du))
    # act'(gate) = s (1 + g (1 - s)) may cancel: an absolute error of 2^-18 of its terms, which stay below 1.2 for the values it has
    # (|dh| (|up| + 1) for the gate, |dh gate| for up)
    near_g, near_u = 2.0**-18 * dh.double().abs() * (u.detach().abs() + 1), 2.0**-18 * (dh.double() * g.detach()).abs()
    for name, got, pairs, red in (
        ("dx", dx, ((dg, near_g, wg), (du, near_u, wu)), 2 * n), ("dw_gate", dwg, ((dg.t(), near_g.t(), x),), m), ("dw_up", dwu, ((du.t(), near_u.t(), x),), m)):  # fmt: skip
        want, s = sum(a @ b for a, _, b in pairs), sum(a.abs() @ b.abs() for a, _, b in pairs)
        off = s * (e + trunc(red)) + sum((near + step) @ b.abs() for _, near, b in pairs)
        within(got, want, e * (want.abs() + off) + off + tiny, name)


def test_float16_gradients_with_infinities_and_zeros():
    """An infinite or NaN value reaches its own row of dx and its own row of dw only, and does not decide the scale of the others; a
    gradient of nothing but zeros gives zeros."""
    import cudnn_frontend_b200 as cf

    gen = torch.Generator(device="cuda").manual_seed(21)
    for m, k, n in ((20, 64, 40), (1500, 512, 2048)):
        x, w = rows(gen, m, k, FP16, 0, 64.0), rows(gen, n, k, FP16, 0, 64.0)
        dy = rows(gen, m, n, torch.float32, 0, 1e-7)
        clean = cf.linear_backward(dy, x, w)
        bad = dy.clone()
        bad[3, 7], bad[4, 8] = float("nan"), float("inf")
        dx, dw, _ = cf.linear_backward(bad, x, w)
        rest = [i for i in range(m) if i not in (3, 4)]
        cols = [i for i in range(n) if i not in (7, 8)]
        assert rel_fro(dx[rest], clean[0][rest].double()) <= eps(FP16) and torch.isnan(dx[3]).all() and not torch.isfinite(dx[4]).any()
        assert torch.isnan(dw[7]).all() and not torch.isfinite(dw[8]).any()
        # (dw's other rows read dz's rows 3 and 4 as well, where their values are finite: 2 of m terms)
        assert rel_fro(dw[cols], clean[1][cols].double()) <= eps(FP16)
        zero = cf.linear_backward(torch.zeros_like(dy), x, w, bias_grad=True)
        assert not any(t.any() for t in zero)
        h = torch.zeros((m, n), dtype=FP16, device="cuda")
        assert not any(t.any() for t in cf.gated_ffn_backward(h, x, w, w, h, h))


def test_captured_float16_gradients_follow_new_magnitudes():
    """The scale of an fp16 call is found by every replay anew."""
    import cudnn_frontend_b200 as cf

    gen = torch.Generator(device="cuda").manual_seed(22)
    m, k, n = 130, 256, 384
    x, w, u = rows(gen, m, k, FP16, 0, 30.0), rows(gen, n, k, FP16, 0, 30.0), rows(gen, n, k, FP16, 0, 30.0)
    z = rows(gen, m, n, FP16, 0, 2.0)
    dy, dh = torch.zeros((m, n), device="cuda"), torch.zeros((m, n), dtype=FP16, device="cuda")

    def step():
        return (*cf.linear_backward(dy, x, w, preact=z, act_func="silu", bias_grad=True), *cf.gated_ffn_backward(dh, x, w, u, z, z))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for size in (1e-6, 1.0, 1e-9, 0.0, 1e-3):
        dy.copy_(size * torch.randn((m, n), device="cuda", generator=gen))
        dh.copy_(dy)
        graph.replay()
        want = step()
        assert all(torch.equal(a, b) and torch.isfinite(a).all() for a, b in zip(out, want))
        assert bool(want[1].any()) == (size > 0)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("m,k,n", [(40, 64, 96), (2049, 264, 1290), (4096, 512, 2304)])
def test_gradients_of_unlike_alignment(m, k, n, gated):
    """dx and the weights' gradients need no alignment: where one of them has none, each equals what aligned memory gets.  (Both
    products may share a launch, whose blocks leave through shared memory by bulk copies, or row by row.)"""
    import ctypes

    import cudnn_frontend_b200 as cf
    from cudnn_frontend_b200 import _lib

    gen = torch.Generator(device="cuda").manual_seed(23)
    x, w, u = rows(gen, m, k, BF16), rows(gen, n, k, BF16, scale=k**-0.5), rows(gen, n, k, BF16, scale=k**-0.5)
    dy, gate, up = rows(gen, m, n, BF16, 6), rows(gen, m, n, BF16, 6), rows(gen, m, n, BF16, 6)
    want = cf.gated_ffn_backward(dy, x, w, u, gate, up) if gated else cf.linear_backward(dy, x, w)[:2]
    lib, act = _lib.load(), _lib.ACT_SWIGLU if gated else _lib.ACT_NONE
    work = torch.empty((lib.b200moe_dense_workspace_bytes(m, n, int(gated)),), dtype=torch.uint8, device="cuda")
    for odd in range(1, 1 << len(want)):  # which outputs start between two 16-byte boundaries
        outs = [torch.full((t.numel() + 8,), 3.0, dtype=BF16, device="cuda") for t in want]
        at = [3 * (odd >> i & 1) for i in range(len(want))]
        args = dict(x=x.data_ptr(), w0=w.data_ptr(), dy=dy.data_ptr(), workspace=work.data_ptr(), workspace_bytes=work.numel(), m=m, n=n, k=k, ld_x=k, ld_w0=k,
                    ld_dy=n + 6, act=act, **dict(zip(("dx", "dw0", "dw1"), (o.data_ptr() + 2 * a for o, a in zip(outs, at)))))  # fmt: skip
        if gated:
            args |= dict(w1=u.data_ptr(), ld_w1=k, pre0=gate.data_ptr(), pre1=up.data_ptr(), ld_pre0=n + 6, ld_pre1=n + 6)
        fn = lib.b200moe_gated_ffn_backward if gated else lib.b200moe_linear_backward
        _lib.check(fn(ctypes.byref(_lib.DenseArgs(**args)), torch.cuda.current_stream().cuda_stream))
        for o, a, t in zip(outs, at, want):
            assert torch.equal(o[a : a + t.numel()].view(t.shape), t)
            assert (o[:a] == 3).all() and (o[a + t.numel() :] == 3).all()


def dense_call(form, m, k, n, gen):
    """A call of a C entry point on fresh inputs: (function, arguments, outputs, what the outputs have to be)."""
    import cudnn_frontend_b200 as cf
    from cudnn_frontend_b200 import _lib

    lib = _lib.load()
    x, w, u = rows(gen, m, k, BF16), rows(gen, n, k, BF16, scale=k**-0.5), rows(gen, n, k, BF16, scale=k**-0.5)
    args = dict(x=x.data_ptr(), w0=w.data_ptr(), m=m, n=n, k=k, ld_x=k, ld_w0=k, act=_lib.ACT_NONE)
    if form == "linear":
        want = [cf.linear(x, w)]
    elif form == "float32":
        want, args = [cf.linear(x, w, out_dtype=torch.float32)], args | dict(y_dtype=_lib.DTYPE_F32)
    elif form == "gated":
        want, args = list(cf.gated_ffn(x, w, u, return_preact=True)), args | dict(w1=u.data_ptr(), ld_w1=k, act=_lib.ACT_SWIGLU)
    else:
        dy = rows(gen, m, n, BF16, 8)
        want, work = list(cf.linear_backward(dy, x, w)[:2]), torch.empty((lib.b200moe_dense_workspace_bytes(m, n, 0),), dtype=torch.uint8, device="cuda")
        args |= dict(dy=dy.data_ptr(), ld_dy=n + 8, workspace=work.data_ptr(), workspace_bytes=work.numel())
        x = (x, dy, work)
    outs = [torch.full_like(t, 3.0) for t in want]
    names = ("dx", "dw0") if form == "backward" else ("y", "pre0", "pre1")
    args |= dict(zip(names, (o.data_ptr() for o in outs)))
    if form != "backward":
        args |= dict(ld_y=n, ld_pre0=n, ld_pre1=n)
    fn = {"gated": lib.b200moe_gated_ffn, "backward": lib.b200moe_linear_backward}.get(form, lib.b200moe_linear)
    return fn, args, outs, want, (x, w, u)


# one CTA to a tile and several, one stage of the reduction and many more than the ring holds, and the kernel of CTA pairs
WAITS = [(5, 64, 200), (40, 512, 300), (300, 4096, 520), (3, 8192, 256), (2048, 256, 2048), (2304, 2048, 2048)]


@pytest.mark.parametrize("form", ["linear", "float32", "gated", "backward"])
@pytest.mark.parametrize("m,k,n", WAITS)
def test_expired_waits_leave_nothing_in_flight(m, k, n, form):
    """A launch whose operand B never arrives ends after its wait limit, whether its producers had more to issue or not, and what it had
    in flight is no part of the launch behind it on the same stream."""
    import ctypes

    from cudnn_frontend_b200 import _lib, ops

    gen = torch.Generator(device="cuda").manual_seed(24)
    fn, args, outs, want, _ = dense_call(form, m, k, n, gen)
    torch.cuda.synchronize()
    assert ops.device_status(clear=True) == 0
    stream = torch.cuda.current_stream().cuda_stream
    assert fn(ctypes.byref(_lib.DenseArgs(flags=_lib.FLAG_TEST_SKIP_B_LOADS, wait_limit_ms=20, **args)), stream) == 0
    assert fn(ctypes.byref(_lib.DenseArgs(**args)), stream) == 0
    torch.cuda.synchronize()
    assert ops.device_status(clear=True) in (401, 402, 403, 411, 412, 413, 414)
    assert all(torch.equal(a, b) for a, b in zip(outs, want))
    assert ops.device_status(clear=True) == 0


@pytest.mark.parametrize("form", ["linear", "float32", "gated", "backward"])
@pytest.mark.parametrize("m,k,n", WAITS)
def test_expired_waits_store_nothing(m, k, n, form):
    """Where sums are missing, outputs stay as they were, also where CTAs exchange partial sums or gate and up meet in shared memory."""
    import ctypes

    from cudnn_frontend_b200 import _lib, ops

    gen = torch.Generator(device="cuda").manual_seed(25)
    fn, args, outs, want, _ = dense_call(form, m, k, n, gen)
    torch.cuda.synchronize()
    assert ops.device_status(clear=True) == 0
    stream = torch.cuda.current_stream().cuda_stream
    assert fn(ctypes.byref(_lib.DenseArgs(flags=_lib.FLAG_TEST_SKIP_B_LOADS, wait_limit_ms=20, **args)), stream) == 0
    torch.cuda.synchronize()
    assert ops.device_status(clear=True) in (401, 402, 403, 411, 412, 413, 414)
    assert all((t == 3.0).all() for t in outs)
    assert fn(ctypes.byref(_lib.DenseArgs(**args)), stream) == 0
    torch.cuda.synchronize()
    assert ops.device_status(clear=True) == 0
    assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_float16_gated_workspace_without_the_scale_is_refused():
    """The size that bf16 needs is 256 bytes short in fp16: refused with the size, nothing written."""
    import ctypes

    from cudnn_frontend_b200 import _lib

    lib, (m, k, n) = _lib.load(), (16, 64, 32)
    gen = torch.Generator(device="cuda").manual_seed(26)
    x, w, t = rows(gen, m, k, FP16), rows(gen, n, k, FP16), rows(gen, m, n, FP16)
    dx = torch.full_like(x, 3.0)
    need = lib.b200moe_dense_workspace_bytes(m, n, 1 | _lib.DENSE_WORKSPACE_F16)
    work = torch.empty((need,), dtype=torch.uint8, device="cuda")
    for size, code in ((lib.b200moe_dense_workspace_bytes(m, n, 1), _lib.E_WORKSPACE), (need, 0)):
        args = _lib.DenseArgs(x=x.data_ptr(), w0=w.data_ptr(), w1=w.data_ptr(), dy=t.data_ptr(), pre0=t.data_ptr(), pre1=t.data_ptr(), dx=dx.data_ptr(),
                              workspace=work.data_ptr(), workspace_bytes=size, m=m, n=n, k=k, ld_x=k, ld_w0=k, ld_w1=k, ld_dy=n, ld_pre0=n, ld_pre1=n,
                              dtype=_lib.DTYPE_F16, act=_lib.ACT_SWIGLU)  # fmt: skip
        assert lib.b200moe_gated_ffn_backward(ctypes.byref(args), torch.cuda.current_stream().cuda_stream) == code
        assert str(need) in _lib.last_error() if code else True
        assert bool((dx == 3.0).all()) == (code != 0)
