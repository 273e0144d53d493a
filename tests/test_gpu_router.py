"""The router's gate against a plain float64 implementation: the choice exactly, weights and gradients to float32 rounding.

Tolerance of a float32 result: the exponentials, logarithms and quotients of the formulas are each within 2 steps (2^-23 relative),
their argument differences within 2^-24 of the arguments (at most 2^-24 * 100 absolute here, which is relative in the exponential), sums of up
to 1024 positive terms within 10 * 2^-24 (a tree): 1e-5 relative covers all of it for the values used here; gradients are differences
of such terms and are bounded by the same share of the terms' sizes.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def plain(logits, topk, score, normalize, bias, scale, dw=None):
    wide = logits.double().requires_grad_()
    on = wide > -math.inf
    if score == "sigmoid":
        s = torch.sigmoid(wide)
    else:
        s = torch.softmax(torch.where(on.any(1, keepdim=True), wide, torch.zeros_like(wide)), 1)
    order = (wide if bias is None else s + bias.double()).detach().masked_fill(~on, -math.inf)
    top, ids = torch.sort(order, dim=1, descending=True, stable=True)
    top, ids = top[:, :topk], ids[:, :topk]
    there = top > -math.inf
    if score == "sigmoid" and normalize:
        a = torch.nn.functional.logsigmoid(wide).gather(1, ids)
        w = torch.softmax(torch.where(there, a, torch.full_like(a, -1e300)), 1)
    elif normalize:
        a = wide.gather(1, ids)
        w = torch.softmax(torch.where(there, a, torch.full_like(a, -1e300)), 1)
    else:
        w = s.gather(1, ids)
    w = scale * torch.where(there, w, torch.zeros_like(w))
    out = [w.detach(), ids.masked_fill(~there, -1).to(torch.int32)]
    if dw is not None:
        (g,) = torch.autograd.grad(w, wide, dw.double())
        out.append(torch.nan_to_num(g))
    return out


CASES = [(1, 1, 1), (3, 4, 2), (64, 8, 2), (5, 33, 7), (130, 64, 6), (257, 60, 4), (100, 256, 8), (9, 300, 16), (33, 512, 32), (17, 1024, 1), (2000, 128, 8), (8195, 60, 8), (9000, 256, 3), (8193, 8, 2)]


@pytest.mark.parametrize("t,e,k", CASES)
@pytest.mark.parametrize("score,normalize", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
@pytest.mark.parametrize("dt,bias,masked,pad", [(torch.float32, False, False, 0), (torch.float32, True, True, 5), (torch.bfloat16, False, True, 0), (torch.float16, True, False, 3)])
def test_router(t, e, k, score, normalize, dt, bias, masked, pad):
    import cudnn_frontend_b200 as cf

    gen = torch.Generator(device="cuda").manual_seed(t + e + k)
    wide = 2.0 * torch.randn((t, e + pad), device="cuda", generator=gen)
    if masked:
        wide[torch.rand((t, e + pad), device="cuda", generator=gen) < 0.4] = -math.inf
        wide[::5] = -math.inf  # rows with no expert at all
    logits = wide.to(dt)[:, :e]
    b = 0.1 * torch.randn((e,), device="cuda", generator=gen) if bias else None
    dw = torch.randn((t, k), device="cuda", generator=gen)
    weights, ids = cf.router_topk(logits, k, score_func=score, normalize=normalize, bias=b, scale=1.5)
    grad = cf.router_topk_backward(dw, logits, ids, score_func=score, normalize=normalize, scale=1.5)
    w64, i64, g64 = plain(logits, k, score, normalize, b, 1.5, dw)
    assert torch.equal(ids, i64)
    assert ((weights.double() - w64).abs() <= 1e-5 * w64 + 1e-30).all()
    assert grad.dtype == dt and torch.isfinite(grad).all()
    terms = (w64 * dw.double().abs()).sum(1, keepdim=True) / min(1.5, 1.0) + 1e-30
    size = torch.zeros_like(g64).scatter(1, ids.clamp(min=0).long(), (w64 * dw.double().abs()).masked_fill(ids < 0, 0.0))
    share = 1.0 if score == "softmax" and not normalize else torch.zeros_like(g64).scatter(1, ids.clamp(min=0).long(), w64.masked_fill(ids < 0, 0.0))
    half = torch.finfo(dt).eps / 2
    tol = 1e-5 * (size + share * terms) + half * g64.abs() + (torch.finfo(dt).tiny * torch.finfo(dt).eps if dt != torch.float32 else 1e-30)
    assert ((grad.double() - g64).abs() <= tol).all()
    outside = torch.ones_like(g64, dtype=torch.bool).scatter(1, ids.clamp(min=0).long(), ids < 0)
    if normalize or score == "sigmoid":
        assert not grad[outside & (g64 == 0)].any()


def test_ties_go_to_the_lowest_index():
    import cudnn_frontend_b200 as cf

    logits = torch.zeros((40, 96), device="cuda")
    logits[1::2] = -0.0
    logits[:, 50] = 1.0
    for b in (None, torch.zeros(96, device="cuda")):
        for score in ("softmax", "sigmoid"):
            _, ids = cf.router_topk(logits, 4, score_func=score, bias=b)
            assert ids.tolist() == [[50, 0, 1, 2]] * 40
    # signed zeros of both kinds in one row are equal
    logits = torch.tensor([[-0.0, 0.0, -0.0, 0.0]], device="cuda")
    assert cf.router_topk(logits, 3)[1].tolist() == [[0, 1, 2]]


def test_far_sigmoids_keep_their_ratio():
    """Scores that underflow in float32 still give weights: the quotient is formed from the logarithms."""
    import cudnn_frontend_b200 as cf

    logits = torch.tensor([[-200.0, -201.0, -300.0, -500.0]], device="cuda")
    w, ids = cf.router_topk(logits, 2, score_func="sigmoid")
    assert ids.tolist() == [[0, 1]]
    want = torch.softmax(torch.tensor([-200.0, -201.0], dtype=torch.float64), 0)
    assert (w[0].cpu().double() - want).abs().max() < 2e-5  # one float32 step of the arguments, 2^-16


def test_biased_choice_where_float32_cannot_decide():
    """Scores that differ by less than a float32 step, many equal ones (more candidates than a warp has lanes), saturated
    sigmoids, biases far above the scores and infinite ones: the choice is that of float64."""
    import cudnn_frontend_b200 as cf

    gen = torch.Generator(device="cuda").manual_seed(2)
    e, k = 200, 8
    rows = [torch.full((e,), 0.3, device="cuda"), 0.3 + 1e-7 * torch.randn((e,), device="cuda", generator=gen),
            20 + 3 * torch.rand((e,), device="cuda", generator=gen), torch.randn((e,), device="cuda", generator=gen)]  # fmt: skip
    logits = torch.stack(rows)
    logits[3, 17] = float("inf")
    small = 1e-7 * torch.randn((e,), device="cuda", generator=gen)
    far = 1e4 * torch.randn((e,), device="cuda", generator=gen)
    off = torch.zeros((e,), device="cuda")
    off[:30], off[40] = -math.inf, math.inf
    for bias in (torch.zeros((e,), device="cuda"), small, far, off, torch.full((e,), -math.inf, device="cuda")):
        for score in ("sigmoid", "softmax"):
            l = logits if score == "sigmoid" else logits[:3]  # (softmax of +inf is NaN)
            _, ids = cf.router_topk(l, k, score_func=score, bias=bias)
            s = torch.sigmoid(l.double()) if score == "sigmoid" else torch.softmax(l.double(), 1)
            top, want = torch.sort(s + bias.double(), dim=1, descending=True, stable=True)
            want = torch.where(top[:, :k] > -math.inf, want[:, :k], -1)
            if score == "sigmoid":
                assert torch.equal(ids.long(), want)
            else:  # float64's own last bits may differ between two sums over a row: the scores agree, and so does the set of clear ones
                got = torch.where(ids >= 0, (s + bias.double()).gather(1, ids.clamp(min=0).long()), -math.inf)
                assert torch.allclose(got, top[:, :k], rtol=1e-14, atol=1e-15)


def test_nan_stays_in_its_row():
    import cudnn_frontend_b200 as cf

    logits = torch.randn((6, 40), device="cuda")
    clean = cf.router_topk(logits, 3)
    logits[2, 11] = float("nan")
    w, ids = cf.router_topk(logits, 3)
    assert int(ids[2, 0]) == 11 and torch.isnan(w[2]).all()
    keep = [0, 1, 3, 4, 5]
    assert torch.equal(w[keep], clean[0][keep]) and torch.equal(ids[keep], clean[1][keep])


def test_gradient_sums_repeated_and_skips_missing_experts():
    import cudnn_frontend_b200 as cf

    logits = torch.randn((3, 20), device="cuda")
    dw = torch.randn((3, 3), device="cuda")
    ids = torch.tensor([[4, 4, 7], [-1, 3, 25], [-1, -1, -1]], dtype=torch.int32, device="cuda")
    g = cf.router_topk_backward(dw, logits, ids, score_func="sigmoid", normalize=False)
    s = torch.sigmoid(logits.double())
    d = s * (1 - s)
    want = torch.zeros_like(d)
    want[0, 4] = d[0, 4] * (dw[0, 0].double() + dw[0, 1].double())
    want[0, 7] = d[0, 7] * dw[0, 2].double()
    want[1, 3] = d[1, 3] * dw[1, 1].double()
    assert ((g.double() - want).abs() <= 1e-6).all() and not g[want == 0].any()


def test_no_tokens_and_other_streams():
    import cudnn_frontend_b200 as cf

    w, ids = cf.router_topk(torch.empty((0, 16), device="cuda"), 2)
    assert w.shape == ids.shape == (0, 2)
    assert cf.router_topk_backward(w, torch.empty((0, 16), device="cuda"), ids).shape == (0, 16)
    logits = torch.randn((500, 64), device="cuda")
    want = cf.router_topk(logits, 6)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got = cf.router_topk(logits, 6, stream=s), cf.router_topk(logits, 6, stream=s.cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))


def test_refusals():
    import cudnn_frontend_b200 as cf

    l = torch.randn((4, 16), device="cuda")
    w, ids = cf.router_topk(l, 2)
    with pytest.raises(NotImplementedError):
        cf.router_topk(l.double(), 2)
    for call in (
        lambda: cf.router_topk(l, 0),
        lambda: cf.router_topk(l, 17),
        lambda: cf.router_topk(torch.randn((2, 64), device="cuda"), 33),
        lambda: cf.router_topk(torch.randn((2, 1025), device="cuda"), 2),
        lambda: cf.router_topk(l, 2, score_func="relu"),
        lambda: cf.router_topk(l, 2, bias=torch.zeros(15, device="cuda")),
        lambda: cf.router_topk(l, 2, bias=torch.zeros(16, device="cuda", dtype=torch.float16)),
        lambda: cf.router_topk(l.t(), 2),
        lambda: cf.router_topk(l[:1].expand(4, 16), 2),
        lambda: cf.router_topk(l.cpu(), 2),
        lambda: cf.router_topk_backward(w, l, ids.long()),
        lambda: cf.router_topk_backward(w.half(), l, ids),
        lambda: cf.router_topk_backward(w[:3], l, ids),
    ):
        with pytest.raises(ValueError):
            call()


def test_gate_feeds_the_expert_path():
    """The run of a whole MoE layer on one GPU: router projection in float32, gate, routing, quantised experts, combine, and the
    shared expert whose projection adds the combined rows.  The parts that are new are checked on what they were given."""
    import cudnn_frontend_b200 as cf
    from cudnn_frontend_b200 import moe, ops

    gen = torch.Generator(device="cuda").manual_seed(9)
    t, h, inter, e, k = 200, 512, 256, 8, 2
    bf = torch.bfloat16
    r = lambda *s, f=1.0: (f * torch.randn(s, device="cuda", generator=gen)).to(bf)  # noqa: E731
    x, wr = r(t, h), r(e, h, f=h**-0.5)
    logits = cf.linear(x, wr, out_dtype=torch.float32)
    weights, ids = cf.router_topk(logits, k)
    assert torch.equal(ids, plain(logits, k, "softmax", True, None, 1.0)[1])
    counts, offs, dst = cf.route(ids, e, 128)
    m_rows = int(offs[-1])
    a = torch.zeros((m_rows, h), dtype=bf, device="cuda")
    prob = torch.zeros((m_rows,), device="cuda")
    cf.scatter_rows(x, dst, a, k, weights.view(-1), prob)
    w1 = [moe.interleave_gate_up(r(inter, h, f=h**-0.5), r(inter, h, f=h**-0.5)) for _ in range(e)]
    w2 = [r(h, inter, f=inter**-0.5) for _ in range(e)]

    def quantised(ws, n, kk):
        q = [cf.quantize_mxfp8(w) for w in ws]
        sf = ops.empty_sf(n, kk, e)
        flat = torch.as_strided(sf.view(torch.uint8), (sf.numel(),), (1,))
        flat.copy_(torch.cat([torch.as_strided(s.view(torch.uint8), (s.numel(),), (1,)) for _, s in q]))
        return torch.stack([w for w, _ in q]).permute(1, 2, 0), sf

    b1, sf1 = quantised(w1, 2 * inter, h)
    b2, sf2 = quantised(w2, h, inter)
    qa, sfa = cf.quantize_mxfp8(a)
    alpha = torch.ones(e, device="cuda")
    one = torch.ones(1, device="cuda")
    f1 = cf.grouped_gemm_swiglu_wrapper_sm100(qa.view(m_rows, h, 1), b1, sfa, sf1, offs, alpha, norm_const_tensor=one,
                                              prob_tensor=torch.ones((m_rows, 1, 1), device="cuda"), d_dtype=torch.float8_e4m3fn, sf_vec_size=32, m_aligned=128)  # fmt: skip
    f2 = cf.grouped_gemm_quant_wrapper_sm100(f1["d_tensor"], f1["sfd_row_tensor"], offs, alpha, b_tensor=b2, sfb_tensor=sf2,
                                             prob_tensor=prob.view(m_rows, 1, 1), sf_vec_size=32, m_aligned=128)  # fmt: skip
    routed = cf.combine_rows(f2["d_tensor"][:, :, 0].contiguous(), dst, t, k)
    wg, wu, wd = r(inter, h, f=h**-0.5), r(inter, h, f=h**-0.5), r(h, inter, f=inter**-0.5)
    hidden = cf.gated_ffn(x, wg, wu)
    y = cf.linear(hidden, wd, residual=routed)
    assert ops.device_status(clear=True) == 0
    # the routed part against float64 experts: MXFP8 keeps 3 bits of mantissa, 2^-4 relative per value at worst in four operands
    want = torch.zeros((t, h), dtype=torch.float64, device="cuda")
    for j in range(e):
        g, u = (w1[j].view(inter // 32, 2, 32, h)[:, q].reshape(inter, h).double() for q in (0, 1))
        z = x.double() @ g.t()
        out = (z * torch.sigmoid(z) * (x.double() @ u.t())) @ w2[j].double().t()
        want += out * torch.where(ids == j, weights.double(), 0.0).sum(1, keepdim=True)
    assert float((routed.double() - want).norm() / want.norm()) <= 4 * 2.0**-4
    # the shared expert on the rows it was given: one rounding of y, and of hidden through the product (2-norm)
    z = x.double() @ wg.double().t()
    full = routed.double() + (z * torch.sigmoid(z) * (x.double() @ wu.double().t())) @ wd.double().t()
    assert float((y.double() - full).norm() / full.norm()) <= torch.finfo(bf).eps
    # and back: the gate's gradient reaches the router's weights
    dlogits = cf.router_topk_backward(torch.randn((t, k), device="cuda", generator=gen), logits, ids)
    dx, dwr, _ = cf.linear_backward(dlogits, x, wr)
    assert rel(dwr, dlogits.double().t() @ x.double()) <= torch.finfo(bf).eps and rel(dx, dlogits.double() @ wr.double()) <= torch.finfo(bf).eps


def rel(got, want):
    return float((got.double() - want).norm() / want.norm())


def test_numbers_beyond_32_bits_are_refused():
    """2^32 + 2 choices are refused before anything of that size is allocated; the C entry point would see 2."""
    import cudnn_frontend_b200 as cf

    logits = torch.zeros((4, 8), device="cuda")
    held = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    wide = torch.zeros((1, 1), device="cuda").as_strided((0, 2**32 + 8), (2**32 + 8, 1))  # (no rows: nothing to allocate)
    for call in (
        lambda: cf.router_topk(logits, 2**32 + 2),
        lambda: cf.router_topk(wide, 2),
        lambda: cf.router_topk_backward(logits[:0, :2], wide, torch.zeros((0, 2), dtype=torch.int32, device="cuda")),
    ):
        with pytest.raises(ValueError):
            call()
    assert torch.cuda.max_memory_allocated() <= held + 4096
