"""The block around a layer of experts: its operators' functions with their first and second gradients, and the block as it trains and serves."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F32 = torch.bfloat16, torch.float32
u = 2.0 ** -24


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(g, *shape, dtype=F32):
    return torch.randn(shape, device=DEV, generator=g).to(dtype)


def first_and_second(f, operands, seed):
    """f's outputs, their gradient along given values, and that gradient's own along others, for every operand and the given values."""
    g = gen(seed)
    leaves = [t.detach().clone().requires_grad_() for t in operands]
    outs = f(*leaves)
    along = [randn(g, *o.shape).to(o.dtype).requires_grad_() for o in outs]
    first = torch.autograd.grad(outs, leaves, along, create_graph=True)
    second = torch.autograd.grad(sum((d * randn(g, *d.shape).to(d.dtype)).sum() for d in first), [*leaves, *along], allow_unused=True)
    plain = torch.autograd.grad(f(*leaves), leaves, along)                 # (with no graph of its own: the operators' gradients)
    return [t.detach() for t in (*outs, *first)], [torch.zeros_like(t) if d is None else d for t, d in zip([*leaves, *along], second)], plain


def alike(f, plain, operands, seed, tolerance):
    """fp32 against 64 bits, by the norms: sums of at most 64 values in a few steps of relative error 2^-22 each, `tolerance` of what they are made of."""
    got, want = first_and_second(f, operands, seed), first_and_second(plain, [t.double() for t in operands], seed)
    for a, b in zip(got, want):
        for x, y in zip(a, b):
            assert x.dtype == F32 and (x.double() - y).norm() <= tolerance * max(float(y.norm()), 1.0)


def test_gradients_of_the_norm():
    from mm_rs_with_catlass_amd.experts import rms_norm
    g = gen(1)
    x, w, r = randn(g, 5, 48), 1 + 0.2 * randn(g, 48), randn(g, 5, 48)

    def plain(a, b, c=None):
        s = a if c is None else a + c
        y = s * (s.square().mean(1, keepdim=True) + 1e-3).rsqrt() * b
        return (y,) if c is None else (y, s)
    alike(lambda a, b: (rms_norm(a, b, eps=1e-3),), plain, [x, w], 2, 2.0 ** -16)
    alike(lambda a, b, c: rms_norm(a, b, c, eps=1e-3), plain, [x, w, r], 3, 2.0 ** -16)
    # the sum alone: its gradient goes through, the weight has none
    x, w, r = (t.clone().requires_grad_() for t in (x, w, r))
    dx, dr, dw = torch.autograd.grad(rms_norm(x, w, r)[1].sum(), (x, r, w), allow_unused=True)
    assert (dx == 1).all() and (dr == 1).all() and dw is None


def test_gradients_of_a_residual_stream_in_32_bits():
    from mm_rs_with_catlass_amd import ops
    from mm_rs_with_catlass_amd.experts import rms_norm
    g = gen(4)
    x, w, r, dy, ds = randn(g, 20, 300, dtype=BF16), randn(g, 300), randn(g, 20, 300), randn(g, 20, 300, dtype=BF16), randn(g, 20, 300)
    leaves = [t.requires_grad_() for t in (x, w, r)]
    y, s = rms_norm(*leaves, eps=1e-5)
    dx, dw, dr = torch.autograd.grad((y, s), leaves, (dy, ds))
    want = ops.rms_norm_backward(dy, s.detach(), w.detach(), ds, eps=1e-5)
    assert torch.equal(dr, want[0]) and torch.equal(dx, want[0].to(BF16)) and torch.equal(dw, want[1])


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [False, True])
def test_gradients_of_the_router(score, renormalize):
    from mm_rs_with_catlass_amd import ops
    from mm_rs_with_catlass_amd.experts import route
    logits = randn(gen(5), 9, 12)
    logits[3, 4:] = -20.0
    choice, _ = ops.route(logits, 4, score=score)

    def plain(v):
        p = (torch.softmax(v, 1) if score == "softmax" else torch.sigmoid(v)).gather(1, choice.long())
        return ((p / p.sum(1, keepdim=True) if renormalize else p) * 1.5,)
    alike(lambda v: (route(v, 4, score=score, renormalize=renormalize, scale=1.5)[1],), plain, [logits], 6, 2.0 ** -16)


def test_gradients_of_rows_there_and_back():
    from mm_rs_with_catlass_amd.experts import Gather, Spread
    g = gen(7)
    back = torch.randperm(24, device=DEV, generator=g).to(torch.int32).view(8, 3)
    x, y, share = randn(g, 8, 40), randn(g, 24, 40), randn(g, 8, 3)
    at = back.long()
    place = torch.argsort(at.view(-1)) // 3
    alike(lambda a: (Spread.apply(a, back),), lambda a: (a[place],), [x], 8, 2.0 ** -18)
    alike(lambda a: (Gather.apply(a, back, None),), lambda a: (a[at].sum(1),), [y], 9, 2.0 ** -18)
    alike(lambda a, s: (Gather.apply(a, back, s),), lambda a, s: ((a[at] * s[:, :, None]).sum(1),), [y, share], 10, 2.0 ** -18)


class Layer:
    def __init__(self, seed, tokens, hidden=256, inter=128, count=8, dtype=BF16, wide=True):
        g = gen(seed)
        self.x, self.residual = randn(g, tokens, hidden, dtype=dtype), randn(g, tokens, hidden, dtype=F32 if wide else dtype)
        self.norm = (1 + 0.1 * randn(g, hidden)).to(dtype)
        self.router = randn(g, count, hidden) / hidden ** 0.5
        self.w1, self.w2 = (randn(g, count, 2 * inter, hidden) / hidden ** 0.5).to(dtype), (randn(g, count, hidden, inter) / inter ** 0.5).to(dtype)
        self.shared = [(randn(g, 2 * inter, hidden) / hidden ** 0.5).to(dtype), (randn(g, hidden, inter) / inter ** 0.5).to(dtype)]
        self.bias = 0.1 * randn(g, count)

    def weights(self):
        return self.norm, self.router, self.w1, self.w2

    def operands(self):
        return self.x, self.residual, *self.weights()


HOW = [{}, dict(score="sigmoid", groups=4, top_groups=2, group_top=2, scale=2.5), dict(renormalize=False)]


@pytest.mark.parametrize("how", HOW)
@pytest.mark.parametrize("tokens", [0, 1, 90, 700])
@pytest.mark.parametrize("dtype,wide", [(BF16, True), (torch.float16, False)])
def test_block_is_its_operators(how, tokens, dtype, wide):
    """The block's results and gradients are those of the operators called one after the other, bit for bit."""
    from mm_rs_with_catlass_amd import ops
    from mm_rs_with_catlass_amd.experts import block, experts
    e = Layer(20, tokens, dtype=dtype, wide=wide)
    bias = e.bias if how.get("score") == "sigmoid" else None
    leaves = [t.detach().clone().requires_grad_() for t in e.operands()]
    out, s = block(*leaves, 2, bias=bias, **how)
    dout, ds = randn(gen(21), *out.shape, dtype=dtype), randn(gen(22), *s.shape).to(s.dtype)
    grads = torch.autograd.grad((out, s), leaves, (dout, ds))

    y, kept = ops.rms_norm(e.x, e.norm, e.residual)
    logits = y.float() @ e.router.t()
    choice, share = ops.route(logits, 2, bias=bias, **how)
    inner = [t.detach().clone().requires_grad_() for t in (y, e.w1, e.w2, share)]
    want = experts(*inner[:3], choice, inner[3])
    assert torch.equal(out, want) and torch.equal(s, kept)
    dy, dw1, dw2, dshare = torch.autograd.grad(want, inner, dout)
    dlogits = ops.route_backward(dshare, logits, choice, **{k: v for k, v in how.items() if k in ("score", "renormalize", "scale")})
    dy = dy + (dlogits @ e.router).to(dtype)
    dsum, dnorm = ops.rms_norm_backward(dy, kept, e.norm, ds)
    for got, w in zip(grads, (dsum.to(dtype), dsum, dnorm, dlogits.t() @ y.float(), dw1, dw2)):
        assert got.dtype == w.dtype and (torch.equal(got, w) or (got.shape == e.router.shape and (got - w).abs().max() <= 1e-4 * w.abs().max()))
    if tokens == 0:
        assert not any(g.any() for g in grads)


@pytest.mark.parametrize("how", HOW)
@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("tokens", [0, 1, 90, 700])
def test_served_block_is_its_operators(how, shared, tokens):
    from mm_rs_with_catlass_amd import ops
    from mm_rs_with_catlass_amd.experts import ServedBlock, ServedExperts
    e = Layer(23, tokens)
    extra = e.shared if shared else []
    out, s = ServedBlock(*e.weights(), 2, *extra, **how)(e.x, e.residual)
    y, kept = ops.rms_norm(e.x, e.norm, e.residual)
    choice, share = ops.route(y.float() @ e.router.t().contiguous(), 2, **how)
    q, scale, _ = ops.rms_norm_fp8(kept, e.norm.float(), keep=True)     # (the sum's norm: the same values before their rounding)
    served = ServedExperts(e.w1, e.w2, *extra)
    assert torch.equal(s, kept) and torch.equal(out, served(y, choice, share, codes=(q, scale)))
    # codes of the 16-bit rows in the place of codes of the norm itself: 2^-8 of a value more, beside an e4m3 rounding of 2^-4 at most
    late = served(y, choice, share)
    assert (out.double() - late.double()).norm() <= 2 * 0.105 * late.double().norm()


@pytest.mark.parametrize("served", [False, True])
def test_the_block_in_a_captured_graph(served):
    from mm_rs_with_catlass_amd.experts import ServedBlock, block
    e = Layer(24, 130)
    whole = ServedBlock(*e.weights(), 2, *e.shared, bias=e.bias, score="sigmoid")

    def call():
        return whole(e.x, e.residual) if served else block(*e.operands(), 2, bias=e.bias, score="sigmoid")
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for i in range(6):
        other = Layer(30 + i, 130)
        e.x.copy_(other.x)
        e.residual.copy_(other.residual)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, call())), i


def test_a_training_step_in_a_captured_graph():
    from mm_rs_with_catlass_amd.experts import block
    e = Layer(25, 200)
    leaves = [t.requires_grad_() for t in e.operands()]
    dout = randn(gen(26), 200, 256, dtype=BF16)

    def call():
        out, s = block(*leaves, 2)
        return (out.detach(), *torch.autograd.grad((out, s), leaves, (dout, torch.ones_like(s))))
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for i in range(5):
        other = Layer(40 + i, 200)
        with torch.no_grad():
            e.x.copy_(other.x)
            e.residual.copy_(other.residual)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, call())), i


def test_experts_past_what_the_operators_take():
    """More experts than the sort takes, or more choices of a token: the layer's rows go through torch, with the same results."""
    from mm_rs_with_catlass_amd import experts as E
    g = gen(27)
    x, w1, w2 = randn(g, 40, 64, dtype=BF16), randn(g, 1100, 32, 64, dtype=BF16) / 8, randn(g, 1100, 64, 16, dtype=BF16) / 4
    choice, share = torch.randint(0, 60, (40, 3), device=DEV, generator=g), torch.rand((40, 3), device=DEV, generator=g)
    many, few = E.experts(x, w1, w2, choice, share), E.experts(x, w1[:60].contiguous(), w2[:60].contiguous(), choice, share)
    assert not E._Plan(choice, 1100).kernels and E._Plan(choice, 60).kernels
    assert ((many.double() - few.double()).abs() <= 4 * 2.0 ** -8 * few.double().abs().amax()).all()
    for dtype in (torch.int16, torch.uint8, torch.int32):
        assert torch.equal(E.experts(x, w1[:60].contiguous(), w2[:60].contiguous(), choice.to(dtype), share), few)
    wide = torch.randint(0, 60, (5, 70), device=DEV, generator=g)
    weights = torch.rand((5, 70), device=DEV, generator=g) / 70
    served = E.ServedExperts(w1[:60], w2[:60])
    halves = [served(x[:5], wide[:, i:i + 35], weights[:, i:i + 35]) for i in (0, 35)]
    assert not E._Plan(wide, 60).kernels
    assert ((served(x[:5], wide, weights).double() - sum(h.double() for h in halves)).abs() <= 4 * 2.0 ** -8 * sum(h.double().abs().amax() for h in halves)).all()


def test_gathers_make_the_gradients_that_are_wanted():
    """Rows are kept for the shares' gradient alone, and not read for the other; both as where both are wanted, first and second."""
    from mm_rs_with_catlass_amd.experts import Gather
    g = gen(40)
    back = torch.randperm(24, device=DEV, generator=g).to(torch.int32).view(8, 3)
    y, share, d = randn(g, 24, 40), randn(g, 8, 3), randn(g, 8, 40)
    a, s = y.clone().requires_grad_(), share.clone().requires_grad_()
    want = torch.autograd.grad(Gather.apply(a, back, s), (a, s), d)
    for graph in (False, True):
        out = Gather.apply(a, back, share)
        assert out.grad_fn.saved_tensors[0] is None
        assert torch.equal(torch.autograd.grad(out, a, d, create_graph=graph)[0], want[0])
        out = Gather.apply(y, back, s)
        got, = torch.autograd.grad(out, s, d, create_graph=graph)
        # (with a graph torch adds up the dot products of 40 values in another order)
        assert torch.equal(got, want[1]) if not graph else ((got - want[1]).abs() <= 2 * 40 * u * (d.abs()[:, None, :] * y.abs()[back.long()]).sum(2)).all()
    at = back.long()
    alike(lambda v: (Gather.apply(v, back, share),), lambda v: ((v[at] * share.to(v.dtype)[:, :, None]).sum(1),), [y], 41, 2.0 ** -18)
    alike(lambda v: (Gather.apply(y, back, v),), lambda v: ((y.to(v.dtype)[at] * v[:, :, None]).sum(1),), [share], 42, 2.0 ** -18)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [False, True])
def test_gradient_of_far_logits_with_a_graph_of_its_own(score, renormalize):
    """Chosen experts far below the others, or all far below zero: the gradient that keeps a graph is the operator's."""
    from mm_rs_with_catlass_amd.experts import route
    logits = randn(gen(30), 8, 12)
    logits[1] -= 120.0
    logits[2] -= 300.0
    logits[3, 4:] += 110.0
    logits[4] = -float("inf")
    logits[5, 2:] = -float("inf")
    logits[6, 1:] = torch.finfo(F32).min
    bias = torch.zeros(12, device=DEV)
    bias[4:] = -2.0                                 # (the far ones are chosen)
    d = randn(gen(31), 8, 4)
    grads = []
    for graph in (False, True):
        v = logits.clone().requires_grad_()
        _, share = route(v, 4, bias=bias, score=score, renormalize=renormalize)
        got, = torch.autograd.grad(share, v, d, create_graph=graph)
        grads.append(got.detach())
    # two evaluations in fp32 of w (g - sum w g): each within 110 half steps of max |g| times the shares' sum
    size = 4 * d.abs().amax(1, keepdim=True) if not renormalize else d.abs().amax(1, keepdim=True)
    assert grads[0].isfinite().all() and ((grads[0] - grads[1]).abs() <= 2 * 2 * 110 * u * size).all()
    if renormalize:
        assert grads[1][1:4].abs().amax(1).min() > 1e-3
