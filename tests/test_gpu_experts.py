"""The layer of experts that calls the grouped and e4m3 operators together, against the same layer in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}   # what a rounding to nearest moves a value by, relative, at most


class Near:
    """A value in 64 bits and how far, element by element, a computation of it in fewer bits can be off."""

    def __init__(self, v, e=None):
        self.v, self.e = v, torch.zeros_like(v) if e is None else e

    def rounded(self, dtype):
        # (below fp16's normal numbers: half of 2^-24)
        return Near(self.v, self.e + U[dtype] * (self.v.abs() + self.e) + 2.0 ** -25)

    def t(self):
        return Near(self.v.t(), self.e.t())

    def __matmul__(self, o):
        a, b = self.v.abs(), o.v.abs()
        size = (a + self.e) @ (b + o.e)
        # (sums in fp32, in any order: at most as many roundings of 2^-24 as there are addends)
        return Near(self.v @ o.v, a @ o.e + self.e @ b + self.e @ o.e + self.v.shape[1] * 2.0 ** -23 * size)

    def __mul__(self, o):
        return Near(self.v * o.v, self.v.abs() * o.e + self.e * o.v.abs() + self.e * o.e + 2.0 ** -21 * (self.v * o.v).abs())

    def __add__(self, o):
        return Near(self.v + o.v, self.e + o.e + 2.0 ** -22 * (self.v.abs() + o.v.abs()))

    def of(self, f, slope):   # |f'| <= slope; f itself is computed in fp32, to 2^-20 of its argument's size
        return Near(f(self.v), slope * self.e + 2.0 ** -20 * (f(self.v).abs() + self.v.abs()))

    def holds(self, got, name):
        off = (got.double().cpu() - self.v).abs() - self.e
        assert off.max() <= 0, "%s is off by %g more than its roundings explain" % (name, off.max())


def silu(v):
    return v * torch.sigmoid(v)


def silu_slope(v):
    s = torch.sigmoid(v)
    return s * (1 + v * (1 - s))


def layer(seed, tokens, hidden, inter, count, top, dtype, chosen=None):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(tokens, hidden, generator=g).to(dtype)
    w1 = (torch.randn(count, 2 * inter, hidden, generator=g) / hidden ** 0.5).to(dtype)
    w2 = (torch.randn(count, hidden, inter, generator=g) / inter ** 0.5).to(dtype)
    share, choice = torch.rand(tokens, chosen or count, generator=g).topk(top)
    return x, w1, w2, choice, share


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,hidden,inter,count,top,chosen", [(1, 64, 32, 4, 2, None), (37, 200, 72, 5, 2, 3), (130, 256, 136, 3, 1, None), (70, 66, 30, 8, 8, None)])
def test_forward_and_gradients(tokens, hidden, inter, count, top, chosen, dtype):
    from mm_rs_with_catlass_amd.experts import experts
    x, w1, w2, choice, share = layer(3, tokens, hidden, inter, count, top, dtype, chosen)
    dout = torch.randn(tokens, hidden, generator=torch.Generator().manual_seed(4)).to(dtype)
    dev = [t.cuda().requires_grad_() for t in (x, w1, w2, share)]
    out = experts(dev[0], dev[1], dev[2], choice.cuda(), dev[3])
    out.backward(dout.cuda())

    want_out, want_dx = Near(torch.zeros(tokens, hidden).double()), Near(torch.zeros(tokens, hidden).double())
    want_share = Near(torch.zeros(tokens, top).double())
    for e in range(count):
        at, which = (choice == e).nonzero(as_tuple=True)
        if at.numel() == 0:
            assert not dev[1].grad[e].any() and not dev[2].grad[e].any()
            continue
        xs, a1, a2, p, do = Near(x[at].double()), Near(w1[e].double()), Near(w2[e].double()), Near(share[at, which].double()[:, None]), Near(dout[at].double())
        h = (xs @ a1.t()).rounded(dtype)
        gate, up = Near(h.v[:, :inter], h.e[:, :inter]), Near(h.v[:, inter:], h.e[:, inter:])
        a = (gate.of(silu, 1.1) * up).rounded(dtype)
        y = (a @ a2.t()).rounded(dtype)
        part = p * y
        want_out.v[at] += part.v
        want_out.e[at] += part.e + 2.0 ** -21 * part.v.abs()
        dshare = do * y
        want_share.v[at, which] = dshare.v.sum(1)
        want_share.e[at, which] = dshare.e.sum(1) + hidden * 2.0 ** -23 * dshare.v.abs().sum(1)
        dy = (p * do).rounded(dtype)
        da = (dy @ a2).rounded(dtype)
        (dy.t() @ a).rounded(dtype).holds(dev[2].grad[e], "the gradient of w_down")
        dh_gate, dh_up = da * up * gate.of(silu_slope, 0.51), da * gate.of(silu, 1.1)
        dh = Near(torch.cat((dh_gate.v, dh_up.v), 1), torch.cat((dh_gate.e, dh_up.e), 1)).rounded(dtype)
        (dh.t() @ xs).rounded(dtype).holds(dev[1].grad[e], "the gradient of w_gate_up")
        dx = (dh @ a1).rounded(dtype)
        want_dx.v[at] += dx.v
        want_dx.e[at] += dx.e + 2.0 ** -21 * dx.v.abs()
    want_out.rounded(dtype).holds(out.detach(), "the output")
    want_dx.rounded(dtype).holds(dev[0].grad, "the gradient of x")
    want_share.holds(dev[3].grad, "the gradient of share")


@pytest.mark.parametrize("ranks", [1, 4])
@pytest.mark.parametrize("tokens,hidden,inter,count,top", [(1, 512, 256, 4, 2), (65, 1024, 320, 6, 3)])
def test_served(tokens, hidden, inter, count, top, ranks):
    """An e4m3 rounding moves a value by 2^-4 of it at most, rms 2^-4 / sqrt(3) = 3.6 %.  A product of two rounded operands: 5.1 % of its norm;
    gate and up together at most 1.8 times that (9.2 %, |g silu'/silu| up to 1.5 where results are large); the second product adds its 5.1 %: 10.5 %."""
    from mm_rs_with_catlass_amd.experts import ServedExperts
    x, w1, w2, choice, share = layer(5, tokens, hidden, inter, count, top, torch.bfloat16)
    _, s1, s2, _, _ = layer(6, tokens, hidden, inter, 1, 1, torch.bfloat16)
    peers = [torch.randn(tokens, hidden, generator=torch.Generator().manual_seed(7 + r)) for r in range(ranks - 1)]
    served = ServedExperts(w1.cuda(), w2.cuda(), s1[0].cuda(), s2[0].cuda())
    got = served(x.cuda(), choice.cuda(), share.cuda(), [p.cuda() for p in peers], ranks - 1).double().cpu()
    alone = ServedExperts(w1.cuda(), w2.cuda())(x.cuda(), choice.cuda(), share.cuda()).double().cpu()

    def expert(v, a1, a2):
        h = v @ a1.double().t()
        return (silu(h[:, :inter]) * h[:, inter:]) @ a2.double().t()
    want = torch.zeros(tokens, hidden).double()
    for t in range(tokens):
        for j in range(top):
            e = choice[t, j]
            want[t] += share[t, j].double() * expert(x[t:t + 1].double(), w1[e], w2[e])[0]
    assert (alone - want).norm() <= 0.105 * want.norm()
    both = expert(x.double(), s1[0], s2[0])
    # (the peers' partials come in fp32: what is off is this rank's product, and three roundings to bf16, 2^-8 of what they round)
    total = want + both + sum(p.double() for p in peers)
    assert (got - total).norm() <= 0.105 * (want.norm() + both.norm()) + 2.0 ** -8 * (want.norm() + 2 * total.norm() + both.norm())


def test_sorting():
    from mm_rs_with_catlass_amd.experts import sort_by_expert
    choice = torch.tensor([[3, 1], [1, 5], [3, 0]], device="cuda")
    order, back, ends = sort_by_expert(choice, 7)
    assert ends.tolist() == [1, 3, 3, 5, 5, 6, 6] and ends.dtype == torch.int32
    assert choice.flatten()[order].tolist() == [0, 1, 1, 3, 3, 5] and order[back].tolist() == list(range(6))


def test_command(capsys):
    from mm_rs_with_catlass_amd import experts
    experts.main()
    lines = capsys.readouterr().out.splitlines()
    losses = [float(s.split()[-1]) for s in lines[:-1]]
    assert losses[-1] < 0.5 * losses[0]
    assert float(lines[-1].split("%")[0].split()[-1]) <= 10.5


def test_second_gradients():
    """L = <c, dx> + <d, dw> of a grouped product's first gradients: each of L's gradients is one or two products of given values."""
    from mm_rs_with_catlass_amd.experts import GroupedLinear
    dtype, counts, k, n = torch.bfloat16, [5, 0, 70, 33], 72, 136
    g = torch.Generator().manual_seed(8)
    rows, groups = sum(counts) + 4, len(counts)           # (four rows of no group)
    x, dy, c = (torch.randn(rows, width, generator=g).to(dtype) for width in (k, n, k))
    w, d = (torch.randn(groups, n, k, generator=g).to(dtype) for _ in range(2))
    ends = torch.tensor(counts).cumsum(0).to(torch.int32).cuda()
    x1, w1, dy1 = (t.cuda().requires_grad_() for t in (x, w, dy))
    dx, dw = torch.autograd.grad(GroupedLinear.apply(x1, w1, ends), (x1, w1), dy1, create_graph=True)
    got = torch.autograd.grad((dx.float() * c.cuda().float()).sum() + (dw.float() * d.cuda().float()).sum(), (x1, w1, dy1))
    at = 0
    for e, count in enumerate(counts):
        i = slice(at, at + count)
        at += count
        if count == 0:
            assert not got[1][e].any()
            continue
        xs, ys, cs, ws, ds = (Near(t.double()) for t in (x[i], dy[i], c[i], w[e], d[e]))
        (ys @ ds).rounded(dtype).holds(got[0][i], "the gradient of x")
        (ys.t() @ cs).rounded(dtype).holds(got[1][e], "the gradient of w")
        ((cs @ ws.t()).rounded(dtype) + (xs @ ds.t()).rounded(dtype)).rounded(dtype).holds(got[2][i], "the gradient of dy")
    assert not got[0][at:].any() and not got[2][at:].any()


def test_tokens_without_an_expert():
    from mm_rs_with_catlass_amd.experts import ServedExperts, experts
    x, w1, w2, choice, share = (t.cuda() for t in layer(9, 50, 256, 128, 5, 2, torch.bfloat16))
    whole = experts(x, w1, w2, choice, share), ServedExperts(w1, w2)(x, choice, share)
    choice[7], choice[20, 1], choice[21, 0] = -1, -1, 5
    kept = torch.where((choice >= 0) & (choice < 5), share, 0)       # the same with no weight, which changes no product
    same = torch.where((choice >= 0) & (choice < 5), choice, 0)
    for got, want, before in zip((experts(x, w1, w2, choice, share), ServedExperts(w1, w2)(x, choice, share)),
                                 (experts(x, w1, w2, same, kept), ServedExperts(w1, w2)(x, same, kept)), whole):
        # (the choice of a tile, and with it the order of a sum in fp32, may differ: a rounding of each sum, and of what is added up)
        assert ((got.double() - want.double()).abs() <= 4 * U[torch.bfloat16] * before.double().abs().amax()).all()
        assert not got[7].any()
        rest = torch.ones(50, dtype=torch.bool)
        rest[[7, 20, 21]] = False
        assert ((got[rest].double() - before[rest].double()).abs() <= 4 * U[torch.bfloat16] * before.double().abs().amax()).all()


@pytest.mark.parametrize("shared", [False, True])
def test_no_tokens(shared):
    from mm_rs_with_catlass_amd.experts import ServedExperts, experts
    x, w1, w2, choice, share = (t.cuda() for t in layer(10, 3, 256, 128, 4, 2, torch.float16))
    leaves = [t.requires_grad_() for t in (x[:0].clone(), w1, w2, share[:0].clone())]
    out = experts(*leaves[:3], choice[:0], leaves[3])
    assert out.shape == (0, 256)
    for grad, leaf in zip(torch.autograd.grad(out.sum(), leaves), leaves):
        assert grad.shape == leaf.shape and not grad.any()
    served = ServedExperts(w1.detach(), w2.detach(), *((w1[0].detach(), w2[0].detach()) if shared else ()))
    assert served(x[:0], choice[:0], share[:0]).shape == (0, 256)


@pytest.mark.parametrize("served", [False, True])
def test_the_layer_in_a_captured_graph(served):
    from mm_rs_with_catlass_amd.experts import ServedExperts, experts
    x, w1, w2, choice, share = (t.cuda() for t in layer(11, 90, 256, 128, 6, 2, torch.bfloat16))
    whole = ServedExperts(w1, w2, w1[0], w2[0])

    def call():
        return whole(x, choice, share) if served else experts(x, w1, w2, choice, share)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for i in range(6):                                  # other tokens, other experts for them
        for to, values in zip((x, choice, share), (layer(20 + i, 90, 256, 128, 6, 2, torch.bfloat16)[j] for j in (0, 3, 4))):
            to.copy_(values)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, call()), i
