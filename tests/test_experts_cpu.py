"""The layer of experts without a GPU: plain products stand in for the grouped operators.  As the kernels' do, their results carry no graph."""
import pytest
import torch

from mm_rs_with_catlass_amd import experts as E


def groups_of(ends, rows):
    begin = 0
    for e, end in enumerate(ends.tolist()):
        yield e, begin, end
        begin = end
    assert begin <= rows


@torch.no_grad()
def grouped_matmul(x, w, ends, trans_b=False):
    y = x.new_zeros((x.shape[0], w.shape[1 if trans_b else 2]))
    for e, i, j in groups_of(ends, x.shape[0]):
        y[i:j] = x[i:j] @ (w[e].t() if trans_b else w[e])
    return y


@torch.no_grad()
def grouped_matmul_dw(x, dy, ends, out_dtype=None, trans_b=False):
    a, b = (dy, x) if trans_b else (x, dy)
    dw = a.new_zeros((ends.numel(), a.shape[1], b.shape[1]), dtype=out_dtype or x.dtype)
    for e, i, j in groups_of(ends, x.shape[0]):
        dw[e] = a[i:j].t() @ b[i:j]
    return dw


@pytest.fixture(autouse=True)
def stand_in(monkeypatch):
    monkeypatch.setattr(E.ops, "grouped_matmul", grouped_matmul)
    monkeypatch.setattr(E.ops, "grouped_matmul_dw", grouped_matmul_dw)


def randn(seed, *shape, dtype=torch.float64):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed), dtype=dtype)


def test_first_and_second_gradients_of_a_grouped_product_against_differences():
    ends = torch.tensor([2, 2, 5], dtype=torch.int32)     # (one group without rows, two rows of no group)
    x, w = randn(1, 7, 4).requires_grad_(), randn(2, 3, 5, 4).requires_grad_()

    def f(a, b):
        return E.GroupedLinear.apply(a, b, ends)
    assert torch.autograd.gradcheck(f, (x, w))
    assert torch.autograd.gradgradcheck(f, (x, w))


def plain_experts(x, w_gate_up, w_down, choice, share):
    rows = []
    for t in range(x.shape[0]):
        row = torch.zeros_like(x[t])
        for j in range(choice.shape[1]):
            gate, up = (w_gate_up[choice[t, j]] @ x[t]).chunk(2)
            row = row + share[t, j] * (w_down[choice[t, j]] @ (torch.nn.functional.silu(gate) * up))
        rows.append(row)
    return torch.stack(rows)


def test_a_penalty_on_first_gradients_reaches_all_operands():
    # everything in fp32 against 64 bits: sums of at most 12 x 16 products, five of them behind each other
    tokens, hidden, inter, count, top = 6, 12, 8, 4, 2
    choice = torch.stack([torch.randperm(count, generator=torch.Generator().manual_seed(t))[:top] for t in range(tokens)])
    values = [randn(11, tokens, hidden), 0.5 * randn(12, count, 2 * inter, hidden), 0.5 * randn(13, count, hidden, inter), randn(14, tokens, top).abs()]
    results = []
    for layer, dtype in ((E.experts, torch.float32), (plain_experts, torch.float64)):
        x, w1, w2, share = leaves = [v.to(dtype).requires_grad_() for v in values]
        first = torch.autograd.grad(layer(x, w1, w2, choice, share).square().sum(), leaves, create_graph=True)
        results.append(torch.autograd.grad(sum(g.square().sum() for g in first), leaves))
    for got, want in zip(*results):
        assert (got.double() - want).norm() <= 1e-4 * want.norm()


@pytest.mark.parametrize("dtype", [torch.int64, torch.int32, torch.int16])
def test_choices_of_no_expert_take_part_in_nothing(dtype):
    choice = torch.tensor([[3, -1], [1, 5], [-7, 9], [0, 3]], dtype=dtype)
    order, back, ends = E.sort_by_expert(choice, 4)
    assert ends.tolist() == [1, 2, 2, 4] and ends.dtype == torch.int32
    few = torch.tensor([[127], [-1], [0]], dtype=torch.int8)       # (as many experts as the type has)
    assert E.sort_by_expert(few, 128)[2].tolist() == [1] * 127 + [2]
    assert choice.flatten()[order[:4]].tolist() == [0, 1, 3, 3] and order[back].tolist() == list(range(8))

    tokens, hidden, inter = 4, 6, 5
    values = [randn(21, tokens, hidden), randn(22, 4, 2 * inter, hidden), randn(23, 4, hidden, inter), randn(24, tokens, 2).abs()]
    dropped = (choice < 0) | (choice >= 4)
    results = []
    for mine in (choice, torch.where(dropped, 0, choice)):     # (as expert 0's with no weight)
        leaves = [v.float().requires_grad_() for v in values]
        x, w1, w2, share = leaves
        out = E.experts(x, w1, w2, mine, torch.where(dropped, 0, share) if mine is not choice else share)
        results.append([out, *torch.autograd.grad(out.square().sum(), leaves)])
    for got, want in zip(*results):
        assert torch.allclose(got, want, rtol=1e-5, atol=1e-5)      # sums of the same values, in another order
    assert not results[0][0][2].any()


def test_no_tokens():
    x, w1, w2 = randn(31, 0, 6).float(), randn(32, 3, 8, 6).float(), randn(33, 3, 6, 4).float()
    leaves = [t.requires_grad_() for t in (x, w1, w2, torch.zeros(0, 2))]
    out = E.experts(*leaves[:3], torch.zeros((0, 2), dtype=torch.int64), leaves[3])
    assert out.shape == (0, 6)
    for grad, leaf in zip(torch.autograd.grad(out.sum(), leaves), leaves):
        assert grad.shape == leaf.shape and not grad.any()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [False, True])
@pytest.mark.parametrize("down", [0.0, -60.0, -120.0, -2000.0])
def test_gradient_of_the_router_with_a_graph_of_its_own(score, renormalize, down):
    """The formula behind second gradients, where the chosen experts' scores are as far down as they may be: against autograd in 64 bits of shares made from logarithms."""
    from types import SimpleNamespace

    from mm_rs_with_catlass_amd.experts import Route
    g = torch.Generator().manual_seed(3)
    logits, dshare, t = torch.randn((7, 12), generator=g), torch.randn((7, 4), generator=g), torch.randn((7, 12), generator=g)
    choice = torch.stack([torch.randperm(6, generator=g)[:4] for _ in range(7)]).int()
    logits[:, :6] += down                       # (the choices', by a bias)
    if score == "sigmoid":
        logits[3:, 6:] += down
    logits[1, choice[1, 3].long()] = -float("inf")
    choice[1, 3], choice[2] = -1, -1
    logits[4, 8:] = -float("inf")

    def gradients(l, d, along):
        l, d = l.clone().requires_grad_(), d.clone().requires_grad_()
        ctx = SimpleNamespace(saved_tensors=(l, choice), score=score, renormalize=renormalize, scale=1.5)
        with torch.enable_grad():
            first = Route.backward(ctx, None, d)[0]
            return [first, *torch.autograd.grad((first * along).sum(), (l, d))]

    def exact(l, d, along):
        l, d = l.double().requires_grad_(), d.double().requires_grad_()
        on, at = choice >= 0, choice.long().clamp_min(0)
        u = torch.nn.functional.logsigmoid(l) if score == "sigmoid" else torch.log_softmax(l, 1)
        u = torch.where(on, u.gather(1, at), -float("inf"))
        if renormalize:
            u = torch.where(on, u - torch.where(on.any(1, keepdim=True), u, 0.0).logsumexp(1, keepdim=True), -float("inf"))
        share = torch.where(on, torch.exp(torch.where(on, u, 0.0)), 0.0) * 1.5
        first, = torch.autograd.grad(share, l, d, create_graph=True)
        return [first, *torch.autograd.grad((first * along.double()).sum(), (l, d))]
    got, want = gradients(logits, dshare, t), exact(logits, dshare, t)
    assert not got[0][2].any()
    for a, b in zip(got, want):
        b = torch.where(torch.isnan(b), 0.0, b)     # (a gradient through -inf)
        # differences of products of shares (at most 1), |dshare| and |t| (at most 4 each), whose logarithms move by 2^-24 of logits and sums of some hundreds at most where the shares are
        # taken relative to each other, and of |down| where they are not and not below fp32
        assert a.isfinite().all() and (a.double() - b).abs().max() <= 1.5 * 4 * 4 * 200 * 2.0 ** -24
    if renormalize:
        assert got[0].abs().amax(1)[[0, 1, 3, 4, 5, 6]].min() > 1e-3
