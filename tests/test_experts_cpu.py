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
