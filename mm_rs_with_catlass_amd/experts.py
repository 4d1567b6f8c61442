"""A feed-forward layer of experts on the grouped and e4m3 operators: how they are called together.

`experts()` is the layer in 16 bits with its backward pass, `ServedExperts` the same layer on e4m3 weights, with an expert that every token
takes (its down projection split over ranks: one rank's all-reduce share).  An expert is w_down (silu(w_gate x) * (w_up x)); gate and up are
one matrix [2 inter, hidden], weights lie as [out, in].

    python -m mm_rs_with_catlass_amd.experts      # a few training steps, then the trained weights served in e4m3
"""
import torch

from . import ops


class GroupedLinear(torch.autograd.Function):
    """y[i] = w[e] x[i] for the rows i of group e; w [groups, out, in] ([groups, in, out] without trans_b).  Both gradients are grouped
    products as well, and differentiable in their turn."""

    @staticmethod
    def forward(ctx, x, w, ends, trans_b=True):
        ctx.save_for_backward(x, w, ends)
        ctx.trans_b = trans_b
        return ops.grouped_matmul(x, w, ends, trans_b=trans_b)

    @staticmethod
    def backward(ctx, dy):
        x, w, ends = ctx.saved_tensors
        dy = dy.contiguous()
        # (a gradient that nobody differentiates needs no function of its own: 64 tokens' forward and backward 480 us, 550 with one)
        linear, outer = (GroupedLinear.apply, GroupedOuter.apply) if torch.is_grad_enabled() else (ops.grouped_matmul, _outer)
        dx = linear(dy, w, ends, not ctx.trans_b) if ctx.needs_input_grad[0] else None
        dw = outer(x, dy, ends, ctx.trans_b) if ctx.needs_input_grad[1] else None
        return dx, dw, None, None


def _outer(x, dy, ends, trans_b):
    return ops.grouped_matmul_dw(x, dy, ends, trans_b=trans_b)


class GroupedOuter(torch.autograd.Function):
    """The weight gradient of GroupedLinear: dw[e] = sum over the rows i of group e of dy[i] x[i]^T (of x[i] dy[i]^T without trans_b)."""

    @staticmethod
    def forward(ctx, x, dy, ends, trans_b):
        ctx.save_for_backward(x, dy, ends)
        ctx.trans_b = trans_b
        return _outer(x, dy, ends, trans_b)

    @staticmethod
    def backward(ctx, g):
        x, dy, ends = ctx.saved_tensors
        g = g.contiguous()
        dx = GroupedLinear.apply(dy, g, ends, not ctx.trans_b) if ctx.needs_input_grad[0] else None
        ddy = GroupedLinear.apply(x, g, ends, ctx.trans_b) if ctx.needs_input_grad[1] else None
        return dx, ddy, None, None


def sort_by_expert(choice, experts):
    """choice [tokens, top], each token's experts -> (order, back, ends): row i of the sorted rows is choice order[i] of the flattened ones,
    back undoes it, group_ends for the operators.  Nothing is read back to the host.  Choices below 0 or past the last expert (a dropped token) are
    sorted behind the last group: rows of no group, whose results and gradients are zeros."""
    flat = choice.reshape(-1).long() & (2 ** 63 - 1)     # (a negative number without its sign is larger than any expert's)
    flat, order = torch.sort(flat, stable=True)
    back = torch.empty_like(order).scatter_(0, order, torch.arange(order.numel(), device=order.device))
    ends = torch.searchsorted(flat, torch.arange(experts, device=flat.device), right=True, out_int32=True)
    return order, back, ends


def spread(x, top, order):
    """Every token's row once for each of its experts, sorted by expert."""
    return x.unsqueeze(1).expand(-1, top, -1).reshape(-1, x.shape[1])[order]


def gather(y, share, back):
    """The experts' rows back at their tokens, weighted (summed in fp32, rounded once)."""
    return (y[back].view(*share.shape, y.shape[1]).float() * share.float().unsqueeze(-1)).sum(1).to(y.dtype)


def experts(x, w_gate_up, w_down, choice, share):
    """x [tokens, hidden] fp16 or bf16, w_gate_up [experts, 2 inter, hidden], w_down [experts, hidden, inter], choice and share [tokens, top]:
    each token's experts (none: -1) and their weights.  Returns [tokens, hidden]; differentiable in x, both weights and share."""
    order, back, ends = sort_by_expert(choice, w_gate_up.shape[0])
    h = GroupedLinear.apply(spread(x, choice.shape[1], order), w_gate_up, ends)
    gate, up = h.float().chunk(2, 1)
    y = GroupedLinear.apply((torch.nn.functional.silu(gate) * up).to(x.dtype), w_down, ends)
    return gather(y, share, back)


def _quantize_each(w):
    """e4m3 codes and scales of each expert's matrix."""
    codes = torch.empty(w.shape, dtype=torch.float8_e4m3fn, device=w.device)
    scales = torch.empty((w.shape[0], -(-w.shape[1] // 128), -(-w.shape[2] // 128)), dtype=torch.float32, device=w.device)
    for e in range(w.shape[0]):
        ops.quantize_fp8(w[e], block_rows=128, out=codes[e], scale=scales[e])
    return codes, scales


class ServedExperts:
    """The layer on e4m3 weights, quantized once; rows are quantized on their way into each product, the second time together with the gate.

    shared_gate_up [2 inter, hidden], shared_down [hidden, inter] (both or neither): the expert of every token, this rank's share of inter."""

    def __init__(self, w_gate_up, w_down, shared_gate_up=None, shared_down=None):
        self.experts = w_gate_up.shape[0]
        self.gate_up, self.down = _quantize_each(w_gate_up), _quantize_each(w_down)
        self.shared = None if shared_gate_up is None else [ops.quantize_fp8(w, block_rows=128) for w in (shared_gate_up, shared_down)]

    def __call__(self, x, choice, share, peers=(), rank=0):
        """peers: the other ranks' fp32 partials [tokens, hidden] of the shared expert."""
        order, back, ends = sort_by_expert(choice, self.experts)
        rows, scale = ops.quantize_fp8(spread(x, choice.shape[1], order))
        h = ops.grouped_fp8_matmul(rows, self.gate_up[0], scale, self.gate_up[1], ends, out_dtype=x.dtype)
        rows, scale = ops.quantize_fp8(h, gated=True)
        out = gather(ops.grouped_fp8_matmul(rows, self.down[0], scale, self.down[1], ends, out_dtype=x.dtype), share, back)
        if self.shared is None:
            return out
        (gate_up, gate_up_scale), (down, down_scale) = self.shared
        rows, scale = ops.quantize_fp8(x)
        h = ops.fp8_matmul_allreduce(rows, gate_up, scale, gate_up_scale, out_dtype=x.dtype)
        rows, scale = ops.quantize_fp8(h, gated=True)
        return out + ops.fp8_matmul_allreduce(rows, down, scale, down_scale, peers, rank, len(peers) + 1, out_dtype=x.dtype)


def main():
    torch.manual_seed(0)
    tokens, hidden, inter, count, top, dev = 512, 1024, 512, 8, 2, "cuda"
    x = torch.randn(tokens, hidden, device=dev, dtype=torch.bfloat16)
    aim = torch.randn(tokens, hidden, device=dev)
    router = torch.randn(hidden, count, device=dev) / hidden ** 0.5
    masters = [torch.randn(count, 2 * inter, hidden, device=dev) / hidden ** 0.5, torch.randn(count, hidden, inter, device=dev) / inter ** 0.5]
    share, choice = (x.float() @ router).softmax(1).topk(top)
    optimizer = torch.optim.Adam(masters, lr=3e-3)
    for step in range(20):
        weights = [m.to(torch.bfloat16).requires_grad_() for m in masters]
        loss = (experts(x, *weights, choice, share).float() - aim).square().mean()
        loss.backward()
        for m, w in zip(masters, weights):
            m.grad = w.grad.float()
        optimizer.step()
        if step % 5 == 4:
            print("step %d  loss %.4f" % (step + 1, loss.item()), flush=True)
    weights = [m.to(torch.bfloat16) for m in masters]
    trained, served = experts(x, *weights, choice, share).float(), ServedExperts(*weights)(x, choice, share).float()
    print("served in e4m3: %.1f %% from the 16-bit layer" % (100 * ((served - trained).norm() / trained.norm()).item()))


if __name__ == "__main__":
    main()
