"""A feed-forward layer of experts on the grouped and e4m3 operators, and the block around it: how they are called together.

`experts()` is the layer in 16 bits with its backward pass, `ServedExperts` the same layer on e4m3 weights, with an expert that every token
takes (its down projection split over ranks: one rank's all-reduce share).  An expert is w_down (silu(w_gate x) * (w_up x)); gate and up are
one matrix [2 inter, hidden], weights lie as [out, in].

`block()` goes from the residual stream to what is added to it next: norm, router, experts; `ServedBlock` is the same on e4m3 weights, its rows
quantized by the norm.  `rms_norm()` and `route()` are the operators of ops.py with their gradients.

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


class Spread(torch.autograd.Function):
    """Every token's row at its choices' places (ops.spread_rows)."""

    @staticmethod
    def forward(ctx, x, back):
        ctx.save_for_backward(back)
        return ops.spread_rows(x.contiguous(), back)

    @staticmethod
    def backward(ctx, d):
        back, = ctx.saved_tensors
        return Gather.apply(d, back, None), None


class Gather(torch.autograd.Function):
    """The choices' rows summed at their tokens, by share where there is one (ops.gather_rows).  The rows are kept for the shares' gradient, where that is wanted."""

    @staticmethod
    def forward(ctx, y, back, share):
        ctx.save_for_backward(y if ctx.needs_input_grad[2] else None, back, share)
        ctx.rows, ctx.dtype = ctx.needs_input_grad[0], y.dtype
        return ops.gather_rows(y.contiguous(), back, share)

    @staticmethod
    def backward(ctx, dout):
        y, back, share = ctx.saved_tensors
        if share is None:
            return Spread.apply(dout, back), None, None
        if torch.is_grad_enabled():     # (gradients of gradients: from operators that have them)
            d, at = Spread.apply(dout, back).float(), back.reshape(-1).long()
            sorted_share = share.new_zeros(at.numel()).index_put((at,), share.reshape(-1))
            return ((d * sorted_share.unsqueeze(-1)).to(ctx.dtype) if ctx.rows else None, None,
                    None if y is None else (d * y.float()).sum(1)[at].view(share.shape))
        dy, dshare = ops.gather_rows_backward(dout.contiguous(), None if y is None else y.contiguous(), back, share, rows=ctx.rows)
        return dy, None, dshare


class _Plan:
    """Where the rows of a call's choices lie.  Tensors on the GPU go through the operators, those on the host, and more experts or choices than the operators
    take, through torch."""

    def __init__(self, choice, experts):
        self.top, self.kernels = choice.shape[1], choice.is_cuda and experts <= ops.MOST_EXPERTS and 1 <= choice.shape[1] <= ops.MOST_TOP
        if self.kernels:
            choice = choice if choice.dtype in (torch.int32, torch.int64) else choice.int()
            self.order, self.back, self.ends = ops.sort_by_expert(choice.contiguous(), experts)
        else:
            self.order, self.back, self.ends = sort_by_expert(choice, experts)

    def spread(self, x):
        return Spread.apply(x, self.back) if self.kernels else spread(x, self.top, self.order)

    def spread_fp8(self, x, scale):
        """e4m3 rows and their scales."""
        if self.kernels:
            return ops.spread_rows(x, self.back, scale)
        token = torch.div(self.order, self.top, rounding_mode="floor")
        return x.view(torch.uint8)[token].view(x.dtype), scale[:, token]

    def gather(self, y, share):
        return Gather.apply(y, self.back, share.float().contiguous()) if self.kernels else gather(y, share, self.back)


def experts(x, w_gate_up, w_down, choice, share):
    """x [tokens, hidden] fp16 or bf16, w_gate_up [experts, 2 inter, hidden], w_down [experts, hidden, inter], choice and share [tokens, top]:
    each token's experts (none: -1) and their weights.  Returns [tokens, hidden]; differentiable in x, both weights and share."""
    plan = _Plan(choice, w_gate_up.shape[0])
    h = GroupedLinear.apply(plan.spread(x), w_gate_up, plan.ends)
    gate, up = h.float().chunk(2, 1)
    y = GroupedLinear.apply((torch.nn.functional.silu(gate) * up).to(x.dtype), w_down, plan.ends)
    return plan.gather(y, share)


class RmsNorm(torch.autograd.Function):
    """ops.rms_norm with its gradients; without a residual the sum is None."""

    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        y, s = (ops.rms_norm(x, weight, eps=eps), None) if residual is None else ops.rms_norm(x, weight, residual, eps=eps)
        ctx.save_for_backward(x if s is None else s, weight)
        ctx.eps, ctx.types = eps, (x.dtype, None if residual is None else residual.dtype)
        ctx.set_materialize_grads(False)
        return y, s

    @staticmethod
    def backward(ctx, dy, dsum):
        s, weight = ctx.saved_tensors
        x_type, residual_type = ctx.types
        if dy is None:
            ds, dw = dsum, None
        elif torch.is_grad_enabled():   # (gradients of gradients: the formula in torch)
            v, w, d = s.float(), weight.float(), dy.float()
            r = (v.square().mean(1, keepdim=True) + ctx.eps).rsqrt()
            n, g = v * r, d * w
            ds = r * (g - n * (g * n).mean(1, keepdim=True)) + (0 if dsum is None else dsum.float())
            ds, dw = ds.to(s.dtype), (d * n).sum(0).to(weight.dtype)
        else:
            ds, dw = ops.rms_norm_backward(dy.contiguous(), s, weight, None if dsum is None else dsum.contiguous(), eps=ctx.eps)
        return ds.to(x_type) if ds is not None and ctx.needs_input_grad[0] else None, dw, ds if residual_type is not None else None, None


def rms_norm(x, weight, residual=None, eps=1e-6):
    """ops.rms_norm(), differentiable in x, weight and residual: y, or (y, x + residual)."""
    y, s = RmsNorm.apply(x, weight, residual, eps)
    return y if residual is None else (y, s)


class Route(torch.autograd.Function):
    """ops.route with the shares' gradient; how: its arguments by name."""

    @staticmethod
    def forward(ctx, logits, top, bias, how):
        choice, share = ops.route(logits, top, bias=bias, **how)
        ctx.save_for_backward(logits, choice)
        ctx.score, ctx.renormalize, ctx.scale = how.get("score", "softmax"), how.get("renormalize", True), how.get("scale", 1.0)
        ctx.mark_non_differentiable(choice)
        return choice, share

    @staticmethod
    def backward(ctx, _, dshare):
        logits, choice = ctx.saved_tensors
        if not torch.is_grad_enabled():
            return ops.route_backward(dshare.contiguous(), logits, choice, score=ctx.score, renormalize=ctx.renormalize, scale=ctx.scale), None, None, None
        return _route_gradient(dshare, logits, choice, ctx.score, ctx.renormalize, ctx.scale), None, None, None


def _route_gradient(dshare, logits, choice, score, renormalize, scale):
    """ops.route_backward()'s formula in torch, for gradients of gradients."""
    at = choice.long().clamp_min(0)
    l = logits.float().gather(1, at)
    on = (choice >= 0) & (l != -torch.inf)
    l, g = torch.where(on, l, 0.0), torch.where(on, dshare * scale, 0.0)
    if renormalize:     # (shares from logarithms: the scores of experts that are all far down are nothing in fp32)
        u = torch.where(on, torch.nn.functional.logsigmoid(l) if score == "sigmoid" else l, -torch.inf)
        w = torch.where(on, torch.softmax(torch.where(on.any(1, keepdim=True), u, 0.0), 1), 0.0)
        d = w * (g - (w * g).sum(1, keepdim=True))
        rest = torch.zeros_like(logits, dtype=torch.float32)
    elif score == "sigmoid":
        d, rest = torch.sigmoid(l) * g, torch.zeros_like(logits, dtype=torch.float32)
    else:               # every expert's logit moves the shares
        v = logits.float()
        p = torch.softmax(torch.where((v != -torch.inf).any(1, keepdim=True), v, 0.0), 1)
        d = torch.where(on, p.gather(1, at), 0.0) * g
        rest = -p * d.sum(1, keepdim=True)
    if score == "sigmoid":
        d = d * torch.sigmoid(-l)
    return rest.scatter_add(1, at, torch.where(on, d, 0.0)).to(logits.dtype)


def route(logits, top, bias=None, **how):
    """ops.route(), its shares differentiable in logits: (choice, share)."""
    return Route.apply(logits, top, bias, how)


def block(x, residual, norm, router, w_gate_up, w_down, top, bias=None, eps=1e-6, **how):
    """From the residual stream to what is added to it next: x [tokens, hidden] fp16 or bf16, the last layer's output; residual [tokens, hidden] of its type or fp32, what it is
    added to; norm [hidden], router [experts, hidden]; top, bias and how: of route().  Returns the experts' output and the sum x + residual; differentiable in all
    floating operands but bias."""
    y, s = rms_norm(x, norm, residual, eps)
    choice, share = route(y.float() @ router.float().t(), top, bias, **how)
    return experts(y, w_gate_up, w_down, choice, share), s


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

    def __call__(self, x, choice, share, peers=(), rank=0, codes=None):
        """peers: the other ranks' fp32 partials [tokens, hidden] of the shared expert; codes: x in e4m3 with its scales, where it was quantized before."""
        plan = _Plan(choice, self.experts)
        codes = ops.quantize_fp8(x.contiguous()) if codes is None else codes
        rows, scale = plan.spread_fp8(*codes)    # (a row's codes are the same before and after)
        h = ops.grouped_fp8_matmul(rows, self.gate_up[0], scale, self.gate_up[1], plan.ends, out_dtype=x.dtype)
        rows, scale = ops.quantize_fp8(h, gated=True)
        out = plan.gather(ops.grouped_fp8_matmul(rows, self.down[0], scale, self.down[1], plan.ends, out_dtype=x.dtype), share)
        if self.shared is None:
            return out
        (gate_up, gate_up_scale), (down, down_scale) = self.shared
        rows, scale = codes
        h = ops.fp8_matmul_allreduce(rows, gate_up, scale, gate_up_scale, out_dtype=x.dtype)
        rows, scale = ops.quantize_fp8(h, gated=True)
        return out + ops.fp8_matmul_allreduce(rows, down, scale, down_scale, peers, rank, len(peers) + 1, out_dtype=x.dtype)


class ServedBlock:
    """block() on e4m3 weights: the norm's rows leave it in 16 bits for the router and in e4m3 for the experts, the shared one too."""

    def __init__(self, norm, router, w_gate_up, w_down, top, shared_gate_up=None, shared_down=None, bias=None, eps=1e-6, **how):
        self.norm, self.router, self.eps, self.top, self.bias, self.how = norm, router.float().t().contiguous(), eps, top, bias, how
        self.experts = ServedExperts(w_gate_up, w_down, shared_gate_up, shared_down)

    def __call__(self, x, residual, peers=(), rank=0):
        q, scale, y, s = ops.rms_norm_fp8(x, self.norm, residual, eps=self.eps, keep=True)
        choice, share = ops.route(y.float() @ self.router, self.top, bias=self.bias, **self.how)
        return self.experts(y, choice, share, peers, rank, codes=(q, scale)), s


def main():
    torch.manual_seed(0)
    tokens, hidden, inter, count, top, dev = 512, 1024, 512, 8, 2, "cuda"
    x, residual = torch.randn(tokens, hidden, device=dev, dtype=torch.bfloat16), torch.randn(tokens, hidden, device=dev)
    aim = torch.randn(tokens, hidden, device=dev)
    masters = [torch.ones(hidden, device=dev), torch.randn(count, hidden, device=dev) / hidden ** 0.5, torch.randn(count, 2 * inter, hidden, device=dev) / hidden ** 0.5,
               torch.randn(count, hidden, inter, device=dev) / inter ** 0.5]
    optimizer = torch.optim.Adam(masters, lr=3e-3)
    for step in range(20):
        weights = [m.to(torch.bfloat16).requires_grad_() for m in masters]
        loss = (block(x, residual, *weights, top, renormalize=False)[0].float() - aim).square().mean()
        loss.backward()
        for m, w in zip(masters, weights):
            m.grad = w.grad.float()
        optimizer.step()
        if step % 5 == 4:
            print("step %d  loss %.4f" % (step + 1, loss.item()), flush=True)
    weights = [m.to(torch.bfloat16) for m in masters]
    trained = block(x, residual, *weights, top, renormalize=False)[0].float()
    served = ServedBlock(*weights, top, renormalize=False)(x, residual)[0].float()
    print("served in e4m3: %.1f %% from the 16-bit layer" % (100 * ((served - trained).norm() / trained.norm()).item()))


if __name__ == "__main__":
    main()
