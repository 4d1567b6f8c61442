"""Cases of the operators around a layer of experts: from the residual stream to the experts' sorted rows, and back at their tokens.

`listed()` names the cases, `draw()` gives more of the same ranges, `prepare()` makes what a program has in hand before the call,
`run()` is one call of a public operator or, with `own` false, the same mathematics in elementary torch operations; `exact()` is the
operator's definition in 64 bits and `work()` the bytes and operations it cannot do without.

Operators:
  norm, norm_fp8, norm_backward   s = x + residual; y = s / sqrt(mean(s^2) + eps) * weight, in 16 bits, or in e4m3 with one fp32 scale per 128 values
                                  of a row, or both; and the gradients of s and weight
  route, route_backward           scores of the experts by softmax or sigmoid of their logits; the best groups of experts, where they come in groups, and the
                                  `top` best experts in them by score + bias, ties to the lowest index; their scores as shares, of the sum where
                                  renormalised.  Logits of -inf: not to be had; where none is left -1 with a share of 0.  And the gradient of the logits
  sort                            the choices' rows by expert, in order of tokens within one; where each choice went, where each expert's rows end
  spread, gather, gather_backward every token's row once for each of its choices, at that choice's place; the choices' rows summed at their tokens by
                                  share; and the gradients of rows and shares

Sizes: hidden widths 256 to 8192, 8 to 256 experts, one to eight of them for a token, one token to long prompts.
"""
import math
import random

import torch

own = False
DEV = "cuda:0"
_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4, "e4m3": 1}
_BLOCK = 128
_TOP = 448.0          # largest e4m3 value
_FLOOR = 2.0 ** -40   # smallest amax of a block
_EPS = 1e-6


def _norm(name, op, rows, cols, dtype, residual, weight="same", keep=False):
    """residual: its type, "none" for no addition (norm_backward: whether a gradient of the sum comes in besides); keep: norm_fp8 returns y too."""
    return {"name": name, "op": op, "rows": rows, "cols": cols, "dtype": dtype, "residual": residual, "weight": weight, "keep": keep}


def _route(name, op, tokens, experts, top, dtype, score, bias=False, groups=1, top_groups=1, group_top=1, renormalize=True, scale=1.0, padded=0):
    """padded: that many tokens at the end are none, all their logits -inf."""
    return {"name": name, "op": op, "tokens": tokens, "experts": experts, "top": top, "dtype": dtype, "score": score, "bias": bias, "groups": groups,
            "top_groups": top_groups, "group_top": group_top, "renormalize": renormalize, "scale": scale, "padded": padded}


def _sort(name, tokens, top, experts, dropped=0):
    """dropped: that many choices are -1."""
    return {"name": name, "op": "sort", "tokens": tokens, "top": top, "experts": experts, "dropped": dropped}


def _rows(name, op, tokens, top, cols, dtype, shares=True):
    return {"name": name, "op": op, "tokens": tokens, "top": top, "cols": cols, "dtype": dtype, "shares": shares}


def listed():
    return [
        # a decode batch between attention and a layer of experts: 16 bits for the router, e4m3 for the experts; latency is all
        _norm("norm_fp8_16", "norm_fp8", 16, 4096, "bf16", "bf16", keep=True),
        # a long prompt, or a training step's forward pass
        _norm("norm_16384", "norm", 16384, 4096, "bf16", "bf16"),
        # a packed batch that is no multiple of anything, a residual stream in 32 bits, rows that end inside a block
        _norm("norm_fp8_4099", "norm_fp8", 4099, 1808, "fp16", "fp32"),
        # a training step's backward pass, weights in 32 bits, the residual's own gradient added
        _norm("norm_backward_8192", "norm_backward", 8192, 4096, "bf16", "bf16", weight="fp32"),
        # a decode batch over few experts, logits in 16 bits with many ties
        _route("route_32", "route", 32, 64, 8, "bf16", "softmax"),
        # a long prompt over many experts in groups, balanced by a bias, its last tokens padding
        _route("route_16384", "route", 16384, 256, 8, "fp32", "sigmoid", bias=True, groups=8, top_groups=4, group_top=2, scale=2.5, padded=100),
        # a training step's backward pass, shares that keep the softmax's sum
        _route("route_backward_4099", "route_backward", 4099, 60, 4, "fp32", "softmax", renormalize=False),
        # the plan of a decode batch
        _sort("sort_256", 32, 8, 64),
        # of a long prompt, some of whose choices were dropped
        _sort("sort_131072", 16384, 8, 128, dropped=1000),
        # a prompt's e4m3 rows on their way into the experts, with their scales
        _rows("spread_fp8_16384", "spread", 2048, 8, 4096, "e4m3"),
        # a decode batch's rows back from the experts
        _rows("gather_256", "gather", 32, 8, 4096, "bf16"),
        # a training step's gradients of odd size on their way back into the experts
        _rows("gather_backward_8198", "gather_backward", 4099, 2, 1808, "fp16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A width: mostly whole blocks, sometimes whole 16-byte pieces, sometimes neither."""
    s = rng.choice([128, 128, 128, 64, 16, 4, 1])
    return max(lo, s * max(1, int(round(_log(rng, lo, hi) / s))))


def draw(rng):
    op = rng.choice(["norm", "norm", "norm_fp8", "norm_fp8", "norm_backward", "route", "route", "route_backward", "sort", "spread", "gather", "gather_backward"])
    if op.startswith("norm"):
        while True:
            dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
            c = _norm("", op, _log(rng, 1, 16384), _width(rng, 256, 8192), dtype, rng.choice(["none", dtype, dtype, "fp32"]), rng.choice(["same", "fp32"]),
                      op == "norm_fp8" and rng.random() < 0.5)
            if c["rows"] * c["cols"] <= 6e7:
                break
    elif op.startswith("route"):
        experts, groups = rng.choice([8, 16, 32, 60, 64, 128, 160, 256]), 1
        if experts >= 60 and rng.random() < 0.4:
            groups = 4 if experts == 60 else 8
        top = min(rng.choice([1, 2, 4, 6, 8] if op == "route" else [2, 4, 6, 8]), experts // 2)    # (one share of its own sum is 1: no gradient)
        tokens = _log(rng, 1, 16384)
        c = _route("", op, tokens, experts, top, rng.choice(["bf16", "fp16", "fp32", "fp32"]), rng.choice(["softmax", "sigmoid"]), rng.random() < 0.5, groups,
                   max(1, groups // 2), rng.choice([1, 2]) if groups > 1 else 1, rng.random() < 0.6, rng.choice([1.0, 1.0, 2.5]), rng.choice([0, 0, tokens // 8]))
    elif op == "sort":
        experts = rng.choice([8, 16, 32, 60, 64, 128, 160, 256])
        c = _sort("", _log(rng, 1, 16384), rng.choice([1, 2, 4, 6, 8]), experts, 0)
        c["dropped"] = rng.choice([0, c["tokens"] * c["top"] // 10])
    else:
        while True:
            c = _rows("", op, _log(rng, 1, 16384), rng.choice([1, 2, 4, 6, 8]), _width(rng, 256, 8192), rng.choice(["bf16", "fp16"]), op == "gather_backward" or rng.random() < 0.7)
            if op == "spread" and rng.random() < 0.5:
                c["dtype"] = "e4m3"
            if c["tokens"] * c["top"] * c["cols"] <= 1.2e8:
                break
    del c["name"]
    return c


# ---- inputs ---------------------------------------------------------------------------------------------------------------------

def _stream(g, rows, cols):
    """Activations: rows of different size, some columns much larger than the others."""
    v = torch.randn((rows, cols), device=DEV, generator=g)
    v *= torch.exp(0.5 * torch.randn((rows, 1), device=DEV, generator=g))
    v *= 1.0 + 15.0 * (torch.rand((1, cols), device=DEV, generator=g) < 0.01)
    return v


def _choices(g, tokens, top, experts):
    """Different experts for each token, some of them more wanted than others."""
    wanted = torch.rand((tokens, experts), device=DEV, generator=g) + 0.3 * torch.rand((1, experts), device=DEV, generator=g)
    return wanted.topk(top, 1).indices.to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    s, op = dict(case), case["op"]
    if op.startswith("norm"):
        rows, cols, dt = case["rows"], case["cols"], _DT[case["dtype"]]
        summed = case["residual"] != "none"
        rt = _DT[case["residual"]] if summed else dt
        s["w"] = (1.0 + 0.2 * torch.randn(cols, device=DEV, generator=g)).to(dt if case["weight"] == "same" else torch.float32)
        if op == "norm_backward":
            s["x"] = _stream(g, rows, cols).to(rt)
            s["dy"] = (0.01 * _stream(g, rows, cols)).to(dt)
            s["more"] = (0.01 * torch.randn((rows, cols), device=DEV, generator=g)).to(rt) if summed else None
        else:
            s["x"] = _stream(g, rows, cols).to(dt)
            s["r"] = (2.0 * _stream(g, rows, cols)).to(rt) if summed else None
    elif op.startswith("route"):
        tokens, experts = case["tokens"], case["experts"]
        logits = torch.randn((tokens, experts), device=DEV, generator=g) + 0.5 * torch.randn((1, experts), device=DEV, generator=g)
        if case["padded"]:
            logits[tokens - case["padded"]:] = -math.inf
        s["logits"] = logits.to(_DT[case["dtype"]])
        s["b"] = 0.05 * torch.randn(experts, device=DEV, generator=g) if case["bias"] else None
        if op == "route_backward":
            s["choice"] = _choose(s)[0]
            s["dshare"] = torch.randn((tokens, case["top"]), device=DEV, generator=g)
    elif op == "sort":
        s["choice"] = _choices(g, case["tokens"], case["top"], case["experts"])
        if case["dropped"]:
            s["choice"].view(-1)[torch.randperm(s["choice"].numel(), device=DEV, generator=g)[:case["dropped"]]] = -1
    else:
        tokens, top, cols = case["tokens"], case["top"], case["cols"]
        flat = _choices(g, tokens, top, 64).view(-1)
        s["back"] = torch.empty_like(flat)
        s["back"][flat.sort(stable=True).indices] = torch.arange(flat.numel(), dtype=torch.int32, device=DEV)
        s["back"] = s["back"].view(tokens, top)
        s["share"] = torch.rand((tokens, top), device=DEV, generator=g).softmax(1) if case["shares"] else None
        if case["dtype"] == "e4m3":
            s["x"] = (60.0 * torch.randn((tokens, cols), device=DEV, generator=g)).clamp_(-_TOP, _TOP).to(torch.float8_e4m3fn)
            s["scale"] = torch.rand((-(-cols // _BLOCK), tokens), device=DEV, generator=g)
        else:
            s["x"] = _stream(g, tokens, cols).to(_DT[case["dtype"]])
            s["scale"] = None
        if op != "spread":
            s["y"] = _stream(g, tokens * top, cols).to(_DT[case["dtype"]])
    return s


# ---- one pass -------------------------------------------------------------------------------------------------------------------

def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    from mm_rs_with_catlass_amd import ops
    op = s["op"]
    if op == "norm":
        return ops.rms_norm(s["x"], s["w"], residual=s["r"], eps=_EPS)
    if op == "norm_fp8":
        return ops.rms_norm_fp8(s["x"], s["w"], residual=s["r"], eps=_EPS, keep=s["keep"])
    if op == "norm_backward":
        return ops.rms_norm_backward(s["dy"], s["x"], s["w"], dsum=s["more"], eps=_EPS)
    if op == "route":
        return ops.route(s["logits"], s["top"], score=s["score"], bias=s["b"], groups=s["groups"], top_groups=s["top_groups"], group_top=s["group_top"],
                         renormalize=s["renormalize"], scale=s["scale"])
    if op == "route_backward":
        return ops.route_backward(s["dshare"], s["logits"], s["choice"], score=s["score"], renormalize=s["renormalize"], scale=s["scale"])
    if op == "sort":
        return ops.sort_by_expert(s["choice"], s["experts"])
    if op == "spread":
        return ops.spread_rows(s["x"], s["back"], scale=s["scale"])
    if op == "gather":
        return ops.gather_rows(s["y"], s["back"], share=s["share"])
    return ops.gather_rows_backward(s["x"], s["y"], s["back"], s["share"])


def _encode(v):
    """e4m3 codes, and scales as [blocks of columns, rows]."""
    rows, cols = v.shape
    blocks = -(-cols // _BLOCK)
    p = torch.zeros((rows, blocks * _BLOCK), device=v.device)
    p[:, :cols] = v
    p = p.view(rows, blocks, _BLOCK)
    scale = p.abs().amax(2).clamp_min(_FLOOR) / _TOP
    q = (p / scale[:, :, None]).view(rows, -1)[:, :cols].contiguous().to(torch.float8_e4m3fn)
    return q, scale.t().contiguous()


def _plain_norm(s):
    op, x, w = s["op"], s["x"], s["w"].float()
    if op == "norm_backward":
        v, dy = x.float(), s["dy"].float()
        r = 1.0 / torch.sqrt((v * v).mean(1, keepdim=True) + _EPS)
        n, g = v * r, dy * w
        ds = r * (g - n * (g * n).mean(1, keepdim=True))
        if s["more"] is not None:
            ds = ds + s["more"].float()
        dw = (dy * n).sum(0, dtype=torch.float64)
        return ds.to(x.dtype), dw.to(s["w"].dtype)
    summed = s["r"] is not None
    if summed:
        kept = (x.float() + s["r"].float()).to(s["r"].dtype)
    v = kept.float() if summed else x.float()
    y = v / torch.sqrt((v * v).mean(1, keepdim=True) + _EPS) * w
    out = [y.to(x.dtype)] if op == "norm" or s["keep"] else []
    if op == "norm_fp8":
        out = [*_encode(y), *out]
    if summed:
        out.append(kept)
    return out[0] if len(out) == 1 else tuple(out)


def _scores(s):
    """In 64 bits: which of two experts is the better one is a matter of their scores' last bits now and then."""
    v = s["logits"].double()
    if s["score"] == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-v))
    e = torch.exp(v - v.amax(1, keepdim=True))
    return e / e.sum(1, keepdim=True)


def _choose(s):
    """The experts chosen, and all scores."""
    p = _scores(s)
    v = p if s["b"] is None else p + s["b"].double()
    v = torch.where(s["logits"].float() == -math.inf, -math.inf, v)
    if s["groups"] > 1:
        by_group = v.view(v.shape[0], s["groups"], -1)
        best = by_group.sort(dim=2, descending=True).values[:, :, :s["group_top"]].sum(2)
        order = best.sort(dim=1, descending=True, stable=True).indices[:, :s["top_groups"]]
        taken = (torch.arange(s["groups"], device=DEV)[None, :, None] == order[:, None, :]).any(2)
        v = torch.where(taken[:, :, None], by_group, -math.inf).reshape(v.shape)
    v, choice = v.sort(dim=1, descending=True, stable=True)
    v, choice = v[:, :s["top"]], choice[:, :s["top"]]
    return torch.where(v == -math.inf, -1, choice).to(torch.int32), p


def _plain_route(s):
    if s["op"] == "route":
        choice, p = _choose(s)
        share = torch.where(choice >= 0, p.gather(1, choice.long().clamp_min(0)), 0.0)
        if s["renormalize"]:
            total = share.sum(1, keepdim=True)
            share = torch.where(total > 0, share / total, 0.0)
        return choice, (share * s["scale"]).float()
    chosen, at = s["choice"] >= 0, s["choice"].long().clamp_min(0)
    v = s["logits"].float()
    d = torch.where(chosen, s["dshare"] * s["scale"], 0.0)
    if s["score"] == "sigmoid":
        p = 1.0 / (1.0 + torch.exp(-v))
    else:
        p = torch.exp(v - v.amax(1, keepdim=True))
        p = p / p.sum(1, keepdim=True)
    mine = torch.where(chosen, p.gather(1, at), 0.0)
    if s["renormalize"]:
        total = mine.sum(1, keepdim=True)
        d = (d - (d * mine).sum(1, keepdim=True) / total) / total
    if s["score"] == "sigmoid":
        d = d * mine * (1.0 - mine)
        rest = torch.zeros_like(v)
    else:
        rest = -p * (d * mine).sum(1, keepdim=True)
        d = d * mine
    out = rest.scatter_add(1, at, torch.where(chosen, d, 0.0))
    return torch.where(v == -math.inf, 0.0, out).to(s["logits"].dtype)


def _plain_sort(s):
    flat = s["choice"].view(-1).long()
    experts = s["experts"]
    flat, order = torch.where(flat < 0, experts, flat).sort(stable=True)
    back = torch.empty_like(order)
    back[order] = torch.arange(order.numel(), device=DEV)
    ends = (flat[None, :] <= torch.arange(experts, device=DEV)[:, None]).sum(1)
    return order.to(torch.int32), back.view(s["choice"].shape).to(torch.int32), ends.to(torch.int32)


def _plain_rows(s):
    op, back = s["op"], s["back"].long()
    if op == "spread":
        tokens = torch.empty(back.numel(), dtype=torch.int64, device=DEV)
        tokens[back.view(-1)] = torch.arange(back.numel(), device=DEV) // s["top"]
        rows = s["x"].view(torch.uint8)[tokens].view(s["x"].dtype) if s["scale"] is not None else s["x"][tokens]
        return rows if s["scale"] is None else (rows, s["scale"][:, tokens])
    v = s["y"][back].float()
    if op == "gather":
        return (v if s["share"] is None else v * s["share"][:, :, None]).sum(1).to(s["y"].dtype)
    d = s["x"].float()[:, None, :]
    dy = torch.empty_like(s["y"])
    dy[back] = (d * s["share"][:, :, None]).to(dy.dtype)
    return dy, (v * d).sum(2)


def _run_plain(s):
    if s["op"].startswith("norm"):
        return _plain_norm(s)
    if s["op"].startswith("route"):
        return _plain_route(s)
    return _plain_sort(s) if s["op"] == "sort" else _plain_rows(s)


# ---- what is exact, and what it takes -------------------------------------------------------------------------------------------

def _exact_norm(s):
    op, w = s["op"], s["w"].double()
    if op == "norm_backward":
        x, w = s["x"].double().requires_grad_(), w.requires_grad_()
        y = x * (x.square().mean(1, keepdim=True) + _EPS).rsqrt() * w
        dx, dw = torch.autograd.grad(y, (x, w), s["dy"].double())
        return dx if s["more"] is None else dx + s["more"].double(), dw
    total = s["x"].double() if s["r"] is None else s["x"].double() + s["r"].double()
    v = total if s["r"] is None else total.to(s["r"].dtype).double()        # (what is kept is what is normalised)
    y = v * (v.square().mean(1, keepdim=True) + _EPS).rsqrt() * w
    out = [y] if op == "norm" or s["keep"] else []
    if op == "norm_fp8":
        rows, cols = y.shape
        padded = torch.nn.functional.pad(y, (0, -cols % _BLOCK)).view(rows, -1, _BLOCK)
        scale = padded.abs().amax(2).clamp_min(_FLOOR) / _TOP
        out = [(padded / scale[:, :, None]).reshape(rows, -1)[:, :cols], scale.t().contiguous(), *out]    # (the codes' values before their rounding)
    if s["r"] is not None:
        out.append(total)
    return out[0] if len(out) == 1 else tuple(out)


def _exact_route(s):
    """Shares of the plain form's choice, from the logarithms of the scores."""
    choice = s["choice"] if s["op"] == "route_backward" else _choose(s)[0]
    on, at = choice >= 0, choice.long().clamp_min(0)
    v = s["logits"].double().requires_grad_(s["op"] == "route_backward")
    row = s["logits"] > -math.inf
    u = torch.where(row, v, -1e4)
    u = torch.nn.functional.logsigmoid(u) if s["score"] == "sigmoid" else torch.log_softmax(u, 1)
    u = torch.where(on, u.gather(1, at), -math.inf)
    if s["renormalize"]:
        u = torch.where(on, u - torch.where(on.any(1, keepdim=True), u, 0.0).logsumexp(1, keepdim=True), -math.inf)
    share = torch.exp(u) * s["scale"]
    if s["op"] == "route":
        return None, share
    return torch.autograd.grad(share, v, s["dshare"].double())[0]


def _exact_rows(s):
    op, back = s["op"], s["back"].long()
    if op == "spread":
        tokens = torch.div(torch.argsort(back.view(-1)), s["top"], rounding_mode="floor")
        rows = s["x"].float().double()[tokens]
        return rows if s["scale"] is None else (rows, s["scale"].double()[:, tokens])
    share = torch.ones(back.shape, dtype=torch.float64, device=DEV) if s["share"] is None else s["share"].double()
    if op == "gather":
        out = torch.zeros((s["tokens"], s["cols"]), dtype=torch.float64, device=DEV)
        for j in range(s["top"]):
            out.addcmul_(s["y"].double()[back[:, j]], share[:, j:j + 1])
        return out
    d = s["x"].double()
    dy, dshare = torch.zeros(s["y"].shape, dtype=torch.float64, device=DEV), torch.zeros_like(share)
    for j in range(s["top"]):
        dy[back[:, j]] = d * share[:, j:j + 1]
        dshare[:, j] = torch.linalg.vecdot(s["y"].double()[back[:, j]], d)
    return dy, dshare


def exact(case, seed):
    if case["op"] == "sort":
        return None
    s = prepare(case, seed)
    if case["op"].startswith("norm"):
        return _exact_norm(s)
    return _exact_route(s) if case["op"].startswith("route") else _exact_rows(s)


def work(case):
    op = case["op"]
    if op.startswith("norm"):
        rows, cols, es = case["rows"], case["cols"], _SIZE[case["dtype"]]
        rs = 0 if case["residual"] == "none" else _SIZE[case["residual"]]
        w = cols * (es if case["weight"] == "same" else 4)
        values = rows * cols
        if op == "norm_backward":
            return {"bytes": values * (es + (3 * rs if rs else 2 * es)) + 2 * w, "flops": 12 * values}
        out = (es if op == "norm" or case["keep"] else 0) + (1 if op == "norm_fp8" else 0)
        scales = 4 * rows * -(-cols // _BLOCK) if op == "norm_fp8" else 0
        return {"bytes": values * (es + 2 * rs + out) + w + scales, "flops": (8 if op == "norm_fp8" else 5) * values}
    if op.startswith("route"):
        logits, chosen = case["tokens"] * case["experts"], case["tokens"] * case["top"]
        if op == "route":
            return {"bytes": logits * _SIZE[case["dtype"]] + 8 * chosen + (4 * case["experts"] if case["bias"] else 0), "flops": 4 * logits + 4 * chosen}
        return {"bytes": 2 * logits * _SIZE[case["dtype"]] + 8 * chosen, "flops": 6 * logits + 6 * chosen}
    if op == "sort":
        return {"bytes": 12 * case["tokens"] * case["top"] + 4 * case["experts"], "flops": 0}
    tokens, chosen, cols, es = case["tokens"], case["tokens"] * case["top"], case["cols"], _SIZE[case["dtype"]]
    scales = 4 * -(-cols // _BLOCK) if case["dtype"] == "e4m3" else 0
    index = 4 * chosen + (4 * chosen if case["shares"] and op != "spread" else 0)
    if op == "gather_backward":
        return {"bytes": (tokens + 2 * chosen) * cols * es + index + 4 * chosen, "flops": 3 * chosen * cols}
    return {"bytes": (tokens + chosen) * (cols * es + scales) + index, "flops": 0 if op == "spread" else 2 * chosen * cols}
