"""The operators around a layer of experts (norm, router, sort, rows to their experts and back) against plain implementations in 64 bits.

Tolerances, from the arithmetic alone, with u = 2^-24 and U the half step of a result's type (below its normal numbers: half its smallest step):
  norms       a thread adds at most 32 squares one after the other, lanes, waves and groups add another 24 levels at most: a mean of squares is within 64 u, its root
              within 34 u, y (three more products) within 40 u and its rounding.  A signed sum is within 64 u of its magnitudes' sum.
  dw          a sum of so many rows in any order: rows u of the magnitudes' sum, and the 40 u of n
  shares      e^x in fp32 is within 2 u of its value and moves by |x| u with its argument's rounding; sums of at most 1024 positive values within 64 u
  gathers     a sum of `top` products in fp32: (top + 1) u of the magnitudes' sum; dot products of `cols`: cols u
Whole numbers are equal, sums that are rounded as the formula says are equal bit for bit."""
import numpy as np
import pytest
import torch

from mm_rs_with_catlass_amd import lib as L
from mm_rs_with_catlass_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F8 = torch.float8_e4m3fn
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
u = 2.0 ** -24
HALF = {t: torch.finfo(t).eps / 2 for t in (BF16, F16, F32)}
LEAST = {BF16: 2.0 ** -134, F16: 2.0 ** -25, F32: 2.0 ** -150}      # half of the smallest step


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(g, *shape, dtype=F32):
    return torch.randn(shape, device=DEV, generator=g).to(dtype)


def near(got, want, bound, dtype=None):
    """|got - want| <= bound, and the rounding to dtype; every value."""
    got, want = got.double(), want.double()
    assert got.shape == want.shape
    if dtype is not None:
        bound = bound + HALF[dtype] * (want.abs() + bound) + LEAST[dtype]
    off = (got - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), "%d of %d off, worst %.3g times the bound" % (int(bad.sum()), bad.numel(), float((off / bound).nan_to_num(1e30).max()))


def bits(t):
    return t.contiguous().view(torch.uint8)


def moved(t, by):
    """The same values `by` elements behind the start of their memory."""
    room = torch.empty(t.numel() + by, dtype=t.dtype, device=t.device)
    room[by:] = t.reshape(-1)
    return room[by:].view(t.shape)


def blocks(n):
    return -(-n // 128)


def stream(g, rows, cols, dtype):
    v = randn(g, rows, cols) * torch.exp(0.5 * randn(g, rows, 1))
    return (v * (1 + 15 * (torch.rand((1, cols), device=DEV, generator=g) < 0.02))).to(dtype)


# ---- norm -------------------------------------------------------------------------------------------------------------------------------

def plain_norm(x, w, r, eps):
    """(s as it is kept, y in 64 bits)"""
    s = x if r is None else (x.float() + r.float()).to(r.dtype)
    v = s.double()
    return s, v / (v.square().mean(1, keepdim=True) + eps).sqrt() * w.double()


def codes_are_near(q, scale, y, slack):
    rows, cols = y.shape
    top = torch.nn.functional.pad(y.abs(), (0, -cols % 128)).view(rows, -1, 128).amax(2)
    want = top.clamp_min(2.0 ** -40).t() / 448
    assert scale.shape == want.shape and ((scale.double() - want).abs() <= (slack + 3 * u) * want).all()
    t = y / scale.double().t()[:, torch.arange(cols, device=y.device) // 128]
    step = torch.exp2(torch.floor(torch.log2(t.abs().clamp_min(2.0 ** -6))) - 3)      # e4m3: three bits behind the leading one, 2^-9 at least
    assert ((q.double() - t).abs() <= step / 2 + (slack + 4 * u) * t.abs()).all()


NORMS = [(1, 1), (1, 128), (3, 127), (5, 512), (7, 513), (64, 1000), (130, 1024), (33, 1025), (16, 2048), (9, 2050), (257, 1808), (5, 4096), (6, 4097), (3, 8192), (4, 7777), (3, 8193), (2, 16384),
         (1030, 1500), (4110, 300), (1025, 4100), (4099, 1000)]
TYPES = [(BF16, None, BF16), (BF16, BF16, F32), (BF16, F32, BF16), (F16, F16, F16), (F16, F32, F32), (F32, None, F32), (F32, F32, F32)]


@pytest.mark.parametrize("rows,cols", NORMS)
@pytest.mark.parametrize("dtype,rtype,wtype", TYPES)
def test_norm(rows, cols, dtype, rtype, wtype):
    g = gen(rows + 7 * cols)
    x, w, r = stream(g, rows, cols, dtype), (1 + 0.3 * randn(g, cols)).to(wtype), None if rtype is None else stream(g, rows, cols, rtype)
    s, y = plain_norm(x, w, r, 1e-5)
    got = ops.rms_norm(x, w, r, eps=1e-5)
    q = ops.rms_norm_fp8(x, w, r, eps=1e-5, keep=True)
    short = ops.rms_norm_fp8(x, w, r, eps=1e-5)
    if r is not None:
        assert torch.equal(got[1], s) and torch.equal(q[3], s) and torch.equal(short[2], s)
        got = got[0]
    assert got.dtype == dtype
    near(got, y, 40 * u * y.abs(), dtype)
    assert torch.equal(got, q[2])
    codes_are_near(q[0], q[1], y, 40 * u)
    assert torch.equal(bits(q[0]), bits(short[0])) and torch.equal(q[1], short[1])


def test_norm_in_place_and_into_given_tensors():
    g = gen(1)
    for cols in (200, 1500, 9000):
        x, w, r = stream(g, 70, cols, BF16), randn(g, cols, dtype=BF16), stream(g, 70, cols, BF16)
        want = ops.rms_norm(x, w, r)
        y, s = x.clone(), r.clone()
        got = ops.rms_norm(y, w, s, out=y, residual_out=s)
        assert got[0] is y and got[1] is s and torch.equal(y, want[0]) and torch.equal(s, want[1])
        want = ops.rms_norm_fp8(x, w, r, keep=True)
        q, scale, y, s = (torch.empty_like(t) for t in want)
        got = ops.rms_norm_fp8(x, w, r, keep=True, out=q, scale=scale, kept=y, residual_out=s)
        assert [a is b for a, b in zip(got, (q, scale, y, s))] == [True] * 4
        assert all(torch.equal(bits(a), bits(b)) for a, b in zip(got, want))


@pytest.mark.parametrize("by", [1, 2, 4, 8])
def test_norm_at_any_address(by):
    g = gen(by)
    for cols in (130, 1001, 4096):
        x, w, r = stream(g, 20, cols, BF16), randn(g, cols), stream(g, 20, cols, F32)
        want = ops.rms_norm_fp8(x, w, r, keep=True)
        got = ops.rms_norm_fp8(moved(x, by), moved(w, by), moved(r, by), keep=True, out=moved(want[0], by), scale=moved(want[1], by), kept=moved(want[2], by),
                               residual_out=moved(want[3], by))
        assert all(torch.equal(bits(a), bits(b)) for a, b in zip(got, want))
        dy = stream(g, 20, cols, BF16)
        want = ops.rms_norm_backward(dy, r, w, r)
        got = ops.rms_norm_backward(moved(dy, by), moved(r, by), moved(w, by), moved(r, by), dx=moved(r, by), dw=moved(w, by))
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_norm_of_zeros_and_of_values_that_are_not_finite():
    x = torch.ones((5, 300), device=DEV)
    x[0] = 0
    x[1, 7], x[2, 8] = float("nan"), float("inf")
    x[3] = 2.0 ** -70                     # whose squares are nothing beside eps
    w = torch.full((300,), 2.0, device=DEV)
    y = ops.rms_norm(x, w, eps=1e-6)
    assert (y[0] == 0).all() and y[1].isnan().all()
    assert y[2, 8].isnan() and (y[2, :8] == 0).all()
    near(y[3], torch.full((300,), 2.0 ** -69 * 1e3, dtype=torch.float64, device=DEV), 2.0 ** -69 * 1e3 * 40 * u)
    near(y[4], torch.full((300,), 2.0, dtype=torch.float64, device=DEV) / (1 + 1e-6) ** 0.5, 80 * u)
    q, scale = ops.rms_norm_fp8(x, w, eps=1e-6)
    want_q, want_scale = ops.quantize_fp8(y)
    assert torch.equal(scale.isnan(), want_scale.isnan()) and torch.equal(q.float().isnan(), want_q.float().isnan())
    assert (q[0].float() == 0).all() and torch.equal(bits(q[4]), bits(want_q[4]))
    assert (ops.rms_norm(x[:1], w, eps=0.0).isnan()).all()                # (0 / 0)


@pytest.mark.parametrize("rows,cols", [(0, 64), (1, 1), (1, 300), (7, 513), (8, 1024), (600, 1000), (1025, 2048), (37, 1999), (1500, 4096), (130, 4100), (515, 8192), (20, 8200), (5, 16384), (5000, 256), (2050, 2100), (2049, 4100), (300, 16000)])
@pytest.mark.parametrize("dtype,stype,wtype", [(BF16, BF16, BF16), (BF16, F32, F32), (F16, F16, F32), (F16, F32, F16), (F32, F32, F32)])
@pytest.mark.parametrize("more", [False, True])
def test_norm_backward(rows, cols, dtype, stype, wtype, more):
    g = gen(rows + 3 * cols)
    x, dy, w = stream(g, rows, cols, stype), stream(g, rows, cols, dtype), (1 + 0.3 * randn(g, cols)).to(wtype)
    dsum = stream(g, rows, cols, stype) if more else None
    dx, dw = ops.rms_norm_backward(dy, x, w, dsum, eps=1e-5)
    assert dx.dtype == stype and dw.dtype == wtype
    v, d, c = x.double(), dy.double(), w.double()
    r = 1 / (v.square().mean(1, keepdim=True) + 1e-5).sqrt()
    n, gr = v * r, d * c
    mean, size = (gr * n).mean(1, keepdim=True), (gr * n).abs().mean(1, keepdim=True)
    want = r * (gr - n * mean) + (dsum.double() if more else 0)
    # (n within 36 u, the mean within 64 + 36 + 4 u of its magnitudes', their product and r within another 80)
    bound = u * r * (44 * gr.abs() + 190 * n.abs() * size) + (2 * u * want.abs() + 2 * u * dsum.double().abs() if more else 2 * u * want.abs())
    near(dx, want, bound, stype)
    near(dw, (d * n).sum(0), (rows + 40) * u * (d * n).abs().sum(0), wtype)
    if more and rows:                                    # into the sum's own gradient
        again = ops.rms_norm_backward(dy, x, w, dsum, eps=1e-5, dx=dsum)
        assert again[0] is dsum and torch.equal(dsum, dx) and torch.equal(again[1], dw)


def test_norm_gradient_against_differences():
    """In fp32 along one direction: central differences of step h are off by h^2 of a third derivative, and by the values' roundings over h."""
    g = gen(3)
    rows, cols, h = 6, 96, 2.0 ** -6
    x, w, dy, tx, tw = randn(g, rows, cols), 1 + 0.2 * randn(g, cols), randn(g, rows, cols), randn(g, rows, cols), randn(g, cols)

    def f(a, b):
        return (ops.rms_norm(a, b).double() * dy.double()).sum()
    dx, dw = ops.rms_norm_backward(dy, x, w)
    for got, want in (((dx * tx).double().sum(), (f(x + h * tx, w) - f(x - h * tx, w)) / (2 * h)), ((dw * tw).double().sum(), (f(x, w + h * tw) - f(x, w - h * tw)) / (2 * h))):
        # third derivative along t: at most about 15 |t|^3 / |x|^3 of y's own size, all of them together 6 * 96 * 15 / 6 h^2; roundings 2^-22 * 6 * 96 / h
        assert abs(got - want) <= 1440 * h * h + 576 * 2.0 ** -22 / h


def test_norm_past_4_gib():
    rows, cols = 140000, 16384
    w = torch.ones(cols, dtype=BF16, device=DEV)
    x = torch.empty((rows, cols), dtype=BF16, device=DEV)
    last = stream(gen(4), 3, cols, BF16)
    x[-3:] = last
    x[:3] = last
    q, scale, y = ops.rms_norm_fp8(x, w, keep=True)
    want = ops.rms_norm_fp8(last, w, keep=True)
    assert torch.equal(y[-3:], want[2]) and torch.equal(bits(q[-3:]), bits(want[0])) and torch.equal(scale[:, -3:], want[1])
    assert torch.equal(y[:3], want[2])
    del q, scale
    dx, _ = ops.rms_norm_backward(y, x, w)
    assert torch.equal(dx[-3:], ops.rms_norm_backward(want[2], last, w)[0])


# ---- router -----------------------------------------------------------------------------------------------------------------------------

def plain_route(logits, top, score="softmax", bias=None, groups=1, top_groups=1, group_top=1, renormalize=True, scale=1.0):
    """Token by token, in 64 bits, on the host: (choice, share)."""
    l = logits.double().cpu().numpy()
    b = None if bias is None else bias.double().cpu().numpy()
    tokens, experts = l.shape
    choice, share = np.full((tokens, top), -1, np.int32), np.zeros((tokens, top))
    with np.errstate(all="ignore"):
        for t in range(tokens):
            v = l[t]
            if score == "softmax":
                p = np.exp(v - v.max()) / np.exp(v - v.max()).sum()
            else:
                p = 1 / (1 + np.exp(-v))
            plain = b is None and group_top == 1
            key = v.copy() if plain else p + (0 if b is None else b)
            key[np.isnan(key)] = np.inf
            key[v == -np.inf] = -np.inf
            if top_groups < groups:
                by = key.reshape(groups, -1)
                best = -np.sort(-by, 1)[:, :group_top]
                best = np.where(best[:, 0] == -np.inf, -np.inf, np.where(best == -np.inf, 0, best).sum(1))
                out = np.argsort(-best, kind="stable")[top_groups:]
                by[out] = -np.inf
            order = np.argsort(-key, kind="stable")[:top]
            order = order[key[order] > -np.inf]
            if order.size == 0:
                continue
            if renormalize:
                a = v[order] - v[order].max()
                a = np.exp(a) if score == "softmax" else np.exp(-np.logaddexp(0, -v[order]) - (-np.logaddexp(0, -v[order])).max())
                w = a / a.sum()
            else:
                w = p[order]
            choice[t, :order.size], share[t, :order.size] = order, w * scale
    return torch.from_numpy(choice).to(DEV), torch.from_numpy(share).to(DEV)


def shares_are_near(got, want, logits, scale=1.0):
    spread = torch.where(logits.double().abs() < 200, logits.double(), 0.0)
    spread = (spread.amax(1, keepdim=True) - spread.amin(1, keepdim=True)).clamp_min(spread.abs().amax(1, keepdim=True))
    near(got, want, (2 * spread + 80) * u * want.abs() + 2.0 ** -126 * abs(scale))


ROUTES = [(1, 8, 2, {}), (33, 64, 8, {}), (1000, 60, 4, {}), (5, 1, 1, {}), (7, 3, 3, {}), (19, 16, 16, {}), (70, 256, 8, {}), (9, 257, 5, {}), (65, 512, 10, {}), (11, 1024, 8, {}),
          (6, 100, 17, {}), (4, 64, 64, {}), (5, 1000, 64, {}), (21, 31, 7, {}), (50, 2, 1, {}),
          (100, 256, 8, dict(groups=8, top_groups=4, group_top=2)), (40, 256, 8, dict(groups=8, top_groups=3)), (33, 60, 4, dict(groups=4, top_groups=2, group_top=2)),
          (30, 160, 6, dict(groups=8, top_groups=3)), (13, 24, 2, dict(groups=3, top_groups=1, group_top=2)), (12, 64, 2, dict(groups=64, top_groups=5)),
          (9, 1020, 3, dict(groups=17, top_groups=4, group_top=2)), (9, 660, 20, dict(groups=33, top_groups=16, group_top=2)), (9, 96, 8, dict(groups=6, top_groups=6, group_top=2)),
          (17, 32, 4, dict(groups=16, top_groups=4, group_top=2)), (8, 63, 5, dict(groups=63, top_groups=7, group_top=2))]


@pytest.mark.parametrize("tokens,experts,top,how", ROUTES)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype,biased,renormalize,scale", [(F32, False, True, 1.0), (BF16, False, False, 1.0), (F16, True, True, 2.5), (F32, True, False, 0.5)])
def test_route(tokens, experts, top, how, score, dtype, biased, renormalize, scale):
    g = gen(tokens + 5 * experts + top)
    logits = (randn(g, tokens, experts) * 1.5).to(dtype)
    bias = 0.1 * randn(g, experts) if biased else None
    choice, share = ops.route(logits, top, score=score, bias=bias, renormalize=renormalize, scale=scale, **how)
    want = plain_route(logits, top, score, bias, renormalize=renormalize, scale=scale, **how)
    assert choice.dtype == torch.int32 and share.dtype == F32
    assert torch.equal(choice, want[0])
    shares_are_near(share, want[1], logits, scale)


@pytest.mark.parametrize("how", [{}, dict(groups=4, top_groups=2), dict(groups=4, top_groups=2, group_top=2)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("renormalize", [False, True])
def test_route_of_ties_masks_and_values_that_are_not_finite(how, score, biased, renormalize):
    low, inf, nan = torch.finfo(F32).min, float("inf"), float("nan")
    rows = torch.zeros((14, 16), device=DEV)
    rows[1] = -1.0
    rows[2, 5:] = -inf                              # five experts are left
    rows[3, 1:] = -inf                              # one
    rows[4] = -inf                                  # none
    rows[5] = low                                   # all masked by the type's lowest value
    rows[6, 3:] = low
    rows[7, ::2], rows[7, 1::2] = 0.0, -0.0         # equal all the same
    rows[8] = torch.arange(16, device=DEV) // 4     # ties within and across groups
    rows[9] = -torch.arange(16, device=DEV) % 3
    rows[10] = 50.0
    rows[11] = -95.0                                # whose sigmoids are below fp32's normal numbers
    rows[11, 7] = -94.0
    rows[12, 9] = nan
    rows[13, 4], rows[13, 11] = inf, 1.0
    bias = torch.zeros(16, device=DEV) if biased else None
    choice, share = ops.route(rows, 6, score=score, bias=bias, renormalize=renormalize, **how)
    want, want_share = plain_route(rows[:12], 6, score, bias, renormalize=renormalize, **how)
    if score == "sigmoid" and renormalize:          # (all scores are 0: as many equal ones)
        want_share[5] = torch.where(want[5] >= 0, 1 / 6, 0.0)
    if score == "softmax" and not biased and how.get("group_top") != 2:
        assert choice[13, 0] == 4
    assert torch.equal(choice[:12], want)
    shares_are_near(share[:12], want_share, rows[:12])
    assert choice[12, 0] == 9 or score == "softmax"
    assert share[12, 0].isnan() and (share[12].isnan().all() or (score == "sigmoid" and not renormalize))
    assert (choice[4] == -1).all() and (share[4] == 0).all()
    for line in choice.tolist():
        got = [c for c in line if c >= 0]
        assert len(set(got)) == len(got) and all(c < 16 for c in got)


def test_route_biases_that_mask():
    g = gen(6)
    logits, bias = randn(g, 40, 12), torch.zeros(12, device=DEV)
    bias[3] = bias[7] = -float("inf")
    choice, share = ops.route(logits, 11, score="sigmoid", bias=bias)
    assert not ((choice == 3) | (choice == 7)).any() and (choice[:, 10] == -1).all() and (share[:, 10] == 0).all()
    near(share.double().sum(1), torch.ones(40, device=DEV), 80 * u)
    apart = logits.clone()
    apart[:, [3, 7]] = -float("inf")
    assert torch.equal(choice, ops.route(apart, 11, score="sigmoid")[0])


def test_route_decides_by_more_than_fp32():
    """Scores that differ by 2^-27 of themselves: the same in fp32, not in the order."""
    logits = torch.zeros((64, 8), device=DEV)
    for i in range(64):
        logits[i, i % 8] = 2.0 ** -26
    for score in ("softmax", "sigmoid"):
        choice, _ = ops.route(logits, 3, score=score, bias=torch.ones(8, device=DEV))
        want = plain_route(logits, 3, score, torch.ones(8, device=DEV))[0]
        assert torch.equal(choice, want) and torch.equal(choice[:, 0].cpu(), torch.arange(64, dtype=torch.int32) % 8)


@pytest.mark.parametrize("tokens,experts,top", [(1, 8, 2), (33, 64, 8), (1000, 60, 4), (19, 16, 16), (70, 256, 8), (9, 257, 5), (11, 1024, 64), (5, 1, 1), (21, 31, 7)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype,renormalize,scale", [(F32, True, 1.0), (BF16, False, 2.5), (F16, True, 0.5), (F32, False, 1.0)])
def test_route_backward(tokens, experts, top, score, dtype, renormalize, scale):
    g = gen(tokens + experts + top)
    logits, dshare = (randn(g, tokens, experts) * 1.5).to(dtype), randn(g, tokens, top)
    choice, _ = ops.route(logits, top, score=score)
    got = ops.route_backward(dshare, logits, choice, score=score, renormalize=renormalize, scale=scale)
    assert got.dtype == dtype
    v = logits.double().requires_grad_()
    p = (torch.softmax(v, 1) if score == "softmax" else torch.sigmoid(v)).gather(1, choice.long())
    share = (p / p.sum(1, keepdim=True) if renormalize else p) * scale
    want, = torch.autograd.grad(share, v, dshare.double())
    # each logit's gradient is a share times a difference of two values no larger than the largest |g|, shares being within (2 * 12 + 80) u
    size = (share.detach().sum(1, keepdim=True) * dshare.double().abs().amax(1, keepdim=True))
    near(got, want, 2 * 110 * u * size, dtype)


def test_route_backward_of_choices_that_are_none_or_come_twice():
    g = gen(8)
    logits = randn(g, 5, 6)
    logits[3] = -float("inf")
    logits[4, 2:] = -float("inf")
    choice = torch.tensor([[1, -1, 4], [2, 2, 0], [6, -5, 3], [-1, -1, -1], [1, 0, -1]], dtype=torch.int32, device=DEV)
    dshare = randn(g, 5, 3)
    for score in ("softmax", "sigmoid"):
        for renormalize in (False, True):
            got = ops.route_backward(dshare, logits, choice, score=score, renormalize=renormalize)
            assert got.isfinite().all() and not got[3].any() and not got[4, 2:].any()
            v = logits.double().requires_grad_()
            p = torch.softmax(v, 1) if score == "softmax" else torch.sigmoid(v)
            on = (choice >= 0) & (choice < 6)
            p = torch.where(on, p.gather(1, choice.long().clamp(0, 5)), 0.0)
            share = p / p.sum(1, keepdim=True) if renormalize else p
            keep = [0, 1, 2, 4]
            want, = torch.autograd.grad(share[keep], v, dshare.double()[keep])
            near(got[keep], want[keep].nan_to_num(0.0), 2 * 110 * u * dshare.double().abs().amax(1, keepdim=True)[keep])


def test_route_gradient_against_differences():
    g = gen(9)
    logits, dshare, t, h = randn(g, 7, 20), randn(g, 7, 5), randn(g, 7, 20), 2.0 ** -7
    choice, _ = ops.route(logits, 5)
    for score in ("softmax", "sigmoid"):
        for renormalize in (False, True):
            def f(v):
                v = v.double()
                p = (torch.softmax(v, 1) if score == "softmax" else torch.sigmoid(v)).gather(1, choice.long())
                return ((p / p.sum(1, keepdim=True) if renormalize else p) * dshare.double()).sum()
            got = (ops.route_backward(dshare, logits, choice, score=score, renormalize=renormalize).double() * t.double()).sum()
            want = (f(logits.double() + h * t.double()) - f(logits.double() - h * t.double())) / (2 * h)
            # a share's third derivative along t is at most (2 max |t|)^3 of it, and |g| at most 4: 7 rows of shares that sum to 5 at most, h^2 / 6 of that
            assert abs(got - want) <= 7 * 5 * 4 * (2 * float(t.abs().max())) ** 3 * h * h / 6 + 1e-5


# ---- rows by expert ---------------------------------------------------------------------------------------------------------------------

def plain_sort(choice, experts):
    flat = choice.cpu().numpy().reshape(-1).astype(np.int64)
    flat = np.where((flat < 0) | (flat >= experts), experts, flat)
    order = np.argsort(flat, kind="stable")
    back = np.empty_like(order)
    back[order] = np.arange(order.size)
    ends = np.searchsorted(flat[order], np.arange(experts), side="right")
    return [torch.from_numpy(a.astype(np.int32)).to(DEV) for a in (order, back.reshape(choice.shape), ends)]


SORTS = [(0, 2, 5), (1, 1, 1), (1, 8, 64), (63, 1, 7), (64, 1, 7), (65, 2, 8), (300, 3, 60), (1024, 1, 256), (1025, 7, 255), (4096, 2, 256), (4097, 2, 257), (8192, 1, 128), (8193, 1, 128),
         (9000, 4, 1024), (16384, 8, 128), (40000, 8, 160), (300001, 1, 31), (70000, 6, 1000), (600001, 1, 8), (1200003, 1, 5), (16384, 1, 9), (16385, 1, 9), (4096, 8, 100), (4097, 8, 100), (5000, 3, 3),
         (150000, 8, 64)]


@pytest.mark.parametrize("tokens,top,experts", SORTS)
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("kind", ["even", "few", "dropped"])
def test_sort(tokens, top, experts, dtype, kind):
    g = gen(tokens + top + experts)
    choice = torch.randint(0, experts if kind == "even" else min(experts, 2), (tokens, top), device=DEV, generator=g).to(dtype)
    if kind == "dropped":
        choice = torch.randint(-3, experts + 5, (tokens, top), device=DEV, generator=g).to(dtype)
    for got, want in zip(ops.sort_by_expert(choice, experts), plain_sort(choice, experts)):
        assert got.dtype == torch.int32 and torch.equal(got, want)


def test_sort_of_choices_past_32_bits():
    choice = torch.tensor([[2 ** 32, 1], [-2 ** 32 + 1, 0], [2 ** 40 + 1, 2]], device=DEV)       # (whose low halves are experts)
    for got, want in zip(ops.sort_by_expert(choice, 3), plain_sort(choice, 3)):
        assert torch.equal(got, want)
    choice = torch.tensor([[2 ** 31 - 1, -2 ** 31, 0]], dtype=torch.int32, device=DEV)
    assert ops.sort_by_expert(choice, 1)[0].tolist() == [2, 0, 1]


# ---- rows to their experts and back -----------------------------------------------------------------------------------------------------

def places(g, tokens, top):
    return torch.randperm(tokens * top, device=DEV, generator=g).to(torch.int32).view(tokens, top)


ROWS = [(0, 2, 64), (1, 1, 1), (1, 8, 4096), (3, 2, 7), (37, 3, 129), (65, 8, 512), (20, 1, 513), (33, 6, 1000), (9, 2, 1025), (130, 4, 2048), (17, 9, 2050), (5, 64, 300), (600, 2, 1808),
        (4100, 2, 256), (2100, 1, 8192), (9, 5, 20001)]


@pytest.mark.parametrize("tokens,top,cols", ROWS)
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_rows_there_and_back(tokens, top, cols, dtype):
    g = gen(tokens + top + cols)
    back, share = places(g, tokens, top), torch.rand((tokens, top), device=DEV, generator=g) - 0.3
    x, y = stream(g, tokens, cols, dtype), stream(g, tokens * top, cols, dtype)
    rows = ops.spread_rows(x, back)
    want = torch.empty_like(rows)
    want[back.long().view(-1)] = x.repeat_interleave(top, 0)
    assert torch.equal(rows, want)
    at = y.double()[back.long()]                                        # [tokens, top, cols]
    for s in (None, share):
        part = at if s is None else at * s.double()[:, :, None]
        near(ops.gather_rows(y, back, s), part.sum(1), (top + 1) * u * part.abs().sum(1), dtype)
    dy, dshare = ops.gather_rows_backward(x, y, back, share)
    want = torch.empty((tokens * top, cols), dtype=torch.float64, device=DEV)
    want[back.long()] = x.double()[:, None, :] * share.double()[:, :, None]
    near(dy, want, 2 * u * want.abs(), dtype)
    part = at * x.double()[:, None, :]
    near(dshare, part.sum(2), (cols + 1) * u * part.abs().sum(2))


@pytest.mark.parametrize("tokens,top,cols", [(0, 2, 256), (1, 1, 1), (3, 8, 4096), (40, 2, 1000), (70, 3, 129), (65, 4, 130), (2048, 8, 512), (9, 2, 15), (5, 3, 9000)])
def test_e4m3_rows_go_with_their_scales(tokens, top, cols):
    g = gen(tokens + cols)
    back = places(g, tokens, top)
    q, scale = (randn(g, tokens, cols) * 60).clamp(-448, 448).to(F8), torch.rand((blocks(cols), tokens), device=DEV, generator=g)
    rows, scales = ops.spread_rows(q, back, scale)
    to = back.long().view(-1)
    want, want_scales = torch.empty_like(bits(rows)), torch.empty_like(scales)
    want[to] = bits(q).repeat_interleave(top, 0)
    want_scales[:, to] = scale.repeat_interleave(top, 1)
    assert torch.equal(bits(rows), want) and torch.equal(scales, want_scales)
    assert torch.equal(bits(ops.spread_rows(q, back)), want)
    if tokens:                                      # quantizing before and after is the same
        x = randn(g, tokens, cols, dtype=BF16)
        late = ops.quantize_fp8(ops.spread_rows(x, back))
        early = ops.spread_rows(*(t if i else ops.quantize_fp8(x)[0] for i, t in enumerate([None, back])), scale=ops.quantize_fp8(x)[1])
        assert torch.equal(bits(late[0]), bits(early[0])) and torch.equal(late[1], early[1])


@pytest.mark.parametrize("by", [1, 2, 3, 4, 8])
def test_rows_at_any_address(by):
    g = gen(by)
    for cols in (130, 1001, 2048):
        back, share = places(g, 30, 3), torch.rand((30, 3), device=DEV, generator=g)
        x, y = stream(g, 30, cols, BF16), stream(g, 90, cols, BF16)
        q, scale = ops.quantize_fp8(x)
        mb, ms = moved(back, by), moved(share, by)
        assert torch.equal(ops.spread_rows(moved(x, by), mb, out=moved(y, by)), ops.spread_rows(x, back))
        a, b = ops.spread_rows(moved(q, by), mb, moved(scale, by)), ops.spread_rows(q, back, scale)
        assert torch.equal(bits(a[0]), bits(b[0])) and torch.equal(a[1], b[1])
        assert torch.equal(ops.gather_rows(moved(y, by), mb, ms, out=moved(x, by)), ops.gather_rows(y, back, share))
        a, b = ops.gather_rows_backward(moved(x, by), moved(y, by), mb, ms, dy=moved(y, by)), ops.gather_rows_backward(x, y, back, share)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_places_outside_the_rows_are_left_out():
    g = gen(10)
    back = torch.tensor([[0, -1], [5, 3], [6, -2 ** 31]], dtype=torch.int32, device=DEV)        # six rows: 0..5
    x, y, share = randn(g, 3, 200, dtype=BF16), randn(g, 6, 200, dtype=BF16), torch.full((3, 2), 0.5, device=DEV)
    y[1] = y[2] = y[4] = float("nan")               # rows that no choice has
    marked = torch.full((6, 200), 7.0, dtype=BF16, device=DEV)
    want = marked.clone()
    want[0], want[5], want[3] = x[0], x[1], x[1]
    assert torch.equal(ops.spread_rows(x, back, out=marked.clone()), want)
    out = ops.gather_rows(y, back, share)
    assert torch.equal(out[0], (0.5 * y[0].float()).to(BF16)) and torch.equal(out[1], (0.5 * y[5].float() + 0.5 * y[3].float()).to(BF16)) and not out[2].any()
    dy, dshare = ops.gather_rows_backward(x, y, back, share, dy=marked.clone())
    want[[0, 5, 3]] = (0.5 * want[[0, 5, 3]].float()).to(BF16)
    assert torch.equal(dy, want) and dshare[0, 1] == 0 and not dshare[2].any() and dshare.isfinite().all()


def test_outputs_on_their_rows_are_refused():
    g = gen(17)
    choice = torch.randint(0, 5, (40, 1), device=DEV, dtype=torch.int32, generator=g)
    x, back = randn(g, 40, 64, dtype=BF16), torch.randperm(40, device=DEV, generator=g).int()[:, None].contiguous()
    kept = choice.clone(), x.clone()
    for match, fn, a, kw in [("back lies", ops.sort_by_expert, (choice, 5), {"back": choice}), ("order lies", ops.sort_by_expert, (choice, 5), {"order": choice.view(-1)}),
                             ("out lies", ops.spread_rows, (x, back), {"out": x}), ("out lies", ops.gather_rows, (x, back), {"out": x}),
                             ("dy lies", ops.gather_rows_backward, (x, x.clone(), back, torch.ones(40, 1, device=DEV)), {"dy": x})]:
        with pytest.raises(L.CatcocError, match=match):
            fn(*a, **kw)
    assert torch.equal(choice, kept[0]) and torch.equal(x, kept[1])


def test_rows_past_4_gib():
    tokens, top, cols = 70000, 4, 8192
    g = gen(11)
    back = torch.arange(tokens * top, dtype=torch.int32, device=DEV).view(tokens, top)
    x = torch.zeros((tokens, cols), dtype=BF16, device=DEV)
    x[-2:] = randn(g, 2, cols, dtype=BF16)
    rows = ops.spread_rows(x, back)
    assert torch.equal(rows[-8:].view(2, top, cols), x[-2:, None].expand(-1, top, -1)) and not rows[-12:-8].any()
    share = torch.full((tokens, top), 0.25, device=DEV)
    assert torch.equal(ops.gather_rows(rows, back, share), x)
    dy, dshare = ops.gather_rows_backward(x, rows, back, share)
    assert torch.equal(dy[-8:], (rows[-8:].float() * 0.25).to(BF16)) and not dy[-12:-8].any()
    near(dshare[-2:], (x[-2:].double() ** 2).sum(1, keepdim=True).expand(-1, top), (cols + 1) * u * (x[-2:].double() ** 2).sum(1, keepdim=True))
    del rows, dy
    q, scale = ops.quantize_fp8(x)
    many = torch.arange(tokens * 8, dtype=torch.int32, device=DEV).view(tokens, 8)
    rows, scales = ops.spread_rows(q, many, scale)
    assert torch.equal(bits(rows[-8:]), bits(q[-1:]).expand(8, -1)) and torch.equal(scales[:, -8:], scale[:, -1:].expand(-1, 8))


def test_logits_past_4_gib():
    tokens, experts = 4_200_000, 260
    g = gen(12)
    logits = torch.zeros((tokens, experts), device=DEV)
    logits[-5:] = randn(g, 5, experts)
    choice, share = ops.route(logits, 4, renormalize=False)
    want = ops.route(logits[-5:], 4, renormalize=False)
    assert torch.equal(choice[-5:], want[0]) and torch.equal(share[-5:], want[1]) and torch.equal(choice[:3].cpu(), torch.arange(4, dtype=torch.int32).expand(3, 4))
    dshare = randn(g, tokens, 4)
    got = ops.route_backward(dshare, logits, choice, renormalize=False)
    assert torch.equal(got[-5:], ops.route_backward(dshare[-5:], logits[-5:], want[0], renormalize=False))


# ---- together, on streams, in graphs ----------------------------------------------------------------------------------------------------

class Everything:
    """One call of each operator, the later ones on what the earlier ones give."""

    def __init__(self, seed):
        g = gen(seed)
        self.tokens, self.cols, self.experts, self.top = 300, 1100, 24, 3
        self.x, self.r, self.w = stream(g, self.tokens, self.cols, BF16), stream(g, self.tokens, self.cols, F32), 1 + 0.1 * randn(g, self.cols)
        self.logits, self.bias = randn(g, self.tokens, self.experts), 0.1 * randn(g, self.experts)
        self.many = torch.randint(-1, 200, (9000, 4), device=DEV, generator=g)

    def inputs(self):
        return [self.x, self.r, self.w, self.logits, self.bias, self.many]

    def run(self):
        q, scale, y, s = ops.rms_norm_fp8(self.x, self.w, self.r, keep=True)
        choice, share = ops.route(self.logits, self.top, score="sigmoid", bias=self.bias, groups=4, top_groups=2, group_top=2)
        order, back, ends = ops.sort_by_expert(choice, self.experts)
        rows, scales = ops.spread_rows(q, back, scale)
        wide = ops.spread_rows(y, back)
        out = ops.gather_rows(wide, back, share)
        dwide, dshare = ops.gather_rows_backward(out, wide, back, share)
        dlogits = ops.route_backward(dshare, self.logits, choice, score="sigmoid")
        dx, dw = ops.rms_norm_backward(ops.gather_rows(dwide, back), s, self.w, s)
        return [bits(q), scale, y, s, choice, share, order, back, ends, bits(rows), scales, wide, out, dwide, dshare, dlogits, dx, dw, *ops.sort_by_expert(self.many, 190),
                ops.rms_norm(self.x, self.w)]


def same(got, want):
    return all(torch.equal(a, b) for a, b in zip(got, want))


def test_together():
    e = Everything(20)
    q, scale, y, s, choice, share, order, back, ends, rows, scales, wide, out = e.run()[:13]
    assert torch.equal(choice, plain_route(e.logits, 3, "sigmoid", e.bias, 4, 2, 2)[0])
    flat = choice.view(-1).long()
    assert torch.equal(flat[order.long()], flat.sort(stable=True).values) and ends[-1] == flat.numel()
    assert torch.equal(wide, y[order.long() // 3]) and torch.equal(rows, q[order.long() // 3]) and torch.equal(scales, scale[:, order.long() // 3])
    near(out, y.double() * share.double().sum(1, keepdim=True), 4 * u * y.double().abs() * share.double().sum(1, keepdim=True), BF16)
    assert same(e.run(), e.run())


def test_behind_their_stream():
    """Operands are written by work that has not run yet when the call is made, results are read by work behind it."""
    e, other = Everything(21), Everything(22)
    want = [t.clone() for t in other.run()]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        for to, values in zip(e.inputs(), other.inputs()):
            to.copy_(values, non_blocking=True)
        got = [t.clone() for t in e.run()]
    side.synchronize()
    assert same(got, want)


def test_calls_on_two_streams_at_once():
    a, b = Everything(25), Everything(26)
    want = [[t.clone() for t in e.run()] for e in (a, b)]
    torch.cuda.synchronize()
    sides = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for i, (e, side) in enumerate(zip((a, b), sides)):
            with torch.cuda.stream(side):
                got[i].append(e.run())
    torch.cuda.synchronize()
    for runs, w in zip(got, want):
        assert all(same(r, w) for r in runs)


def test_two_graphs_replayed_in_turn():
    a, b = Everything(23), Everything(24)
    graphs = []
    for e in (a, b):
        e.run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = e.run()
        graphs.append((e, graph, out))
    for i in range(4):
        other = Everything(30 + i)
        for e, graph, out in graphs:
            for to, values in zip(e.inputs(), other.inputs()):
                to.copy_(values)
        for e, graph, out in graphs:
            graph.replay()
        torch.cuda.synchronize()
        want = other.run()
        for e, graph, out in graphs:
            assert same(out, want), i


class Nothing:
    """In the place of the compiled calls: leaves every call to the Python path."""

    def __getattr__(self, name):
        return lambda *a: None


def test_the_compiled_call_and_the_python_path_answer_alike(monkeypatch):
    g = gen(31)
    x, w, r = stream(g, 20, 300, BF16), randn(g, 300, dtype=BF16), stream(g, 20, 300, F32)
    logits, bias, many = randn(g, 20, 16), randn(g, 16), torch.randint(0, 9, (9000, 2), device=DEV, generator=g)
    choice, share = ops.route(logits, 4)
    order, back, ends = ops.sort_by_expert(choice, 16)
    rows, (q, scale) = ops.spread_rows(x, back), ops.quantize_fp8(x)

    def alike(fn, *a, **kw):
        seen = []
        for host in (None, Nothing()):
            with monkeypatch.context() as m:
                if host is not None:
                    m.setattr(ops, "_host", host)
                try:
                    got = fn(*a, **kw)
                    seen.append([bits(t).clone() for t in (got if isinstance(got, tuple) else (got,))])
                except L.CatcocError as e:
                    seen.append(str(e))
        assert type(seen[0]) is type(seen[1])
        if isinstance(seen[0], str):
            assert seen[0] == seen[1]
            return False
        assert len(seen[0]) == len(seen[1]) and same(*seen)
        return True
    n, f, b, t, tb, s, p, c, cb = (ops.rms_norm, ops.rms_norm_fp8, ops.rms_norm_backward, ops.route, ops.route_backward, ops.sort_by_expert, ops.spread_rows, ops.gather_rows,
                                   ops.gather_rows_backward)
    for fn, a, kw in ((n, (x, w), {}), (n, (x, w, r), {"eps": 1e-3}), (n, (x, w, x), {"eps": 1}), (n, (torch.nn.Parameter(x), w), {}), (n, (x[:0], w), {}),
                      (n, (x, w), {"out": torch.empty_like(x)}), (f, (x, w), {}), (f, (x, w, r, 1e-5, True), {}), (f, (x, w.float(), r), {}), (f, (x, w, None, 1e-6, True), {}),
                      (f, (x, w), {"out": torch.empty_like(q), "scale": torch.empty_like(scale)}), (b, (x, x, w), {}), (b, (x, r, w, r), {}), (b, (x[:0], r[:0], w), {}),
                      (t, (logits, 4), {}), (t, (logits.half(), 4, "sigmoid", bias, 4, 2, 2, False, 2.0), {}), (t, (logits, 4), {"scale": 2}), (t, (logits[:0], 4), {}),
                      (t, (logits, 4), {"choice": torch.empty_like(choice), "share": torch.empty_like(share)}), (tb, (share, logits, choice), {}),
                      (tb, (share, logits.bfloat16(), choice, "sigmoid", False, 2.0), {}), (s, (choice, 16), {}), (s, (many, 9), {}), (s, (many[:0], 9), {}), (s, (many.int(), 700), {}),
                      (p, (x, back), {}), (p, (q, back, scale), {}), (p, (x, back), {"out": torch.empty_like(rows)}), (c, (rows, back), {}), (c, (rows, back, share), {}),
                      (cb, (x, rows, back, share), {}), (cb, (x, rows, back, share), {"dshare": torch.empty_like(share)})):
        assert alike(fn, *a, **kw), (fn.__name__, kw)
    far = torch.zeros((20, 16400), device=DEV)
    for fn, a, kw in ((n, (x, w[1:]), {}), (n, (x[:, ::2], w[::2].contiguous()), {}), (n, (x, w.half()), {}), (n, (x, w, None, -1.0), {}), (n, (far, far[0]), {}), (n, (x.cpu(), w), {}),
                      (n, (x, w), {"residual_out": x}), (f, (x, w), {"kept": x}), (b, (x, x, w, r), {}), (b, (x, r, w), {"dx": x}), (t, (logits, 17), {}), (t, (logits, 4, "relu"), {}),
                      (t, (logits, 4, "softmax", bias.half()), {}), (t, (logits, 4), {"groups": 3}), (t, (logits, 4), {"groups": 8, "top_groups": 1}), (t, (logits, 4), {"group_top": 3}),
                      (t, (logits, 4), {"scale": float("nan")}), (t, (torch.zeros((2, 1025), device=DEV), 4), {}), (tb, (share, logits, choice.long()), {}),
                      (tb, (share[:, 1:], logits, choice), {}), (s, (choice, 0), {}), (s, (choice, 1025), {}), (s, (choice.short(), 16), {}), (p, (x, back[1:]), {}),
                      (p, (x, back.cpu()), {}), (p, (x, back, scale), {}), (p, (x, back[:, :0]), {}), (c, (rows[1:], back), {}), (c, (rows, back, share.half()), {}), (cb, (x, rows, back, None), {}),
                      (cb, (x.float(), rows, back, share), {})):
        assert not alike(fn, *a, **kw), (fn.__name__, kw)


def test_results_are_those_of_their_mode():
    x, w = randn(gen(32), 4, 256, dtype=BF16), torch.ones(256, dtype=BF16, device=DEV)
    with torch.inference_mode():
        got = [ops.rms_norm(x, w), *ops.quantize_fp8(x), *ops.route(x, 2)]
        assert all(t.is_inference() and not t.requires_grad for t in got)
    got = [ops.rms_norm(x, w), *ops.quantize_fp8(x), *ops.route(x, 2)]
    assert not any(t.is_inference() or t.requires_grad for t in got) and all(t.device == x.device and t.is_contiguous() for t in got)
    assert got[0].clone().requires_grad_().sum().backward() is None


def test_launches_of_more_rows_than_one_dimension_holds():
    """2^24 rows of 256 threads: workgroups go on in the launch's second dimension."""
    rows = 2 ** 24 + 5
    x = torch.zeros((rows, 1032), dtype=BF16, device=DEV)
    w = torch.ones(1032, dtype=BF16, device=DEV)
    last = stream(gen(33), 6, 1032, BF16)
    x[-6:] = last
    y = ops.rms_norm(x, w)
    assert torch.equal(y[-6:], ops.rms_norm(last, w)) and not y[:10].any() and not y[-20:-6].any()
    del y
    back = torch.arange(rows, dtype=torch.int32, device=DEV).view(-1, 1)
    assert torch.equal(ops.gather_rows(x, back)[-6:], last)
    dy, dshare = ops.gather_rows_backward(x, x, back, torch.ones((rows, 1), device=DEV))
    assert torch.equal(dy[-6:], last) and not dshare[:-6].any()


@pytest.mark.parametrize("experts,top,how", [(12, 8, {}), (60, 8, {}), (256, 8, {}), (300, 20, {}), (1024, 8, {}), (64, 6, dict(groups=8, top_groups=4, group_top=2)),
                                             (256, 8, dict(groups=8, top_groups=4))])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [False, True])
def test_biases_mask_rows_that_are_not_finite_too(experts, top, how, score, renormalize):
    """A bias of -inf stands whatever a row's logits are: NaN or infinite ones, its own among them, and those that make every score of a softmax NaN."""
    g = gen(experts + top)
    logits, bias = randn(g, 9, experts), 0.1 * randn(g, experts)
    gone = torch.arange(0, experts, 3, device=DEV)
    bias[gone] = -float("inf")
    nan, inf = float("nan"), float("inf")
    logits[1, 4], logits[2, 4], logits[3, 3], logits[4, 3] = nan, inf, nan, inf     # (3 is masked, 4 is not)
    logits[5, 3], logits[5, 4], logits[6, gone], logits[7] = nan, inf, nan, nan
    logits[8, 1:] = -inf
    choice, share = ops.route(logits, top, score=score, bias=bias, renormalize=renormalize, **how)
    assert not (torch.isin(choice, gone.int())).any() and (choice[8] < 0).all() and (share[8] == 0).all()
    want = plain_route(logits[:1], top, score, bias, renormalize=renormalize, **how)
    assert torch.equal(choice[:1], want[0])
    for line in choice.tolist():
        got = [c for c in line if c >= 0]
        assert len(set(got)) == len(got) and all(c < experts for c in got)
    assert (share[choice < 0] == 0).all() and not share[0].isnan().any()
    if score == "softmax":
        assert share[1:8][choice[1:8] >= 0].isnan().all()
    else:
        assert (choice[1, 0] == 4 and share[1, 0].isnan() and share[3:5].isfinite().all() and share[6].isfinite().all())


def test_launches_of_more_long_rows_than_one_dimension_holds():
    """2^22 rows of 1024 threads, in place (69 GB)."""
    rows, cols = 2 ** 22 + 3, 8200
    x = torch.zeros((rows, cols), dtype=BF16, device=DEV)
    w = torch.ones(cols, dtype=BF16, device=DEV)
    ends = stream(gen(34), 5, cols, BF16)
    x[-5:], x[:5], x[2 ** 20 - 2:2 ** 20 + 3] = ends, ends, ends
    want = ops.rms_norm(ends, w)
    ops.rms_norm(x, w, out=x)
    assert torch.equal(x[-5:], want) and torch.equal(x[:5], want) and torch.equal(x[2 ** 20 - 2:2 ** 20 + 3], want)
    assert not x[5:100].any() and not x[-100:-5].any()
    del x
    torch.cuda.empty_cache()


@pytest.mark.parametrize("tokens,top,cols", [(0, 2, 64), (1, 8, 4096), (3, 2, 7), (37, 3, 129), (9, 2, 1025), (600, 2, 1808), (5, 3, 9000)])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_one_gradient_of_gathered_rows(tokens, top, cols, dtype):
    """What is wanted alone is what both together give; places outside the rows as there."""
    g = gen(tokens + cols)
    back, share = places(g, tokens, top), torch.rand((tokens, top), device=DEV, generator=g)
    if tokens > 2:
        back[1, 0], back[2, 1] = -1, tokens * top
    x, y = stream(g, tokens, cols, dtype), stream(g, tokens * top, cols, dtype)
    mark = torch.full_like(y, 3.0)
    dy, dshare = ops.gather_rows_backward(x, y, back, share, dy=mark.clone())
    only, none = ops.gather_rows_backward(x, None, back, share, dy=mark.clone())
    assert none is None and torch.equal(only, dy)
    none, only = ops.gather_rows_backward(x, y, back, share, rows=False)
    assert none is None and torch.equal(only, dshare)
    only, none = ops.gather_rows_backward(x, None, back, share)
    assert only.dtype == dtype and only.shape == y.shape


@pytest.mark.parametrize("cols", [40, 700, 1500, 4096, 9000])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_outputs_in_the_place_of_operands(cols, dtype):
    """Every output that may take an operand's place, against one of its own."""
    g = gen(cols)
    x, r, w, dy, more = stream(g, 77, cols, dtype), stream(g, 77, cols, dtype), 1 + 0.1 * randn(g, cols, dtype=dtype), stream(g, 77, cols, dtype), stream(g, 77, cols, dtype)
    want = ops.rms_norm(x, w, r)
    for out, kept in ((0, 1), (1, 0), (0, None), (1, None), (None, 0), (None, 1)):
        own = x.clone(), r.clone()
        got = ops.rms_norm(own[0], w, own[1], out=None if out is None else own[out], residual_out=None if kept is None else own[kept])
        assert same(got, want)
    want = ops.rms_norm_fp8(x, w, r, keep=True)
    own = x.clone(), r.clone()
    assert same([bits(t) for t in ops.rms_norm_fp8(own[0], w, own[1], keep=True, kept=own[1], residual_out=own[0])], [bits(t) for t in want])
    want = ops.rms_norm_backward(dy, x, w, more)
    for place in range(3):
        own = dy.clone(), x.clone(), more.clone()
        weight = w.clone()
        assert same(ops.rms_norm_backward(own[0], own[1], weight, own[2], dx=own[place], dw=weight), want)
    back, share, y = places(g, 77, 3), randn(g, 77, 3), stream(g, 231, cols, dtype)
    want = ops.gather_rows_backward(x, y, back, share)
    own, parts = y.clone(), share.clone()
    assert same(ops.gather_rows_backward(x, own, back, parts, dy=own, dshare=parts), want)
    experts = min(cols, 1000)
    for renormalize in (True, False):
        logits = x[:, :experts].contiguous()
        choice, _ = ops.route(logits, 3, score="sigmoid")
        for score in ("softmax", "sigmoid"):
            want = ops.route_backward(share, logits, choice, score=score, renormalize=renormalize)
            own = logits.clone()
            assert torch.equal(ops.route_backward(share, own, choice, score=score, renormalize=renormalize, out=own), want)


def test_outputs_a_row_off_their_operands_are_refused():
    g = gen(50)
    room = randn(g, 9, 64, dtype=BF16)
    w, x, off = torch.ones(64, dtype=BF16, device=DEV), room[:8], room[1:]
    kept = room.clone()
    back, share, logits = torch.randperm(8, device=DEV, generator=g).int()[:, None].contiguous(), torch.ones(8, 1, device=DEV), room[:8]
    for match, fn, a, kw in [("out lies in the memory of x", ops.rms_norm, (x, w), {"out": off}), ("sum lies in the memory of residual", ops.rms_norm, (x.clone(), w, x), {"residual_out": off}),
                             ("sum lies in the memory of out", ops.rms_norm, (x.clone(), w, x.clone()), {"out": x, "residual_out": x}),
                             ("q lies in the memory of x", ops.rms_norm_fp8, (x, w), {"out": room.view(-1)[:256].view(F8).view(8, 64)}),
                             ("dx lies in the memory of dy", ops.rms_norm_backward, (x, x.clone(), w), {"dx": off}), ("dx lies in the memory of x", ops.rms_norm_backward, (x.clone(), x, w), {"dx": off}),
                             ("dy lies in the memory of y", ops.gather_rows_backward, (x.clone(), x, back, share), {"dy": off}),
                             ("dlogits lies in the memory of logits", ops.route_backward, (share, logits, back), {"out": off})]:
        with pytest.raises(L.CatcocError, match=match):
            fn(*a, **kw)
    assert torch.equal(room, kept)


@pytest.mark.parametrize("tokens,experts,top,groups,top_groups", [(60, 8, 2, 4, 2), (60, 16, 4, 4, 2), (50, 60, 4, 4, 2), (40, 256, 8, 8, 4), (20, 160, 6, 8, 3), (20, 96, 4, 6, 2), (15, 640, 8, 10, 4),
                                                                  (30, 64, 4, 64, 9)])
@pytest.mark.parametrize("score,biased", [("softmax", False), ("softmax", True), ("sigmoid", False), ("sigmoid", True)])
def test_groups_with_one_expert_left(tokens, experts, top, groups, top_groups, score, biased):
    """A group's score is the sum of its best two that are to be had: of one where one is left, whose group may still be the best."""
    g = gen(experts + groups)
    logits, each = randn(g, tokens, experts), experts // groups
    gone = torch.rand((tokens, groups, each), device=DEV, generator=g) < 0.3
    gone[:, 0] = True                                                   # one left in the first group,
    gone[:, 0, each // 2] = False
    gone[::3, 1 % groups] = True                                        # none in the second
    logits[:, each // 2] += torch.where(torch.arange(tokens, device=DEV) % 2 == 0, 12.0, -2.0)
    logits[gone.view(tokens, experts)] = -float("inf")
    bias = 0.1 * randn(g, experts) if biased else None
    how = dict(groups=groups, top_groups=top_groups, group_top=2)
    choice, share = ops.route(logits, top, score=score, bias=bias, **how)
    want = plain_route(logits, top, score, bias, **how)
    assert torch.equal(choice, want[0]) and (score == "sigmoid" or (choice[::2, 0] == each // 2).all())
    shares_are_near(share, want[1], logits)


@pytest.mark.parametrize("tokens,experts,top", [(21, 128, 8), (13, 100, 6), (6, 128, 40), (4, 64, 64), (17, 65, 3), (9, 250, 16), (7, 300, 12), (5, 600, 33), (3, 512, 64)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype,renormalize,scale", [(F32, True, 1.0), (BF16, False, 2.5), (F16, True, 0.5), (F32, False, 1.0)])
def test_route_backward_in_every_shape(tokens, experts, top, score, dtype, renormalize, scale):
    test_route_backward(tokens, experts, top, score, dtype, renormalize, scale)


@pytest.mark.parametrize("experts", [6, 30, 64, 100, 128, 250, 300, 500, 1000])
@pytest.mark.parametrize("top", [3, 5, 16, 20])
def test_route_backward_of_none_and_doubled_choices_in_every_shape(experts, top):
    if top > experts:
        pytest.skip("more choices than experts are refused")
    g = gen(experts + top)
    logits, dshare = randn(g, 9, experts), randn(g, 9, top)
    choice = torch.randint(0, experts, (9, top), device=DEV, generator=g, dtype=torch.int32)
    choice[1, 1:] = choice[1, :1]                               # one expert, always
    choice[2, ::2], choice[2, 1::2] = experts - 1, 0            # two, in turn
    choice[3, 0], choice[3, -1] = -1, experts                   # none
    choice[4] = -5
    choice[5], choice[5, 1] = 2 ** 31 - 1, experts - 1
    choice[6, :2] = 0
    choice[7], choice[7, 0], choice[7, -1] = -2 ** 31, experts // 2, experts // 2
    for score in ("softmax", "sigmoid"):
        for renormalize in (False, True):
            got = ops.route_backward(dshare, logits, choice, score=score, renormalize=renormalize)
            assert got.isfinite().all() and not got[4].any()
            v = logits.double().requires_grad_()
            p = torch.softmax(v, 1) if score == "softmax" else torch.sigmoid(v)
            on = (choice >= 0) & (choice < experts)
            p = torch.where(on, p.gather(1, choice.long().clamp(0, experts - 1)), 0.0)
            share = p / p.sum(1, keepdim=True) if renormalize else p
            keep = [0, 1, 2, 3, 5, 6, 7, 8]
            want, = torch.autograd.grad(share[keep], v, dshare.double()[keep])
            # as test_route_backward; an expert that is chosen `top` times gets as many gradients, each within its share's bound
            size = share.detach()[keep].sum(1, keepdim=True) * dshare.double().abs().amax(1, keepdim=True)[keep]
            near(got[keep], want[keep], 2 * (110 + top) * u * size)


def test_one_gradient_of_gathered_rows_from_the_compiled_call(monkeypatch):
    g = gen(60)
    x, y, back, share = randn(g, 12, 200, dtype=BF16), randn(g, 36, 200, dtype=BF16), places(g, 12, 3), randn(g, 12, 3)
    compiled, given = ops._host or ops._compiled(), (torch.empty_like(y), torch.empty_like(share))
    for a, kw in (((x, None, back, share), {}), ((x, y, back, share), {"rows": False}), ((x, None, back, share), {"dy": given[0]}), ((x, y, back, share), {"dshare": given[1], "rows": False}),
                  ((x[:0], None, back[:0], share[:0]), {}), ((x[:0], y[:0], back[:0], share[:0]), {"rows": False})):
        host = compiled.gather_rows_backward(*a, kw.get("dy"), kw.get("dshare"), kw.get("rows", True))
        assert host is not None
        host = [None if t is None else t.clone() for t in host]
        with monkeypatch.context() as m:
            m.setattr(ops, "_host", Nothing())
            python = ops.gather_rows_backward(*a, **kw)
        assert [t is None for t in host] == [t is None for t in python] and all(p is None or torch.equal(h, p) for h, p in zip(host, python))
    for a in ((x, None, back, share, None, share, True), (x, None, back, share, None, None, False), (x, y, back, share, y.clone(), None, False), (x[1:], None, back, share, None, None, True),
              (x, y[1:], back, share, None, None, False)):
        assert compiled.gather_rows_backward(*a) is None
