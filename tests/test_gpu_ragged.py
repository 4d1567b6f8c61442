"""e4m3 products with block scales, products grouped by expert, their gradients and the quantizer, against plain implementations in 64 bits.

Tolerances, from the arithmetic alone: a product of two 16-bit or two e4m3 values is exact in fp32, a sum of K of them taken in any order in fp32 is off by at
most K 2^-24 of the sum of magnitudes (scaled: two more roundings), and the output's one rounding by half of its type's epsilon of the value
(fp16: at least 2^-25, half the smallest denormal).

The e4m3 matrix instructions of this GPU (16x16x128 and 16x16x32 alike) are no exact fp32 sums: of up to eight adjacent products they keep 13 bits below
the leading one of the largest (2^14 - 2^14 + 1 is 0, 2^13 - 2^13 + 1 is 1; products further apart add exactly).  Each product is off by at most
2^-13 of the largest in its group, independently: together about 2^-13 sqrt(8) times the products' 2-norm at most, and 2^-10 leaves that nearly three times over."""
import numpy as np
import pytest
import torch

from mm_rs_with_catlass_amd import lib as L
from mm_rs_with_catlass_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
ROUND = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16, torch.float32)}
F8 = torch.float8_e4m3fn


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(g, *shape, dtype=torch.float32):
    return torch.randn(shape, device=DEV, generator=g).to(dtype)


def close(got, want, magnitude, terms, dtype, norm=None):
    """|got - want| against terms * 2^-24 * magnitude + the rounding to dtype, e4m3 products (norm: their 2-norm) 2^-10 norm too; every value."""
    got = got.double()
    assert got.shape == want.shape
    bound = (terms + 2) * 2.0 ** -24 * magnitude + ROUND[dtype] * want.abs() * (1 + 2.0 ** -8) + (2.0 ** -25 if dtype == torch.float16 else 2.0 ** -130)
    if norm is not None:
        bound = bound + 2.0 ** -10 * norm
    off = (got - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), "%d of %d off, worst %.3g times the bound" % (int(bad.sum()), bad.numel(), float((off / bound).nan_to_num(1e30).max()))


def norm2(a, b):
    return ((a * a) @ (b * b).t()).sqrt()


def blocks(n):
    return -(-n // 128)


def spread(scale, rows, cols, br):
    i = torch.arange(rows, device=scale.device) // br
    j = torch.arange(cols, device=scale.device) // 128
    return scale.double()[..., i, :][..., j]


def ends_of(counts):
    return torch.tensor(np.cumsum(counts), dtype=torch.int32, device=DEV)


def ranges(counts):
    at = 0
    for c in counts:
        yield at, at + c
        at += c


def fp8_operand(g, rows, k, br):
    codes = (randn(g, rows, k) * 60).clamp(-448, 448).to(F8)
    scale = torch.rand((blocks(k), rows) if br == 1 else (blocks(rows), blocks(k)), device=DEV, generator=g) + 0.5
    return codes, scale


# ---- quantizer --------------------------------------------------------------------------------------------------------------------

def plain_quantize(v, br):
    """The definition, with numpy's correctly rounded fp32 divisions."""
    rows, cols = v.shape
    p = np.zeros((-(-rows // br) * br, blocks(cols) * 128), np.float32)
    p[:rows, :cols] = v
    p = p.reshape(-1, br, blocks(cols), 128)
    top = np.abs(p).max((1, 3))
    scale = np.where(top < np.float32(2.0 ** -40), np.float32(2.0 ** -40), top) / np.float32(448)
    q = (p / scale[:, None, :, None]).reshape(-1, blocks(cols) * 128)[:rows, :cols]
    return q, (scale.T if br == 1 else scale)


@pytest.mark.parametrize("rows,cols,br", [(1, 1, 1), (1, 128, 1), (3, 129, 1), (5, 7, 1), (16, 1024, 1), (127, 1792, 1), (130, 255, 1), (1000, 643, 1),
                                          (1, 1, 128), (128, 128, 128), (129, 130, 128), (300, 1000, 128), (127, 513, 128)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_quantize_is_its_definition_bit_for_bit(rows, cols, br, dtype):
    g = gen(rows * 1000 + cols)
    x = randn(g, rows, cols) * torch.exp(3 * randn(g, rows, 1))
    x[0, 0] = 0
    x = x.to(dtype)
    q, s = ops.quantize_fp8(x, block_rows=br)
    with np.errstate(invalid="ignore"):      # (fp16: some rows overflow)
        want_q, want_s = plain_quantize(x.float().cpu().numpy(), br)
    assert np.array_equal(s.cpu().numpy(), want_s)
    want = torch.from_numpy(np.ascontiguousarray(want_q)).to(F8)     # (torch rounds to nearest even)
    assert torch.equal(q.cpu().view(torch.uint8), want.view(torch.uint8))


def test_quantize_zeros_tiny_and_values_that_are_not_finite():
    x = torch.zeros((6, 256), device=DEV)
    x[1, 3] = 2.0 ** -50            # under the floor of a block's largest magnitude
    x[2, 5] = float("nan")
    x[3, 7] = float("inf")
    x[4, :] = torch.finfo(torch.float32).max
    x[5, 0], x[5, 1] = 448.0, -1.0
    q, s = ops.quantize_fp8(x)
    q, s = q.float().cpu(), s.cpu()
    floor = np.float32(2.0 ** -40) / np.float32(448)
    assert (q[0] == 0).all() and (s[:, 0] == floor).all()
    assert s[0, 1] == floor and abs(q[1, 3] - 448 * 2.0 ** -10) <= 2.0 ** -10 and (q[1, 4:] == 0).all()
    assert s[0, 2].isnan() and q[2, :128].isnan().all() and (q[2, 128:] == 0).all() and s[1, 2] == floor
    assert s[0, 3].isinf() and q[3, 7].isnan() and (q[3, 8:] == 0).all()
    assert (q[4] == 448).all()
    assert s[0, 5] == 1 and q[5, 0] == 448 and q[5, 1] == -1


@pytest.mark.parametrize("rows,cols", [(1, 128), (7, 130), (33, 1792), (4, 1), (5, 1003)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_quantize_gated(rows, cols, dtype):
    g = gen(rows + cols)
    x = (randn(g, rows, 2 * cols) * 3).to(dtype)
    x[0, 0] = -60.0
    q, s = ops.quantize_fp8(x, gated=True)
    v = x.double()
    v = v[:, :cols] * torch.sigmoid(v[:, :cols]) * v[:, cols:]
    # a handful of fp32 operations, each off by a few 2^-24: the scale within 2^-20, a code within half its spacing and as much again of the value
    want_s = torch.nn.functional.pad(v.abs(), (0, blocks(cols) * 128 - cols)).view(rows, -1, 128).amax(2).clamp_min(2.0 ** -40).t() / 448
    assert ((s.double() - want_s).abs() <= 2.0 ** -20 * want_s).all()
    t = v / spread(s.t(), rows, cols, 1)
    step = torch.exp2(torch.floor(torch.log2(t.abs().clamp_min(2.0 ** -6))) - 3)      # e4m3: three bits behind the leading one, 2^-9 at least
    assert ((q.double() - t).abs() <= step / 2 + 2.0 ** -19 * t.abs() + 2.0 ** -30).all()


# ---- e4m3 products ----------------------------------------------------------------------------------------------------------------

FP8 = [(1, 128, 128), (1, 1, 1), (2, 8192, 256), (3, 130, 5), (16, 129, 127), (17, 1000, 1000), (31, 4096, 513), (63, 257, 260), (64, 512, 1024), (65, 640, 384),
       (100, 1808, 515), (128, 256, 256), (130, 1024, 768), (203, 1808, 1100), (256, 384, 512), (257, 131, 513), (300, 4100, 260), (512, 1792, 1024),
       (777, 2048, 1284), (1025, 900, 1000), (2048, 1024, 2048)]


@pytest.mark.parametrize("m,k,n", FP8)
@pytest.mark.parametrize("dtype,ranks", [(torch.bfloat16, 1), (torch.float16, 3)])
def test_fp8_matmul_allreduce(m, k, n, dtype, ranks):
    g = gen(m + 3 * k + 7 * n)
    x, sx = fp8_operand(g, m, k, 1)
    w, sw = fp8_operand(g, n, k, 128)
    sx *= 0.05 / 60
    peers = [randn(g, m + 2, n + 3) for _ in range(ranks - 1)]    # (rows and columns past the ones read)
    out = ops.fp8_matmul_allreduce(x, w, sx, sw, peers, rank=ranks - 1, rank_size=ranks, out_dtype=dtype, peer_row_offset=2)
    a, b = x.double() * spread(sx.t(), m, k, 1), w.double() * spread(sw, n, k, 128)
    want, mag, norm = a @ b.t(), a.abs() @ b.abs().t(), norm2(a, b)
    for p in peers:
        want += p[2:, :n].double()
        mag += p[2:, :n].double().abs()
    close(out, want, mag, k + ranks, dtype, norm)


def test_fp8_matmul_keeps_rows_with_values_that_are_not_finite_apart():
    g = gen(5)
    m, k, n = 70, 300, 200
    x, sx = fp8_operand(g, m, k, 1)
    w, sw = fp8_operand(g, n, k, 128)
    clean = ops.fp8_matmul_allreduce(x, w, sx, sw)
    x2, sx2, w2 = x.clone(), sx.clone(), w.clone()
    x2.view(torch.uint8)[3, 299] = 0x7f             # a NaN in one row's last value of k,
    sx2[1, 20] = float("inf")                        # an infinite scale of another row,
    w2.view(torch.uint8)[77, 0] = 0xff              # a NaN in one column
    out = ops.fp8_matmul_allreduce(x2, w2, sx2, sw)
    rows = torch.ones(m, dtype=torch.bool, device=DEV)
    rows[3] = rows[20] = False
    cols = torch.ones(n, dtype=torch.bool, device=DEV)
    cols[77] = False
    assert torch.equal(out[rows][:, cols], clean[rows][:, cols])
    assert out[3].isnan().all() and not out[20].isfinite().any() and out[:, 77].isnan().all()


@pytest.mark.parametrize("offset", [1, 2, 4, 8])
def test_fp8_operands_at_any_address(offset):
    g = gen(offset)
    m, k, n = 75, 384, 320
    x, sx = fp8_operand(g, m, k, 1)
    w, sw = fp8_operand(g, n, k, 128)
    want = ops.fp8_matmul_allreduce(x, w, sx, sw).double()

    def moved(t, by):
        room = torch.empty(t.numel() + by, dtype=t.dtype, device=DEV)
        room[by:] = t.reshape(-1)
        return room[by:].view(t.shape)
    got = ops.fp8_matmul_allreduce(moved(x, offset), moved(w, offset), moved(sx, offset), moved(sw, offset),
                                   out=moved(torch.empty((m, n), dtype=torch.bfloat16, device=DEV), offset))
    a, b = x.double() * spread(sx.t(), m, k, 1), w.double() * spread(sw, n, k, 128)
    close(got, a @ b.t(), a.abs() @ b.abs().t(), k, torch.bfloat16, norm2(a, b))
    assert ((got.double() - want).abs() <= 2.0 ** -7 * want.abs() + 1e-3 * want.abs().max()).all()


# ---- rows in groups ---------------------------------------------------------------------------------------------------------------

COUNTS = {
    "one": [1], "none_between": [3, 0, 5, 0, 0, 1], "first_and_last_empty": [0, 17, 64, 0], "edges": [15, 16, 17, 31, 33, 63, 64, 65], "long": [700, 1, 0, 300],
    "many": [(7 * i) % 11 for i in range(70)], "very_many": [1 if i % 3 else 0 for i in range(200)], "decode": [0] * 20 + [1, 2, 0, 1] + [0] * 8 + [4],
    "around_256": [255, 256, 257, 0, 129],
}
WIDTHS = [(128, 128), (64, 256), (1, 1), (130, 77), (200, 516), (1000, 264), (513, 1025), (4, 12), (1792, 384)]


@pytest.mark.parametrize("name", sorted(COUNTS))
@pytest.mark.parametrize("k,n", WIDTHS)
@pytest.mark.parametrize("trans_b", [False, True])
def test_grouped_matmul(name, k, n, trans_b):
    counts = COUNTS[name]
    if len(counts) > 60 and k * n > 200000:
        pytest.skip("the same widths run with fewer groups")
    dtype = torch.bfloat16 if (k + n) % 3 else torch.float16
    g = gen(k + n)
    rows, groups, past = sum(counts), len(counts), 5
    x = randn(g, rows + past, k, dtype=dtype)
    w = randn(g, groups, n, k, dtype=dtype) if trans_b else randn(g, groups, k, n, dtype=dtype)
    out = ops.grouped_matmul(x, w, ends_of(counts), trans_b=trans_b)
    for e, (i, j) in enumerate(ranges(counts)):
        a, b = x[i:j].double(), w[e].double()
        b = b.t() if trans_b else b
        close(out[i:j], a @ b, a.abs() @ b.abs(), k, dtype)
    assert (out[rows:] == 0).all()      # rows past the last group


@pytest.mark.parametrize("name", sorted(COUNTS))
@pytest.mark.parametrize("k,n", WIDTHS)
@pytest.mark.parametrize("trans_b", [False, True])
def test_grouped_matmul_dw(name, k, n, trans_b):
    counts = COUNTS[name]
    if len(counts) > 60 and k * n > 200000:
        pytest.skip("the same widths run with fewer groups")
    dtype = torch.bfloat16 if (k + n) % 3 else torch.float16
    out_dtype = [torch.float32, dtype][(k + len(counts)) % 2]
    g = gen(k + n + 1)
    rows, groups = sum(counts), len(counts)
    x, dy = randn(g, rows + 3, k, dtype=dtype), randn(g, rows + 3, n, dtype=dtype)
    x[rows:] = float("nan")             # rows of no group
    dw = ops.grouped_matmul_dw(x, dy, ends_of(counts), out_dtype=out_dtype, trans_b=trans_b)
    assert dw.shape == ((groups, n, k) if trans_b else (groups, k, n)) and dw.dtype == out_dtype
    for e, (i, j) in enumerate(ranges(counts)):
        a, b = x[i:j].double().t(), dy[i:j].double()
        want, mag = a @ b, a.abs() @ b.abs()
        close(dw[e].t() if trans_b else dw[e], want, mag, j - i, out_dtype)


@pytest.mark.parametrize("name", sorted(COUNTS))
@pytest.mark.parametrize("k,n", [(128, 128), (64, 256), (1, 1), (130, 77), (260, 516), (1000, 264), (515, 1025), (4, 12), (1792, 384)])
def test_grouped_fp8_matmul(name, k, n):
    counts = COUNTS[name]
    if len(counts) > 60 and k * n > 200000:
        pytest.skip("the same widths run with fewer groups")
    dtype = torch.bfloat16 if (k + n) % 3 else torch.float16
    g = gen(k + n + 2)
    rows, groups, past = sum(counts), len(counts), 2
    x, sx = fp8_operand(g, rows + past, k, 1)
    sx *= 0.05 / 60
    w = (randn(g, groups, n, k) * 60).clamp(-448, 448).to(F8)
    sw = torch.rand((groups, blocks(n), blocks(k)), device=DEV, generator=g) + 0.5
    out = ops.grouped_fp8_matmul(x, w, sx, sw, ends_of(counts), out_dtype=dtype)
    for e, (i, j) in enumerate(ranges(counts)):
        a, b = x[i:j].double() * spread(sx[:, i:j].t(), j - i, k, 1), w[e].double() * spread(sw[e], n, k, 128)
        close(out[i:j], a @ b.t(), a.abs() @ b.abs().t(), k, dtype, norm2(a, b))
    assert (out[rows:] == 0).all()


def test_groups_keep_values_that_are_not_finite_to_themselves():
    g = gen(9)
    counts, k, n = [33, 40, 0, 7], 200, 136
    x = randn(g, sum(counts), k, dtype=torch.bfloat16)
    w = randn(g, len(counts), n, k, dtype=torch.bfloat16)
    dy = randn(g, sum(counts), n, dtype=torch.bfloat16)
    ends = ends_of(counts)
    clean, dclean = ops.grouped_matmul(x, w, ends, trans_b=True), ops.grouped_matmul_dw(x, dy, ends)
    x[33:73] = float("inf")
    w[2] = float("nan")                 # the matrix of a group without rows
    out, dw = ops.grouped_matmul(x, w, ends, trans_b=True), ops.grouped_matmul_dw(x, dy, ends)
    assert torch.equal(out[:33], clean[:33]) and torch.equal(out[73:], clean[73:])
    assert torch.equal(dw[[0, 2, 3]], dclean[[0, 2, 3]])
    assert not out[33:73].isfinite().any() and not dw[1].isfinite().any()


@pytest.mark.parametrize("ends", [[5, 3, 60, 40], [-7, 20, 2000, 100], [0, 0, 0, 0], [64, 64, 64, 64]])
def test_group_ends_that_make_no_sense_stay_in_bounds(ends):
    # the rows of a group that is well formed come out right; nothing else is promised but that no access leaves the buffers
    g = gen(11)
    rows, k, n = 64, 96, 80
    x, w = randn(g, rows, k, dtype=torch.bfloat16), randn(g, 4, k, n, dtype=torch.bfloat16)
    room = torch.full((rows + 2, n), 7.0, dtype=torch.bfloat16, device=DEV)
    ops.grouped_matmul(x, w, torch.tensor(ends, dtype=torch.int32, device=DEV), out=room[1:-1])
    ops.grouped_matmul_dw(x, randn(g, rows, n, dtype=torch.bfloat16), torch.tensor(ends, dtype=torch.int32, device=DEV))
    torch.cuda.synchronize()
    assert (room[0] == 7).all() and (room[-1] == 7).all()


def test_gradients_against_differences():
    # L = sum(y * r) is linear in x and in w: in 64 bits a difference quotient is the gradient up to its own rounding, so what remains
    # is the gradient's one rounding to fp32 (dw) or bf16 (dx) and its sums
    g = gen(13)
    counts, k, n = [5, 0, 9, 2], 40, 24
    rows = sum(counts)
    ends = ends_of(counts)
    x, w = randn(g, rows, k, dtype=torch.bfloat16), randn(g, len(counts), n, k, dtype=torch.bfloat16)
    r = randn(g, rows, n, dtype=torch.bfloat16)
    dx = ops.grouped_matmul(r, w, ends, trans_b=False)
    dw = ops.grouped_matmul_dw(x, r, ends, out_dtype=torch.float32, trans_b=True)

    def loss(x64, w64):
        return sum(((x64[i:j] @ w64[e].t()) * r[i:j].double()).sum() for e, (i, j) in enumerate(ranges(counts)))
    x64, w64, h = x.double(), w.double(), 2.0 ** -6
    for i, j in [(0, 0), (4, 39), (5, 7), (13, 20), (15, 39)]:
        step = torch.zeros_like(x64)
        step[i, j] = h
        d = float((loss(x64 + step, w64) - loss(x64 - step, w64)) / (2 * h))
        assert abs(float(dx[i, j]) - d) <= 2.0 ** -8 * abs(d) + n * 2.0 ** -20
    for e, i, j in [(0, 0, 0), (0, 23, 39), (2, 11, 5), (3, 1, 38), (1, 3, 3)]:
        step = torch.zeros_like(w64)
        step[e, i, j] = h
        d = float((loss(x64, w64 + step) - loss(x64, w64 - step)) / (2 * h))
        assert abs(float(dw[e, i, j]) - d) <= 1e-5 * (1 + abs(d))


FAR_TILES = [None, (256, 256, 1), (128, 128, 1), (64, 128, 2), (64, 64, 1)]


@pytest.mark.parametrize("trans_b", [False, True])
def test_matrices_past_4_gib(trans_b):
    groups, k, n, rows = 34, 8192, 8192, 11
    w = torch.zeros((groups, n, k) if trans_b else (groups, k, n), dtype=torch.bfloat16, device=DEV)
    assert w[-1].data_ptr() - w.data_ptr() > 2 ** 32
    g = gen(21)
    w[-1] = randn(g, *w.shape[1:])
    x = randn(g, rows, k, dtype=torch.bfloat16)
    counts = [4] + [0] * (groups - 2) + [7]
    b = w[-1].double().t() if trans_b else w[-1].double()
    for tile in FAR_TILES + (SMALL_NK if trans_b else SMALL_KN):
        out = ops.grouped_matmul(x, w, ends_of(counts), trans_b=trans_b, tile=tile)
        assert (out[:4] == 0).all()
        close(out[4:], x[4:].double() @ b, x[4:].double().abs() @ b.abs(), k, torch.bfloat16)


def test_rows_past_4_gib():
    rows, k, n, last = 2 ** 18 + 300, 8192, 136, 150
    x, dy = torch.zeros((rows, k), dtype=torch.bfloat16, device=DEV), torch.zeros((rows, n), dtype=torch.bfloat16, device=DEV)
    assert x[-last].data_ptr() - x.data_ptr() > 2 ** 32
    g = gen(22)
    x[-last:], dy[-last:] = randn(g, last, k), randn(g, last, n)
    w = randn(g, 2, k, n, dtype=torch.bfloat16)
    ends = ends_of([rows - last, last])
    a, d = x[-last:].double(), dy[-last:].double()
    for tile in FAR_TILES:
        out = ops.grouped_matmul(x, w, ends, tile=tile)
        assert (out[:-last] == 0).all()
        close(out[-last:], a @ w[1].double(), a.abs() @ w[1].double().abs(), k, torch.bfloat16)
    back = torch.zeros((rows, k), dtype=torch.bfloat16, device=DEV)   # (results past 4 GiB)
    ops.grouped_matmul(dy, w, ends, trans_b=True, out=back)
    assert (back[:-last] == 0).all()
    close(back[-last:], d @ w[1].double().t(), d.abs() @ w[1].double().abs().t(), n, torch.bfloat16)
    for tile in (None, (256, 256, 1), (128, 128, 1), (64, 64, 1)):
        dw = ops.grouped_matmul_dw(x, dy, ends, out_dtype=torch.float32, tile=tile)
        assert (dw[0] == 0).all()
        close(dw[1], a.t() @ d, a.abs().t() @ d.abs(), last, torch.float32)
    for br in (1, 128):
        q, sx = ops.quantize_fp8(x, block_rows=br)
        first = rows - rows % 128 - 128
        want, scale = plain_quantize(x[first:].float().cpu().numpy(), br)
        assert (q[first:].float().cpu().numpy() == torch.from_numpy(want).to(F8).float().numpy()).all()
        got = sx[:, first:] if br == 1 else sx[first // 128:]
        assert (got.cpu().numpy() == scale).all()


def test_fp8_rows_past_4_gib():
    rows, k, n, last = 2 ** 19 + 300, 8192, 130, 150
    x = torch.zeros((rows, k), dtype=torch.uint8, device=DEV).view(F8)
    sx = torch.ones((blocks(k), rows), device=DEV)
    g = gen(23)
    x[-last:], sx[:, -last:] = fp8_operand(g, last, k, 1)
    w, sw = fp8_operand(g, n, k, 128)
    a, b = x[-last:].double() * spread(sx[:, -last:].t().contiguous(), last, k, 1), w.double() * spread(sw, n, k, 128)
    for tile in FAR_TILES:
        out = ops.fp8_matmul_allreduce(x, w, sx, sw, tile=tile)
        assert (out[:-last] == 0).all()
        close(out[-last:], a @ b.t(), a.abs() @ b.abs().t(), k + 1, torch.bfloat16, norm2(a, b))


def test_no_rows():
    ends = torch.zeros(3, dtype=torch.int32, device=DEV)
    x, dy = torch.empty((0, 64), dtype=torch.bfloat16, device=DEV), torch.empty((0, 32), dtype=torch.bfloat16, device=DEV)
    assert ops.grouped_matmul(x, torch.ones((3, 64, 32), dtype=torch.bfloat16, device=DEV), ends).shape == (0, 32)
    dw = torch.full((3, 64, 32), 5.0, device=DEV)
    assert (ops.grouped_matmul_dw(x, dy, ends, out=dw) == 0).all()
    q, s = ops.quantize_fp8(x)
    assert q.shape == (0, 64) and s.shape == (1, 0)
    w, sw = ops.quantize_fp8(torch.ones((128, 64), dtype=torch.bfloat16, device=DEV), block_rows=128)
    assert ops.fp8_matmul_allreduce(q, w, s, sw).shape == (0, 128)
    assert ops.grouped_fp8_matmul(q, w.expand(3, -1, -1).contiguous(), s, sw.expand(3, -1, -1).contiguous(), ends).shape == (0, 128)


def test_equal_calls_give_equal_bits_and_other_streams_see_their_inputs():
    g = gen(17)
    counts, k, n = [100, 0, 300, 57], 512, 384
    rows = sum(counts)
    x, w, dy = randn(g, rows, k, dtype=torch.bfloat16), randn(g, 4, n, k, dtype=torch.bfloat16), randn(g, rows, n, dtype=torch.bfloat16)
    ends = ends_of(counts)
    calls = [lambda: ops.grouped_matmul(x, w, ends, trans_b=True), lambda: ops.grouped_matmul_dw(x, dy, ends, out_dtype=torch.float32),
             lambda: ops.quantize_fp8(x)[0].view(torch.uint8)]
    want = [c() for c in calls]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = [[c() for c in calls] for _ in range(3)]
    side.synchronize()
    for them in got:
        assert all(torch.equal(a, b) for a, b in zip(them, want))


def test_replay_from_a_hip_graph():
    g = gen(19)
    counts, k, n = [30, 2, 0, 50], 256, 384
    rows = sum(counts)
    x, w, ends = randn(g, rows, 2 * k, dtype=torch.bfloat16), randn(g, 4, n, k, dtype=torch.bfloat16), ends_of(counts)
    codes = torch.empty((4, n, k), dtype=F8, device=DEV)
    scales = torch.empty((4, 3, 2), device=DEV)
    for e in range(4):
        ops.quantize_fp8(w[e], block_rows=128, out=codes[e], scale=scales[e])

    def step():
        q, s = ops.quantize_fp8(x, gated=True)
        return ops.grouped_fp8_matmul(q, codes, s, scales, ends)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        x.copy_(randn(g, rows, 2 * k, dtype=torch.bfloat16))
        counts = counts[1:] + counts[:1]          # the same graph serves other group sizes
        ends.copy_(ends_of(counts))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, step()), i


def test_calls_say_what_they_ran():
    x, sx = fp8_operand(gen(1), 8, 131, 1)
    w, sw = fp8_operand(gen(2), 8, 131, 128)
    ops.fp8_matmul_allreduce(x, w, sx, sw)
    info = L.last_launch()
    assert (info.kernel, info.tileRows, info.tileCols) == (L.KERNEL_RAGGED_CHECKED, 64, 64)


TILES = [(256, 256, 1), (224, 256, 1), (160, 256, 1), (96, 256, 1), (128, 128, 1), (128, 128, 2), (64, 128, 2), (64, 64, 1)]
TILES_DW = [(256, 256, 1), (128, 128, 1), (64, 64, 1)]
SMALL_NK, SMALL_KN = [(16, 32, 4), (32, 32, 4)], [(16, 64, 4), (32, 64, 4), (64, 64, 4)]
UNEVEN = {"large": [513, 0, 31, 900, 260, 1], "one_group": [1300], "full": [512, 256], "few": [1, 0, 15, 16, 17, 0, 40, 70, 129], "many": [(5 * i) % 23 for i in range(75)]}


def ran(tile):
    info = L.last_launch()
    return (info.tileRows, info.tileCols, info.kSlices) == tile and info.kernel == (L.KERNEL_RAGGED_CHECKED if tile == (64, 64, 1) else L.KERNEL_RAGGED)


@pytest.mark.parametrize("name", sorted(UNEVEN))
@pytest.mark.parametrize("k,n", [(1024, 512), (1096, 776), (514, 1030), (66, 2), (64, 128), (192, 250), (2050, 130)])
@pytest.mark.parametrize("tile,trans_b", [(t, b) for b in (False, True) for t in TILES + (SMALL_NK if b else SMALL_KN)])
def test_every_tile_of_grouped_products(name, k, n, tile, trans_b):
    counts = UNEVEN[name]
    g = gen(k * n)
    rows, groups = sum(counts), len(counts)
    ends = ends_of(counts)
    x = randn(g, rows + 40, k, dtype=torch.bfloat16)
    x[rows:] = float("nan")
    w = randn(g, groups, n, k, dtype=torch.bfloat16) if trans_b else randn(g, groups, k, n, dtype=torch.bfloat16)
    out = ops.grouped_matmul(x, w, ends, trans_b=trans_b, tile=tile)
    assert ran(tile)
    for e, (i, j) in enumerate(ranges(counts)):
        a, b = x[i:j].double(), w[e].double()
        b = b.t() if trans_b else b
        close(out[i:j], a @ b, a.abs() @ b.abs(), k, torch.bfloat16)
    assert (out[rows:] == 0).all()


@pytest.mark.parametrize("name", sorted(UNEVEN))
@pytest.mark.parametrize("k,n", [(1024, 512), (1096, 776), (514, 1030), (66, 2), (256, 130)])
@pytest.mark.parametrize("tile", TILES_DW)
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.float16])
def test_every_tile_of_weight_gradients(name, k, n, tile, out_dtype):
    counts = UNEVEN[name]
    g = gen(k * n + 2)
    rows = sum(counts)
    ends = ends_of(counts)
    x, dy = randn(g, rows + 40, k, dtype=torch.bfloat16), randn(g, rows + 40, n, dtype=torch.bfloat16)
    x[rows:], dy[rows:] = float("nan"), float("nan")
    for trans_b in (False, True):
        dw = ops.grouped_matmul_dw(x, dy, ends, out_dtype=out_dtype, trans_b=trans_b, tile=tile)
        assert ran(tile)
        for e, (i, j) in enumerate(ranges(counts)):
            a, d = x[i:j].double(), dy[i:j].double()
            close(dw[e].t() if trans_b else dw[e], a.t() @ d, a.abs().t() @ d.abs(), j - i, out_dtype)


# Groups of very different heights, rows past the last one, more row tiles than a band has: each group's tiles go to all XCDs (fewer rows than matrices) ...
@pytest.mark.parametrize("tile,trans_b", [(t, b) for b in (False, True) for t in TILES + (SMALL_NK if b else SMALL_KN) + [None]])
@pytest.mark.parametrize("groups", [28, 48, 64])   # (... but not with 64)
def test_tiles_of_uneven_groups(groups, tile, trans_b):
    k, n = 192, 776
    counts = [900, 0, 3, 64] + [0] * (groups - 8) + [130, 131, 1, 259]
    g = gen(groups)
    rows = sum(counts)
    x = randn(g, rows + 333, k, dtype=torch.bfloat16)
    x[rows:] = float("nan")
    w = randn(g, groups, n, k, dtype=torch.bfloat16) if trans_b else randn(g, groups, k, n, dtype=torch.bfloat16)
    out = ops.grouped_matmul(x, w, ends_of(counts), trans_b=trans_b, tile=tile)
    for e, (i, j) in enumerate(ranges(counts)):
        a, b = x[i:j].double(), w[e].double()
        b = b.t() if trans_b else b
        close(out[i:j], a @ b, a.abs() @ b.abs(), k, torch.bfloat16)
    assert (out[rows:] == 0).all()


# Several tiles for each workgroup, with every number of steps, of rows in the last one and of tiles without rows between them.
@pytest.mark.parametrize("tile", TILES_DW)
@pytest.mark.parametrize("k,n", [(1024, 768), (1030, 700), (896, 1032)])
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
def test_weight_gradients_of_many_tiles(k, n, tile, out_dtype):
    counts = [0, 0] + [(131 * i * i + 64 * i) % 450 if i % 7 else 0 for i in range(34)] + [64, 128, 192, 256, 320, 63, 65, 1, 0]
    g = gen(k + n)
    x, dy = randn(g, sum(counts), k, dtype=torch.float16), randn(g, sum(counts), n, dtype=torch.float16)
    dw = ops.grouped_matmul_dw(x, dy, ends_of(counts), out_dtype=out_dtype, tile=tile)
    assert ran(tile)
    for e, (i, j) in enumerate(ranges(counts)):
        a, d = x[i:j].double(), dy[i:j].double()
        close(dw[e], a.t() @ d, a.abs().t() @ d.abs(), j - i, out_dtype)


@pytest.mark.parametrize("name", sorted(UNEVEN))
@pytest.mark.parametrize("k,n", [(1024, 512), (1100, 777), (516, 1030), (132, 3), (128, 128), (260, 250), (4, 100)])
@pytest.mark.parametrize("tile", TILES + SMALL_NK)
def test_every_tile_of_fp8_products(name, k, n, tile):
    counts = UNEVEN[name]
    g = gen(k * n + 1)
    rows, groups = sum(counts), len(counts)
    x, sx = fp8_operand(g, rows + 3, k, 1)
    sx *= 0.05 / 60
    w = (randn(g, groups, n, k) * 60).clamp(-448, 448).to(F8)
    sw = torch.rand((groups, blocks(n), blocks(k)), device=DEV, generator=g) + 0.5
    out = ops.grouped_fp8_matmul(x, w, sx, sw, ends_of(counts), tile=tile)
    assert ran(tile)
    for e, (i, j) in enumerate(ranges(counts)):
        a, b = x[i:j].double() * spread(sx[:, i:j].t(), j - i, k, 1), w[e].double() * spread(sw[e], n, k, 128)
        close(out[i:j], a @ b.t(), a.abs() @ b.abs().t(), k, torch.bfloat16, norm2(a, b))
    assert (out[rows:] == 0).all()


@pytest.mark.parametrize("m,k,n", [(300, 1000, 390), (33, 384, 130), (1, 4100, 260), (129, 132, 65)])
@pytest.mark.parametrize("tile", TILES + SMALL_NK)
def test_every_tile_adds_its_peers(m, k, n, tile):
    g = gen(m * k)
    x, sx = fp8_operand(g, m, k, 1)
    w, sw = fp8_operand(g, n, k, 128)
    sx *= 0.05 / 60
    peers = [randn(g, m, n) for _ in range(9)]
    out = ops.fp8_matmul_allreduce(x, w, sx, sw, peers, rank=3, rank_size=10, out_dtype=torch.float16, tile=tile)
    assert ran(tile)
    a, b = x.double() * spread(sx.t(), m, k, 1), w.double() * spread(sw, n, k, 128)
    want, mag = a @ b.t(), a.abs() @ b.abs().t()
    for p in peers:
        want, mag = want + p.double(), mag + p.double().abs()
    close(out, want, mag, k + 10, torch.float16, norm2(a, b))


@pytest.mark.parametrize("rows,groups,k,n", [(64, 64, 512, 512), (512, 8, 512, 512), (1024, 8, 512, 2048), (4096, 8, 512, 2048), (4096, 2, 256, 8192), (16384, 4, 128, 4096), (300, 4, 509, 640)])
def test_the_choice_of_tiles_changes_no_more_than_the_order_of_sums(rows, groups, k, n):
    g = gen(rows + k)
    ends = ends_of([rows // groups] * groups)
    x, w = randn(g, rows, k, dtype=torch.bfloat16), randn(g, groups, n, k, dtype=torch.bfloat16)
    out = ops.grouped_matmul(x, w, ends, trans_b=True)
    same = ops.grouped_matmul(x, w, ends, trans_b=True, tile=(64, 64, 1))
    e = 1 % groups
    i = slice(e * (rows // groups), e * (rows // groups) + min(7, rows // groups))
    a, b = x[i].double(), w[e].double().t()
    close(out[i], a @ b, a.abs() @ b.abs(), k, torch.bfloat16)
    assert ((out.double() - same.double()).abs() <= 2.0 ** -7 * same.double().abs() + 1e-3).all()


def test_tiles_that_do_not_exist_are_refused():
    x, w, ends = torch.ones((8, 64), dtype=torch.bfloat16, device=DEV), torch.ones((2, 64, 32), dtype=torch.bfloat16, device=DEV), ends_of([3, 5])
    dy = torch.ones((8, 32), dtype=torch.bfloat16, device=DEV)
    for call in (lambda t: ops.grouped_matmul(x, w, ends, tile=t), lambda t: ops.grouped_matmul_dw(x, dy, ends, tile=t)):
        for t in ((256, 128, 1), (16, 32, 4), (1, 1, 1), (64, 64, 2)):
            with pytest.raises(L.CatcocError, match="no kernel of"):
                call(t)
    with pytest.raises(L.CatcocError, match="do not start on 4 bytes"):
        ops.grouped_matmul(x[:, :63].contiguous(), w[:, :63].contiguous(), ends, tile=(128, 128, 1))
    with pytest.raises(L.CatcocError, match="no kernel of"):
        ops.grouped_matmul_dw(x, dy, ends, tile=(128, 128, 2))


class Nothing:
    """In the place of the compiled calls: leaves every call to the Python path."""

    def __getattr__(self, name):
        return lambda *a: None


def both_calls(monkeypatch, fn, *a, **kw):
    """What the compiled and the Python path make of a call: results, or the error's text."""
    seen = []
    for host in (None, Nothing()):
        with monkeypatch.context() as m:
            if host is not None:
                m.setattr(ops, "_host", host)
            try:
                r = fn(*a, **kw)
                seen.append([t.clone().view(torch.uint8) if t.dtype == F8 else t.clone() for t in (r if isinstance(r, tuple) else (r,))])
            except L.CatcocError as e:
                seen.append(str(e))
    assert type(seen[0]) is type(seen[1])
    if isinstance(seen[0], str):
        assert seen[0] == seen[1]
        return False
    assert all(torch.equal(p, q) for p, q in zip(*seen))
    return True


def test_the_compiled_call_and_the_python_path_answer_alike(monkeypatch):
    g = gen(31)
    rows, k, n, groups = 20, 256, 130, 3
    x, dy = randn(g, rows, k, dtype=torch.bfloat16), randn(g, rows, n, dtype=torch.bfloat16)
    w, ends = randn(g, groups, n, k, dtype=torch.bfloat16), ends_of([4, 0, 16])
    (x8, sx), (w8, sw) = ops.quantize_fp8(x), ops.quantize_fp8(w[0], block_rows=128)
    ws8, ssw = torch.stack([w8.view(torch.uint8)] * groups).view(F8), torch.stack([sw] * groups)
    peers = [randn(g, rows + 3, n + 2) for _ in range(2)]
    wide = randn(g, rows, 2 * k, dtype=torch.bfloat16)
    q, f, m, d, e = ops.quantize_fp8, ops.fp8_matmul_allreduce, ops.grouped_matmul, ops.grouped_matmul_dw, ops.grouped_fp8_matmul

    def alike(fn, *a, **kw):
        return both_calls(monkeypatch, fn, *a, **kw)
    for fn, a, kw in ((q, (x,), {}), (q, (x.float(), 128), {}), (q, (wide,), {"gated": True}), (q, (torch.nn.Parameter(x),), {}),
                      (q, (x,), {"out": torch.empty_like(x8), "scale": torch.empty_like(sx)}),
                      (f, (x8, w8, sx, sw), {}), (f, (x8, w8, sx, sw, peers, 1, 3, torch.float16, 2), {}), (f, (x8, w8, sx, sw, tuple(peers)), {"rank_size": 3}),
                      (f, (x8, w8, sx, sw), {"out": torch.empty((rows, n), dtype=torch.float16, device=DEV)}),
                      (m, (x, w, ends), {"trans_b": True}), (m, (dy, w, ends), {}), (d, (x, dy, ends), {}), (d, (x, dy, ends, torch.float32, True), {}),
                      (d, (x, dy, ends), {"out": torch.empty((groups, k, n), device=DEV)}), (e, (x8, ws8, sx, ssw, ends), {}), (e, (x8, ws8, sx, ssw, ends, torch.float16), {})):
        assert alike(fn, *a, **kw), (fn.__name__, kw)
    for fn, a, kw in ((q, (x.int(),), {}), (q, (wide[:, ::2],), {}), (q, (x, 64), {}), (q, (x, 128, True), {}), (q, (x,), {"out": x}), (q, (x,), {"scale": sx[:, 1:]}),
                      (q, (x.cpu(),), {}), (q, (x[0],), {}),
                      (f, (x8, w8, sx.cpu(), sw), {}), (f, (x8, w8[:, 1:], sx, sw), {}), (f, (x8, w8, sx, sw, peers), {}), (f, (x8, w8, sx, sw, peers, 3, 3), {}),
                      (f, (x8, w8, sx, sw, peers, 0, 3, torch.bfloat16, 4), {}), (f, (x8, w8, sx, sw, [peers[0], peers[1].half()], 0, 3), {}),
                      (f, (x8, w8, sx, sw), {"out_dtype": torch.float32}), (f, (x8, w8, sx, sw), {"out": torch.empty((rows, n), device=DEV)}),
                      (m, (x, w, ends), {}), (m, (x, w.half(), ends, True), {}), (m, (x, w, ends.long(), True), {}), (m, (x, w, ends[:2], True), {}),
                      (m, (x, w, ends, True), {"out": torch.empty((rows, n), device=DEV)}), (m, (x[:, ::2], w[:, :, ::2], ends, True), {}),
                      (d, (x, dy[1:], ends), {}), (d, (x, dy, ends, torch.float64), {}), (d, (x, dy, ends.cpu()), {}), (d, (x, dy, [4, 4, 20]), {}),
                      (e, (x8, ws8, sx, sw, ends), {}), (e, (x8, ws8, sx, ssw, ends, torch.float32), {}), (e, (x, ws8, sx, ssw, ends), {})):
        assert not alike(fn, *a, **kw), (fn.__name__, kw)


# ---- launches of more workgroups than one dimension of a grid holds (2^32 threads) --------------------------------------------------

@pytest.mark.parametrize("br", [1, 128])
def test_quantize_as_many_rows_as_there_can_be(br):
    rows = 2 ** 31 - 1
    x = torch.empty((rows, 1), dtype=torch.bfloat16, device=DEV).normal_(generator=gen(41)).clamp_(2.0 ** -10)
    q, s = ops.quantize_fp8(x, block_rows=br)
    if br == 1:
        # a block of one value: its code is the largest one
        assert all(bool((part == 0x7e).all()) for part in q.view(torch.uint8).split(2 ** 28))
    for first in (0, 2 ** 28 - 128, 2 ** 30 - 256, rows - rows % 128 - 256):
        part = slice(first, min(first + 1024, rows))
        want, scale = plain_quantize(x[part].float().cpu().numpy(), br)
        assert torch.equal(q[part].cpu().view(torch.uint8), torch.from_numpy(want).to(F8).view(torch.uint8))
        got = s[:, part] if br == 1 else s[first // 128:first // 128 + scale.shape[0]]
        assert np.array_equal(got.cpu().numpy(), scale)


def test_grouped_products_of_as_many_rows_as_there_can_be():
    rows, groups = 2 ** 31 - 1, 3
    g = gen(42)
    table = torch.randint(-2, 3, (2 ** 20, 2), device=DEV, generator=g).to(torch.bfloat16)      # (small whole numbers: every product and sum is exact)
    x = table.repeat(2 ** 11, 1)[:rows]
    w = torch.randint(-2, 3, (groups, 2, 2), device=DEV, generator=g).to(torch.bfloat16)
    ends = [2 ** 30 + 5, 2 ** 30 + 5, rows - 7]
    for tile in ((16, 64, 4), (128, 128, 1), (256, 256, 1)):       # (each one or more tiles too many)
        with pytest.raises(L.CatcocError, match="tiles are more than one launch holds"):
            ops.grouped_matmul(x, w, torch.tensor(ends, dtype=torch.int32, device=DEV), tile=tile)
    for tile in (None, (64, 64, 1)):
        out = ops.grouped_matmul(x, w, torch.tensor(ends, dtype=torch.int32, device=DEV), tile=tile)
        assert ran((64, 64, 1))
        for first in range(0, rows, 2 ** 27):
            last = min(first + 2 ** 27, rows)
            for begin, end, e in ((0, ends[0], 0), (ends[0], ends[2], 2)):
                i, j = max(first, begin), min(last, end)
                if i < j:
                    want = x[i:j, :1] * w[e, 0] + x[i:j, 1:] * w[e, 1]
                    assert torch.equal(out[i:j], want), (tile, i, j)
        assert not out[ends[2]:].any()
        del out
    fewer = 2 ** 31 - 2 ** 20        # whole tiles of 128 rows that one launch holds
    ops.grouped_matmul(x[:fewer], w, torch.tensor(ends, dtype=torch.int32, device=DEV).clamp_(max=fewer))
    assert L.last_launch().tileCols >= 128


def test_weight_gradients_of_as_many_groups_as_there_can_be():
    groups, k = 65536, 64 * 256 + 1
    g = gen(43)
    x, dy = randn(g, groups, k, dtype=torch.float16), randn(g, groups, 1, dtype=torch.float16)
    dw = ops.grouped_matmul_dw(x, dy, torch.arange(1, groups + 1, dtype=torch.int32, device=DEV))
    assert ran((64, 64, 1))
    for i in range(0, groups, 4096):
        assert torch.equal(dw[i:i + 4096, :, 0], (x[i:i + 4096].float() * dy[i:i + 4096].float()).half())      # (one row a group: one rounding)


# ---- gated rows at the ends of the range --------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantize_gated_where_the_gate_is_nearly_shut(dtype):
    """silu(g) = g e^g / (1 + e^g) of gates down to -180 is far below fp32's range, times a large value it is not.  One value a row: its scale says it."""
    g = gen(51)
    gates = torch.tensor([-80.0, -86.0, -87.0, -87.25, -87.5, -88.0, -88.5, -89.0, -92.0, -100.0, -104.0, -120.0, -150.0, 0.0, -1e-30, 1e-30, 30.0, 100.0], device=DEV)
    gates = torch.cat([gates, torch.rand(2000, device=DEV, generator=g) * 300 - 180])
    ups = torch.tensor([1.0, 1e10, -1e30, 3e38], device=DEV)
    x = torch.cartesian_prod(gates, torch.cat([ups, torch.exp2(torch.rand(20, device=DEV, generator=g) * 190 - 64)])).to(dtype)
    v = x.double()
    v = v[:, 0] * torch.sigmoid(v[:, 0]) * v[:, 1]
    x, v = x[v.abs() < 3.4e38], v[v.abs() < 3.4e38]
    q, s = ops.quantize_fp8(x.contiguous(), gated=True)
    # (a dozen fp32 operations, each off by a few 2^-24, two of them counted twice)
    want = v.abs().clamp_min(2.0 ** -40) / 448
    assert ((s[0].double() - want).abs() <= 2.0 ** -20 * want).all()
    t = v / want
    step = torch.exp2(torch.floor(torch.log2(t.abs().clamp_min(2.0 ** -6))) - 3)
    assert ((q[:, 0].double() - t).abs() <= step / 2 + 2.0 ** -19 * t.abs() + 2.0 ** -30).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_quantize_gated_values_that_are_not_finite(dtype):
    inf, nan = float("inf"), float("nan")
    pairs = [(inf, 1.0), (inf, -2.0), (-inf, 1.0), (nan, 1.0), (1.0, inf), (-1.0, inf), (-100.0, inf), (1.0, nan), (0.0, inf), (inf, 0.0), (inf, inf), (-100.0, nan)]
    x = torch.zeros((len(pairs) + 1, 2 * 130), device=DEV)
    x[:, :130], x[:, 130:] = 1.0, 2.0
    for i, (gate, up) in enumerate(pairs):
        x[i, 7], x[i, 137] = gate, up
    q, s = ops.quantize_fp8(x.to(dtype), gated=True)
    for i, (gate, up) in enumerate(pairs):
        want = torch.tensor(gate).double() * torch.sigmoid(torch.tensor(gate).double()) * up      # what the definition makes of it: an infinity or NaN
        assert not want.isfinite()
        assert s[0, i].isnan() if want.isnan() else s[0, i].isinf(), (gate, up)
        assert q[i, 7].float().isnan()
        assert (q[i, :128].float()[torch.arange(128) != 7] == 0).all() if want.isinf() else q[i, :128].float().isnan().all()
    assert torch.equal(s[1], s[1, -1:].expand(len(pairs) + 1)) and torch.equal(q[:, 128:].view(torch.uint8), q[-1:, 128:].view(torch.uint8).expand(len(pairs) + 1, -1))
    assert s[0, -1].isfinite()


@pytest.mark.parametrize("rows,cols", [(3, 8), (130, 264), (1000, 1792)])
def test_quantize_gated_small_and_large_gates_beside_each_other(rows, cols):
    x = randn(gen(52 + rows), rows, 2 * cols)
    x[:, :cols] *= 60
    q, s = ops.quantize_fp8(x, gated=True)
    v = x.double()
    v = v[:, :cols] * torch.sigmoid(v[:, :cols]) * v[:, cols:]
    want = torch.nn.functional.pad(v.abs(), (0, blocks(cols) * 128 - cols)).view(rows, -1, 128).amax(2).clamp_min(2.0 ** -40).t() / 448
    assert ((s.double() - want).abs() <= 2.0 ** -20 * want).all()
    t = v / spread(s.t(), rows, cols, 1)
    step = torch.exp2(torch.floor(torch.log2(t.abs().clamp_min(2.0 ** -6))) - 3)
    assert ((q.double() - t).abs() <= step / 2 + 2.0 ** -19 * t.abs() + 2.0 ** -30).all()


@pytest.mark.parametrize("k", [128, 1000])
@pytest.mark.parametrize("tile", [(64, 64, 1), (16, 32, 4), (32, 32, 4), (64, 128, 2), (128, 128, 1), (256, 256, 1)])
def test_fp8_products_that_cancel_keep_what_the_instruction_promises(k, tile):
    """Of eight adjacent products 13 bits below the leading one of the largest are kept: each is off by less than 2^-13 of the largest.  Eights without a large
    product lose nothing by another's; all else is fp32."""
    g = gen(61 + k)
    m, n = 40, 300
    x = torch.randint(-8, 9, (m, k), device=DEV, generator=g).float() / 8
    w = torch.randint(-8, 9, (n, k), device=DEV, generator=g).float() / 8
    at = torch.stack([torch.randperm(k, device=DEV, generator=g)[:2] for _ in range(m)])
    at[::4, 1] = at[::4, 0] ^ 1           # the same eight, another one, another block
    at.clamp_(max=k - 1)
    i = torch.arange(m, device=DEV)
    x[i, at[:, 0]], x[i, at[:, 1]] = 128.0, -128.0
    w[: n // 2, :] = torch.where(torch.rand(n // 2, k, device=DEV, generator=g) < 0.5, 128.0, w[: n // 2])     # (2^14 less 2^14 in some of the results)
    x8, w8 = x.to(F8), w.to(F8)
    assert torch.equal(x8.float(), x) and torch.equal(w8.float(), w)
    out = ops.fp8_matmul_allreduce(x8, w8, torch.ones((blocks(k), m), device=DEV), torch.ones((blocks(n), blocks(k)), device=DEV), tile=tile)
    want, lost = torch.zeros((m, n), dtype=torch.float64, device=DEV), torch.zeros((m, n), dtype=torch.float64, device=DEV)
    mag = torch.zeros((m, n), dtype=torch.float64, device=DEV)
    for j in range(0, k, 8):
        p = x[:, None, j:j + 8].double() * w[None, :, j:j + 8].double()
        want += p.sum(2)
        mag += p.abs().sum(2)
        top = torch.exp2(torch.floor(torch.log2(p.abs().amax(2).clamp_min(2.0 ** -20))))
        lost += (torch.frac(p / top[:, :, None] * 2.0 ** 13) != 0).sum(2) * top * 2.0 ** -13
    bound = lost + k * 2.0 ** -23 * mag + ROUND[torch.bfloat16] * (want.abs() + lost)
    off = (out.double() - want).abs()
    assert (off <= bound).all(), float((off / bound).max())
    assert (want.abs() < 2.0 ** -10 * mag).any()       # (some results are what is left of large products)


# ---- streams and graphs: every operator ----------------------------------------------------------------------------------------------

class Everything:
    """One call of each operator on the same few operands, with results of their own."""

    def __init__(self, seed):
        g = self.g = gen(seed)
        self.counts, self.k, self.n = [100, 0, 300, 57], 512, 384
        rows = sum(self.counts)
        self.x, self.dy = randn(g, rows, self.k, dtype=torch.bfloat16), randn(g, rows, self.n, dtype=torch.bfloat16)
        self.w, self.ends = randn(g, 4, self.n, self.k, dtype=torch.bfloat16), ends_of(self.counts)
        self.x8, self.sx = fp8_operand(g, rows, self.k, 1)
        self.w8 = (randn(g, 4, self.n, self.k) * 60).clamp(-448, 448).to(F8)
        self.sw = torch.rand((4, blocks(self.n), blocks(self.k)), device=DEV, generator=g) + 0.5
        self.peers = [randn(g, rows, self.n) for _ in range(2)]

    def inputs(self):
        return [self.x, self.dy, self.x8, self.sx, self.ends, *self.peers]

    def others(self):
        """Other values for the same operands, other groups among them."""
        v = Everything.__new__(Everything)
        Everything.__init__(v, 71)
        v.ends = ends_of([57, 300, 100, 0])
        return v

    def run(self):
        return [*ops.quantize_fp8(self.x), ops.quantize_fp8(self.x, gated=True)[0], ops.quantize_fp8(self.dy, block_rows=128)[0],
                ops.fp8_matmul_allreduce(self.x8, self.w8[1], self.sx, self.sw[1], self.peers, 1, 3), ops.grouped_matmul(self.x, self.w, self.ends, trans_b=True),
                ops.grouped_matmul(self.dy, self.w, self.ends), ops.grouped_matmul_dw(self.x, self.dy, self.ends, out_dtype=torch.float32),
                ops.grouped_fp8_matmul(self.x8, self.w8, self.sx, self.sw, self.ends)]


def same(a, b):
    return all(torch.equal(p.view(torch.uint8), q.view(torch.uint8)) for p, q in zip(a, b))


def test_every_operator_waits_for_its_streams_work():
    now = Everything(70)
    then = now.others()
    then.w, then.w8, then.sw = now.w, now.w8, now.sw
    before, want = now.run(), then.run()
    assert not any(torch.equal(p.view(torch.uint8), q.view(torch.uint8)) for p, q in zip(before, want))
    long = torch.zeros((8192, 8192), dtype=torch.float16, device=DEV)
    side, done = torch.cuda.Stream(), torch.cuda.Event()
    with torch.cuda.stream(side):                   # (memory for all results: allocating may wait for the GPU)
        room = [now.run(), long @ long, long @ long]
    torch.cuda.synchronize()
    del room
    with torch.cuda.stream(side):
        for _ in range(40):
            long = long @ long                      # (20 ms and more before the operands get their values)
        for a, b in zip(now.inputs(), then.inputs()):
            a.copy_(b)
        got = now.run()
        done.record()
    assert not done.query()                         # nothing so far has waited for it
    side.synchronize()
    assert same(got, want)


def test_every_operator_in_a_captured_graph():
    now = Everything(72)
    then = now.others()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        now.run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = now.run()
    for i in range(6):
        for a, b in zip(now.inputs(), then.inputs()):
            keep = a.clone()
            a.copy_(b)
            b.copy_(keep)
        for t in out:
            t.view(torch.uint8).fill_(0xff)
        graph.replay()
        torch.cuda.synchronize()
        assert same(out, now.run()), i


# ---- ends that descend or lie outside the rows ---------------------------------------------------------------------------------------

ODD_ENDS = {"descending": [5, 3, 600, 400], "outside": [-7, 20, 2000, 100], "none": [0, 0, 0, 0], "all_in_the_first": [700, 700, 700, 700], "turning": [700, 0, 700, 0],
            "extremes": [2 ** 31 - 1, -2 ** 31, 300, 2 ** 31 - 1], "one_step_back": [100, 350, 349, 700], "many": [(37 * i) % 700 for i in range(90)],
            "as_many_as_are_dealt": [(53 * i) % 700 for i in range(48)]}


def claims(ends, rows):
    """The rows of every group as the operators bound them, and which rows are one group's alone."""
    mine, times, at = [], np.zeros(rows, int), 0
    for e, end in enumerate(list(ends) + [rows]):
        begin = min(max(ends[e - 1], 0), rows) if e else 0
        mine.append((begin, max(min(end, rows), begin)))
        times[mine[-1][0]:mine[-1][1]] += 1
    return mine, times == 1


@pytest.mark.parametrize("name", sorted(ODD_ENDS))
@pytest.mark.parametrize("kind,tile", [(kind, t) for kind in ("kn", "nk", "f8") for t in [None] + TILES + (SMALL_KN if kind == "kn" else SMALL_NK)])
def test_odd_ends_on_every_tile(name, kind, tile):
    ends, rows, k, n = ODD_ENDS[name], 700, 128, 2600 if name == "as_many_as_are_dealt" else 136
    groups = len(ends)
    g = gen(groups)
    room = torch.full((rows + 8, n), 7.0, dtype=torch.bfloat16, device=DEV)
    on_gpu = torch.tensor(ends, dtype=torch.int32, device=DEV)
    if kind == "f8":
        x, sx = fp8_operand(g, rows, k, 1)
        w = (randn(g, groups, n, k) * 60).clamp(-448, 448).to(F8)
        sw = torch.rand((groups, blocks(n), blocks(k)), device=DEV, generator=g) + 0.5
        ops.grouped_fp8_matmul(x, w, sx, sw, on_gpu, out=room[4:-4], tile=tile)
        a, b = x.double() * spread(sx.t(), rows, k, 1), torch.stack([(w[e].double() * spread(sw[e], n, k, 128)).t() for e in range(groups)])
    else:
        x = randn(g, rows, k, dtype=torch.bfloat16)
        w = randn(g, groups, n, k, dtype=torch.bfloat16) if kind == "nk" else randn(g, groups, k, n, dtype=torch.bfloat16)
        ops.grouped_matmul(x, w, on_gpu, trans_b=kind == "nk", out=room[4:-4], tile=tile)
        a, b = x.double(), w.double().transpose(1, 2) if kind == "nk" else w.double()
    assert (room[:4] == 7).all() and (room[-4:] == 7).all()
    mine, alone = claims(ends, rows)
    height = (tile or (16,))[0]
    most = (rows - groups - 1) // height + groups + 1       # (row tiles of a launch: as many as ascending ends can have)
    if sum(-(-(j - i) // height) for i, j in mine) > most:
        return
    alone, out = torch.from_numpy(alone).to(DEV), room[4:-4]
    for e, (i, j) in enumerate(mine):
        keep = alone[i:j]
        if e == groups:
            assert (out[i:j][keep] == 0).all()
        elif keep.any():
            p, q = a[i:j][keep], b[e]
            close(out[i:j][keep], p @ q, p.abs() @ q.abs(), k, torch.bfloat16, norm2(p, q.t()) if kind == "f8" else None)


@pytest.mark.parametrize("name", sorted(ODD_ENDS))
@pytest.mark.parametrize("tile", [None] + TILES_DW)
def test_odd_ends_of_weight_gradients(name, tile):
    ends, rows, k, n = ODD_ENDS[name], 700, 130, 136
    g = gen(len(ends) + 1)
    x, dy = randn(g, rows, k, dtype=torch.bfloat16), randn(g, rows, n, dtype=torch.bfloat16)
    room = torch.full((len(ends) + 2, k, n), 7.0, device=DEV)
    ops.grouped_matmul_dw(x, dy, torch.tensor(ends, dtype=torch.int32, device=DEV), out=room[1:-1], tile=tile)
    assert (room[0] == 7).all() and (room[-1] == 7).all()
    for e, (i, j) in enumerate(claims(ends, rows)[0][:-1]):      # (a gradient's groups may share rows)
        a, d = x[i:j].double().t(), dy[i:j].double()
        close(room[1 + e], a @ d, a.abs() @ d.abs(), j - i, torch.float32)
