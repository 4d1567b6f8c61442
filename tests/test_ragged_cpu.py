"""Refusals of the e4m3 and grouped operators: by the Python entry points on host tensors, and by the C ABI before any device is touched."""
import ctypes as C

import pytest
import torch

from mm_rs_with_catlass_amd import lib as L
from mm_rs_with_catlass_amd import ops

F8 = torch.float8_e4m3fn


def refuses(match, fn, *a, **kw):
    with pytest.raises(L.CatcocError, match=match):
        fn(*a, **kw)


def test_quantize_refuses():
    x = torch.zeros((4, 256), dtype=torch.bfloat16)
    q = ops.quantize_fp8
    refuses("x must be", q, x.int())
    refuses("2 dimensions", q, x[0])
    refuses("block_rows must be", q, x, block_rows=64)
    refuses("block_rows=1", q, x, block_rows=128, gated=True)
    refuses("gate and up", q, x[:, :255], gated=True)
    refuses("out must have shape", q, x, out=torch.empty((4, 255), dtype=F8))
    refuses("out must be", q, x, out=torch.empty((4, 256), dtype=torch.uint8))
    refuses("scale must have shape", q, x, scale=torch.empty((4, 2)))
    refuses("must live on the GPU", q, x)


def test_fp8_matmul_refuses():
    m, k, n = 8, 300, 200
    x, w = torch.zeros((m, k), dtype=F8), torch.zeros((n, k), dtype=F8)
    sx, sw = torch.ones((3, m)), torch.ones((2, 3))
    f = ops.fp8_matmul_allreduce
    refuses("x1 must be", f, x.view(torch.uint8), w, sx, sw)
    refuses("x2 must be", f, x, w.float(), sx, sw)
    refuses("k extent", f, x, w[:, :-1], sx, sw)
    refuses("scale_x1 must have shape", f, x, w, sx.t(), sw)
    refuses("scale_x2 must have shape", f, x, w, sx, sw[:1])
    refuses("scale_x1 must be", f, x, w, sx.half(), sw)
    refuses("out_dtype must be float16 or bfloat16", f, x, w, sx, sw, out_dtype=torch.float32)
    refuses("out must have shape", f, x, w, sx, sw, out=torch.empty((m, n + 1), dtype=torch.bfloat16))
    refuses("rank_size - 1", f, x, w, sx, sw, rank_size=2)
    refuses(r"peers\[0\] has shape", f, x, w, sx, sw, [torch.zeros((m, n))], rank_size=2, peer_row_offset=1)
    refuses(r"peers\[0\] must be", f, x, w, sx, sw, [torch.zeros((m, n), dtype=torch.float16)], rank_size=2)
    refuses("peer_row_offset", f, x, w, sx, sw, peer_row_offset=-1)
    refuses("out of range", f, x, w, sx, sw, rank=1)
    refuses("must live on the GPU", f, x, w, sx, sw)


def test_grouped_operators_refuse():
    rows, k, n, groups = 10, 64, 48, 3
    x, dy = torch.zeros((rows, k), dtype=torch.float16), torch.zeros((rows, n), dtype=torch.float16)
    w, ends = torch.zeros((groups, k, n), dtype=torch.float16), torch.tensor([1, 2, 10], dtype=torch.int32)
    f = ops.grouped_matmul
    refuses("x must be float16 or bfloat16", f, x.float(), w, ends)
    refuses("w must be", f, x, w.bfloat16(), ends)
    refuses("3 dimensions", f, x, w[0], ends)
    refuses("k extent", f, x, w, ends, trans_b=True)
    refuses("group_ends must be", f, x, w, ends.long())
    refuses("group_ends must have shape", f, x, w, ends[:2])
    refuses("at least one group", f, x, w[:0], ends[:0])
    refuses("out must have shape", f, x, w, ends, out=torch.empty((rows, k), dtype=torch.float16))
    refuses("must live on the GPU", f, x, w, ends)
    d = ops.grouped_matmul_dw
    refuses("dy must be", d, x, dy.bfloat16(), ends)
    refuses("dy has 9 rows", d, x, dy[:9], ends)
    refuses("out_dtype must be", d, x, dy, ends, out_dtype=torch.float64)
    refuses("out must have shape", d, x, dy, ends, out=torch.empty((groups, n, k), dtype=torch.float32))
    refuses("group_ends must be", d, x, dy, ends.float())
    refuses("group_ends must be", d, x, dy, [1, 2, 10])
    refuses("must live on the GPU", d, x, dy, ends)
    q = ops.grouped_fp8_matmul
    x8, w8 = torch.zeros((rows, k), dtype=F8), torch.zeros((groups, n, k), dtype=F8)
    sx, sw = torch.ones((1, rows)), torch.ones((groups, 1, 1))
    refuses("x must be", q, x, w8, sx, sw, ends)
    refuses("w must be", q, x8, w, sx, sw, ends)
    refuses("scale_w must have", q, x8, w8, sx, sw[0], ends)
    refuses("scale_x must have shape", q, x8, w8, sx.t(), sw, ends)
    refuses("out_dtype must be", q, x8, w8, sx, sw, ends, out_dtype=torch.float32)
    refuses("must live on the GPU", q, x8, w8, sx, sw, ends)


def test_c_abi_refuses():
    so = L.load()

    def says(match, fn, *a):
        fn(None, *a)
        assert so.catcoc_last_status() != 0 and match in L.last_error(), L.last_error()
    says("blockRows", so.catcoc_quantize_fp8, 16, 16, 16, 4, 128, 2, 0, L.BF16)
    says("gated", so.catcoc_quantize_fp8, 16, 16, 16, 4, 128, 128, 1, L.BF16)
    says("dataType", so.catcoc_quantize_fp8, 16, 16, 16, 4, 128, 1, 0, L.INT8)
    says("non-NULL", so.catcoc_quantize_fp8, 16, None, 16, 4, 128, 1, 0, L.BF16)
    says("empty problem", so.catcoc_quantize_fp8, 16, 16, 16, 4, 0, 1, 0, L.BF16)
    f = so.catcoc_fp8_matmul_allreduce
    says("outDataType", f, 16, 16, 16, 16, 16, None, 4, 4, 4, L.INT8, None)
    says("must be below", f, 16, 16, 16, 16, 16, None, 4, 1 << 22, 4, L.BF16, None)
    says("non-NULL", f, 16, 16, 16, None, 16, None, 4, 4, 4, L.BF16, None)
    d = L.make_desc(0, 3, [16])
    d.peerLd = 4
    says("peers[1] is NULL", f, 16, 16, 16, 16, 16, C.addressof(d), 4, 4, 4, L.BF16, None)
    d.magic = 0
    says("bad magic", f, 16, 16, 16, 16, 16, C.addressof(d), 4, 4, 4, L.BF16, None)
    g = so.catcoc_grouped_matmul
    for match, a in [("dataType", (L.INT8, 16, 16, 16, 16, 4, 4, 4, 2, 0)), ("groups out of range", (L.BF16, 16, 16, 16, 16, 4, 4, 4, 0, 0)),
                     ("non-NULL", (L.BF16, 16, 16, None, 16, 4, 4, 4, 2, 0)), ("empty problem", (L.BF16, 16, 16, 16, 16, 4, 0, 4, 2, 0)),
                     ("rows", (L.BF16, 16, 16, 16, 16, 1 << 31, 4, 4, 2, 0))]:
        says(match, g, *a, None)
    says("outDataType", so.catcoc_grouped_matmul_dw, L.BF16, 16, 16, 16, 16, 4, 4, 4, 2, 0, L.INT8, None)
    says("non-NULL", so.catcoc_grouped_matmul_dw, L.BF16, 16, 16, 16, None, 4, 4, 4, 2, 0, 0, None)
    says("non-NULL", so.catcoc_grouped_fp8_matmul, 16, 16, 16, 16, 16, None, 4, 4, 4, 2, L.BF16, None)
    says("no kernel of 48x48", g, L.BF16, 16, 16, 16, 16, 4, 4, 4, 2, 0, C.byref(L.CatcocTile(48, 48, 1)))
    # no rows: accepted, nothing launched
    g(None, L.BF16, None, None, None, None, 0, 4, 4, 2, 0, None)
    assert so.catcoc_last_status() == 0


def test_sizes_past_32_bits_are_refused():
    """The C ABI has 32-bit sizes: 2^32 + 5 rows must not become five."""
    def wide(*shape, dtype=F8):
        return torch.zeros((1,) * len(shape), dtype=dtype).expand(*shape)
    far, h = 2 ** 32 + 5, torch.float16
    ends = torch.ones(1, dtype=torch.int32)
    refuses("x has 4294967301 rows", ops.quantize_fp8, wide(far, 1, dtype=h))
    refuses("x has 4294967301 columns", ops.quantize_fp8, wide(1, far, dtype=h))
    refuses("x has 4294967301 columns", ops.quantize_fp8, wide(1, 2 * far, dtype=h), gated=True)
    f = ops.fp8_matmul_allreduce
    refuses("x1 has 4294967301 rows", f, wide(far, 1), wide(4, 1), wide(1, far, dtype=torch.float32), wide(1, 1, dtype=torch.float32))
    refuses("x2 has 4294967301 rows", f, wide(4, 1), wide(far, 1), wide(1, 4, dtype=torch.float32), wide(-(-far // 128), 1, dtype=torch.float32))
    refuses("x1 has 4294967301 columns", f, wide(4, far), wide(4, far), wide(-(-far // 128), 4, dtype=torch.float32), wide(1, -(-far // 128), dtype=torch.float32))
    m, d, e = ops.grouped_matmul, ops.grouped_matmul_dw, ops.grouped_fp8_matmul
    refuses("x has 4294967301 rows", m, wide(far, 1, dtype=h), wide(1, 1, 1, dtype=h), ends)
    refuses("x has 4294967301 columns", m, wide(1, far, dtype=h), wide(1, far, 1, dtype=h), ends)
    refuses("w has 4294967301 columns", m, wide(1, 1, dtype=h), wide(1, 1, far, dtype=h), ends)
    refuses("w has 4294967301 rows", m, wide(1, 1, dtype=h), wide(1, far, 1, dtype=h), ends, trans_b=True)
    refuses("w has 4294967301 groups", m, wide(1, 1, dtype=h), wide(far, 1, 1, dtype=h), wide(far, dtype=torch.int32))
    refuses("x has 4294967301 rows", d, wide(far, 1, dtype=h), wide(far, 1, dtype=h), ends)
    refuses("x has 4294967301 columns", d, wide(1, far, dtype=h), wide(1, 1, dtype=h), ends)
    refuses("dy has 4294967301 columns", d, wide(1, 1, dtype=h), wide(1, far, dtype=h), ends)
    refuses("group_ends has 4294967301 groups", d, wide(1, 1, dtype=h), wide(1, 1, dtype=h), wide(far, dtype=torch.int32))
    refuses("x has 4294967301 rows", e, wide(far, 1), wide(1, 1, 1), wide(1, far, dtype=torch.float32), wide(1, 1, 1, dtype=torch.float32), ends)
    refuses("w has 4294967301 rows", e, wide(1, 1), wide(1, far, 1), wide(1, 1, dtype=torch.float32), wide(1, -(-far // 128), 1, dtype=torch.float32), ends)
