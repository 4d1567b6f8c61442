"""Refusals of the operators around a layer of experts: by the Python entry points on host tensors, and by the C ABI before any device is touched."""
import ctypes as C

import pytest
import torch

from mm_rs_with_catlass_amd import lib as L
from mm_rs_with_catlass_amd import ops

F8 = torch.float8_e4m3fn


def refuses(match, fn, *a, **kw):
    with pytest.raises(L.CatcocError, match=match):
        fn(*a, **kw)


def test_norm_refuses():
    x, w = torch.zeros((4, 256), dtype=torch.bfloat16), torch.zeros(256, dtype=torch.bfloat16)
    for n in (ops.rms_norm, ops.rms_norm_fp8):
        refuses("x must be float16, bfloat16 or float32", n, x.int(), w)
        refuses("2 dimensions", n, x[0], w)
        refuses("weight must be", n, x, w.half())
        refuses("weight must have shape", n, x, w[1:])
        refuses("weight must have 1 dimensions", n, x, x)
        refuses("residual must be", n, x, w, x.half())
        refuses("residual must have shape", n, x, w, x[1:])
        refuses("residual_out without", n, x, w, residual_out=x)
        refuses("residual_out must be", n, x, w, x, residual_out=x.float())
        refuses("residual_out must have shape", n, x, w, x, residual_out=x[1:])
        refuses("must live on the GPU", n, x, w, x)
    refuses("out must be", ops.rms_norm, x, w, out=x.float())
    refuses("out must have shape", ops.rms_norm, x, w, out=x[:, 1:])
    refuses("out must be", ops.rms_norm_fp8, x, w, out=x)
    refuses("scale must have shape", ops.rms_norm_fp8, x, w, scale=torch.zeros((4, 2)))
    refuses("kept without keep", ops.rms_norm_fp8, x, w, kept=x)
    refuses("kept must have shape", ops.rms_norm_fp8, x, w, keep=True, kept=x[1:])
    b = ops.rms_norm_backward
    refuses("dy must be float16", b, x.double(), x, w)
    refuses("x must be", b, x, x.half(), w)
    refuses("x must have shape", b, x, x[1:], w)
    refuses("weight must be", b, x, x, w.half())
    refuses("weight must have shape", b, x, x, w[1:])
    refuses("dsum must be", b, x, x, w, x.float())
    refuses("dx must be", b, x, x.float(), w, dx=x)
    refuses("dw must be", b, x, x, w.float(), dw=w)
    refuses("dw must have shape", b, x, x, w, dw=w[1:])
    refuses("must live on the GPU", b, x, x, w)


def test_route_refuses():
    x, r = torch.zeros((5, 12)), ops.route
    refuses("logits must be float16", r, x.double(), 2)
    refuses("2 dimensions", r, x[0], 2)
    refuses("top must be a positive number", r, x, 0)
    refuses("top must be a positive number", r, x, 2.0)
    refuses("score must be one of", r, x, 2, score="relu")
    refuses("groups must be a positive", r, x, 2, groups=0)
    refuses("top_groups must be a positive", r, x, 2, groups=3, top_groups=None)
    refuses("group_top must be a positive", r, x, 2, group_top=-1)
    refuses("bias must be", r, x, 2, bias=torch.zeros(12, dtype=torch.half))
    refuses("bias must have shape", r, x, 2, bias=torch.zeros(11))
    refuses("choice must be", r, x, 2, choice=torch.zeros((5, 2), dtype=torch.int64))
    refuses("choice must have shape", r, x, 2, choice=torch.zeros((5, 3), dtype=torch.int32))
    refuses("share must have shape", r, x, 2, share=torch.zeros((4, 2)))
    refuses("must live on the GPU", r, x, 2)
    b, choice, d = ops.route_backward, torch.zeros((5, 2), dtype=torch.int32), torch.zeros((5, 2))
    refuses("logits must be float16", b, d, x.int(), choice)
    refuses("choice must be", b, d, x, choice.long())
    refuses("choice has 4 rows", b, d, x, choice[1:])
    refuses("dshare must have shape", b, d[:, 1:], x, choice)
    refuses("dshare must be", b, d.half(), x, choice)
    refuses("out must be", b, d, x, choice, out=x.half())
    refuses("score must be one of", b, d, x, choice, score=1)
    refuses("must live on the GPU", b, d, x, choice)


def test_rows_refuse():
    choice, s = torch.zeros((5, 2), dtype=torch.int32), ops.sort_by_expert
    refuses("choice must be", s, choice.short(), 4)
    refuses("2 dimensions", s, choice[0], 4)
    refuses("experts must be a number in 1..1024", s, choice, 0)
    refuses("experts must be a number in 1..1024", s, choice, 1025)
    refuses("order must have shape", s, choice, 4, order=torch.zeros(9, dtype=torch.int32))
    refuses("back must be", s, choice, 4, back=choice.long())
    refuses("back must have shape", s, choice, 4, back=torch.zeros((2, 5), dtype=torch.int32))
    refuses("ends must have shape", s, choice, 4, ends=torch.zeros(5, dtype=torch.int32))
    refuses("must live on the GPU", s, choice, 4)
    x, p = torch.zeros((5, 300), dtype=torch.half), ops.spread_rows
    refuses("x must be", p, x.int(), choice)
    refuses("back must be", p, x, choice.long())
    refuses("back has 4 rows", p, x, choice[1:])
    refuses("scale must have shape", p, x.to(F8), choice, torch.zeros((5, 3)))
    refuses("x with scale must be", p, x, choice, torch.zeros((3, 5)))
    refuses("out_scale without scale", p, x, choice, out_scale=torch.zeros((3, 10)))
    refuses("out_scale must have shape", p, x.to(F8), choice, torch.zeros((3, 5)), out_scale=torch.zeros((3, 5)))
    refuses("out must have shape", p, x, choice, out=x)
    refuses("out must be", p, x, choice, out=torch.zeros((10, 300)))
    refuses("must live on the GPU", p, x, choice)
    y, g = torch.zeros((10, 300), dtype=torch.half), ops.gather_rows
    refuses("y must be float16", g, y.to(F8), choice)
    refuses("y must have shape", g, y[1:], choice)
    refuses("share must be", g, y, choice, torch.zeros((5, 2), dtype=torch.half))
    refuses("share must have shape", g, y, choice, torch.zeros((2, 5)))
    refuses("out must have shape", g, y, choice, out=y)
    refuses("must live on the GPU", g, y, choice)
    b, share = ops.gather_rows_backward, torch.zeros((5, 2))
    refuses("dout must have shape", b, x[1:], y, choice, share)
    refuses("dout must be", b, x.float(), y, choice, share)
    refuses("share must be a tensor", b, x, y, choice, None)
    refuses("dy must have shape", b, x, y, choice, share, dy=x)
    refuses("dshare must be", b, x, y, choice, share, dshare=share.half())
    refuses("must live on the GPU", b, x, y, choice, share)


def test_c_abi_refuses():
    so = L.load()

    def says(match, fn, *a):
        fn(None, *a)
        assert so.catcoc_last_status() != 0 and match in L.last_error(), L.last_error()
    n = so.catcoc_rms_norm
    #            x  res  w  out  sum  q  scale rows cols eps type rt wt
    says("dataType 2", n, 16, None, 16, 16, None, None, None, 4, 128, 1e-6, L.INT8, 0, 0)
    says("residualType 1", n, 16, 16, 16, 16, 16, None, None, 4, 128, 1e-6, L.BF16, L.FP16, 0)
    says("weightType 27", n, 16, None, 16, 16, None, None, None, 4, 128, 1e-6, 0, 0, L.BF16)
    says("columns out of range", n, 16, None, 16, 16, None, None, None, 4, 0, 1e-6, 0, 0, 0)
    says("columns out of range", n, 16, None, 16, 16, None, None, None, 4, 16385, 1e-6, 0, 0, 0)
    says("rows", n, 16, None, 16, 16, None, None, None, 1 << 31, 128, 1e-6, 0, 0, 0)
    says("eps", n, 16, None, 16, 16, None, None, None, 4, 128, -1.0, 0, 0, 0)
    says("eps", n, 16, None, 16, 16, None, None, None, 4, 128, float("nan"), 0, 0, 0)
    says("out or q", n, 16, None, 16, None, None, None, None, 4, 128, 1e-6, 0, 0, 0)
    says("q and scale", n, 16, None, 16, 16, None, 16, None, 4, 128, 1e-6, 0, 0, 0)
    says("residual and sum", n, 16, 16, 16, 16, None, None, None, 4, 128, 1e-6, 0, 0, 0)
    says("non-NULL", n, 16, None, None, 16, None, None, None, 4, 128, 1e-6, 0, 0, 0)
    b = so.catcoc_rms_norm_backward
    need = so.catcoc_rms_norm_backward_workspace_size(100, 1000)
    assert need > 0 and need % 4000 == 0 and so.catcoc_rms_norm_backward_workspace_size(0, 1000) == 0
    #                  dy  x   w  dsum  dx  dw  work bytes rows cols eps type st wt
    says("sumType", b, 16, 16, 16, None, 16, 16, 16, need, 100, 1000, 1e-6, L.FP16, L.BF16, 0)
    says("workspace holds", b, 16, 16, 16, None, 16, 16, 16, need - 1, 100, 1000, 1e-6, 0, 0, 0)
    says("4-byte aligned", b, 16, 16, 16, None, 16, 16, 18, need, 100, 1000, 1e-6, 0, 0, 0)
    says("non-NULL", b, 16, 16, 16, None, 16, None, 16, need, 100, 1000, 1e-6, 0, 0, 0)
    says("non-NULL", b, 16, 16, 16, None, 16, 16, None, need, 100, 1000, 1e-6, 0, 0, 0)
    says("eps", b, 16, 16, 16, None, 16, 16, 16, need, 100, 1000, float("inf"), 0, 0, 0)

    def how(score=0, groups=1, top_groups=1, group_top=1, renormalize=1, scale=1.0):
        return C.byref(L.CatcocRouting(score, groups, top_groups, group_top, renormalize, scale))
    r = so.catcoc_route
    says("how must be", r, 16, None, 16, 16, None, 4, 8, 2, 0)
    for match, a, tail in [("dataType", how(), (4, 8, 2, L.INT8)), ("score 2", how(2), (4, 8, 2, 0)), ("experts out of range", how(), (4, 1025, 2, 0)),
                           ("experts out of range", how(), (4, 0, 2, 0)), ("top 9", how(), (4, 8, 9, 0)), ("top 65", how(), (4, 100, 65, 0)), ("top 0", how(), (4, 8, 0, 0)),
                           ("do not come in 3 groups", how(groups=3), (4, 8, 2, 0)), ("topGroups 5", how(groups=4, top_groups=5), (4, 8, 2, 0)),
                           ("groupTop 3", how(groups=4, group_top=3), (4, 8, 2, 0)), ("fewer than top 3", how(groups=4), (4, 8, 3, 0)),
                           ("at most 64", how(groups=65, top_groups=2), (4, 130, 3, 0)), ("scale", how(scale=float("inf")), (4, 8, 2, 0)),
                           ("tokens", how(), (1 << 31, 8, 2, 0))]:
        says(match, r, 16, None, 16, 16, a, *tail)
    says("non-NULL", r, 16, None, 16, None, how(), 4, 8, 2, 0)
    says("non-NULL", so.catcoc_route_backward, 16, 16, None, 16, how(), 4, 8, 2, 0)
    says("top 9", so.catcoc_route_backward, 16, 16, 16, 16, how(), 4, 8, 9, 0)
    s = so.catcoc_sort_by_expert
    assert so.catcoc_sort_by_expert_workspace_size(100, 8) == 0
    need = so.catcoc_sort_by_expert_workspace_size(1 << 20, 8)
    assert need > 0
    #                   choice order back ends work bytes rows experts bits
    says("choiceBits", s, 16, 16, 16, 16, None, 0, 100, 8, 16)
    says("experts out of range", s, 16, 16, 16, 16, None, 0, 100, 1025, 32)
    says("rows", s, 16, 16, 16, 16, None, 0, 1 << 31, 8, 32)
    says("non-NULL", s, 16, 16, 16, None, None, 0, 0, 8, 32)
    says("non-NULL", s, 16, None, 16, 16, None, 0, 100, 8, 32)
    says("workspace holds", s, 16, 16, 16, 16, 16, need - 1, 1 << 20, 8, 32)
    says("workspace holds 0 bytes", s, 16, 16, 16, 16, None, need, 1 << 20, 8, 32)
    says("4-byte aligned", s, 16, 16, 16, 16, 17, need, 1 << 20, 8, 32)
    p, g, gb = so.catcoc_spread_rows, so.catcoc_gather_rows, so.catcoc_gather_rows_backward
    #                  x  scale back out outScale tokens top cols bytes
    says("valueBytes", p, 16, None, 16, 16, None, 4, 2, 8, 8)
    says("columns out of range", p, 16, None, 16, 16, None, 4, 2, 0, 2)
    says("columns out of range", p, 16, None, 16, 16, None, 4, 2, 1 << 22, 2)
    says("top 65", p, 16, None, 16, 16, None, 4, 65, 8, 2)
    says("top 0", p, 16, None, 16, 16, None, 4, 0, 8, 2)
    says("choices each", p, 16, None, 16, 16, None, 1 << 30, 2, 8, 2)
    says("scale and outScale", p, 16, 16, 16, 16, None, 4, 2, 8, 1)
    says("non-NULL", p, 16, None, None, 16, None, 4, 2, 8, 1)
    says("values of 1 byte", p, 16, 16, 16, 16, 16, 4, 2, 8, 2)
    says("more than one launch holds", p, 16, None, 16, 16, None, 1 << 30, 1, 1 << 21, 2)
    says("dataType", g, 16, 16, None, 16, 4, 2, 8, L.INT8)
    says("non-NULL", g, 16, None, None, 16, 4, 2, 8, L.BF16)
    says("dataType", gb, 16, 16, 16, 16, 16, 16, 4, 2, 8, L.INT8)
    says("non-NULL", gb, 16, 16, 16, None, 16, 16, 4, 2, 8, L.BF16)
    # outputs in the memory of what other waves still read: the last and the first value of an overlap
    for shift in (0, 399, -399):
        says("order lies in the memory of choice", s, 4096, 4096 + shift, 8192, 16384, None, 0, 100, 8, 32)
        says("back lies in the memory of choice", s, 4096, 8192, 4096 + shift, 16384, None, 0, 100, 8, 32)
    says("back lies in the memory of choice", s, 4096, 8192, 4096 + 799, 16384, None, 0, 100, 8, 64)
    says("ends lies in the memory of choice", s, 4096, 8192, 16384, 4096 - 31, None, 0, 100, 8, 32)
    says("out lies in the memory of x", p, 4096, None, 16, 4096 + 63, None, 4, 2, 8, 2)
    says("out lies in the memory of x", p, 4096, None, 16, 4096 - 127, None, 4, 2, 8, 2)
    says("outScale lies in the memory of scale", p, 4096, 16384, 16, 8192, 16384, 4, 2, 8, 1)
    says("out lies in the memory of y", g, 4096, 16, None, 4096 + 127, 4, 2, 8, L.BF16)
    says("out lies in the memory of y", g, 4096, 16, None, 4096 - 127, 4, 2, 8, 0)
    says("dy lies in the memory of dout", gb, 4096, 8192, 16, 16, 4096 - 127, 16, 4, 2, 8, L.BF16)
    # nothing to do: accepted, nothing launched
    for fn, a in ((n, (None, None, None, 16, None, None, None, 0, 128, 1e-6, 0, 0, 0)), (r, (None, None, None, None, how(), 0, 8, 2, 0)),
                  (p, (None, None, None, None, None, 0, 2, 8, 2)), (g, (None, None, None, None, 0, 2, 8, 0)), (gb, (None,) * 6 + (0, 2, 8, 0))):
        fn(None, *a)
        assert so.catcoc_last_status() == 0


def test_sizes_past_32_bits_are_refused():
    """The C ABI has 32-bit sizes: 2^32 + 5 rows must not become five."""
    def wide(*shape, dtype=torch.float16):
        return torch.zeros((1,) * len(shape), dtype=dtype).expand(*shape)
    far = 2 ** 32 + 5
    for n in (ops.rms_norm, ops.rms_norm_fp8):
        refuses("x has 4294967301 rows", n, wide(far, 1), wide(1))
        refuses("x has 4294967301 columns", n, wide(1, far), wide(far))
    refuses("dy has 4294967301 rows", ops.rms_norm_backward, wide(far, 1), wide(far, 1), wide(1))
    refuses("logits has 4294967301 rows", ops.route, wide(far, 4), 1)
    refuses("logits has 4294967301 columns", ops.route, wide(4, far), 1)
    refuses("top must be", ops.route, wide(4, 4), far)
    refuses("logits has 4294967301 rows", ops.route_backward, wide(far, 1, dtype=torch.float32), wide(far, 4), wide(far, 1, dtype=torch.int32))
    i32 = torch.int32
    refuses("choice has 4294967301 rows", ops.sort_by_expert, wide(far, 1, dtype=i32), 4)
    refuses("x has 4294967301 rows", ops.spread_rows, wide(far, 1), wide(far, 1, dtype=i32))
    refuses("x has 4294967301 columns", ops.spread_rows, wide(4, far), wide(4, 1, dtype=i32))
    refuses("back has 4294967301 rows", ops.gather_rows, wide(far, 1), wide(far, 1, dtype=i32))
    refuses("y has 4294967301 columns", ops.gather_rows, wide(4, far), wide(4, 1, dtype=i32))
    refuses("y has 4294967301 columns", ops.gather_rows_backward, wide(4, far), wide(4, far), wide(4, 1, dtype=i32), wide(4, 1, dtype=torch.float32))


def test_grids_hold_every_workgroup_and_fewer_than_2_32_threads_a_dimension(tmp_path):
    """The arithmetic of launches in two dimensions, compiled for the host: every block size, from one workgroup to 2^31."""
    import os
    import subprocess
    csrc = os.path.join(os.path.dirname(os.path.abspath(L.__file__)), "csrc")
    source, program = tmp_path / "grid.cpp", tmp_path / "grid"
    source.write_text(r"""
#include <stdio.h>
#include <initializer_list>
#include "launch_grid.h"
int main()
{
    for (uint32_t threads = 64; threads <= 1024; threads *= 2)
        for (uint64_t wgs : {1ull, 4099ull, (1ull << 22) - 1, 1ull << 22, (1ull << 22) + 5, (1ull << 32) / threads - 1, (1ull << 32) / threads, (1ull << 32) / threads + 1, 1ull << 29, 1ull << 30, 1ull << 31}) {
            const catcoc::LaunchGrid g = catcoc::launch_grid(wgs, threads);
            printf("%u %llu %u %u\n", threads, (unsigned long long)wgs, g.x, g.y);
        }
}
""")
    subprocess.run([os.environ.get("CXX", "g++"), "-std=c++17", "-I", csrc, str(source), "-o", str(program)], check=True)
    lines = subprocess.run([str(program)], check=True, capture_output=True, text=True).stdout.split("\n")[:-1]
    assert len(lines) == 5 * 11
    for line in lines:
        threads, wgs, x, y = map(int, line.split())
        assert 0 < x * threads < 2 ** 32 and 0 < y <= 65535 and x * y >= wgs and (y == 1 or x * (y - 1) < wgs), line
        assert y == 1 or x & (x - 1) == 0
        if wgs * threads < 2 ** 32:
            assert (x, y) == (wgs, 1)


def test_one_gradient_of_gathered_rows_refuses():
    choice, share, x, y = torch.zeros((5, 2), dtype=torch.int32), torch.zeros((5, 2)), torch.zeros((5, 300), dtype=torch.half), torch.zeros((10, 300), dtype=torch.half)
    b = ops.gather_rows_backward
    refuses("dshare without y", b, x, None, choice, share, dshare=share)
    refuses("no gradient is wanted", b, x, None, choice, share, rows=False)
    refuses("dy without rows", b, x, y, choice, share, dy=y, rows=False)
    refuses("dout must have shape", b, x[1:], None, choice, share)
    refuses("dout must be float16", b, x.int(), None, choice, share)
    refuses("dy must be", b, x, None, choice, share, dy=y.float())
    refuses("dy must have shape", b, x, None, choice, share, dy=x)
    refuses("must live on the GPU", b, x, None, choice, share)
    refuses("must live on the GPU", b, x, y, choice, share, rows=False)
    so = L.load()
    for match, a in [("dy or dshare", (16, 16, 16, 16, None, None)), ("y and dshare come", (16, None, 16, 16, 16, 16)), ("y and dshare come", (16, 16, 16, 16, 16, None)),
                     ("non-NULL", (None, 16, 16, 16, 16, 16)), ("non-NULL", (16, 16, None, 16, 16, 16)), ("non-NULL", (16, 16, 16, None, 16, 16))]:
        so.catcoc_gather_rows_backward(None, *a, 4, 2, 8, L.BF16)
        assert so.catcoc_last_status() != 0 and match in L.last_error(), L.last_error()


def test_outputs_in_the_memory_of_operands_are_refused():
    """Every pair of an output and an operand or another output: one byte of them in common, at either end; and the outputs that may take an operand's place, a row off it."""
    so = L.load()
    how = C.byref(L.CatcocRouting(0, 1, 1, 1, 1, 1.0))
    T = 32                                                      # tokens or rows, of 256 values; two choices each
    need = so.catcoc_rms_norm_backward_workspace_size(T, 256)
    sorted_rows = 1 << 20
    sort_need = so.catcoc_sort_by_expert_workspace_size(sorted_rows, 8)
    values, wide, choices, scales = T * 256 * 2, T * 512 * 2, T * 2 * 4, T * 2 * 4
    calls = [
        (so.catcoc_rms_norm, [("x", values), ("residual", 2 * values), ("weight", 512), ("out", values), ("sum", 2 * values), ("q", values // 2), ("scale", scales)],
         (T, 256, 1e-6, L.BF16, 0, L.BF16), ["out", "sum", "q", "scale"]),
        (so.catcoc_rms_norm, [("x", values), ("residual", values), ("weight", 1024), ("out", values), ("sum", values), ("q", values // 2), ("scale", scales)],
         (T, 256, 1e-6, L.BF16, L.BF16, 0), ["out", "sum", "q", "scale"]),
        (so.catcoc_rms_norm_backward, [("dy", values), ("x", 2 * values), ("weight", 512), ("dsum", 2 * values), ("dx", 2 * values), ("dw", 512), ("workspace", need)],
         (need, T, 256, 1e-6, L.FP16, 0, L.FP16), ["dx", "dw", "workspace"]),
        (so.catcoc_route, [("logits", values), ("bias", 1024), ("choice", choices), ("share", choices)], (how, T, 256, 2, L.BF16), ["choice", "share"]),
        (so.catcoc_route_backward, [("dshare", choices), ("logits", values), ("choice", choices), ("dlogits", values)], (how, T, 256, 2, L.BF16), ["dlogits"]),
        (so.catcoc_sort_by_expert, [("choice", sorted_rows * 8), ("order", sorted_rows * 4), ("back", sorted_rows * 4), ("ends", 32), ("workspace", sort_need)],
         (sort_need, sorted_rows, 8, 64), ["order", "back", "ends", "workspace"]),
        (so.catcoc_spread_rows, [("x", values // 2), ("scale", scales), ("back", choices), ("out", wide // 2), ("outScale", 2 * scales)], (T, 2, 256, 1), ["out", "outScale"]),
        (so.catcoc_gather_rows, [("y", wide), ("back", choices), ("share", choices), ("out", values)], (T, 2, 256, L.BF16), ["out"]),
        (so.catcoc_gather_rows_backward, [("dout", values), ("y", wide), ("back", choices), ("share", choices), ("dy", wide), ("dshare", choices)],
         (T, 2, 256, L.BF16), ["dy", "dshare"]),
        # (values of one column: as many bytes as the shares, but not in their order)
        (so.catcoc_gather_rows_backward, [("dout", T * 4), ("y", choices), ("back", choices), ("share", choices), ("dy", choices), ("dshare", choices)], (T, 2, 1, 0), ["dy", "dshare"]),
    ]
    seen = 0
    for fn, operands, tail, outs in calls:
        size = dict(operands)
        apart = {name: (i + 1) << 32 for i, name in enumerate(size)}
        for out in outs:
            for other in size:
                if other == out:
                    continue
                # (addresses of floats and indexes may be any here: nothing is launched; the workspaces' are multiples of four)
                for shift in (size[other] - 4, 4 - size[out], 4 if size[other] > 4 else -4):
                    at = dict(apart)
                    at[out] = apart[other] + shift
                    fn(None, *at.values(), *tail)
                    said = L.last_error()
                    assert so.catcoc_last_status() != 0 and set(said.split(" lies in the memory of ")) == {out, other}, (fn.__name__, out, other, shift, said)
                    seen += 1
    assert seen > 100
    # in an operand's very place, but not of its rows: dy in share's, dshare in y's (one column)
    fn, operands, tail, _ = calls[-1]
    for out, other in (("dy", "share"), ("dshare", "y"), ("dy", "back"), ("dshare", "dout")):
        at = {name: (i + 1) << 32 for i, (name, _) in enumerate(operands)}
        at[out] = at[other]
        fn(None, *at.values(), *tail)
        assert so.catcoc_last_status() != 0 and "%s lies in the memory of %s" % (out, other) in L.last_error()
    # and of values of another size
    fn, operands, tail, _ = calls[0]
    for out, other in (("out", "residual"), ("sum", "x"), ("q", "x")):
        at = {name: (i + 1) << 32 for i, (name, _) in enumerate(operands)}
        at[out] = at[other]
        fn(None, *at.values(), *tail)
        assert so.catcoc_last_status() != 0 and "%s lies in the memory of %s" % (out, other) in L.last_error()
