"""CPU tests of the mixture-of-experts steps: what the C ABI refuses before it touches CUDA (made-up addresses do), and the work
list's own arithmetic, compiled for the host."""
import os
import shutil
import subprocess

import pytest

from conftest import ROOT

A, B, C, D, E, F = (0x10000 * i for i in range(1, 7))


def test_norm_refuses(capi):
    L = capi.load()

    def call(x=A, residual=B, weight=C, eps=1e-6, rows=8, n=128, residual_out=B, norm_out=None, codes=D, scales=E):
        return L.catccos_b200_add_rms_norm_mx_quant(None, x, residual, weight, eps, rows, n, residual_out, norm_out, codes, scales)

    for bad in (dict(x=None), dict(weight=None), dict(codes=None), dict(scales=None), dict(residual=None), dict(residual_out=None),
                dict(n=0), dict(n=48), dict(n=32800), dict(rows=2**31), dict(eps=0.0), dict(eps=1e-31), dict(eps=float("nan")), dict(x=A + 8), dict(residual=B + 2),
                dict(weight=C + 4), dict(residual_out=B + 8), dict(norm_out=F + 8), dict(codes=D + 8), dict(scales=E + 2),
                # overlaps: one output in another, or in what is read, other than the whole of x or residual
                dict(norm_out=B), dict(norm_out=B + 16), dict(residual_out=A + 32), dict(residual_out=B + 1024), dict(norm_out=A + 1024),
                dict(codes=A), dict(codes=B + 16), dict(scales=D + 512), dict(scales=C), dict(residual_out=C), dict(codes=F, norm_out=F)):
        assert call(**bad) == -1, bad
    assert call(rows=0) == 0  # an empty batch needs no addresses and no device


def test_route_refuses(capi):
    L = capi.load()

    def call(logits=A, bf16=0, bias=B, tokens=4, experts=64, top_k=4, groups=1, top_groups=1, group_best=1, score=0, renormalize=1,
             scale=1.0, ids=C, weights=D):
        return L.catccos_b200_moe_route(None, logits, bf16, bias, tokens, experts, top_k, groups, top_groups, group_best, score, renormalize,
                                        scale, ids, weights)

    for bad in (dict(logits=None), dict(ids=None), dict(weights=None), dict(logits=A + 2), dict(logits=A + 1, bf16=1), dict(bias=B + 2),
                dict(ids=C + 1), dict(weights=D + 2), dict(experts=0), dict(experts=1025), dict(top_k=0), dict(top_k=33), dict(groups=0),
                dict(groups=7), dict(groups=64), dict(groups=8, top_groups=9), dict(top_groups=0), dict(groups=32, top_groups=1),
                dict(group_best=0), dict(group_best=3), dict(score=2), dict(score=-1), dict(bf16=2), dict(scale=float("inf")),
                dict(tokens=2**31), dict(ids=D), dict(weights=C + 32), dict(ids=A + 64), dict(weights=B)):
        assert call(**bad) == -1, bad
    assert call(tokens=0) == 0


def test_row_plan_refuses(capi):
    L = capi.load()

    def call(ids=A, routes=8, experts=4, first=0, index=B, offsets=C):
        return L.catccos_b200_moe_row_plan(None, ids, routes, experts, first, index, offsets)

    for bad in (dict(ids=None), dict(index=None), dict(offsets=None), dict(ids=A + 2), dict(index=B + 1), dict(offsets=C + 2),
                dict(experts=0), dict(experts=1025), dict(first=-1), dict(routes=2**31), dict(index=A + 4),
                dict(offsets=A), dict(offsets=B + 16)):
        assert call(**bad) == -1, bad


def test_combine_refuses(capi):
    L = capi.load()

    def call(y=A, rows=8, index=B, weights=C, shared=D, out=E, tokens=4, n=64, top_k=2, f16=0):
        return L.catccos_b200_moe_combine(None, y, rows, index, weights, shared, out, tokens, n, top_k, f16)

    for bad in (dict(y=None), dict(index=None), dict(weights=None), dict(out=None), dict(y=A + 8), dict(shared=D + 8), dict(out=E + 8),
                dict(index=B + 2), dict(weights=C + 2), dict(n=0), dict(n=12), dict(top_k=0), dict(f16=2), dict(rows=2**31),
                dict(out=A), dict(out=D + 16), dict(out=B), dict(shared=None, out=A + 512), dict(weights=E)):
        assert call(**bad) == -1, bad
    assert call(tokens=0) == 0


def test_grouped_gemm_refuses(capi):
    L = capi.load()

    def call(a=A, step=128, a_scale=B, scale_step=4, b=C, b_scale=D, offsets=E, c=F, rows=8, experts=2, n=64, k=128):
        return L.catccos_b200_mx_grouped_gemm(None, a, step, a_scale, scale_step, b, b_scale, offsets, c, rows, experts, n, k)

    for bad in (dict(a=None), dict(a_scale=None), dict(b=None), dict(b_scale=None), dict(offsets=None), dict(c=None), dict(a=A + 8),
                dict(a_scale=B + 2), dict(b=C + 8), dict(b_scale=D + 1), dict(offsets=E + 2), dict(c=F + 16), dict(step=127),
                dict(step=136), dict(scale_step=3), dict(scale_step=6), dict(n=0), dict(n=24), dict(k=0), dict(k=64), dict(experts=0),
                dict(experts=1025), dict(experts=1024, k=2**22, step=2**22), dict(rows=2**31), dict(c=A), dict(c=A + 1024 - 128),
                dict(c=C + 128 * 128 - 32), dict(a_scale=F), dict(b_scale=F + 32), dict(offsets=F + 1020)):
        assert call(**bad) == -1, bad
    assert call(rows=0) == 0
    for option in (b"a_dtype", b"b_dtype"):
        L.catccos_b200_set_option(option, 2)
        assert call() == -1
        L.catccos_b200_set_option(option, 0)


def test_matvec_refuses(capi):
    L = capi.load()

    def call(x=A, w=B, w_scale=C, ids=D, out=E, rows=8, x_rows=4, experts=2, n=64, k=128):
        return L.catccos_b200_mx_fp4_matvec(None, x, w, w_scale, ids, out, rows, x_rows, experts, n, k)

    for bad in (dict(x=None), dict(w=None), dict(w_scale=None), dict(out=None), dict(x=A + 8), dict(w=B + 8), dict(w_scale=C + 8),
                dict(ids=D + 2), dict(out=E + 2), dict(n=0), dict(n=24), dict(k=0), dict(k=96), dict(experts=0), dict(x_rows=0),
                dict(x_rows=3), dict(rows=65536, x_rows=65536), dict(ids=None), dict(ids=None, experts=1),
                dict(out=A), dict(out=B + 64), dict(w_scale=E), dict(ids=E + 64)):
        assert call(**bad) == -1, bad
    assert call(rows=0) == 0


def test_typed_calls_refuse(capi):
    L = capi.load()

    def grouped(types, rows=8):
        return L.catccos_b200_mx_grouped_gemm_typed(None, A, 128, B, 4, C, D, E, F, rows, 2, 64, 128, *types)

    def matvec(c_type, rows=8):
        return L.catccos_b200_mx_fp4_matvec_typed(None, A, B, C, D, E, rows, rows // 2, 2, 64, 128, c_type)

    for bad in ((2, 0, 0), (-2, 0, 0), (0, 2, 0), (0, 0, 2), (0, 0, -2)):
        assert grouped(bad) == -1, bad
    assert matvec(2) == -1 and matvec(-2) == -1
    for types in ((0, 1, 0), (1, 0, 1), (-1, -1, -1)):
        assert grouped(types, rows=0) == 0
    assert matvec(1, rows=0) == 0 and matvec(-1, rows=0) == 0
    for option in (b"a_dtype", b"b_dtype"):  # an option counts only where the call leaves its type to it
        L.catccos_b200_set_option(option, 2)
        assert grouped((-1, -1, -1), rows=0) == -1 and grouped((0, 0, 0), rows=0) == 0
        L.catccos_b200_set_option(option, 0)


@pytest.mark.skipif(shutil.which("nvcc") is None, reason="needs nvcc")
def test_rows_of_an_expert_stay_inside_the_matrix(tmp_path):
    exe = tmp_path / "grouped_rows_selftest"
    src = os.path.join(ROOT, "tests", "host", "grouped_rows_selftest.cu")
    subprocess.check_call(["nvcc", "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", "-o", str(exe), src])
    assert "grouped rows ok" in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout
