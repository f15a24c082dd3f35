"""Refusals of the FP8 layer operators: every check comes before the device is touched, so it runs without one."""
import ctypes as C

import pytest

INVALID = 1
P = 1 << 20          # an address that is aligned for everything and never read


@pytest.fixture(scope="module")
def handle(pkg):
    """A handle; where there is no GPU, the one that a failed creation leaves for its error message."""
    lib, h = pkg.lib(), C.c_void_p()
    cfg = pkg.MoeConfig(64, 64, 8, 4, 1, 7.0, 1.702, 8, 1, 0, 0, 0)
    lib.moe_create(C.byref(cfg), C.byref(h))
    assert h
    yield h
    lib.moe_destroy(h)


def refused(pkg, handle, rc, *words):
    assert rc == INVALID
    text = pkg.lib().moe_last_error(handle).decode()
    assert all(w in text for w in words), text


def test_null_handle(pkg):
    lib = pkg.lib()
    assert lib.moe_route_scored(None, pkg.RouteRule(8, 2), P, 0, 8, None, 1, P, P, None) == INVALID
    assert lib.moe_group_pairs(None, P, 1, 1, 8, P, P, P, None) == INVALID
    assert lib.moe_quantize_fp8(None, P, 0, 8, 1, 8, 0, 7.0, 1.0, None, 1, 1, None, P, 8, P, 1, None) == INVALID
    assert lib.moe_quantize_fp8_blocks(None, P, 0, 8, 1, 8, 8, P, 8, P, None) == INVALID
    assert lib.moe_gemm_fp8(None, P, 16, P, 1, 1, P, 16, P, 8, 16, 1, None, None, P, 0, 8, None) == INVALID
    assert lib.moe_combine_pairs(None, P, 0, 8, 1, P, P, 1, 1, 8, None, 0, P, 0, 8, None) == INVALID


@pytest.mark.parametrize("change", [
    dict(n_experts=0), dict(n_experts=513), dict(top_k=0), dict(top_k=33), dict(top_k=65), dict(score=2), dict(score=-1), dict(n_groups=0),
    dict(n_groups=3), dict(n_groups=64), dict(n_groups=4, top_groups=5), dict(top_groups=0), dict(group_top=0), dict(group_top=3),
    dict(scale=float("nan")), dict(scale=float("inf"))])
def test_route_rules(change, pkg, handle):
    rule = pkg.RouteRule(**{**dict(n_experts=64, top_k=4), **change})
    refused(pkg, handle, pkg.lib().moe_route_scored(handle, rule, P, 0, 1024, None, 1, P, P, None), "moe_route_scored")


@pytest.mark.parametrize("logits,dtype,ld,bias,rows,idx,w", [
    (0, 0, 64, 0, 1, P, P), (P, 0, 64, 0, 1, 0, P), (P, 0, 64, 0, 1, P, 0), (P, 3, 64, 0, 1, P, P), (P, -1, 64, 0, 1, P, P), (P, 0, 63, 0, 1, P, P),
    (P, 0, 64, 0, -1, P, P), (P + 2, 0, 64, 0, 1, P, P), (P + 1, 1, 64, 0, 1, P, P), (P, 0, 64, P + 2, 1, P, P), (P, 0, 64, 0, 1, P + 1, P)])
def test_route_tensors(logits, dtype, ld, bias, rows, idx, w, pkg, handle):
    refused(pkg, handle, pkg.lib().moe_route_scored(handle, pkg.RouteRule(64, 4), logits, dtype, ld, bias, rows, idx, w, None), "moe_route_scored")


def test_route_null_rule(pkg, handle):
    refused(pkg, handle, pkg.lib().moe_route_scored(handle, None, P, 0, 64, None, 1, P, P, None), "null rule")


@pytest.mark.parametrize("idx,rows,top_k,experts,offsets,pair_row,row_pair", [
    (0, 1, 1, 8, P, P, P), (P, 1, 1, 8, 0, P, P), (P, 1, 1, 8, P, 0, P), (P, -1, 1, 8, P, P, P), (P, 1, 0, 8, P, P, P), (P, 1, 1, 0, P, P, P),
    (P, 1, 1, 1025, P, P, P), (P, 1 << 30, 2, 8, P, P, P), (P + 2, 1, 1, 8, P, P, P), (P, 1, 1, 8, P, P, P + 1)])
def test_group(idx, rows, top_k, experts, offsets, pair_row, row_pair, pkg, handle):
    refused(pkg, handle, pkg.lib().moe_group_pairs(handle, idx, rows, top_k, experts, offsets, pair_row, row_pair, None), "moe_group_pairs")


QUANT = dict(x=P, dtype=1, ld_x=256, rows=4, cols=256, act=0, limit=7.0, alpha=1.7, pair_row=0, fanout=1, out_rows=4, n_rows=0, codes=P, ld_codes=256,
             scales=P, ld_scales=2)


@pytest.mark.parametrize("change", [
    dict(x=0), dict(codes=0), dict(scales=0), dict(dtype=3), dict(ld_x=255), dict(rows=-1), dict(cols=0), dict(ld_codes=255), dict(ld_scales=1),
    dict(act=3), dict(act=1), dict(act=1, ld_x=512, limit=-1.0), dict(act=1, ld_x=512, limit=float("nan")), dict(act=1, ld_x=512, alpha=float("inf")),
    dict(fanout=0), dict(fanout=2), dict(out_rows=3), dict(out_rows=-1, pair_row=P), dict(pair_row=P, fanout=1 << 30), dict(x=P + 1), dict(scales=P + 2),
    dict(pair_row=P + 2, fanout=2), dict(n_rows=P + 3), dict(ld_x=1 << 31), dict(ld_codes=1 << 31), dict(ld_scales=1 << 31),
    dict(rows=1 << 30, out_rows=1 << 30)])
def test_quantise(change, pkg, handle):
    refused(pkg, handle, pkg.lib().moe_quantize_fp8(handle, *{**QUANT, **change}.values(), None), "moe_quantize_fp8")


@pytest.mark.parametrize("w,dtype,ld_w,mats,rows,cols,codes,ld_codes,scales", [
    (0, 0, 64, 1, 8, 64, P, 64, P), (P, 0, 64, 1, 8, 64, 0, 64, P), (P, 0, 64, 1, 8, 64, P, 64, 0), (P, 5, 64, 1, 8, 64, P, 64, P),
    (P, 0, 63, 1, 8, 64, P, 64, P), (P, 0, 64, -1, 8, 64, P, 64, P), (P, 0, 64, 70000, 8, 64, P, 64, P), (P, 0, 64, 1, 0, 64, P, 64, P),
    (P, 0, 64, 1, 8, 0, P, 64, P), (P, 0, 64, 1, 8, 64, P, 63, P), (P + 2, 0, 64, 1, 8, 64, P, 64, P), (P, 0, 64, 1, 65535 * 128 + 1, 64, P, 64, P)])
def test_quantise_blocks(w, dtype, ld_w, mats, rows, cols, codes, ld_codes, scales, pkg, handle):
    refused(pkg, handle, pkg.lib().moe_quantize_fp8_blocks(handle, w, dtype, ld_w, mats, rows, cols, codes, ld_codes, scales, None), "moe_quantize_fp8_blocks")


GEMM = dict(a=P, ld_a=256, sa=P, ld_sa=2, rows=4, b=P, ld_b=256, sb=P, n=64, k=256, n_groups=1, offsets=0, bias=0, out=P, out_dtype=1, ld_out=64)


@pytest.mark.parametrize("change", [
    dict(a=0), dict(sa=0), dict(b=0), dict(sb=0), dict(out=0), dict(ld_a=255), dict(ld_a=264), dict(ld_b=240), dict(ld_b=264), dict(ld_sa=1), dict(rows=-1),
    dict(n=0), dict(k=0), dict(n_groups=0), dict(n_groups=2), dict(n_groups=1025, offsets=P), dict(out_dtype=7), dict(ld_out=63), dict(a=P + 8),
    dict(b=P + 1), dict(sa=P + 2), dict(sb=P + 1), dict(offsets=P + 2), dict(bias=P + 1), dict(out=P + 1)])
def test_gemm(change, pkg, handle):
    refused(pkg, handle, pkg.lib().moe_gemm_fp8(handle, *{**GEMM, **change}.values(), None), "moe_gemm_fp8")


COMBINE = dict(y=P, y_dtype=1, ld_y=64, n_y_rows=8, pair_row=P, w=P, rows=4, top_k=2, cols=64, residual=0, ld_residual=0, out=P, out_dtype=1, ld_out=64)


@pytest.mark.parametrize("change", [
    dict(y=0), dict(pair_row=0), dict(w=0), dict(out=0), dict(y_dtype=3), dict(out_dtype=-1), dict(ld_y=63), dict(ld_out=63), dict(n_y_rows=-1),
    dict(rows=-1), dict(top_k=0), dict(cols=0), dict(residual=P, ld_residual=63), dict(rows=1 << 30, top_k=4), dict(y=P + 1), dict(w=P + 2),
    dict(out=P + 1), dict(residual=P + 1, ld_residual=64)])
def test_combine(change, pkg, handle):
    refused(pkg, handle, pkg.lib().moe_combine_pairs(handle, *{**COMBINE, **change}.values(), None), "moe_combine_pairs")


def test_no_rows_is_a_call_that_does_nothing(pkg, handle):
    lib = pkg.lib()
    assert lib.moe_route_scored(handle, pkg.RouteRule(64, 4), None, 0, 64, None, 0, None, None, None) == 0
    assert lib.moe_quantize_fp8(handle, *{**QUANT, "rows": 0, "x": 0, "codes": 0, "scales": 0}.values(), None) == 0
    assert lib.moe_quantize_fp8_blocks(handle, None, 0, 64, 0, 8, 64, None, 64, None, None) == 0
    assert lib.moe_gemm_fp8(handle, *{**GEMM, "rows": 0, "a": 0, "out": 0}.values(), None) == 0
    assert lib.moe_combine_pairs(handle, *{**COMBINE, "rows": 0, "out": 0}.values(), None) == 0


@pytest.mark.parametrize("change", [dict(rows=2 ** 31 - 255), dict(rows=2 ** 31 - 1), dict(n=2 ** 31 - 255, ld_out=2 ** 31), dict(n=2 ** 31 - 1, ld_out=2 ** 31)])
def test_gemm_of_more_rows_or_columns_than_an_index_holds(change, pkg, handle):
    refused(pkg, handle, pkg.lib().moe_gemm_fp8(handle, *{**GEMM, **change}.values(), None), "moe_gemm_fp8", "in one call")
