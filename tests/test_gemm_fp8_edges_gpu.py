"""The FP8 product beside values that are not finite, and output rows of 16-byte pieces that end inside one."""
import math

import pytest
import torch

import fp8_reference as ref
from test_fp8_layer_gpu import TYPES, check_product, kind, make_product, run_product, stream

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def handle(pkg):
    h = pkg.MoeBlock(64, 64, 8, max_rows=8)
    yield h
    h.synchronize()
    h.close()


# rows, n, k, rows of the groups: 16, 64 and 128 token columns and the wide form, whole and split over clusters of two, four and eight
SHAPES = [(12, 200, 300, None), (16, 256, 7168, None), (40, 260, 1040, None), (214, 225, 7912, None), (200, 1030, 2000, None), (512, 1536, 1024, None),
          (2100, 520, 300, None), (60, 300, 640, [20, 0, 25, 15]), (300, 200, 300, [120, 0, 80, 100]), (700, 520, 400, [300, 0, 250, 150])]


@pytest.mark.parametrize("rows,n,k,counts", SHAPES)
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_scales_that_are_not_finite_reach_what_they_scale(rows, n, k, counts, value, pkg, handle):
    """A row's scale: that row's outputs.  A block's scale: the block's columns in the rows of its group."""
    groups = len(counts) if counts else 1
    p = make_product(5, rows, n, k, groups=groups, counts=counts)
    clean = run_product(pkg, handle, p, "f32")
    bad, block, group = rows // 2, (n - 1) // 128, groups - 1
    p["sa"][bad, ref.blocks(k) // 2] = value
    p["sb"][group, block, ref.blocks(k) - 1] = value
    got = run_product(pkg, handle, p, "f32")
    hit = torch.zeros(rows, n, dtype=torch.bool, device="cuda")
    hit[bad] = True
    first = int(p["offsets"][group]) if counts else 0
    hit[first:, 128 * block:] = True
    assert torch.equal(got[~hit], clean[~hit])
    assert not got[hit].isfinite().any()      # (a sum of 128 random products is not zero: no inf x 0)


@pytest.mark.parametrize("rows,k", [(9, 300), (60, 640), (120, 2000), (200, 4096), (700, 400), (5000, 200)])
@pytest.mark.parametrize("n", [257, 260, 262, 519])
@pytest.mark.parametrize("out", ["f16", "bf16", "f32"])
def test_aligned_output_rows_that_end_inside_a_piece(rows, n, k, out, pkg, handle):
    """Rows 16-byte aligned, columns not made of 16-byte pieces: what lies between the last column and the next row stays."""
    p = make_product(n, rows, n, k, bias=True)
    p["sa"] *= 0.01          # inside the range of fp16
    check_product(p, run_product(pkg, handle, p, out, ld_out=(n + 7) // 8 * 8 + 8), out)


@pytest.mark.parametrize("n", [130, 262])
@pytest.mark.parametrize("out", ["bf16", "f32"])
def test_aligned_output_rows_of_groups_that_end_inside_a_piece(n, out, pkg, handle):
    for counts in ([5, 0, 20], [130, 1, 0, 127, 128, 129]):
        p = make_product(n, sum(counts), n, 384, groups=len(counts), counts=counts, bias=True)
        check_product(p, run_product(pkg, handle, p, out, ld_out=(n + 7) // 8 * 8), out)


def test_product_of_as_many_rows_as_an_index_holds(pkg, handle):
    """2^31 - 256 rows of 16 codes: the first and the last rows are random, those between them alike."""
    rows, edge = 2 ** 31 - 256, 2000
    p = make_product(8, 2 * edge, 1, 16)
    large = {**p, "rows": rows, "a": torch.full((rows, 16), 0x38, dtype=torch.uint8, device="cuda"), "sa": torch.ones(rows, 1, device="cuda")}   # 0x38: 1
    for name in ("a", "sa"):
        large[name][:edge], large[name][-edge:] = p[name][:edge], p[name][edge:]
    out = run_product(pkg, handle, large, "bf16")
    check_product(p, torch.cat([out[:edge], out[-edge:]]), "bf16")
    between = out[edge:rows - edge]
    want = p["b"].view(torch.float8_e4m3fn).double().sum() * p["sb"].double()[0, 0, 0]
    # 16 products and their scale, each off by at most 2^-23 of the magnitudes, and the rounding to bf16
    mag = p["b"].view(torch.float8_e4m3fn).double().abs().sum() * p["sb"].double()[0, 0, 0]
    assert abs(float(between[0]) - float(want)) <= abs(float(want)) * 2.0 ** -8 + float(mag) * 17 * 2.0 ** -23
    assert (between == between[0]).all()
    del large, out, between
    torch.cuda.empty_cache()


# all but one in the form of many rows per group, whole: the copy engine writes pieces of 16 bytes
WIDE = [(809, 146, 2, [300, 300, 209]), (2132, 129, 4, [700, 732, 700]), (4886, 410, 4, [1600, 1600, 1686]), (4707, 745, 1500, None), (2600, 1271, 1863, None),
        (6000, 500, 1500, None), (9000, 257, 130, None), (3000, 515, 260, [1000, 0, 1999])]


@pytest.mark.parametrize("rows,n,k,counts", WIDE)
@pytest.mark.parametrize("out", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("beside", [0, 8, 40])
def test_an_output_inside_a_wider_tensor(rows, n, k, counts, out, beside, pkg, handle):
    """`beside` columns on its left, at least as many on its right; they stay, and so does what lies behind the last row."""
    p = make_product(rows, rows, n, k, groups=len(counts) if counts else 1, counts=counts, bias=True)
    p["sa"] *= 0.003         # inside the range of fp16
    ld = (beside + n + 7) // 8 * 8 + beside
    whole = torch.full((rows * ld + 64,), 77.0, dtype=TYPES[out], device="cuda")
    view = whole[:rows * ld].view(rows, ld)[:, beside:]
    handle.gemm_fp8(p["a"].data_ptr(), p["a"].shape[1], p["sa"].data_ptr(), p["sa"].shape[1], rows, p["b"].data_ptr(), p["b"].shape[2], p["sb"].data_ptr(), n, k,
                    view.data_ptr(), kind(pkg, out), ld, bias_ptr=p["bias"].data_ptr(), n_groups=p["groups"],
                    offsets_ptr=0 if p["offsets"] is None else p["offsets"].data_ptr(), stream=stream())
    check_product(p, view, out)
    assert (whole[rows * ld:] == 77).all() and (whole[:rows * ld].view(rows, ld)[:, :beside] == 77).all()
