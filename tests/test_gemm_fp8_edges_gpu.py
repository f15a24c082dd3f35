"""The FP8 product at the ends of its range."""
import pytest
import torch

from test_fp8_layer_gpu import check_product, make_product, run_product

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def handle(pkg):
    h = pkg.MoeBlock(64, 64, 8, max_rows=8)
    yield h
    h.synchronize()
    h.close()


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
