"""The FP8 quantiser at the ends of its arguments' ranges, against its definition in 64 bits (fp8_reference.py)."""
import pytest
import torch

import fp8_reference as ref
from test_fp8_layer_gpu import TYPES, kind, stream

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def handle(pkg):
    h = pkg.MoeBlock(64, 64, 8, max_rows=8)
    yield h
    h.close()


@pytest.mark.parametrize("alpha", [3.4e38, -3.4e38, 2.4e38, 1e30, 0.0, -1.702])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("cols", [128, 200, 345])
def test_swiglu_of_any_finite_alpha(alpha, dtype, cols, pkg, handle):
    """Gates of 0 among others: a sigmoid of 0 is a half whatever alpha is."""
    x = (4 * torch.randn(6, 2 * cols, generator=torch.Generator().manual_seed(cols))).cuda().to(TYPES[dtype])
    x[1::2, ::4] = 0
    x[2] = 0
    codes, scales = torch.zeros(6, cols, dtype=torch.uint8, device="cuda"), torch.zeros(6, ref.blocks(cols), device="cuda")
    handle.quantize_fp8(x.data_ptr(), kind(pkg, dtype), 2 * cols, 6, cols, codes.data_ptr(), cols, scales.data_ptr(), ref.blocks(cols),
                        act=pkg.ACT_SWIGLU, alpha=alpha, stream=stream())
    v = ref.activation(x, "swiglu", alpha=alpha)
    step = scales.double()[:, torch.arange(cols) // 128]
    # half a step of the code (its smallest is 2^-9) and 2^-16 for exponential, quotient and scale
    far = (codes.view(torch.float8_e4m3fn).double() * step - v).abs()
    assert (far <= v.abs() * (2.0 ** -4 + 2.0 ** -16) + step * 2.0 ** -10).all()
