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


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,cols,ld", [(128, 128, 128), (200, 300, 304), (130, 257, 260)])
def test_blocks_beside_values_that_are_not_finite(rows, cols, ld, dtype, pkg, handle):
    """A NaN becomes a NaN code, an infinity +-448, and the scale is that of the block's finite values."""
    w = torch.randn(2, rows, ld, generator=torch.Generator().manual_seed(rows)).cuda().to(TYPES[dtype])
    w[0, 3, 5], w[0, 7, 100], w[1, rows - 1, cols - 1] = float("nan"), float("inf"), -float("inf")
    w[1, :, :128] = float("inf")      # blocks without a finite value
    codes = torch.full((2, rows, ld), 0x55, dtype=torch.uint8, device="cuda")
    scales = torch.empty(2, ref.blocks(rows), ref.blocks(cols), device="cuda")
    handle.quantize_fp8_blocks(w.data_ptr(), kind(pkg, dtype), ld, 2, rows, cols, codes.data_ptr(), ld, scales.data_ptr(), stream())
    x = w[:, :, :cols].float()
    want, want_s = ref.quantise_blocks(torch.where(x.isfinite(), x, 0.0))
    want = want.view(torch.uint8).clone()
    want[x == float("inf")], want[x == -float("inf")], want[x.isnan()] = 0x7e, 0xfe, 0x7f
    got = codes[:, :, :cols].contiguous()
    got[x.isnan()] &= 0x7f
    assert torch.equal(got, want) and torch.equal(scales, want_s)
    assert (codes[:, :, cols:] == 0x55).all()
