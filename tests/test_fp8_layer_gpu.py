"""Operators of an FP8 expert layer on the GPU against their definitions in 64 bits (fp8_reference.py).

Tolerances, by arithmetic.  A stored value of type t is off by half a step, eps(t) / 2 relative (fp16: and half of its
smallest step, 2^-25).  Sums: products of two e4m3 values are exact in fp32; a block of 128 is summed by the tensor core in
fp32 and at most 128 + n_blocks additions follow one another, each off by at most one last place (2^-23) of a partial sum,
which the sum of the magnitudes bounds; scales add two roundings, inside the same count.  Routing weights: at most sixteen
roundings of 2^-24 (score, sum, quotient, scale) = 2^-20 relative.  Activations: exp and quotient within 2^-18 relative.
"""
import math

import pytest
import torch

import fp8_reference as ref

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module")
def handle(pkg):
    h = pkg.MoeBlock(64, 64, 8, max_rows=8)
    yield h
    h.synchronize()      # also reports a bounded wait that ran out
    h.close()


def kind(pkg, name):
    return {"f32": pkg.F32, "bf16": pkg.BF16, "f16": pkg.F16}[name]


def stream():
    return torch.cuda.current_stream().cuda_stream


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def half_step(out, name):
    return out.abs() * torch.finfo(TYPES[name]).eps / 2 + (2.0 ** -25 if name == "f16" else 0.0)


# ------------------------------------------------------------------------------------------------ routing
def run_route(pkg, handle, logits, bias, top_k, score, n_groups=1, top_groups=1, group_top=1, renorm=True, scale=1.0, dtype="f32"):
    rows, experts = logits.shape
    idx = torch.full((rows, top_k), -7, dtype=torch.int32, device="cuda")
    w = torch.full((rows, top_k), math.nan, device="cuda")
    rule = pkg.RouteRule(experts, top_k, pkg.SCORE_SIGMOID if score == "sigmoid" else pkg.SCORE_SOFTMAX, n_groups, top_groups,
                         group_top, int(renorm), scale)
    handle.route_scored(rule, logits.data_ptr(), kind(pkg, dtype), logits.stride(0), 0 if bias is None else bias.data_ptr(), rows,
                        idx.data_ptr(), w.data_ptr(), stream())
    return idx.cpu(), w.cpu()


def check_route(got, want):
    assert torch.equal(got[0], want[0])
    assert ((got[1].double() - want[1]).abs() <= want[1].abs() * 2.0 ** -20).all()


@pytest.mark.parametrize("rows,experts,top_k,groups,top_groups,group_top,score,dtype,bias,pad", [
    (40, 510, 8, 2, 1, 2, "sigmoid", "f32", True, 0),      # groups that are not whole lanes
    (40, 496, 6, 16, 5, 2, "softmax", "bf16", False, 0),
    (1, 128, 4, 1, 1, 1, "softmax", "f32", False, 0),
    (1, 256, 8, 8, 4, 2, "sigmoid", "f32", True, 0),
    (5, 1, 1, 1, 1, 1, "sigmoid", "f32", True, 0),
    (3, 7, 7, 7, 3, 1, "softmax", "f32", True, 1),
    (37, 32, 2, 4, 2, 2, "sigmoid", "bf16", True, 0),
    (33, 160, 6, 8, 3, 2, "softmax", "f16", True, 5),
    (64, 60, 4, 1, 1, 1, "sigmoid", "bf16", False, 4),
    (41, 384, 8, 8, 4, 2, "sigmoid", "f32", True, 8),
    (19, 512, 32, 32, 16, 2, "softmax", "bf16", True, 0),
    (129, 72, 8, 3, 1, 2, "sigmoid", "f16", True, 3),
    (300, 256, 8, 1, 1, 1, "softmax", "f32", True, 0),
])
@pytest.mark.parametrize("renorm,scale", [(True, 2.5), (False, 1.0)])
def test_route_matches_definition(rows, experts, top_k, groups, top_groups, group_top, score, dtype, bias, pad, renorm, scale, pkg, handle):
    g = gen(experts * 31 + rows)
    buf = (1.5 * randn(g, rows, experts + pad)).to(TYPES[dtype])
    logits, b = buf[:, :experts], 0.1 * randn(g, experts) if bias else None
    args = dict(top_k=top_k, score=score, n_groups=groups, top_groups=top_groups, group_top=group_top, renorm=renorm, scale=scale)
    check_route(run_route(pkg, handle, logits, b, dtype=dtype, **args), ref.route(logits, b, **args))


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups", [1, 4])
def test_route_masked_equal_and_extreme_logits(score, groups, pkg, handle):
    experts, top_k = 32, 6
    x = randn(gen(7), 16, experts)
    x[0] = -math.inf                                  # nothing left
    x[1, 3:] = -math.inf                              # fewer than top_k left
    x[2] = 0.25                                       # all equal: the lowest indices
    x[3, 1::2] = x[3, 0::2]                           # equal pairs
    x[4, 5], x[4, 9] = math.nan, math.nan             # NaN is off
    x[5, 30] = math.inf                               # counts as the largest finite value
    x[6, 30], x[6, 2] = math.inf, math.inf
    x[7] = torch.finfo(torch.float32).min             # a mask by the type's lowest value: on, scores 0 or equal
    x[8, :] = torch.finfo(torch.float32).min
    x[8, 17] = 0.0
    x[9] = 40.0 + torch.arange(experts, device="cuda") * 2.0 ** -10     # sigmoid next to 1
    x[10, 8:16] = -math.inf                           # a whole group off
    x[11, 8:15] = -math.inf                           # a group with one expert left
    b = 0.1 * randn(gen(8), experts)
    b[12], b[20] = -math.inf, math.nan                # off for every row
    args = dict(top_k=top_k, score=score, n_groups=groups, top_groups=max(1, groups // 2), group_top=2, renorm=True, scale=1.5)
    check_route(run_route(pkg, handle, x, b, **args), ref.route(x, b, **args))
    check_route(run_route(pkg, handle, x, None, **args), ref.route(x, None, **args))


def test_route_next_to_a_tie_is_decided_in_64_bits(pkg, handle):
    """Scores whose fp32 sums with the bias would be equal, or in the other order."""
    experts = 64
    x = torch.zeros(8, experts, device="cuda")
    b = torch.full((experts,), 0.5, device="cuda")
    for t in range(8):
        up = torch.tensor(-1.0 - 0.3 * t)
        for j in range(6):
            x[t, 60 - 7 * j] = float(up)
            up = torch.nextafter(up, torch.tensor(9.0))
    x[x == 0] = -9.0
    for score in ("sigmoid", "softmax"):
        args = dict(top_k=6, score=score)
        check_route(run_route(pkg, handle, x, b, **args), ref.route(x, b, **args))


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts,groups,group_top,top_k", [(256, 1, 1, 8), (256, 8, 2, 8), (64, 8, 1, 6), (512, 4, 2, 32), (30, 1, 1, 4)])
@pytest.mark.parametrize("bias", ["none", "zero", "steps"])
def test_route_values_a_few_steps_apart(score, experts, groups, group_top, top_k, bias, pkg, handle):
    """Rows of few levels, every value of a level some last places off, with exact ties among them.  Sums of two differ by the
    second order of a step, 4e-15 at the upper levels, ten last places of 64 bits; under a bias that few values share, sums of
    the same parts in another pairing would not, so every expert has its own there."""
    g = gen(experts + groups)
    levels = torch.tensor([-3.0, -0.5, 0.25, 1.0, 1.5, 2.0, 2.5], device="cuda")
    level = levels[torch.randint(0, 7, (400, experts), generator=g, device="cuda")]
    x = level * (1 + torch.randint(0, 40, (400, experts), generator=g, device="cuda") * 2.0 ** -23)
    b = {"none": None, "zero": torch.zeros(experts, device="cuda"),
         "steps": 0.125 + 2.0 ** -20 * (randn(g, experts) if group_top == 2 else torch.randint(0, 3, (experts,), generator=g, device="cuda"))}[bias]
    top_groups = max(1, groups // 2)
    got = run_route(pkg, handle, x, b, top_k, score, groups, top_groups, group_top)
    check_route(got, ref.route(x, b, top_k, score, groups, top_groups, group_top))


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,group_top", [(1, 1), (8, 1), (8, 2)])
@pytest.mark.parametrize("bias", ["none", "zero", "steps"])
def test_route_many_equal_scores(score, groups, group_top, bias, pkg, handle):
    """Logits of a coarse grid: equal scores, equal groups and, under a bias of the same grid, equal sums of different parts."""
    g = gen(11)
    x = (randn(g, 400, 64) * 4).round() / 4
    x[300:] *= 12                                     # sigmoids that 64 bits no longer tell apart
    b = None if bias == "none" else torch.zeros(64, device="cuda") if bias == "zero" else (randn(g, 64) * 4).round() / 16
    args = dict(top_k=8, score=score, n_groups=groups, top_groups=max(1, groups // 2), group_top=group_top)
    check_route(run_route(pkg, handle, x.bfloat16(), b, dtype="bf16", **args), ref.route(x.bfloat16(), b, **args))


def test_route_agrees_with_the_softmax_rule_of_the_block(pkg):
    """Without bias and groups and with renormalised softmax weights this is moe_route_topk's rule."""
    blk = pkg.MoeBlock(64, 64, 128, top_k=4, max_rows=8)
    try:
        x = randn(gen(3), 500, 128)
        idx, w = torch.empty(500, 4, dtype=torch.int32, device="cuda"), torch.empty(500, 4, device="cuda")
        blk.route_topk(x.data_ptr(), 500, idx.data_ptr(), w.data_ptr(), stream())
        got = run_route(pkg, blk, x, None, 4, "softmax")
        assert torch.equal(got[0], idx.cpu())
        assert ((got[1] - w.cpu()).abs() <= w.cpu() * 2.0 ** -20).all()
    finally:
        blk.close()


# ------------------------------------------------------------------------------------------------ grouping
def run_group(handle, idx, experts):
    rows, k = idx.shape
    offsets = torch.full((experts + 1,), -9, dtype=torch.int32, device="cuda")
    pair_row, row_pair = torch.full_like(idx, -9), torch.full((rows * k,), -9, dtype=torch.int32, device="cuda")
    handle.group_pairs(idx.data_ptr(), rows, k, experts, offsets.data_ptr(), pair_row.data_ptr(), row_pair.data_ptr(), stream())
    return offsets.cpu(), pair_row.cpu(), row_pair.cpu()


@pytest.mark.parametrize("rows,top_k,experts", [(1, 1, 1), (1, 4, 128), (2, 8, 256), (31, 1, 7), (33, 3, 60), (64, 4, 32), (257, 8, 512),
                                                (1000, 5, 1024), (4100, 8, 256), (20000, 3, 33)])
@pytest.mark.parametrize("spread", ["even", "one expert", "none", "with gaps"])
def test_group_matches_definition(rows, top_k, experts, spread, handle):
    g = gen(rows + experts)
    idx = torch.randint(0, experts, (rows, top_k), generator=g, device="cuda", dtype=torch.int32)
    if spread == "one expert":
        idx[:] = experts - 1
    elif spread == "none":
        idx[:] = -1
    elif spread == "with gaps":
        idx[::3, 0] = -1
        idx[1::4, -1] = experts + 5      # not an expert either
        idx[2::5, 0] = -2 ** 31
    for got, want in zip(run_group(handle, idx, experts), ref.group(idx, experts)):
        assert torch.equal(got, want)


def test_group_of_no_rows_and_without_row_pair(handle):
    offsets = torch.full((9,), 5, dtype=torch.int32, device="cuda")
    handle.group_pairs(0, 0, 4, 8, offsets.data_ptr(), 0, 0, stream())
    assert not offsets.any()
    idx = torch.tensor([[1, 0], [1, 7]], dtype=torch.int32, device="cuda")
    pair_row = torch.empty_like(idx)
    handle.group_pairs(idx.data_ptr(), 2, 2, 8, offsets.data_ptr(), pair_row.data_ptr(), 0, stream())
    assert pair_row.tolist() == [[1, 0], [2, 3]]


# ------------------------------------------------------------------------------------------------ quantiser
def run_quantise(pkg, handle, x, cols, act="none", dtype="f32", pair_row=None, out_rows=None, n_rows=None, ld_codes=None, ld_scales=None, shift=0):
    rows = x.shape[0]
    out_rows = rows if out_rows is None else out_rows
    ld_codes, ld_scales = ld_codes or cols, ld_scales or ref.blocks(cols)
    codes = torch.full((out_rows * ld_codes + shift,), 0x55, dtype=torch.uint8, device="cuda")
    scales = torch.full((out_rows, ld_scales), -5.0, device="cuda")
    a = {"none": pkg.ACT_NONE, "swiglu": pkg.ACT_SWIGLU, "silu": pkg.ACT_SILU_MUL}[act]
    handle.quantize_fp8(x.data_ptr(), kind(pkg, dtype), x.stride(0), rows, cols, codes.data_ptr() + shift, ld_codes, scales.data_ptr(), ld_scales,
                        act=a, pair_row_ptr=0 if pair_row is None else pair_row.data_ptr(), fanout=1 if pair_row is None else pair_row.shape[1],
                        out_rows=out_rows, n_rows_ptr=0 if n_rows is None else n_rows.data_ptr(), stream=stream())
    return codes[shift:].view(out_rows, ld_codes), scales


@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 128), (3, 127), (2, 129), (5, 2880), (17, 1000), (300, 264), (2, 7168)])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("pad,shift", [(0, 0), (8, 0), (3, 1)])
def test_quantise_rows_bit_for_bit(rows, cols, dtype, pad, shift, pkg, handle):
    x = (randn(gen(cols), rows, cols + pad) * torch.exp(2 * randn(gen(3), cols + pad))).clamp(-6e4, 6e4).to(TYPES[dtype])
    x[0, : max(1, cols // 2)] = 0
    codes, scales = run_quantise(pkg, handle, x, cols, dtype=dtype, ld_codes=cols + pad, ld_scales=ref.blocks(cols) + (pad > 0), shift=shift)
    want, want_s = ref.quantise_rows(x[:, :cols])
    assert torch.equal(codes[:, :cols].contiguous(), want.view(torch.uint8))
    assert torch.equal(scales[:, :ref.blocks(cols)], want_s)
    assert (codes[:, cols:] == 0x55).all() and (scales[:, ref.blocks(cols):] == -5).all()      # left as they were
    # against 64 bits: half a step of the code (its smallest step is 2^-9) and the roundings of the two quotients
    v = x[:, :cols].double()
    far = (codes[:, :cols].contiguous().view(torch.float8_e4m3fn).double() * scales.double()[:, torch.arange(cols) // 128] - v).abs()
    assert (far <= v.abs() * (2.0 ** -4 + 2.0 ** -21) + scales.double()[:, torch.arange(cols) // 128] * 2.0 ** -10).all()


@pytest.mark.parametrize("act", ["none", "swiglu", "silu"])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,cols,fanout", [(1, 128, 1), (3, 300, 2), (70, 1000, 6), (257, 2881, 4)])
def test_quantise_alignment_does_not_change_results(rows, cols, fanout, dtype, act, pkg, handle):
    """Rows of x at any element, codes in 16-byte rows or not: the same codes and scales, bit for bit."""
    wide = cols if act == "none" else 2 * cols
    g = gen(rows + cols)
    aligned = torch.zeros(rows, ref.pad16(wide), device="cuda", dtype=TYPES[dtype])
    aligned[:, :wide] = 4 * randn(g, rows, wide)
    odd = torch.zeros(rows * (wide + 3) + 1, device="cuda", dtype=TYPES[dtype])[1:].view(rows, wide + 3)
    odd[:, :wide] = aligned[:, :wide]
    place = torch.randperm(rows * fanout, generator=g, device="cuda").int().view(rows, fanout).contiguous()
    results = []
    for x in (aligned, odd):
        for ld, shift in ((ref.pad16(cols), 0), (ref.pad16(cols) + 3, 1)):
            codes, scales = run_quantise(pkg, handle, x, cols, act=act, dtype=dtype, pair_row=place, out_rows=rows * fanout, ld_codes=ld, shift=shift)
            assert (codes[:, cols:] == 0x55).all()
            results.append((codes[:, :cols], scales))
    for codes, scales in results[1:]:
        assert torch.equal(codes, results[0][0]) and torch.equal(scales, results[0][1])
    if act == "none":
        want, want_s = ref.quantise_rows(aligned[:, :cols])
        assert torch.equal(results[0][0][place.long().flatten()], want.view(torch.uint8).repeat_interleave(fanout, 0))
        assert torch.equal(results[0][1][place.long().flatten()], want_s.repeat_interleave(fanout, 0))


def test_quantise_extreme_values(pkg, handle):
    x = randn(gen(1), 8, 256)
    x[0] = 0
    x[1] = 1e-38                      # below the smallest maximum that counts
    x[2, 5] = torch.finfo(torch.float32).max
    x[3, 7], x[3, 9] = math.inf, -math.inf
    x[4, 11] = math.nan
    x[5] = math.nan
    x[6] = math.inf
    x[7] *= 2.0 ** -126
    codes, scales = run_quantise(pkg, handle, x, 256)
    want, want_s = ref.quantise_rows(torch.nan_to_num(x, nan=0.0, posinf=math.inf, neginf=-math.inf))
    want = want.view(torch.uint8).clone()
    want[x.isnan()] = 0x7f
    want[x == math.inf], want[x == -math.inf] = 0x7e, 0xfe
    assert torch.equal(codes & torch.where(x.isnan(), 0x7f, 0xff).to(torch.uint8), want)
    assert torch.equal(scales, want_s)


@pytest.mark.parametrize("rows,cols", [(1, 128), (7, 100), (30, 2880), (65, 345)])
@pytest.mark.parametrize("act", ["swiglu", "silu"])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_quantise_through_an_activation(rows, cols, act, dtype, pkg, handle):
    x = (4.0 * randn(gen(cols + 1), rows, 2 * cols)).to(TYPES[dtype])
    codes, scales = run_quantise(pkg, handle, x, cols, act=act, dtype=dtype)
    v = ref.activation(x, act)
    b = torch.nn.functional.pad(v.abs(), (0, ref.blocks(cols) * 128 - cols)).view(rows, -1, 128).amax(2).clamp_min(ref.AMAX_FLOOR)
    assert ((scales.double() - b / 448).abs() <= b / 448 * 2.0 ** -17).all()
    step = scales.double()[:, torch.arange(cols) // 128]
    far = (codes.contiguous().view(torch.float8_e4m3fn).double() * step - v).abs()
    assert (far <= v.abs() * (2.0 ** -4 + 2.0 ** -16) + step * 2.0 ** -10).all()


def test_quantise_activation_keeps_nan_and_saturates(pkg, handle):
    x = torch.zeros(2, 256, device="cuda")
    x[0, 0], x[0, 1] = math.nan, 1.0          # gate
    x[0, 2], x[0, 3] = 1.0, math.nan          # up
    x[0, 4], x[0, 5] = math.inf, math.inf     # both clamped
    x[0, 6], x[0, 7] = -1e4, 3.0              # sigmoid 0
    codes, _ = run_quantise(pkg, handle, x, 128, act="swiglu")
    c = codes[0].tolist()
    assert c[0] & 0x7f == 0x7f and c[1] & 0x7f == 0x7f and c[2] == 0x7e and c[3] & 0x7f == 0 and not any(codes[1].tolist())


@pytest.mark.parametrize("rows,cols,fanout", [(1, 2880, 4), (9, 200, 1), (40, 129, 8), (257, 2880, 2)])
def test_quantise_to_several_places(rows, cols, fanout, pkg, handle):
    """Every row arrives at each of its places; places outside the output are left out, other rows stay as they were."""
    out_rows = rows * fanout + 3
    g = gen(rows)
    pair_row = torch.randperm(out_rows, generator=g, device="cuda")[: rows * fanout].int().view(rows, fanout).contiguous()
    pair_row[0, 0], pair_row[-1, -1] = -1, out_rows
    x = randn(g, rows, cols).bfloat16()
    codes, scales = run_quantise(pkg, handle, x, cols, dtype="bf16", pair_row=pair_row, out_rows=out_rows)
    one, one_s = ref.quantise_rows(x)
    want, want_s = torch.full_like(codes, 0x55), torch.full_like(scales, -5.0)
    for t, places in enumerate(pair_row.tolist()):
        for r in places:
            if 0 <= r < out_rows:
                want[r], want_s[r] = one[t].view(torch.uint8), one_s[t]
    assert torch.equal(codes, want) and torch.equal(scales, want_s)


@pytest.mark.parametrize("n_rows", [-3, 0, 1, 11, 99])
def test_quantise_row_count_on_the_device(n_rows, pkg, handle):
    x = randn(gen(5), 20, 300)
    codes, scales = run_quantise(pkg, handle, x, 300, n_rows=torch.tensor([n_rows], dtype=torch.int32, device="cuda"))
    live = min(max(n_rows, 0), 20)
    want, want_s = ref.quantise_rows(x)
    assert torch.equal(codes[:live], want.view(torch.uint8)[:live]) and torch.equal(scales[:live], want_s[:live])
    assert (codes[live:] == 0x55).all() and (scales[live:] == -5).all()


@pytest.mark.parametrize("mats,rows,cols,pad", [(1, 1, 1, 0), (1, 128, 128, 0), (3, 130, 257, 0), (2, 300, 200, 8), (2, 127, 2880, 5), (1, 5760, 384, 0)])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_quantise_blocks_bit_for_bit(mats, rows, cols, pad, dtype, pkg, handle):
    w = (0.02 * randn(gen(rows), mats, rows, cols + pad)).to(TYPES[dtype])
    codes = torch.full((mats, rows, cols + pad), 0x55, dtype=torch.uint8, device="cuda")
    scales = torch.empty(mats, ref.blocks(rows), ref.blocks(cols), device="cuda")
    handle.quantize_fp8_blocks(w.data_ptr(), kind(pkg, dtype), cols + pad, mats, rows, cols, codes.data_ptr(), cols + pad, scales.data_ptr(), stream())
    want, want_s = ref.quantise_blocks(w[:, :, :cols])
    assert torch.equal(codes[:, :, :cols].contiguous(), want.view(torch.uint8)) and torch.equal(scales, want_s)
    assert (codes[:, :, cols:] == 0x55).all()


# ------------------------------------------------------------------------------------------------ product
def codes_of(g, scale, *shape):
    """Random e4m3 codes over the whole range, stored with rows padded to 16 bytes; what lies behind the columns is NaN."""
    k = shape[-1]
    full = torch.full((*shape[:-1], ref.pad16(k)), 0x7f, dtype=torch.uint8, device="cuda")
    full[..., :k] = (scale * randn(g, *shape)).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    return full


def make_product(seed, rows, n, k, groups=1, counts=None, bias=False):
    g = gen(seed)
    p = {"a": codes_of(g, 120.0, rows, k), "b": codes_of(g, 120.0, groups, n, k), "n": n, "k": k, "rows": rows, "groups": groups}
    p["sa"] = torch.exp(0.7 * randn(g, rows, ref.blocks(k))) / 100
    p["sb"] = torch.exp(0.7 * randn(g, groups, ref.blocks(n), ref.blocks(k))) / 1000
    p["bias"] = randn(g, groups, n).bfloat16() if bias else None
    p["offsets"] = None
    if counts is not None:
        p["offsets"] = torch.tensor([0] + list(torch.tensor(counts).cumsum(0)), dtype=torch.int32, device="cuda")
    return p


def run_product(pkg, handle, p, out="bf16", ld_out=None, st=None):
    ld_out = ld_out or p["n"]
    buf = torch.full((p["rows"], ld_out), 77.0, dtype=TYPES[out], device="cuda")
    handle.gemm_fp8(p["a"].data_ptr(), p["a"].shape[1], p["sa"].data_ptr(), p["sa"].shape[1], p["rows"], p["b"].data_ptr(), p["b"].shape[2],
                    p["sb"].data_ptr(), p["n"], p["k"], buf.data_ptr(), kind(pkg, out), ld_out, bias_ptr=0 if p["bias"] is None else p["bias"].data_ptr(),
                    n_groups=p["groups"], offsets_ptr=0 if p["offsets"] is None else p["offsets"].data_ptr(), stream=stream() if st is None else st)
    return buf


def check_product(p, buf, out):
    k, n = p["k"], p["n"]
    a, b = p["a"][:, :k].contiguous().view(torch.float8_e4m3fn), p["b"][:, :, :k].contiguous().view(torch.float8_e4m3fn)
    want, mag = ref.gemm(a, p["sa"], b, p["sb"], p["offsets"], p["bias"])
    covered = p["rows"] if p["offsets"] is None else int(p["offsets"][-1])
    got, want, mag = buf[:covered, :n].double(), want[:covered], mag[:covered]
    bound = half_step(want, out) + mag * (128 + ref.blocks(k)) * 2.0 ** -23
    far = (got - want).abs()
    assert (far <= bound).all(), (float((far / bound).max()), int((far > bound).sum()), far.numel())
    assert (buf[covered:] == 77).all() and (buf[:, n:] == 77).all()      # left as they were


DENSE = [(1, 1, 1), (1, 128, 128), (1, 4096, 512), (3, 5, 17), (16, 256, 7168), (17, 130, 1000), (33, 2880, 2880), (64, 512, 129),
         (100, 200, 300), (127, 129, 128), (128, 256, 256), (129, 257, 640), (256, 1024, 96), (300, 5760, 384), (513, 384, 2944), (1000, 136, 1040),
         (2049, 520, 272), (2500, 128, 200), (9, 300, 4100), (60, 130, 4096), (250, 100, 4300), (214, 225, 7912), (256, 1536, 14336), (300, 700, 2000)]


@pytest.mark.parametrize("rows,n,k", DENSE)
@pytest.mark.parametrize("out,bias", [("bf16", True), ("f32", False)])
def test_dense_product(rows, n, k, out, bias, pkg, handle):
    p = make_product(rows + n + k, rows, n, k, bias=bias)
    check_product(p, run_product(pkg, handle, p, out), out)


@pytest.mark.parametrize("pad", [0, 1, 2, 8])
@pytest.mark.parametrize("out", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("rows", [5, 40, 100, 200, 9000])
def test_product_output_types_and_strides(rows, out, pad, pkg, handle):
    p = make_product(pad, rows, 264, 400, bias=True)
    p["sa"] *= 0.01          # inside the range of fp16
    check_product(p, run_product(pkg, handle, p, out, ld_out=264 + pad), out)


GROUPED = [([1], 96, 200), ([0, 0, 5, 0], 300, 256), ([8] * 8, 384, 512), ([3, 0, 17, 1, 0, 64, 2, 9], 260, 1040), ([130, 1, 0, 127, 128, 129], 520, 384),
           ([700, 5, 0, 300, 33], 256, 640), ([0, 0, 0], 128, 128), ([1] * 40, 144, 2880), ([257, 255, 256, 0, 31, 32, 33], 1152, 128),
           ([16] * 200, 64, 64), ([1700, 5, 0, 2300, 33], 520, 384), ([1] * 1024, 130, 144), ([1900, 0, 300], 100, 256), ([9, 11], 300, 4200), ([0, 100, 90], 260, 5000)]


@pytest.mark.parametrize("counts,n,k", GROUPED)
@pytest.mark.parametrize("out,extra", [("bf16", 0), ("f32", 7)])
def test_grouped_product(counts, n, k, out, extra, pkg, handle):
    """Groups of any size, empty ones among them; `extra` rows behind the last group."""
    p = make_product(n + k, sum(counts) + extra, n, k, groups=len(counts), counts=counts, bias=extra == 0)
    if p["rows"] == 0:
        p["rows"] = 4
        p = {**p, "a": codes_of(gen(1), 1.0, 4, k), "sa": torch.ones(4, ref.blocks(k), device="cuda")}
    check_product(p, run_product(pkg, handle, p, out), out)


@pytest.mark.parametrize("rows,first", [(60, 7), (700, 130)])
def test_rows_before_the_first_group_stay(rows, first, pkg, handle):
    p = make_product(3, rows, 200, 260, groups=2, counts=[rows // 2 - first, rows // 2])
    p["offsets"] = p["offsets"] + first
    buf = run_product(pkg, handle, p, "f32")
    want, mag = ref.gemm(p["a"][:, :260].contiguous().view(torch.float8_e4m3fn), p["sa"], p["b"][:, :, :260].contiguous().view(torch.float8_e4m3fn), p["sb"],
                         p["offsets"])
    last = int(p["offsets"][-1])
    assert ((buf.double() - want).abs() <= half_step(want, "f32") + mag * 131 * 2.0 ** -23)[first:last].all()
    assert (buf[:first] == 77).all() and (buf[last:] == 77).all()


@pytest.mark.parametrize("rows,counts", [(20, None), (400, None), (200, [120, 0, 80])])
def test_nan_stays_in_its_row(rows, counts, pkg, handle):
    """A NaN code in a row of a, or a NaN or infinite scale, reaches that row's outputs and no others."""
    groups = len(counts) if counts else 1
    p = make_product(4, rows, 192, 300, groups=groups, counts=counts)
    clean = run_product(pkg, handle, p, "f32")
    bad = rows // 2
    p["a"][bad, 170] = 0x7f
    p["sa"][bad + 1, 1] = math.nan
    got = run_product(pkg, handle, p, "f32")
    assert got[bad:bad + 2].isnan().all()
    keep = torch.ones(rows, dtype=torch.bool, device="cuda")
    keep[bad:bad + 2] = False
    assert torch.equal(got[keep], clean[keep])


@pytest.mark.parametrize("rows", [8, 1500])
def test_product_is_the_same_every_time(rows, pkg, handle):
    p = make_product(2, rows, 1024, 3000, bias=True)
    first = run_product(pkg, handle, p, "f32")
    for _ in range(3):
        assert torch.equal(run_product(pkg, handle, p, "f32"), first)


def test_a_row_does_not_depend_on_its_batch_when_grouped(pkg, handle):
    """Rows of one group, and the same rows behind other groups (other tile borders): the same bits."""
    p = make_product(6, 90, 256, 512, groups=3, counts=[40, 7, 43])
    both = run_product(pkg, handle, p, "f32")
    lone = {**p, "a": p["a"][47:].contiguous(), "sa": p["sa"][47:].contiguous(), "b": p["b"][2:3].contiguous(), "sb": p["sb"][2:3].contiguous(),
            "rows": 43, "groups": 1, "offsets": torch.tensor([0, 43], dtype=torch.int32, device="cuda")}
    assert torch.equal(run_product(pkg, handle, lone, "f32"), both[47:])


def test_product_with_offsets_that_pass_32_bits(pkg, handle):
    """Weights of more than 2^32 bytes: the last group's product."""
    groups, n, k = 18, 16384, 16384
    p = {"n": n, "k": k, "rows": 5, "groups": groups, "bias": None}
    p["b"] = torch.empty(groups, n, k, dtype=torch.uint8, device="cuda")
    p["sb"] = torch.empty(groups, n // 128, k // 128, device="cuda")
    last = make_product(9, 5, n, k)
    p["b"][-1], p["sb"][-1], p["a"], p["sa"] = last["b"][0], last["sb"][0], last["a"], last["sa"]
    p["offsets"] = torch.tensor([0] * groups + [5], dtype=torch.int32, device="cuda")
    buf = run_product(pkg, handle, p, "f32")
    last["offsets"] = None
    check_product(last, buf, "f32")


# ------------------------------------------------------------------------------------------------ combine
@pytest.mark.parametrize("rows,top_k,cols,pad", [(1, 1, 1, 0), (1, 4, 2880, 0), (7, 3, 100, 3), (64, 8, 2880, 0), (130, 2, 2881, 7), (33, 32, 64, 8), (500, 4, 1024, 0)])
@pytest.mark.parametrize("y_type,out", [("bf16", "bf16"), ("f16", "bf16"), ("f32", "f32"), ("bf16", "f32"), ("f32", "f16"), ("f16", "f16")])
@pytest.mark.parametrize("residual", [False, True])
def test_combine(rows, top_k, cols, pad, y_type, out, residual, pkg, handle):
    g = gen(cols)
    n_y = rows * top_k
    y = torch.full((n_y, cols + pad), math.nan, device="cuda", dtype=TYPES[y_type])
    y[:, :cols] = randn(g, n_y, cols).to(TYPES[y_type])
    pair_row = torch.randperm(n_y, generator=g, device="cuda").int().view(rows, top_k)
    w = randn(g, rows, top_k)
    if rows > 3:
        pair_row[1, 0], pair_row[2, :], w[2, :], pair_row[3, -1] = -1, -1, math.nan, n_y      # a weight without a row counts for nothing
    res = randn(g, rows, cols + pad).to(TYPES[out]) if residual else None
    buf = torch.full((rows, cols + pad), 33.0, device="cuda", dtype=TYPES[out])
    handle.combine_pairs(y.data_ptr(), kind(pkg, y_type), cols + pad, n_y, pair_row.data_ptr(), w.data_ptr(), rows, top_k, cols, buf.data_ptr(),
                         kind(pkg, out), cols + pad, residual_ptr=0 if res is None else res.data_ptr(), ld_residual=cols + pad, stream=stream())
    w = torch.where((pair_row < 0) | (pair_row >= n_y), 0.0, w)
    want, mag = ref.combine(y[:, :cols], pair_row, w, None if res is None else res[:, :cols])
    assert ((buf[:, :cols].double() - want).abs() <= half_step(want, out) + mag * (top_k + 1) * 2.0 ** -24).all()
    assert (buf[:, cols:] == 33).all()


def test_combine_over_its_residual(pkg, handle):
    g = gen(2)
    y, x = randn(g, 60, 320).bfloat16(), randn(g, 20, 320).bfloat16()
    pair_row, w = torch.arange(60, device="cuda").int().view(20, 3), randn(g, 20, 3)
    apart = torch.empty_like(x)
    handle.combine_pairs(y.data_ptr(), pkg.BF16, 320, 60, pair_row.data_ptr(), w.data_ptr(), 20, 3, 320, apart.data_ptr(), pkg.BF16, 320,
                         residual_ptr=x.data_ptr(), ld_residual=320, stream=stream())
    handle.combine_pairs(y.data_ptr(), pkg.BF16, 320, 60, pair_row.data_ptr(), w.data_ptr(), 20, 3, 320, x.data_ptr(), pkg.BF16, 320,
                         residual_ptr=x.data_ptr(), ld_residual=320, stream=stream())
    assert torch.equal(x, apart)


# ------------------------------------------------------------------------------------------------ a layer of them
class Layer:
    """One FP8 expert layer: weights quantised by the library, buffers for up to `rows` tokens, the calls in order."""

    def __init__(self, pkg, handle, rows, hidden, inter, experts, top_k, seed=0):
        self.pkg, self.h, self.rows, self.H, self.D, self.E, self.K = pkg, handle, rows, hidden, inter, experts, top_k
        g = gen(seed)
        self.w1, self.s1 = self.quantised(0.05 * randn(g, experts, 2 * inter, hidden))
        self.w2, self.s2 = self.quantised(0.05 * randn(g, experts, hidden, inter))
        self.b1, self.b2 = 0.1 * randn(g, experts, 2 * inter), 0.1 * randn(g, experts, hidden)
        self.b1, self.b2 = self.b1.bfloat16(), self.b2.bfloat16()
        self.bias = 0.1 * randn(g, experts)
        self.rule = pkg.RouteRule(experts, top_k, pkg.SCORE_SIGMOID, n_groups=4, top_groups=2, group_top=2, renormalise=1, scale=1.5)
        P, dev = rows * top_k, dict(device="cuda")
        self.idx, self.wt = torch.empty(rows, top_k, dtype=torch.int32, **dev), torch.empty(rows, top_k, **dev)
        self.offsets, self.pair_row = torch.empty(experts + 1, dtype=torch.int32, **dev), torch.empty(rows, top_k, dtype=torch.int32, **dev)
        self.xq, self.xs = torch.zeros(P, ref.pad16(hidden), dtype=torch.uint8, **dev), torch.zeros(P, ref.blocks(hidden), **dev)
        self.h1 = torch.zeros(P, 2 * inter, dtype=torch.bfloat16, **dev)
        self.hq, self.hs = torch.zeros(P, ref.pad16(inter), dtype=torch.uint8, **dev), torch.zeros(P, ref.blocks(inter), **dev)
        self.y = torch.zeros(P, hidden, dtype=torch.bfloat16, **dev)

    def quantised(self, w):
        mats, rows, cols = w.shape
        codes = torch.zeros(mats, rows, ref.pad16(cols), dtype=torch.uint8, device="cuda")
        scales = torch.empty(mats, ref.blocks(rows), ref.blocks(cols), device="cuda")
        self.h.quantize_fp8_blocks(w.data_ptr(), self.pkg.F32, cols, mats, rows, cols, codes.data_ptr(), codes.shape[2], scales.data_ptr(), stream())
        torch.cuda.synchronize()
        return codes, scales

    def __call__(self, logits, x, out):
        """out = x + the layer's output for the rows x (bf16), with router logits fp32."""
        h, p, s = self.h, self.pkg, stream()
        T, P, H, D, E, K = self.rows, self.rows * self.K, self.H, self.D, self.E, self.K
        h.route_scored(self.rule, logits.data_ptr(), p.F32, E, self.bias.data_ptr(), T, self.idx.data_ptr(), self.wt.data_ptr(), s)
        h.group_pairs(self.idx.data_ptr(), T, K, E, self.offsets.data_ptr(), self.pair_row.data_ptr(), 0, s)
        h.quantize_fp8(x.data_ptr(), p.BF16, H, T, H, self.xq.data_ptr(), self.xq.shape[1], self.xs.data_ptr(), self.xs.shape[1],
                       pair_row_ptr=self.pair_row.data_ptr(), fanout=K, out_rows=P, stream=s)
        h.gemm_fp8(self.xq.data_ptr(), self.xq.shape[1], self.xs.data_ptr(), self.xs.shape[1], P, self.w1.data_ptr(), self.w1.shape[2],
                   self.s1.data_ptr(), 2 * D, H, self.h1.data_ptr(), p.BF16, 2 * D, bias_ptr=self.b1.data_ptr(), n_groups=E,
                   offsets_ptr=self.offsets.data_ptr(), stream=s)
        h.quantize_fp8(self.h1.data_ptr(), p.BF16, 2 * D, P, D, self.hq.data_ptr(), self.hq.shape[1], self.hs.data_ptr(), self.hs.shape[1],
                       act=p.ACT_SWIGLU, n_rows_ptr=self.offsets[E:].data_ptr(), stream=s)
        h.gemm_fp8(self.hq.data_ptr(), self.hq.shape[1], self.hs.data_ptr(), self.hs.shape[1], P, self.w2.data_ptr(), self.w2.shape[2],
                   self.s2.data_ptr(), H, D, self.y.data_ptr(), p.BF16, H, bias_ptr=self.b2.data_ptr(), n_groups=E,
                   offsets_ptr=self.offsets.data_ptr(), stream=s)
        h.combine_pairs(self.y.data_ptr(), p.BF16, H, P, self.pair_row.data_ptr(), self.wt.data_ptr(), T, K, H, out.data_ptr(), p.BF16, H,
                        residual_ptr=x.data_ptr(), ld_residual=H, stream=s)

    def inputs(self, seed):
        g = gen(seed)
        logits, x = randn(g, self.rows, self.E), randn(g, self.rows, self.H).bfloat16()
        if self.rows > 3:
            logits[1] = -math.inf          # a padding row: no expert
            logits[2, 1:] = -math.inf      # one expert only
        return logits, x

    def check(self, logits, x, out):
        """Every step against its definition on what the step before it left."""
        f8 = torch.float8_e4m3fn
        idx, w = ref.route(logits, self.bias, self.K, "sigmoid", 4, 2, 2, True, 1.5)
        check_route((self.idx.cpu(), self.wt.cpu()), (idx, w))
        offsets, pair_row, _ = ref.group(idx, self.E)
        assert torch.equal(self.offsets.cpu(), offsets) and torch.equal(self.pair_row.cpu(), pair_row)
        P, H, D = int(offsets[-1]), self.H, self.D
        codes, scales = ref.quantise_rows(x)
        at = self.pair_row.view(-1) >= 0
        token = torch.arange(self.rows, device="cuda").repeat_interleave(self.K)[at]
        place = self.pair_row.view(-1)[at].long()
        assert torch.equal(self.xq[place, :H], codes[token].view(torch.uint8)) and torch.equal(self.xs[place], scales[token])
        def product(a, s, b, sb, bias, got, n, k):
            p = {"a": a, "sa": s, "b": b, "sb": sb, "bias": bias, "offsets": self.offsets, "n": n, "k": k, "rows": len(a)}
            want, mag = ref.gemm(a[:, :k].contiguous().view(f8), s, b[:, :, :k].contiguous().view(f8), sb, self.offsets, bias)
            bound = half_step(want, "bf16") + mag * (128 + ref.blocks(k)) * 2.0 ** -23
            assert ((got.double() - want).abs() <= bound)[:P].all(), p["n"]
        product(self.xq, self.xs, self.w1, self.s1, self.b1, self.h1, 2 * D, H)
        v, step = ref.activation(self.h1[:P], "swiglu"), self.hs[:P].double()[:, torch.arange(D) // 128]
        far = (self.hq[:P, :D].contiguous().view(f8).double() * step - v).abs()
        assert (far <= v.abs() * (2.0 ** -4 + 2.0 ** -16) + step * 2.0 ** -10).all()
        product(self.hq, self.hs, self.w2, self.s2, self.b2, self.y, H, D)
        want, mag = ref.combine(self.y, self.pair_row, self.wt, x)
        assert ((out.double() - want).abs() <= half_step(want, "bf16") + mag * (self.K + 1) * 2.0 ** -24).all()


@pytest.mark.parametrize("rows,hidden,inter,experts,top_k", [(1, 256, 128, 16, 4), (5, 192, 96, 8, 2), (70, 288, 352, 32, 4), (600, 384, 200, 12, 3)])
def test_layer_of_operators(rows, hidden, inter, experts, top_k, pkg, handle):
    layer = Layer(pkg, handle, rows, hidden, inter, experts, top_k)
    logits, x = layer.inputs(1)
    out = torch.empty_like(x)
    layer(logits, x, out)
    layer.check(logits, x, out)


def test_layer_in_a_graph_beside_a_layer_on_another_stream(pkg, handle):
    """Captured once and replayed on new inputs, while the same handle runs another layer on a second stream."""
    a, b = Layer(pkg, handle, 130, 320, 160, 16, 4, seed=1), Layer(pkg, handle, 40, 256, 256, 8, 2, seed=2)
    inputs = [a.inputs(s) for s in (1, 2, 3)]
    logits, x = (t.clone() for t in inputs[0])
    out = torch.empty_like(x)
    want = []
    for l, r in inputs:
        o = torch.empty_like(r)
        a(l, r, o)
        want.append(o)
    lb, xb = b.inputs(9)
    ob, want_b = torch.empty_like(xb), torch.empty_like(xb)
    b(lb, xb, want_b)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a(logits, x, out)
    side = torch.cuda.Stream()
    for (l, r), o in zip(inputs, want):
        logits.copy_(l)
        x.copy_(r)
        with torch.cuda.stream(side):
            for _ in range(5):
                b(lb, xb, ob)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, o) and torch.equal(ob, want_b)


def test_first_calls_of_a_handle_are_captured_across_streams(pkg):
    """A handle whose first calls are made under capture, on two streams that fork and join."""
    h = pkg.MoeBlock(64, 64, 8, max_rows=8)
    try:
        small, large = make_product(1, 12, 260, 1024, bias=True), make_product(2, 300, 260, 1024, bias=True)
        idx = torch.randint(0, 40, (500, 4), generator=gen(5), device="cuda", dtype=torch.int32)
        offsets, pair_row, row_pair = torch.zeros(41, dtype=torch.int32, device="cuda"), torch.zeros_like(idx), torch.zeros(2000, dtype=torch.int32, device="cuda")
        outs = [torch.zeros(p["rows"], 260, device="cuda") for p in (small, large)]
        side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()

        def product(p, buf):
            h.gemm_fp8(p["a"].data_ptr(), p["a"].shape[1], p["sa"].data_ptr(), p["sa"].shape[1], p["rows"], p["b"].data_ptr(), p["b"].shape[2],
                       p["sb"].data_ptr(), p["n"], p["k"], buf.data_ptr(), pkg.F32, 260, bias_ptr=p["bias"].data_ptr(), stream=stream())
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            h.group_pairs(idx.data_ptr(), 500, 4, 40, offsets.data_ptr(), pair_row.data_ptr(), row_pair.data_ptr(), stream())
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                product(small, outs[0])
            product(large, outs[1])
            torch.cuda.current_stream().wait_stream(side)
            h.group_pairs(idx.data_ptr(), 500, 4, 40, offsets.data_ptr(), pair_row.data_ptr(), 0, stream())
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip((offsets, pair_row, row_pair), ref.group(idx, 40)):
            assert torch.equal(got.cpu(), want)
        for p, buf in zip((small, large), outs):
            check_product(p, buf, "f32")
        h.synchronize()
    finally:
        h.close()
