"""Routing by scores where 32 bits are not enough, against the definition in 64 bits (fp8_reference.py).

Tolerance of a weight, by arithmetic: scores that are normal numbers of 32 bits carry at most sixteen roundings of 2^-24 to the
weight (score, sum, quotient, scale) = 2^-20 relative; rows with smaller scores are formed in 64 bits and rounded once, which below
2^-126 is half of the smallest step, 2^-150.
"""
import math

import pytest
import torch

import fp8_reference as ref
from test_fp8_layer_gpu import TYPES, run_route

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def handle(pkg):
    h = pkg.MoeBlock(64, 64, 8, max_rows=8)
    yield h
    h.synchronize()
    h.close()


def check(pkg, handle, x, bias, dtype="f32", want_bias=None, **args):
    """x and the biases on the CPU; want_bias: what the biases count as."""
    x = x.to(TYPES[dtype])
    got = run_route(pkg, handle, x.cuda(), None if bias is None else bias.cuda(), dtype=dtype, **args)
    want = ref.route(x, bias if want_bias is None else want_bias, **args)
    assert torch.equal(got[0], want[0])
    far, bound = (got[1].double() - want[1]).abs(), want[1].abs() * 2.0 ** -20 + 2.0 ** -150
    assert (far <= bound).all(), float((far / bound).max())
    return want


# ------------------------------------------------------------------------------------------------ small scores
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("renorm,scale", [(True, 1.0), (False, 1.0), (False, 2.0 ** 100)])
@pytest.mark.parametrize("experts,groups", [(4, 1), (64, 1), (64, 8), (512, 4)])
def test_sigmoid_weights_of_low_logits(experts, groups, renorm, scale, bias, dtype, pkg, handle):
    """Every selected score is small: exp(-x) is near the largest of 32 bits, or past it."""
    g = torch.Generator().manual_seed(experts + groups)
    lows = torch.tensor([-60.0, -69.0, -80.0, -85.0, -87.0, -87.5, -88.5, -89.0, -90.0, -95.0, -100.0, -104.0, -110.0, -300.0, -600.0, -700.0])
    x = lows[:, None] - 0.5 * torch.argsort(torch.rand(len(lows), experts, generator=g), dim=1).clamp(max=8)
    b = 0.1 * torch.randn(experts, generator=g) if bias else None
    check(pkg, handle, x, b, dtype, top_k=4, score="sigmoid", n_groups=groups, top_groups=max(1, groups // 2), group_top=2, renorm=renorm, scale=scale)


def test_sigmoid_weights_of_the_smallest_rows(pkg, handle):
    want = check(pkg, handle, torch.tensor([[-90.0, -91.0, -92.0, -93.0], [-87.5, -88.5, -89.0, -90.0]]), None, top_k=4, score="sigmoid")
    assert (want[1].sum(1) - 1).abs().max() < 1e-12


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("renorm,scale", [(True, 2.5), (False, 1.0), (False, 2.0 ** 100)])
@pytest.mark.parametrize("experts,groups", [(32, 1), (256, 8), (512, 32)])
def test_softmax_weights_far_below_the_largest_logit(experts, groups, renorm, scale, dtype, pkg, handle):
    """A bias selects experts whose logits lie 30 to 600 below the row's largest."""
    g = torch.Generator().manual_seed(experts)
    below = torch.tensor([30.0, 50.0, 68.0, 70.0, 80.0, 86.0, 87.0, 88.0, 90.0, 100.0, 104.0, 110.0, 200.0, 400.0, 600.0])
    x = torch.randn(len(below), experts, generator=g)
    chosen = torch.argsort(torch.rand(experts, generator=g))[:6]
    b = 0.01 * torch.randn(experts, generator=g)
    b[chosen] = 3.0 + 0.25 * torch.arange(6)
    x[:, chosen] = 0.5 * torch.randn(len(below), 6, generator=g) - below[:, None]
    check(pkg, handle, x, b, dtype, top_k=4, score="softmax", n_groups=groups, top_groups=max(1, groups // 2), renorm=renorm, scale=scale)


def test_softmax_weights_below_a_largest_logit_whose_expert_is_off(pkg, handle):
    x = torch.tensor([[0.0, -120.0, -121.0, -122.0, -125.0, -300.0, -301.0, -302.0], [500.0, 1.0, 0.5, 0.25, 0.0, -1.0, -2.0, -3.0]])
    b = torch.zeros(8)
    b[0] = -math.inf
    for renorm in (True, False):
        check(pkg, handle, x, b, top_k=4, score="softmax", renorm=renorm)


# ------------------------------------------------------------------------------------------------ groups by sums of two
def opposite_signs(experts, groups, size_of_bias, rows=60):
    """Groups worth nearly the same: their two best have biases near +- size_of_bias, whose sums lie a few 1e-6 apart."""
    g = torch.Generator().manual_seed(experts + int(8 * size_of_bias))
    size = experts // groups
    b = torch.full((groups, size), -9.0 * size_of_bias)
    at = torch.argsort(torch.rand(groups, size, generator=g), dim=1)[:, :2]
    u, step = torch.rand(groups, 1, generator=g), 4e-6 * (torch.rand(groups, 1, generator=g) - 0.5)
    b.scatter_(1, at, torch.cat([size_of_bias + u, step - size_of_bias - u], 1))
    return 0.3 + 1e-5 * torch.randn(rows, experts, generator=g), b.view(-1)


@pytest.mark.parametrize("size_of_bias", [0.5, 4.0, 10.0, 100.0])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("experts,groups", [(32, 16), (256, 32), (512, 32)])      # 1, 8 and 16 experts a lane
@pytest.mark.parametrize("share", [1, 2])
def test_group_sums_of_opposite_signs(experts, groups, share, score, size_of_bias, pkg, handle):
    x, b = opposite_signs(experts, groups, size_of_bias)
    top_groups = 1 if share == 1 else groups // 2
    # rows whose order the last places of 64 bits would decide are not asked for
    s = torch.sigmoid(x.double()) if score == "sigmoid" else torch.softmax(x.double(), 1)
    worth = (s + b.double()).view(len(x), groups, -1).topk(2, dim=2).values.sum(2).sort(dim=1, descending=True).values
    x = x[worth[:, top_groups - 1] - worth[:, top_groups] > 1e-11]
    assert len(x) > 50
    check(pkg, handle, x, b, top_k=2, score=score, n_groups=groups, top_groups=top_groups, group_top=2)


def test_group_sums_whose_parts_lose_their_last_places(pkg, handle):
    """64 bits: group 1 is worth 0.210505247 + 1, group 0 0.210505009 + 1."""
    b = torch.full((512,), -9.0)
    b[0], b[1], b[16], b[17] = 2.9504035, -3.7398984, 2.4139395, -3.2034342
    want = check(pkg, handle, torch.zeros(1, 512), b, top_k=2, score="sigmoid", n_groups=32, top_groups=1, group_top=2)
    assert want[0].tolist() == [[16, 17]]


# ------------------------------------------------------------------------------------------------ biases that are not finite
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups", [1, 4])
@pytest.mark.parametrize("experts", [32, 60, 256])
@pytest.mark.parametrize("renorm", [False, True])
def test_an_expert_off_by_its_bias_still_counts_in_the_softmax(score, groups, experts, renorm, pkg, handle):
    """A bias decides the selection, not the weights: at -inf or NaN its expert is never selected, and the others' scores stay."""
    g = torch.Generator().manual_seed(experts)
    x, b = torch.randn(30, experts, generator=g), 0.1 * torch.randn(experts, generator=g)
    x[::5, 3::7] = -math.inf
    off = torch.zeros(experts, dtype=torch.bool)
    off[::3] = True
    b[::3], b[::6] = -math.inf, math.nan
    args = dict(top_k=6, score=score, n_groups=groups, top_groups=max(1, groups // 2), group_top=2, renorm=renorm)
    idx, w = check(pkg, handle, x, b, **args)
    assert not off[idx[idx >= 0].long()].any()
    if not renorm:
        s = torch.sigmoid(x.double()) if score == "sigmoid" else torch.softmax(x.double(), 1)
        found = idx >= 0
        assert torch.allclose(w[found], s.gather(1, idx.clamp(min=0).long())[found], rtol=1e-12, atol=0)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts,groups", [(32, 1), (32, 4), (60, 4), (256, 8)])
@pytest.mark.parametrize("group_top", [1, 2])
def test_an_infinite_bias_counts_as_the_largest_finite_one(score, experts, groups, group_top, pkg, handle):
    """Two of them in a group are worth more than one, and one is worth what the largest finite bias is."""
    g = torch.Generator().manual_seed(experts + group_top)
    x, b = torch.randn(20, experts, generator=g), 0.1 * torch.randn(experts, generator=g)
    size, most = experts // groups, torch.finfo(torch.float32).max
    b[1] = math.inf
    b[2 * size % experts + 2], b[2 * size % experts + 4] = math.inf, most
    b[-1] = most
    check(pkg, handle, x, b, want_bias=b.clamp(max=most), top_k=4, score=score, n_groups=groups, top_groups=1, group_top=group_top)


# ------------------------------------------------------------------------------------------------ the sum of a softmax
@pytest.mark.parametrize("experts", [128, 256, 512])
@pytest.mark.parametrize("bias", [False, True])
def test_weights_of_a_softmax_that_is_not_renormalised(experts, bias, pkg, handle):
    """One logit of 0 and all others at the same distance: roundings of their exponentials and of the sum would all go one way.
    Roundings of 2^-24: two of an exponential (one last place), once in the sum and once in the selected score, which takes one
    more; the sum, the quotient and the scaled weight, one each: eight."""
    d = torch.linspace(-16.0, -0.5, 20000, device="cuda")
    x = d[:, None].repeat(1, experts)
    x[:, 7] = 0
    b = torch.zeros(experts, device="cuda") if bias else None
    got = run_route(pkg, handle, x, b, 1, "softmax", renorm=False)
    want = (1 / torch.exp(x.double()).sum(1, keepdim=True)).cpu()
    assert (got[0] == 7).all()
    assert ((got[1].double() - want).abs() <= want * 8 * 2.0 ** -24).all()
