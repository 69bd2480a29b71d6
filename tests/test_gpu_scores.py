"""Routing, the gradient for stored values and distillation against their definitions in 64 bits.

Tolerances count roundings.  u = 2^-24 is half a step of fp32 relative to the value; a result in a 16-bit type is off by half a step of that type
on top, or half its smallest step.
"""
import math

import numpy as np
import pytest
import torch

from csrspmm_b200 import ops, torch_library as TL

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
SMALLEST = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def _rounding(want, dtype):
    """Half a step of `dtype` at values of this size (nothing for fp32, whose roundings are counted with the others)."""
    return SMALLEST[dtype] + (0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2 * want.abs())


# ---- routing ------------------------------------------------------------------------------------------

def route_f64(x, k, bias=None, score="softmax", groups=1, top_groups=1, group_top=1, renormalize=True, scale=1.0, g=None):
    """(columns T x k, values, gradient of x or None, magnitude of what the gradient's terms cancel)"""
    x = x.detach().double()
    T, E = x.shape
    open_ = x > -math.inf
    s = torch.sigmoid(x) if score == "sigmoid" else torch.softmax(x.masked_fill(~open_.any(1, keepdim=True), 0.0), 1)
    s = s.masked_fill(~open_, 0.0)
    c = s if bias is None else s + bias.double()
    if bias is None:  # the order of s is the order of x, where s itself rounds to 0 or 1 too
        c = torch.where(open_, s, -math.inf)
        order = x
    else:
        c = order = c.masked_fill(~open_, -math.inf)
    inside = torch.ones_like(open_)
    if top_groups < groups:
        per = (order if group_top == 1 else c).view(T, groups, E // groups)
        best = per.topk(group_top, 2).values.sum(2)
        kept = torch.sort(best, dim=1, descending=True, stable=True).indices[:, :top_groups]
        inside = torch.zeros(T, groups, dtype=torch.bool, device=x.device).scatter_(1, kept, True).repeat_interleave(E // groups, 1)
    by_order = torch.sort(order, dim=1, descending=True, stable=True).indices
    behind = torch.sort((~inside).gather(1, by_order).to(torch.int8), dim=1, stable=True).indices
    cols = by_order.gather(1, behind)[:, :k].sort(1).values
    chosen = s.gather(1, cols)
    # s / sum s through logarithms, ln s = x - ln(sum of all) or -ln(1 + exp(-x)): the scores may all be below what 64 bits hold, their shares not
    there = x.gather(1, cols)
    log_s = torch.nn.functional.logsigmoid(there) if score == "sigmoid" else there
    p = torch.softmax(log_s.masked_fill(there == -math.inf, -math.inf), 1).nan_to_num(0.0)  # NaN: nothing available
    w = scale * (p if renormalize else chosen)
    if g is None:
        return cols, w, None, None
    g = g.double().view(T, k)
    dx, mag = torch.zeros_like(x), torch.zeros_like(x)
    if renormalize:
        slope = (1 - chosen) if score == "sigmoid" else 1.0
        dx.scatter_(1, cols, w * slope * (g - (p * g).sum(1, keepdim=True)))
        mag.scatter_(1, cols, (w * slope).abs() * (g.abs() + (p * g.abs()).sum(1, keepdim=True)))
    elif score == "sigmoid":
        dx.scatter_(1, cols, w * (1 - chosen) * g)
        mag = dx.abs()
    else:
        mean, mean_abs = (w * g).sum(1, keepdim=True), (w * g).abs().sum(1, keepdim=True)
        dx = s * (torch.zeros_like(x).scatter_(1, cols, scale * g) - mean)
        mag = s * (torch.zeros_like(x).scatter_(1, cols, abs(scale) * g.abs()) + mean_abs)
    return cols, w, dx, mag


def check_route(x, k, **how):
    T, E = x.shape
    g = torch.randn(T * k, device="cuda", generator=_gen(k))
    leaf = x.detach().requires_grad_(True)
    rp, ci, va = ops.route(leaf, k, **how)
    (dx,) = torch.autograd.grad(va, leaf, g)
    plain = ops.route(x.detach(), k, **how)
    assert all(torch.equal(a, b) for a, b in zip((rp, ci, va.detach()), plain))
    assert not plain[2].requires_grad and rp.dtype == ci.dtype == torch.int32
    cols, w, want, mag = route_f64(x, k, g=g, **how)
    assert torch.equal(rp.long(), torch.arange(0, T * k + 1, k, device="cuda"))
    assert torch.equal(ci.long().view(T, k), cols)
    # an exponential (2) of a rounded difference (at most 64 units, logits are within 32 of one another where it counts), a sum of 32
    # terms a lane and 5 steps, a division, a product: less than 128 roundings; the backward makes fewer of its own on top
    err = (va.detach().double().view(T, k) - w).abs()
    assert (err <= 128 * U * w.abs() + 1e-37).all(), float((err / (w.abs() + 1e-30)).max())
    assert dx.shape == x.shape and dx.dtype == x.dtype
    err = (dx.double() - want).abs()
    assert (err <= 256 * U * mag + _rounding(want, x.dtype)).all(), float((err - _rounding(want, x.dtype)).max())


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("T,E,k", [(1, 2, 1), (1, 64, 4), (7, 5, 5), (9, 60, 6), (64, 128, 8), (33, 129, 3), (17, 200, 32), (40, 256, 8), (11, 511, 16),
                                   (5, 1000, 7), (3, 1024, 32)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
def test_route(cuda_lib, dtype, T, E, k, score, renormalize):
    x = (3 * torch.randn(T, E, device="cuda", generator=_gen(T + E))).to(dtype)
    bias = 0.3 * torch.randn(E, device="cuda", generator=_gen(E))
    check_route(x, k, score=score, renormalize=renormalize, scale=2.5)
    check_route(x, k, score=score, renormalize=renormalize, bias=bias)


@pytest.mark.parametrize("E,groups,top_groups,group_top,k", [(64, 8, 4, 2, 8), (640, 10, 4, 1, 5), (752, 8, 2, 2, 8), (768, 8, 2, 2, 8), (769, 1, 1, 1, 8), (60, 4, 1, 2, 6), (60, 5, 2, 1, 3), (256, 8, 4, 2, 8), (256, 32, 3, 2, 8),
                                                             (96, 3, 2, 1, 16), (512, 16, 5, 2, 4), (1024, 4, 3, 2, 8), (32, 32, 7, 1, 7)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_route_with_groups(cuda_lib, E, groups, top_groups, group_top, k, score, with_bias, dtype):
    x = (2 * torch.randn(50, E, device="cuda", generator=_gen(E + k))).to(dtype)
    x[3] = -math.inf
    x[4, : E // 2] = -math.inf
    x[5, 1:] = -math.inf
    bias = 0.2 * torch.randn(E, device="cuda", generator=_gen(E)) if with_bias else None
    check_route(x, k, score=score, bias=bias, groups=groups, top_groups=top_groups, group_top=group_top)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,top_groups", [(1, 1), (8, 3)])
def test_route_makes_the_exact_choice_between_near_equals(cuda_lib, score, groups, top_groups):
    """Biases that bring every expert to the same sum but for their own rounding: fp32 sums cannot tell them apart."""
    x = torch.randn(200, 64, device="cuda", generator=_gen(1))
    s = torch.sigmoid(x.double()) if score == "sigmoid" else torch.softmax(x.double(), 1)
    for row in range(0, 200, 10):
        bias = (1.5 - s[row]).float()
        check_route(x[row : row + 1], 6, score=score, bias=bias, groups=groups, top_groups=top_groups, group_top=2 if groups > 1 else 1)


def test_route_takes_the_lower_index_of_equals(cuda_lib):
    x = torch.randint(-2, 3, (300, 96), device="cuda", generator=_gen(2)).float()
    for how in (dict(), dict(bias=torch.zeros(96, device="cuda")), dict(groups=8, top_groups=2, group_top=2),
                dict(groups=8, top_groups=2, group_top=1, bias=torch.zeros(96, device="cuda"))):
        for score in ("softmax", "sigmoid"):
            check_route(x, 8, score=score, **how)
    x = torch.zeros(4, 1024, device="cuda", dtype=torch.bfloat16)
    assert torch.equal(ops.route(x, 32)[1].view(4, 32), torch.arange(32, device="cuda", dtype=torch.int32).expand(4, 32))


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_route_of_masked_rows(cuda_lib, score, renormalize, dtype):
    x = torch.randn(8, 40, device="cuda", generator=_gen(3)).to(dtype)
    x[0] = -math.inf  # nothing available
    x[1, 3:] = -math.inf  # fewer than k
    x[2, ::2] = -math.inf
    x[3, :37] = torch.finfo(dtype).min  # the type's lowest is a number like others
    x[4, 5] = torch.finfo(dtype).max if score == "sigmoid" else 30.0
    bias = torch.randn(40, device="cuda", generator=_gen(4))
    for how in (dict(), dict(bias=bias)):
        check_route(x, 6, score=score, renormalize=renormalize, **how)
    rp, ci, va = ops.route(x, 6, score=score, renormalize=renormalize)
    assert (va[:6] == 0).all() and torch.equal(ci[:6], torch.arange(6, device="cuda", dtype=torch.int32))
    assert torch.equal(ci[6:12], torch.arange(6, device="cuda", dtype=torch.int32)) and (va[9:12] == 0).all() and (va[6:9] > 0).all()


def test_route_of_far_logits_keeps_their_shares(cuda_lib):
    """Scores that all round to zero or one, whose shares do not."""
    x = torch.tensor([[-200.0, -201.0, -203.0, -300.0], [200.0, 100.0, 50.0, -50.0]], device="cuda")
    for score in ("softmax", "sigmoid"):
        _, ci, va = ops.route(x, 2, score=score)
        assert ci.tolist() == [0, 1, 0, 1]
        e = math.e / (1 + math.e)
        want = [e, 1 - e, 0.5, 0.5] if score == "sigmoid" else [e, 1 - e, 1.0, math.exp(-100.0)]
        assert np.allclose(va.cpu().numpy(), want, rtol=128 * U, atol=1e-44)


def test_route_passes_nan_on(cuda_lib):
    for score, bad in (("softmax", math.nan), ("sigmoid", math.nan), ("softmax", math.inf)):
        for how in (dict(), dict(renormalize=False), dict(bias=torch.ones(24, device="cuda")), dict(groups=4, top_groups=2, group_top=2)):
            x = torch.randn(5, 24, device="cuda", generator=_gen(5))
            x[2, 7] = bad
            x[3] = bad
            leaf = x.clone().requires_grad_(True)
            rp, ci, va = ops.route(leaf, 4, score=score, **how)
            ci, va = ci.view(5, 4), va.view(5, 4)
            assert va[2:4].isnan().all() and not va[[0, 1, 4]].isnan().any()
            assert (ci >= 0).all() and (ci < 24).all() and (ci[:, 1:] > ci[:, :-1]).all()
            (dx,) = torch.autograd.grad(va.sum(), leaf)
            assert dx[2:4].isnan().all() and not dx[[0, 1, 4]].isnan().any()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_route_of_views(cuda_lib, dtype):
    base = torch.randn(40, 3 * 66, device="cuda", generator=_gen(6)).to(dtype)
    for x in (base[:, :64], base[:, 1:65], base[::2, 5:69], base.t()[:64, :40], base[:1, :64].expand(40, 64), base[7:8, 3:67]):
        check_route(x, 5, renormalize=False)
        check_route(x, 5, score="sigmoid", bias=torch.randn(200, device="cuda", generator=_gen(7))[: x.shape[1]].contiguous())


def test_route_gradients_of_broadcast_and_strided_kinds(cuda_lib):
    x = torch.randn(9, 48, device="cuda", generator=_gen(8), requires_grad=True)
    g = torch.randn(2 * 36, device="cuda", generator=_gen(9))[::2]
    va = ops.route(x, 4, score="sigmoid", renormalize=False)[2]
    one, = torch.autograd.grad(va.sum(), x, retain_graph=True)
    two, = torch.autograd.grad(va, x, torch.ones(36, device="cuda"), retain_graph=True)
    three, = torch.autograd.grad(va, x, g, retain_graph=True)
    four, = torch.autograd.grad(va, x, g.contiguous())
    assert torch.equal(one, two) and torch.equal(three, four)
    assert not torch.equal(one, three)


def test_route_gradient_against_differences(cuda_lib):
    """The definition in 64 bits is itself checked by differences: d(sum g w) along a direction, the choice unchanged."""
    x = torch.randn(6, 24, device="cuda", generator=_gen(10), dtype=torch.float64)
    g = torch.randn(6 * 4, device="cuda", generator=_gen(11))
    way = torch.randn(6, 24, device="cuda", generator=_gen(12), dtype=torch.float64)
    for score in ("softmax", "sigmoid"):
        for renormalize in (True, False):
            f = lambda h: (route_f64(x + h * way, 4, score=score, renormalize=renormalize)[1].flatten() * g.double()).sum()
            dx = route_f64(x, 4, score=score, renormalize=renormalize, g=g)[2]
            h = 1e-5
            assert abs(float((f(h) - f(-h)) / (2 * h) - (dx * way).sum())) < 1e-8


def test_route_of_nothing_and_refusals(cuda_lib):
    rp, ci, va = ops.route(torch.empty(0, 16, device="cuda"), 4)
    assert rp.tolist() == [0] and ci.numel() == va.numel() == 0
    x = torch.zeros(3, 16, device="cuda", requires_grad=True)
    dx, = torch.autograd.grad(ops.route(x[:0], 4)[2].sum(), x)
    assert (dx == 0).all()
    for k, how, message in ((0, {}, "k has"), (17, {}, "k has"), (4, dict(groups=3), "groups"), (4, dict(groups=4, top_groups=5), "top_groups"),
                            (5, dict(groups=4, top_groups=1), "k has"), (4, dict(groups=4, top_groups=2, group_top=3), "group_top"),
                            (4, dict(score="tanh"), "unknown score"), (4, dict(bias=torch.zeros(15, device="cuda")), "one entry per expert"),
                            (4, dict(bias=torch.zeros(16)), "bias"), (4, dict(bias=torch.zeros(16, device="cuda").half()), "bias"),
                            (4, dict(scale=math.inf), "scale")):
        with pytest.raises(RuntimeError, match=message):
            ops.route(x, k, **how)
        with pytest.raises(RuntimeError, match=message):
            ops.route(x.detach(), k, **how)
    with pytest.raises(RuntimeError, match="experts"):
        ops.route(torch.zeros(2, 1025, device="cuda"), 4)
    with pytest.raises(RuntimeError, match="float32, float16 or bfloat16"):
        ops.route(x.detach().double(), 4)
    with pytest.raises(RuntimeError, match="2-D"):
        ops.route(x.detach()[0], 4)
    va = ops.route(x, 4)[2]
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(va.sum(), x, create_graph=True)


# ---- the gradient for stored values ----------------------------------------------------------------------------

def _csr(M, Kd, lens, seed):
    lens = torch.as_tensor(lens, device="cuda")
    rp = torch.zeros(M + 1, dtype=torch.int32, device="cuda")
    rp[1:] = lens.cumsum(0)
    n = int(rp[-1])
    return rp, torch.randint(0, Kd, (n,), device="cuda", generator=_gen(seed), dtype=torch.int32), torch.randn(n, device="cuda", generator=_gen(seed + 1))


def _rows(rp):
    return torch.repeat_interleave(torch.arange(rp.numel() - 1, device="cuda"), (rp[1:] - rp[:-1]).long())


def check_sddmm(rp, ci, G, B, alpha=1.0):
    got = ops.sddmm(rp, ci, G, B, alpha)
    rows = _rows(rp)
    terms = G.double()[rows] * B.double()[ci.long()]
    # a lane sums at most an eighth of the columns in turn, and five steps join the lanes
    bound = (B.shape[1] / 8 + 16) * U * abs(alpha) * terms.abs().sum(1)
    assert got.dtype == torch.float32 and got.shape == ci.shape
    assert ((got.double() - alpha * terms.sum(1)).abs() <= bound).all()
    return got


@pytest.mark.parametrize("Nd", [1, 2, 3, 4, 7, 8, 16, 18, 31, 32, 33, 34, 50, 63, 64, 66, 90, 100, 128, 130, 200, 256, 258, 300, 512, 513, 514, 516, 1000, 2048])
def test_sddmm(cuda_lib, Nd):
    M, Kd = 150, 90
    lens = torch.randint(0, 9, (M,), generator=torch.Generator().manual_seed(Nd))
    lens[:5] = torch.tensor([0, 0, 1, 0, 700])
    lens[-3:] = 0
    rp, ci, _ = _csr(M, Kd, lens, Nd)
    G, B = torch.randn(M, Nd, device="cuda", generator=_gen(1)), torch.randn(Kd, Nd, device="cuda", generator=_gen(2))
    got = check_sddmm(rp, ci, G, B, -1.5)
    assert torch.equal(got, ops.sddmm(rp, ci, G, B, -1.5))  # the same bits again


@pytest.mark.parametrize("M,lens", [(1, [1]), (1, [5000]), (1, [40000]), (3000, [0] * 2999 + [1]), (3000, [1] + [0] * 2998 + [1]), (20000, [0, 3] * 10000),
                                    (40, [0] * 20 + [4000] + [0] * 19), (5, [0, 0, 0, 0, 2]), (100_000, [1] * 100_000)])
@pytest.mark.parametrize("Nd", [20, 128, 700])
def test_sddmm_of_uneven_rows(cuda_lib, M, lens, Nd):
    rp, ci, _ = _csr(M, 33, lens, 7)
    check_sddmm(rp, ci, torch.randn(M, Nd, device="cuda", generator=_gen(3)), torch.randn(33, Nd, device="cuda", generator=_gen(4)))


def test_sddmm_of_views_and_nothing(cuda_lib):
    rp, ci, _ = _csr(50, 40, [6] * 50, 9)
    wide = torch.randn(60, 300, device="cuda", generator=_gen(5))
    for G, B in ((wide[:50, :64], wide[10:50, 100:164]), (wide[:50, 1:65], wide[:40, 4:68]), (wide[:50, 2:66], wide[:40, 6:70]), (wide.t()[:50, :60], wide.t()[100:140, :60]),
                 (wide[:1, :64].expand(50, 64), wide[:40, :64]), (wide[::1][:50, :50], wide[20:60, :50])):
        check_sddmm(rp, ci, G, B)
    empty = torch.zeros(51, dtype=torch.int32, device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda")
    assert ops.sddmm(*empty, wide[:50], wide[:40]).numel() == 0
    assert (ops.sddmm(rp, ci, torch.empty(50, 0, device="cuda"), torch.empty(40, 0, device="cuda")) == 0).all()
    with pytest.raises(RuntimeError, match="same number of columns"):
        ops.sddmm(rp, ci, wide[:50, :64], wide[:40, :63])
    with pytest.raises(RuntimeError, match="row for each row"):
        ops.sddmm(rp, ci, wide[:49, :64], wide[:40, :64])
    with pytest.raises(RuntimeError, match="float32"):
        ops.sddmm(rp, ci, wide[:50].half(), wide[:40].half())
    with pytest.raises(RuntimeError, match="int32"):
        ops.sddmm(rp, ci.long(), wide[:50], wide[:40])


def test_sddmm_takes_the_nearest_column_inside(cuda_lib):
    rp, ci, _ = _csr(10, 8, [3] * 10, 11)
    ci[4], ci[7], ci[20] = 8, -1, 2 ** 31 - 1
    G, B = torch.randn(10, 24, device="cuda", generator=_gen(6)), torch.randn(8, 24, device="cuda", generator=_gen(7))
    assert torch.equal(ops.sddmm(rp, ci, G, B), ops.sddmm(rp, ci.clamp(0, 7), G, B))


@pytest.mark.parametrize("Nd", [5, 64, 130])
def test_weighted_spmm_and_its_gradients(cuda_lib, Nd):
    rp, ci, va = _csr(200, 120, torch.randint(0, 12, (200,), generator=torch.Generator().manual_seed(3)), 13)
    B = torch.randn(120, Nd, device="cuda", generator=_gen(8))
    W = torch.randn(200, Nd, device="cuda", generator=_gen(9))
    A = torch.zeros(200, 120, device="cuda", dtype=torch.float64).index_put_((_rows(rp), ci.long()), va.double(), accumulate=True)
    for for_values, for_B in ((True, True), (True, False), (False, True), (False, False)):
        v, b = va.clone().requires_grad_(for_values), B.clone().requires_grad_(for_B)
        C = ops.weighted_spmm(rp, ci, v, b, 0.75)
        assert torch.equal(C.detach(), torch.ops.csrspmm_b200.spmm(rp, ci, va, B, 0.75, "auto")) and C.requires_grad == (for_values or for_B)
        if not C.requires_grad:
            continue
        C.backward(W)
        if for_values:
            assert torch.equal(v.grad, ops.sddmm(rp, ci, W, B, 0.75))
            check_sddmm(rp, ci, W, B, 0.75)
        if for_B:
            assert torch.allclose(b.grad.double(), 0.75 * A.T @ W.double(), rtol=1e-4, atol=1e-4)
    v = va.clone().requires_grad_(True)
    s, = torch.autograd.grad(ops.weighted_spmm(rp, ci, v, B).sum(), v)  # a gradient that is one number for all
    assert torch.equal(s, ops.sddmm(rp, ci, torch.ones_like(W), B))
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(ops.weighted_spmm(rp, ci, v, B).sum(), v, create_graph=True)
    step = 2.0 ** -6  # along a direction the product is linear: the difference is the gradient but for rounding
    way = torch.randn(va.numel(), device="cuda", generator=_gen(10))
    f = lambda h: float((ops.weighted_spmm(rp, ci, va + h * way, B).double() * W.double()).sum())
    grad = ops.sddmm(rp, ci, W, B).double()
    assert abs((f(step) - f(-step)) / (2 * step) - float((grad * way.double()).sum())) <= 1e-3 * float((grad * way.double()).abs().sum())


@pytest.mark.parametrize("Nd", [1, 2, 6, 24, 130, 512, 515, 1024, 2050])
def test_small_product_with_the_transpose(cuda_lib, Nd):
    rp, ci, va = _csr(150, 70, torch.randint(0, 6, (150,), generator=torch.Generator().manual_seed(Nd)), 17)
    ci[3], ci[9] = 70, -4  # the nearest inside, as in a product
    wide = torch.randn(150, Nd + 3, device="cuda", generator=_gen(18))
    for G in (wide[:, :Nd], wide[:, 1 : Nd + 1], wide[:, :Nd].contiguous()):
        got = torch.ops.csrspmm_b200.spmm_transposed(rp, ci, va, G, 70, -0.5)
        terms = va.double()[:, None] * G.double()[_rows(rp)]
        index = ci.long().clamp(0, 69)
        want = torch.zeros(70, Nd, dtype=torch.float64, device="cuda").index_add(0, index, terms)
        most = int(torch.bincount(index).max())
        bound = (most + 1) * U * 0.5 * torch.zeros_like(want).index_add(0, index, terms.abs())  # a sum in turn and the factor
        assert got.shape == want.shape and ((got.double() + 0.5 * want).abs() <= bound + 1e-38).all()
        assert torch.equal(got, torch.ops.csrspmm_b200.spmm_transposed(rp, ci, va, G, 70, -0.5))
    none = torch.zeros(4, dtype=torch.int32, device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda"), torch.zeros(0, device="cuda")
    assert (torch.ops.csrspmm_b200.spmm_transposed(*none, wide[:3], 5, 1.0) == 0).all()
    assert torch.ops.csrspmm_b200.spmm_transposed(*none, wide[:3], 0, 1.0).shape == (0, Nd + 3)


def test_both_ways_to_the_gradient_of_b_agree(cuda_lib):
    from csrspmm_b200 import _lib
    pays = _lib.lib().csrspmm_b200_spmm_transposed_pays
    for M, Kd, Nd, mean in ((300, 200, 64, 4), (5000, 4000, 48, 9)):
        rp, ci, va = _csr(M, Kd, [mean] * M, 19)
        G = torch.randn(M, Nd, device="cuda", generator=_gen(20))
        assert bool(pays(Kd, Nd, ci.numel())) == (M == 300)
        got = torch.ops.csrspmm_b200.spmm_transposed(rp, ci, va, G, Kd, 1.5)
        t = TL.transpose_csr(rp, ci, va, Kd)
        assert torch.allclose(got, torch.ops.csrspmm_b200.spmm(*t, G, 1.5, "auto"), rtol=1e-4, atol=1e-4)
        B = torch.randn(Kd, Nd, device="cuda", generator=_gen(21), requires_grad=True)
        (dB,) = torch.autograd.grad(ops.weighted_spmm(rp, ci, va, B, 1.5), B, G)
        assert torch.equal(dB, got)


# ---- distillation ------------------------------------------------------------------------------------------------

def distill_f64(x, rp, ci, va, g, t=1.0, log_probs=False):
    """(loss, dx, and the magnitudes that their terms cancel) row by row, on the host"""
    X = x.detach().double().cpu()
    T, V = X.shape
    torch.set_num_threads(8)
    at, cols, vals = rp.cpu().long().tolist(), ci.cpu().long().clamp(0, max(V - 1, 0)), va.double().cpu()
    loss, dx = torch.zeros(T, dtype=torch.float64), torch.zeros(T, V, dtype=torch.float64)
    lmag, dmag = torch.zeros_like(loss), torch.zeros_like(dx)
    for r in range(T):
        c, v = cols[at[r] : at[r + 1]], vals[at[r] : at[r + 1]]
        if not log_probs and (len(c) == 0 or bool((v == -math.inf).all())):
            continue
        p = v.exp() if log_probs else torch.softmax(v / t, 0)
        if len(c) == 0 or bool((p == 0).all()):
            continue
        z = X[r] / t
        m = z.max()
        logq = torch.log_softmax(z, 0)
        on = p > 0
        loss[r] = t * t * (p[on] * (p[on].log() - logq[c[on]])).sum()
        near = (z[c[on]] - m).abs()
        lmag[r] = t * t * (p[on] * (1 + p[on].log().abs() + (v[on] / t).abs().max() + near + math.log(max(V, 2)))).sum()
        P = torch.zeros(V, dtype=torch.float64).index_add_(0, c, p)
        w = float(g[r]) * t
        dx[r] = w * (p.sum() * logq.exp() - P)
        dmag[r] = abs(w) * (p.sum() * logq.exp() * (1 + (z - m).abs().clamp_max(200)) + P)
    return loss, dx, lmag, dmag


def check_distill(x, rp, ci, va, t=1.0, log_probs=False):
    T, V = x.shape
    g = torch.rand(T, device="cuda", generator=_gen(V)) + 0.5
    want, want_dx, lmag, dmag = distill_f64(x, rp, ci, va, g.cpu(), t, log_probs)
    how = dict(temperature=t, log_probs=log_probs)
    leaf = x.detach().requires_grad_(True)
    loss = ops.distill_loss(leaf, rp, ci, va, **how)
    (dx,) = torch.autograd.grad(loss, leaf, g)
    loss2, dx2 = ops.distill_loss_grad(x.detach(), rp, ci, va, g, **how)
    plain = ops.distill_loss(x.detach(), rp, ci, va, **how)
    assert torch.equal(plain, loss.detach()) and loss.dtype == loss2.dtype == torch.float32 and dx.dtype == dx2.dtype == x.dtype
    # a thread sums at most V / 128 exponentials in turn and the parts meet in a dozen steps; an exponential is off by 4 and by twice its
    # argument (counted in the magnitudes), the entries' sums by their number at most
    most = int((rp[1:] - rp[:-1]).max()) if T else 0
    units = 64 + V / 128 + most
    for l, d in ((loss.detach(), dx), (loss2, dx2)):
        err = (l.cpu().double() - want).abs()
        assert (err <= units * U * lmag).all(), (float(err.max()), float((err / lmag.clamp_min(1e-30)).max() / U))
        err = (d.cpu().double() - want_dx).abs()
        room = units * U * dmag + _rounding(want_dx, x.dtype)
        # exponentials below 2^-126 are taken as zero
        room = room + g.abs().cpu().double()[:, None] * t * 2.0 ** -126
        assert (err <= room).all(), float((err - room).max())


def teacher(T, V, lens, seed, spread=3.0):
    lens = torch.as_tensor(lens)
    rng = np.random.default_rng(seed)
    cols = [rng.choice(V, size=int(n), replace=False) for n in lens]
    rp = torch.zeros(T + 1, dtype=torch.int32)
    rp[1:] = lens.cumsum(0)
    ci = torch.from_numpy(np.concatenate(cols) if T else np.zeros(0)).to(torch.int32)
    va = torch.from_numpy(rng.standard_normal(len(ci)) * spread).float()
    return rp.cuda(), ci.cuda(), va.cuda()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("T,V,k", [(1, 1, 1), (3, 7, 7), (5, 100, 8), (40, 1000, 3), (2, 4097, 64), (300, 513, 10), (9, 8192, 16), (7, 8195, 16), (2, 40001, 100),
                                   (1, 131072, 64), (1, 262145, 5), (3, 65536, 1000), (5000, 700, 4), (9000, 3000, 6), (2, 1_000_003, 9),
                                   (1500, 20000, 12)])
def test_distill(cuda_lib, dtype, T, V, k):
    x = (4 * torch.randn(T, V, device="cuda", generator=_gen(V + T))).to(dtype)
    check_distill(x, *teacher(T, V, [k] * T, V))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("t", [0.5, 1.0, 3.0])
@pytest.mark.parametrize("log_probs", [False, True])
def test_distill_of_ragged_rows(cuda_lib, dtype, t, log_probs):
    T, V = 60, 3001
    lens = torch.randint(0, 80, (T,), generator=torch.Generator().manual_seed(1))
    lens[[0, 5, 59]] = 0
    lens[7] = 1
    rp, ci, va = teacher(T, V, lens, 5)
    if log_probs:
        va = -va.abs() - 3.0
    x = (3 * torch.randn(T, V, device="cuda", generator=_gen(2))).to(dtype)
    check_distill(x, rp, ci, va, t, log_probs)


@pytest.mark.parametrize("log_probs", [False, True])
@pytest.mark.parametrize("V", [300, 20000, 150_000, 470_000])
def test_distill_of_masked_places(cuda_lib, log_probs, V):
    T = 9
    rp, ci, va = teacher(T, V, [6] * T, 8)
    if log_probs:
        va = -va.abs() - 0.5
    x = torch.randn(T, V, device="cuda", generator=_gen(3))
    hit = ci.long().view(T, 6)
    masked = torch.rand(T, V, device="cuda", generator=_gen(4)) < 0.3
    masked.scatter_(1, hit, False)
    x[0][masked[0]] = -math.inf
    x[1][masked[1]] = torch.finfo(torch.float32).min
    x[2] = torch.finfo(torch.float32).min  # all of them: a uniform row
    va[3 * 6 : 3 * 6 + 4] = -math.inf  # a teacher who rules some out
    va[4 * 6 : 5 * 6] = -math.inf  # or all: the row is left out
    x[4] = math.nan
    x[5] = x[5] * 1000.0
    keep = torch.ones(T, dtype=torch.bool)
    check_distill(x, rp, ci, va, 1.0, log_probs)
    # the student rules out what the teacher wants: an infinite loss, a finite gradient
    x[6, hit[6, 0]] = -math.inf
    x[7, 5] = math.nan
    x[8] = -math.inf
    loss, dx = ops.distill_loss_grad(x, rp, ci, va, 1.0, log_probs=log_probs)
    assert loss[6] == math.inf and dx[6].isfinite().all() and loss[7:].isnan().all() and dx[7:].isnan().all()
    assert loss[4] == 0 and (dx[4] == 0).all()
    assert keep.all() and loss[:6].isfinite().all() and dx[:6].isfinite().all()
    leaf = x.clone().requires_grad_(True)
    again = ops.distill_loss(leaf, rp, ci, va, log_probs=log_probs)
    again.sum().backward()
    assert torch.equal(again.detach().isnan(), loss.isnan()) and torch.equal(leaf.grad.isnan(), dx.isnan()) and (leaf.grad[4] == 0).all()


def test_distill_passes_a_teachers_nan_on(cuda_lib):
    rp, ci, va = teacher(4, 500, [3] * 4, 8)
    x = torch.randn(4, 500, device="cuda", generator=_gen(3))
    va[3:6] = math.nan
    va[7] = math.nan
    va[9] = math.inf
    for log_probs in (False, True):
        leaf = x.clone().requires_grad_(True)
        loss = ops.distill_loss(leaf, rp, ci, va, log_probs=log_probs)
        loss.sum().backward()
        loss2, dx2 = ops.distill_loss_grad(x, rp, ci, va, log_probs=log_probs)
        assert not loss[1:3].isfinite().any() and not loss2[1:3].isfinite().any() and loss[0].isfinite() and loss2[0].isfinite()
        assert leaf.grad[1:3].isnan().all() and dx2[1:3].isnan().all() and leaf.grad[0].isfinite().all() and dx2[0].isfinite().all()


def test_distill_counts_a_column_named_twice_with_both(cuda_lib):
    T, V = 6, 9001
    rp, ci, va = teacher(T, V, [40] * T, 9)
    c = ci.view(T, 40)
    c[0, 1] = c[0, 0]
    c[1, 20:30] = c[1, 3]
    c[2] = c[2, 0]
    c[3] = c[3].sort().values
    c[4] = c[4].sort().values
    c[4, 11] = c[4, 10]
    c[5, 0], c[5, 1] = -5, V + 3  # and one outside with the nearest inside
    x = torch.randn(T, V, device="cuda", generator=_gen(5))
    check_distill(x, rp, ci, va)
    a, b = ops.distill_loss_grad(x, rp, ci, va), ops.distill_loss_grad(x, rp, ci, va)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("V,k", [(1500, 300), (9001, 600), (60000, 300)])
def test_distill_of_many_entries_with_repeated_columns(cuda_lib, V, k):
    rp, ci, va = teacher(5, V, [k, 10, k, 0, 7], 21)
    ci[::3] = ci[1::3][: len(ci[::3])] if len(ci[1::3]) >= len(ci[::3]) else torch.cat([ci[1::3], ci[:1]])[: len(ci[::3])]
    check_distill(torch.randn(5, V, device="cuda", generator=_gen(22)), rp, ci, va)


@pytest.mark.parametrize("k", [3000, 9001])
def test_distill_from_a_dense_teacher(cuda_lib, k):
    rp, ci, va = teacher(2, 9001, [k, k], 10)
    x = torch.randn(2, 9001, device="cuda", generator=_gen(6)).bfloat16()
    check_distill(x, rp, ci, va)
    order = ci.view(2, k).sort(1)
    check_distill(x, rp, order.values.flatten().contiguous(), va.view(2, k).gather(1, order.indices).flatten().contiguous())


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_distill_of_views(cuda_lib, dtype):
    base = torch.randn(12, 5003, device="cuda", generator=_gen(7)).to(dtype)
    for x in (base[:, :4000], base[:, 1:4001], base[::3, 3:4100], base.t()[:4096, :12].t(), base[:1].expand(12, 5003), base[:, 7:8]):
        check_distill(x, *teacher(x.shape[0], x.shape[1], [min(5, x.shape[1])] * x.shape[0], 11))


def test_distill_weights_of_all_kinds(cuda_lib):
    rp, ci, va = teacher(8, 777, [5] * 8, 12)
    x = torch.randn(8, 777, device="cuda", generator=_gen(8))
    w = torch.rand(16, device="cuda", generator=_gen(9))
    one = ops.distill_loss_grad(x, rp, ci, va)[1]
    assert torch.equal(one, ops.distill_loss_grad(x, rp, ci, va, torch.ones(8, device="cuda"))[1])
    assert torch.equal(one, ops.distill_loss_grad(x, rp, ci, va, torch.ones(1, device="cuda").expand(8))[1])
    assert torch.equal(2 * one, ops.distill_loss_grad(x, rp, ci, va, 2.0)[1])
    assert torch.equal(ops.distill_loss_grad(x, rp, ci, va, w[::2])[1], ops.distill_loss_grad(x, rp, ci, va, w[::2].contiguous())[1])
    assert (ops.distill_loss_grad(x, rp, ci, va, 0.0)[1] == 0).all()
    leaf = x.clone().requires_grad_(True)
    loss = ops.distill_loss(leaf, rp, ci, va)
    one, = torch.autograd.grad(loss.sum(), leaf, retain_graph=True)
    two, = torch.autograd.grad(loss, leaf, torch.ones(8, device="cuda"))
    assert torch.equal(one, two)


def test_distill_gradient_against_differences(cuda_lib):
    """The definition in 64 bits against differences of itself, along a direction."""
    rp, ci, va = teacher(5, 60, [7, 0, 3, 1, 60], 13)
    x, way = (torch.randn(5, 60, dtype=torch.float64, generator=torch.Generator().manual_seed(s)) for s in (1, 2))
    g = torch.rand(5, dtype=torch.float64)
    for t, log_probs, v in ((1.0, False, va), (2.5, False, va), (2.5, True, -va.abs() - 2)):
        f = lambda h: (distill_f64(x + h * way, rp, ci, v, g, t, log_probs)[0] * g).sum()
        dx = distill_f64(x, rp, ci, v, g, t, log_probs)[1]
        h = 1e-5
        assert abs(float((f(h) - f(-h)) / (2 * h) - (dx * way).sum())) < 1e-8


def test_distill_of_nothing_and_refusals(cuda_lib):
    none = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda"), torch.zeros(0, device="cuda")
    loss, dx = ops.distill_loss_grad(torch.empty(0, 50, device="cuda"), *none)
    assert loss.shape == (0,) and dx.shape == (0, 50)
    rp = torch.zeros(5, dtype=torch.int32, device="cuda")
    x = torch.full((4, 50), math.nan, device="cuda", requires_grad=True)
    loss = ops.distill_loss(x, rp, *none[1:])
    loss.sum().backward()
    assert (loss == 0).all() and (x.grad == 0).all()  # rows without a teacher are left out, whatever they hold
    loss, dx = ops.distill_loss_grad(torch.empty(4, 0, device="cuda"), rp, *none[1:])
    assert (loss == 0).all() and dx.shape == (4, 0)
    x = torch.zeros(4, 50, device="cuda")
    rp, ci, va = teacher(4, 50, [2] * 4, 14)
    for args, how, message in (((x.double(), rp, ci, va), {}, "float32, float16 or bfloat16"), ((x[0], rp, ci, va), {}, "2-D"),
                               ((x, rp[:-1], ci, va), {}, "row_ptr must have"), ((x, rp.long(), ci, va), {}, "row_ptr"), ((x, rp, ci.long(), va), {}, "col_idx"),
                               ((x, rp, ci, va.double()), {}, "values"), ((x, rp, ci[:-1], va), {}, "differ in length"), ((x, rp, ci, va.cpu()), {}, "values"),
                               ((x, rp, ci, va), dict(temperature=0.0), "temperature"), ((x, rp, ci, va), dict(temperature=math.nan), "temperature"),
                               ((x, rp, ci[::2], va[::2]), {}, "contiguous")):
        with pytest.raises(RuntimeError, match=message):
            ops.distill_loss(*args, **how)
        with pytest.raises(RuntimeError, match=message):
            ops.distill_loss_grad(*args, 1.0, **how)
    for w in (torch.ones(3, device="cuda"), torch.ones(4), torch.ones(4, device="cuda").double(), torch.ones(4, 1, device="cuda")):
        with pytest.raises(RuntimeError, match="weights"):
            ops.distill_loss_grad(x, rp, ci, va, w)
    leaf = x.clone().requires_grad_(True)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(ops.distill_loss(leaf, rp, ci, va).sum(), leaf, create_graph=True)


# ---- all of them together ------------------------------------------------------------------------------------------

def _experts_step(x, scores, W, head, k, rp_t, ci_t, va_t):
    """A layer of experts between a router and a teacher: route, each expert's tokens by transposition, the answers combined by the routing
    matrix, logits, distillation."""
    T, H = x.shape
    E = W.shape[0]
    rp, ci, va = ops.route(scores, k, score="sigmoid")
    with torch.no_grad():
        by_expert, token, _ = TL.transpose_csr(rp, ci, va.detach(), E)
        expert = torch.repeat_interleave(torch.arange(E, device="cuda"), (by_expert[1:] - by_expert[:-1]).long())
        # the slot of entry e of the routing matrix: its place among the transposed entries
        slot = torch.empty(T * k, dtype=torch.int32, device="cuda")
        order = torch.sort(ci.long(), stable=True).indices
        slot[order] = torch.arange(T * k, device="cuda", dtype=torch.int32)
        assert torch.equal(torch.div(order, k, rounding_mode="floor"), token.long())
    answers = torch.bmm(x[token.long()].unsqueeze(1), W[expert]).squeeze(1)
    y = ops.weighted_spmm(rp, slot, va, answers)
    logits = y @ head
    return ops.distill_loss(logits, rp_t, ci_t, va_t)


def _experts_f64(x, scores, W, head, k, rp_t, ci_t, va_t):
    s = torch.sigmoid(scores)
    top = s.topk(k, 1)
    w = top.values / top.values.sum(1, keepdim=True)
    dense = torch.zeros_like(s).scatter(1, top.indices, w)
    y = torch.einsum("te,th,ehd->td", dense, x, W)
    logq = torch.log_softmax(y @ head, 1)
    rows = _rows(rp_t)
    p = torch.cat([torch.softmax(v, 0) for v in torch.split(va_t.double(), (rp_t[1:] - rp_t[:-1]).tolist())])
    return torch.zeros(len(x), dtype=torch.float64, device="cuda").index_add(0, rows, p * (p.log() - logq[rows, ci_t.long()]))


def test_a_layer_of_experts_learns_from_a_teacher(cuda_lib):
    torch.backends.cuda.matmul.allow_tf32 = False
    T, H, E, V, k = 50, 32, 12, 1000, 3
    new = lambda *s: torch.randn(*s, device="cuda", generator=_gen(sum(s)), dtype=torch.float64) / math.sqrt(s[-1])
    x, scores, W, head = new(T, H), 4 * new(T, E), new(E, H, H), 8 * new(H, V)
    rp, ci, va = teacher(T, V, [6] * T, 20)
    leaves = [v.float().requires_grad_(True) for v in (x, scores, W, head)]
    loss = _experts_step(*leaves, k, rp, ci, va)
    loss.mean().backward()
    wide = [v.detach().double().requires_grad_(True) for v in leaves]
    want = _experts_f64(*wide, k, rp, ci, va)
    want.mean().backward()
    # fp32 through four products of at most 1000 terms
    assert torch.allclose(loss.double(), want, rtol=1e-4, atol=1e-4)
    for got, ref in zip(leaves, wide):
        assert torch.allclose(got.grad.double(), ref.grad, rtol=1e-3, atol=1e-4 * float(ref.grad.abs().max()))


def test_on_another_stream_and_replayed_from_a_graph(cuda_lib):
    T, E, V, k = 64, 64, 5001, 4
    scores, logits = torch.randn(T, E, device="cuda", generator=_gen(30)), torch.randn(T, V, device="cuda", generator=_gen(31)).bfloat16()
    rp_t, ci_t, va_t = teacher(T, V, [9] * T, 21)
    answers = torch.randn(T * k, 48, device="cuda", generator=_gen(32))
    slots = torch.randperm(T * k, device="cuda", generator=_gen(33)).int()
    g_route, g_loss = torch.randn(T, 48, device="cuda", generator=_gen(34)), torch.rand(T, device="cuda", generator=_gen(35))

    def step(scores, logits, answers):
        rp, ci, va = ops.route(scores, k)
        y = ops.weighted_spmm(rp, slots, va, answers)
        loss = ops.distill_loss(logits, rp_t, ci_t, va_t)
        dx, da = torch.autograd.grad(y, (scores, answers), g_route)
        (dl,) = torch.autograd.grad(loss, logits, g_loss)
        both = ops.distill_loss_grad(logits.detach(), rp_t, ci_t, va_t, g_loss)
        return [ci, va.detach(), y.detach(), loss.detach(), dx, da, dl, *both]

    new = lambda: [v.clone().requires_grad_(True) for v in (scores, logits, answers)]
    eager = new()
    want = step(*eager)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(*eager)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # (an eager graph of the same leaves that lives through a capture of their backward pass invalidates it, for any operator of torch's too)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(*eager)
    for seed in (1, 2):
        with torch.no_grad():
            for v in eager:
                v.copy_(torch.randn(v.shape, device="cuda", generator=_gen(seed)))
        graph.replay()
        torch.cuda.synchronize()
        want = step(*[v.detach().clone().requires_grad_(True) for v in eager])
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_padding_behind_rows_is_left_alone(cuda_lib):
    """The C ABI writes rows of the given width and nothing behind them, at any alignment."""
    import ctypes as C
    from csrspmm_b200 import _lib
    L = _lib.lib()
    for dtype, kind in ((torch.float32, 0), (torch.bfloat16, 2)):
        for T, V, k in ((3, 37, 4), (5, 1001, 8), (4, 9003, 8), (2, 70001, 8), (3, 5, 2)):
            x = torch.randn(T, V, device="cuda", generator=_gen(V)).to(dtype)
            rp, ci, va = teacher(T, V, [k] * T, 40)
            loss, stats, w = torch.empty(T, device="cuda"), torch.empty(4 * T, device="cuda"), torch.ones(T, device="cuda")
            a = _lib.DistillArgs(C.sizeof(_lib.DistillArgs), T, V, kind, x.data_ptr(), V, ci.numel(), rp.data_ptr(), ci.data_ptr(), va.data_ptr(), 1.0, 0)
            want = ops.distill_loss_grad(x, rp, ci, va)[1]
            for pad in (1, 3, 8):
                out = torch.full((T + 1, V + pad), 7.0, device="cuda", dtype=dtype)
                assert L.csrspmm_b200_distill_grad(C.byref(a), w.data_ptr(), 1, loss.data_ptr(), out[0, 1:].data_ptr(), V + pad, None) == 0
                flat = out.flatten()[1 : 1 + T * (V + pad)].view(T, V + pad)
                assert torch.equal(flat[:, :V], want) and (flat[:, V:] == 7).all() and out[0, 0] == 7
                out.fill_(7.0)
                assert L.csrspmm_b200_distill(C.byref(a), loss.data_ptr(), stats.data_ptr(), None) == 0
                assert L.csrspmm_b200_distill_backward(C.byref(a), stats.data_ptr(), w.data_ptr(), 1, out.data_ptr(), V + pad, None) == 0
                assert torch.allclose(out[:T, :V].float(), want.float(), rtol=2.0 ** -7, atol=1e-6) and (out[:T, V:] == 7).all() and (out[T] == 7).all()
        x = torch.randn(9, 60, device="cuda", generator=_gen(1)).to(dtype)
        rp, ci, va = ops.route(x, 5)
        r = _lib.RouteArgs(struct_size=C.sizeof(_lib.RouteArgs), T=9, E=60, k=5, scores=x.data_ptr(), ld=60, score_type=kind, score=0, groups=1, top_groups=1,
                           group_top=1, renormalize=1, scale=1.0)
        out = torch.full((10, 63), 7.0, device="cuda", dtype=dtype)
        g = torch.randn(45, device="cuda", generator=_gen(2))
        assert L.csrspmm_b200_route_backward(C.byref(r), ci.data_ptr(), va.data_ptr(), g.data_ptr(), 1, out.data_ptr(), 63, None) == 0
        want = torch.ops.csrspmm_b200.route_backward(g, x, ci, va, 5, "softmax", True, 1.0)
        assert torch.equal(out[:9, :60], want) and (out[:9, 60:] == 7).all() and (out[9] == 7).all()
        guard = torch.full((60,), 7, dtype=torch.int32, device="cuda")
        values = torch.full((60,), 7.0, device="cuda")
        offsets = torch.full((20,), 7, dtype=torch.int32, device="cuda")
        assert L.csrspmm_b200_route(C.byref(r), offsets.data_ptr(), guard.data_ptr(), values.data_ptr(), None) == 0
        assert torch.equal(offsets[:10], rp) and (offsets[10:] == 7).all()
        assert torch.equal(guard[:45], ci) and (guard[45:] == 7).all() and torch.equal(values[:45], va) and (values[45:] == 7).all()
    out = torch.full((40,), 7.0, device="cuda")
    rp, ci, _ = _csr(10, 8, [3] * 10, 11)
    G, B = torch.randn(10, 24, device="cuda", generator=_gen(6)), torch.randn(8, 24, device="cuda", generator=_gen(7))
    assert L.csrspmm_b200_sddmm(10, 8, 24, 30, rp.data_ptr(), ci.data_ptr(), G.data_ptr(), 24, B.data_ptr(), 24, 1.0, out.data_ptr(), None) == 0
    assert torch.equal(out[:30], ops.sddmm(rp, ci, G, B)) and (out[30:] == 7).all()


def test_more_elements_than_32_bits_count(cuda_lib):
    """Rows that begin beyond 2^31 elements, in each operator."""
    T, V = 16_500, 131_100
    x = torch.zeros(T, V, device="cuda", dtype=torch.bfloat16)
    last = torch.arange(T - 3, T, device="cuda")
    x[-3:] = torch.randn(3, V, device="cuda", generator=_gen(70)).bfloat16()
    lens = torch.zeros(T, dtype=torch.long)
    lens[-3:] = 20
    rp, ci, va = teacher(T, V, lens, 71)
    g = torch.ones(T, device="cuda")
    loss, dx = ops.distill_loss_grad(x, rp, ci, va, g)
    leaf = x.requires_grad_(True)
    again = ops.distill_loss(leaf, rp, ci, va)
    (dx2,) = torch.autograd.grad(again, leaf, g)
    small = teacher(3, V, [20] * 3, 71)  # the same entries
    want = ops.distill_loss_grad(x.detach()[last], *small)
    assert torch.equal(small[1], ci) and torch.equal(small[2], va)
    assert torch.equal(loss[-3:], want[0]) and torch.equal(again.detach()[-3:], want[0]) and (loss[:-3] == 0).all()
    assert torch.equal(dx[-3:], want[1]) and torch.allclose(dx2[-3:].float(), want[1].float(), rtol=2.0 ** -7, atol=1e-7)
    assert not dx[:100].any() and not dx2[T - 100 : T - 3].any()
    del x, leaf, dx, dx2, again
    T, E = 8_400_000, 256
    x = torch.zeros(T, E, device="cuda", dtype=torch.bfloat16)
    x[-2:] = torch.randn(2, E, device="cuda", generator=_gen(72)).bfloat16()
    x.requires_grad_(True)
    rp, ci, va = ops.route(x, 4, score="sigmoid", renormalize=False)
    (dx,) = torch.autograd.grad(va.sum(), x)
    few = x.detach()[-2:].clone().requires_grad_(True)
    want = ops.route(few, 4, score="sigmoid", renormalize=False)
    (want_dx,) = torch.autograd.grad(want[2].sum(), few)
    assert torch.equal(ci[-8:], want[1]) and torch.equal(va[-8:], want[2]) and torch.equal(dx[-2:], want_dx) and int(rp[-1]) == 4 * T
    assert torch.equal(ci[:4], torch.arange(4, device="cuda", dtype=torch.int32))
    del x, dx, va
    Kd, Nd = (1 << 22) + 7, 513
    B = torch.empty(Kd, Nd, device="cuda").normal_(generator=_gen(73))
    G = torch.randn(5, Nd, device="cuda", generator=_gen(74))
    rp = torch.tensor([0, 2, 2, 5, 6, 8], dtype=torch.int32, device="cuda")
    ci = torch.tensor([Kd - 1, 0, Kd - 2, Kd - 3, 5, Kd - 1, 4_190_000, Kd - 1], dtype=torch.int32, device="cuda")
    check_sddmm(rp, ci, G, B)


def test_two_threads_at_once(cuda_lib):
    import threading
    x = torch.randn(500, 64, device="cuda", generator=_gen(50))
    logits = torch.randn(40, 20001, device="cuda", generator=_gen(51))
    rp, ci, va = teacher(40, 20001, [9] * 40, 52)
    want = [*ops.route(x, 6, score="sigmoid", bias=x[0].contiguous()), *ops.distill_loss_grad(logits, rp, ci, va)]
    torch.cuda.synchronize()
    found = []

    def work():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                leaf = logits.detach().requires_grad_(True)
                got = [*ops.route(x, 6, score="sigmoid", bias=x[0].contiguous()), *ops.distill_loss_grad(logits, rp, ci, va)]
                ops.distill_loss(leaf, rp, ci, va).sum().backward()
                torch.cuda.current_stream().synchronize()
                found.append(all(torch.equal(a, b) for a, b in zip(got, want)) and torch.allclose(leaf.grad, want[4], rtol=1e-5, atol=1e-8))

    threads = [threading.Thread(target=work) for _ in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert len(found) == 80 and all(found)


def test_what_was_saved_and_then_changed_is_refused(cuda_lib):
    x = torch.randn(6, 32, device="cuda", generator=_gen(60))
    leaf = x.clone().requires_grad_(True)
    h = leaf * 1.0
    va = ops.route(h, 4, renormalize=False)[2]
    with torch.no_grad():
        h.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        va.sum().backward()
    rp, ci, t = teacher(6, 32, [3] * 6, 61)
    h = leaf * 1.0
    loss = ops.distill_loss(h, rp, ci, t)
    with torch.no_grad():
        t.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.sum().backward()
    with torch.inference_mode():
        assert not ops.route(leaf, 4)[2].requires_grad and not ops.distill_loss(leaf, rp, ci, t).requires_grad
    with torch.no_grad():
        assert not ops.route(leaf, 4)[2].requires_grad and not ops.weighted_spmm(rp, ci, t.requires_grad_(True), torch.randn(32, 5, device="cuda")).requires_grad


def test_registration(cuda_lib):
    O = torch.ops.csrspmm_b200
    how = dict(test_utils=("test_schema", "test_faketensor", "test_autograd_registration"))
    x = torch.randn(6, 16, device="cuda")
    rp, ci, va = O.route(x, 4, None, "softmax", 1, 1, 1, True, 1.0)
    for leaf in (x, x.clone().requires_grad_(True)):
        torch.library.opcheck(O.route, (leaf, 4, None, "sigmoid", 4, 2, 1, True, 1.0), **how)
        torch.library.opcheck(O.distill_loss, (leaf, rp, ci, va, 2.0, False), **how)
        torch.library.opcheck(O.weighted_spmm, (rp, ci, va, torch.randn(16, 5, device="cuda", requires_grad=leaf.requires_grad), 1.0), **how)
    torch.library.opcheck(O.sddmm, (rp, ci, torch.randn(6, 5, device="cuda"), torch.randn(16, 5, device="cuda"), 1.0), **how)
    torch.library.opcheck(O.spmm_transposed, (rp, ci, va, torch.randn(6, 5, device="cuda"), 16, 1.0), **how)
    torch.library.opcheck(O.route_backward, (va, x, ci, va, 4, "softmax", False, 1.0), **how)
    torch.library.opcheck(O.distill_loss_grad, (x, rp, ci, va, torch.ones(6, device="cuda"), 1.0, False), **how)
    loss, stats = O.distill_with_stats(x, rp, ci, va, 1.0, False)
    torch.library.opcheck(O.distill_backward, (loss, x, rp, ci, va, stats, 1.0, False), **how)


def test_the_operators_and_their_gradients_trace(cuda_lib):
    O = torch.ops.csrspmm_b200
    x, B = (torch.randn(*shape, device="cuda", generator=_gen(80), requires_grad=True) for shape in ((16, 64), (64, 24)))
    slots = torch.randperm(64, device="cuda", generator=_gen(81)).int()
    rp_t, ci_t, va_t = teacher(16, 24, [4] * 16, 82)

    def loss(x, B):
        rp, ci, va = O.route(x, 4, None, "sigmoid", 1, 1, 1, True, 1.0)
        return O.distill_loss(O.weighted_spmm(rp, slots, va, B, 1.0), rp_t, ci_t, va_t, 1.0, False).mean()

    want = torch.autograd.grad(loss(x, B), (x, B))
    got = torch.autograd.grad(torch.compile(loss, backend="aot_eager", fullgraph=True)(x, B), (x, B))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
