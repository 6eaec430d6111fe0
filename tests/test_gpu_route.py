"""Routing of tokens to experts against the definition in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def definition(z, k, bias=None, score="softmax", renormalize=True, scale=1.0, num_groups=1, topk_groups=1):
    """(weights, indices) in float64, differentiable in z (float64)."""
    T, E = z.shape
    dead = ~(z.detach() > -math.inf)
    if score == "softmax":
        m = z.detach().amax(dim=1, keepdim=True)
        p = torch.where(dead, torch.zeros_like(z), torch.exp(z - torch.where(m > -math.inf, m, torch.zeros_like(m))))
        total = p.sum(dim=1, keepdim=True)
        s = p / torch.where(total > 0, total, torch.ones_like(total))
    else:
        s = torch.where(dead, torch.zeros_like(z), torch.sigmoid(z))
    c = s.detach() + (0 if bias is None else bias.double())
    c = c.masked_fill(dead, -math.inf)
    order = c.clone() if bias is not None else z.detach().masked_fill(dead, -math.inf)
    if num_groups > 1:
        size = E // num_groups
        two = torch.sort(c.view(T, num_groups, size), dim=2, descending=True).values[:, :, :2]
        two = torch.where(two[:, :, :1] > -math.inf, two.clamp_min(-1e300), two)
        gs = torch.where(two <= -1e300, torch.zeros_like(two), two).sum(dim=2)
        gs = gs.masked_fill(two[:, :, 0] == -math.inf, -math.inf)
        best = torch.sort(gs, dim=1, descending=True, stable=True).indices[:, :topk_groups]
        keep = torch.zeros(T, num_groups, dtype=torch.bool, device=z.device).scatter_(1, best, True)
        keep = keep.repeat_interleave(size, dim=1)
        # eligible but masked experts stay ahead of experts of dropped groups
        order = torch.where(keep, order.clamp_min(-1e301), torch.full_like(order, -math.inf))
    idx = torch.sort(order, dim=1, descending=True, stable=True).indices[:, :k]
    w = torch.gather(s, 1, idx)
    if renormalize:
        total = w.sum(dim=1, keepdim=True)
        w = torch.where(total > 0, w / torch.where(total > 0, total, torch.ones_like(total)), torch.zeros_like(w))
    return w * scale, idx


def check(z, k, weight_tol=None, grad=True, **kw):
    from fusedswiglu_b200 import _lib, route

    leaf = z.detach().clone().requires_grad_(grad)
    w, idx = route(leaf, k, **kw)
    z64 = z.detach().double().requires_grad_(grad)
    w64, idx64 = definition(z64, k, **kw)
    assert w.dtype == torch.float32 and idx.dtype == torch.int32
    assert torch.equal(idx.long(), idx64)
    # a score: exp and the division 4 half steps, the row's sum of E terms held in a tree of
    # at most E/32 + 5, the rounded difference z - max up to |z - max| half steps of the result
    spread = 100.0
    tol = weight_tol or HALF[torch.float32] * (16 + z.shape[1] / 32 + spread)
    assert ((w.double() - w64).abs() <= tol * w64.abs() + 1e-37).all()
    if not grad:
        return w, idx
    dw = torch.randn(w.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    (got,) = torch.autograd.grad(w, [leaf], dw)
    (want,) = torch.autograd.grad(w64, [z64], dw.double())
    assert got.dtype == z.dtype and got.shape == z.shape
    # p (ds - sum p ds): the difference cancels, so errors count against |p| sum |ds|
    size = (w64.detach().abs() * dw.abs()).sum(dim=1, keepdim=True) + w64.detach().abs().amax(dim=1, keepdim=True) * dw.abs().amax(dim=1, keepdim=True)
    bound = HALF[z.dtype] * want.abs() + 4 * tol * size.double() + 2.0 ** -24
    assert ((got.double() - want).abs() <= bound).all()
    assert _lib.device_status() == 0
    return w, idx


def logits(T, E, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(T, E, device="cuda", generator=g) * 1.5).to(dtype)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("T,E,k,groups,topk_groups,dtype", [
    (1, 1, 1, 1, 1, torch.float32), (1, 64, 6, 1, 1, torch.bfloat16), (5, 33, 33 - 1, 1, 1, torch.float16),
    (129, 256, 8, 8, 4, torch.float32), (1000, 160, 6, 8, 3, torch.bfloat16), (77, 1024, 32, 32, 7, torch.float16),
    (64, 60, 4, 5, 2, torch.float32), (31, 8, 2, 8, 2, torch.bfloat16), (257, 96, 8, 3, 1, torch.bfloat16),
])
def test_selection_weights_and_gradients(T, E, k, groups, topk_groups, dtype, score, renormalize):
    z = logits(T, E, dtype, seed=T + E)
    check(z, k, score=score, renormalize=renormalize, scale=2.5, num_groups=groups, topk_groups=topk_groups)
    bias = (torch.randn(E, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)) * 8).round() * 1e-3
    check(z, k, bias=bias, score=score, renormalize=renormalize, num_groups=groups, topk_groups=topk_groups)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,topk_groups", [(1, 1), (4, 2)])
def test_scores_closer_than_fp32_are_ordered_as_in_64_bits(score, groups, topk_groups):
    """Experts whose scores agree to 1e-8: their fp32 sums with the bias round together."""
    T, E, k = 300, 64, 8
    g = torch.Generator(device="cuda").manual_seed(5)
    z = torch.full((T, E), 0.75, device="cuda") + torch.randint(-2, 3, (T, E), device="cuda", generator=g) * 2.0 ** -24
    z = z + (torch.randint(0, 3, (T, E), device="cuda", generator=g) == 0) * 0.5
    bias = torch.randint(0, 2, (E,), device="cuda", generator=g) * 0.25
    check(z, k, bias=bias, score=score, num_groups=groups, topk_groups=topk_groups)
    check(z, k, score=score, num_groups=groups, topk_groups=topk_groups)


@pytest.mark.parametrize("groups,topk_groups", [(1, 1), (8, 4)])
@pytest.mark.parametrize("with_bias", [False, True])
def test_equal_scores_go_to_the_lowest_index(groups, topk_groups, with_bias):
    from fusedswiglu_b200 import route

    z = torch.zeros(40, 64, device="cuda", dtype=torch.bfloat16)
    bias = torch.zeros(64, device="cuda") if with_bias else None
    w, idx = route(z, 6, bias=bias, num_groups=groups, topk_groups=topk_groups)
    assert torch.equal(idx, torch.arange(6, device="cuda", dtype=torch.int32).expand(40, 6))
    assert torch.equal(w, torch.full_like(w, 1 / 6)) or (w - 1 / 6).abs().max() < 1e-7


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("groups,topk_groups", [(1, 1), (4, 3)])
def test_masked_experts(score, renormalize, with_bias, groups, topk_groups):
    """-inf masks; rows with fewer open experts than k, and with none, get weight 0 there."""
    T, E, k = 200, 32, 6
    z = logits(T, E, torch.float32, seed=9)
    g = torch.Generator(device="cuda").manual_seed(10)
    open_ = torch.rand(T, E, device="cuda", generator=g) < torch.linspace(0, 1, T, device="cuda")[:, None]
    open_[:20] = False
    z = z.masked_fill(~open_, -math.inf)
    bias = torch.randn(E, device="cuda", generator=g) * 0.1 if with_bias else None
    w, idx = check(z, k, bias=bias, score=score, renormalize=renormalize, num_groups=groups, topk_groups=topk_groups)
    assert (w[:20] == 0).all()
    assert (torch.sort(idx, dim=1).values.diff(dim=1) > 0).all()
    masked = torch.gather(z, 1, idx.long()) == -math.inf
    assert (w[masked] == 0).all() and masked.any()


def test_lowest_finite_values_are_scores_not_masks():
    low = torch.finfo(torch.float32).min
    z = torch.full((3, 16), low, device="cuda")
    z[1, 3] = 0.0
    from fusedswiglu_b200 import route

    w, idx = route(z, 2)
    assert torch.equal(w[0], torch.tensor([0.5, 0.5], device="cuda")) and idx[0].tolist() == [0, 1]
    assert w[1].tolist() == [1.0, 0.0] and idx[1].tolist() == [3, 0]
    w, idx = route(z, 2, renormalize=False)
    assert (w[0] - 1 / 16).abs().max() < 1e-7 and w[1].tolist() == [1.0, 0.0]


def test_nan_and_inf_logits_keep_indices_valid():
    from fusedswiglu_b200 import route

    z = logits(64, 48, torch.float32, seed=3)
    z[0] = math.nan
    z[1, 5] = math.nan
    z[2, 7] = math.inf
    for kw in (dict(), dict(renormalize=False), dict(bias=torch.zeros(48, device="cuda")),
               dict(num_groups=4, topk_groups=2)):
        for score in ("softmax", "sigmoid"):
            w, idx = route(z, 5, score=score, **kw)
            assert ((idx >= 0) & (idx < 48)).all()
            assert (torch.sort(idx, dim=1).values.diff(dim=1) > 0).all()
            assert w[0].isnan().any() and not w[3:].isnan().any()
            if score == "softmax":
                assert w[:3].isnan().all()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_gradient_against_differences(score):
    z = logits(6, 24, torch.float32, seed=4)
    from fusedswiglu_b200 import route

    for renormalize in (True, False):
        leaf = z.clone().requires_grad_(True)
        w, idx = route(leaf, 3, score=score, renormalize=renormalize)
        dw = torch.randn(w.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
        (got,) = torch.autograd.grad(w, [leaf], dw)
        h = 1e-4
        for e in range(24):
            step = torch.zeros(24, dtype=torch.float64, device="cuda")
            step[e] = h

            def value(shift):
                zz = z.double() + shift
                s = torch.softmax(zz, dim=1) if score == "softmax" else torch.sigmoid(zz)
                v = torch.gather(s, 1, idx.long())
                v = v / v.sum(dim=1, keepdim=True) if renormalize else v
                return (v * dw).sum(dim=1)

            want = (value(step) - value(-step)) / (2 * h)
            # the difference quotient is off by h^2 times a third derivative of at most |dw| k
            assert ((got[:, e].double() - want).abs() < 1e-6).all()


def test_strided_rows_leading_axes_and_other_streams():
    from fusedswiglu_b200 import route

    wide = logits(40, 100, torch.bfloat16, seed=6)
    view = wide[:, 4:68]
    w, idx = route(view, 4)
    w2, idx2 = route(view.contiguous(), 4)
    assert torch.equal(w, w2) and torch.equal(idx, idx2)
    w3, idx3 = route(view.t().contiguous().t(), 4)
    assert torch.equal(w, w3) and torch.equal(idx, idx3)
    w4, idx4 = route(view.reshape(5, 8, 64), 4)
    assert w4.shape == (5, 8, 4) and torch.equal(idx4.view(40, 4), idx)
    e, i = route(view[:0], 4)
    assert e.shape == (0, 4) and i.shape == (0, 4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        w5, idx5 = route(view, 4)
    side.synchronize()
    assert torch.equal(w, w5) and torch.equal(idx, idx5)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w6, idx6 = route(view, 4)
    wide.copy_(wide.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(w6, w.flip(0)) and torch.equal(idx6, idx.flip(0))
