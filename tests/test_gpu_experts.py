"""Routed SwiGLU experts against the formulas in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

# half a step of each type, relative: what one rounding is off by at most
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def inputs(T, E, k, d, f, o, dtype, seed=0, spread=1.0, wdtype=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *s: torch.randn(*s, device="cuda", generator=g)
    x, dy = rn(T, d).to(dtype), rn(T, o).to(dtype)
    logits = rn(T, E) + spread * rn(E)
    top, idx = torch.topk(logits, k, dim=1)
    w = torch.softmax(top, dim=1).to(wdtype or dtype)
    wg, wu = (rn(E, d, f) / math.sqrt(d)).to(dtype), (rn(E, d, f) / math.sqrt(d)).to(dtype)
    wd = (rn(E, f, o) / math.sqrt(f)).to(dtype)
    return x, w, idx.to(torch.int32), wg, wu, wd, dy


def definition(x, w, idx, wg, wu, wd, dy=None):
    """y, or (y, dx, dw, dwg, dwu, dwd), in float64 by autograd of the formula."""
    leaves = [t.detach().double().requires_grad_(dy is not None) for t in (x, w, wg, wu, wd)]
    x, w, wg, wu, wd = leaves
    y = torch.zeros(x.shape[0], wd.shape[2], dtype=torch.float64, device="cuda")
    for e in range(wg.shape[0]):
        t, j = torch.nonzero(idx == e, as_tuple=True)
        if t.numel():
            h = torch.nn.functional.silu(x[t] @ wg[e]) * (x[t] @ wu[e])
            y = y.index_add(0, t, w[t, j][:, None] * (h @ wd[e]))
    if dy is None:
        return [y]
    return [y.detach(), *torch.autograd.grad(y, leaves, dy.double())]


def rel(a, b):
    n = torch.linalg.norm(b)
    d = torch.linalg.norm(a.double() - b)
    return (d / n).item() if n > 0 else d.item()


def run(x, w, idx, wg, wu, wd, dy=None):
    from fusedswiglu_b200 import FusedSwiGLUExperts, _lib

    if dy is None:
        out = [FusedSwiGLUExperts.apply(x, w, idx, wg, wu, wd)]
    else:
        leaves = [t.detach().requires_grad_(True) for t in (x, w, wg, wu, wd)]
        y = FusedSwiGLUExperts.apply(leaves[0], leaves[1], idx, *leaves[2:])
        out = [y.detach(), *torch.autograd.grad(y, leaves, dy)]
    torch.cuda.synchronize()
    assert _lib.device_status() == 0
    return out


# 16-bit roundings between an input and each output: y passes h and its own, dx passes dg, du and
# its own, a weight's gradient one operand and its own; 7 are allowed for.  Each moves a value by
# HALF of it at most and, evenly spread over a step, by less than half of that in the norm; they
# are independent: sqrt(7) * 0.5 HALF < 1.5 HALF.
NAMES = ("y", "dx", "dweights", "dw_gate", "dw_up", "dw_down")


def compare(got, want, dtype):
    for name, a, b in zip(NAMES, got, want):
        assert a.shape == b.shape
        assert rel(a, b) <= 1.5 * HALF[dtype], (name, rel(a, b))


SHAPES = [  # T, E, k, d, f, o
    (1, 8, 2, 64, 64, 64), (3, 64, 6, 136, 72, 200), (33, 4, 4, 256, 128, 256), (130, 5, 3, 72, 264, 8),
    (500, 60, 4, 264, 136, 264), (1500, 4, 2, 512, 384, 512), (2000, 2, 1, 256, 1032, 520), (64, 1, 1, 128, 128, 128),
    (700, 3, 2, 8, 8, 8), (600, 400, 3, 16, 24, 16), (2100, 352, 2, 16, 16, 16),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,E,k,d,f,o", SHAPES)
def test_forward(T, E, k, d, f, o, dtype):
    a = inputs(T, E, k, d, f, o, dtype, seed=T)[:6]
    compare(run(*a), definition(*a), dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,E,k,d,f,o", SHAPES)
def test_gradients(T, E, k, d, f, o, dtype):
    a = inputs(T, E, k, d, f, o, dtype, seed=T + 1, wdtype=torch.float32 if T % 2 else None)
    compare(run(*a), definition(*a), dtype)


def test_gradient_against_differences():
    """d<y, dy> along one direction of each input, of the 64-bit definition at the kernel's
    own inputs, against the kernel's gradients."""
    a = list(inputs(40, 4, 2, 64, 64, 64, torch.float16, seed=3, wdtype=torch.float32))
    got = run(*a)[1:]
    g = torch.Generator(device="cuda").manual_seed(9)
    for slot, grad in zip((0, 1, 3, 4, 5), got):
        v = torch.randn(a[slot].shape, device="cuda", generator=g).double()
        h = 1e-5

        def value(sign):
            b = [t.double() if t.is_floating_point() else t for t in a]
            b[slot] = b[slot] + sign * h * v
            return (definition(*b[:6])[0] * b[6]).sum()

        want = ((value(1) - value(-1)) / (2 * h)).item()
        have = (grad.double() * v).sum().item()
        size = torch.linalg.norm(grad.double()).item() * torch.linalg.norm(v).item()
        # a norm-wise error of 1.5 steps in the gradient moves the product by at most that of |grad| |v|
        assert abs(have - want) <= 1.5 * HALF[torch.float16] * size


def test_experts_without_rows_dropped_pairs_and_repeated_indices():
    x, w, idx, wg, wu, wd, dy = inputs(200, 12, 4, 128, 96, 128, torch.bfloat16, seed=5)
    idx = idx.clamp(max=5)                       # experts 6.. have no rows; repeats within a row
    idx[::7, 1] = -1
    idx[::5, 2] = 12
    idx[11] = -5                                 # a token without any expert
    a = (x, w, idx, wg, wu, wd, dy)
    got, want = run(*a), definition(*a)
    compare(got, want, torch.bfloat16)
    assert (got[0][11] == 0).all() and (got[1][11] == 0).all()
    for t in got[3:]:
        assert (t[6:] == 0).all()
    assert (got[2][(idx < 0) | (idx >= 12)] == 0).all()
    assert torch.equal(run(*a[:2], idx.long(), *a[3:])[0], got[0])


def test_all_pairs_dropped_and_no_tokens():
    x, w, idx, wg, wu, wd, dy = inputs(20, 4, 2, 64, 64, 64, torch.bfloat16, seed=6)
    for t in run(x, w, torch.full_like(idx, -1), wg, wu, wd, dy):
        assert (t == 0).all()
    got = run(x[:0], w[:0], idx[:0], wg, wu, wd, dy[:0])
    assert got[0].shape == (0, 64) and all((t == 0).all() for t in got)


@pytest.mark.parametrize("T", [9000, 300])
def test_all_tokens_to_one_expert(T):
    x, w, idx, wg, wu, wd, dy = inputs(T, 16, 2, 64, 72, 64, torch.bfloat16, seed=7)
    idx = torch.full_like(idx, 9)
    compare(run(x, w, idx, wg, wu, wd, dy), definition(x, w, idx, wg, wu, wd, dy), torch.bfloat16)


def test_inf_and_nan_of_one_expert_or_token_stay_there():
    x, w, idx, wg, wu, wd, dy = inputs(150, 6, 2, 136, 72, 64, torch.bfloat16, seed=8)
    clean = run(x, w, idx, wg, wu, wd, dy)
    wg2 = wg.clone()
    wg2[3, :, 5] = math.nan
    x2 = x.clone()
    x2[17] = math.inf
    got = run(x2, w, idx, wg2, wu, wd, dy)
    touched = (idx == 3).any(dim=1)
    touched[17] = True
    assert torch.equal(got[0][~touched], clean[0][~touched]) and torch.equal(got[1][~touched], clean[1][~touched])
    assert got[0][touched].isnan().any(dim=1).all()
    hit = torch.zeros(6, dtype=torch.bool, device="cuda")
    hit[3] = True
    hit[idx[17].long()] = True
    for a, b in zip(got[3:], clean[3:]):
        assert torch.equal(a[~hit], b[~hit])


def test_deterministic_strided_other_stream_and_graph():
    from fusedswiglu_b200 import FusedSwiGLUExperts

    a = inputs(700, 8, 2, 128, 136, 128, torch.bfloat16, seed=10)
    first = run(*a)
    for t, u in zip(first, run(*a)):
        assert torch.equal(t, u)
    x, w, idx, wg, wu, wd, dy = a
    strided = (x.t().contiguous().t(), w.t().contiguous().t(), idx.t().contiguous().t(),
               wg.transpose(1, 2).contiguous().transpose(1, 2), wu, wd, dy)
    for t, u in zip(first, run(*strided)):
        assert torch.equal(t, u)
    y3 = FusedSwiGLUExperts.apply(x.view(7, 100, 128), w.view(7, 100, 2), idx.view(7, 100, 2), wg, wu, wd)
    assert torch.equal(y3.view(700, 128), first[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = FusedSwiGLUExperts.apply(x, w, idx, wg, wu, wd)
    other = FusedSwiGLUExperts.apply(x.flip(0).contiguous(), w, idx, wg, wu, wd)
    side.synchronize()
    torch.cuda.synchronize()
    assert torch.equal(y, first[0])

    xs, ids = x.clone(), idx.clone()
    FusedSwiGLUExperts.apply(xs, w, ids, wg, wu, wd)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        yg = FusedSwiGLUExperts.apply(xs, w, ids, wg, wu, wd)
    xs.copy_(x.flip(0))
    ids.copy_(idx.roll(1, 0))          # another routing through the same graph
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(yg, FusedSwiGLUExperts.apply(xs, w, ids, wg, wu, wd))
    del other


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_moe_block_router_and_experts_together(score):
    """SwiGLUMoE: router logits, selection, experts and all gradients, as a user runs them."""
    from fusedswiglu_b200 import SwiGLUMoE, route

    torch.manual_seed(0)
    m = SwiGLUMoE(128, 96, 16, 3, score=score, num_groups=4, topk_groups=2, use_balance_bias=True, device="cuda")
    m.balance_bias.normal_(0, 0.05)
    x = torch.randn(2, 37, 128, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    dy = torch.randn(2, 37, 128, device="cuda", dtype=torch.bfloat16)
    y = m(x)
    y.backward(dy)
    # the same in 64 bits, with the block's own rounded logits and selection
    with torch.no_grad():
        from fusedswiglu_b200.experts import RouterLogits
        logits = RouterLogits.apply(x, m.w_router)
        _, idx = route(logits, 3, bias=m.balance_bias, score=score, num_groups=4, topk_groups=2)
    leaves = [t.detach().double().requires_grad_(True) for t in (x.view(74, 128), m.w_router, m.w_gate, m.w_up, m.w_down)]
    x64, wr, wg, wu, wd = leaves
    z = x64 @ wr
    s = torch.softmax(z, dim=1) if score == "softmax" else torch.sigmoid(z)
    w = torch.gather(s, 1, idx.view(74, 3).long())
    w = w / w.sum(dim=1, keepdim=True)
    out = torch.zeros(74, 128, dtype=torch.float64, device="cuda")
    for e in range(16):
        t, j = torch.nonzero(idx.view(74, 3) == e, as_tuple=True)
        if t.numel():
            h = torch.nn.functional.silu(x64[t] @ wg[e]) * (x64[t] @ wu[e])
            out = out.index_add(0, t, w[t, j][:, None] * (h @ wd[e]))
    want = torch.autograd.grad(out, leaves, dy.view(74, 128).double())
    assert rel(y.view(74, 128), out.detach()) < 2 * HALF[torch.bfloat16]
    got = [x.grad.view(74, 128), m.w_router.grad, m.w_gate.grad, m.w_up.grad, m.w_down.grad]
    for name, a, b in zip(("x", "router", "gate", "up", "down"), got, want):
        # the logits' rounding (half a step of values up to 3) moves a weight by that much too
        assert rel(a, b) < 3 * HALF[torch.bfloat16], (name, rel(a, b))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,E,k,d,f,o", [(1, 1, 1, 8, 8, 8), (1, 64, 32, 136, 72, 40), (4, 8, 8, 1032, 264, 520),
                                        (2, 3, 2, 4096, 136, 2056), (3, 16, 4, 520, 1408, 1024), (4, 6, 1, 256, 128, 264)])
def test_a_handful_of_tokens(T, E, k, d, f, o, dtype):
    """Inference on up to four tokens: fp32 and 16-bit weights, dropped pairs, repeated experts."""
    for wdtype in (torch.float32, dtype):
        x, w, idx, wg, wu, wd, _ = inputs(T, E, k, d, f, o, dtype, seed=T + k, wdtype=wdtype)
        compare(run(x, w, idx, wg, wu, wd), definition(x, w, idx, wg, wu, wd), dtype)
        idx[0, k // 2] = -1 if k > 1 else E
        idx[-1] = int(idx[-1, 0])
        wg[0, 0] = math.nan if k > 1 else 0.0
        keep = (idx != 0).all(dim=1)
        got, want = run(x, w, idx, wg, wu, wd), definition(x, w, idx, wg, wu, wd)
        compare([got[0][keep]], [want[0][keep]], dtype)


def test_the_number_of_tokens_does_not_change_a_token():
    """The same tokens alone and among others, through the forms for few and for many rows: apart
    by the roundings of the second, not by more."""
    x, w, idx, wg, wu, wd, _ = inputs(64, 8, 2, 256, 136, 256, torch.bfloat16, seed=20)
    many = run(x, w, idx, wg, wu, wd)[0]
    for T in (1, 3, 4, 5, 16):
        few = run(x[:T], w[:T], idx[:T], wg, wu, wd)[0]
        assert rel(few, many[:T].double()) < 3 * HALF[torch.bfloat16]
