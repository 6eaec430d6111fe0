"""Routed experts and 8-bit products under odd circumstances: a wait that runs out, two streams
at once, one captured graph beside another, layers in a row, and the serving form of a block."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def weights(E, d, f, dtype=torch.bfloat16, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *s: torch.randn(*s, device="cuda", generator=g)
    return ((rn(E, d, f) / math.sqrt(d)).to(dtype), (rn(E, d, f) / math.sqrt(d)).to(dtype),
            (rn(E, f, d) / math.sqrt(f)).to(dtype))


def tokens(T, E, k, d, dtype=torch.bfloat16, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(T, d, device="cuda", generator=g).to(dtype)
    top, idx = torch.topk(torch.randn(T, E, device="cuda", generator=g), k, dim=1)
    return x, torch.softmax(top, dim=1), idx.to(torch.int32)


def calls():
    """(name, call) of every kind of kernel with waits, at sizes that take each of its forms."""
    from fusedswiglu_b200 import FusedSwiGLUExperts, fp8_linear, fp8_quantize_weight, fp8_swiglu_experts, fp8_swiglu_mlp

    E, d, f = 4, 256, 256
    wg, wu, wd = weights(E, d, f)
    q = [t for w in (wg, wu, wd) for t in fp8_quantize_weight(w)]
    first = [t[0] for t in q]
    out = []
    for T, k in ((40, 2), (700, 2)):
        x, w, i = tokens(T, E, k, d)
        out.append((f"experts {T}", lambda x=x, w=w, i=i: FusedSwiGLUExperts.apply(x, w, i, wg, wu, wd)))
        out.append((f"fp8 experts {T}", lambda x=x, w=w, i=i: fp8_swiglu_experts(x, w, i, *q)))
    for T in (3, 300, 5000):
        x = tokens(T, E, 1, d)[0]
        out.append((f"fp8 linear {T}", lambda x=x: fp8_linear(x, first[0], first[1])))
        out.append((f"fp8 mlp {T}", lambda x=x: fp8_swiglu_mlp(x, *first)))
    long = fp8_quantize_weight(weights(1, 4096, 256, seed=3)[0][0])
    x = torch.randn(2, 4096, device="cuda", dtype=torch.bfloat16)
    out.append(("fp8 linear, divided", lambda: fp8_linear(x, *long)))
    return out


def test_waits_that_run_out_end_and_are_reported():
    """The loads are held back, as the library's test hook does: every kernel gives up by itself,
    says so in the status word, and the next calls are right again."""
    from fusedswiglu_b200 import _lib

    cases = calls()
    want = [c() for _, c in cases]
    assert _lib.device_status() == 0
    old = _lib.get_option("wait_limit_ms")
    _lib.set_option("wait_limit_ms", 50)
    _lib.set_option("stall_producer", 1)
    try:
        for name, c in cases:
            c()
            torch.cuda.synchronize()
            assert _lib.load().fsw_status() != 0, name
            assert "bounded wait" in _lib.last_error()
    finally:
        _lib.set_option("stall_producer", 0)
        _lib.set_option("wait_limit_ms", old)
    assert _lib.device_status() == 0
    for (name, c), w in zip(cases, want):
        assert torch.equal(c(), w), name
    assert _lib.device_status() == 0


def test_two_streams_at_once_and_two_graphs():
    cases = calls()
    want = [c() for _, c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        for order, s, g in zip((cases, cases[::-1]), streams, got):
            with torch.cuda.stream(s):
                g.append([c() for _, c in order])
    torch.cuda.synchronize()
    for r in got[0]:
        assert all(torch.equal(a, b) for a, b in zip(r, want))
    for r in got[1]:
        assert all(torch.equal(a, b) for a, b in zip(r[::-1], want))
    graphs, outs = [], []
    for part in (cases[:5], cases[5:]):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append([c() for _, c in part])
        graphs.append(g)
    for s, g in zip(streams, graphs):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for _ in range(3):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs[0] + outs[1], want))


def test_training_step_captured_in_a_graph():
    """Router, experts and all gradients of one step, replayed with other tokens."""
    from fusedswiglu_b200 import FusedSwiGLUExperts, route

    T, E, k, d, f = 300, 8, 2, 128, 136
    wg, wu, wd = weights(E, d, f)
    wr = torch.randn(d, E, device="cuda", dtype=torch.bfloat16) / math.sqrt(d)
    x, _, _ = tokens(T, E, k, d)
    dy = torch.randn(T, d, device="cuda", dtype=torch.bfloat16)
    fixed = x.clone()

    def step(inp):
        leaves = [t.detach().requires_grad_(True) for t in (inp, wr, wg, wu, wd)]
        w, i = route(leaves[0] @ leaves[1], k)
        y = FusedSwiGLUExperts.apply(leaves[0], w, i, *leaves[2:])
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(fixed)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(fixed)
    for seed in (5, 6):
        other = tokens(T, E, k, d, seed=seed)[0]
        fixed.copy_(other)
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step(other)):
            assert torch.equal(a, b)


def test_layers_in_a_row_with_a_padded_batch():
    """Several blocks one after another, as a model runs them; padded tokens (index -1) stay
    zero and change nothing for the others."""
    from fusedswiglu_b200 import FusedSwiGLUExperts, fp8_quantize_weight, fp8_swiglu_experts

    T, E, k, d, f = 260, 16, 4, 256, 128
    x, w, i = tokens(T, E, k, d)
    layers = [weights(E, d, f, seed=s) for s in range(4)]
    eight = [[t for m in layer for t in fp8_quantize_weight(m)] for layer in layers]

    def run(x, w, i):
        a, b = x, x
        for layer, q in zip(layers, eight):
            a = FusedSwiGLUExperts.apply(a, w, i, *layer)
            b = fp8_swiglu_experts(b, w, i, *q)
        return a, b

    whole = run(x, w, i)
    pad = torch.cat([x, torch.full((50, d), math.nan, device="cuda", dtype=x.dtype)])
    wp = torch.cat([w, torch.full((50, k), math.nan, device="cuda")])
    ip = torch.cat([i, torch.full((50, k), -1, device="cuda", dtype=torch.int32)])
    for a, b in zip(run(pad, wp, ip), whole):
        assert torch.equal(a[:T], b)
        assert (a[T:] == 0).all()


def test_a_block_without_tokens():
    from fusedswiglu_b200 import Fp8SwiGLUMoE, SwiGLUMoE

    m = SwiGLUMoE(64, 64, 8, 2, device="cuda")
    x = torch.zeros(3, 0, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    y = m(x)
    y.sum().backward()
    assert y.shape == x.shape == x.grad.shape
    assert all((p.grad == 0).all() and p.grad.shape == p.shape for p in m.parameters())
    assert Fp8SwiGLUMoE(m)(x.detach()).shape == x.shape


def test_shared_and_broadcast_inputs_get_summed_gradients():
    from fusedswiglu_b200 import FusedSwiGLUExperts

    E, d, f, T = 4, 64, 64, 50
    wg, _, wd = weights(E, d, f)
    x, w, i = tokens(1, E, 2, d)
    one, both, r = (t.detach().requires_grad_(True) for t in (x, wg, w))
    y = FusedSwiGLUExperts.apply(one.expand(T, d), r.expand(T, 2), i.expand(T, 2), both, both, wd)
    dy = torch.randn(T, d, device="cuda", dtype=torch.bfloat16)
    got = torch.autograd.grad(y, [one, r, both], dy)
    leaves = [t.detach().requires_grad_(True) for t in (x.expand(T, d), w.expand(T, 2), wg, wg)]
    y2 = FusedSwiGLUExperts.apply(leaves[0], leaves[1], i.expand(T, 2), leaves[2], leaves[3], wd)
    gx, gr, gg, gu = torch.autograd.grad(y2, leaves, dy)
    assert torch.equal(y, y2)
    # autograd's own sums, in the tensors' types
    assert torch.equal(got[0], gx.sum(0, keepdim=True)) and torch.equal(got[2], gg + gu)
    assert torch.allclose(got[1], gr.sum(0, keepdim=True), rtol=1e-5, atol=1e-6)
