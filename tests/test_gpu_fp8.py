"""8-bit products with a scale per block of 128 against the definition in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

# half a step of each type, relative: what one rounding is off by at most
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def rel(a, b):
    n = torch.linalg.norm(b)
    d = torch.linalg.norm(a.double() - b)
    return (d / n).item() if n > 0 else d.item()


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def e4m3(r):
    """Nearest e4m3 values of |r| <= 448 in 64 bits: 4 bits of significand down to 2^-6, steps
    of 2^-9 below.  (Powers of two by ldexp: pow is not exact on a GPU.)"""
    _, e = torch.frexp(r.abs().clamp_min(2.0 ** -6))
    return torch.ldexp(torch.round(torch.ldexp(r, 4 - e)), e - 4)


def quantised(v):
    """(values q, scale per row and block) of rows in 64 bits, from the type's definition."""
    T, d = v.shape
    nb = -(-d // 128)
    q, s = torch.zeros_like(v), torch.ones(T, nb, dtype=torch.float64, device="cuda")
    for b in range(nb):
        x = v[:, 128 * b:128 * b + 128]
        m, e = torch.frexp(x.abs().amax(dim=1))
        power = torch.where(m <= 0.875, e - 9, e - 8).clamp_min(-126)
        s[:, b] = torch.where(m > 0, torch.ldexp(torch.ones_like(m), power), torch.ones_like(m))
        q[:, 128 * b:128 * b + 128] = e4m3(x / s[:, b:b + 1])
    return q, s


def values(q, s):
    """Values a quantised weight (N, K) holds, in 64 bits."""
    full = s.double().repeat_interleave(128, 0)[:q.shape[0]].repeat_interleave(128, 1)[:, :q.shape[1]]
    return q.to(torch.float64) * full


def row_values(q, s):
    return q.to(torch.float64) * s.double().repeat_interleave(128, 1)[:, :q.shape[1]]


def weight(N, K, seed, scale_like=1.0):
    """A weight in 8 bits with fp32 scales that are not powers of two."""
    g = gen(seed)
    q = (torch.randn(N, K, device="cuda", generator=g) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    s = torch.rand(-(-N // 128), -(-K // 128), device="cuda", generator=g) + 0.5
    return q, s * (scale_like / (100 * math.sqrt(K)))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,d", [(1, 16), (3, 128), (7, 144), (130, 2064), (1030, 4112), (2, 14336)])
def test_rows_are_quantised_exactly(T, d, dtype):
    from fusedswiglu_b200 import fp8_quantize

    x = torch.randn(T, d, device="cuda", generator=gen(T)) * torch.exp2(torch.randint(-9, 9, (T, 1), device="cuda", generator=gen(d)).float())
    x = x.to(dtype)
    x[0, :16] = 0.0
    if d >= 256:
        x[-1, 128:256] = 0.0
        x[-1, 129] = 448.0       # exactly the largest value at scale 1
        x[0, 128:256] = 0.0
        x[0, 130] = torch.finfo(dtype).tiny
    q, s = fp8_quantize(x)
    wq, ws = quantised(x.double())
    assert q.dtype == torch.float8_e4m3fn and s.dtype == torch.float32 and s.shape == (T, -(-d // 128))
    assert torch.equal(s.double(), ws)
    assert torch.equal(q.to(torch.float64), wq)


def test_inf_and_nan_make_their_block_nan():
    from fusedswiglu_b200 import fp8_quantize, fp8_linear

    x = torch.randn(4, 384, device="cuda", generator=gen(0)).to(torch.bfloat16)
    x[1, 200] = math.inf
    x[2, 5] = math.nan
    q, s = fp8_quantize(x)
    assert torch.equal(s.isnan(), torch.tensor([[0, 0, 0], [0, 1, 0], [1, 0, 0], [0, 0, 0]], device="cuda").bool())
    w, ws = weight(128, 384, 1)
    y = fp8_linear(x, w, ws)
    assert y[1:3].isnan().all() and not y[0].isnan().any() and not y[3].isnan().any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(16, 8), (128, 128), (272, 200), (3, 144, 264)])
def test_weights_are_quantised_and_transposed(shape, dtype):
    from fusedswiglu_b200 import fp8_quantize_weight

    w = torch.randn(*shape, device="cuda", generator=gen(2)).to(dtype)
    q, s = fp8_quantize_weight(w)
    for e, we in enumerate(w if w.ndim == 3 else w[None]):
        qe, se = (q[e], s[e]) if w.ndim == 3 else (q, s)
        wt = we.t().double()
        assert qe.shape == wt.shape and se.shape == (-(-wt.shape[0] // 128), -(-wt.shape[1] // 128))
        for i in range(se.shape[0]):
            for j in range(se.shape[1]):
                block = wt[128 * i:128 * i + 128, 128 * j:128 * j + 128]
                m, ex = torch.frexp(block.abs().max())
                want = 2.0 ** (ex - 9 if m <= 0.875 else ex - 8).item()
                assert se[i, j].item() == want
                assert torch.equal(qe[128 * i:128 * i + 128, 128 * j:128 * j + 128].to(torch.float64), e4m3(block / want))


# fp32 sums: 128 products, exact (two significands of 4 bits), added in tensor memory and then over K / 128 blocks: each addition at most half a
# step of the running sum, of which a random walk keeps about the square root of their number;
# (128 + K / 128) / 2 half steps 2^-24 bound it from above at these sizes by 2^-17, next to the
# one rounding of the output: HALF at most, and evenly spread over a step less than half of that in the norm.
def bound(dtype):
    return 0.5 * HALF[dtype] + 2.0 ** -15


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,K,N", [
    (1, 16, 8), (1, 128, 128), (1, 4096, 1024), (5, 1040, 264), (77, 2064, 520), (120, 4096, 256), (129, 512, 384),
    (300, 272, 2000), (1000, 4096, 4104), (2100, 1168, 4096), (8, 14336, 512),
])
def test_linear(T, K, N, dtype):
    from fusedswiglu_b200 import _lib, fp8_linear, fp8_matmul, fp8_quantize

    x = torch.randn(T, K, device="cuda", generator=gen(T + K)).to(dtype)
    w, ws = weight(N, K, N)
    y = fp8_linear(x, w, ws)
    q, s = quantised(x.double())
    want = row_values(q, s) @ values(w, ws).t()
    torch.cuda.synchronize()
    assert _lib.device_status() == 0
    assert y.dtype == dtype and y.shape == (T, N)
    assert rel(y, want) <= bound(dtype)
    # element by element: no stripe, tile or block is off
    assert ((y.double() - want).abs() <= HALF[dtype] * want.abs() + 1e-3 * HALF[dtype] / 2 ** -8 * want.abs().max()).all()
    # the same rows, quantised apart, with scales stored row by row
    xq, xs = fp8_quantize(x)
    assert torch.equal(fp8_matmul(xq, xs.contiguous(), w, ws, dtype), y)


def test_each_block_has_its_own_scale():
    """One nonzero block of the row and of the weight at a time."""
    from fusedswiglu_b200 import fp8_matmul

    T, K, N = 3, 640, 384
    w, ws = weight(N, K, 4)
    q = torch.zeros(T, K, device="cuda").to(torch.float8_e4m3fn)
    s = torch.rand(T, 5, device="cuda", generator=gen(5)) + 0.5
    for b in range(5):
        one = q.to(torch.float32)
        one[:, 128 * b + 3] = 2.0
        y = fp8_matmul(one.to(torch.float8_e4m3fn), s, w, ws, torch.float16)
        want = 2.0 * s[:, b:b + 1].double() * values(w, ws)[:, 128 * b + 3][None]
        # one rounding to fp16, at most half a step, 2^-11 of the value; three fp32 products before it
        assert ((y.double() - want).abs() <= HALF[torch.float16] * 1.001 * want.abs() + 2.0 ** -25).all()


def mlp_definition(x, wg, sg, wu, su, wd, sd):
    q, s = quantised(x.double())
    xv = row_values(q, s)
    h = torch.nn.functional.silu(xv @ values(wg, sg).t()) * (xv @ values(wu, su).t())
    q, s = quantised(h)
    return row_values(q, s) @ values(wd, sd).t()


# A value of h next to a border between two e4m3 numbers may round the other way when fp32
# moves it: with g and u off by about 2^-20 that is a fraction of 2^-20 / 2^-4 of the values, each by
# a step of 2^-3: in the norm sqrt(2^-16) * 2^-3 = 2^-11 at most, besides the output's rounding.
def mlp_bound(dtype):
    return 0.5 * HALF[dtype] + 2.0 ** -11


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,d,f,o", [(1, 128, 128, 128), (2, 272, 144, 264), (33, 512, 1040, 256), (300, 1024, 400, 1000),
                                     (1500, 512, 1408, 520)])
def test_mlp(T, d, f, o, dtype):
    from fusedswiglu_b200 import fp8_swiglu_mlp, _lib

    x = torch.randn(T, d, device="cuda", generator=gen(T)).to(dtype)
    args = (*weight(f, d, 1), *weight(f, d, 2), *weight(o, f, 3))
    y = fp8_swiglu_mlp(x, *args)
    torch.cuda.synchronize()
    assert _lib.device_status() == 0
    assert rel(y, mlp_definition(x, *args)) <= mlp_bound(dtype)


def stack(E, N, K, seed):
    ws = [weight(N, K, seed + e) for e in range(E)]
    return torch.stack([q for q, _ in ws]), torch.stack([s for _, s in ws])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,E,k,d,f,o", [(1, 8, 2, 128, 128, 128), (4, 16, 6, 272, 144, 264), (60, 4, 3, 256, 400, 128),
                                        (700, 12, 4, 144, 272, 136), (1600, 3, 2, 512, 256, 512)])
def test_experts(T, E, k, d, f, o, dtype):
    from fusedswiglu_b200 import fp8_swiglu_experts, _lib

    x = torch.randn(T, d, device="cuda", generator=gen(T)).to(dtype)
    logits = torch.randn(T, E, device="cuda", generator=gen(1)) + torch.randn(E, device="cuda", generator=gen(2))
    top, idx = torch.topk(logits, k, dim=1)
    r = torch.softmax(top, dim=1)
    if T > 50:
        idx[::9, 0] = -1
        idx[5] = E
    args = (*stack(E, f, d, 10), *stack(E, f, d, 50), *stack(E, o, f, 90))
    y = fp8_swiglu_experts(x, r, idx.to(torch.int32), *args)
    torch.cuda.synchronize()
    assert _lib.device_status() == 0
    want = torch.zeros(T, o, dtype=torch.float64, device="cuda")
    for e in range(E):
        t, j = torch.nonzero(idx == e, as_tuple=True)
        if t.numel():
            want.index_add_(0, t, r[t, j, None].double() * mlp_definition(x[t], *(a[e] for a in args)))
    # one more rounding than the dense block: the expert's row before the weighted sum
    assert rel(y, want) <= mlp_bound(dtype) + 0.5 * HALF[dtype]
    assert torch.equal(fp8_swiglu_experts(x, r, idx, *args), y)
    if T > 50:
        assert (y[5] == 0).all()


def test_modules_agree_with_their_16_bit_blocks():
    """Serving forms next to the blocks they come from: off by the quantisation only, two
    roundings to 4 bits (half a step 2^-4 at most, 0.3 of that in the norm each way) per product."""
    from fusedswiglu_b200 import Fp8SwiGLUMLP, Fp8SwiGLUMoE, SwiGLUMoE
    from fusedswiglu_b200.mlp import SwiGLUMLP

    torch.manual_seed(0)
    x = torch.randn(3, 50, 256, device="cuda", dtype=torch.bfloat16)
    for block, served in ((SwiGLUMLP(256, 512, device="cuda"), Fp8SwiGLUMLP),
                          (SwiGLUMoE(256, 128, 16, 4, use_balance_bias=True, device="cuda"), Fp8SwiGLUMoE)):
        with torch.no_grad():
            want = block(x)
        got = served(block)(x)
        assert got.shape == want.shape and got.dtype == want.dtype
        assert rel(got, want.double()) < 6 * 0.3 * 2.0 ** -4
        assert not got.requires_grad
        moved = served(block).state_dict()
        assert any(v.dtype == torch.float8_e4m3fn for v in moved.values())


def test_no_rows_streams_graphs_and_leading_axes():
    from fusedswiglu_b200 import fp8_linear, fp8_quantize, fp8_swiglu_experts, fp8_swiglu_mlp

    K, N = 256, 512
    w, ws = weight(N, K, 1)
    d, sd = weight(K, N, 2)
    x = torch.randn(6, 10, K, device="cuda", generator=gen(3)).to(torch.bfloat16)
    y = fp8_linear(x, w, ws)
    assert y.shape == (6, 10, N) and torch.equal(y.view(60, N), fp8_linear(x.view(60, K).t().contiguous().t(), w, ws))
    assert fp8_linear(x[:0], w, ws).shape == (0, 10, N)
    assert fp8_quantize(x[:0].view(0, K))[0].shape == (0, K)
    assert fp8_swiglu_mlp(x[:0], w, ws, w, ws, d, sd).shape == (0, 10, K)
    args = [t[None] for t in (w, ws, w, ws, d, sd)]
    assert fp8_swiglu_experts(x[0, :0], torch.zeros(0, 1, device="cuda"), torch.zeros(0, 1, device="cuda", dtype=torch.int32), *args).shape == (0, K)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y2 = fp8_swiglu_mlp(x, w, ws, w, ws, d, sd)
    y1 = fp8_swiglu_mlp(x.flip(0).contiguous(), w, ws, w, ws, d, sd)
    torch.cuda.synchronize()
    assert torch.equal(y2, fp8_swiglu_mlp(x, w, ws, w, ws, d, sd)) and torch.equal(y1.flip(0), y2)
    xs = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        yg = fp8_swiglu_mlp(xs, w, ws, w, ws, d, sd)
    xs.copy_(x.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(yg, y1)
