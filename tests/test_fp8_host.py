"""Refusals of the 8-bit entry points, without a GPU."""
import pytest
import torch

from fusedswiglu_b200 import _lib, fp8_linear, fp8_matmul, fp8_quantize, fp8_swiglu_experts, fp8_swiglu_mlp

P = 16  # never dereferenced: every call below is refused before any CUDA call
BIG = 1 << 40


def linear(x=P, T=4, K=256, N=64, dtype=0, scratch=P, nbytes=BIG):
    return _lib.load().fsw_fp8_linear(x, P, P, P, scratch, nbytes, T, K, N, dtype, None)


@pytest.mark.parametrize("kw,what", [
    (dict(dtype=2), "dtype"), (dict(K=24), "multiple of 16"), (dict(N=12), "of 8"), (dict(T=-1), "rows"), (dict(K=0), "sizes"),
    (dict(T=1 << 31), "rows"), (dict(x=None), "NULL"), (dict(scratch=None), "NULL"), (dict(x=8), "aligned"),
    (dict(nbytes=64), "too small"),
])
def test_linear_refusals(kw, what):
    assert linear(**kw) == -1
    assert what in _lib.last_error()


def test_other_refusals():
    lib = _lib.load()
    assert lib.fsw_fp8_gemm(P, P, -1, 1, P, P, P, 4, 128, 64, 0, None) == -1 and "stride" in _lib.last_error()
    assert lib.fsw_fp8_gemm(P, None, 1, 1, P, P, P, 4, 128, 64, 0, None) == -1 and "NULL" in _lib.last_error()
    assert lib.fsw_fp8_quantize_rows(P, P, P, 4, 100, 0, None) == -1 and "multiple" in _lib.last_error()
    assert lib.fsw_fp8_quantize_weight(P, P, P, 0, 128, 128, 0, None) == -1 and "weights" in _lib.last_error()
    assert lib.fsw_fp8_mlp(P, P, P, P, P, P, P, P, P, 8, 4, 128, 128, 128, 0, None) == -1 and "too small" in _lib.last_error()
    assert lib.fsw_fp8_mlp(P, P, P, P, P, P, P, P, P, BIG, 4, 128, 136, 128, 0, None) == -1 and "multiple of 16" in _lib.last_error()
    args = [P] * 11
    assert lib.fsw_fp8_experts_forward(*args, BIG, 4, 2, 8, 128, 136, 128, 0, 2, None) == -1
    assert lib.fsw_fp8_experts_forward(*args, 8, 4, 2, 8, 128, 128, 128, 0, 2, None) == -1 and "too small" in _lib.last_error()
    assert lib.fsw_fp8_experts_forward(*args, BIG, 4, 0, 8, 128, 128, 128, 0, 2, None) == -1 and "top_k" in _lib.last_error()
    assert lib.fsw_fp8_linear_scratch_bytes(4, 100) < 0 and lib.fsw_fp8_mlp_scratch_bytes(4, 100, 128) < 0
    assert linear(T=0) == 0


def test_python_refusals():
    x = torch.zeros(4, 256, dtype=torch.bfloat16)
    q, s = torch.zeros(384, 256).to(torch.float8_e4m3fn), torch.ones(3, 2)
    with pytest.raises(RuntimeError, match="CUDA"):
        fp8_linear(x, q, s)
    with pytest.raises(AssertionError, match="scales"):
        fp8_linear(x, q, s[:2])
    with pytest.raises(AssertionError, match="scales"):
        fp8_linear(x, q, s.double())
    with pytest.raises(AssertionError, match="float8"):
        fp8_linear(x, q.float(), s)
    with pytest.raises(AssertionError, match="mismatch"):
        fp8_linear(x[:, :128], q, s)
    with pytest.raises(AssertionError, match="inference"):
        fp8_linear(x.requires_grad_(True), q, s)
    x = x.detach()
    with pytest.raises(AssertionError, match="bfloat16 or"):
        fp8_linear(x.float(), q, s)
    with pytest.raises(AssertionError, match="dimensions"):
        fp8_quantize(x[0])
    with pytest.raises(AssertionError, match="row scales"):
        fp8_matmul(x.float().to(torch.float8_e4m3fn), torch.ones(4, 3), q, s)
    down, sd = torch.zeros(64, 384).to(torch.float8_e4m3fn), torch.ones(1, 3)
    with pytest.raises(AssertionError, match="mismatch"):
        fp8_swiglu_mlp(x, q, s, q, s, down[:, :256], sd[:, :2])
    with pytest.raises(AssertionError, match="same shape"):
        fp8_swiglu_mlp(x, q, s, q[:128], s[:1], down, sd)
    with pytest.raises(AssertionError, match="top_k"):
        fp8_swiglu_experts(x, torch.ones(3, 2), torch.zeros(3, 2, dtype=torch.int32),
                           *(t[None] for t in (q, s, q, s, down, sd)))
