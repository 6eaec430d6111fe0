"""Refusals of the routing entry points, without a GPU."""
import pytest
import torch

from fusedswiglu_b200 import _lib, route

P = 16  # never dereferenced: every call below is refused before any CUDA call


def call(T=4, ld=8, E=8, k=2, dtype=0, score=0, scale=1.0, groups=1, topk_groups=1):
    return _lib.load().fsw_route(P, ld, None, P, P, T, E, k, dtype, score, 1, scale, groups, topk_groups, None)


@pytest.mark.parametrize("kw,what", [
    (dict(dtype=3), "dtype"), (dict(score=2), "score"), (dict(T=-1), "tokens"), (dict(E=0), "experts"),
    (dict(E=1025, ld=1025), "experts"), (dict(k=0), "top_k"), (dict(k=9), "top_k"),
    (dict(E=64, ld=64, k=33), "top_k"), (dict(groups=3), "num_groups"), (dict(groups=0), "num_groups"),
    (dict(E=64, ld=64, groups=64), "num_groups"), (dict(groups=4, topk_groups=5), "topk_groups"),
    (dict(groups=4, topk_groups=0), "topk_groups"), (dict(groups=4, topk_groups=1, k=3), "exceeds"),
    (dict(scale=float("inf")), "finite"), (dict(scale=float("nan")), "finite"), (dict(ld=7), "stride"),
])
def test_refusals(kw, what):
    assert call(**kw) == -1
    assert what in _lib.last_error()


def test_null_pointers_and_empty_batches():
    lib = _lib.load()
    assert lib.fsw_route(None, 8, None, P, P, 4, 8, 2, 0, 0, 1, 1.0, 1, 1, None) == -1
    assert "NULL" in _lib.last_error()
    assert lib.fsw_route_backward(P, 8, None, P, P, 4, 8, 2, 0, 0, 1, 1.0, None) == -1
    assert "NULL" in _lib.last_error()
    assert call(T=0) == 0


def test_python_refusals():
    z = torch.zeros(4, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        route(z, 2)
    with pytest.raises(AssertionError, match="score"):
        route(z, 2, score="relu")
    with pytest.raises(AssertionError, match="bias"):
        route(z, 2, bias=torch.zeros(7))
    with pytest.raises(AssertionError, match="logits"):
        route(torch.zeros(8), 2)
    with pytest.raises(AssertionError, match="fp32 logits"):
        route(z.double(), 2)
