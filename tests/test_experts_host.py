"""Refusals and sizes of the routed experts' entry points, without a GPU."""
import ctypes

import pytest
import torch

from fusedswiglu_b200 import FusedSwiGLUExperts, SwiGLUMoE, _launch, _lib

P = 16  # never dereferenced: every call below is refused before any CUDA call


def forward(T=4, k=2, E=8, d=64, f=64, o=64, dtype=0, wtype=2, x=P, saved=None, saved_bytes=0, scratch=P, nbytes=1 << 40):
    return _lib.load().fsw_experts_forward(x, P, P, P, P, P, P, saved, saved_bytes, scratch, nbytes, T, k, E, d, f, o,
                                           dtype, wtype, None)


@pytest.mark.parametrize("kw,what", [
    (dict(dtype=2), "dtype"), (dict(wtype=1), "weights"), (dict(k=0), "top_k"), (dict(k=33), "top_k"),
    (dict(E=0), "experts"), (dict(E=1025), "experts"), (dict(d=60), "multiples of 8"), (dict(f=60), "multiples of 8"),
    (dict(o=60), "multiples of 8"), (dict(d=0), "feature"), (dict(T=1 << 31), "many"), (dict(T=1 << 30), "many"),
    (dict(T=-1), "tokens"), (dict(x=None), "NULL"), (dict(scratch=None), "NULL"), (dict(x=8), "aligned"),
    (dict(nbytes=100), "too small"), (dict(saved=P, saved_bytes=100), "too small"),
])
def test_forward_refusals(kw, what):
    assert forward(**kw) == -1
    assert what in _lib.last_error()


def test_backward_refusals():
    lib = _lib.load()

    def backward(dy=P, saved_bytes=1 << 40, nbytes=1 << 40, dwg=P, dwu=P, dtype=0):
        return lib.fsw_experts_backward(dy, P, P, P, P, P, saved_bytes, P, nbytes, P, P, dwg, dwu, P, 4, 2, 8, 64, 64, 64,
                                        dtype, 2, None)

    for kw, what in ((dict(dy=None), "NULL"), (dict(saved_bytes=8), "too small"), (dict(nbytes=8), "too small"),
                     (dict(dwu=None), "together"), (dict(dy=8), "aligned"), (dict(dtype=9), "dtype")):
        assert backward(**kw) == -1
        assert what in _lib.last_error()


def test_sizes_cover_every_split_of_the_pairs_over_the_experts():
    """Rows of all experts, each padded to whole tiles, never exceed the bound the buffers
    are sized by, whatever the routing."""
    for T, k, E in [(1, 1, 1), (1, 6, 64), (5, 3, 4), (100, 4, 8), (1000, 2, 3), (4096, 8, 128)]:
        pairs = T * k
        tile = 256 if pairs >= 256 * E else 128
        saved, fwd, inf, back = _launch._expert_sizes(T, k, E, 64, 64, 64)
        used = min(pairs, E)
        for spread in ([pairs - (used - 1)] + [1] * (used - 1), [pairs // used + (i < pairs % used) for i in range(used)]):
            assert sum(spread) == pairs
            rows = sum(-(-c // tile) * tile for c in spread)
            # saved holds xs, g, u: 3 arrays of `rows` x 64 16-bit values behind the plan
            assert 3 * rows * 64 * 2 <= saved and 2 * rows * 64 * 2 <= fwd
    assert _launch._expert_sizes(0, 2, 8, 64, 64, 64)[0] > 0


def test_python_refusals():
    z = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype)
    x, w, i = z(4, 64), z(4, 2, dtype=torch.float32), z(4, 2, dtype=torch.int32)
    wg, wd = z(8, 64, 32), z(8, 32, 64)
    with pytest.raises(RuntimeError, match="CUDA"):
        FusedSwiGLUExperts.apply(x, w, i, wg, wg, wd)
    for args, what in (((x, w, i, wg, z(8, 64, 40), wd), "same shape"), ((z(4, 72), w, i, wg, wg, wd), "mismatch"),
                       ((x, w, i, wg, wg, z(7, 32, 64)), "mismatch"), ((x, w[:3], i, wg, wg, wd), "top_k"),
                       ((x, w, i.float(), wg, wg, wd), "indices"), ((x, w.double(), i, wg, wg, wd), "weights"),
                       ((x, w, i, wg.half(), wg.half(), wd), "one dtype"), ((x[0], w, i, wg, wg, wd), "dimensions")):
        with pytest.raises(AssertionError, match=what):
            FusedSwiGLUExperts.apply(*args)
    with pytest.raises(ValueError):
        SwiGLUMoE(64, 64, 6, 2)
    with pytest.raises(ValueError):
        SwiGLUMoE(64, 64, 8, 2, dtype=torch.float32)


def test_indices_that_do_not_fit_32_bits_stay_out_of_range():
    idx = torch.tensor([[0, 2 ** 32], [-(2 ** 32) + 3, 7]])
    got = _launch.expert_indices(idx, 8)
    assert got.dtype == torch.int32 and got[0, 0] == 0 and got[1, 1] == 7
    assert not (0 <= got[0, 1] < 8) and not (0 <= got[1, 0] < 8)
