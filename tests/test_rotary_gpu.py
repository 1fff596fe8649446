"""Rotary positions (tq_rotary, rope.py) against float64.

Tolerance: angles are exact to 2^-52 of their turns, sincospif to 2 ulp, the two products and their sum round three times in float32, then
once to the type: |error| <= (eps(type) / 2) |y| + 8 eps32 (|a| + |b|) factor."""

import pytest
import torch

from blocks_util import rotary as exact_rotary

pytestmark = pytest.mark.gpu


def make(b, h, length, d, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(b, length, h, d, generator=g).to(dtype).cuda().transpose(1, 2)


def check(got, x, freqs, positions, interleaved, factor):
    ref = exact_rotary(x.cpu(), freqs, positions, interleaved, factor)
    big = x.double().abs().cpu().amax(-1, keepdim=True)
    tol = torch.finfo(x.dtype).eps / 2 * ref.abs() + 16 * torch.finfo(torch.float32).eps * big * max(factor, 1.0)
    if x.dtype is torch.float16:
        tol = tol + 2.0 ** -25                             # (half a step of the subnormals)
    err = (got.double().cpu() - ref).abs()
    assert got.is_contiguous() and got.dtype is x.dtype and got.shape == x.shape
    assert bool((err <= tol).all()), float((err - tol).max())


@pytest.mark.parametrize("dtype", (torch.float16, torch.bfloat16, torch.float32))
@pytest.mark.parametrize("interleaved", (False, True))
@pytest.mark.parametrize("d,dims", ((128, 128), (96, 24), (64, 32), (256, 64), (128, 6), (80, 2), (33, 20)))
def test_against_float64(d, dims, interleaved, dtype):
    from mlx_turboquant_b200 import rope
    f, factor = rope.frequencies(dims, 10000.0)
    for b, hq, hkv, length, offset in ((1, 4, 2, 1, 0), (3, 5, 1, 7, 12345), (1, 32, 8, 130, 70000)):
        q, k = make(b, hq, length, d, dtype, 1), make(b, hkv, length, d, dtype, 2)
        pos = torch.arange(offset, offset + length)
        gq, gk = rope.apply_rotary(q, k, f, offset, interleaved=interleaved, factor=1.25)
        check(gq, q, f, pos, interleaved, 1.25)
        check(gk, k, f, pos, interleaved, 1.25)


def test_far_positions_and_positions_of_their_own():
    from mlx_turboquant_b200 import rope
    f, _ = rope.frequencies(128, 500000.0)
    q, k = make(2, 8, 5, 128, torch.bfloat16, 3), make(2, 2, 5, 128, torch.bfloat16, 4)
    pos = torch.tensor([[0, 1, 2 ** 20 + 1, 2 ** 24 + 3, 2 ** 33 + 5], [7, 7, 3, 2, 1]])
    gq, gk = rope.apply_rotary(q, k, f, positions=pos.cuda())
    check(gq, q, f, pos, False, 1.0)
    check(gk, k, f, pos, False, 1.0)
    gq, gk = rope.apply_rotary(q, None, f, positions=pos[0].cuda())
    assert gk is None
    check(gq, q, f, pos[0], False, 1.0)
    assert torch.equal(rope.apply_rotary(q, k, f, 2 ** 24)[0], rope.apply_rotary(q, k, f, positions=torch.arange(2 ** 24, 2 ** 24 + 5).cuda())[0])


def test_strides_and_slow_path(monkeypatch):
    """Views of a fused projection, unaligned and padded rows, and the path without the native host module: the same bits."""
    from mlx_turboquant_b200 import _lib, rope
    f, _ = rope.frequencies(64, 10000.0)
    base = torch.randn(2, 9, 12, 70, device="cuda").to(torch.float16)
    views = [base.transpose(1, 2)[:, :8, :, 3:67], base.transpose(1, 2)[:, 8:12, :, 3:67]]
    gq, gk = rope.apply_rotary(views[0], views[1], f, 11)
    check(gq, views[0].contiguous(), f, torch.arange(11, 20), False, 1.0)
    check(gk, views[1].contiguous(), f, torch.arange(11, 20), False, 1.0)
    turned = base.permute(0, 2, 3, 1)[:, :, :64]                                  # last axis not contiguous: the caller's path copies
    t = turned.transpose(2, 3)
    monkeypatch.setattr(_lib, "_host", _lib._NoHost())
    sq, sk = rope.apply_rotary(views[0], views[1], f, 11)
    assert torch.equal(gq, sq) and torch.equal(gk, sk)
    st, _ = rope.apply_rotary(t, None, f, 3)
    check(st, t.contiguous(), f, torch.arange(3, 12), False, 1.0)


def test_empty_and_refusals():
    from mlx_turboquant_b200 import rope
    f, _ = rope.frequencies(64)
    q = torch.randn(1, 2, 0, 64, device="cuda", dtype=torch.float16)
    assert rope.apply_rotary(q, q, f, 0)[0].shape == q.shape
    q = torch.randn(1, 2, 3, 64, device="cuda", dtype=torch.float16)
    with pytest.raises(ValueError):
        rope.apply_rotary(q, q.bfloat16(), f)
    with pytest.raises(ValueError):
        rope.apply_rotary(q, q, f.float())
    with pytest.raises(ValueError):
        rope.apply_rotary(q[..., :32], None, f)
    with pytest.raises(ValueError):
        rope.apply_rotary(q, q, f, positions=torch.zeros(4, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError):
        rope.apply_rotary(q, q, f, positions=torch.zeros(3, dtype=torch.int32, device="cuda"))
    with pytest.raises(TypeError):
        rope.apply_rotary(q.double(), None, f)
    with pytest.raises(RuntimeError, match="CUDA"):
        rope.apply_rotary(q.cpu(), None, f)
    with pytest.raises(RuntimeError, match="backward"):
        rope.apply_rotary(q.requires_grad_(), None, f)
    with torch.no_grad():
        rope.apply_rotary(q, None, f)


def test_captured_and_on_a_side_stream():
    from mlx_turboquant_b200 import rope
    f, _ = rope.frequencies(128)
    q, k = make(2, 8, 3, 128, torch.bfloat16, 5), make(2, 4, 3, 128, torch.bfloat16, 6)
    pos = torch.zeros(3, dtype=torch.int64, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        rope.apply_rotary(q, k, f, positions=pos)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gq, gk = rope.apply_rotary(q, k, f, positions=pos)
    for start in (5, 1000):
        pos.copy_(torch.arange(start, start + 3))
        graph.replay()
        eq, ek = rope.apply_rotary(q, k, f, start)
        assert torch.equal(gq, eq) and torch.equal(gk, ek)
