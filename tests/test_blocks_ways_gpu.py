"""Every way that attention over the 8-bit block cache can take (tq_blocks_attend_choice), at every head_dim that has it: shapes for which it is the one that runs, each lane with tokens of
its own, results against float64 within a bound relative to sum(w |v|).  And what runs where there is no room for the scratch."""

import ctypes as C
import math

import pytest
import torch

from test_blocks_gpu import storage

pytestmark = pytest.mark.gpu

ALONE, RUNS, CLUSTER, FUSED, FUSED_CUT, EXPANDED, EXPANDED_CUT = range(2, 9)
# sequences, KV heads, query heads, tokens, queries, window
SHAPES = {
    (ALONE, 64): (1, 1, 1, 2, 1, 0), (ALONE, 96): (2, 2, 4, 33, 1, 20), (ALONE, 128): (1, 3, 3, 70, 1, 0), (ALONE, 256): (1, 1, 2, 20, 2, 0),
    (RUNS, 64): (40, 8, 8, 2289, 1, 0), (RUNS, 96): (1, 1, 4, 7724, 1, 0), (RUNS, 128): (1, 1, 2, 6579, 1, 0), (RUNS, 256): (1, 1, 1, 5446, 1, 0),
    (CLUSTER, 64): (1, 2, 2, 667, 1, 0), (CLUSTER, 96): (1, 1, 1, 528, 1, 0), (CLUSTER, 128): (1, 1, 1, 550, 1, 0), (CLUSTER, 256): (1, 1, 1, 460, 1, 0),
    (FUSED, 64): (20, 8, 96, 50, 2, 0), (FUSED, 96): (20, 8, 96, 50, 2, 40), (FUSED, 128): (20, 8, 56, 40, 3, 0),
    (FUSED_CUT, 64): (1, 1, 4, 652, 652, 0), (FUSED_CUT, 96): (1, 2, 8, 1891, 93, 0), (FUSED_CUT, 128): (1, 1, 8, 7227, 7, 0),
    (EXPANDED, 64): (9, 3, 36, 300, 33, 291), (EXPANDED, 96): (9, 3, 36, 265, 35, 0), (EXPANDED, 128): (5, 8, 96, 210, 19, 0), (EXPANDED, 256): (40, 2, 14, 30, 5, 0),
    (EXPANDED_CUT, 64): (5, 3, 36, 4359, 18, 0), (EXPANDED_CUT, 96): (2, 2, 24, 4245, 81, 0), (EXPANDED_CUT, 128): (2, 1, 12, 1783, 412, 0), (EXPANDED_CUT, 256): (1, 3, 24, 1496, 25, 0),
}


def tokens(b, h, t, d, dtype, seed, std=0.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(b, h, t, d, generator=g, device="cuda") * torch.exp(std * torch.randn(b, h, t, 1, generator=g, device="cuda"))).to(dtype)


def held(codes, scales, tail, length):
    """float64 on the GPU: what the storage stands for"""
    n = tail.shape[2]
    cut = length // n * n
    return torch.cat([codes[:, :, :cut].float().double() * scales[:, :, :cut // n].double().repeat_interleave(n, dim=2)[..., None], tail[:, :, :length - cut].double()], dim=2)


def check(got, q, store, length, window=0, sinks=0, weights=2.0 ** -11):
    """Lane by lane.  `weights`: what a weight may be rounded by; 2^-14 beside it for the rest, then the result's own rounding.

    A weight's fp16 parts end at 2^-24 (half of that is the rounding), where the largest value scale of the tokens seen stands at 2^4 or more and the row's reference, no larger than
    its largest weight, at 1: each token is off by up to 2^-25 |code| / 2^4 of that value scale, 2^-29 max|v|, whatever its weight.  That is all there is in coordinates where the one
    token that a row is about has the code 0."""
    b, hq, t, d = q.shape
    h = store[0].shape[1]
    j, pos = torch.arange(length, device="cuda")[None, :], torch.arange(length - t, length, device="cuda")[:, None]
    seen = (j <= pos) & ((pos - j < window) | (j < sinks)) if window else j <= pos
    for i in range(b):
        k, v = held(*(x[i:i + 1] for x in store[0:2]), store[4][i:i + 1], length), held(*(x[i:i + 1] for x in store[2:4]), store[5][i:i + 1], length)
        s = (q[i:i + 1].double().reshape(1, h, -1, d) @ k.transpose(-1, -2)).reshape(1, h, hq // h, t, length) / math.sqrt(d)
        w = torch.softmax(s.masked_fill(~seen, -math.inf), dim=-1).reshape(1, h, -1, length)
        ref, wv = (w @ v).reshape(1, hq, t, d), (w @ v.abs()).reshape(1, hq, t, d)
        err, tol = (got[i:i + 1].double() - ref).abs(), torch.finfo(got.dtype).eps / 2 * ref.abs() + (weights + 2.0 ** -14) * wv + length * 2.0 ** -29 * v.abs().max() + 2.0 ** -25
        assert bool((err <= tol).all()), (i, float((err / tol).max()))


def arguments(q, out, store, length, window=0, sinks=0):
    from mlx_turboquant_b200 import _lib, blocks
    a = _lib.BlocksAttendArgs()
    a.store = blocks._store(*store, length)
    a.n_q_heads, a.t_q, a.q, a.scale, a.window, a.sinks, a.out = q.shape[1], q.shape[2], blocks._rows(q), q.shape[3] ** -0.5, window, sinks, out.data_ptr()
    return a


def attend_within(room, q, store, length, window=0, sinks=0):
    """-> (result of a call that is given at most `room` bytes of scratch, the way it takes, the scratch it has)"""
    from mlx_turboquant_b200 import _lib
    lib, out = _lib.lib(), torch.full_like(q, math.nan)
    a = arguments(q, out, store, length, window, sinks)
    need = lib.tq_blocks_attend_workspace_within(C.byref(a), room)
    assert need <= room
    ws = torch.full((need + 256,), 0xff, dtype=torch.uint8, device="cuda")          # (any content; NaN as floats)
    a.workspace, a.workspace_bytes = (ws.data_ptr(), need) if need else (None, 0)
    way = lib.tq_blocks_attend_choice(C.byref(a))
    assert lib.tq_blocks_attend(C.byref(a), torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert bool((ws[need:] == 0xff).all())                                           # nothing behind what it asked for
    return out, way, need


def filled(b, h, total, d, block, codes, dtype, seed):
    from mlx_turboquant_b200 import blocks
    store = storage(b, h, total, d, block, codes, dtype)
    blocks.write_blocks(tokens(b, h, total, d, dtype, seed), tokens(b, h, total, d, dtype, seed + 1), *store, 0)
    return store


@pytest.mark.parametrize("way,d", SHAPES)
@pytest.mark.parametrize("codes", (torch.int8, torch.float8_e4m3fn))
@pytest.mark.parametrize("dtype", (torch.float16, torch.bfloat16))
def test_every_way(way, d, codes, dtype):
    from mlx_turboquant_b200 import _lib, blocks
    b, h, hq, total, t, window = SHAPES[way, d]
    sinks = 4 if window else 0
    store, q = filled(b, h, total, d, 64, codes, dtype, 7), tokens(b, hq, t, d, dtype, 9, std=0)
    a = arguments(q, q, store, total, window, sinks)
    a.workspace_bytes = (1 << 64) - 1
    assert _lib.lib().tq_blocks_attend_choice(C.byref(a)) == way
    got = blocks.attend_blocks(q, *store, total, window=window or None, sinks=sinks)
    check(got, q, store, total, window, sinks, 2.0 ** -11 if dtype is torch.bfloat16 and way >= FUSED else 0.0)
    again, its_way, _ = attend_within((1 << 64) - 1, q, store, total, window, sinks)
    assert its_way == way and torch.equal(again, got)                                 # (whatever the scratch held)
    assert _lib.lib().tq_device_status() == 0


@pytest.mark.parametrize("d,codes,dtype", ((64, torch.float8_e4m3fn, torch.bfloat16), (96, torch.int8, torch.float16), (128, torch.int8, torch.bfloat16), (256, torch.float8_e4m3fn, torch.float16)))
def test_less_scratch_than_the_fastest_way_wants(d, codes, dtype):
    """From all that it would like down to none: the ways get leaner, lanes are done in more rounds, results stay within their bounds.  Lanes of different tokens: a round that
    took another's would show."""
    total, t, ways = 6000, 400, []
    store, q = filled(14, 1, total, d, 32, codes, dtype, 3), tokens(14, 8, t, d, dtype, 5, std=0)
    room = (1 << 64) - 1
    while True:
        got, way, need = attend_within(room, q, store, total)
        ways.append(way)
        check(got, q, store, total, weights=2.0 ** -11)
        if need == 0:
            break
        room = min(need - 1, int(need * 0.8))
    assert way in (ALONE, CLUSTER) and sum(x in (EXPANDED, EXPANDED_CUT) for x in ways) > 1, ways


@pytest.mark.parametrize("native", (True, False))
@pytest.mark.parametrize("room", ("some", "none"))
def test_a_card_without_room_for_the_scratch(monkeypatch, native, room):
    """The allocator refuses what the fastest way wants: the call runs all the same."""
    from mlx_turboquant_b200 import _lib, blocks, kernels
    if not native:
        monkeypatch.setattr(_lib, "_host", _lib._NoHost())
    store, q = filled(2, 8, 32000, 128, 64, torch.int8, torch.bfloat16, 3), tokens(2, 32, 200, 128, torch.bfloat16, 5, std=0)
    a = arguments(q, q, store, 32000)
    assert _lib.lib().tq_blocks_attend_workspace(C.byref(a)) > 4 * blocks.SMALL
    want = blocks.attend_blocks(q, *store, 32000)
    check(want, q, store, 32000)
    out, asked, scratch = torch.empty_like(q), [], kernels.scratch

    def limited(dev, *sizes):
        asked.append([size() for size in sizes])
        return scratch(dev, *sizes) if room == "some" else None
    monkeypatch.setattr(kernels, "scratch", limited)
    torch.cuda.empty_cache()
    total = torch.cuda.get_device_properties(0).total_memory
    try:
        torch.cuda.set_per_process_memory_fraction((torch.cuda.memory_reserved() + 2 * blocks.SMALL) / total)
        got = blocks.attend_blocks(q, *store, 32000, out=out)
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
    assert got is out and len(asked) == 1 and asked[0][0] > 4 * blocks.SMALL and 0 < asked[0][1] <= blocks.SMALL
    check(got, q, store, 32000)
    monkeypatch.setattr(kernels, "scratch", scratch)
    assert torch.equal(blocks.attend_blocks(q, *store, 32000), want)
