"""The 8-bit block cache (blocks.py) against plain implementations.

Codes and scales are defined by float32 steps and compared bit for bit.  Read-back: codes times scales round once to float32 (product) and once
to the type.

Attention against float64 over what the storage holds.  Relative to the result's largest magnitude: scores are float32 sums of products of exact
codes (tensor cores keep 2^-22 or better of the largest term), a score of magnitude up to S then moves a weight by S 2^-20 relative; a weight
is rounded to fp16, at most 2^-11 relative; the sum of weights is not rounded with them, so all of them may be off one way: 2^-11 in all, plus 2^-11
for rows of bfloat16 tails rounded to fp16 under their power of two (exact for 8 of its 11 bits), plus the rounding of the result to its type,
eps / 2.  Bound: max |v| 2^-11 + eps / 2 |out| + 2^-14 max |v| for the rest.  The rest, for scores of some units: queries in fixed
point of 15 bits (bfloat16) or 22 (fp16) move a score by 2^-16 of its terms, exponentials have 2^-18, weights far below their row's reference are
off by 2^-29 of it each.  float32 tokens: scores up to 64 (in powers of two) are
added up with seven roundings of 2^-19, which moves a weight by 2^-16; twice that for the rest."""

import pytest
import torch

from blocks_util import attention, encode, values

pytestmark = pytest.mark.gpu

CODES = (torch.int8, torch.float8_e4m3fn)


def storage(b, h, cap, d, block, codes, dtype):
    z = torch.zeros
    cap = -(-cap // block) * block
    out = []
    for _ in range(2):
        out += [z(b, h, cap, d, dtype=torch.int8, device="cuda").view(codes), z(b, h, cap // block, device="cuda")]
    return out + [z(b, h, block, d, dtype=dtype, device="cuda") for _ in range(2)]


def rows(b, h, t, d, dtype, seed, std=0.5):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(b, h, t, d, generator=g) * torch.exp(std * torch.randn(b, h, t, 1, generator=g))
    return x.to(dtype).cuda()


def dense(store, length):
    """float64 on the CPU: what the storage stands for."""
    kc, ks, vc, vs, kt, vt = store
    n = kt.shape[2]
    cut = length // n * n
    return tuple(torch.cat([values(c[:, :, :cut].cpu(), s[:, :, :cut // n].cpu()), t[:, :, :length - cut].cpu().double()], dim=2) for c, s, t in ((kc, ks, kt), (vc, vs, vt)))


def filled(b, h, total, d, block, codes, dtype, seed=0, room=1):
    from mlx_turboquant_b200 import blocks
    store = storage(b, h, total + room, d, block, codes, dtype)
    assert blocks.write_blocks(rows(b, h, total, d, dtype, seed), rows(b, h, total, d, dtype, seed + 1), *store, 0) == total
    return store


def check_attention(got, q, k, v, scale, window=None, sinks=0):
    ref = attention(q.cpu(), k, v, scale, window, sinks)
    top = v.abs().amax().item()
    tol = torch.finfo(q.dtype).eps / 2 * ref.abs() + top * (2.0 ** -11 + 2.0 ** -14 if q.dtype is not torch.float32 else 2.0 ** -15)
    err = (got.double().cpu() - ref).abs()
    assert bool((err <= tol).all()), (float((err - tol).max()), float(err.max()), top)


# ---- writing, reading back ----------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("dtype", (torch.float16, torch.bfloat16, torch.float32))
@pytest.mark.parametrize("d,block", ((64, 16), (96, 32), (128, 64), (256, 128), (32, 16), (160, 64)))
def test_write_is_bit_exact_in_any_pieces(d, block, codes, dtype):
    from mlx_turboquant_b200 import blocks
    b, h, total = 2, 3, 5 * block + 7
    k, v = rows(b, h, total, d, dtype, 1), rows(b, h, total, d, dtype, 2)
    k[:, 0, :block] = 0                                                             # a block of zeros
    whole = storage(b, h, total, d, block, codes, dtype)
    assert blocks.write_blocks(k, v, *whole, 0) == total
    cut = total // block * block
    for c, s, t, x in ((whole[0], whole[1], whole[4], k), (whole[2], whole[3], whole[5], v)):
        rc, rs = encode(x[:, :, :cut].cpu().reshape(b, h, cut // block, block, d), codes)
        assert torch.equal(c[:, :, :cut].view(torch.int8).cpu(), rc.view(torch.int8).reshape(b, h, cut, d))
        assert torch.equal(s[:, :, :cut // block].cpu(), rs)
        assert torch.equal(t[:, :, :total - cut], x[:, :, cut:]) and not t[:, :, total - cut:].any()
    pieces = storage(b, h, total, d, block, codes, dtype)
    n = 0
    for size in (1, block - 2, 1, 0, block, 2 * block + 3, 1, 1, total):
        size = min(size, total - n)
        n = blocks.write_blocks(k[:, :, n:n + size], v[:, :, n:n + size], *pieces, n)      # (views: strided rows)
    assert n == total
    for i, (x, y) in enumerate(zip(whole, pieces)):
        if i < 4:
            assert torch.equal(x.view(torch.int8) if i % 2 == 0 else x, y.view(torch.int8) if i % 2 == 0 else y)
        else:
            assert torch.equal(x[:, :, :total - cut], y[:, :, :total - cut])


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("d,block,total", ((128, 64, 200), (96, 16, 47), (64, 32, 31), (256, 128, 256), (32, 16, 1)))
def test_read_back(d, block, total, codes):
    from mlx_turboquant_b200 import blocks
    for dtype in (torch.float16, torch.bfloat16, torch.float32):
        store = filled(2, 2, total, d, block, codes, dtype)
        ref = dense(store, total)
        for out in (None, torch.float16, torch.bfloat16, torch.float32):
            got = blocks.read_blocks(*store, total, dtype=out)
            for x, y in zip(got, ref):
                # codes times scales are rounded to float32 first
                assert torch.equal(x.cpu(), y.float().to(out or dtype)) and x.shape == (2, 2, total, d)


def test_rows_behind_the_last_token_stay(monkeypatch):
    """Capacity that is not reached, and tail rows behind the last token, are left as they were; both host paths do the same."""
    from mlx_turboquant_b200 import _lib, blocks
    k, v = rows(1, 2, 70, 64, torch.float16, 1), rows(1, 2, 70, 64, torch.float16, 2)
    a, z = (storage(1, 2, 320, 64, 32, torch.int8, torch.float16) for _ in range(2))
    for s in (a, z):
        for x in s:
            x.view(torch.uint8 if x.dtype is torch.int8 else x.dtype).fill_(7)
    blocks.write_blocks(k, v, *a, 0)
    monkeypatch.setattr(_lib, "_host", _lib._NoHost())
    blocks.write_blocks(k, v, *z, 0)
    for x, y in zip(a, z):
        assert torch.equal(x, y)
    assert bool((a[0][:, :, 64:] == 7).all()) and bool((a[1][:, :, 2:] == 7).all()) and bool((a[4][:, :, 6:] == 7).all())


def test_not_finite_and_tiny_blocks():
    from mlx_turboquant_b200 import blocks
    for bad in (float("nan"), float("inf")):
        k = rows(1, 1, 48, 64, torch.float32, 3)
        k[0, 0, 20, 5] = bad
        store = storage(1, 1, 48, 64, 16, torch.int8, torch.float32)
        blocks.write_blocks(k, k, *store, 0)
        got, _ = blocks.read_blocks(*store, 48)
        assert bool(got[:, :, 16:32].isnan().all()) and bool(got[:, :, :16].isfinite().all()) and bool(got[:, :, 32:].isfinite().all())
    k = rows(1, 1, 16, 64, torch.float32, 3, std=0) * 1e-39
    store = storage(1, 1, 16, 64, 16, torch.float8_e4m3fn, torch.float32)
    blocks.write_blocks(k, k, *store, 0)
    got, _ = blocks.read_blocks(*store, 16)
    assert bool(got.isfinite().all()) and float((got - k).abs().max()) <= float(k.abs().max())


# ---- attention ------------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("dtype", (torch.float16, torch.bfloat16, torch.float32))
@pytest.mark.parametrize("d,block", ((64, 32), (96, 16), (128, 64), (256, 128), (160, 64)))
def test_decode(d, block, codes, dtype):
    from mlx_turboquant_b200 import blocks
    for b, hq, h, total in ((1, 1, 1, 1), (2, 4, 2, 15), (1, 8, 2, block), (3, 7, 1, 3 * block + 9), (1, 18, 2, 1000)):
        store = filled(b, h, total, d, block, codes, dtype, seed=total)
        q = rows(b, hq, 1, d, dtype, 9, std=0)
        k, v = dense(store, total)
        check_attention(blocks.attend_blocks(q, *store, total), q, k, v, d ** -0.5)
        check_attention(blocks.attend_blocks(q, *store, total, scale=0.3), q, k, v, 0.3)


@pytest.mark.parametrize("d,block,codes,dtype", ((128, 64, torch.int8, torch.bfloat16), (64, 16, torch.float8_e4m3fn, torch.float16), (96, 32, torch.int8, torch.float16),
                                                 (256, 16, torch.float8_e4m3fn, torch.bfloat16), (224, 64, torch.int8, torch.float16)))
@pytest.mark.parametrize("total", (5, 64, 129, 1050))
def test_windows_and_sinks(d, block, codes, dtype, total):
    from mlx_turboquant_b200 import blocks
    store = filled(2, 2, total, d, block, codes, dtype, seed=3)
    q = rows(2, 6, 1, d, dtype, 5, std=0)
    k, v = dense(store, total)
    for window in (1, 3, 16, 33, 100, 1000, 5000):
        for sinks in (0, 1, 4, 17, 200):
            check_attention(blocks.attend_blocks(q, *store, total, window=window, sinks=sinks), q, k, v, d ** -0.5, window, sinks)


@pytest.mark.parametrize("d,block,codes,dtype", ((128, 64, torch.int8, torch.bfloat16), (64, 16, torch.float8_e4m3fn, torch.float16), (96, 32, torch.float8_e4m3fn, torch.bfloat16),
                                                 (256, 64, torch.int8, torch.float16), (128, 128, torch.int8, torch.float32)))
def test_several_tokens(d, block, codes, dtype):
    from mlx_turboquant_b200 import blocks
    for b, hq, h, total, t in ((1, 4, 1, 2, 2), (2, 8, 2, 77, 5), (1, 6, 2, 300, 130), (1, 3, 3, 200, 200), (2, 8, 8, 1100, 33), (1, 8, 2, 2500, 700), (1, 12, 1, 1337, 150)):
        store = filled(b, h, total, d, block, codes, dtype, seed=t)
        q = rows(b, hq, t, d, dtype, 5, std=0)
        k, v = dense(store, total)
        for window, sinks in ((None, 0), (1, 0), (20, 3), (64, 70), (300, 4)):
            check_attention(blocks.attend_blocks(q, *store, total, window=window, sinks=sinks), q, k, v, d ** -0.5, window, sinks)
    from mlx_turboquant_b200 import _lib
    assert _lib.lib().tq_device_status() == 0


@pytest.mark.parametrize("d,codes,dtype", ((128, torch.int8, torch.bfloat16), (64, torch.float8_e4m3fn, torch.float16), (96, torch.int8, torch.float16), (256, torch.float8_e4m3fn, torch.bfloat16)))
def test_pieces_of_a_prompt(d, codes, dtype):
    """Many row blocks: runs of key tiles that end inside them, whole ones in between, rows of several lanes and head groups."""
    from mlx_turboquant_b200 import _lib, blocks
    for b, hq, h, total, t in ((3, 8, 2, 1500, 600), (1, 20, 1, 900, 333), (2, 5, 5, 700, 700), (1, 1, 1, 4500, 4100), (9, 32, 8, 130, 40)):
        store = filled(b, h, total, d, 64, codes, dtype, seed=t)
        q = rows(b, hq, t, d, dtype, 5, std=0)
        k, v = dense(store, total)
        for window, sinks in ((None, 0), (100, 0), (333, 70)):
            check_attention(blocks.attend_blocks(q, *store, total, window=window, sinks=sinks), q, k, v, d ** -0.5, window, sinks)
    assert _lib.lib().tq_device_status() == 0


def repeated(store, n):
    return [x.repeat(n, *[1] * (x.dim() - 1)) for x in store]


def check_repeated(q, store, n, kd, vd, total, kernel=None, **kw):
    """n times the batch: every copy's results within the bounds, and by the kernel that is meant."""
    from mlx_turboquant_b200 import blocks
    got = None
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA], acc_events=True) as p:
        got = blocks.attend_blocks(q.repeat(n, 1, 1, 1), *store, total, **kw)
        torch.cuda.synchronize()
    names = " ".join(e.key for e in p.key_averages())
    assert kernel is None or not names or kernel in names, names          # (no names where the profiler cannot record)
    for x in got.chunk(n):
        check_attention(x, q, kd, vd, q.shape[-1] ** -0.5, kw.get("window"), kw.get("sinks", 0))


@pytest.mark.parametrize("d,codes,dtype", ((128, torch.int8, torch.bfloat16), (128, torch.float8_e4m3fn, torch.float16), (64, torch.float8_e4m3fn, torch.bfloat16), (96, torch.int8, torch.float16),
                                           (256, torch.int8, torch.bfloat16)))
def test_many_lanes_of_several_tokens(d, codes, dtype):
    """What takes the tile products: row blocks that fill a tile in part, one to eight heads on a KV head and more, tails of every length, windows and sinks."""
    for b, hq, h, total, t, n in ((1, 4, 1, 100, 60, 130), (1, 16, 2, 257, 33, 70), (2, 6, 2, 300, 130, 40), (1, 3, 3, 200, 200, 50), (1, 20, 2, 191, 17, 80), (1, 7, 1, 640, 64, 150)):
        store = filled(b, h, total, d, 64, codes, dtype, seed=t)
        q = rows(b, hq, t, d, dtype, 5, std=0)
        kd, vd = dense(store, total)
        many = repeated(store, n)
        check_repeated(q, many, n, kd, vd, total, "blocks_fa")
        for window, sinks in ((1, 0), (20, 3), (64, 70), (150, 4)):
            check_repeated(q, many, n, kd, vd, total, window=window, sinks=sinks)


@pytest.mark.parametrize("t", (40, 190))
@pytest.mark.parametrize("dtype", (torch.float16, torch.bfloat16))
def test_many_lanes_where_tokens_are_not_finite(dtype, t):
    from mlx_turboquant_b200 import blocks
    for total, at, side, bad in ((250, 247, 0, float("nan")), (250, 248, 1, float("nan")), (250, 246, 1, float("inf")), (200, 199, 1, float("-inf"))):
        store, q = filled(1, 2, total, 64, 128, torch.int8, dtype, room=0), rows(1, 8, t, 64, dtype, 3, std=0)
        kd, vd = dense(store, total)
        store[4 + side][:, :, at - 128, 7] = bad
        got = blocks.attend_blocks(q.repeat(64, 1, 1, 1), *repeated(store, 64), total)
        first = t - (total - at)
        for x in got.chunk(64):
            check_attention(x[:, :, :first], q[:, :, :first], kd[:, :, :at], vd[:, :, :at], 0.125)
            assert bool((~x[:, :, first:].isfinite()).any(-1).all())
        # behind every query's window, or behind the last token
        store = filled(1, 2, total, 64, 128, torch.int8, dtype, room=0)
        ref = blocks.attend_blocks(q.repeat(64, 1, 1, 1), *repeated(store, 64), total, window=5)
        low, cut = total - t + 1 - 5, 128
        for x, s in ((store[4], store[1]), (store[5], store[3])):
            x[:, :, total - cut:] = bad
            x[:, :, :max(low - cut, 0)] = bad
            if low >= cut:
                s[:, :, 0] = float("nan")
        assert torch.equal(blocks.attend_blocks(q.repeat(64, 1, 1, 1), *repeated(store, 64), total, window=5), ref)


def test_query_magnitudes():
    """bfloat16 queries of very different rows, outside the fp16 range."""
    from mlx_turboquant_b200 import blocks
    store = filled(1, 1, 500, 128, 64, torch.int8, torch.bfloat16)
    store[1].mul_(2.0 ** -60)
    tail = store[4]
    tail.mul_(2.0 ** -60)
    k, v = dense(store, 500)
    for t in (1, 20, 200):
        q = (rows(1, 4, t, 128, torch.float32, 2, std=0) * torch.exp2(60 - 30 * torch.rand(1, 4, t, 1).cuda())).bfloat16()
        check_attention(blocks.attend_blocks(q, *store, 500), q, k, v, 128 ** -0.5)
        if t > 1:
            check_repeated(q, repeated(store, 150), 150, k, v, 500, "blocks_fa")


@pytest.mark.parametrize("dtype", (torch.float16, torch.bfloat16, torch.float32))
@pytest.mark.parametrize("length", (0, 5, 62, 63, 64, 200, 1000))
def test_the_new_token_joins(length, dtype):
    """attend_blocks(new=...) leaves the storage as write_blocks does and attends over it, also where the token completes a block."""
    from mlx_turboquant_b200 import blocks
    args = (2, 2, max(length, 1), 128, 64, torch.int8, dtype)
    a, z = filled(*args, seed=4, room=64), filled(*args, seed=4, room=64)
    kv = torch.randn(2, 1, 4, 128, device="cuda").to(dtype).transpose(1, 2)
    k, v = kv[:, :2], kv[:, 2:]
    q = rows(2, 8, 1, 128, dtype, 6, std=0)
    got = blocks.attend_blocks(q, *a, length, new=(k, v))
    assert blocks.write_blocks(k, v, *z, length) == length + 1
    for x, y in zip(a, z):
        assert torch.equal(x, y)
    kd, vd = dense(z, length + 1)
    check_attention(got, q, kd, vd, 128 ** -0.5)


def test_the_new_token_joins_many_heads():
    """Several groups of query heads a lane, of which one appends, over runs and clusters of CTAs."""
    from mlx_turboquant_b200 import blocks
    for b, hq, h, length in ((1, 20, 1, 5000), (3, 32, 2, 700), (2, 17, 1, 37), (40, 16, 1, 900)):
        a, z = (filled(b, h, length, 128, 64, torch.int8, torch.bfloat16, seed=2, room=64) for _ in range(2))
        k, v, q = rows(b, h, 1, 128, torch.bfloat16, 4), rows(b, h, 1, 128, torch.bfloat16, 5), rows(b, hq, 1, 128, torch.bfloat16, 6, std=0)
        got = blocks.attend_blocks(q, *a, length, new=(k, v), window=4000, sinks=3)
        blocks.write_blocks(k, v, *z, length)
        assert all(torch.equal(x, y) for x, y in zip(a, z))
        kd, vd = dense(z, length + 1)
        check_attention(got, q, kd, vd, 128 ** -0.5, 4000, 3)


def test_scales_and_windows_at_their_ends():
    from mlx_turboquant_b200 import blocks
    for dtype in (torch.bfloat16, torch.float32):
        store = filled(2, 2, 300, 64, 32, torch.int8, dtype)
        k, v = dense(store, 300)
        for t in (1, 3, 150):
            q = rows(2, 8, t, 64, dtype, 1, std=0)
            for scale in (0.0, -0.2):
                check_attention(blocks.attend_blocks(q, *store, 300, scale=scale), q, k, v, scale)
            assert torch.equal(blocks.attend_blocks(q, *store, 300, window=1 << 70, sinks=1 << 70), blocks.attend_blocks(q, *store, 300))
            assert torch.equal(blocks.attend_blocks(q, *store, 300, window=1 << 40, sinks=1 << 40), blocks.attend_blocks(q, *store, 300))


def test_lanes_in_several_rounds():
    """More expanded tiles than the workspace is given: some lanes after the others."""
    total, t, n = 16500, 130, 70
    store = filled(1, 1, total, 128, 64, torch.int8, torch.bfloat16)
    q = rows(1, 4, t, 128, torch.bfloat16, 3, std=0)
    from mlx_turboquant_b200 import blocks
    got = blocks.attend_blocks(q.expand(n, -1, -1, -1), *repeated(store, n), total)
    k, v = dense(store, total)
    for i in (0, n // 2, n - 1):
        check_attention(got[i:i + 1], q, k, v, 128 ** -0.5)
    tol = 2 * (2.0 ** -11 + 2.0 ** -14 + 2.0 ** -8) * float(v.abs().max())           # (each within the bound of one result)
    assert float((got.float() - got[:1].float()).abs().max()) <= tol


def test_hidden_values_do_not_count():
    """NaN and infinities in tokens that no query sees: behind the window in blocks and in the tail, behind the last token."""
    from mlx_turboquant_b200 import blocks
    for dtype in (torch.float16, torch.bfloat16, torch.float32):
        for total, window in ((300, 40), (310, 5), (64, 64), (20, 3)):
            store = filled(1, 2, total, 128, 64, torch.int8, dtype, seed=1)
            q = rows(1, 8, 1, 128, dtype, 2, std=0)
            ref = blocks.attend_blocks(q, *store, total, window=window, sinks=2).clone()
            low = total - window
            for t, s in ((store[4], store[1]), (store[5], store[3])):
                cut = total // 64 * 64
                if low > cut:
                    t[:, :, :low - cut] = float("nan")
                    if cut == 0:                                                     # (the sinks sit in the tail)
                        t[:, :, :2] = 0.5
                t[:, :, total - cut:] = float("inf")
                s[:, :, 1:low // 64] = float("nan")
                s[:, :, cut // 64:] = float("nan")
            if total == 20:
                ref = blocks.attend_blocks(q, *store, total, window=window, sinks=2)
                assert bool(ref.isfinite().all())
            else:
                assert torch.equal(blocks.attend_blocks(q, *store, total, window=window, sinks=2), ref)


@pytest.mark.parametrize("t", (5, 40, 190))
@pytest.mark.parametrize("dtype", (torch.float16, torch.bfloat16, torch.float32))
def test_what_is_not_finite_reaches_those_who_see_it(dtype, t):
    """A NaN or an infinity in one token: not finite for the queries that see it, the others' results as without it.  (Not the same bits: the rows of a warp
    move their reference maxima together, which a NaN does not ask for, and weights are rounded to fp16 from another reference.  Each is within the bound.)"""
    from mlx_turboquant_b200 import blocks
    for total, at, side, bad in ((250, 247, 0, float("nan")), (250, 248, 1, float("nan")), (250, 246, 1, float("inf")), (200, 199, 1, float("-inf"))):
        k, v = rows(1, 2, total, 64, dtype, 1), rows(1, 2, total, 64, dtype, 2)
        q = rows(1, 8, t, 64, dtype, 3, std=0)
        store = storage(1, 2, total, 64, 128, torch.int8, dtype)
        blocks.write_blocks(k, v, *store, 0)
        kd, vd = dense(store, total)
        for window in (None, 3):
            tail = store[4 + side]
            kept = tail.clone()
            tail[:, :, at - 128, 7] = bad
            got = blocks.attend_blocks(q, *store, total, window=window)
            tail.copy_(kept)
            pos = torch.arange(total - t, total)
            sees = (pos >= at) & ((pos - at < window) if window else True)
            assert bool(sees.any())
            first = int(sees.nonzero()[0])
            if first > 0:
                check_attention(got[:, :, :first], q[:, :, :first], kd[:, :, :total - t + first], vd[:, :, :total - t + first], 0.125, window)
            last = int(sees.nonzero()[-1]) + 1
            if last < t:
                check_attention(got[:, :, last:], q[:, :, last:], kd, vd, 0.125, window)
            hit = got[:, :, sees]
            assert bool((~hit.isfinite()).any(-1).all())


def test_extreme_scales():
    """Scales from 2^-60 to 2^60 of the values, and scores that grow along the sequence."""
    from mlx_turboquant_b200 import blocks
    for dtype in (torch.bfloat16, torch.float32):
        total = 1000
        grow = torch.exp2(torch.linspace(-60, 60, total)).view(1, 1, total, 1).cuda()
        k, v = rows(1, 1, total, 64, dtype, 1), (rows(1, 1, total, 64, torch.float32, 2) * grow).to(dtype)
        store = storage(1, 1, total, 64, 16, torch.int8, dtype)
        blocks.write_blocks(k, v, *store, 0)
        q = rows(1, 4, 1, 64, dtype, 3, std=0)
        kd, vd = dense(store, total)
        check_attention(blocks.attend_blocks(q, *store, total), q, kd, vd, 0.125)
        k = (rows(1, 1, total, 64, torch.float32, 1) + q[:, :1].float() * torch.linspace(0, 3, total, device="cuda").view(1, 1, total, 1)).to(dtype)
        store = storage(1, 1, total, 64, 16, torch.int8, dtype)
        blocks.write_blocks(k, v, *store, 0)
        kd, vd = dense(store, total)
        check_attention(blocks.attend_blocks(q, *store, total), q, kd, vd, 0.125)


def test_strided_queries_outs_and_the_other_host_path(monkeypatch):
    from mlx_turboquant_b200 import _lib, blocks
    store = filled(2, 2, 300, 128, 64, torch.int8, torch.bfloat16)
    q = torch.randn(2, 3, 8, 128, device="cuda").bfloat16().transpose(1, 2)
    a = blocks.attend_blocks(q, *store, 300, window=100, sinks=4)
    out = torch.empty(2, 8, 3, 128, device="cuda", dtype=torch.bfloat16)
    assert blocks.attend_blocks(q, *store, 300, window=100, sinks=4, out=out) is out and torch.equal(out, a)
    odd = torch.randn(2, 8, 3, 131, device="cuda").bfloat16()[..., 1:129].copy_(q)
    assert torch.equal(blocks.attend_blocks(odd, *store, 300, window=100, sinks=4), a)
    monkeypatch.setattr(_lib, "_host", _lib._NoHost())
    assert torch.equal(blocks.attend_blocks(q, *store, 300, window=100, sinks=4), a)
    assert torch.equal(blocks.attend_blocks(q, *store, 300, window=None), blocks.attend_blocks(q, *store, 300, window=300))


def test_long_cache_offsets_pass_32_bits():
    """Lanes whose codes lie past 2^31 bytes; results do not depend on how the work is split."""
    from mlx_turboquant_b200 import blocks
    b, h, total, d = 9, 8, 262144, 128                                              # 2.4 GB a side
    store = storage(b, h, total, d, 128, torch.int8, torch.float16)
    g = torch.Generator(device="cuda").manual_seed(1)
    for i in (0, 2):
        store[i].copy_(torch.randint(-127, 128, (1, 1, total, d), generator=g, device="cuda", dtype=torch.int8).expand(b, h, total, d))
        store[i + 1].copy_((torch.rand(1, 1, total // 128, generator=g, device="cuda") + 0.5).expand(b, h, total // 128) / 100)
    q = torch.randn(1, 1, 1, d, device="cuda").half().expand(b, h, 1, d)
    got = blocks.attend_blocks(q, *store, total)
    k, v = dense([x[:1, :1] for x in store], total)
    check_attention(got[:1, :1], q[:1, :1], k, v, d ** -0.5)
    assert float((got.float() - got[:1, :1].float()).abs().max()) <= 2.0 ** -10 * float(v.abs().max())
    again = blocks.attend_blocks(q, *store, total)
    assert torch.equal(got, again)


def test_refusals():
    from mlx_turboquant_b200 import blocks
    store = filled(1, 2, 100, 64, 32, torch.int8, torch.float16)
    q = rows(1, 4, 1, 64, torch.float16, 1)
    new = rows(1, 2, 1, 64, torch.float16, 1)
    for bad in (dict(window=0), dict(window=-3), dict(sinks=-1)):
        with pytest.raises(ValueError):
            blocks.attend_blocks(q, *store, 100, **bad)
    with pytest.raises(ValueError):
        blocks.attend_blocks(q[:, :3], *store, 100)
    with pytest.raises(ValueError):
        blocks.attend_blocks(q, *store, 0)
    with pytest.raises(ValueError):
        blocks.attend_blocks(rows(1, 4, 3, 64, torch.float16, 1), *store, 2)
    with pytest.raises(ValueError):
        blocks.attend_blocks(rows(1, 4, 2, 64, torch.float16, 1), *store, 100, new=(new, new))
    with pytest.raises(ValueError):
        blocks.attend_blocks(q, *store, 200)                                         # more than the storage holds
    with pytest.raises(TypeError):
        blocks.attend_blocks(q.bfloat16(), *store, 100)
    with pytest.raises(TypeError):
        blocks.write_blocks(new.bfloat16(), new.bfloat16(), *store, 100)
    with pytest.raises(ValueError):
        blocks.write_blocks(rows(1, 2, 200, 64, torch.float16, 1), rows(1, 2, 200, 64, torch.float16, 1), *store, 100)
    with pytest.raises(ValueError):
        blocks.write_blocks(new[:, :1], new[:, :1], *store, 100)
    with pytest.raises(ValueError):
        blocks.read_blocks(*store, 1000)
    with pytest.raises(ValueError):
        blocks.read_blocks(store[0][:, :, :32], *store[1:], 30)                       # not contiguous, and the scales disagree
    with pytest.raises(TypeError):
        blocks.read_blocks(store[0].view(torch.uint8), *store[1:], 30)
    with pytest.raises(RuntimeError, match="CUDA"):
        blocks.read_blocks(store[0].cpu(), *store[1:], 30)
    with pytest.raises(RuntimeError, match="backward"):
        blocks.attend_blocks(q.clone().requires_grad_(), *store, 100)
    with pytest.raises(NotImplementedError):
        blocks.read_blocks(*storage(1, 1, 16, 48, 16, torch.int8, torch.float16), 3)


def test_captured_graphs_do_not_share_scratch():
    """Two graphs, captured on one stream, replayed on two at once."""
    from mlx_turboquant_b200 import blocks
    store = filled(1, 2, 4000, 128, 64, torch.int8, torch.bfloat16)
    qs = [rows(1, 16, 1, 128, torch.bfloat16, s, std=0) for s in (1, 2)]
    want = [blocks.attend_blocks(q, *store, 4000).clone() for q in qs]
    graphs, outs = [], []
    for q in qs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(blocks.attend_blocks(q, *store, 4000))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o, w)
