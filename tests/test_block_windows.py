"""Block caches with a window for callers that run their own attention: what update_and_fetch returns, and the mask over it."""

import pytest
import torch

from blocks_util import attention
from mlx_turboquant_b200 import BlockKVCache
from mlx_turboquant_b200.blocks import window_mask


def seen(offset, n, window, sinks):
    """By definition: (n, offset + n)"""
    return torch.tensor([[j <= p and (p - j < window or j < sinks) for j in range(offset + n)] for p in range(offset, offset + n)])


@pytest.mark.parametrize("window", (1, 2, 5, 16, 40))
@pytest.mark.parametrize("sinks", (0, 1, 4, 30))
def test_the_mask_is_the_definition(window, sinks):
    c = BlockKVCache(64, 1, window=window, sinks=sinks)
    for offset in (0, 1, 4, 15, 16, 33, 60):
        for n in (1, 2, 7, 30):
            want = seen(offset, n, window, sinks)
            low = max(0, offset - window + 1)
            kept = [*range(min(sinks, low)), *range(low, offset + n)]
            assert not want[:, [j for j in range(offset + n) if j not in kept]].any()             # nothing that some query sees is left out
            assert torch.equal(window_mask(offset, n, window, sinks, "cpu"), want[:, kept])
            c.offset = offset
            if n == 1:
                assert c.make_mask(1) is None and bool(want[:, kept].all())
            elif bool((want == seen(offset, n, offset + n, 0)).all()):                             # the window hides nothing
                assert c.make_mask(n) == "causal" and len(kept) == offset + n


def test_the_models_own_size_names_the_window():
    c = BlockKVCache(64, 1, window=124, sinks=4)
    assert c.make_mask(5, window_size=128) == "causal" and c.make_mask(5, window_size=124) == "causal" and c.make_mask(1, window_size=128) is None
    for other in (4, 100, 120, 132):
        with pytest.raises(NotImplementedError):
            c.make_mask(5, window_size=other)
    with pytest.raises(NotImplementedError):
        BlockKVCache(64, 1).make_mask(5, window_size=128)


def tokens(b, h, t, d, dtype, seed):
    return torch.randn(b, h, t, d, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks,block", ((100, 0, 32), (100, 4, 32), (33, 40, 16), (1, 0, 16), (64, 64, 64)))
@pytest.mark.parametrize("dtype", (torch.float16, torch.bfloat16, torch.float32))
def test_dense_rows_and_their_mask(window, sinks, block, dtype):
    """A life of a cache through update_and_fetch: what a cache without a window returns, at the tokens that the mask's columns stand for."""
    b, h, hq, d = 2, 2, 4, 64
    c, every = BlockKVCache(d, h, "int8", block, window, sinks), BlockKVCache(d, h, "int8", block)
    for i, t in enumerate((7, 200, 1, 1, 300, 5) + (1,) * 70 + (64, 3) + (1,) * 40):
        k, v, q = tokens(b, h, t, d, dtype, 3 * i), tokens(b, h, t, d, dtype, 3 * i + 1), tokens(b, hq, t, d, dtype, 3 * i + 2)
        offset, mask, array = c.offset, c.make_mask(t), c.make_mask(t, return_array=True)
        got, all_k = c.update_and_fetch(k, v), every.update_and_fetch(k, v)
        low = max(0, offset - window + 1)
        kept = [*range(min(sinks, low)), *range(low, offset + t)]
        for x, y in zip(got, all_k):
            assert x.dtype is dtype and torch.equal(x, y[:, :, kept])
        want = seen(offset, t, window, sinks)[:, kept]
        assert array.device == k.device and torch.equal(array.cpu(), want)
        if isinstance(mask, torch.Tensor):
            assert torch.equal(mask, array)
        elif mask is None:
            assert t == 1 and bool(want.all())
        else:
            assert torch.equal(want, seen(offset, t, offset + t, 0))
        if i % 9 == 0:
            # the caller's own attention over them is what attend computes (its bound as test_blocks_gpu derives it, and float64 here)
            kd, vd = got[0].double().cpu(), got[1].double().cpu()
            s = (q.double().cpu() @ kd.repeat_interleave(hq // h, 1).transpose(-1, -2) * d ** -0.5).masked_fill(~want, float("-inf"))
            ref = torch.softmax(s, -1) @ vd.repeat_interleave(hq // h, 1)
            held = attention(q.cpu(), *(x.double().cpu() for x in all_k), d ** -0.5, window, sinks)
            assert torch.allclose(ref, held, rtol=1e-12, atol=1e-12)
            # (the dense rows are rounded to the type once more than what attend reads: half a step of each value, and of each key in the scores)
            eps = torch.finfo(dtype).eps / 2
            terms = float((q.double().cpu().abs() @ kd.abs().repeat_interleave(hq // h, 1).transpose(-1, -2)).max()) * d ** -0.5
            top = float(vd.abs().max())
            tol = eps * ref.abs() + top * (2.0 ** -11 + 2.0 ** -14 + eps + 2 * eps * terms)
            assert bool(((c.attend(q).double().cpu() - ref).abs() <= tol).all())
    assert c._dropped > 0 and every.offset == c.offset


@pytest.mark.gpu
@pytest.mark.parametrize("keep", (0, 4))
def test_the_caller_by_both_routes(keep):
    """A model whose layers have sliding windows, patched: packed and dense, a prompt in pieces and steps."""
    from mlx_turboquant_b200 import apply_turboquant
    from mlx_turboquant_b200.consumer import LlamaShaped, ModelArgs

    class RotatingKVCache:
        def __init__(self):
            self.max_size, self.keep = 48, keep

    class Model(LlamaShaped):
        def make_cache(self):
            return [RotatingKVCache() for _ in self.layers]

    args = ModelArgs(hidden_size=256, num_hidden_layers=3, num_attention_heads=8, num_key_value_heads=4, head_dim=128, intermediate_size=512, vocab_size=512)
    m = apply_turboquant(Model(args, dtype=torch.bfloat16, seed=5, std=0.05), auto_detect_outliers=False, block_cache="int8")
    packed, dense, whole = m.make_cache(), m.make_cache(), [BlockKVCache(128, 4) for _ in range(3)]
    assert all((c.window, c.sinks) == (48 - keep, keep) for c in packed + dense)
    assert dense[0].make_mask(60, window_size=48).shape == (60, 60)
    prompt = torch.randint(0, 512, (2, 190), generator=torch.Generator().manual_seed(1)).cuda()
    apart = []
    for first, last in ((0, 100), (100, 101), (101, 160), (160, 161), (161, 162), (162, 190)):
        a, z, w = (m(prompt[:, first:last], cache=c, packed=p).float() for c, p in ((packed, True), (dense, False), (whole, True)))
        # bfloat16 activations: both routes round every layer's result, 2^-8 of it; six of them in a row and the logits' sum over 256
        assert float((a - z).abs().max()) <= 0.06 * float(z.abs().max())
        apart.append(float((a - w).abs().max()) / float(z.abs().max()))
    assert max(apart) > 0.06                                # (the windows do hide something here)
    assert dense[0].offset == 190


@pytest.mark.parametrize("head_dim", (80, 112, 288, 48))
def test_head_dims_without_kernels_leave_the_layers_as_they_were(head_dim):
    from test_block_cache import _model, _RotatingKVCache
    from mlx_turboquant_b200 import apply_turboquant
    from mlx_turboquant_b200.patch import KVCache
    m = _model(lambda i: _RotatingKVCache() if i == 2 else KVCache())
    with pytest.warns(UserWarning, match="no kernels for head_dim"):
        apply_turboquant(m, head_dim=head_dim, skip_layers=[0], block_cache="int8")
    assert [type(c).__name__ for c in m.make_cache()] == ["KVCache", "TurboQuantKVCache", "_RotatingKVCache", "TurboQuantKVCache"]
    assert "block_cache" not in m._turboquant_config


def test_what_a_call_wants_and_what_it_makes_do_with():
    """Host logic of the library: no GPU is asked."""
    import ctypes as C
    from mlx_turboquant_b200 import _lib
    lib = _lib.lib()
    for b, h, hq, d, total, t, dtype in ((1, 8, 32, 128, 16384, 2048, 1), (40, 8, 32, 64, 700, 64, 0), (3, 1, 4, 256, 5000, 300, 1), (1, 1, 1, 96, 9000, 1, 0), (2, 2, 4, 128, 300, 5, 2)):
        a = _lib.BlocksAttendArgs()
        a.store = _lib.BlockStore(b, h, d, 64, 0, dtype, *(4096,) * 6, -(-total // 64) * 64, total)
        a.n_q_heads, a.t_q, a.q, a.out, a.scale = hq, t, _lib.NewRows(4096, 0, 128, 128), 4096, 1.0
        most = lib.tq_blocks_attend_workspace(C.byref(a))
        a.workspace_bytes = (1 << 64) - 1
        way, room, last = lib.tq_blocks_attend_choice(C.byref(a)), most, None
        assert way > 0 and lib.tq_blocks_attend_workspace_within(C.byref(a), most) == most
        while room:
            a.workspace_bytes = room
            assert room != most or lib.tq_blocks_attend_choice(C.byref(a)) == way
            last, room = room, lib.tq_blocks_attend_workspace_within(C.byref(a), room - 1)
            assert room < last
        a.workspace_bytes = 0
        assert lib.tq_blocks_attend_choice(C.byref(a)) in (1, 2, 4)
        a.workspace = 4100
        assert lib.tq_blocks_attend_choice(C.byref(a)) == -1                          # 256-byte aligned


def test_storage_from_inference_mode_is_written_to_outside_of_it():
    """A prompt under torch.inference_mode(), steps under torch.no_grad(): what the window has passed is dropped in place.  (The storage's own bookkeeping; no kernel runs.)"""
    c = BlockKVCache(32, 1, "int8", 16, window=20, sinks=3)
    row = torch.zeros(1, 1, 1, 32)
    with torch.inference_mode():
        c._reserve(row.expand(1, 1, 600, 32), 600)
    cap = c._store[0].shape[2]
    for t in c._store:
        assert not t.is_inference()
        t.view(torch.uint8 if t.element_size() == 1 else t.dtype).zero_()
    c.offset = cap + 15
    c._store[0][0, 0, :, 0] = torch.arange(cap) // 16 % 100
    c._store[1][0, 0] = torch.arange(cap // 16).float()
    with torch.no_grad():
        c._reserve(row, 1)
    low = c.offset - 20 + 1
    assert c._dropped == low // 16 * 16 - 16 and c._store[0].shape[2] == cap
    kept = [0, *range(low // 16, cap // 16)]                # the sinks' block, and the window's
    assert c._store[1][0, 0, :len(kept)].tolist() == kept and c._store[0][0, 0, :16 * len(kept):16, 0].tolist() == [k % 100 for k in kept]


@pytest.mark.gpu
def test_a_windowed_life_across_modes():
    c, z = (BlockKVCache(64, 2, "int8", 32, 50, 4) for _ in range(2))
    x = tokens(1, 2, 1400, 64, torch.float16, 1)
    q = tokens(1, 4, 1, 64, torch.float16, 2)
    with torch.inference_mode():
        c.update(x[:, :, :1000], -x[:, :, :1000])
    z.update(x[:, :, :1000], -x[:, :, :1000])
    for i in range(1000, 1400):
        k = x[:, :, i:i + 1]
        assert torch.equal(c.decode_step(q, k, -k), z.decode_step(q, k, -k))
    assert c._dropped > 0
    with torch.inference_mode():
        y = BlockKVCache(64, 2, "int8", 32, 50, 4)
        y.state, y.meta_state = c.state, c.meta_state
    for i in range(400):
        k = x[:, :, i:i + 1]
        assert torch.equal(y.decode_step(q, k, -k), c.decode_step(q, k, -k))


def test_the_callers_dense_route_asks_a_windowed_cache_for_its_mask():
    """On the CPU, with a cache that keeps everything and returns what a windowed one would: the same logits whatever pieces the tokens come in."""
    from mlx_turboquant_b200.consumer import LlamaShaped, ModelArgs

    class Windowed:
        window, sinks = 6, 2

        def __init__(self):
            self.offset, self.kv = 0, None

        def make_mask(self, n):
            return None if n == 1 else "causal" if self.offset + n - self.window <= self.sinks else window_mask(self.offset, n, self.window, self.sinks, "cpu")

        def update_and_fetch(self, k, v):
            low = max(0, self.offset - self.window + 1)
            self.kv = (k, v) if self.kv is None else tuple(torch.cat(x, 2) for x in zip(self.kv, (k, v)))
            self.offset += k.shape[2]
            return tuple(torch.cat([x[:, :, :min(self.sinks, low)], x[:, :, low:]], 2) for x in self.kv)

    m = LlamaShaped(ModelArgs(hidden_size=64, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, head_dim=32, intermediate_size=64, vocab_size=64), dtype=torch.float32, device="cpu", std=0.2)
    tok = torch.randint(0, 64, (2, 25), generator=torch.Generator().manual_seed(3))
    whole = m(tok, cache=[Windowed() for _ in range(2)], packed=False)
    assert float((whole - m(tok)).abs().max()) > 1e-2                       # (the window does hide something)
    for pieces in ((1,) * 25, (7, 1, 12, 5), (3, 22), (20, 1, 1, 3)):
        cache, at, got = [Windowed() for _ in range(2)], 0, []
        for n in pieces:
            got.append(m(tok[:, at:at + n], cache=cache, packed=False))
            at += n
        assert torch.allclose(torch.cat(got, 1), whole, atol=2e-4)
