"""BlockKVCache, its place in apply_turboquant and in the Llama-shaped caller; refusals that need no GPU."""

import ctypes as C

import pytest
import torch

from blocks_util import attention, encode
from mlx_turboquant_b200 import BlockKVCache, apply_turboquant
from mlx_turboquant_b200.patch import KVCache

TINY = dict(hidden_size=256, num_hidden_layers=3, num_attention_heads=8, num_key_value_heads=4, head_dim=128, intermediate_size=512, vocab_size=512)


# ---- without a GPU ------------------------------------------------------------------------------------------------------------------

def test_arguments():
    for bad in (dict(codes="int4"), dict(block=48), dict(window=0), dict(sinks=-1), dict(sinks=4)):
        with pytest.raises(ValueError):
            BlockKVCache(**bad)
    c = BlockKVCache(window=128, sinks=4)
    assert c.empty() and c.size() == 0 and c.nbytes == 0 and not c.is_trimmable() and c.state == (None,) * 6
    assert c.make_mask(1) is None and c.make_mask(5) == "causal" and c.make_mask(5, window_size=128) == "causal"
    with pytest.raises(NotImplementedError):
        c.make_mask(5, window_size=64)
    with pytest.raises(ValueError):
        c.attend(torch.zeros(1, 1, 1, 128))
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        c.update(torch.zeros(1, 1, 3, 128), torch.zeros(1, 1, 3, 128))
    with pytest.raises(NotImplementedError):
        c.update_and_fetch(torch.zeros(1, 1, 3, 128), torch.zeros(1, 1, 3, 128))


def test_frequencies():
    from mlx_turboquant_b200 import rope
    f, m = rope.frequencies(8, 10000.0, device="cpu")
    assert m == 1.0 and f.dtype == torch.float64 and torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-12)
    assert torch.equal(rope.frequencies(8, 10000.0, {"rope_type": "linear", "factor": 4}, "cpu")[0], f / 4)
    g, _ = rope.frequencies(128, 500000.0, {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original_max_position_embeddings": 8192}, "cpu")
    b = rope.frequencies(128, 500000.0, device="cpu")[0]
    turns = 8192 * b / (2 * torch.pi)
    assert torch.equal(g[turns > 4], b[turns > 4]) and torch.allclose(g[turns < 1], b[turns < 1] / 8) and bool(((g <= b) & (g >= b / 8 * (1 - 1e-12))).all())
    y, m = rope.frequencies(128, 10000.0, {"type": "yarn", "factor": 16.0}, "cpu")
    b = rope.frequencies(128, 10000.0, device="cpu")[0]
    assert y[0] == b[0] and torch.isclose(y[-1], b[-1] / 16) and m == pytest.approx(0.1 * torch.log(torch.tensor(16.0)).item() + 1)
    for bad in (dict(dims=7), dict(dims=0), dict(dims=8, scaling={"rope_type": "nope"})):
        with pytest.raises(ValueError):
            rope.frequencies(**{"device": "cpu", **bad})


def test_scalings_that_are_not_understood():
    from mlx_turboquant_b200 import rope
    for bad in ({"rope_type": "linear"}, {"rope_type": "linear", "factor": 0.0}, {"rope_type": "llama3", "factor": None}, {"rope_type": "yarn", "factor": 4.0, "mscale": 1.0},
                {"rope_type": "yarn", "factor": 4.0, "truncate": False}, {"rope_type": "default", "factor": 2.0}, {"rope_type": "longrope", "factor": 4.0}):
        with pytest.raises(ValueError):
            rope.frequencies(16, scaling=bad, device="cpu")
    rope.frequencies(16, scaling={"rope_type": "yarn", "factor": 4.0, "attention_factor": None}, device="cpu")


def test_head_dims_that_have_no_kernel():
    from mlx_turboquant_b200 import BlockKVCache
    for d in (0, -32, 80, 288):
        with pytest.raises(ValueError):
            BlockKVCache(head_dim=d)


def test_library_refuses_bad_arguments():
    """Host checks in front of any launch; the addresses are never followed."""
    from mlx_turboquant_b200 import _lib
    lib = _lib.lib()
    good = dict(batch=1, n_kv_heads=2, d=128, block=64, code_type=0, dtype=1, k_codes=4096, v_codes=4096, k_scales=4096, v_scales=4096, k_tail=4096, v_tail=4096, capacity=256, length=100)
    rows = _lib.NewRows(4096, 0, 128, 128)

    def store(**kw):
        return _lib.BlockStore(**{**good, **kw})

    for kw, code in ((dict(block=48), -1), (dict(capacity=250), -1), (dict(length=400), -1), (dict(length=-1), -1), (dict(dtype=7), -1), (dict(code_type=2), -1), (dict(d=48), -2),
                     (dict(d=512), -2), (dict(k_codes=0), -1), (dict(v_tail=0), -1), (dict(k_codes=4100), -2)):
        assert lib.tq_blocks_read(C.byref(store(**kw)), 4096, 4096, 1, None) == code, kw
        assert lib.tq_blocks_write(C.byref(store(**kw)), C.byref(rows), C.byref(rows), 1, None) == code, kw
        a = _lib.BlocksAttendArgs()
        a.store, a.n_q_heads, a.t_q, a.q, a.out = store(**kw), 2, 1, rows, 4096
        assert lib.tq_blocks_attend(C.byref(a), None) == code, kw
    s = store()
    assert lib.tq_blocks_write(C.byref(s), C.byref(rows), C.byref(rows), 0, None) == 0                            # nothing to do
    assert lib.tq_blocks_write(C.byref(s), C.byref(rows), C.byref(rows), 300, None) == -1                         # no room
    assert lib.tq_blocks_write(C.byref(s), C.byref(_lib.NewRows(4098, 0, 128, 128)), C.byref(rows), 1, None) == -2
    assert lib.tq_blocks_write(C.byref(s), C.byref(_lib.NewRows(4096, 0, 132, 128)), C.byref(rows), 1, None) == -2
    assert lib.tq_blocks_read(C.byref(s), 4096, 4104, 1, None) == -2
    assert lib.tq_blocks_read(C.byref(s), 4096, 4096, 5, None) == -1

    def attend(**kw):
        a = _lib.BlocksAttendArgs()
        a.store, a.n_q_heads, a.t_q, a.q, a.out, a.scale = store(length=kw.pop("length", 100)), 4, 1, rows, 4096, 1.0
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.tq_blocks_attend(C.byref(a), None)

    assert attend(n_q_heads=3) == -1 and attend(t_q=101) == -1 and attend(window=-1) == -1 and attend(sinks=-1) == -1 and attend(out=0) == -1 and attend(out=4100) == -2
    assert attend(k_new=rows) == -1                                                                                # keys without values
    assert attend(k_new=rows, v_new=rows, t_q=2) == -1 and attend(k_new=rows, v_new=rows, length=127) == -1        # more than one query; completes a block
    assert attend(t_q=0) == 0
    r = _lib.RotaryArgs()
    r.dtype, r.batch, r.d, r.dims, r.length, r.freqs = 1, 1, 64, 64, 4, 4096
    r.part[0] = _lib.RotaryRows(4096, 0, 64, 64, 4096, 1)
    for field, value in (("dims", 7), ("dims", 66), ("dims", 0), ("dtype", 4), ("freqs", 0), ("d", 0)):
        b = _lib.RotaryArgs.from_buffer_copy(r)
        setattr(b, field, value)
        assert lib.tq_rotary(C.byref(b), None) == -1, field
    r.length = 0
    assert lib.tq_rotary(C.byref(r), None) == 0


class _Rotating:
    """A sliding-window model's default cache, as mlx-lm has it: max_size tokens in all, the first `keep` among them."""

    def __init__(self, max_size=128, keep=4):
        self.max_size, self.keep = max_size, keep


class _RotatingKVCache(_Rotating):
    pass


def _model(default):
    class Layer:
        self_attn = object()

    class Model:
        class args:
            hidden_size, head_dim, num_key_value_heads, num_hidden_layers, num_attention_heads = 256, 64, 4, 4, 4

        layers = [Layer() for _ in range(4)]

        def make_cache(self):
            return [default(i) for i in range(4)]

    return Model()


@pytest.mark.filterwarnings("ignore::UserWarning")
def test_which_layers_get_block_caches():
    from mlx_turboquant_b200 import TurboQuantKVCache
    default = lambda i: _RotatingKVCache() if i == 2 else KVCache()  # noqa: E731
    plain = apply_turboquant(_model(default), skip_layers=[0]).make_cache()
    assert [type(c).__name__ for c in plain] == ["KVCache", "TurboQuantKVCache", "_RotatingKVCache", "TurboQuantKVCache"]
    caches = apply_turboquant(_model(default), skip_layers=[0], block_cache="e4m3").make_cache()
    assert [type(c) for c in caches] == [BlockKVCache, TurboQuantKVCache, BlockKVCache, TurboQuantKVCache]
    assert caches[0].window is None and caches[0].codes == "e4m3" and (caches[2].window, caches[2].sinks) == (124, 4) and caches[2].head_dim == 64
    with pytest.raises(ValueError):
        apply_turboquant(_model(default), block_cache="fp8")
    unknown = apply_turboquant(_model(lambda i: type("RotatingThing", (), {})()), skip_layers=[0], block_cache="int8").make_cache()
    assert all(type(c).__name__ == "RotatingThing" for c in unknown)                  # (a window of unknown size stays the model's)


# ---- on the GPU ---------------------------------------------------------------------------------------------------------------------

def tokens(b, h, t, d, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(b, h, t, d, generator=g).to(dtype).cuda()


def held(x, block, codes):
    """What a cache without a window holds of tokens x: float64 on the CPU."""
    cut = x.shape[2] // block * block
    c, s = encode(x[:, :, :cut].cpu().unflatten(2, (-1, block)) if cut else x[:, :, :0].cpu().unflatten(2, (0, block)), codes)
    return torch.cat([(c.float().double() * s.double()[..., None, None]).flatten(2, 3), x[:, :, cut:].cpu().double()], dim=2)


@pytest.mark.gpu
@pytest.mark.parametrize("codes,dtype,window,sinks", (("int8", torch.bfloat16, None, 0), ("e4m3", torch.float16, None, 0), ("int8", torch.float16, 100, 4), ("int8", torch.bfloat16, 64, 70),
                                                      ("e4m3", torch.float32, 33, 0)))
def test_a_life_of_a_cache(codes, dtype, window, sinks):
    """A prompt in pieces, steps, drafts: what every call returns, over what a cache without dropping would hold."""
    b, h, hq, d, block = 2, 2, 8, 64, 32
    c = BlockKVCache(d, h, codes, block, window, sinks)
    ct = torch.int8 if codes == "int8" else torch.float8_e4m3fn
    ks, vs = [], []
    for i, t in enumerate((7, 200, 1, 1, 300, 5) + (1,) * 70 + (64, 3) + (1,) * 40):
        k, v, q = tokens(b, h, t, d, dtype, 3 * i), tokens(b, h, t, d, dtype, 3 * i + 1), tokens(b, hq, t, d, dtype, 3 * i + 2)
        ks.append(k)
        vs.append(v)
        if t == 1:
            got = c.decode_step(q, k, v) if i % 2 else c.decode_step(q[:, :, 0], k, v).unsqueeze(2)
        else:
            c.update(k, v)
            got = c.attend(q)
        if i % 9 == 0 or t > 1:
            kd, vd = held(torch.cat(ks, 2), block, ct), held(torch.cat(vs, 2), block, ct)
            ref = attention(q.cpu(), kd, vd, d ** -0.5, window, sinks)
            top = vd.abs().max().item()
            tol = torch.finfo(dtype).eps / 2 * ref.abs() + top * (2.0 ** -11 + 2.0 ** -14 if dtype is not torch.float32 else 2.0 ** -15)      # (as test_blocks_gpu derives it)
            err = (got.double().cpu() - ref).abs()
            assert bool((err <= tol).all()), (i, float((err - tol).max()))
    assert c.size() == c.offset == sum(x.shape[2] for x in ks)
    if window is not None:
        assert c._dropped > 0
        for i in range(30):                                # (storage stays within twice what the window, the sinks and the longest piece fill)
            c.update(tokens(b, h, 90, d, dtype, i), tokens(b, h, 90, d, dtype, i))
        assert c._store[0].shape[2] <= 2 * (window + sinks + 300 + 3 * block) < c.offset
        with pytest.raises(ValueError, match="no longer stored"):
            c.attend(tokens(b, hq, c._length - 10, d, dtype, 1))
    else:
        k2, v2 = c.update_and_fetch(ks[0], vs[0])
        assert torch.equal(k2.cpu(), held(torch.cat(ks + [ks[0]], 2), block, ct).float().to(dtype))


@pytest.mark.gpu
def test_state_goes_round():
    c = BlockKVCache(128, 2, "int8", 64, 200, 4)
    for i in range(5):
        c.update(tokens(1, 2, 150, 128, torch.bfloat16, i), tokens(1, 2, 150, 128, torch.bfloat16, 10 + i))
    assert c._dropped > 0
    z = BlockKVCache(128, 2, "int8", 64, 200, 4)
    z.state = tuple(t.clone() for t in c.state)
    z.meta_state = c.meta_state
    assert z.nbytes == c.nbytes and z.offset == c.offset
    for i in range(3):
        q, k, v = tokens(1, 8, 1, 128, torch.bfloat16, 30 + i), tokens(1, 2, 1, 128, torch.bfloat16, 40 + i), tokens(1, 2, 1, 128, torch.bfloat16, 50 + i)
        assert torch.equal(c.decode_step(q, k, v), z.decode_step(q, k, v))
    with pytest.raises(ValueError):
        z.state = c.state[:4]
    with pytest.raises(RuntimeError):
        z.state = tuple(t.cpu() for t in c.state)
    with pytest.raises(ValueError):
        BlockKVCache(128, 2, "int8", 32).state = c.state
    with pytest.raises(ValueError):
        z.meta_state = {**c.meta_state, "offset": "100000"}


@pytest.mark.gpu
def test_a_restored_cache_writes_to_its_own_storage():
    from mlx_turboquant_b200 import BlockKVCache
    x = torch.randn(1, 2, 70, 64, device="cuda").half()
    a, z = BlockKVCache(64, 2, block=32), BlockKVCache(64, 2, block=32)
    a.update(x[:, :, :64], -x[:, :, :64])                         # (whole blocks: the state is the storage from end to end)
    z.state, z.meta_state = a.state, a.meta_state
    z.update(torch.ones_like(x[:, :, :6]), torch.ones_like(x[:, :, :6]))
    k, v = a.update_and_fetch(x[:, :, 64:], -x[:, :, 64:])
    assert torch.equal(k[:, :, 64:], x[:, :, 64:]) and torch.equal(v[:, :, 64:], -x[:, :, 64:])
    z.state = (None,) * 6
    assert z.empty()
    z.update(x, x)
    assert z.offset == 70


@pytest.mark.gpu
def test_a_refused_first_update_leaves_nothing():
    from mlx_turboquant_b200 import BlockKVCache
    c, x = BlockKVCache(64, 2), torch.randn(1, 2, 5, 64, device="cuda")
    for bad in ((x.double(), x.double()), (x, x.half()), (x, x[:, :, :4])):
        with pytest.raises((TypeError, ValueError)):
            c.update(*bad)
        with pytest.raises((TypeError, ValueError)):
            c.decode_step(x[:, :, :1], bad[0][:, :, :1], bad[1][:, :1, :1])
        assert c.empty() and c.state == (None,) * 6
    c.update(x.half(), x.half())
    assert c.offset == 5


@pytest.mark.gpu
def test_refusals_leave_the_cache_as_it_was():
    c = BlockKVCache(64, 2)
    with pytest.raises(ValueError):
        c.update(tokens(1, 3, 5, 64, torch.float16, 1), tokens(1, 3, 5, 64, torch.float16, 1))
    c.update(tokens(1, 2, 5, 64, torch.float16, 1), tokens(1, 2, 5, 64, torch.float16, 1))
    q = tokens(1, 4, 1, 64, torch.float16, 2)
    before = c.attend(q).clone()
    with pytest.raises(TypeError):
        c.update(tokens(1, 2, 1, 64, torch.bfloat16, 1), tokens(1, 2, 1, 64, torch.bfloat16, 1))
    with pytest.raises(TypeError):
        c.decode_step(q, tokens(1, 2, 1, 64, torch.bfloat16, 1), tokens(1, 2, 1, 64, torch.bfloat16, 1))
    with pytest.raises(ValueError):
        c.decode_step(q, tokens(2, 2, 1, 64, torch.float16, 1), tokens(2, 2, 1, 64, torch.float16, 1))
    with pytest.raises(ValueError):
        c.attend(tokens(1, 4, 6, 64, torch.float16, 1))
    assert c.offset == 5 and torch.equal(c.attend(q), before)


@pytest.mark.gpu
def test_the_caller_with_block_caches_and_scaled_positions():
    """Prompt pieces and steps through a model whose layers are skipped (8-bit blocks), windowed and packed: packed route, dense route, replayed graphs."""
    from mlx_turboquant_b200.consumer import GraphedDecoder, LlamaShaped, ModelArgs, generate
    scaling = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original_max_position_embeddings": 64}
    args = ModelArgs(**TINY, rope_scaling=scaling, rope_traditional=True, partial_rotary_factor=0.5)
    m = LlamaShaped(args, dtype=torch.bfloat16, seed=5, std=0.05)
    apply_turboquant(m, skip_layers=[0, 1, 2], block_cache="int8")
    prompt = torch.randint(0, 512, (2, 150), generator=torch.Generator().manual_seed(1)).cuda()
    packed, dense = m.make_cache(), m.make_cache()
    assert all(isinstance(c, BlockKVCache) for c in packed)
    for piece in (prompt[:, :100], prompt[:, 100:149], prompt[:, 149:]):
        a, z = m(piece, cache=packed, packed=True), m(piece, cache=dense, packed=False)
        # bfloat16 activations: both routes round every layer's result, 2^-8 of it; six of them in a row and the logits' sum over 256
        assert float((a.float() - z.float()).abs().max()) <= 0.06 * float(z.float().abs().max())
    windowed = [BlockKVCache(128, 4, "int8", 64, 40, 4) for _ in range(3)]
    out = generate(m, prompt, 6, cache=windowed, prefill_chunk=64)
    assert out.shape == (2, 6) and windowed[0].offset == 155
    # replayed graphs against eager steps
    first = torch.randint(0, 512, (2, 1), generator=torch.Generator().manual_seed(2)).cuda()
    eager_caches, graph_caches = m.make_cache(), m.make_cache()
    m(prompt, cache=eager_caches)
    m(prompt, cache=graph_caches)
    dec = GraphedDecoder(m, graph_caches, first)
    tok = first
    for _ in range(20):
        tok = m(tok, cache=eager_caches, last_only=True)[:, -1].argmax(-1, keepdim=True)
        assert torch.equal(dec.step(), tok)


@pytest.mark.gpu
def test_the_rotary_kernel_is_the_torch_code():
    """Plain embeddings through either: float32 angles are 2^-24 of a position off, the rest is rounding."""
    from mlx_turboquant_b200 import rope
    from mlx_turboquant_b200.consumer import rope as torch_rope
    x = tokens(1, 8, 50, 128, torch.bfloat16, 3)
    f, _ = rope.frequencies(128, 500000.0)
    a, z = rope.apply_rotary(x, None, f, 100)[0].float(), torch_rope(x, 100, 500000.0).float()
    # angles up to 150 with relative error 2^-23 move a value by 150 * 2^-23 of the largest of the pair; then half a bfloat16 step each, eps / 2 = 2^-8
    tol = 2 * 2.0 ** -8 * torch.maximum(a.abs(), z.abs()) + 2.0 ** -14 * float(x.float().abs().max())
    assert bool(((a - z).abs() <= tol).all())
