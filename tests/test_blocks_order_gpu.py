"""Calls over the 8-bit block cache one after the other, with temporaries that the allocator hands on: results as when every call has ended before the next begins."""

import pytest
import torch

from test_blocks_gpu import rows, storage

pytestmark = pytest.mark.gpu


def tokens(b, h, t, d, dtype, seed):
    """Rows made on the GPU, as a view of a fused projection: (B, H, T, D) of (B, T, H, D) memory."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(b, t, h, d, generator=g, device="cuda").to(dtype).transpose(1, 2)


def after(sync, x):
    if sync:
        torch.cuda.synchronize()
    return x


@pytest.mark.parametrize("d,codes,window", ((128, torch.int8, 1000), (64, torch.float8_e4m3fn, 300), (256, torch.int8, 500)))
def test_attention_behind_a_write_of_temporaries(d, codes, window):
    """A prompt's piece is written from copies that are dropped, and attended to in scratch that fits where they were."""
    from mlx_turboquant_b200 import blocks
    dtype, b, h, hq, total, t = torch.bfloat16, 2, 4, 16, 20000, 256

    def run(sync, seed):
        store = storage(b, h, total + 64, d, 64, codes, dtype)
        k, v, q = (tokens(b, n, total, d, dtype, seed + i) for i, n in enumerate((h, h, 1)))
        q = q[:, :, :t].expand(b, hq, t, d).contiguous()
        torch.cuda.synchronize()
        kc, vc = k.contiguous(), v.contiguous()
        blocks.write_blocks(kc, vc, *store, 0)
        if sync:
            torch.cuda.synchronize()
        del kc, vc                                             # (as a caller's temporaries: their memory is the next allocation's)
        out = after(sync, blocks.attend_blocks(q, *store, total, window=window, sinks=4))
        torch.cuda.synchronize()
        return [out, *store]

    for seed in range(0, 60, 3):
        for x, y in zip(run(False, seed), run(True, seed)):
            assert torch.equal(x.view(torch.int8) if x.element_size() == 1 else x, y.view(torch.int8) if y.element_size() == 1 else y)


def test_one_graph_of_many_calls():
    """Decode with partials to join, a dense read, tokens written from copies, a prompt's piece: captured into one pool, temporaries dropped, replayed again and again."""
    from mlx_turboquant_b200 import blocks, rope
    dtype, d, b, h, hq, total, t = torch.bfloat16, 128, 1, 8, 32, 9000, 512
    store = storage(b, h, total + 2 * t + 64, d, 64, torch.int8, dtype)
    blocks.write_blocks(rows(b, h, total, d, dtype, 1), rows(b, h, total, d, dtype, 2), *store, 0)
    start = [x.clone() for x in store]
    freqs, factor = rope.frequencies(d)
    qkv = tokens(b, hq + 2 * h, t, d, dtype, 5)
    q1 = rows(b, hq, 1, d, dtype, 6, std=0)

    def calls(sync):
        a = after(sync, blocks.attend_blocks(q1, *store, total))
        k, v = after(sync, blocks.read_blocks(*store, total))
        sums = after(sync, (k.float().sum(-1), v.float().sum(-1)))
        del k, v
        q, kk = after(sync, rope.apply_rotary(qkv[:, :hq], qkv[:, hq:hq + h], freqs, total, factor=factor))
        vv = qkv[:, hq + h:].contiguous()
        n = after(sync, blocks.write_blocks(kk, vv, *store, total))
        del kk, vv
        z = after(sync, blocks.attend_blocks(q, *store, n))
        w = after(sync, blocks.attend_blocks(q, *store, n, window=700, sinks=4))
        return [a, *sums, z, w]

    def restore():
        for x, y in zip(store, start):
            x.copy_(y)
        torch.cuda.synchronize()

    want = [x.clone() for x in calls(True)]
    held = [x.clone() for x in store]
    restore()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        calls(False)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = calls(False)
    for _ in range(30):
        restore()
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(got, want):
            assert torch.equal(x, y)
        for x, y in zip(store, held):
            assert torch.equal(x, y)
