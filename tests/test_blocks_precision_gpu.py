"""How far attention over the 8-bit block cache is from float64, held to bounds relative to sum(w |v|), the weights' own sum over the values: errors of the weights, each
relative to its weight, cannot move a result by more than that.  (Relative to the largest value, as test_blocks_gpu has it, a result that averages many tokens may be off by several
per cent of itself.)"""

import pytest
import torch

from blocks_util import attention
from test_blocks_gpu import dense, rows, storage

pytestmark = pytest.mark.gpu

CODES = (torch.int8, torch.float8_e4m3fn)


@pytest.mark.parametrize("d", (64, 96, 128, 256))
@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("dtype", (torch.float16, torch.bfloat16))
@pytest.mark.parametrize("t", (1, 3, 40, 300))
def test_queries_with_one_large_coordinate(d, codes, dtype, t):
    """A coordinate of the queries 2048 times as large as the others, where the keys are zero: the others decide.

    Queries may be held in 22 bits of their largest element: 2^-22 of it off each, which moves a score by delta = 2^-22 max|q| sum|k| scale at most and the result by
    2 delta sum(w |v|) - here 0.002 to 0.004 of it; the keys have eight coordinates only so that this is small.  Beside it: weights rounded once to fp16, 2^-11 of sum(w |v|),
    2^-14 of it for the rest (scores in float32, exponentials), the result's own rounding."""
    from mlx_turboquant_b200 import blocks
    b, hq, h, total, scale = 2, 8, 2, 330, d ** -0.5
    k, v = rows(b, h, total, d, dtype, 1, std=0), rows(b, h, total, d, dtype, 2)
    few = torch.zeros(d, device="cuda")
    few[5:d:d // 8] = 3.0
    k = (k * few).to(dtype)
    k[..., 0] = 0
    q = rows(b, hq, t, d, dtype, 3, std=0)
    q[..., 0] = 2048.0
    store = storage(b, h, total, d, 32, codes, dtype)
    blocks.write_blocks(k, v, *store, 0)
    kd, vd = dense(store, total)
    for length in (total, 320):                            # (with and without a tail)
        if length < t:
            continue
        ref = attention(q.cpu(), kd[:, :, :length], vd[:, :, :length], scale)
        delta = 2.0 ** -22 * 2048 * float(kd.abs().sum(-1).max()) * scale
        wv = attention(q.cpu(), kd[:, :, :length], vd[:, :, :length].abs(), scale)
        tol = torch.finfo(dtype).eps / 2 * ref.abs() + wv * (2.0 ** -11 + 2.0 ** -14 + 2 * delta)
        err = (blocks.attend_blocks(q, *store, length).double().cpu() - ref).abs()
        assert bool((err <= tol).all()), (float((err / tol).max()), float(err.max()), delta)


@pytest.mark.parametrize("d", (64, 96, 128, 256))
@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("dtype", (torch.float16, torch.bfloat16))
@pytest.mark.parametrize("total", (2, 3, 17, 40, 330, 1000))
def test_weights_of_few_queries_are_not_rounded_to_16_bits(d, codes, dtype, total):
    """One token, and three: beside the result's own rounding 2^-14 of sum(w |v|), where weights rounded once would take 2^-11.

    Queries in 22 bits move scores by 2^-22 max|q| sum|k| scale < 2^-22 * 5 * 256 * 2 / 8, 2^-15 of a weight at most, twice; exponentials, float32 scores and scales
    2^-20; two fp16 parts 2^-22, or where they end 2^-25 of the largest weight for each token, 2^-15 over a thousand."""
    from mlx_turboquant_b200 import blocks
    b, hq, h, scale = 2, 16, 2, d ** -0.5
    store = storage(b, h, total, d, 16, codes, dtype)
    blocks.write_blocks(rows(b, h, total, d, dtype, 1, std=0), rows(b, h, total, d, dtype, 2), *store, 0)
    kd, vd = dense(store, total)
    for t in (1, 3):
        if t > total:
            continue
        q = rows(b, hq, t, d, dtype, 3, std=0)
        ref, wv = (attention(q.cpu(), kd, x, scale) for x in (vd, vd.abs()))
        err = (blocks.attend_blocks(q, *store, total).double().cpu() - ref).abs()
        tol = torch.finfo(dtype).eps / 2 * ref.abs() + 2.0 ** -14 * wv + (2.0 ** -25 if dtype is torch.float16 else 0.0)       # (half a step of fp16's subnormals)
        assert bool((err <= tol).all()), (float((err / tol).max()), t)


@pytest.mark.parametrize("d", (64, 96, 128, 256))
@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("block", (16, 64))
@pytest.mark.parametrize("b,total,t", ((1, 70, 70), (1, 1000, 130), (2, 1500, 600), (16, 330, 40)))
def test_fp16_prompts_are_as_precise_as_their_decoding(d, codes, block, b, total, t):
    """Many query rows of fp16 tokens: 2^-14 of sum(w |v|) beside the result's own rounding, as above (exponentials to 2^-16.9, twice; fp16 queries are exact here)."""
    from mlx_turboquant_b200 import blocks
    h, hq, scale, dtype = 2, 16, d ** -0.5, torch.float16
    store = storage(b, h, total, d, block, codes, dtype)
    blocks.write_blocks(rows(b, h, total, d, dtype, 1, std=0), rows(b, h, total, d, dtype, 2), *store, 0)
    kd, vd = dense(store, total)
    q = rows(b, hq, t, d, dtype, 3, std=0)
    for window, sinks in ((None, 0), (50, 4)):
        ref, wv = (attention(q.cpu(), kd, x, scale, window, sinks) for x in (vd, vd.abs()))
        err = (blocks.attend_blocks(q, *store, total, window=window, sinks=sinks).double().cpu() - ref).abs()
        tol = torch.finfo(dtype).eps / 2 * ref.abs() + 2.0 ** -14 * wv + 2.0 ** -25
        assert bool((err <= tol).all()), (float((err / tol).max()), window)
