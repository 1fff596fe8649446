"""The settings of scaled rotary positions: what a table is kept under, what is refused.  No GPU."""

import math

import numpy as np
import pytest
import torch

from mlx_turboquant_b200 import rope


def table(dims=64, base=10000.0, **scaling):
    return rope.frequencies(dims, base, scaling, "cpu")


@pytest.mark.parametrize("number", (float, int, str, np.float32, np.float64, np.int64, torch.tensor))
@pytest.mark.parametrize("kind,other", (("linear", {}), ("llama3", {"original_max_position_embeddings": 8192}), ("yarn", {"original_max_position_embeddings": 4096})))
def test_every_setting_counts(kind, other, number):
    """Two tables in a row whose settings differ in one number, of whatever type it comes in; each is that of a plain float."""
    names = {"linear": ("factor",), "llama3": ("factor", "low_freq_factor", "high_freq_factor", "original_max_position_embeddings"),
             "yarn": ("factor", "original_max_position_embeddings", "beta_fast", "beta_slow")}[kind]
    values = {"factor": (4, 8), "low_freq_factor": (1, 2), "high_freq_factor": (4, 16), "original_max_position_embeddings": (8192, 1024), "beta_fast": (32, 8), "beta_slow": (1, 2)}
    for name in names:
        got = [table(rope_type=kind, **{"factor": 16.0, **other, name: number(v)}) for v in values[name]]
        rope._tables.clear()
        want = [table(rope_type=kind, **{"factor": 16.0, **other, name: float(v)}) for v in values[name]]
        assert not torch.equal(got[0][0], got[1][0]), name
        for g, w in zip(got, want):
            assert torch.equal(g[0], w[0]) and g[1] == w[1], name
    if kind == "yarn":
        assert table(rope_type=kind, factor=4.0, **other, attention_factor=number(2))[1] == 2.0 and table(rope_type=kind, factor=4.0, **other, attention_factor=number(3))[1] == 3.0


def test_none_is_as_good_as_absent():
    for kind, names in (("llama3", ("low_freq_factor", "high_freq_factor")), ("yarn", ("beta_fast", "beta_slow", "attention_factor"))):
        given = {"rope_type": kind, "factor": 8.0, "original_max_position_embeddings": 8192}
        plain = table(**given)
        for name in names:
            f, m = table(**given, **{name: None})
            assert torch.equal(f, plain[0]) and m == plain[1], name
    assert torch.equal(table(rope_type="default", factor=None)[0], table()[0])


def test_the_defaults_are_the_published_ones():
    f, m = table(rope_type="yarn", factor=8.0, original_max_position_embeddings=4096)
    g, n = table(rope_type="yarn", factor=8.0, original_max_position_embeddings=4096, beta_fast=32, beta_slow=1, attention_factor=0.1 * math.log(8.0) + 1)
    assert torch.equal(f, g) and m == n
    f, _ = table(rope_type="llama3", factor=8.0, original_max_position_embeddings=8192)
    assert torch.equal(f, table(rope_type="llama3", factor=8.0, original_max_position_embeddings=8192, low_freq_factor=1, high_freq_factor=4)[0])


def test_a_scaling_without_its_length():
    """Left out of a model's configuration, the length is the model's own: no number of this package's stands for it unsaid."""
    from mlx_turboquant_b200.consumer import ModelArgs
    for missing in ({}, {"original_max_position_embeddings": None}):
        with pytest.raises(ValueError, match="original_max_position_embeddings"):
            table(rope_type="llama3", factor=8.0, **missing)
        with pytest.warns(UserWarning, match="4096 positions"):
            f, _ = table(rope_type="yarn", factor=8.0, **missing)
        assert torch.equal(f, table(rope_type="yarn", factor=8.0, original_max_position_embeddings=4096)[0])
        for kind in ("llama3", "yarn"):
            with pytest.raises(ValueError, match="original_max_position_embeddings"):
                ModelArgs(head_dim=64, rope_scaling={"rope_type": kind, "factor": 8.0, **missing}).rotary_frequencies("cpu")
    f, _ = ModelArgs(head_dim=64, rope_theta=10000.0, rope_scaling={"type": "yarn", "factor": 8.0, "original_max_position_embeddings": 2048}).rotary_frequencies("cpu")
    assert torch.equal(f, table(rope_type="yarn", factor=8.0, original_max_position_embeddings=2048)[0])


def test_numbers_that_give_no_angles():
    for bad in (float("inf"), float("nan"), -2.0, 0.0):
        for kind in ("linear", "llama3", "yarn"):
            with pytest.raises(ValueError):
                table(rope_type=kind, factor=bad, **({} if kind == "linear" else {"original_max_position_embeddings": 4096}))
        for kind, name in (("llama3", "original_max_position_embeddings"), ("yarn", "original_max_position_embeddings"), ("yarn", "beta_fast"), ("yarn", "beta_slow"), ("llama3", "low_freq_factor")):
            with pytest.raises(ValueError):
                table(**{"rope_type": kind, "factor": 2.0, "original_max_position_embeddings": 4096, name: bad})
        with pytest.raises(ValueError):
            table(base=bad)
    for low, high in ((2, 2), (4, 1)):
        with pytest.raises(ValueError):
            table(rope_type="llama3", factor=8.0, original_max_position_embeddings=8192, low_freq_factor=low, high_freq_factor=high)
    with pytest.raises(ValueError):
        table(base=1.0, rope_type="yarn", factor=2.0, original_max_position_embeddings=4096)


def test_no_table_is_made_inside_a_capture(monkeypatch):
    """Nothing of a refused call stays: the table is made by the next one outside."""
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="before the capture"):
        rope.frequencies(48, 77.0, device="cuda:0")
    assert not any(k[:2] == (48, 77.0) for k in rope._tables)
    f, _ = table(48, 77.0)
    assert rope.frequencies(48, 77.0, device="cpu")[0] is f                 # (the CPU's are never captured)


def test_a_forward_pass_looks_its_table_up_once(monkeypatch):
    """Not for each layer of each step: the settings are read anew every time."""
    from mlx_turboquant_b200 import consumer
    args = consumer.ModelArgs(hidden_size=64, num_hidden_layers=5, num_attention_heads=2, num_key_value_heads=1, head_dim=32, intermediate_size=64, vocab_size=32, rope_scaling={"rope_type": "linear", "factor": 2.0})
    m, calls, made = consumer.LlamaShaped(args, dtype=torch.float32, device="cpu"), [], rope.frequencies
    monkeypatch.setattr(consumer.rotary, "frequencies", lambda *a, **kw: calls.append(a) or made(*a, **kw))
    monkeypatch.setattr(consumer.rotary, "apply_rotary", lambda q, k, *a, **kw: (q, k))
    for n in (1, 2):
        m(torch.zeros(1, 3, dtype=torch.int64))
        assert len(calls) == n
