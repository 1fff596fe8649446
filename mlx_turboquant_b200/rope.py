"""Rotary positions on the GPU: queries and keys turned and laid out for a cache in one launch.

The reference's models turn queries and keys with ``mlx.nn.RoPE`` before they reach its cache (docs/attention_source_dump.txt:78-86):
``traditional`` there is ``interleaved`` here, ``dims`` the coordinates of a head that are turned, ``scale`` one of the scalings below.

``apply_rotary(q, k, freqs, offset)`` takes the angles per position as a float64 tensor, ``frequencies(...)`` makes it.
"""

from __future__ import annotations

import ctypes as C
import math
import warnings

import torch

from . import _lib

_tables: dict[tuple, tuple[torch.Tensor, float]] = {}
# what each kind of scaling understands besides its name, and what stands for a setting that is absent or None (REQUIRED: it has to be there); anything else is
# refused rather than left out
REQUIRED = object()
_SETTINGS = {"default": {}, "linear": {"factor": REQUIRED},
             "llama3": {"factor": REQUIRED, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original_max_position_embeddings": REQUIRED},
             "yarn": {"factor": REQUIRED, "original_max_position_embeddings": 4096.0, "beta_fast": 32.0, "beta_slow": 1.0, "attention_factor": None}}


def _settings(scaling: dict | None) -> tuple[str, dict]:
    """The kind of a model's ``rope_scaling`` entry and its settings as Python floats (or None)."""
    s = dict(scaling or {})
    kind = s.get("rope_type", s.get("type", "default"))
    if kind not in _SETTINGS:
        raise ValueError(f"unsupported rope scaling {kind!r}: default, linear, llama3 or yarn")
    unknown = [k for k, v in s.items() if v is not None and k not in ("rope_type", "type", *_SETTINGS[kind])]
    if unknown:
        raise ValueError(f"rope scaling {kind!r} does not know {', '.join(sorted(unknown))}")
    out = {}
    for name, default in _SETTINGS[kind].items():
        value = s.get(name)
        if value is None and default is REQUIRED:
            raise ValueError(f"rope scaling {kind!r} needs a {name}")
        out[name] = default if value is None else float(value)
    bad = [f"{k} = {s[k]!r}" for k, v in out.items() if v is not None and not 0.0 < v < math.inf and (k != "attention_factor" or v != 0.0)]       # (0: the default)
    if bad:
        raise ValueError(f"rope scaling {kind!r} needs positive numbers, got {', '.join(bad)}")
    if kind == "llama3" and not out["high_freq_factor"] > out["low_freq_factor"]:
        raise ValueError(f"rope scaling 'llama3' blends between low_freq_factor and a larger high_freq_factor, got {out['low_freq_factor']} and {out['high_freq_factor']}")
    # a configuration without the length means the model's own, which only the caller knows
    if kind == "yarn" and s.get("original_max_position_embeddings") is None:
        warnings.warn(f"rope scaling 'yarn' without original_max_position_embeddings: {int(out['original_max_position_embeddings'])} positions are assumed; "
                      "give the length that the model was trained on", UserWarning, stacklevel=3)
    return kind, out


def frequencies(dims: int, base: float = 10000.0, scaling: dict | None = None, device="cuda") -> tuple[torch.Tensor, float]:
    """(radians per position of each of the ``dims / 2`` pairs, float64 on ``device``; the factor on the result), shared between calls.
    The first call for a table copies it to the device: not inside a graph's capture.

    ``scaling`` is the ``rope_scaling`` entry of a model's config: ``{"rope_type": ..., "factor": ...}`` with

    * ``"linear"``: positions divided by ``factor``;
    * ``"llama3"``: pairs that turn less than ``low_freq_factor`` (1) times in ``original_max_position_embeddings`` positions are slowed by ``factor``,
      those that turn more than ``high_freq_factor`` (4) times stay, a blend in between;
    * ``"yarn"``: the same with a ramp over the pairs' index between ``beta_fast`` (32) and ``beta_slow`` (1) turns, and a factor on the result
      (``attention_factor``, otherwise ``0.1 ln(factor) + 1``).

    The length that a model was trained on, ``original_max_position_embeddings``, is wanted with both: configurations that leave it out mean the model's
    ``max_position_embeddings``.  llama3 refuses without it; yarn assumes 4096 and says so in a warning.
    """
    if dims <= 0 or dims % 2:
        raise ValueError(f"an even number of coordinates is turned, got {dims}")
    if not (0.0 < float(base) < math.inf):
        raise ValueError(f"the base of the frequencies must be positive, got {base}")
    kind, s = _settings(scaling)
    if kind == "yarn" and float(base) <= 1.0:
        raise ValueError(f"rope scaling 'yarn' needs a base above 1, got {base}")
    device = torch.device(device)
    if device.type == "cuda" and device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    key = (dims, float(base), kind, tuple(s.values()), device)
    if key not in _tables:
        if device.type == "cuda" and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("rope.frequencies: this table is not made yet, and making it copies from the host, which a graph cannot capture; call it once before the capture")
        f = float(base) ** (-torch.arange(0, dims, 2, dtype=torch.float64) / dims)
        result = 1.0
        if kind == "linear":
            f = f / s["factor"]
        elif kind == "llama3":
            low, high = s["low_freq_factor"], s["high_freq_factor"]
            turns = s["original_max_position_embeddings"] * f / (2 * math.pi)
            keep = ((turns - low) / (high - low)).clamp(0.0, 1.0)
            f = f * ((1 - keep) / s["factor"] + keep)
        elif kind == "yarn":
            length, slow = s["original_max_position_embeddings"], s["factor"]
            at = [dims * math.log(length / (t * 2 * math.pi)) / (2 * math.log(base)) for t in (s["beta_fast"], s["beta_slow"])]
            first, last = max(math.floor(at[0]), 0), min(math.ceil(at[1]), dims - 1)
            ramp = ((torch.arange(dims // 2, dtype=torch.float64) - first) / max(last - first, 0.001)).clamp(0.0, 1.0)
            f = f * (ramp / slow + (1 - ramp))
            result = s["attention_factor"] or (0.1 * math.log(slow) + 1.0 if slow > 1 else 1.0)
        _tables[key] = (f.to(device), result)
    return _tables[key]


def _part(r, x: torch.Tensor, out: torch.Tensor) -> None:
    r.x, r.sb, r.sh, r.st, r.out, r.heads = x.data_ptr(), x.stride(0), x.stride(1), x.stride(2), out.data_ptr(), x.shape[1]


def apply_rotary(q: torch.Tensor, k: torch.Tensor | None, freqs: torch.Tensor, offset: int = 0, *, positions: torch.Tensor | None = None,
                 interleaved: bool = False, factor: float = 1.0):
    """Queries (B, H_q, L, D) and keys (B, H_kv, L, D) at positions ``offset``, ``offset + 1``, ... turned by ``position * freqs`` -> (q, k),
    contiguous, of their type (k may be None).

    The first ``2 * len(freqs)`` coordinates of each head are turned, in pairs of the two halves or, ``interleaved``, of neighbours; the others are
    copied; turned ones are multiplied by ``factor``.  ``positions`` (int64 on the device, (L,) or (B, L)) gives every token its own position in
    place of ``offset``.  Any strides with contiguous heads are read as they are: the views of a fused projection need no copy.  Angles
    are formed in float64, products in float32, one rounding.  Inference only."""
    res = _lib.host().rotary(q, k, freqs, offset, positions, interleaved, factor)
    if res is not None:
        if type(res) is int:
            _lib.check(res)
        return res
    dev = _lib.require_cuda(q, k, freqs, positions)
    for x in (q, k):
        if x is None:
            continue
        if x.dim() != 4 or x.shape[0] != q.shape[0] or x.shape[2:] != q.shape[2:] or x.dtype != q.dtype:
            raise ValueError("queries and keys must be (B, heads, L, D) of one B, L, D and type")
        if torch.is_grad_enabled() and x.requires_grad:
            raise RuntimeError("apply_rotary has no backward pass: call it under torch.no_grad()")
    code = _lib.dtype_code(q.dtype)
    b, _, length, d = q.shape
    if freqs.dtype != torch.float64 or freqs.dim() != 1 or not freqs.is_contiguous():
        raise ValueError("freqs must be a contiguous float64 vector (rope.frequencies)")
    if freqs.numel() == 0 or 2 * freqs.numel() > d:
        raise ValueError(f"{freqs.numel()} pairs in heads of {d}")
    a = _lib.RotaryArgs()
    if positions is not None:
        if positions.dtype != torch.int64 or tuple(positions.shape) not in ((length,), (b, length)) or (length > 1 and positions.stride(-1) != 1):
            raise ValueError("positions must be int64, (L,) or (B, L), contiguous along L")
        a.positions, a.pos_sb = positions.data_ptr(), (positions.stride(0) if positions.dim() == 2 and b > 1 else 0)
    a.dtype, a.batch, a.d, a.dims, a.interleaved, a.length = code, b, d, 2 * freqs.numel(), bool(interleaved), length
    a.freqs, a.factor, a.offset = freqs.data_ptr(), float(factor), int(offset)
    outs = []
    for r, x in zip(a.part, (q, k)):
        if x is None:
            outs.append(None)
            continue
        if x.stride(3) != 1 and d > 1:
            x = x.contiguous()
        out = torch.empty(x.shape, dtype=x.dtype, device=dev)
        _part(r, x, out)
        outs.append((out, x))                              # (x stays alive until the launch)
    _lib.check(_lib.launch(dev, "tq_rotary", C.byref(a), _lib.stream_ptr(dev)))
    return tuple(None if o is None else o[0] for o in outs)
