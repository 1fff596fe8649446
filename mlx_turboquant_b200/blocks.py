"""A KV cache held in 8 bits: a scale for each block of tokens and head, written as tokens come, read back, attended to.

For the layers that 2 to 4 bits would hurt (``apply_turboquant(..., skip_layers=...)``, outliers) and for sliding-window layers, which the
reference leaves on the model's uncompressed default cache (patch.py:238-340).

Storage, six tensors: ``k_codes`` and ``v_codes`` (B, H, capacity, D), ``torch.int8`` or ``torch.float8_e4m3fn``; ``k_scales`` and ``v_scales``
(B, H, capacity / block), float32; ``k_tail`` and ``v_tail`` (B, H, block, D), the tokens behind the last whole block as they came.  Blocks of
16, 32, 64 or 128 tokens.  A block is quantised once, when its last token arrives: what the cache holds depends on the tokens, not on the calls
they came in.

* ``write_blocks`` appends tokens, ``read_blocks`` gives all of them dense, ``attend_blocks`` computes attention from the storage;
* ``BlockKVCache`` keeps the storage of a layer behind the protocol of ``TurboQuantKVCache``.
"""

from __future__ import annotations

import ctypes as C
from typing import Any

import torch

from . import _lib

CODE_TYPES = {torch.int8: _lib.TQ_CODE_INT8, torch.float8_e4m3fn: _lib.TQ_CODE_E4M3}
BLOCKS = (16, 32, 64, 128)


def _no_grad(*tensors) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError("the block cache has no backward pass: call it under torch.no_grad()")


def _store(k_codes, k_scales, v_codes, v_scales, k_tail, v_tail, length: int) -> "_lib.BlockStore":
    """Checked storage as the library's argument block."""
    if k_codes.dtype not in CODE_TYPES or v_codes.dtype != k_codes.dtype:
        raise TypeError(f"codes must be int8 or float8_e4m3fn, keys and values alike; got {k_codes.dtype} and {v_codes.dtype}")
    if k_scales.dtype != torch.float32 or v_scales.dtype != torch.float32:
        raise TypeError("scales must be float32")
    if k_tail.dtype != v_tail.dtype:
        raise TypeError("the tails must have one type")
    if k_codes.dim() != 4 or k_scales.dim() != 3 or k_tail.dim() != 4:
        raise ValueError("codes and tails have four axes, scales three")
    b, h, cap, d = k_codes.shape
    n = k_tail.shape[2]
    if n not in BLOCKS:
        raise ValueError(f"blocks have 16, 32, 64 or 128 tokens, got a tail of {n}")
    if (v_codes.shape != k_codes.shape or tuple(k_tail.shape) != (b, h, n, d) or v_tail.shape != k_tail.shape or cap % n
            or tuple(k_scales.shape) != (b, h, cap // n) or v_scales.shape != k_scales.shape):
        raise ValueError("storage shapes disagree: codes (B, H, capacity, D), scales (B, H, capacity / block), tails (B, H, block, D)")
    if not all(t.is_contiguous() for t in (k_codes, v_codes, k_scales, v_scales, k_tail, v_tail)):
        raise ValueError("storage must be contiguous")
    if length < 0 or length // n * n > cap:
        raise ValueError(f"{length} tokens in storage for {cap}")
    s = _lib.BlockStore()
    s.batch, s.n_kv_heads, s.d, s.block = b, h, d, n
    s.code_type, s.dtype = CODE_TYPES[k_codes.dtype], _lib.dtype_code(k_tail.dtype)
    s.k_codes, s.v_codes, s.k_scales, s.v_scales = k_codes.data_ptr(), v_codes.data_ptr(), k_scales.data_ptr(), v_scales.data_ptr()
    s.k_tail, s.v_tail, s.capacity, s.length = k_tail.data_ptr(), v_tail.data_ptr(), cap, length
    return s


def _aligned(x: torch.Tensor) -> torch.Tensor:
    """Rows (B, H, T, D) as the kernels read them: contiguous coordinates, 16-byte aligned; copied where they are not."""
    n = 16 // x.element_size()
    st = x.stride()
    if ((st[3] == 1 or x.shape[3] == 1) and x.data_ptr() % 16 == 0 and (x.shape[2] == 1 or st[2] % n == 0) and (x.shape[1] == 1 or st[1] % n == 0)
            and (x.shape[0] == 1 or st[0] % n == 0)):
        return x
    return x.clone(memory_format=torch.contiguous_format)


def _rows(x: torch.Tensor) -> "_lib.NewRows":
    st, shape = x.stride(), x.shape
    return _lib.NewRows(x.data_ptr(), *(st[i] if shape[i] > 1 else 0 for i in range(3)))


def _new_tokens(keys: torch.Tensor, values: torch.Tensor, tail: torch.Tensor) -> None:
    b, h, _, d = tail.shape
    if keys.dim() != 4 or keys.shape != values.shape or keys.shape[0] != b or keys.shape[1] != h or keys.shape[3] != d:
        raise ValueError(f"new tokens must be (B, H, T, D) = ({b}, {h}, T, {d}), got {tuple(keys.shape)} and {tuple(values.shape)}")
    if keys.dtype != tail.dtype or values.dtype != tail.dtype:
        raise TypeError(f"the cache takes {tail.dtype} tokens, got {keys.dtype} and {values.dtype}")


def write_blocks(keys: torch.Tensor, values: torch.Tensor, k_codes, k_scales, v_codes, v_scales, k_tail, v_tail, length: int) -> int:
    """Append (B, H, T, D) tokens of the tails' type behind the ``length`` that the storage holds; returns the new length.  The storage must have
    room for the whole blocks that they fill."""
    res = _lib.host().blocks_write(keys, values, k_codes, k_scales, v_codes, v_scales, k_tail, v_tail, length)
    if res is not None:
        if res < 0:
            _lib.check(res)
        return res
    dev = _lib.require_cuda(keys, values, k_codes, k_scales, v_codes, v_scales, k_tail, v_tail)
    _no_grad(keys, values)
    s = _store(k_codes, k_scales, v_codes, v_scales, k_tail, v_tail, length)
    _new_tokens(keys, values, k_tail)
    t = keys.shape[2]
    if (length + t) // s.block * s.block > s.capacity:
        raise ValueError(f"{length} tokens and {t} more in storage for {s.capacity}")
    if t == 0 or s.batch * s.n_kv_heads == 0:
        return length + t
    keys, values = _aligned(keys), _aligned(values)
    _lib.check(_lib.launch(dev, "tq_blocks_write", C.byref(s), C.byref(_rows(keys)), C.byref(_rows(values)), t, _lib.stream_ptr(dev)))
    return length + t


def read_blocks(k_codes, k_scales, v_codes, v_scales, k_tail, v_tail, length: int, dtype: torch.dtype | None = None):
    """All ``length`` tokens as dense (keys, values), (B, H, length, D) of ``dtype`` (default: the tails')."""
    res = _lib.host().blocks_read(k_codes, k_scales, v_codes, v_scales, k_tail, v_tail, length) if dtype is None or dtype is k_tail.dtype else None
    if res is not None:
        if type(res) is int:
            _lib.check(res)
        return res
    dev = _lib.require_cuda(k_codes, k_scales, v_codes, v_scales, k_tail, v_tail)
    s = _store(k_codes, k_scales, v_codes, v_scales, k_tail, v_tail, length)
    dtype = k_tail.dtype if dtype is None else dtype
    code = _lib.dtype_code(dtype)
    k, v = (torch.empty((s.batch, s.n_kv_heads, length, s.d), dtype=dtype, device=dev) for _ in range(2))
    if k.numel():
        _lib.check(_lib.launch(dev, "tq_blocks_read", C.byref(s), k.data_ptr(), v.data_ptr(), code, _lib.stream_ptr(dev)))
    return k, v


def attend_blocks(queries: torch.Tensor, k_codes, k_scales, v_codes, v_scales, k_tail, v_tail, length: int, *, window: int | None = None,
                  sinks: int = 0, scale: float | None = None, out: torch.Tensor | None = None, new=None) -> torch.Tensor:
    """softmax(scale q K^T) V of the last T_q of ``length`` tokens, causal, from the storage.

    ``queries`` (B, H_q, T_q, D) of the tails' type; H_q a multiple of H.  With ``window`` a query sees the last ``window`` tokens up to its own and
    the first ``sinks`` of the cache.  ``new`` = (keys, values), (B, H, 1, D): one more token, which joins the cache and is attended to, in the
    same launch unless it completes a block (the cache then holds ``length + 1`` tokens).  ``out`` (contiguous, the queries' shape and type)
    receives the result."""
    if out is None:
        res = _lib.host().blocks_attend(queries, k_codes, k_scales, v_codes, v_scales, k_tail, v_tail, length, window or 0, sinks,
                                        scale, *(new if new is not None else (None, None))) if window != 0 else None
        if res is not None:
            if type(res) is int:
                _lib.check(res)
            return res
    k_new, v_new = new if new is not None else (None, None)
    dev = _lib.require_cuda(queries, k_codes, k_scales, v_codes, v_scales, k_tail, v_tail, k_new, v_new, out)
    _no_grad(queries, k_new, v_new)
    if window is not None and window < 1:
        raise ValueError(f"a window holds the query's own token at least, got {window}")
    if sinks < 0:
        raise ValueError(f"sinks must not be negative, got {sinks}")
    a = _lib.BlocksAttendArgs()
    a.store = s = _store(k_codes, k_scales, v_codes, v_scales, k_tail, v_tail, length)
    if queries.dim() != 4 or queries.shape[0] != s.batch or queries.shape[3] != s.d or s.n_kv_heads == 0 or queries.shape[1] % s.n_kv_heads:
        raise ValueError(f"queries must be (B, H_q, T_q, D) with B = {s.batch}, D = {s.d} and H_q a multiple of {s.n_kv_heads}, got {tuple(queries.shape)}")
    if queries.dtype != k_tail.dtype:
        raise TypeError(f"the cache takes {k_tail.dtype} queries, got {queries.dtype}")
    t = queries.shape[2]
    if out is None:
        out = torch.empty(queries.shape, dtype=queries.dtype, device=dev)
    elif out.shape != queries.shape or out.dtype != queries.dtype or not out.is_contiguous():
        raise ValueError("out must be contiguous and of the queries' shape and type")
    q = _aligned(queries)
    if new is not None:
        _new_tokens(k_new, v_new, k_tail)
        if k_new.shape[2] != 1 or t != 1:
            raise ValueError("one new token, attended to by its own queries; write_blocks takes several")
        if length % s.block + 1 == s.block:                # it completes a block
            s.length = write_blocks(k_new, v_new, k_codes, k_scales, v_codes, v_scales, k_tail, v_tail, length)
            a.store.length = s.length
        else:
            k_new, v_new = _aligned(k_new), _aligned(v_new)
            a.k_new, a.v_new = _rows(k_new), _rows(v_new)
    if t > s.length + (a.k_new.x is not None):
        raise ValueError(f"{t} query tokens over {s.length} in the cache: write their keys and values first")
    a.n_q_heads, a.t_q, a.q = queries.shape[1], t, _rows(q)
    a.scale, a.window, a.sinks, a.out = float(s.d ** -0.5 if scale is None else scale), int(window or 0), int(sinks), out.data_ptr()
    if out.numel() == 0:
        return out
    # Any content, so that the allocator's memory serves: one call's scratch is its own, in captured graphs and on every stream.
    need = int(_lib.launch(dev, "tq_blocks_attend_workspace", C.byref(a)))
    if need:
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        a.workspace, a.workspace_bytes = ws.data_ptr(), need
    _lib.check(_lib.launch(dev, "tq_blocks_attend", C.byref(a), _lib.stream_ptr(dev)))
    return out
