"""A KV cache held in 8 bits: a scale for each block of tokens and head, written as tokens come, read back, attended to.

For the layers that 2 to 4 bits would hurt (``apply_turboquant(..., skip_layers=...)``, outliers) and for sliding-window layers, which the
reference leaves on the model's uncompressed default cache (patch.py:238-340).

Storage, six tensors: ``k_codes`` and ``v_codes`` (B, H, capacity, D), ``torch.int8`` or ``torch.float8_e4m3fn``; ``k_scales`` and ``v_scales``
(B, H, capacity / block), float32; ``k_tail`` and ``v_tail`` (B, H, block, D), the tokens behind the last whole block as they came.  Blocks of
16, 32, 64 or 128 tokens.  A block is quantised once, when its last token arrives: what the cache holds depends on the tokens, not on the calls
they came in.  Codes are finite (the scale of a block that is not is NaN); storage from elsewhere must keep to that.

* ``write_blocks`` appends tokens, ``read_blocks`` gives all of them dense, ``attend_blocks`` computes attention from the storage;
* ``BlockKVCache`` keeps the storage of a layer behind the protocol of ``TurboQuantKVCache``.
"""

from __future__ import annotations

import ctypes as C
from typing import Any

import torch

from . import _lib, kernels

CODE_TYPES = {torch.int8: _lib.TQ_CODE_INT8, torch.float8_e4m3fn: _lib.TQ_CODE_E4M3}
BLOCKS = (16, 32, 64, 128)
SMALL = 64 << 20               # scratch that a call makes do with on a card without room for what it would like


def head_dim_ok(d: int) -> bool:
    """Whether the kernels of the block cache take this head_dim."""
    return 0 < d <= 256 and d % 32 == 0


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
    receives the result and must not overlap what is read.

    Long pieces of a prompt take up to some 600 MB of scratch while they run; without room for that the call takes ways that need less."""
    if window != 0:
        res = _lib.host().blocks_attend(queries, k_codes, k_scales, v_codes, v_scales, k_tail, v_tail, length, window or 0, sinks, scale,
                                        *(new if new is not None else (None, None)), out)
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
    a.scale, a.out = float(s.d ** -0.5 if scale is None else scale), out.data_ptr()
    a.window, a.sinks = min(int(window or 0), 1 << 62), min(int(sinks), 1 << 62)
    if out.numel() == 0:
        return out
    # Any content, so that the allocator's memory serves: one call's scratch is its own, in captured graphs and on every stream.  On a card without room for it, slower ways run that
    # make do with little, or with none.
    need = int(_lib.launch(dev, "tq_blocks_attend_workspace", C.byref(a)))
    if need:
        ws = kernels.scratch(dev, lambda: need, lambda: int(_lib.launch(dev, "tq_blocks_attend_workspace_within", C.byref(a), min(need - 1, SMALL))))
        a.workspace, a.workspace_bytes = (None, 0) if ws is None else (ws.data_ptr(), ws.numel())
    _lib.check(_lib.launch(dev, "tq_blocks_attend", C.byref(a), _lib.stream_ptr(dev)))
    return out


def window_mask(offset: int, n: int, window: int, sinks: int, device) -> torch.Tensor:
    """Which tokens ``n`` queries behind ``offset`` tokens see: (n, sinks before the window + tokens from the first query's window on)."""
    low = max(0, offset - window + 1)
    pos = torch.arange(offset, offset + n, device=device)[:, None]
    tok = torch.cat([torch.arange(min(sinks, low), device=device), torch.arange(low, offset + n, device=device)])[None, :]
    return (tok <= pos) & ((pos - tok < window) | (tok < sinks))


class BlockKVCache:
    """KV cache of a layer in 8-bit blocks, behind the protocol of ``TurboQuantKVCache``.

    ``codes``: ``"int8"`` or ``"e4m3"``; ``block``: tokens that share a scale (16, 32, 64 or 128).  With ``window`` a query sees the last ``window`` tokens
    up to its own and the first ``sinks`` ones; blocks that no later query can see are dropped when their room is wanted, so that the storage stays bounded
    by the window and the longest piece of prompt.  float16, bfloat16 (or, on slower kernels, float32) tokens, of one type per cache."""

    step = 256

    def __init__(self, head_dim: int = 128, num_kv_heads: int = 1, codes: str = "int8", block: int = 64, window: int | None = None, sinks: int = 0):
        if codes not in ("int8", "e4m3"):
            raise ValueError(f"codes must be 'int8' or 'e4m3', got {codes!r}")
        if block not in BLOCKS:
            raise ValueError(f"blocks have 16, 32, 64 or 128 tokens, got {block}")
        if not head_dim_ok(head_dim):
            raise ValueError(f"head_dim must be a multiple of 32 up to 256, got {head_dim}")
        if window is not None and window < 1:
            raise ValueError(f"a window holds the query's own token at least, got {window}")
        if sinks < 0 or (sinks and window is None):
            raise ValueError("sinks are the first tokens that stay visible next to a window")
        self.head_dim, self.num_kv_heads, self.codes, self.block = head_dim, num_kv_heads, codes, block
        self.window, self.sinks = window, sinks
        self.offset = 0                # tokens seen
        self._dropped = 0              # of them no longer stored: whole blocks between the sinks and the window
        self._store: tuple | None = None

    # ---- storage ------------------------------------------------------------------------------------
    @property
    def _length(self) -> int:
        return self.offset - self._dropped

    def _sink_end(self) -> int:
        return -(-self.sinks // self.block) * self.block

    def _allocate(self, b: int, h: int, cap: int, dtype, device) -> tuple:
        codes = torch.int8 if self.codes == "int8" else torch.float8_e4m3fn
        out = []
        with torch.inference_mode(False):                      # (the storage outlives the mode that its first tokens came in, and is written to in any)
            for _ in range(2):
                out += [torch.empty((b, h, cap, self.head_dim), dtype=codes, device=device), torch.empty((b, h, cap // self.block), dtype=torch.float32, device=device)]
            return tuple(out + [torch.empty((b, h, self.block, self.head_dim), dtype=dtype, device=device) for _ in range(2)])

    def _reserve(self, keys: torch.Tensor, t: int) -> None:
        """Room for the whole blocks that ``t`` more tokens fill: drops what no query can see any more, or grows."""
        n = self.block
        if self._store is None:
            if keys.dim() != 4 or keys.shape[3] != self.head_dim or keys.shape[1] != self.num_kv_heads:
                raise ValueError(f"tokens must be (B, {self.num_kv_heads}, T, {self.head_dim}), got {tuple(keys.shape)}")
            cap = max(-(-(t + n) // n) * n, self.step)
            self._store = self._allocate(keys.shape[0], keys.shape[1], -(-cap // n) * n, keys.dtype, keys.device)
            return
        cap = self._store[0].shape[2]
        need = (self._length + t) // n * n
        if need <= cap:
            return
        first, last = self._sink_end(), self._length // n * n                  # (blocks [first, last) are the window's)
        drop = 0 if self.window is None else max(0, (self._length - self.window + 1) // n * n - first)
        if drop and 2 * (need - drop) <= cap:                                  # (half of the storage at least comes free: copies stay rare)
            for i in (0, 2):
                codes, scales = self._store[i].view(torch.int8), self._store[i + 1]
                codes[:, :, first:last - drop] = codes[:, :, first + drop:last].clone()
                scales[:, :, first // n:(last - drop) // n] = scales[:, :, (first + drop) // n:last // n].clone()
            self._dropped += drop
            return
        keep = last - drop if drop else last
        new = self._allocate(*self._store[0].shape[:2], -(-max(need - drop, 2 * cap if not drop else 2 * (need - drop)) // n) * n, self._store[4].dtype, self._store[0].device)
        for i in (0, 2):
            old, to = self._store[i].view(torch.int8), new[i].view(torch.int8)
            to[:, :, :min(first, keep)] = old[:, :, :min(first, keep)]
            to[:, :, first:keep] = old[:, :, first + drop:last]
            new[i + 1][:, :, :min(first, keep) // n] = self._store[i + 1][:, :, :min(first, keep) // n]
            new[i + 1][:, :, first // n:keep // n] = self._store[i + 1][:, :, (first + drop) // n:last // n]
        self._store = (*new[:4], *self._store[4:])
        self._dropped += drop

    # ---- protocol -------------------------------------------------------------------------------------
    def update(self, keys: torch.Tensor, values: torch.Tensor) -> None:
        """Append (B, H, T, D) tokens."""
        _lib.require_cuda(keys, values)
        t = keys.shape[2] if keys.dim() == 4 else 0
        fresh = self._store is None
        self._reserve(keys, t)
        try:
            write_blocks(keys, values, *self._store, self._length)
        except Exception:
            if fresh:                                          # (the storage took its type and batch from tokens that were refused)
                self._store = None
            raise
        self.offset += t

    def attend(self, queries: torch.Tensor, scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
        """softmax(scale q K^T) V for the last T_q tokens: (B, H_q, T_q, D), or (B, H_q, D) for the last one; ``out`` receives the result."""
        if self._store is None or self.offset == 0:
            raise ValueError("attend on an empty cache")
        if queries.dim() == 3:
            res = self.attend(queries.unsqueeze(2), scale, None if out is None else out.view(*queries.shape[:2], 1, queries.shape[2]))
            return out if out is not None else res.squeeze(2)
        if self._dropped and self._length - queries.shape[2] - self.window + 1 < self._sink_end():
            raise ValueError(f"the window of the first of {queries.shape[2]} query tokens is no longer stored: attend to the tokens of the last update")
        return attend_blocks(queries, *self._store, self._length, window=self.window, sinks=self.sinks, scale=scale, out=out)

    def decode_step(self, queries: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
        """``update`` with one token, then ``attend``: one launch unless the token completes a block."""
        if keys.dim() != 4 or keys.shape[2] != 1 or (queries.dim() == 4 and queries.shape[2] != 1):
            self.update(keys, values)
            return self.attend(queries, scale, out)
        if queries.dim() == 3:
            res = self.decode_step(queries.unsqueeze(2), keys, values, scale, None if out is None else out.view(*queries.shape[:2], 1, queries.shape[2]))
            return out if out is not None else res.squeeze(2)
        _lib.require_cuda(queries, keys, values)
        fresh = self._store is None
        self._reserve(keys, 1)
        try:
            res = attend_blocks(queries, *self._store, self._length, window=self.window, sinks=self.sinks, scale=scale, out=out, new=(keys, values))
        except Exception:
            if fresh:
                self._store = None
            raise
        self.offset += 1
        return res

    def update_and_fetch(self, keys: torch.Tensor, values: torch.Tensor):
        """Append, and return dense, of the tokens' type, what queries of the new tokens may see: all tokens, or with a window the first ``sinks`` of them
        and those from the first new token's window on.  Which of these each query sees, ``make_mask`` says, asked before this call."""
        if self.window is None:
            self.update(keys, values)
            return read_blocks(*self._store, self._length)
        if not (keys.is_cuda and values.is_cuda):
            raise NotImplementedError("mlx_turboquant_b200 runs on CUDA tensors only; a cache with a window has nothing to return on " + str(keys.device))
        low, sinks = self._seen_from()
        self.update(keys, values)
        return tuple(self._visible(x, low - self._dropped, sinks) for x in read_blocks(*self._store, self._length))

    def _seen_from(self) -> tuple[int, int]:
        """The first token that the next one sees through its window, and how many sinks lie before that."""
        low = max(0, self.offset - self.window + 1)
        return low, min(self.sinks, low)

    @staticmethod
    def _visible(x: torch.Tensor, at: int, sinks: int) -> torch.Tensor:
        return x[:, :, at - sinks:] if at == sinks or sinks == 0 else torch.cat([x[:, :, :sinks], x[:, :, at:]], dim=2)

    def make_mask(self, N: int, offset: int = 0, return_array: bool = False, window_size: int | None = None) -> Any | None:
        """The mask of ``N`` new tokens over what ``update_and_fetch`` returns for them; asked before that call.  ``None`` for a single token, ``"causal"`` where
        that is all, otherwise a boolean tensor (N, tokens returned), true where a query sees a token (before the first tokens on the current device).  ``attend`` needs none: the window is part of it.
        ``window_size`` may be the window, or what the model's own cache calls its size: window and sinks together."""
        if window_size is not None and (self.window is None or window_size not in (self.window, self.window + self.sinks)):
            raise NotImplementedError(f"this cache has a window of {self.window} and {self.sinks} sinks, not {window_size}")
        if N == 1 and not return_array:
            return None
        if self.window is None or (not return_array and self.offset + N - self.window <= self.sinks):
            return "causal"
        return window_mask(self.offset, N, self.window, self.sinks, torch.device("cuda") if self._store is None else self._store[0].device)

    def size(self) -> int:
        return self.offset

    def empty(self) -> bool:
        return self.offset == 0

    def is_trimmable(self) -> bool:
        return False

    @property
    def nbytes(self) -> int:
        """Bytes of the stored tokens: codes, scales and the tail's rows."""
        if self._store is None:
            return 0
        b, h, _, d = self._store[0].shape
        whole, rest = self._length // self.block, self._length % self.block
        return 2 * b * h * (whole * (self.block * d + 4) + rest * d * self._store[4].element_size())

    # ---- checkpoint -----------------------------------------------------------------------------------
    @property
    def state(self):
        """k_codes, k_scales, v_codes, v_scales (whole blocks only), k_tail, v_tail; or six ``None``."""
        if self._store is None:
            return (None,) * 6
        whole = self._length // self.block
        return tuple(t[:, :, :whole * self.block] if i in (0, 2) else t[:, :, :whole] if i in (1, 3) else t for i, t in enumerate(self._store))

    @state.setter
    def state(self, v):
        if len(v) != 6:
            raise ValueError(f"state must have 6 elements, got {len(v)}")
        if all(t is None for t in v):
            self._store, self.offset, self._dropped = None, 0, 0
            return
        _lib.require_cuda(*v)
        with torch.inference_mode(False):
            store = tuple(t.clone(memory_format=torch.contiguous_format) for t in v)   # (the cache that the state came from goes on writing to its own)
        _store(*store, 0)
        if store[4].shape[2] != self.block or store[0].shape[3] != self.head_dim or store[0].dtype is not (torch.int8 if self.codes == "int8" else torch.float8_e4m3fn):
            raise ValueError("the state is of a cache with other blocks, codes or head_dim")
        self._store = store

    @property
    def meta_state(self):
        return {"offset": str(self.offset), "dropped": str(self._dropped), "head_dim": str(self.head_dim), "codes": self.codes, "block": str(self.block),
                "window": "" if self.window is None else str(self.window), "sinks": str(self.sinks)}

    @meta_state.setter
    def meta_state(self, v):
        offset, dropped = int(v["offset"]), int(v["dropped"])
        if self._store is not None and (offset - dropped) // self.block * self.block > self._store[0].shape[2]:
            raise ValueError(f"{offset - dropped} tokens in storage for {self._store[0].shape[2]}")
        self.offset, self._dropped = offset, dropped
        self.window, self.sinks = (int(v["window"]) if v["window"] else None), int(v["sinks"])
