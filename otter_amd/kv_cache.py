"""K/V history held in 4 or 8 bits: the cache object, and its kernels as ``torch.ops.otter_hip.*`` operators.

The policy's fp32 history costs 9 kB a position and layer (q | k | v rows of 768) and its kernels end at 64 positions.  A
:class:`KVCache` holds keys and values only, in blocks of 32 numbers with a power of two as scale: 0.8 kB a position and layer
in 4 bits (e2m1 codes), 1.6 kB in 8 (e4m3), and histories of any length.  Numbers are quantised as they are written
(:meth:`KVCache.write`, or :meth:`KVCache.step` together with the attention of a single new position), attended to in that form
(:meth:`KVCache.attend`), and read back (:meth:`KVCache.read`).  The same cache semantics as ``otter/policy/otter.py:153-175`` /
``transformer.py:76-104`` apply: one window per episode, causal attention over the window's earlier positions.

Accuracy is the format's, half a step of the code: a number that is stored in 4 bits is within a fifth of itself if it is at least a
sixth of its block's largest, in 8 bits within 2^-4 of itself if it is at least 2^-14 of the largest; smaller ones are within a
quarter of 2^e (2^-10 of 2^e), e the block's exponent.  The arithmetic on the stored numbers is fp32 for fp32 activations; for 16-bit ones scores
and sums are fp32 and a weight is held to 2^-16, or 2^-11 for bf16 activations with several steps and more than 32 columns (steps x
query heads of a key head), below the output's own rounding (2^-8).

| operator | arithmetic |
|---|---|
| ``kv_cache_write`` | keys and values -> blocks of codes and scales |
| ``kv_cache_read`` | blocks -> numbers |
| ``attn_cache`` | ``softmax(q k^T / sqrt(d)) v`` over the cached positions, one or many new positions a row |
| ``attn_cache_rows`` | one new position a row: write and attend in one call |
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import ops
from .torch_ops import _CODE, _DT

Tensor = torch.Tensor
_lib = torch.library.Library("otter_hip", "FRAGMENT")

_SCHEMAS = (
    "kv_cache_write(Tensor k, Tensor v, Tensor(a!) codes, Tensor(b!) scales, Tensor? pos, Tensor? idx, Tensor? count) -> ()",
    "kv_cache_read(Tensor codes, Tensor scales, int head_dim, int steps, Tensor? pos, Tensor? idx, Tensor? count, int n_rows, int dtype) -> (Tensor, Tensor)",
    "attn_cache(Tensor q, Tensor codes, Tensor scales, Tensor? pos, Tensor? idx, Tensor? count, bool causal, int window, float? scale, int? max_len) -> Tensor",
    "attn_cache_rows(Tensor q, Tensor k, Tensor v, Tensor(a!) codes, Tensor(b!) scales, Tensor? pos, Tensor? idx, int window, float? scale, int? max_len) "
    "-> Tensor",
)
for _s in _SCHEMAS:
    _lib.define(_s)
OP_NAMES = tuple(s.split("(", 1)[0] for s in _SCHEMAS)


def _kv_cache_write(k, v, codes, scales, pos, idx, count):
    ops.kv_cache_write(k, v, codes, scales, pos, idx, count)


def _kv_cache_read(codes, scales, head_dim, steps, pos, idx, count, n_rows, dtype):
    return ops.kv_cache_read(codes, scales, head_dim, steps, pos, idx, count, n_rows=None if n_rows < 0 else n_rows, dtype=_DT[dtype])


def _attn_cache(q, codes, scales, pos, idx, count, causal, window, scale, max_len):
    return ops.attn_cache(q, codes, scales, pos, idx, count, causal=causal, window=window, scale=scale, max_len=max_len)


def _attn_cache_rows(q, k, v, codes, scales, pos, idx, window, scale, max_len):
    return ops.attn_cache_rows(q, k, v, codes, scales, pos, idx, window=window, scale=scale, max_len=max_len)


for _name in OP_NAMES:
    _lib.impl(_name, globals()["_" + _name], "CUDA")            # "CUDA" is PyTorch's dispatch key for HIP devices on ROCm builds


@torch.library.register_fake("otter_hip::kv_cache_write")
def _(k, v, codes, scales, pos, idx, count):
    return None


@torch.library.register_fake("otter_hip::kv_cache_read")
def _(codes, scales, head_dim, steps, pos, idx, count, n_rows, dtype):
    n = idx.shape[0] if idx is not None else (codes.shape[1] if n_rows < 0 else n_rows)
    shape = (n, steps, codes.shape[2], head_dim)
    return codes.new_empty(shape, dtype=_DT[dtype]), codes.new_empty(shape, dtype=_DT[dtype])


@torch.library.register_fake("otter_hip::attn_cache")
def _(q, codes, scales, pos, idx, count, causal, window, scale, max_len):
    return q.new_empty(q.shape)


@torch.library.register_fake("otter_hip::attn_cache_rows")
def _(q, k, v, codes, scales, pos, idx, window, scale, max_len):
    return q.new_empty(q.shape)


class KVCache:
    """Keys and values of ``episodes`` windows of ``capacity`` positions, ``heads`` key heads of ``head_dim`` (32, 64, 96 or 128)
    numbers, in ``bits`` = 4 or 8.  Starts as zeros.  The rows of a call are episodes: row i of its operands is episode ``idx[i]``
    (int32 on the device; None: episode i), and its steps follow on window position ``pos[episode]`` (int32, one per episode;
    None: 0).  ``max_len``: no window is longer than that (it sizes the launch; positions from it on are not looked at)."""

    def __init__(self, episodes: int, heads: int, capacity: int, head_dim: int, bits: int = 4, device="cuda"):
        if bits not in (4, 8):
            raise ValueError(f"KVCache: {bits} bits; 4 or 8")
        if head_dim % 32 != 0 or not 32 <= head_dim <= 128:
            raise ValueError(f"KVCache: head_dim {head_dim} must be 32, 64, 96 or 128")
        if episodes < 0 or heads < 1 or capacity < 1:
            raise ValueError(f"KVCache: {episodes} episodes, {heads} heads, {capacity} positions")
        self.bits, self.head_dim = bits, head_dim
        self.codes = torch.zeros(2, episodes, heads, capacity, head_dim * bits // 8, dtype=torch.uint8, device=device)
        self.scales = torch.zeros(2, episodes, heads, capacity, 4, dtype=torch.uint8, device=device)
        ns = torch.ops.otter_hip
        self._write, self._read = ns.kv_cache_write.default, ns.kv_cache_read.default
        self._attend, self._step = ns.attn_cache.default, ns.attn_cache_rows.default

    @property
    def episodes(self) -> int:
        return self.codes.shape[1]

    @property
    def heads(self) -> int:
        return self.codes.shape[2]

    @property
    def capacity(self) -> int:
        return self.codes.shape[3]

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel()

    def write(self, k: Tensor, v: Tensor, pos: Optional[Tensor] = None, idx: Optional[Tensor] = None, count: Optional[Tensor] = None) -> None:
        """k, v (rows, steps, heads, head_dim) into the cache; ``count`` (rows,): how many of the steps exist."""
        self._write(k, v, self.codes, self.scales, pos, idx, count)

    def read(self, steps: int, pos: Optional[Tensor] = None, idx: Optional[Tensor] = None, count: Optional[Tensor] = None,
             dtype=torch.float32) -> Tuple[Tensor, Tensor]:
        """(k, v), each (rows, steps, heads, head_dim) in ``dtype``; what the cache does not hold reads as zeros."""
        return self._read(self.codes, self.scales, self.head_dim, steps, pos, idx, count, -1, _CODE[dtype])

    def attend(self, q: Tensor, pos: Optional[Tensor] = None, idx: Optional[Tensor] = None, count: Optional[Tensor] = None, *,
               causal: bool = True, window: int = 0, scale: Optional[float] = None, max_len: Optional[int] = None) -> Tensor:
        """q (rows, steps, q_heads, head_dim), already written steps -> their attention outputs (see ``ops.attn_cache``)."""
        return self._attend(q, self.codes, self.scales, pos, idx, count, causal, window, scale, max_len)

    def step(self, q: Tensor, k: Tensor, v: Tensor, pos: Optional[Tensor] = None, idx: Optional[Tensor] = None, *, window: int = 0,
             scale: Optional[float] = None, max_len: Optional[int] = None) -> Tensor:
        """One new position a row: k, v (rows, heads, head_dim) are written and q (rows, q_heads, head_dim) attends to them and to
        everything before."""
        return self._step(q, k, v, self.codes, self.scales, pos, idx, window, scale, max_len)
