"""Streaming attention on the GPU (tgc/analysis/attention.py:97-137).

``streaming_attention(queries, keys, values, block)`` takes float32 CUDA matrices and returns
the same function tgc's version computes, from one fused kernel (``tgcb_streaming_attention_f32``):
one pass over the keys with the running maximum and sum rescaled as blocks arrive, the score
matrix never written to memory. ``block`` is checked as tgc checks it; the kernel's own key
block is 64, which moves rounding, not the result. ``AttentionShape`` mirrors tgc's
(attention.py:44-77).

``cached_attention`` is the same function over a ``tgcb.kv_cache.QuantisedCache``, for the tokens a
program generates: all heads of a batch of sequences in one call, query heads sharing key heads, single tokens,
pieces of prompts and trees of drafted tokens.
"""

from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass

import torch

from tgcb import _lib, heads, kv_cache
from tgcb.errors import ConfigError

WIDTHS = (16, 32, 64, 128)


@dataclass(frozen=True)
class AttentionShape:
    sequence: int
    width: int

    def __post_init__(self) -> None:
        if min(self.sequence, self.width) < 1:
            raise ConfigError(f"a head cannot be {self.sequence} by {self.width}")

    @property
    def input_elements(self) -> int:
        return 3 * self.sequence * self.width

    @property
    def score_elements(self) -> int:
        return self.sequence * self.sequence

    @property
    def arithmetic(self) -> float:
        """Multiply-adds in the two products (attention.py:67-70)."""
        return 4.0 * self.sequence * self.sequence * self.width

    def as_dict(self) -> dict:
        return {"sequence": self.sequence, "width": self.width, "inputs": self.input_elements,
                "scores": self.score_elements}


def streaming_attention_into(queries: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, out: torch.Tensor,
                             stream=None) -> None:
    for name, t in (("queries", queries), ("keys", keys), ("values", values), ("out", out)):
        if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype != torch.float32 or t.dim() != 2:
            raise ConfigError(f"{name} must be a float32 CUDA matrix")
        if not t.is_contiguous():
            raise ConfigError(f"{name} must be contiguous")
    sq, width = queries.shape
    sk = keys.shape[0]
    if width not in WIDTHS:
        raise ConfigError(f"the kernel takes widths {WIDTHS}, got {width}")
    if keys.shape[1] != width or values.shape != keys.shape or out.shape != queries.shape:
        raise ConfigError("keys and values must be [keys, width] and out [queries, width]")
    if sq == 0 or sk == 0:
        raise ConfigError("a head needs at least one query and one key")
    _lib.ensure_device(queries.device.index)
    s = stream if stream is not None else torch.cuda.current_stream(queries.device)
    rc = _lib.load().tgcb_streaming_attention_f32(
        ctypes.c_void_p(queries.data_ptr()), ctypes.c_void_p(keys.data_ptr()), ctypes.c_void_p(values.data_ptr()),
        sq, sk, width, ctypes.c_void_p(out.data_ptr()), ctypes.c_void_p(s.cuda_stream),
    )
    _lib.check(rc, "tgcb_streaming_attention_f32")


def streaming_attention(queries: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, block: int = 128) -> torch.Tensor:
    """softmax(queries keys^T / sqrt(width)) values in one pass over the keys."""
    if block < 1:
        raise ConfigError(f"a block has to hold something, got {block}")
    q, k, v = (t.contiguous() for t in (queries, keys, values))
    out = torch.empty_like(q)
    streaming_attention_into(q, k, v, out)
    return out


def cached_attention(queries: torch.Tensor, cache: kv_cache.QuantisedCache, table: torch.Tensor, starts: torch.Tensor,
                     offsets: torch.Tensor | None = None, *, visible: torch.Tensor | None = None, scale: float | None = None,
                     cap: float | None = None, out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """Attention of each token of a call over its sequence's cached positions.

    ``queries`` [tokens, q_heads, width] with q_heads a multiple of the cache's heads (query head h
    reads key head h // (q_heads // kv_heads)); ``table``, ``starts`` and ``offsets`` as for
    ``QuantisedCache.append``, which must have stored the call's own keys and values before. Row i of
    a sequence sees positions 0 .. starts + i. With ``visible`` (int64 [tokens]) it sees positions 0 .. starts - 1
    and, among the call's own rows of its sequence, row j where bit j is set: a tree's ancestors
    and the token itself. At most 64 rows a sequence can be named so.

    score = scale * q.k (``scale`` None: 1 / sqrt(width)), then with ``cap`` (at most 1e30) cap * tanh(score / cap).
    A token that sees nothing gets zeros. ``out`` (not the queries) receives the result; rows of no sequence are not written.
    A kernel that waits in vain for 4 s gives up, with ``out`` unfinished; ``cache.check`` raises for it.
    """
    if not isinstance(cache, kv_cache.QuantisedCache):
        raise ConfigError("cached_attention reads a QuantisedCache")
    heads.check_rows("queries", queries)
    index = cache.index
    if queries.get_device() != index:
        raise ConfigError(f"queries must be on {cache.device}, where the cache is")
    tokens, q_heads, width = queries.shape
    if width != cache.width or q_heads < 1 or q_heads % cache.kv_heads:
        raise ConfigError(f"queries must be [tokens, a multiple of {cache.kv_heads} heads, {cache.width}], got {tuple(queries.shape)}")
    b = cache.batch_of(table, starts, offsets, tokens)
    if visible is not None:
        heads.check_vector("visible", visible, tokens, (torch.int64,), index)
        if offsets is None and tokens > 64 * table.shape[0]:
            raise ConfigError(f"a tree has at most 64 tokens, got {tokens // table.shape[0]} a sequence")
    scale = 1.0 / math.sqrt(width) if scale is None else float(scale)
    cap = 0.0 if cap is None else float(cap)
    if not math.isfinite(scale) or not math.isfinite(cap) or cap < 0:
        raise ConfigError(f"the scale has to be finite and the cap finite and not negative, got {scale} and {cap}")
    if max(abs(scale), abs(scale) / cap if cap else 0.0, cap) > 1e30:
        raise ConfigError(f"a scale of {scale} under a cap of {cap} is beyond float32")
    if out is not None:
        heads.check_rows("out", out, queries)
        if out.shape != queries.shape:
            raise ConfigError(f"out must have the shape {tuple(queries.shape)}, got {tuple(out.shape)}")
        heads.check_written("out", out)
        heads.check_apart("out", out, "queries", queries)
    lib = _lib.load()
    need = lib.tgcb_cached_attention_scratch_bytes(cache.desc, b, q_heads)
    with heads.on_stream(index, stream):
        if out is None:
            out = heads.empty(queries)
        scratch = torch.empty(need, dtype=torch.uint8, device=cache.device) if need else None
    with heads.on_device(index):
        rc = lib.tgcb_cached_attention(
            cache.desc, b, heads.DTYPES[queries.dtype], q_heads, _lib.Heads(*heads.rows(queries)),
            visible.data_ptr() if visible is not None else None, scale, cap, _lib.Heads(*heads.rows(out)),
            scratch.data_ptr() if need else None, need, heads.raw(index, stream),
        )
    _lib.check(rc, "tgcb_cached_attention")
    return out
