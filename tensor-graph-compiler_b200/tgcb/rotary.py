"""RMS norm of query and key heads with the position rotation in the same pass.

For each head of each token, ``y = x / sqrt(mean(x^2) + epsilon) * gain`` (the arithmetic of
``tgcb.normalisation.rms_norm`` along one head) and then each of the first ``len(frequencies)``
column pairs turned by ``position * frequency`` radians: pairs (i, i + len(frequencies)), or with
``interleaved`` (2i, 2i + 1). One launch takes queries and keys together, as slices of a
projection's output if they lie there. Angles are taken in float64, so far positions keep theirs; everything else
is float32, rounded once to the rows' type.

``norm_rotate`` returns new tensors, ``norm_rotate_into`` writes into given ones (the inputs
themselves, if wanted). ``norm_rotate_backward`` returns the gradients of all four inputs; the
gains' gradients are summed over tokens and heads in a fixed order. Nothing is recorded for
``torch.autograd``: as elsewhere in this package a backward pass is called by its name.
"""

from __future__ import annotations

import torch

from tgcb import _lib, heads
from tgcb.errors import ConfigError

MAX_WIDTH = 1024
_NONE = (0, 0, 0)


def frequencies(rotary: int, base: float = 10000.0, device=None) -> torch.Tensor:
    """base^(-2i / rotary) for i < rotary / 2, in float64: the usual geometric frequencies."""
    if rotary < 2 or rotary % 2:
        raise ConfigError(f"a rotation takes pairs of columns, got {rotary}")
    if base <= 0:
        raise ConfigError(f"the base has to be positive, got {base}")
    half = rotary // 2
    return base ** (-torch.arange(half, dtype=torch.float64, device=device or "cuda") / half)


def _check(queries, keys, query_gain, key_gain, positions, freqs, epsilon) -> None:
    heads.check_rows("queries", queries)
    heads.check_rows("keys", keys, queries)
    tokens, q_heads, width = queries.shape
    k_tokens, k_heads, k_width = keys.shape
    if k_tokens != tokens or k_width != width:
        raise ConfigError("queries and keys must have the same tokens and width")
    if q_heads < 1 or k_heads < 1:
        raise ConfigError("there has to be at least one query head and one key head")
    if not 2 <= width <= MAX_WIDTH:
        raise ConfigError(f"a head's width must be from 2 to {MAX_WIDTH}, got {width}")
    index = queries.get_device()
    heads.check_vector("query_gain", query_gain, width, (torch.float32, queries.dtype), index)
    heads.check_vector("key_gain", key_gain, width, (query_gain.dtype,), index)
    heads.check_vector("positions", positions, tokens, (torch.int32, torch.int64), index)
    half = freqs.shape[0] if isinstance(freqs, torch.Tensor) and freqs.dim() == 1 else 0
    if not 1 <= half <= width // 2:
        raise ConfigError(f"frequencies must be a vector of 1 to {width // 2} values for heads of width {width}")
    heads.check_vector("frequencies", freqs, half, (torch.float64,), index)
    if not 1e-37 <= epsilon < 1e38:
        raise ConfigError(f"the epsilon has to be a positive float32, got {epsilon}")


def _desc(queries, keys, query_gain, key_gain, positions, freqs, epsilon, interleaved, out, grads=(_NONE, _NONE),
          gain_grads=(0, 0), scratch=(0, 0)) -> _lib.RotaryDesc:
    tokens, q_heads, width = queries.shape
    return _lib.RotaryDesc.of(
        heads.DTYPES[queries.dtype], heads.DTYPES[query_gain.dtype], positions.element_size(), bool(interleaved), tokens,
        q_heads, keys.shape[1], width, 2 * freqs.shape[0], epsilon, positions.data_ptr(), freqs.data_ptr(),
        query_gain.data_ptr(), key_gain.data_ptr(), *heads.rows(queries), *heads.rows(keys), *grads[0], *grads[1],
        *heads.rows(out[0]), *heads.rows(out[1]), *gain_grads, *scratch,
    )


def _check_outputs(out: tuple, names: tuple, inputs: tuple) -> None:
    """Outputs shaped like the rows, apart from each other and from all inputs but their own."""
    for name, o, like in zip(names, out, inputs, strict=True):
        heads.check_rows(name, o, like[0][1])
        if o.shape != like[0][1].shape:
            raise ConfigError(f"{name} must have the shape {tuple(like[0][1].shape)}, got {tuple(o.shape)}")
        heads.check_written(name, o)
        for side in inputs:
            for other_name, other in side:
                heads.check_apart(name, o, other_name, other, same_allowed=side is like)
    heads.check_apart(names[0], out[0], names[1], out[1])


def norm_rotate_into(queries: torch.Tensor, keys: torch.Tensor, query_gain: torch.Tensor, key_gain: torch.Tensor,
                     positions: torch.Tensor, frequencies: torch.Tensor, query_out: torch.Tensor, key_out: torch.Tensor, *,
                     epsilon: float = 1e-5, interleaved: bool = False, stream=None) -> None:
    _check(queries, keys, query_gain, key_gain, positions, frequencies, epsilon)
    _check_outputs((query_out, key_out), ("query_out", "key_out"), ((("queries", queries),), (("keys", keys),)))
    _run(queries, keys, query_gain, key_gain, positions, frequencies, epsilon, interleaved, (query_out, key_out), stream)


def _run(queries, keys, query_gain, key_gain, positions, freqs, epsilon, interleaved, out, stream) -> None:
    d = _desc(queries, keys, query_gain, key_gain, positions, freqs, epsilon, interleaved, out)
    index = queries.get_device()
    with heads.on_device(index):
        _lib.check(_lib.load().tgcb_norm_rotate(d, heads.raw(index, stream)), "tgcb_norm_rotate")


def norm_rotate(queries: torch.Tensor, keys: torch.Tensor, query_gain: torch.Tensor, key_gain: torch.Tensor,
                positions: torch.Tensor, frequencies: torch.Tensor, *, epsilon: float = 1e-5, interleaved: bool = False,
                stream=None) -> tuple[torch.Tensor, torch.Tensor]:
    """The normed and turned queries and keys, [tokens, heads, width] each.

    ``queries`` and ``keys`` share their type, tokens and width; the gains are float32 or of that
    type, [width]; ``positions`` int32 or int64, [tokens]; ``frequencies`` float64, [1 .. width / 2].
    """
    _check(queries, keys, query_gain, key_gain, positions, frequencies, epsilon)
    with heads.on_stream(queries.get_device(), stream):
        out = heads.empty(queries), heads.empty(keys)
    _run(queries, keys, query_gain, key_gain, positions, frequencies, epsilon, interleaved, out, stream)
    return out


def norm_rotate_backward(query_grad: torch.Tensor, key_grad: torch.Tensor, queries: torch.Tensor, keys: torch.Tensor,
                         query_gain: torch.Tensor, key_gain: torch.Tensor, positions: torch.Tensor, frequencies: torch.Tensor, *,
                         epsilon: float = 1e-5, interleaved: bool = False, out: tuple[torch.Tensor, torch.Tensor] | None = None,
                         stream=None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """Gradients of ``norm_rotate``'s queries, keys, query_gain and key_gain, given those of its outputs.

    ``out`` names where the first two go (each may be its input or its output's gradient itself).
    """
    _check(queries, keys, query_gain, key_gain, positions, frequencies, epsilon)
    index = queries.get_device()
    for name, g, x in (("query_grad", query_grad, queries), ("key_grad", key_grad, keys)):
        heads.check_rows(name, g, x)
        if g.shape != x.shape:
            raise ConfigError(f"{name} must have the shape {tuple(x.shape)}, got {tuple(g.shape)}")
    if out is not None:
        _check_outputs(tuple(out), ("query gradient", "key gradient"),
                       ((("queries", queries), ("query_grad", query_grad)), (("keys", keys), ("key_grad", key_grad))))
    lib, width = _lib.load(), queries.shape[2]
    with heads.on_stream(index, stream):
        if out is None:
            out = heads.empty(queries), heads.empty(keys)
        gains = query_gain.new_empty((2, width))
        scratch = torch.empty(lib.tgcb_norm_rotate_scratch_bytes(width), dtype=torch.uint8, device=queries.device)
    d = _desc(queries, keys, query_gain, key_gain, positions, frequencies, epsilon, interleaved, out,
              (heads.rows(query_grad), heads.rows(key_grad)), (gains.data_ptr(), gains.data_ptr() + width * gains.element_size()),
              (scratch.data_ptr(), scratch.numel()))
    with heads.on_device(index):
        _lib.check(lib.tgcb_norm_rotate_backward(d, heads.raw(index, stream)), "tgcb_norm_rotate_backward")
    return out[0], out[1], gains[0], gains[1]
