"""The token-generation operators in float64, row by row, and how far float32 arithmetic may be from them.

Each function returns its values and, beside them, the magnitudes that a bound on a float32
computation's error is taken relative to: the sums of the absolute values of what is added up.
"""

from __future__ import annotations

import numpy as np
import torch

from oracle import quantize as oq


def _pairs(width: int, half: int, interleaved: bool) -> tuple[torch.Tensor, torch.Tensor]:
    i = torch.arange(half)
    return (2 * i, 2 * i + 1) if interleaved else (i, i + half)


def turn(x, positions, frequencies, interleaved, back=False):
    """x [tokens, heads, width] float64 with its column pairs turned; and each value's pair's |a| + |b|."""
    a, b = _pairs(x.shape[-1], frequencies.numel(), interleaved)
    angle = positions.double()[:, None, None] * frequencies * (-1 if back else 1)
    out, size = x.clone(), x.abs().clone()
    out[..., a] = x[..., a] * angle.cos() - x[..., b] * angle.sin()
    out[..., b] = x[..., a] * angle.sin() + x[..., b] * angle.cos()
    size[..., a] = size[..., b] = x[..., a].abs() + x[..., b].abs()
    return out, size


def norm_rotate(x, gain, positions, frequencies, epsilon, interleaved):
    x, gain = x.cpu().double(), gain.cpu().double()
    y = x / (x.square().mean(-1, keepdim=True) + epsilon).sqrt() * gain
    return turn(y, positions.cpu(), frequencies.cpu(), interleaved)


def norm_rotate_backward(grad, x, gain, positions, frequencies, epsilon, interleaved):
    """((dx, its magnitudes), (dgain, its magnitudes))."""
    x, gain = x.cpu().double(), gain.cpu().double()
    d, size = turn(grad.cpu().double(), positions.cpu(), frequencies.cpu(), interleaved, back=True)
    r = 1 / (x.square().mean(-1, keepdim=True) + epsilon).sqrt()
    e, e_size = d * gain, size * gain.abs()
    dx = r * (e - x * r * r * (e * x).mean(-1, keepdim=True))
    dx_size = r * (e_size + x.abs() * r * r * (e_size * x.abs()).mean(-1, keepdim=True))
    return (dx, dx_size), ((d * x * r).sum((0, 1)), (size * x.abs() * r).sum((0, 1)))


def quantise(x):
    """Codes (int8) and scales (float32) of rows [..., width] by tgc's rule."""
    flat = x.detach().cpu().float().reshape(-1, x.shape[-1])
    q, s = oq.quantise_rows(flat.numpy())
    return torch.from_numpy(np.ascontiguousarray(q)).reshape(x.shape), torch.from_numpy(np.ascontiguousarray(s)).reshape(x.shape[:-1])


def places(table, starts, offsets, tokens, page):
    """For each token row: (sequence, row in it, first row, rows, page, place), or None where it belongs to no sequence."""
    table, starts = table.cpu(), starts.cpu().tolist()
    batch = table.shape[0]
    ends = offsets.cpu().tolist() if offsets is not None else [b * (tokens // batch) for b in range(batch + 1)]
    found = [None] * tokens
    for b in range(batch):
        for t in range(ends[b], ends[b + 1]):
            position = starts[b] + t - ends[b]
            inside = 0 <= position and position // page < table.shape[1]
            at = int(table[b, position // page]) if inside else -1
            found[t] = (b, t - ends[b], ends[b], ends[b + 1] - ends[b], at, position % page)
    return found


def attention(queries, keys, key_scales, values, value_scales, table, starts, offsets=None, visible=None, scale=1.0, cap=0.0):
    """Every token's attention, its magnitudes sum_j p_j |v_j|, and a bound's worth of its scores:
    the largest scale * sum_i |q_i k_i| of a seen key. Rows of no sequence are NaN."""
    q = queries.cpu().double()
    pages, heads, page, width = keys.shape
    tokens, q_heads, _ = q.shape
    group = q_heads // heads
    k = keys.cpu().double() * key_scales.cpu().double()[..., None]
    v = values.cpu().double() * value_scales.cpu().double()[..., None]
    table, bits = table.cpu(), visible.cpu().tolist() if visible is not None else None
    out = torch.full(q.shape, float("nan"), dtype=torch.float64)
    size, score_size = torch.zeros_like(out), torch.zeros(tokens, q_heads, 1, dtype=torch.float64)
    start_of = starts.cpu().tolist()
    for t, place in enumerate(places(table, starts, offsets, tokens, page)):
        if place is None:
            continue
        b, i, _, rows, _, _ = place
        start = start_of[b]
        if bits is None:
            seen = list(range(max(0, start + i + 1)))
        else:
            seen = list(range(max(0, start))) + [start + j for j in range(min(rows, 64)) if bits[t] >> j & 1 and start + j >= 0]
        seen = [j for j in seen if j // page < table.shape[1] and 0 <= table[b, j // page] < pages]
        out[t] = 0.0
        if not seen:
            continue
        j = torch.tensor(seen)
        at, place_in = table[b, j // page].long(), j % page
        for h in range(heads):
            kk, vv = k[at, h, place_in], v[at, h, place_in]
            qq = q[t, h * group:(h + 1) * group]
            s = qq @ kk.T * scale
            score_size[t, h * group:(h + 1) * group, 0] = (qq.abs() @ kk.abs().T * abs(scale)).amax(-1)
            if cap:
                s = cap * torch.tanh(s / cap)
            p = torch.softmax(s, -1)
            out[t, h * group:(h + 1) * group] = p @ vv
            size[t, h * group:(h + 1) * group] = p @ vv.abs()
    return out, size, score_size
