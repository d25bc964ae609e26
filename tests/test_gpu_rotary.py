"""Head norms with the position rotation on the GPU, forward and backward, against float64.

Tolerances. The forward pass in float32: the sum of squares of `width` values in at most
width / 32 + 5 additions in a row enters with half its relative error, and about 12 more roundings
(the square root, the quotient, three products, the cosine and sine at 2 ulp, the rotation)
follow, each at most 2^-24 of the pair's |a| + |b|: (width / 64 + 16) * 2^-24. The backward pass takes
twice as many, and the gains' gradients add `rows` terms, at most rows / 592 + 64 of them in a row. Then one rounding to the
rows' type: half of its eps of the value, and for float16 half its smallest subnormal.
"""

from __future__ import annotations

import os

import pytest
import torch
from oracle import generation

from tgcb import heads, rotary
from tgcb.errors import ConfigError

pytestmark = pytest.mark.gpu

U = 2.0**-24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def rounding(dtype):
    return 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2


def close(got, want, size, units, dtype):
    tol = (units * U) * size * (1 + rounding(dtype)) + rounding(dtype) * want.abs() + (2.0**-25 if dtype == torch.float16 else 1e-37)
    off = (got.cpu().double() - want).abs()
    assert bool((off <= tol).all()), f"off by {float((off / tol).max())} tolerances"


def make(tokens, q_heads, k_heads, width, rotary_width, dtype, seed=0, far=5000, gain_dtype=None, position_dtype=torch.int32):
    g = torch.Generator().manual_seed(seed)
    qkv = (torch.randn(tokens, q_heads + 2 * k_heads, width, generator=g) * 2).to(dtype).cuda()
    gains = [(1 + 0.3 * torch.randn(width, generator=g)).to(gain_dtype or dtype).cuda() for _ in range(2)]
    positions = torch.randint(0, far, (tokens,), generator=g).to(position_dtype).cuda()
    return qkv[:, :q_heads], qkv[:, q_heads:q_heads + k_heads], *gains, positions, rotary.frequencies(rotary_width)


SHAPES = [
    # tokens, query heads, key heads, width, rotary columns, interleaved
    (1, 1, 1, 2, 2, False),
    (1, 16, 4, 64, 64, False),
    (7, 8, 8, 128, 128, False),
    (33, 5, 1, 128, 64, True),
    (3, 32, 8, 128, 128, True),
    (5, 3, 2, 80, 80, False),
    (5, 3, 2, 80, 40, False),
    (6, 4, 2, 96, 48, True),
    (9, 2, 1, 256, 256, False),
    (4, 71, 3, 256, 64, True),
    (3, 2, 2, 66, 34, True),
    (2, 3, 1, 1024, 1024, False),
    (2, 1, 1, 7, 6, False),
    (601, 6, 3, 32, 32, False),
    (130, 40, 8, 64, 32, False),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,q_heads,k_heads,width,turned,interleaved", SHAPES)
def test_forward(cuda, tokens, q_heads, k_heads, width, turned, interleaved, dtype):
    q, k, qg, kg, pos, freq = make(tokens, q_heads, k_heads, width, turned, dtype)
    got = rotary.norm_rotate(q, k, qg, kg, pos, freq, interleaved=interleaved)
    for y, x, gain in zip(got, (q, k), (qg, kg), strict=True):
        assert y.dtype == dtype and y.shape == x.shape
        close(y, *generation.norm_rotate(x, gain, pos, freq, 1e-5, interleaved), width / 64 + 16, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,q_heads,k_heads,width,turned,interleaved", SHAPES)
def test_backward(cuda, tokens, q_heads, k_heads, width, turned, interleaved, dtype):
    q, k, qg, kg, pos, freq = make(tokens, q_heads, k_heads, width, turned, dtype, seed=1)
    dq, dk = (torch.randn(x.shape, generator=torch.Generator().manual_seed(2)).to(dtype).cuda() for x in (q, k))
    got = rotary.norm_rotate_backward(dq, dk, q, k, qg, kg, pos, freq, interleaved=interleaved)
    for i, (d, x, gain) in enumerate(((dq, q, qg), (dk, k, kg))):
        (dx, dx_size), (dg, dg_size) = generation.norm_rotate_backward(d, x, gain, pos, freq, 1e-5, interleaved)
        close(got[i], dx, dx_size, width / 32 + 40, dtype)
        rows = x.shape[0] * x.shape[1]
        close(got[2 + i], dg, dg_size, width / 32 + 40 + rows / 592 + 64, dtype)


def test_gradients_against_differences(cuda):
    """The gradients of sum(out * w) against central differences of the float64 definition."""
    q, k, qg, kg, pos, freq = make(3, 2, 1, 32, 16, torch.float32, seed=3)
    wq, wk = torch.randn(q.shape, device="cuda"), torch.randn(k.shape, device="cuda")
    got = rotary.norm_rotate_backward(wq, wk, q, k, qg, kg, pos, freq)

    def loss(x, gain, w):
        return float((generation.norm_rotate(x, gain, pos, freq, 1e-5, False)[0] * w.cpu().double()).sum())

    step = 1e-5  # float64: a difference is off by about step^2 and 1e-16 / step
    for i, (x, gain, w) in enumerate(((q, qg, wq), (k, kg, wk))):
        base_x, base_g = x.cpu().double(), gain.cpu().double()
        for at in [(0, 0, 0), (1, 0, 17), (2, 0, 31)]:
            e = torch.zeros_like(base_x)
            e[at] = step
            slope = (loss(base_x + e, base_g, w) - loss(base_x - e, base_g, w)) / (2 * step)
            assert abs(float(got[i][at]) - slope) < 1e-5 * (1 + abs(slope))
        e = torch.zeros_like(base_g)
        e[5] = step
        slope = (loss(base_x, base_g + e, w) - loss(base_x, base_g - e, w)) / (2 * step)
        assert abs(float(got[2 + i][5]) - slope) < 1e-5 * (1 + abs(slope))


@pytest.mark.parametrize("far", [1 << 20, 1 << 40])
def test_far_positions_keep_their_angles(cuda, far):
    q, k, qg, kg, pos, freq = make(64, 2, 1, 64, 64, torch.float32, far=far, position_dtype=torch.int64)
    pos[:8] = -pos[:8]
    got = rotary.norm_rotate(q, k, qg, kg, pos, freq)
    # the angle itself is a float64 product: a relative 2^-53 of up to `far` radians
    want, size = generation.norm_rotate(q, qg, pos, freq, 1e-5, False)
    close(got[0], want, size, 17 + 4 * far * 2.0**-53 / U, torch.float32)


@pytest.mark.parametrize("dtype", DTYPES)
def test_gains_in_float32_and_positions_of_64_bits(cuda, dtype):
    q, k, qg, kg, pos, freq = make(5, 4, 2, 64, 64, dtype, gain_dtype=torch.float32, position_dtype=torch.int64)
    got = rotary.norm_rotate(q, k, qg, kg, pos, freq)
    close(got[1], *generation.norm_rotate(k, kg, pos, freq, 1e-5, False), 17, dtype)
    grads = rotary.norm_rotate_backward(q, k, q, k, qg, kg, pos, freq)
    assert grads[2].dtype == torch.float32
    close(grads[3], *generation.norm_rotate_backward(k, k, kg, pos, freq, 1e-5, False)[1], 200, torch.float32)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shift", [0, 1])
def test_any_strides_and_in_place(cuda, dtype, shift):
    """Heads before tokens, rows that start off a 16-byte boundary, one row for all heads, and outputs in the inputs' place."""
    base = torch.randn(4, 6, 64 + shift, device="cuda").to(dtype)[:, :, shift:]
    q, k = base.transpose(0, 1)[:, :3], base.transpose(0, 1)[:, 3:]
    _, _, qg, kg, pos, freq = make(6, 1, 1, 64, 64, dtype)
    want = [generation.norm_rotate(x, g, pos, freq, 1e-5, False) for x, g in ((q, qg), (k, kg))]
    got = rotary.norm_rotate(q, k, qg, kg, pos, freq)
    for y, w in zip(got, want, strict=True):
        close(y, *w, 17, dtype)
    rotary.norm_rotate_into(q, k, qg, kg, pos, freq, q, k)
    assert torch.equal(q, got[0]) and torch.equal(k, got[1])
    one = torch.randn(6, 1, 64, device="cuda").to(dtype).expand(6, 5, 64)
    close(rotary.norm_rotate(one, k, qg, kg, pos, freq)[0], *generation.norm_rotate(one, qg, pos, freq, 1e-5, False), 17, dtype)


@pytest.mark.parametrize("width", [64, 66])
def test_backward_in_place(cuda, width):
    q, k, qg, kg, pos, freq = make(9, 4, 2, width, 32, torch.bfloat16)
    dq, dk = torch.randn_like(q), torch.randn_like(k)
    want = rotary.norm_rotate_backward(dq, dk, q, k, qg, kg, pos, freq)
    into_grads = rotary.norm_rotate_backward(dq.clone(), dk.clone(), q, k, qg, kg, pos, freq)
    a, b = dq.clone(), dk.clone()
    got = rotary.norm_rotate_backward(a, b, q, k, qg, kg, pos, freq, out=(a, b))
    assert got[0] is a and all(torch.equal(x, y) for x, y in zip(got, want, strict=True))
    assert all(torch.equal(x, y) for x, y in zip(into_grads, want, strict=True))
    got = rotary.norm_rotate_backward(dq, dk, q, k, qg, kg, pos, freq, out=(q, k))
    assert all(torch.equal(x, y) for x, y in zip(got, want, strict=True))


def test_rows_of_zeros_infinities_and_nan_stay_in_their_rows(cuda):
    q, k, qg, kg, pos, freq = make(6, 2, 1, 64, 64, torch.float32)
    clean = rotary.norm_rotate(q, k, qg, kg, pos, freq)[0]
    q = q.clone()
    q[0, 0] = 0
    q[1, 0, 3] = float("inf")
    q[2, 1, 60] = float("nan")
    got = rotary.norm_rotate(q, k, qg, kg, pos, freq)[0]
    assert bool((got[0, 0] == 0).all())
    assert bool(got[1, 0].isnan().any()) and bool(got[2, 1].isnan().all())
    keep = torch.ones(6, 2, dtype=torch.bool)
    keep[0, 0] = keep[1, 0] = keep[2, 1] = False
    assert torch.equal(got[keep], clean[keep])


def test_no_tokens(cuda):
    q, k, qg, kg, pos, freq = make(0, 2, 1, 64, 64, torch.bfloat16)
    assert rotary.norm_rotate(q, k, qg, kg, pos, freq)[0].shape == (0, 2, 64)
    grads = rotary.norm_rotate_backward(q, k, q, k, qg, kg, pos, freq)
    assert bool((grads[2] == 0).all()) and bool((grads[3] == 0).all())


def test_the_same_bits_on_every_run_stream_and_replay(cuda):
    q, k, qg, kg, pos, freq = make(700, 16, 4, 128, 128, torch.bfloat16)
    want = rotary.norm_rotate_backward(q, k, q, k, qg, kg, pos, freq)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = rotary.norm_rotate_backward(q, k, q, k, qg, kg, pos, freq, stream=side)
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want, strict=True))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = rotary.norm_rotate_backward(q, k, q, k, qg, kg, pos, freq)
    for _ in range(2):
        for x in got:
            x.zero_()
        graph.replay()
        assert all(torch.equal(x, y) for x, y in zip(got, want, strict=True))


def test_refusals(cuda):
    q, k, qg, kg, pos, freq = make(4, 2, 1, 64, 64, torch.float32)
    ok = dict(queries=q, keys=k, query_gain=qg, key_gain=kg, positions=pos, frequencies=freq)
    bad = [
        dict(queries=q.cpu()), dict(queries=q.double()), dict(queries=q[0]), dict(keys=k.half()), dict(keys=k[:3]), dict(keys=k[:, :, :32]),
        dict(queries=q[:, :0]), dict(query_gain=qg[:5]), dict(query_gain=qg.half()), dict(key_gain=kg.cpu()), dict(positions=pos.float()),
        dict(positions=pos[:2]), dict(frequencies=freq.float()), dict(frequencies=freq[:0]), dict(frequencies=torch.cat([freq, freq])),
        dict(epsilon=0.0), dict(epsilon=1e-60), dict(queries=torch.randn(4, 64, 2, device="cuda").transpose(1, 2)),
    ]
    for change in bad:
        with pytest.raises(ConfigError):
            rotary.norm_rotate(**{**ok, **change})
    out = torch.empty(4, 2, 64, device="cuda")
    for q_out, k_out in ((out, out[:, :1]), (q, q[:, :1]), (out.half(), k), (out[:3], k), (out[:1].expand(4, 2, 64), k), (k.expand(4, 2, 64), k)):
        with pytest.raises(ConfigError):
            rotary.norm_rotate_into(q, k, qg, kg, pos, freq, q_out, k_out)
    with pytest.raises(ConfigError):
        rotary.norm_rotate_backward(q[:2], k, q, k, qg, kg, pos, freq)
    with pytest.raises(ConfigError):
        rotary.frequencies(7)
    assert heads.overlap(out, out[1:]) and not heads.overlap(q, k)


def test_outputs_that_are_parts_of_the_same_heads(cuda):
    rows = torch.randn(5, 3, 2, 64, device="cuda")
    gain, positions, freqs = torch.ones(64, device="cuda"), torch.arange(5, device="cuda"), rotary.frequencies(64)
    want = rotary.norm_rotate(rows[:, :, 0], rows[:, :, 1], gain, gain, positions, freqs)
    out = torch.zeros_like(rows)
    rotary.norm_rotate_into(rows[:, :, 0], rows[:, :, 1], gain, gain, positions, freqs, out[:, :, 0], out[:, :, 1])
    assert torch.equal(out[:, :, 0], want[0]) and torch.equal(out[:, :, 1], want[1])
    rotary.norm_rotate_into(rows[:, :, 0], rows[:, :, 1], gain, gain, positions, freqs, rows[:, :, 0], rows[:, :, 1])
    assert torch.equal(rows, out)


FIRST = """
import sys
sys.path.insert(0, sys.argv[1])
import torch
from tgcb import attention, kv_cache, rotary

rows, gain, freqs = torch.randn(4, 3, 64, device="cuda"), torch.ones(64, device="cuda"), rotary.frequencies(64)
positions, table, starts = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 1, 2, 3], [[2, 1]], [3]))
cache = kv_cache.QuantisedCache(4, 1, 64, page=16)

def step():
    q, k = rotary.norm_rotate(rows[:, :2], rows[:, 2:], gain, gain, positions, freqs)
    cache.append(k, rows[:, 2:], table, starts)
    return attention.cached_attention(q, cache, table, starts)

graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = step()
graph.replay()
cache.check()
assert bool(got.isfinite().all()) and torch.equal(got, step())
"""


def test_a_process_whose_first_call_is_captured(cuda):
    import subprocess
    import sys

    package = os.path.dirname(os.path.dirname(heads.__file__))
    done = subprocess.run([sys.executable, "-c", FIRST, package], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]
