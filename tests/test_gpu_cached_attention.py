"""Attention over the int8 cache on the GPU against float64, and the step that generates a token.

Tolerance. A score is a sum of `width` products in float32, truncated by the tensor cores at
worst: off by (width + 8) * 2^-23 of scale * sum |q_i k_i| (plus 2^-21 of a cap); a weight is off by
that relatively, and once more through the sum of the weights. The weighted values of n keys are added up in
float32, at most n / 16 + 64 of them in a row. 16-bit rows hold the weights to 16 bits or more and
round the result once: half of the type's eps of the value.
"""

from __future__ import annotations

import pytest
import torch
from oracle import generation

from tgcb import attention, kv_cache, rotary
from tgcb.errors import ConfigError

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def vector(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


WIDE = 80_000  # positions that a table may hold beyond those in use: how a call is cut goes by what it may hold


def make(starts, counts, q_heads, kv_heads, width, page, dtype, seed=0, spare=2, room=0):
    """(queries, cache, table, starts, offsets): sequences with `starts` positions before and `counts` rows in the call, in a
    table with room for `room` positions."""
    g = torch.Generator().manual_seed(seed)
    batch = len(starts)
    each = max(1, max(-(-(s + n) // page) for s, n in zip(starts, counts, strict=True)))
    pages = batch * each + spare
    parts = []
    for _ in range(2):
        parts.append((torch.randn(pages, kv_heads, page, width, generator=g) * 40).round().clamp(-128, 127).to(torch.int8).cuda())
        parts.append(((0.5 + torch.rand(pages, kv_heads, page, generator=g)) / 40).cuda())
    table = torch.randperm(pages, generator=g)[:batch * each].reshape(batch, each).to(torch.int32).cuda()
    if room > each * page:
        table = torch.nn.functional.pad(table, (0, room // page - each), value=-1)
    tokens = sum(counts)
    q = (torch.randn(tokens, q_heads, width, generator=g) * 2).to(dtype).cuda()
    offsets = [0]
    for n in counts:
        offsets.append(offsets[-1] + n)
    return q, kv_cache.QuantisedCache.of(*parts), table, vector(starts), vector(offsets)


def tree_bits(counts, seed=0):
    """Ancestor bits of a random tree per sequence, every row seeing itself."""
    g = torch.Generator().manual_seed(seed)
    bits = []
    for n in counts:
        own = []
        for i in range(n):
            parent = int(torch.randint(-1, i, (1,), generator=g)) if i else -1
            own.append((own[parent] if parent >= 0 else 0) | 1 << i)
        bits += own
    return torch.tensor([b - (1 << 64) if b >> 63 else b for b in bits], dtype=torch.int64, device="cuda")


def check(got, q, cache, table, starts, offsets, visible=None, scale=None, cap=None, longest=0):
    width = q.shape[2]
    scale = width**-0.5 if scale is None else scale
    want, size, scores = generation.attention(q, cache.keys, cache.key_scales, cache.values, cache.value_scales, table, starts, offsets,
                                              visible, scale, cap or 0.0)
    mine = ~want.isnan().all(-1)
    longest = int(starts.max()) + q.shape[0] if not longest else longest
    delta = (width + 8) * 2.0**-23 * scores + (cap or 0.0) * 2.0**-21
    part = 2 * delta + (longest / 16 + 64) * 2.0**-24
    tol = part * size + 1e-37
    if q.dtype != torch.float32:
        tol = (part + 2.0**-16) * size + torch.finfo(q.dtype).eps / 2 * (want.abs() + part * size) + 2.0**-25
    off = (got.cpu().double() - want).abs()
    ratio = (off / tol)[mine]
    assert not bool(got.cpu()[mine].isnan().any())
    assert ratio.numel() == 0 or float(ratio.max()) <= 1, f"off by {float(ratio.max())} tolerances"


SHAPES = [
    # starts, counts, query heads, key heads, width, page
    ([0], [1], 1, 1, 32, 16),
    ([1], [1], 2, 1, 64, 16),
    ([300], [1], 16, 4, 64, 16),
    ([63, 64, 65, 0], [1, 1, 1, 1], 8, 8, 128, 64),
    ([1000, 17, 515], [1, 1, 1], 8, 1, 128, 32),
    ([777], [1], 20, 4, 256, 128),
    ([2500, 5], [1, 1], 12, 3, 32, 64),
    ([129], [7], 6, 2, 64, 16),
    ([0, 40, 200], [33, 1, 0], 4, 4, 128, 32),
    ([100], [70], 16, 2, 128, 64),
    ([0], [150], 5, 1, 64, 128),
    ([31, 0], [17, 40], 17, 1, 32, 16),
    ([500, 3], [5, 64], 8, 2, 256, 64),
    ([3000, 0, 7, 250], [90, 200, 0, 3], 8, 2, 128, 64),
    ([0, 1500], [1, 300], 4, 1, 64, 32),
    ([130], [129], 3, 3, 128, 16),
]


@pytest.mark.parametrize("room", [0, WIDE])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("starts,counts,q_heads,kv_heads,width,page", SHAPES)
def test_causal(cuda, starts, counts, q_heads, kv_heads, width, page, dtype, room):
    q, cache, table, s, o = make(starts, counts, q_heads, kv_heads, width, page, dtype, room=room)
    check(attention.cached_attention(q, cache, table, s, o), q, cache, table, s, o)
    cache.check()


@pytest.mark.parametrize("room", [0, WIDE])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("starts,counts,q_heads,kv_heads,width,page", SHAPES)
def test_capped(cuda, starts, counts, q_heads, kv_heads, width, page, dtype, room):
    q, cache, table, s, o = make(starts, counts, q_heads, kv_heads, width, page, dtype, seed=1, room=room)
    check(attention.cached_attention(q, cache, table, s, o, scale=0.3, cap=20.0), q, cache, table, s, o, scale=0.3, cap=20.0)


@pytest.mark.parametrize("room", [0, WIDE])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("starts,counts,q_heads,kv_heads,width,page", [
    ([0], [1], 1, 1, 64, 16), ([100], [13], 8, 2, 128, 64), ([1000, 3], [60, 64], 16, 2, 128, 32), ([127, 128], [64, 1], 8, 1, 64, 16), ([0, 33, 250], [64, 3, 20], 4, 1, 64, 32), ([5, 6], [16, 16], 32, 4, 128, 16),
    ([200], [64], 16, 2, 32, 64), ([90, 0, 1, 64], [9, 1, 30, 64], 4, 4, 256, 128),
])
def test_trees(cuda, starts, counts, q_heads, kv_heads, width, page, dtype, room):
    q, cache, table, s, o = make(starts, counts, q_heads, kv_heads, width, page, dtype, room=room)
    bits = tree_bits(counts)
    check(attention.cached_attention(q, cache, table, s, o, visible=bits), q, cache, table, s, o, bits)
    check(attention.cached_attention(q, cache, table, s, o, visible=bits, cap=30.0), q, cache, table, s, o, bits, cap=30.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q_heads,room", [(4, 0), (4, WIDE), (32, WIDE)])
def test_rows_behind_the_64th_cannot_be_named(cuda, q_heads, room, dtype):
    """Any bits, rows ahead among them, in sequences of more than 64 rows: bit j is row j, no row is bit 64."""
    counts = [100, 3, 65, 129]
    q, cache, table, s, o = make([30, 0, 127, 500], counts, q_heads, 2, 64, 32, dtype, room=room)
    g = torch.Generator().manual_seed(3)
    bits = torch.randint(-(1 << 63), (1 << 63) - 1, (sum(counts),), generator=g).cuda()
    bits[::7] = -1
    check(attention.cached_attention(q, cache, table, s, o, visible=bits), q, cache, table, s, o, bits)
    cache.check()


def test_one_count_for_all_is_the_same_call(cuda):
    q, cache, table, s, o = make([40, 3, 77], [5, 5, 5], 8, 2, 64, 16, torch.bfloat16)
    assert torch.equal(attention.cached_attention(q, cache, table, s), attention.cached_attention(q, cache, table, s, o))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("length,kv_heads", [(20000, 1), (9001, 8), (33000, 2)])
def test_long_contexts(cuda, length, kv_heads, dtype):
    q, cache, table, s, o = make([length, 700], [1, 1], 4 * kv_heads, kv_heads, 128, 64, dtype)
    check(attention.cached_attention(q, cache, table, s, o), q, cache, table, s, o)


@pytest.mark.parametrize("q_heads", [4, 128])
def test_pages_whose_offsets_pass_32_bits(cuda, q_heads):
    """The same pages at the end of a cache of 4.6 GB of key codes: the same bits, written and read there too."""
    q, near, table, s, o = make([700, 5], [1, 3], q_heads, 2, 128, 128, torch.bfloat16, room=WIDE)
    pages, own = 140_000, near.pages
    far = kv_cache.QuantisedCache(pages, 2, 128, page=128)
    assert far.keys.numel() > 1 << 32
    for a, b in ((near.keys, far.keys), (near.key_scales, far.key_scales), (near.values, far.values), (near.value_scales, far.value_scales)):
        b[pages - own:] = a
    moved = torch.where(table < 0, table, table + (pages - own))
    assert torch.equal(attention.cached_attention(q, far, moved, s, o), attention.cached_attention(q, near, table, s, o))
    rows = torch.randn(4, 2, 128, device="cuda").bfloat16()
    for cache, at in ((near, table), (far, moved)):
        cache.append(rows, -rows, at, s, o)
        cache.check()
    for a, b in zip(near.read(4, table, s, o), far.read(4, moved, s, o), strict=True):
        assert torch.equal(a, b)
    assert torch.equal(near.keys, far.keys[pages - own:]) and not bool(far.keys[:own].any())


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_sequences_of_all_lengths(cuda, dtype):
    starts = [(37 * i) % 400 for i in range(150)]
    q, cache, table, s, o = make(starts, [1] * 150, 8, 2, 64, 32, dtype)
    check(attention.cached_attention(q, cache, table, s), q, cache, table, s, None)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q_heads,room", [(4, 0), (4, WIDE), (64, WIDE)])
def test_a_row_that_sees_nothing_gets_zeros(cuda, q_heads, room, dtype):
    q, cache, table, s, o = make([0, 0, 50], [3, 2, 2], q_heads, 2, 64, 16, dtype, room=room)
    bits = torch.tensor([0, 1, 0, 2, 2, 0, 3], device="cuda")
    got = attention.cached_attention(q, cache, table, s, o, visible=bits)
    assert bool((got[0] == 0).all()) and bool((got[2] == 0).all())
    check(got, q, cache, table, s, o, bits)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("q_heads,room", [(4, 0), (4, WIDE), (128, WIDE)])
def test_what_lies_behind_and_beside_a_sequence_does_not_reach_it(cuda, q_heads, room, dtype):
    """Infinite and NaN scales in places that no token sees, in its own pages too."""
    q, cache, table, s, o = make([20, 3], [1, 2], q_heads, 2, 64, 16, dtype, room=room)
    bits = torch.tensor([1, 1, 2], device="cuda")
    plain, tree = attention.cached_attention(q, cache, table, s, o), attention.cached_attention(q, cache, table, s, o, visible=bits)
    held = torch.zeros(cache.keys.shape[0], 16, dtype=torch.bool, device="cuda")
    for b, length in ((0, 21), (1, 5)):
        for j in range(length):
            held[int(table[b, j // 16]), j % 16] = True
    for scales, codes in ((cache.key_scales, cache.keys), (cache.value_scales, cache.values)):
        scales.copy_(torch.where(held[:, None], scales, float("nan")))
        codes.copy_(torch.where(held[:, None, :, None], codes, -128))
    assert torch.equal(attention.cached_attention(q, cache, table, s, o), plain)
    for value in (float("nan"), float("inf")):
        cache.value_scales[table[1, 0], :, 3] = value  # row 0 of sequence 1, seen by itself alone
        cache.key_scales[table[1, 0], :, 3] = value
        got = attention.cached_attention(q, cache, table, s, o, visible=bits)
        assert torch.equal(got[0], tree[0]) and torch.equal(got[2], tree[2]) and bool(got[1].isnan().all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q_heads,room", [(8, 0), (8, WIDE), (64, WIDE)])
def test_infinite_and_nan_queries_stay_in_their_rows(cuda, q_heads, room, dtype):
    q, cache, table, s, o = make([100], [5], q_heads, 2, 64, 16, dtype, room=room)
    want = attention.cached_attention(q, cache, table, s, o)
    q[1, 3, 7], q[4, 0, 0] = float("inf"), float("nan")
    got = attention.cached_attention(q, cache, table, s, o)
    assert bool(got[1, 3].isnan().all()) and bool(got[4, 0].isnan().all())
    keep = torch.ones(5, q_heads, dtype=torch.bool)
    keep[1, 3] = keep[4, 0] = False
    assert torch.equal(got[keep], want[keep])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q_heads,room", [(4, 0), (40, WIDE)])
@pytest.mark.parametrize("size", [2.0**-12, 2.0**10])
def test_rows_of_very_different_sizes(cuda, dtype, size, q_heads, room):
    """One key with a far larger or smaller value row than the others, and queries of that size."""
    q, cache, table, s, o = make([300], [1], q_heads, 1, 128, 64, dtype, room=room)
    cache.value_scales[table[0, 2], 0, 9] *= size * 64
    q = (q.float() * size).to(dtype)
    check(attention.cached_attention(q, cache, table, s, o, scale=0.1 / size), q, cache, table, s, o, scale=0.1 / size)


@pytest.mark.parametrize("q_heads,room", [(4, 0), (4, WIDE), (64, WIDE)])
def test_rows_of_no_sequence_are_left(cuda, q_heads, room):
    q, cache, table, s, _ = make([30, 5], [4, 8], q_heads, 2, 64, 16, torch.float16, room=room)
    o = vector([1, 4, 9])
    out = torch.full_like(q, 3.0)
    assert attention.cached_attention(q, cache, table, s, o, out=out) is out
    assert bool((out[0] == 3).all()) and bool((out[9:] == 3).all())
    check(out, q, cache, table, s, o)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("q_heads,room", [(4, 0), (4, WIDE), (128, WIDE)])
def test_pages_and_positions_that_are_not_there_are_left_out(cuda, q_heads, room, dtype):
    q, cache, table, s, o = make([60, 40, 3], [1, 1, 1], q_heads, 2, 64, 16, dtype, room=room)
    table[0, 1], table[1, 0] = 10_000, -1
    s[2] = 64  # its 65 positions need a fifth page
    check(attention.cached_attention(q, cache, table, s, o), q, cache, table, s, o, longest=70)
    with pytest.raises(ConfigError):
        cache.check()
    s.copy_(vector([-5, -1, 2]))
    table[:2, :2] = 0
    got = attention.cached_attention(q, cache, table, s, o)
    assert bool((got[:2] == 0).all())
    check(got, q, cache, table, s, o, longest=70)


@pytest.mark.parametrize("start", [-3, 64, 63])
@pytest.mark.parametrize("q_heads,room", [(4, 0), (128, WIDE)])
def test_positions_outside_the_table_are_counted(cuda, q_heads, room, start):
    q, cache, table, s, o = make([62], [2], q_heads, 2, 64, 16, torch.bfloat16, room=room)
    attention.cached_attention(q, cache, table, s, o)
    cache.check()
    s.fill_(start if start < 0 or not room else start - 64 + table.shape[1] * 16)
    attention.cached_attention(q, cache, table, s, o)
    with pytest.raises(ConfigError):
        cache.check()


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_rows_in_short_tables(cuda, dtype):
    """Units that are never cut, enough of them for every kernel."""
    starts = [(29 * i) % 400 for i in range(16)]
    q, cache, table, s, o = make(starts, [40] * 16, 32, 8, 64, 64, dtype, room=512)
    check(attention.cached_attention(q, cache, table, s, o), q, cache, table, s, o)
    bits = tree_bits([40] * 16)
    check(attention.cached_attention(q, cache, table, s, o, visible=bits, cap=25.0), q, cache, table, s, o, bits, cap=25.0)


@pytest.mark.parametrize("offsets", [[0, 100, 3, 9], [-50, 4, 9, 400], [9, 6, 3, 0], [5, 5, 5, 5]])
@pytest.mark.parametrize("q_heads,room", [(4, 0), (4, WIDE), (64, WIDE)])
def test_offsets_that_make_no_sense_reach_nothing_outside(cuda, offsets, q_heads, room):
    q, cache, table, s, _ = make([30, 5, 0], [3, 3, 3], q_heads, 2, 64, 16, torch.bfloat16, room=room)
    out = attention.cached_attention(q, cache, table, s, vector(offsets))
    attention.cached_attention(q, cache, table, s, vector(offsets), visible=tree_bits([9]), out=out)
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q_heads,room", [(4, 0), (4, WIDE), (64, WIDE)])
def test_queries_and_outputs_of_any_stride(cuda, q_heads, room, dtype):
    q, cache, table, s, o = make([30, 5], [3, 2], q_heads, 2, 64, 16, dtype, room=room)
    want = attention.cached_attention(q, cache, table, s, o)
    for shift in (0, 1):
        wide = torch.zeros(q_heads, 5, 80, device="cuda", dtype=dtype)[:, :, shift:64 + shift].transpose(0, 1)
        wide.copy_(q)
        out = torch.zeros(5, 2 * q_heads, 80, device="cuda", dtype=dtype)[:, ::2, shift:64 + shift]
        assert torch.equal(attention.cached_attention(wide, cache, table, s, o, out=out), want)
    one = q[:, :1].expand(5, q_heads, 64)
    check(attention.cached_attention(one, cache, table, s, o), one, cache, table, s, o)


@pytest.mark.parametrize("count", [1, 40])
def test_the_same_bits_on_every_run_and_stream(cuda, count):
    q, cache, table, s, o = make([5000, 300, 12], [count] * 3, 16, 4, 128, 64, torch.bfloat16, room=WIDE)
    want = attention.cached_attention(q, cache, table, s, o)
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for side in streams:
        side.wait_stream(torch.cuda.current_stream())
        for _ in range(5):
            outs.append(attention.cached_attention(q, cache, table, s, o, stream=side))
    for side in streams:
        side.synchronize()
    assert all(torch.equal(x, want) for x in outs)


@pytest.mark.parametrize("count", [1, 30])
def test_two_captured_calls_replay_side_by_side_with_other_lengths(cuda, count):
    a, b = (make([4000, 4000], [count] * 2, 16, 4, 128, 64, torch.bfloat16, seed=i, room=WIDE) for i in range(2))
    graphs, outs = [], []
    for q, cache, table, s, o in (a, b):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(attention.cached_attention(q, cache, table, s, o))
        graphs.append(graph)
    side = torch.cuda.Stream()
    for lengths in ([4000, 100], [0, 4000], [63, 64], [2111, 3000]):
        for call in (a, b):
            call[3].copy_(vector(lengths))
        want = [attention.cached_attention(*call[:4], call[4]) for call in (a, b)]
        for _ in range(3):
            side.wait_stream(torch.cuda.current_stream())
            graphs[0].replay()
            with torch.cuda.stream(side):
                graphs[1].replay()
            torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(x, y) for x, y in zip(outs, want, strict=True))


@pytest.mark.parametrize("dtype", DTYPES)
def test_generating_tokens(cuda, dtype):
    """Prompts, then single tokens, then a drafted tree: heads normed and turned, rows appended, attention
    over what the cache holds, each step against float64 on the cache's own rows."""
    g = torch.Generator().manual_seed(0)
    q_heads, kv_heads, width, page, batch = 8, 2, 64, 16, 3
    cache = kv_cache.QuantisedCache(batch * 8, kv_heads, width, page=page)
    table = torch.randperm(batch * 8, generator=g).reshape(batch, 8).to(torch.int32).cuda()
    gains = [(1 + 0.1 * torch.randn(width, generator=g)).to(dtype).cuda() for _ in range(2)]
    freq, lengths = rotary.frequencies(width), [0] * batch
    for counts, tree in (([30, 1, 17], False), ([1, 1, 1], False), ([1, 1, 1], False), ([9, 4, 14], True), ([1, 1, 1], False)):
        tokens = sum(counts)
        qkv = torch.randn(tokens, q_heads + 2 * kv_heads, width, generator=g).to(dtype).cuda()
        q, k, v = qkv[:, :q_heads], qkv[:, q_heads:q_heads + kv_heads], qkv[:, q_heads + kv_heads:]
        offsets = vector([sum(counts[:b]) for b in range(batch + 1)])
        positions = vector([lengths[b] + i for b in range(batch) for i in range(counts[b])])
        starts = vector(lengths)
        turned_q, turned_k = rotary.norm_rotate(q, k, *gains, positions, freq)
        cache.append(turned_k, v, table, starts, offsets)
        back = cache.read(tokens, table, starts, offsets)
        for x, y in ((turned_k, back[0]), (v, back[1])):  # a code is off by half a step of max|x| / 127
            assert bool(((x.float() - y).abs() <= x.float().abs().amax(-1, keepdim=True) / 127 * 0.5 * 1.0001).all())
        bits = tree_bits(counts) if tree else None
        got = attention.cached_attention(turned_q, cache, table, starts, offsets, visible=bits)
        check(got, turned_q, cache, table, starts, offsets, bits)
        lengths = [n + (2 if tree else c) for n, c in zip(lengths, counts, strict=True)]
    cache.check()


def test_refusals(cuda):
    q, cache, table, s, o = make([30, 5], [3, 3], 4, 2, 64, 16, torch.float32)
    bits = tree_bits([3, 3])
    for change in (
        dict(queries=q.cpu()), dict(queries=q.double()), dict(queries=q[:, :3]), dict(queries=q[:, :, :32]), dict(queries=q[0]),
        dict(queries=q[:5], offsets=None), dict(queries=q[:, :0]), dict(cache=cache.keys), dict(table=table.long()), dict(starts=s[:1]),
        dict(starts=s.long()), dict(offsets=o[:2]), dict(visible=bits.int()), dict(visible=bits[:3]), dict(scale=float("nan")),
        dict(scale=float("inf")), dict(cap=-1.0), dict(cap=float("inf")), dict(out=q), dict(out=torch.empty_like(q).half()),
        dict(scale=1e31), dict(cap=1e-35), dict(out=torch.empty_like(q)[:3]), dict(out=torch.empty(1, 4, 64, device="cuda").expand(6, 4, 64)),
    ):
        with pytest.raises(ConfigError):
            attention.cached_attention(**{**dict(queries=q, cache=cache, table=table, starts=s, offsets=o), **change})
    many = torch.randn(130, 4, 64, device="cuda")
    with pytest.raises(ConfigError, match="64"):
        attention.cached_attention(many, cache, table, s, visible=torch.zeros(130, dtype=torch.int64, device="cuda"))


def check_relative(got, q, cache, table, starts, offsets, visible=None, scale=None, cap=0.0):
    """As `check`, without an error that is a fixed part of the cap or of the values' type: a capped score is off by
    2^-19 of itself (1 - 2 / (1 + e^2x) from |x| = 1/4 on: its quotient, at most 0.76, by 1.8 * 2^-22 of itself, and the
    tangent is 0.24 there; below, the series by 2^-21 and its roundings)."""
    scale = q.shape[2]**-0.5 if scale is None else scale
    want, size, scores = generation.attention(q, cache.keys, cache.key_scales, cache.values, cache.value_scales, table, starts, offsets,
                                              visible, scale, cap)
    mine, eps = ~want.isnan().all(-1), torch.finfo(q.dtype).eps
    delta = ((q.shape[2] + 8) * 2.0**-23 + 2.0**-19 * (cap > 0)) * scores
    part = 2 * delta + ((int(starts.max()) + q.shape[0]) / 16 + 64) * 2.0**-24
    tol = part * size if q.dtype == torch.float32 else (part + 2.0**-16) * size + eps / 2 * (want.abs() + part * size)
    ratio = ((got.cpu().double() - want).abs() / (tol + torch.finfo(q.dtype).tiny * eps))[mine]
    assert bool(got.cpu()[mine].isfinite().all())
    assert float(ratio.max()) <= 1, f"off by {float(ratio.max())} tolerances"


@pytest.mark.parametrize("cap", [100.0, 1e4, 1e6, 1e8, 1e30])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q_heads,room", [(4, 0), (4, WIDE), (64, WIDE)])
def test_large_caps(cuda, q_heads, room, dtype, cap):
    """A cap far above the scores changes next to nothing."""
    q, cache, table, s, o = make([100, 700], [1, 5], q_heads, 2, 64, 32, dtype, seed=2, room=room)
    check_relative(attention.cached_attention(q, cache, table, s, o, scale=0.5, cap=cap), q, cache, table, s, o, scale=0.5, cap=cap)


@pytest.mark.parametrize("cap", [1e31, 3e38])
def test_caps_beyond_float32_are_refused(cuda, cap):
    q, cache, table, s, o = make([100, 700], [1, 5], 4, 2, 64, 32, torch.float32)
    with pytest.raises(ConfigError, match="beyond float32"):
        attention.cached_attention(q, cache, table, s, o, cap=cap)


@pytest.mark.parametrize("power", [-100, 60, 90, 115, 125])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("q_heads,room", [(4, 0), (4, WIDE), (64, WIDE), (128, WIDE)])
def test_values_of_every_magnitude(cuda, q_heads, room, dtype, power):
    q, cache, table, s, o = make([300, 1900], [1, 5], q_heads, 2, 64, 32, dtype, seed=3, room=room)
    cache.value_scales *= 2.0**power  # values up to 4.8 times that
    check_relative(attention.cached_attention(q, cache, table, s, o), q, cache, table, s, o)
    check_relative(attention.cached_attention(q, cache, table, s, o, cap=10.0), q, cache, table, s, o, cap=10.0)
    q.zero_()  # all weights one, all values of one sign: the largest sums
    cache.values.clamp_(min=-127).abs_()
    check_relative(attention.cached_attention(q, cache, table, s, o), q, cache, table, s, o)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("q_heads,room", [(4, 0), (4, WIDE), (64, WIDE), (128, WIDE)])
@pytest.mark.parametrize("place", [0, 40, 200, 1001, 1004])
def test_one_value_far_above_the_others(cuda, place, q_heads, room, dtype):
    """Rows that see it, and rows that do not, whose own values are too small to be held beside it."""
    q, cache, table, s, o = make([1000], [6], q_heads, 1, 64, 32, dtype, seed=4, room=room)
    cache.value_scales *= 2.0**-90
    at = table[0, place // 32], 0, place % 32
    cache.value_scales[at] *= 2.0**105
    cache.value_scales[at] *= 2.0**105
    cache.values[at] += cache.values[at] == 0  # it has a part in every column
    check_relative(attention.cached_attention(q, cache, table, s, o), q, cache, table, s, o)
    bits = tree_bits([6])
    check_relative(attention.cached_attention(q, cache, table, s, o, visible=bits, cap=10.0), q, cache, table, s, o, bits, cap=10.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("q_heads,room", [(4, 0), (4, WIDE), (64, WIDE), (128, WIDE)])
@pytest.mark.parametrize("bits", [30, 95])
def test_a_large_value_of_little_weight(cuda, bits, q_heads, room, dtype):
    """2^120 at a weight 2^-30 or 2^-95 of the largest: it is most of the answer, and not all its weight may be taken from it."""
    q, cache, table, s, o = make([500], [3], q_heads, 1, 64, 32, dtype, seed=5, room=room)
    cache.keys.zero_()
    cache.keys[table[0, 7], 0, 9] = 64
    cache.key_scales.fill_(2.0**-6)
    cache.value_scales[table[0, 7], 0, 9] *= 2.0**120
    q.fill_(-1)  # 64 products of -1 with 1: a score of -64 scale, the others' 0
    scale = bits * 0.6931471805599453 / 64
    check_relative(attention.cached_attention(q, cache, table, s, o, scale=scale), q, cache, table, s, o, scale=scale)


@pytest.mark.parametrize("page", [-1, -2, -3, -(1 << 31), 10_000, (1 << 31) - 1])
@pytest.mark.parametrize("q_heads,room", [(4, 0), (4, WIDE), (128, WIDE)])
def test_every_page_that_is_not_there_is_counted(cuda, q_heads, room, page):
    q, cache, table, s, o = make([300], [2], q_heads, 2, 64, 16, torch.bfloat16, room=room)
    table[0, 3] = page
    check(attention.cached_attention(q, cache, table, s, o), q, cache, table, s, o)
    with pytest.raises(ConfigError):
        cache.check()
    cache.append(q[:, :2], q[:, :2], table, vector([47]), o)
    with pytest.raises(ConfigError, match="^1 accesses"):
        cache.check()
