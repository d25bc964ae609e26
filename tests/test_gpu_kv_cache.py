"""The int8 cache on the GPU: rows quantised as they are written, bit for bit the quantiser's, and read back."""

from __future__ import annotations

import pytest
import torch
from oracle import generation

from tgcb import kv_cache, quantize
from tgcb.errors import ConfigError

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def filled(pages, kv_heads, page, width, seed=0):
    """A cache that holds something everywhere, and copies of its tensors."""
    g = torch.Generator().manual_seed(seed)
    parts = [torch.randint(-128, 128, (pages, kv_heads, page, width), generator=g).to(torch.int8).cuda() if i % 2 == 0
             else torch.rand(pages, kv_heads, page, generator=g).cuda() for i in range(4)]
    return kv_cache.QuantisedCache.of(*parts), [p.clone() for p in parts]


def a_table(batch, each, pages, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randperm(pages, generator=g)[:batch * each].reshape(batch, each).to(torch.int32).cuda()


def vector(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def written(before, keys, values, table, starts, offsets, page):
    """What the cache holds after the rows are written in order, by the oracle."""
    k, ks, v, vs = (p.cpu().clone() for p in before)
    (qk, sk), (qv, sv) = generation.quantise(keys), generation.quantise(values)
    for t, place in enumerate(generation.places(table, starts, offsets, keys.shape[0], page)):
        if place is not None and 0 <= place[4] < k.shape[0]:
            at, row = place[4], place[5]
            k[at, :, row], ks[at, :, row], v[at, :, row], vs[at, :, row] = qk[t], sk[t], qv[t], sv[t]
    return k, ks, v, vs


def same(cache, want):
    for got, w in zip((cache.keys, cache.key_scales, cache.values, cache.value_scales), want, strict=True):
        assert torch.equal(got.cpu(), w)


CASES = [
    # batch, starts, offsets (None: one count for all), tokens, kv heads, width, page
    (1, [0], None, 1, 1, 32, 16),
    (1, [15], None, 2, 2, 64, 16),
    (3, [0, 63, 64], None, 3, 8, 128, 64),
    (2, [5, 200], None, 130, 3, 128, 32),
    (4, [0, 1, 100, 7], [0, 0, 1, 40, 50], 50, 5, 256, 64),
    (3, [9, 0, 31], [2, 5, 5, 80], 90, 4, 64, 32),  # rows before the first and behind the last sequence
    (70, [3 * i for i in range(70)], None, 70, 2, 128, 128),
    (300, [i % 7 for i in range(300)], None, 1500, 1, 32, 16),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,starts,offsets,tokens,kv_heads,width,page", CASES)
def test_append_and_read(cuda, batch, starts, offsets, tokens, kv_heads, width, page, dtype):
    each = 1 + (max(starts) + tokens) // page
    cache, before = filled(batch * each + 2, kv_heads, page, width)
    table, starts = a_table(batch, each, batch * each + 2), vector(starts)
    offsets = vector(offsets) if offsets is not None else None
    g = torch.Generator().manual_seed(3)
    keys, values = ((torch.randn(tokens, kv_heads, width, generator=g) * torch.rand(tokens, kv_heads, 1, generator=g) * 30).to(dtype).cuda()
                    for _ in range(2))
    keys[0, 0] = 0
    cache.append(keys, values, table, starts, offsets)
    cache.check()
    want = written(before, keys, values, table, starts, offsets, page)
    same(cache, want)
    filler = torch.full_like(keys, 7.0), torch.full_like(keys, 7.0)
    cache.read_into(*filler, table, starts, offsets)
    got = cache.read(tokens, table, starts, offsets, dtype=dtype)
    for t, place in enumerate(generation.places(table, starts, offsets, tokens, page)):
        for side, (codes, scales) in enumerate(((want[0], want[1]), (want[2], want[3]))):
            if place is None:
                assert bool((filler[side][t] == 7.0).all())
            else:
                w = (codes[place[4], :, place[5]].float() * scales[place[4], :, place[5]][..., None]).to(dtype)
                assert torch.equal(filler[side][t].cpu(), w) and torch.equal(got[side][t].cpu(), w)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_are_the_quantisers(cuda, dtype):
    """Ties between two codes, rows of zeros, subnormals, infinities and NaN: what quantise_rows gives."""
    g = torch.Generator().manual_seed(5)
    rows = torch.randn(64, 128, generator=g) * torch.exp(torch.randn(64, 1, generator=g) * 4)
    rows[0] = 0
    rows[1] = 1e-42
    rows[1, 5] = -3e-44
    rows[2, 3] = float("inf")
    rows[3, 3] = float("nan")
    rows[4] = torch.arange(128) - 63.5
    rows[4, 0] = 127.0  # scale 1: every other value lies half way between two codes
    rows[5] = torch.arange(128) * 0.5
    rows[5, 0] = -63.5
    rows[6] = 3e38
    rows = rows.to(dtype).cuda()
    codes, scales = quantize.quantise_rows(rows)
    cache = kv_cache.QuantisedCache(2, 2, 128, page=32)
    cache.append(rows.reshape(32, 2, 128), rows.flip(0).reshape(32, 2, 128), vector([[1]]), vector([0]))
    assert torch.equal(cache.keys[1].transpose(0, 1).reshape(64, 128), codes)
    assert torch.equal(cache.key_scales[1].T.reshape(64).nan_to_num(nan=-1.0), scales.nan_to_num(nan=-1.0))
    assert torch.equal(cache.values[1].transpose(0, 1).reshape(64, 128), codes.flip(0))
    read = cache.read(32, vector([[1]]), vector([0]))[0].reshape(64, 128)
    want = codes.float() * scales[:, None]
    assert torch.equal(read.isnan(), want.isnan()) and torch.equal(read.nan_to_num(), want.nan_to_num())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("width", [32, 256])
def test_rows_of_every_magnitude_are_the_quantisers(cuda, width, dtype):
    """Maxima of 2^-140 to 2^127: scales subnormal, at the least normal number, large; halves of the maximum lie between two codes."""
    g = torch.Generator().manual_seed(6)
    rows = torch.rand(268 * 4, width, generator=g, dtype=torch.float64) * 2 - 1
    rows[:, 1::4] = rows[:, :1] * torch.randint(-127, 128, (268 * 4, width // 4), generator=g) / 254
    rows = (rows * 2.0 ** (torch.arange(268 * 4) // 4 - 140.0)[:, None]).float().to(dtype).cuda()
    codes, scales = quantize.quantise_rows(rows)
    cache = kv_cache.QuantisedCache(9, 1, width, page=128)
    cache.append(rows[:, None], rows[:, None], torch.arange(9, dtype=torch.int32, device="cuda")[None], vector([0]))
    for got, got_scales in ((cache.keys, cache.key_scales), (cache.values, cache.value_scales)):
        assert torch.equal(got.reshape(-1, width)[:268 * 4], codes) and torch.equal(got_scales.reshape(-1)[:268 * 4], scales)


@pytest.mark.parametrize("shift", [0, 1])
def test_rows_of_any_stride(cuda, shift):
    base = torch.randn(5, 9, 64 + shift, device="cuda").to(torch.bfloat16)[:, :, shift:]
    keys, values = base[:, :4], base[:, 4:8]
    cache, before = filled(3, 4, 16, 64)
    cache.append(keys, values, vector([[2]]), vector([1]))
    same(cache, written(before, keys, values, vector([[2]]), vector([1]), None, 16))
    want = cache.read(5, vector([[2]]), vector([1]), dtype=torch.bfloat16)
    out = torch.zeros(4, 2, 5, 64 + shift, device="cuda", dtype=torch.bfloat16)[..., shift:]
    got = out[:, 0].transpose(0, 1), out[:, 1].transpose(0, 1)
    cache.read_into(*got, vector([[2]]), vector([1]))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("tokens,batch", [(40, 40), (96, 3), (2100, 2)])
def test_a_place_named_twice_holds_the_last_row(cuda, tokens, batch):
    """All sequences share their pages: the last sequence's rows stay, whole."""
    cache, before = filled(200, 2, 16, 64)
    table = a_table(1, 150, 200).expand(batch, 150).contiguous()
    starts = vector([i % 3 for i in range(batch)])
    keys, values = torch.randn(tokens, 2, 64, device="cuda"), torch.randn(tokens, 2, 64, device="cuda")
    for _ in range(3):
        cache.append(keys, values, table, starts)
        same(cache, written(before, keys, values, table, starts, None, 16))
    table = vector([[4, 9, 4, 9, 9, 1]])  # a page twice in one sequence
    keys, values = keys[:90], values[:90]
    cache, before = filled(20, 2, 16, 64)
    cache.append(keys, values, table, vector([3]))
    same(cache, written(before, keys, values, table, vector([3]), None, 16))


def test_places_that_are_not_there_are_skipped_and_counted(cuda):
    cache, before = filled(4, 1, 16, 32)
    table = vector([[0, 7], [-1, 1], [2, 3], [3, 2]])
    starts, offsets = vector([15, 15, 31, -1]), vector([0, 2, 4, 6, 7])
    keys, values = torch.randn(7, 1, 32, device="cuda"), torch.randn(7, 1, 32, device="cuda")
    cache.append(keys, values, table, starts, offsets)
    want = written(before, keys, values, table, starts, offsets, 16)
    same(cache, want)
    with pytest.raises(ConfigError, match="4 accesses"):  # page 7, page -1, position 32, position -1
        cache.check()
    cache.check()
    k, _ = cache.read(7, table, starts, offsets)
    assert k.isnan().all(-1).flatten().tolist() == [False, True, True, False, False, True, True]
    with pytest.raises(ConfigError):
        cache.check()


@pytest.mark.parametrize("offsets", [[0, 100, 3, 9], [-50, 4, 9, 400], [9, 6, 3, 0], [5, 5, 5, 5]])
def test_offsets_that_make_no_sense_reach_nothing_outside(cuda, offsets):
    cache, _ = filled(8, 1, 16, 32)
    keys, values = torch.randn(9, 1, 32, device="cuda"), torch.randn(9, 1, 32, device="cuda")
    table = a_table(3, 2, 8)
    cache.append(keys, values, table, vector([0, 3, 20]), vector(offsets))
    out = cache.read(9, table, vector([0, 3, 20]), vector(offsets))
    assert out[0].shape == (9, 1, 32)
    torch.cuda.synchronize()


def test_no_tokens_and_replay_with_other_lengths(cuda):
    cache, before = filled(6, 2, 16, 64)
    table, starts = a_table(2, 3, 6), vector([0, 0])
    cache.append(torch.empty(0, 2, 64, device="cuda"), torch.empty(0, 2, 64, device="cuda"), table, starts)
    same(cache, [p.cpu() for p in before])
    keys, values = torch.randn(2, 2, 64, device="cuda"), torch.randn(2, 2, 64, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.append(keys, values, table, starts)
        got = cache.read(2, table, starts)
    want = [p.cpu() for p in before]
    for length in (0, 15, 16, 40):
        starts.copy_(vector([length, 47 - length]))
        keys.normal_()
        graph.replay()
        want = written(want, keys, values, table, starts, None, 16)
        same(cache, want)
        assert float((got[0] - keys).abs().max()) <= float(keys.abs().max()) / 127 * 0.5 * 1.001
    cache.check()


def test_refusals(cuda):
    cache = kv_cache.QuantisedCache(4, 2, 64, page=16)
    assert cache.bytes == 4 * 2 * 16 * 2 * (64 + 4)
    rows, table, starts = torch.randn(2, 2, 64, device="cuda"), vector([[0, 1], [2, 3]]), vector([0, 0])
    for keys, values, t, s, o in (
        (rows.cpu(), rows, table, starts, None), (rows.double(), rows, table, starts, None), (rows, rows.half(), table, starts, None),
        (rows[:, :1], rows[:, :1], table, starts, None), (rows[:1], rows, table, starts, None), (rows, rows, table.long(), starts, None),
        (rows, rows, table[0], starts, None), (rows, rows, table.cpu(), starts, None), (rows, rows, table.T, starts, None),
        (rows, rows, table, starts[:1], None), (rows, rows, table, starts.long(), None), (rows, rows, table, starts, starts),
        (rows[:1], rows[:1], table, starts, None), (rows, rows, table[:, :0], starts, None),
    ):
        with pytest.raises(ConfigError):
            cache.append(keys, values, t, s, o)
    with pytest.raises(ConfigError):
        cache.read(2, table, starts, dtype=torch.float64)
    with pytest.raises(ConfigError):
        cache.read_into(rows, rows, table, starts)
    with pytest.raises(ConfigError):
        cache.read_into(rows[:1].expand(2, 2, 64), rows.clone(), table, starts)
    for pages, kv_heads, width, page in ((0, 1, 64, 16), (1, 0, 64, 16), (1, 1, 48, 16), (1, 1, 64, 24)):
        with pytest.raises(ConfigError):
            kv_cache.QuantisedCache(pages, kv_heads, width, page=page)
    with pytest.raises(ConfigError):
        kv_cache.QuantisedCache.of(cache.keys, cache.key_scales, cache.values.float(), cache.value_scales)
    with pytest.raises(ConfigError):
        kv_cache.QuantisedCache.of(cache.keys, cache.key_scales[:2], cache.values, cache.value_scales)


def test_check_waits_for_every_stream(cuda):
    cache, _ = filled(4, 1, 16, 32)
    rows, bad, starts, side = torch.randn(2, 1, 32, device="cuda"), vector([[7]]), vector([0]), torch.cuda.Stream()
    cache.append(rows, rows, vector([[1]]), starts)  # its kernel is loaded before the streams differ
    cache.check()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)
    cache.append(rows, rows, bad, starts, stream=side)
    with pytest.raises(ConfigError, match="2 accesses"):
        cache.check()
    cache.append(rows[:1], rows[:1], bad, starts)
    with pytest.raises(ConfigError, match="1 accesses"):
        cache.check()
    cache.check()


def test_a_new_cache_counts_on_every_stream(cuda):
    parts = filled(4, 1, 16, 32)[1]
    rows, bad, starts, side = torch.randn(2, 1, 32, device="cuda"), vector([[7]]), vector([0]), torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda._sleep(200_000_000)
    cache = kv_cache.QuantisedCache.of(*parts)
    cache.append(rows, rows, bad, starts, stream=side)
    with pytest.raises(ConfigError, match="2 accesses"):
        cache.check()


def test_read_into_parts_of_the_same_rows(cuda):
    cache, _ = filled(4, 2, 16, 64)
    rows, table, starts = torch.randn(5, 2, 64, device="cuda"), vector([[2]]), vector([1])
    cache.append(rows, -rows, table, starts)
    want = cache.read(5, table, starts)
    for out in (torch.zeros(5, 2, 2, 64, device="cuda").unbind(2), torch.zeros(5, 2, 128, device="cuda").split(64, -1),
                torch.zeros(2, 5, 2, 64, device="cuda").transpose(0, 1).unbind(2)):
        cache.read_into(*out, table, starts)
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
