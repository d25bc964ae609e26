"""The token-generation entry points without a GPU: calls that are refused before anything is launched."""

from __future__ import annotations

import contextlib
import ctypes

import pytest
import torch

from tgcb import _lib, attention, heads, kv_cache, rotary
from tgcb.errors import ConfigError, DeviceError

memory = (ctypes.c_char * 4096)()  # never read: every call here is refused for its arguments
HERE = (ctypes.addressof(memory) + 255) & ~255


def rotary_desc(**change):
    d = _lib.RotaryDesc(dtype=0, gain_dtype=0, position_bytes=4, tokens=3, heads=(2, 1), width=64, rotary=64, epsilon=1e-5, positions=HERE,
                        frequencies=HERE, gain=(HERE, HERE), gain_grad=(HERE, HERE), scratch=HERE, scratch_bytes=1 << 40)
    for i in range(2):
        d.rows_in[i] = d.grad[i] = d.rows_out[i] = _lib.Heads(HERE, 64, 64)
    for name, value in change.items():
        setattr(d, name, value)
    return d


@pytest.mark.parametrize("change,why", [
    (dict(dtype=3), "element type"), (dict(dtype=-1), "element type"), (dict(gain_dtype=1), "gains"), (dict(position_bytes=2), "positions"),
    (dict(tokens=-1), "negative"), (dict(heads=(0, 1)), "head"), (dict(width=1), "width"), (dict(width=1025), "width"), (dict(rotary=0), "rotary"),
    (dict(rotary=63), "rotary"), (dict(rotary=66), "rotary"), (dict(epsilon=0.0), "epsilon"), (dict(epsilon=float("nan")), "epsilon"), (dict(epsilon=1e-60), "epsilon"),
    (dict(positions=None), "null"), (dict(frequencies=None), "null"), (dict(gain=(HERE, None)), "null"), (dict(heads=(1 << 21, 1)), "2\\^20"),
])
def test_norm_rotate_refuses(change, why):
    lib = _lib.load()
    for entry in (lib.tgcb_norm_rotate, lib.tgcb_norm_rotate_backward):
        assert entry(rotary_desc(**change), None) == _lib.TGCB_E_INVALID
        with pytest.raises(Exception, match=why):
            _lib.check(_lib.TGCB_E_INVALID, "norm_rotate")


def test_norm_rotate_backward_refuses_its_scratch():
    lib = _lib.load()
    need = lib.tgcb_norm_rotate_scratch_bytes(64)
    for change in (dict(scratch=None), dict(scratch_bytes=need - 1), dict(scratch=HERE + 4), dict(gain_grad=(HERE, None))):
        assert lib.tgcb_norm_rotate_backward(rotary_desc(**change), None) == _lib.TGCB_E_INVALID
    assert lib.tgcb_norm_rotate(None, None) == _lib.TGCB_E_INVALID
    assert lib.tgcb_norm_rotate_scratch_bytes(0) == 0


def cache_desc(**change):
    return _lib.CacheDesc(**{**dict(keys=HERE, values=HERE, key_scales=HERE, value_scales=HERE, faults=HERE, pages=4, kv_heads=2, page=16,
                                    width=64), **change})


def batch_desc(**change):
    return _lib.BatchDesc(**{**dict(table=HERE, starts=HERE, offsets=None, table_stride=2, tokens=6, batch=3, max_pages=2), **change})


@pytest.mark.parametrize("cache,batch,dtype", [
    (dict(keys=None), {}, 0), (dict(value_scales=None), {}, 0), (dict(faults=None), {}, 0), (dict(values=HERE + 8), {}, 0), (dict(width=48), {}, 0),
    (dict(page=24), {}, 0), (dict(page=0), {}, 0), (dict(kv_heads=0), {}, 0), (dict(pages=0), {}, 0), (dict(pages=1 << 31), {}, 0),
    ({}, dict(table=None), 0), ({}, dict(starts=None), 0), ({}, dict(batch=0), 0), ({}, dict(batch=4097), 0), ({}, dict(max_pages=0), 0),
    ({}, dict(tokens=-1), 0), ({}, dict(tokens=7), 0), ({}, dict(tokens=1 << 32), 0), ({}, {}, 3), ({}, {}, -1),
])
def test_cache_calls_refuse(cache, batch, dtype):
    lib, rows = _lib.load(), _lib.Heads(HERE, 128, 64)
    c, b = cache_desc(**cache), batch_desc(**batch)
    assert lib.tgcb_cache_append(c, b, dtype, rows, rows, None) == _lib.TGCB_E_INVALID
    assert lib.tgcb_cache_read(c, b, dtype, rows, rows, None) == _lib.TGCB_E_INVALID
    assert lib.tgcb_cached_attention(c, b, dtype, 4, rows, None, 1.0, 0.0, rows, HERE, 1 << 40, None) == _lib.TGCB_E_INVALID


def test_null_rows_and_descriptors_are_refused():
    lib, rows, nothing = _lib.load(), _lib.Heads(HERE, 128, 64), _lib.Heads(None, 128, 64)
    c, b = cache_desc(), batch_desc()
    for k, v in ((None, rows), (rows, None), (nothing, rows), (rows, nothing)):
        assert lib.tgcb_cache_append(c, b, 0, k, v, None) == _lib.TGCB_E_INVALID
        assert lib.tgcb_cache_read(c, b, 0, k, v, None) == _lib.TGCB_E_INVALID
        assert lib.tgcb_cached_attention(c, b, 0, 4, k, None, 1.0, 0.0, v, HERE, 1 << 40, None) == _lib.TGCB_E_INVALID
    assert lib.tgcb_cache_append(None, b, 0, rows, rows, None) == _lib.TGCB_E_INVALID
    assert lib.tgcb_cache_append(c, None, 0, rows, rows, None) == _lib.TGCB_E_INVALID


@pytest.mark.parametrize("q_heads,scale,cap", [(3, 1.0, 0.0), (0, 1.0, 0.0), (4, float("nan"), 0.0), (4, float("inf"), 0.0), (4, 1.0, -1.0),
                                               (4, 1.0, float("nan")), (4, 1.0, float("inf")), (4, 1e31, 0.0), (4, 1.0, 1e-35)])
def test_attention_refuses(q_heads, scale, cap):
    lib, rows = _lib.load(), _lib.Heads(HERE, 256, 64)
    rc = lib.tgcb_cached_attention(cache_desc(), batch_desc(), 0, q_heads, rows, None, scale, cap, rows, HERE, 1 << 40, None)
    assert rc == _lib.TGCB_E_INVALID


class Faults:
    """A counter of a device that goes on counting: one more after every read."""

    def __init__(self):
        self.value = 1

    def item(self):
        self.value += 1
        return self.value - 1

    def zero_(self):
        self.value = 0


class Device:
    """The library's status word, read and cleared as on a device."""

    def __init__(self, status=0):
        self.status = status

    def tgcb_status(self, clear, to):
        to._obj.value = self.status
        if clear:
            self.status = 0
        return _lib.TGCB_OK


def counting_cache(monkeypatch, device):
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *_: None)
    monkeypatch.setattr(heads, "on_device", lambda _: contextlib.nullcontext())
    monkeypatch.setattr(_lib, "load", lambda: device)
    cache = kv_cache.QuantisedCache.__new__(kv_cache.QuantisedCache)
    cache.faults, cache.device, cache.index, cache._reported = Faults(), torch.device("cuda:0"), 0, 0
    return cache


def test_check_reports_a_kernel_that_gave_up(monkeypatch):
    device = Device(6)
    cache = counting_cache(monkeypatch, device)
    with pytest.raises(DeviceError, match="status 6"):
        cache.check()
    with pytest.raises(ConfigError, match="^1 accesses"):  # not lost beside it
        cache.check()
    assert device.status == 0


def test_check_loses_no_count(monkeypatch):
    cache = counting_cache(monkeypatch, Device())
    for _ in range(3):
        with pytest.raises(ConfigError, match="^1 accesses"):
            cache.check()
    cache.faults.value, cache._reported = -(1 << 31) + 5, (1 << 31) - 5  # the int32 has wrapped around
    with pytest.raises(ConfigError, match="^10 accesses"):
        cache.check()


def test_parts_of_the_same_rows_are_apart():
    halves, both = torch.zeros(5, 3, 128), torch.zeros(5, 3, 2, 64)
    side_by_side, by_head = torch.zeros(5, 7, 64), torch.zeros(3, 5, 2, 64).transpose(0, 1)
    for a, b in ((halves[..., :64], halves[..., 64:]), both.unbind(2), (side_by_side[:, :3], side_by_side[:, 3:6]), by_head.unbind(2),
                 (side_by_side[:, :2], side_by_side[:, 2:]), (side_by_side[:, ::2], side_by_side[:, 1::2][:, :3]), (side_by_side[:2], side_by_side[2:])):
        assert not heads.overlap(a, b) and not heads.overlap(b, a)
    for a, b in ((halves[..., :65], halves[..., 64:]), (side_by_side[:, :4], side_by_side[:, 3:]), (by_head[:, :, 0], by_head[:, :, 0]),
                 (side_by_side[:3], side_by_side[2:]), (halves, halves[1:2])):
        assert heads.overlap(a, b) and heads.overlap(b, a)


def test_rows_that_share_memory_are_never_taken_as_apart():
    g = torch.Generator().manual_seed(0)
    number = lambda low, high: int(torch.randint(low, high, (1,), generator=g))  # noqa: E731
    memory, apart, shared = torch.arange(400), 0, 0
    for _ in range(3000):
        strides = number(0, 30), number(0, 30)
        shape = number(1, 4), number(1, 4), number(1, 9)
        a = memory.as_strided(shape, (*strides, 1), number(0, 60))
        if number(0, 2):
            shape = number(1, 4), number(1, 4), number(1, 9)
        if not number(0, 3):
            strides = number(0, 30), number(0, 30)
        b = memory.as_strided(shape, (*strides, 1), number(0, 60))
        meet = not set(a.reshape(-1).tolist()).isdisjoint(b.reshape(-1).tolist())
        assert heads.overlap(a, b) or not meet
        apart, shared = apart + (not heads.overlap(a, b)), shared + meet
    assert apart > 500 and shared > 500


@pytest.mark.parametrize("index", [0, 1])
def test_a_call_on_another_device_leaves_the_current_one(monkeypatch, index):
    current, set_up = [0], []

    @contextlib.contextmanager
    def device(i):
        before, current[0] = current[0], i
        yield
        current[0] = before

    def ensure(i):  # as tgcb_init: the first call on a device selects it
        if i not in set_up:
            set_up.append(i)
            current[0] = i

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(_lib, "ensure_device", ensure)
    for _ in range(2):
        with heads.on_device(index):
            assert current[0] == index and set_up == [index]
        assert current[0] == 0


def test_host_tensors_are_refused():
    rows, gain = torch.randn(2, 2, 64), torch.ones(64)
    with pytest.raises(ConfigError):
        rotary.norm_rotate(rows, rows, gain, gain, torch.zeros(2, dtype=torch.int32), torch.ones(32, dtype=torch.float64))
    with pytest.raises(ConfigError):
        kv_cache.QuantisedCache(4, 2, 64, device="cpu")
    with pytest.raises(ConfigError):
        attention.cached_attention(rows, None, torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32))


@pytest.mark.parametrize("cap", [1e31, 3e38])
def test_attention_refuses_caps_beyond_float32(cap):
    lib, rows = _lib.load(), _lib.Heads(HERE, 256, 64)
    assert lib.tgcb_cached_attention(cache_desc(), batch_desc(), 0, 4, rows, None, 1.0, cap, rows, HERE, 1 << 40, None) == _lib.TGCB_E_INVALID
    with pytest.raises(Exception, match="cap is at most"):
        _lib.check(_lib.TGCB_E_INVALID, "cached_attention")
