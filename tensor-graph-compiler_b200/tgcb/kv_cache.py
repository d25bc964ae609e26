"""A paged int8 cache of keys and values, quantised as it is written.

Each cached row (one position of one key head) is ``width`` int8 codes and a float32 scale by
the rule of ``tgcb.quantize.quantise_rows``, bit for bit: scale = max|x| / 127, code =
rint(x / scale). Rows lie in pages of 16 to 128 positions; a page table names each sequence's
pages in order, and pages may be anywhere and shared by sequences that only read them.

A call's token rows belong to sequences: ``offsets`` [batch + 1] says which rows are whose (without it
every sequence has tokens / batch of them), ``starts`` [batch] how many positions each had before, so row i of sequence b
is position ``starts[b] + i``. All three are int32 on the device and are read when the kernels run: a
captured call can be replayed with other lengths. Rows of no sequence are left as they
were. Positions that the table does not hold and pages outside the cache are never accessed; they are
counted, and ``check`` raises for them, as for a kernel that gave up waiting.
"""

from __future__ import annotations

import ctypes

import torch

from tgcb import _lib, heads
from tgcb.errors import ConfigError, DeviceError

PAGES = (16, 32, 64, 128)
WIDTHS = (32, 64, 128, 256)
MAX_BATCH = 4096
MAX_POSITIONS = 1 << 30
_INT32 = (torch.int32,)


def batch_of(table: torch.Tensor, starts: torch.Tensor, offsets: torch.Tensor | None, tokens: int, index: int) -> _lib.BatchDesc:
    """The checked description of a call's sequences, on CUDA device ``index``."""
    if not isinstance(table, torch.Tensor) or table.get_device() != index or table.dtype is not torch.int32 or table.dim() != 2:
        raise ConfigError(f"the page table must be an int32 matrix [batch, pages] on cuda:{index}")
    batch, pages = table.shape
    step, unit = table.stride()
    if not 1 <= batch <= MAX_BATCH or pages < 1:
        raise ConfigError(f"a call takes 1 to {MAX_BATCH} sequences of at least one page, got {batch} of {pages}")
    if pages > 1 and unit != 1:
        raise ConfigError("the page table must have a unit stride along its pages")
    heads.check_vector("starts", starts, batch, _INT32, index)
    if offsets is not None:
        heads.check_vector("offsets", offsets, batch + 1, _INT32, index)
    elif tokens % batch:
        raise ConfigError(f"without offsets every sequence has the same number of tokens: {tokens} over {batch} sequences")
    return _lib.BatchDesc(table.data_ptr(), starts.data_ptr(), offsets.data_ptr() if offsets is not None else None, step, tokens, batch, pages)


class QuantisedCache:
    """The pages: ``keys`` and ``values`` int8 [pages, kv_heads, page, width], ``key_scales`` and
    ``value_scales`` float32 [pages, kv_heads, page]."""

    def __init__(self, pages: int, kv_heads: int, width: int, page: int = 64, device=None):
        if pages < 1 or kv_heads < 1:
            raise ConfigError(f"a cache cannot have {pages} pages of {kv_heads} heads")
        device = torch.device(device if device is not None else "cuda")
        shape = (pages, kv_heads, page)
        self._hold(*(torch.zeros(s, dtype=t, device=device) for _ in range(2) for s, t in (((*shape, width), torch.int8), (shape, torch.float32))))

    @classmethod
    def of(cls, keys: torch.Tensor, key_scales: torch.Tensor, values: torch.Tensor, value_scales: torch.Tensor) -> QuantisedCache:
        """A cache over tensors that hold its pages already; they are used as they are, not copied."""
        cache = cls.__new__(cls)
        cache._hold(keys, key_scales, values, value_scales)
        return cache

    def _hold(self, keys, key_scales, values, value_scales) -> None:
        if not isinstance(keys, torch.Tensor) or not keys.is_cuda or keys.dim() != 4 or keys.dtype != torch.int8:
            raise ConfigError("keys must be an int8 CUDA tensor [pages, kv_heads, page, width]")
        pages, kv_heads, page, width = keys.shape
        if width not in WIDTHS:
            raise ConfigError(f"the cache takes widths {WIDTHS}, got {width}")
        if page not in PAGES:
            raise ConfigError(f"the cache takes pages of {PAGES} positions, got {page}")
        if not 1 <= pages < 1 << 31 or not 1 <= kv_heads <= 1024:
            raise ConfigError(f"a cache cannot have {pages} pages of {kv_heads} heads")
        for name, t, shape, dtype in (("keys", keys, keys.shape, torch.int8), ("values", values, keys.shape, torch.int8),
                                      ("key_scales", key_scales, keys.shape[:3], torch.float32),
                                      ("value_scales", value_scales, keys.shape[:3], torch.float32)):
            if not isinstance(t, torch.Tensor) or t.device != keys.device or t.dtype != dtype or t.shape != shape:
                raise ConfigError(f"{name} must be {dtype} {tuple(shape)} on {keys.device}")
            if not t.is_contiguous() or t.data_ptr() % 16:
                raise ConfigError(f"{name} must be contiguous and 16-byte aligned")
        self.keys, self.key_scales, self.values, self.value_scales = keys, key_scales, values, value_scales
        self.pages, self.kv_heads, self.page, self.width = pages, kv_heads, page, width
        self.device, self.index = keys.device, keys.get_device()
        self.faults = torch.tensor([0], dtype=torch.int32, device=keys.device)  # there when this returns, for calls on any stream
        self._reported = 0
        self.desc = _lib.CacheDesc(keys.data_ptr(), values.data_ptr(), key_scales.data_ptr(), value_scales.data_ptr(),
                                   self.faults.data_ptr(), pages, kv_heads, page, width)

    @property
    def bytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.keys, self.values, self.key_scales, self.value_scales))

    def _check_rows(self, name: str, t: torch.Tensor, like: torch.Tensor | None = None) -> None:
        heads.check_rows(name, t, like)
        if t.get_device() != self.index:
            raise ConfigError(f"{name} must be on {self.device}, where the cache is")
        tokens, kv_heads, width = t.shape
        if kv_heads != self.kv_heads or width != self.width or (like is not None and tokens != like.shape[0]):
            raise ConfigError(f"{name} must be [tokens, {self.kv_heads}, {self.width}], got {tuple(t.shape)}")

    def batch_of(self, table: torch.Tensor, starts: torch.Tensor, offsets: torch.Tensor | None, tokens: int) -> _lib.BatchDesc:
        """The checked description of a call's sequences."""
        b = batch_of(table, starts, offsets, tokens, self.index)
        if b.max_pages * self.page > MAX_POSITIONS:
            raise ConfigError(f"a page table holds at most 2^30 positions a sequence, got {b.max_pages} pages of {self.page}")
        return b

    def _call(self, entry, name: str, keys, values, b: _lib.BatchDesc, stream) -> None:
        with heads.on_device(self.index):
            rc = entry(self.desc, b, heads.DTYPES[keys.dtype], _lib.Heads(*heads.rows(keys)), _lib.Heads(*heads.rows(values)),
                       heads.raw(self.index, stream))
        _lib.check(rc, name)

    def append(self, keys: torch.Tensor, values: torch.Tensor, table: torch.Tensor, starts: torch.Tensor,
               offsets: torch.Tensor | None = None, *, stream=None) -> None:
        """Quantise each token's key and value rows [tokens, kv_heads, width] into their places.

        Where several rows of a call have one place, the last of them is stored.
        """
        self._check_rows("keys", keys)
        self._check_rows("values", values, keys)
        b = self.batch_of(table, starts, offsets, keys.shape[0])
        self._call(_lib.load().tgcb_cache_append, "tgcb_cache_append", keys, values, b, stream)

    def read_into(self, keys: torch.Tensor, values: torch.Tensor, table: torch.Tensor, starts: torch.Tensor,
                  offsets: torch.Tensor | None = None, *, stream=None) -> None:
        """Write code * scale of each token row's position into ``keys`` and ``values``, rounded to their type."""
        self._check_rows("keys", keys)
        self._check_rows("values", values, keys)
        heads.check_written("keys", keys)
        heads.check_written("values", values)
        heads.check_apart("keys", keys, "values", values)
        b = self.batch_of(table, starts, offsets, keys.shape[0])
        self._call(_lib.load().tgcb_cache_read, "tgcb_cache_read", keys, values, b, stream)

    def read(self, tokens: int, table: torch.Tensor, starts: torch.Tensor, offsets: torch.Tensor | None = None, *,
             dtype: torch.dtype = torch.float32, stream=None) -> tuple[torch.Tensor, torch.Tensor]:
        """The cached keys and values of ``tokens`` rows, new tensors [tokens, kv_heads, width].

        Rows of no sequence are not written.
        """
        if dtype not in heads.DTYPES:
            raise ConfigError(f"rows are read as float32, bfloat16 or float16, not {dtype}")
        if tokens < 0:
            raise ConfigError(f"there cannot be {tokens} tokens")
        b = self.batch_of(table, starts, offsets, tokens)
        with heads.on_stream(self.index, stream):
            keys, values = torch.empty((2, tokens, self.kv_heads, self.width), dtype=dtype, device=self.device).unbind()
        self._call(_lib.load().tgcb_cache_read, "tgcb_cache_read", keys, values, b, stream)
        return keys, values

    def check(self) -> None:
        """Synchronise the device and raise ``ConfigError`` if a call on any of its streams named positions or pages that are not
        there, since this was last called; ``DeviceError`` if a kernel gave up waiting, which leaves its call's output unfinished."""
        status = ctypes.c_int(0)
        with heads.on_device(self.index):
            _lib.check(_lib.load().tgcb_status(1, ctypes.byref(status)), "reading the device status")  # synchronises the device
        if status.value:
            raise DeviceError(f"a kernel on {self.device} reported device status {status.value}: an output is not finished")
        counted = int(self.faults.item())
        count, self._reported = (counted - self._reported) % (1 << 32), counted  # the device only ever adds to it
        if count:
            raise ConfigError(f"{count} accesses named a position outside the page table or a page outside the cache")
