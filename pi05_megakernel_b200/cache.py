"""The prefix cache in pages, in BF16 or quantised to 8 bits as it is written.

``KvCache`` holds pools of keys and values for any number of sequences: the prefix that ``Pi05Prefill`` produces, of one observation or of many,
and the tokens that follow it.  ``write`` puts rows into the pages that a table names, ``read`` brings them back as the dense BF16 tensors that
``Pi05Arm.bind`` takes; ``SharedPrefixAttention`` (shared.py) attends over the pages in place.  torch only supplies device memory and the
current stream; the work is done by ``libpi05_b200.so``.
"""

from __future__ import annotations

import ctypes
import math
import struct

import torch

from . import _lib

FORMATS = {"bf16": (_lib.CACHE_BF16, torch.bfloat16), "int8": (_lib.CACHE_INT8, torch.int8), "e4m3": (_lib.CACHE_E4M3, torch.float8_e4m3fn)}

ROWS = struct.Struct("@PP4qPPP6i")           # pi05_cache_rows of the header
MAX_FITS = 256                                # shapes whose checks are kept


def check_table(name: str, t: torch.Tensor, device: torch.device, dim: int) -> None:
    if t.dtype != torch.int32 or t.dim() != dim or t.device != device or (t.numel() > 1 and t.stride(-1) != 1):
        raise ValueError(f"{name} must be an int32 tensor of {dim} dimensions on {device}, contiguous along its last")


# The current stream of a device as an integer; the public way to it makes an object, which takes 2 us of a call that takes 6.
raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


class Fresh:
    """New tensors like those of earlier calls: from a template (one element, expanded) an allocation takes 1.3 us, from sizes, type and device 2.5 to 3.3."""

    def __init__(self, device: torch.device) -> None:
        self.device, self.templates = device, {}

    def __call__(self, shape, dtype: torch.dtype) -> torch.Tensor:
        t = self.templates.get((shape, dtype))
        if t is None:
            if len(self.templates) >= MAX_FITS:
                self.templates.clear()
            t = self.templates[(shape, dtype)] = torch.empty(1, dtype=dtype, device=self.device).expand(shape)
        return torch.empty_like(t, memory_format=torch.contiguous_format)


def describe(t: torch.Tensor | None):
    """What a check of a table goes by."""
    return None if t is None else (t.shape, t.stride(), t.dtype, t.device)


def strides(t: torch.Tensor) -> list[int]:
    """Strides of the dimensions but the last one; those of a single entry do not matter and are 0."""
    return [0 if n == 1 else s for n, s in zip(t.shape[:-1], t.stride()[:-1])]


def meet(lib, a: torch.Tensor, b: torch.Tensor | None = None) -> bool:
    """Whether two rows (along the last dimension) of a tensor lie on one another, or one of ``a`` and one of ``b``."""
    numbers = lambda v: (ctypes.c_longlong * len(v))(*v)
    other = (None, None, 0) if b is None else (numbers(b.shape[:-1]), numbers(strides(b)), (b.data_ptr() - a.data_ptr()) // a.element_size())
    return bool(lib.pi05_rows_meet(a.dim() - 1, numbers(a.shape[:-1]), numbers(strides(a)), *other, a.shape[-1]))


def span(t: torch.Tensor) -> int:
    """Bytes from a tensor's first element to behind its last."""
    return t.element_size() * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))) if t.numel() else 0


class KvCache:
    """``pages`` pages of ``page_tokens`` tokens (a multiple of 16) for ``layers`` layers and ``kv_heads`` heads of ``head_dim`` (64, 128 or 256)
    elements; ``format`` is ``"bf16"``, ``"int8"`` or ``"e4m3"``.

    ``k`` and ``v`` are the pools ``[pages, layers, page_tokens, kv_heads, head_dim]``; of the 8-bit formats ``k_scale`` and ``v_scale``
    ``[pages, layers, kv_heads, page_tokens]`` FP32 hold a scale per token and head, and an element stands for code x scale.  A BF16 cache of
    one head of 256 is a pool that ``PagedPrefix`` takes as it is.
    """

    def __init__(self, pages: int, layers: int, page_tokens: int, kv_heads: int = 1, head_dim: int = 256, format: str = "int8",
                 device: str = "cuda") -> None:
        if format not in FORMATS:
            raise ValueError(f"bad format {format!r}: expected one of {', '.join(FORMATS)}")
        if min(pages, layers, kv_heads) < 1 or page_tokens < 16 or page_tokens % 16 or head_dim not in (64, 128, 256):
            raise ValueError("a cache needs pages, layers and heads, pages of a multiple of 16 tokens, and heads of 64, 128 or 256 elements")
        if not torch.cuda.is_available():
            raise RuntimeError("no CUDA device: the cache has no CPU path")
        shape = (pages, layers, page_tokens, kv_heads, head_dim)
        pools = [torch.zeros(shape, dtype=FORMATS[format][1], device=device) for _ in range(2)]
        scales = [None if format == "bf16" else torch.zeros((pages, layers, kv_heads, page_tokens), device=device) for _ in range(2)]
        self._set(*pools, *scales)

    @classmethod
    def wrap(cls, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None) -> "KvCache":
        """A cache over pools that exist already (the shapes above, contiguous).  The format has no e4m3 NaNs: a row that is not a number has a NaN as its
        scale, which is what ``write`` gives it, and rows that hold such codes (0x7f, 0xff) now get one here.  Pools that something else writes later have to be
        wrapped again."""
        self = cls.__new__(cls)
        self._set(k, v, k_scale, v_scale)
        if self.format == "e4m3":
            with torch.no_grad():
                for codes, scale in ((k, k_scale), (v, v_scale)):
                    step = max(1, (1 << 26) // max(1, codes[0].numel()))
                    for c, s in zip(codes.view(torch.uint8).split(step), scale.split(step)):
                        s.masked_fill_(c.bitwise_and(127).amax(-1).eq(127).transpose(2, 3), math.nan)
        return self

    def _set(self, k, v, k_scale, v_scale) -> None:
        names = {dtype: name for name, (_, dtype) in FORMATS.items()}
        if k.dim() != 5 or k.shape != v.shape or k.dtype != v.dtype or k.dtype not in names or k.device != v.device or k.device.type != "cuda":
            raise ValueError("k and v must be CUDA tensors [pages, layers, page_tokens, kv_heads, head_dim] of one type: bfloat16, int8 or float8_e4m3fn")
        self.pages, self.layers, self.page_tokens, self.kv_heads, self.head_dim = k.shape
        self.format, self.device = names[k.dtype], k.device
        want = (self.pages, self.layers, self.kv_heads, self.page_tokens)
        for t in (k_scale, v_scale):
            if (t is None) != (self.format == "bf16"):
                raise ValueError("8-bit pools need scales, BF16 pools have none")
            if t is not None and (tuple(t.shape) != want or t.dtype != torch.float32 or t.device != k.device):
                raise ValueError(f"scales must be float32 {want} on {k.device}")
        if not all(t is None or t.is_contiguous() for t in (k, v, k_scale, v_scale)):
            raise ValueError("pools and scales must be contiguous")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.lib = _lib.load()
        self.words = torch.zeros(4, dtype=torch.int32, device=self.device)       # the status words
        scale = (None, None) if k_scale is None else (k_scale.data_ptr(), v_scale.data_ptr())
        self.struct = _lib.Cache(k.data_ptr(), v.data_ptr(), *scale, self.words.data_ptr(), FORMATS[self.format][0], *k.shape)
        self.ref, self.index, self.fits, self.fresh = ctypes.byref(self.struct), self.device.index, {}, Fresh(self.device)
        self.call_write, self.call_read = self.lib.pi05_cache_write, self.lib.pi05_cache_read
        # what the library refuses is refused here, before a first call
        nbytes = ctypes.c_size_t()
        _lib.check(self.lib, None, self.lib.pi05_shared_workspace(1, self.ref, self.kv_heads, 1, 1, ctypes.byref(nbytes)))

    def _fit(self, k, v, table, starts, counts, layer):
        """What does not depend on addresses, checked: the strides and sizes of the call.  Kept by shapes and types, since checking costs as much as
        a small call."""
        if k.dim() != 5 or k.shape != v.shape or k.dtype != torch.bfloat16 or v.dtype != torch.bfloat16 or k.device != self.device or v.device != self.device:
            raise ValueError(f"k and v must be bfloat16 [batch, layers, tokens, kv_heads, head_dim] on {self.device}")
        batch, layers, tokens, heads, dim = k.shape
        if heads != self.kv_heads or dim != self.head_dim or layer < 0 or layer + layers > self.layers:
            raise ValueError(f"{tuple(k.shape)} from layer {layer} on does not fit a cache of {self.layers} layers x {self.kv_heads} heads of {self.head_dim}")
        st = strides(k)
        if st != strides(v) or k.stride(4) != 1 or v.stride(4) != 1 or any(s % 8 for s in st):
            raise ValueError("k and v must share their strides (multiples of 8 elements, the last dimension contiguous) and be 16-byte aligned")
        check_table("table", table, self.device, 2)
        if table.shape[0] != batch:
            raise ValueError("the page table needs a row per sequence")
        for name, t in (("starts", starts), ("counts", counts)):
            if t is not None:
                check_table(name, t, self.device, 1)
                if t.shape[0] != batch:
                    raise ValueError(f"{name} needs an entry per sequence")
        return (*st, batch, layers, tokens, layer, table.stride(0) if batch > 1 else table.shape[1], table.shape[1])

    def _rows(self, k, v, table, starts, counts, layer) -> bytes:
        key = (k.shape, v.shape, k.stride(), v.stride(), k.dtype, v.dtype, k.device, v.device, layer, describe(table), describe(starts), describe(counts))
        fit = self.fits.get(key)
        if fit is None:
            if len(self.fits) >= MAX_FITS:
                self.fits.clear()
            fit = self.fits[key] = self._fit(k, v, table, starts, counts, layer)
        kp, vp = k.data_ptr(), v.data_ptr()
        if (kp | vp) & 15:
            raise ValueError("k and v must share their strides (multiples of 8 elements, the last dimension contiguous) and be 16-byte aligned")
        # (a table without pages: a place that is never read, so that what its rows ask for is reported like any other)
        return ROWS.pack(kp, vp, *fit[:4], table.data_ptr() or kp, 0 if starts is None else starts.data_ptr(), 0 if counts is None else counts.data_ptr(), *fit[4:])

    def _apart(self, k, v) -> None:
        """Refuses outputs that several blocks would write at once."""
        key = ("out", k.shape, k.stride())
        reach = self.fits.get(key)
        if reach is None:
            if meet(self.lib, k):
                raise ValueError("the rows of out must lie in different places")
            reach = self.fits[key] = span(k)
        if abs(k.data_ptr() - v.data_ptr()) < reach and meet(self.lib, k, v):
            raise ValueError("the rows of out must lie in different places")

    def write(self, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, starts: torch.Tensor | None = None,
              counts: torch.Tensor | None = None, layer: int = 0) -> None:
        """Rows into their pages, asynchronous on the current stream.  ``k``, ``v`` BF16 ``[batch, layers, tokens, kv_heads, head_dim]`` of any
        strides that they share go to layers ``layer`` .. of the cache and to the tokens ``starts[b]`` .. (None: 0 ..) of sequence ``b``, whose
        pages ``table`` int32 ``[batch, pages]`` names; of a padded batch only the first ``counts[b]`` tokens are taken.  Tokens of one call must
        lie in different places of the cache."""
        rc = self.call_write(self.index, self.ref, self._rows(k, v, table, starts, counts, layer), raw_stream(self.index))
        if rc:
            _lib.check(self.lib, None, rc)

    def read(self, table: torch.Tensor, tokens: int, starts: torch.Tensor | None = None, counts: torch.Tensor | None = None, layer: int = 0,
             layers: int | None = None, out: tuple[torch.Tensor, torch.Tensor] | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """Rows out of their pages, asynchronous on the current stream: BF16 keys and values ``[batch, layers, tokens, kv_heads, head_dim]`` of
        layers ``layer`` .. (all that there are), zeros behind ``counts[b]``; the rest as in ``write``.  The rows of ``out`` lie in different places, those of
        keys and of values too."""
        if layers is None:
            layers = self.layers - layer
        given = out is not None
        if not given:
            shape = (table.shape[0], layers, tokens, self.kv_heads, self.head_dim)
            out = (self.fresh(shape, torch.bfloat16), self.fresh(shape, torch.bfloat16))
        elif out[0].shape[1:3] != (layers, tokens):
            raise ValueError("out does not have the layers and tokens that are read")
        rows = self._rows(*out, table, starts, counts, layer)
        if given:
            self._apart(*out)
        rc = self.call_read(self.index, self.ref, rows, raw_stream(self.index))
        if rc:
            _lib.check(self.lib, None, rc)
        return out

    def status(self) -> None:
        """Synchronise the current stream; raises when a call met a page or a position out of range, or a device-side wait gave up, since the last
        time it was asked."""
        code, where = ctypes.c_int(), ctypes.c_int()
        rc = self.lib.pi05_cache_status(self.device.index, self.ref, torch.cuda.current_stream(self.device).cuda_stream, ctypes.byref(code),
                                        ctypes.byref(where))
        if rc == _lib.ERR_PAGE_TABLE:
            what = "page" if code.value == _lib.CACHE_BAD_PAGE else "start or length"
            raise _lib.EngineError(rc, f"{what} out of range in " + (f"sequence {where.value}" if where.value >= 0 else "the shared prefix"))
        if rc == _lib.ERR_DEVICE_TIMEOUT:
            raise _lib.EngineError(rc, f"device wait kind {code.value} gave up in block {where.value >> 16}")
        _lib.check(self.lib, None, rc)
