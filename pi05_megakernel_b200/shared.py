"""Attention of several sequences that share one prefix.

``SharedPrefixAttention`` attends with the queries of a batch of sequences over the pages of one prefix, which are read once for the whole batch, and
over the pages of every sequence's own tokens: a step of several candidates that continue from one observation, drafted tokens that are checked in
one pass, or the tokens of several action chunks.  torch only supplies device memory and the current stream; the work is done by
``libpi05_b200.so``.
"""

from __future__ import annotations

import ctypes
import struct

import torch

from . import _lib
from .cache import MAX_FITS, KvCache, check_table, describe, meet, raw_stream, span, strides

CALL = struct.Struct("@PPP6qPPPP8if4x")      # pi05_shared_call of the header


class SharedPrefixAttention:
    """For calls of up to ``max_batch`` sequences x ``max_tokens`` queries of ``q_heads`` heads over ``cache``.  One call at a time: the calls
    share a workspace."""

    def __init__(self, cache: KvCache, q_heads: int, max_batch: int, max_tokens: int = 1) -> None:
        if q_heads < 1 or q_heads % cache.kv_heads or max_batch < 1 or max_tokens < 1:
            raise ValueError(f"q_heads must be a multiple of the cache's {cache.kv_heads} heads, max_batch and max_tokens at least 1")
        self.cache, self.q_heads, self.max_batch, self.max_tokens = cache, q_heads, max_batch, max_tokens
        self.lib, self.device = cache.lib, cache.device
        nbytes = ctypes.c_size_t()
        sms = torch.cuda.get_device_properties(self.device).multi_processor_count
        _lib.check(self.lib, None, self.lib.pi05_shared_workspace(sms, cache.ref, q_heads, max_batch, max_tokens, ctypes.byref(nbytes)))
        self.ws = torch.zeros(nbytes.value, dtype=torch.uint8, device=self.device)
        self.fresh = cache.fresh
        self.workspace, self.nbytes, self.index, self.fits, self.call = self.ws.data_ptr(), nbytes.value, self.device.index, {}, self.lib.pi05_shared_attention

    def run(self, q: torch.Tensor, prefix_table: torch.Tensor | None, prefix_tokens: int, table: torch.Tensor | None = None,
            lengths: torch.Tensor | None = None, layer: int = 0, valid: torch.Tensor | None = None, causal: bool = True,
            scale: float | None = None, out: torch.Tensor | None = None, with_lse: bool = False):
        """Asynchronous on the current stream.  ``q`` BF16 ``[batch, tokens, q_heads, head_dim]`` of any strides; returns the outputs in the same
        shape (in ``out``, whose rows lie in different places and not over ``q``) and, ``with_lse``, their log-sum-exp FP32 ``[batch, tokens, q_heads]``.

        ``prefix_table`` int32 ``[pages]`` names the pages of the ``prefix_tokens`` shared tokens, ``valid`` bool ``[prefix_tokens]`` which
        of them count (None: all).  ``table`` int32 ``[batch, pages]`` and ``lengths`` int32 ``[batch]`` are the sequences' own tokens, the
        queries' among them; ``causal``: query t sees own tokens up to its own place, ``lengths[b] - tokens + t``, else all of them.
        ``scale`` defaults to head_dim ** -0.5.  A query that sees no key gets zeros (log-sum-exp: -infinity)."""
        key = (q.shape, q.stride(), q.dtype, q.device, describe(out), describe(prefix_table), prefix_tokens, describe(table), describe(lengths),
               describe(valid), layer, causal, scale)
        given = out is not None
        if not given:
            out = self.fresh(q.shape, torch.bfloat16)
        known = self.fits.get(key)
        if known is None:
            if len(self.fits) >= MAX_FITS:
                self.fits.clear()
            fit = self._fit(q, out, prefix_table, prefix_tokens, table, lengths, layer, valid, causal, scale)
            known = self.fits[key] = (fit, span(q), span(out))
        fit, q_span, out_span = known
        qp, op = q.data_ptr(), out.data_ptr()
        if (qp | op) & 15:
            raise ValueError("q and out need strides of multiples of 8 elements, a contiguous last dimension and 16-byte alignment")
        if given and qp < op + out_span and op < qp + q_span and meet(self.lib, q, out):
            raise ValueError("the rows of out must not lie over those of q")
        lse = self.fresh(q.shape[:3], torch.float32) if with_lse else None
        call = CALL.pack(qp, op, lse.data_ptr() if with_lse else 0, *fit[:6], prefix_table.data_ptr() if prefix_tokens else 0,
                         valid.data_ptr() if prefix_tokens and valid is not None else 0,
                         0 if table is None else table.data_ptr() or lengths.data_ptr(),          # (a table without pages: its lengths are checked all the same)
                         0 if lengths is None else lengths.data_ptr(), *fit[6:])
        rc = self.call(self.index, self.cache.ref, call, self.workspace, self.nbytes, raw_stream(self.index))
        if rc:
            _lib.check(self.lib, None, rc)
        return (out, lse) if with_lse else out

    def _fit(self, q, out, prefix_table, prefix_tokens, table, lengths, layer, valid, causal, scale, shapes_only=False):
        """What does not depend on addresses, checked, as in ``KvCache``."""
        c = self.cache
        if q.dim() != 4 or q.dtype != torch.bfloat16 or (q.device != self.device and not shapes_only) or q.shape[2] != self.q_heads or q.shape[3] != c.head_dim:
            raise ValueError(f"q must be bfloat16 [batch, tokens, {self.q_heads}, {c.head_dim}] on {self.device}")
        batch, tokens = q.shape[:2]
        if batch > self.max_batch or tokens > self.max_tokens:
            raise ValueError(f"{batch} x {tokens} queries: made for up to {self.max_batch} x {self.max_tokens}")
        scale = c.head_dim ** -0.5 if scale is None else scale
        if not 0 <= layer < c.layers or prefix_tokens < 0 or not 0 < scale < float("inf"):
            raise ValueError("no such layer in the cache, a negative prefix_tokens, or a scale that is not positive and finite")
        if out.shape != q.shape or out.dtype != torch.bfloat16 or (out.device != self.device and not shapes_only):
            raise ValueError("out must be like q")
        qs, os_ = strides(q), strides(out)
        if q.stride(3) != 1 or out.stride(3) != 1 or any(s % 8 for s in qs + os_):
            raise ValueError("q and out need strides of multiples of 8 elements, a contiguous last dimension and 16-byte alignment")
        if meet(self.lib, out):
            raise ValueError("the rows of out must lie in different places")
        if prefix_tokens:
            if prefix_table is None:
                raise ValueError("a prefix needs its page table")
            check_table("prefix_table", prefix_table, self.device, 1)
            if prefix_table.shape[0] * c.page_tokens < prefix_tokens:
                raise ValueError("the prefix's page table is too short")
            if valid is not None and (valid.dtype != torch.bool or tuple(valid.shape) != (prefix_tokens,) or not valid.is_contiguous() or valid.device != self.device):
                raise ValueError(f"valid must be a contiguous bool tensor [{prefix_tokens}] on {self.device}")
        if (table is None) != (lengths is None):
            raise ValueError("own tokens need a table and lengths")
        pages = 0
        if table is not None:
            check_table("table", table, self.device, 2)
            check_table("lengths", lengths, self.device, 1)
            if table.shape[0] != batch or lengths.shape[0] != batch:
                raise ValueError("table and lengths need an entry per sequence")
            pages = table.shape[1]
        return (*qs, *os_, batch, tokens, self.q_heads, layer, prefix_tokens, table.stride(0) if pages and batch > 1 else pages, pages, bool(causal), scale)

    def status(self) -> None:
        """``KvCache.status`` of the cache."""
        self.cache.status()
