"""Quantised, paged K/V cache for autoregressive decoding, through the C ABI.

* ``KvCache``                  the pool: pages of tokens held in 4 or 8 bits
* ``gpu_kv_cache_append``      quantises new tokens' K and V into it
* ``gpu_kv_cache_read``        dequantises tokens out of it
* ``gpu_kv_cache_attention``   causal attention of new tokens over it

The three calls name their tokens alike: ``page_table`` Int32 [batch, width]
gives each sequence's pages (position p stands in entry p // page_size),
``seq_lens`` Int32 [batch] its length *with* this call's tokens, and
``cu_tokens`` Int32 [batch + 1] where its tokens start in the packed operands
(sequence b's are rows cu_tokens[b] .. cu_tokens[b+1]-1 and its last
positions).  Without ``cu_tokens`` every sequence has one token.  All three
stay on the device: nothing is read back, so calls can be captured in CUDA
graphs and replayed with other values.

What the device finds wrong is never touched: a position before the start of
its sequence is skipped, and one without a usable page (entry outside the
pool, sequence longer than its row of the table) is skipped and noted as
``ICX_DEVICE_BAD_PAGE`` in ``icx_device_status``.  No gradient flows through
these calls.
"""

from __future__ import annotations

import ctypes
import math

import torch

from . import _lib
from ._lib import IcxError, KvCacheArg, KvTokensArg
from .ops import _float_type, _name, _on, _ptr


class KvCache:
    """A pool of ``pages`` pages of ``page_size`` tokens for ``kv_heads`` heads.

    Per (token, head) each group of ``group`` (32 or 64) dimensions keeps a
    bf16 scale s and low end lo and ``bits`` (4 or 8) per value, which stands
    for ``code * s + lo``: lo is the group's minimum rounded down, s its range
    over 2^bits - 1 rounded up, and codes are rounded half to even.  A group
    with a NaN or an infinity reads back as NaN.  ``page_size`` is a power of
    two in 16..1024, ``head_dim`` 64, 128 or 256.  A new pool is all zeros.
    ``k_codes``, ``v_codes``, ``k_params`` and ``v_params`` are its buffers, to be
    copied from and into (saving and restoring a pool), not to be replaced.
    """

    def __init__(self, pages: int, page_size: int, kv_heads: int, head_dim: int, bits: int = 4,
                 group: int = 64, device="cuda:0"):
        device = torch.device(device)
        if device.type != "cuda":
            raise IcxError(-1, f"KvCache: expected a CUDA device, got {device}")
        if bits not in (4, 8):
            raise IcxError(-1, f"KvCache: bits must be 4 or 8, got {bits}")
        if head_dim not in (64, 128, 256):
            raise IcxError(-1, f"KvCache: head_dim must be 64, 128 or 256, got {head_dim}")
        if group not in (32, 64):
            raise IcxError(-1, f"KvCache: group must be 32 or 64, got {group}")
        if page_size not in (16, 32, 64, 128, 256, 512, 1024):
            raise IcxError(-1, f"KvCache: page_size must be a power of two in 16..1024, got {page_size}")
        if not 1 <= kv_heads <= 1024:
            raise IcxError(-1, f"KvCache: kv_heads must be in 1..1024, got {kv_heads}")
        if not 0 <= pages < 1 << 31:
            raise IcxError(-1, f"KvCache: pages out of range: {pages}")
        self.pages, self.page_size, self.kv_heads = pages, page_size, kv_heads
        self.head_dim, self.bits, self.group = head_dim, bits, group
        rows = (pages, kv_heads, page_size)
        codes = (*rows, head_dim * bits // 8)
        params = (*rows, head_dim // group)
        self._buffers = [torch.zeros(shape, dtype=dtype, device=device)
                         for shape, dtype in ((codes, torch.uint8),) * 2 + ((params, torch.int32),) * 2]
        self.device = self._buffers[0].device
        self._arg = KvCacheArg(*(t.data_ptr() for t in self._buffers), pages, page_size, kv_heads, head_dim, bits,
                               group)
        self._ref = ctypes.byref(self._arg)

    # The calls take the buffers' addresses from _arg, so they stay the same
    # tensors for the pool's life.
    k_codes = property(lambda self: self._buffers[0])
    v_codes = property(lambda self: self._buffers[1])
    k_params = property(lambda self: self._buffers[2])
    v_params = property(lambda self: self._buffers[3])


def _index(t, shape, device, what: str) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or t.device != device:
        raise IcxError(-1, f"{what}: expected a tensor on {device}")
    if t.dtype != torch.int32 or t.dim() != len(shape) or (shape[0] is not None and t.shape[0] != shape[0]):
        raise IcxError(-1, f"{what}: expected Int32 [{', '.join('*' if n is None else str(n) for n in shape)}], "
                           f"got {_name(t.dtype)} {list(t.shape)}")
    return t.contiguous()


def _where(cache: KvCache, page_table, seq_lens, cu_tokens, tokens: int, what: str):
    """The icx_kv_tokens argument and the tensors it points into."""
    table = _index(page_table, (None, None), cache.device, f"{what}: page_table")
    batch, width = table.shape
    lens = _index(seq_lens, (batch,), cache.device, f"{what}: seq_lens")
    if cu_tokens is None:
        if tokens != batch:
            raise IcxError(-1, f"{what}: without cu_tokens there is one token per sequence "
                               f"({tokens} tokens, batch {batch})")
        cu = None
    else:
        cu = _index(cu_tokens, (batch + 1,), cache.device, f"{what}: cu_tokens")
    return KvTokensArg(table.data_ptr(), lens.data_ptr(), _ptr(cu), tokens, batch, width), (table, lens, cu)


def _rows(t, heads, dim, device, what: str) -> torch.Tensor:
    """t [tokens, heads, dim] with a contiguous last axis (copied if it has none)."""
    if not isinstance(t, torch.Tensor) or t.device != device:
        raise IcxError(-1, f"{what}: expected a tensor on {device}")
    if t.dim() != 3 or t.shape[2] != dim or (heads is not None and t.shape[1] != heads):
        raise IcxError(-1, f"{what}: expected [tokens, {'*' if heads is None else heads}, {dim}], "
                           f"got {list(t.shape)}")
    return t if t.stride(2) == 1 else t.contiguous()


def _new_rows(out, shape, dtype, device, what: str) -> torch.Tensor:
    if (not isinstance(out, torch.Tensor) or out.device != device or out.dtype != dtype
            or out.shape != shape or not out.is_contiguous() or out.data_ptr() % 16):
        raise IcxError(-1, f"{what}: expected a contiguous, 16-byte aligned {_name(dtype)} "
                           f"{list(shape)} on {device}")
    return out


def gpu_kv_cache_append(cache: KvCache, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor,
                        seq_lens: torch.Tensor, cu_tokens: torch.Tensor | None = None,
                        return_values: bool = False):
    """Quantises k and v ([tokens, kv_heads, head_dim], any strides over tokens
    and heads) into the cache.

    With ``return_values`` returns ``(k', v')``, contiguous and of k's type:
    the values the cache now stands for, e.g. to attend over a prompt as later
    steps will see it.  Rows that are not stored (rows outside ``cu_tokens``,
    positions without a page) are undefined there.

    A page that receives tokens belongs to one sequence: where two tokens of a
    call fall on one slot, the slot holds an undefined mixture of both.
    """
    what = "KvCacheAppend"
    k = _rows(k, cache.kv_heads, cache.head_dim, cache.device, f"{what}: k")
    v = _rows(v, cache.kv_heads, cache.head_dim, cache.device, f"{what}: v")
    t = _float_type(k.dtype, f"{what}: k")
    if v.dtype != k.dtype or v.shape != k.shape:
        raise IcxError(-1, f"{what}: v is {_name(v.dtype)} {list(v.shape)}, "
                           f"k {_name(k.dtype)} {list(k.shape)}")
    arg, keep = _where(cache, page_table, seq_lens, cu_tokens, k.shape[0], what)
    values = [torch.empty_like(k, memory_format=torch.contiguous_format) for _ in range(2)] if return_values else (None, None)
    _on(cache.device, _lib.load().icx_kv_cache_append, cache._ref, ctypes.byref(arg),
        k.data_ptr(), v.data_ptr(), t, k.stride(0), k.stride(1), v.stride(0), v.stride(1),
        _ptr(values[0]), _ptr(values[1]))
    return tuple(values) if return_values else None


def gpu_kv_cache_read(cache: KvCache, page_table: torch.Tensor, seq_lens: torch.Tensor,
                      cu_tokens: torch.Tensor | None = None, tokens: int | None = None,
                      dtype: torch.dtype = torch.float32, out=None):
    """Dequantises tokens: returns ``(k, v)``, [tokens, kv_heads, head_dim].

    ``tokens`` is the number of packed rows (cu_tokens' last entry, or more;
    the batch without ``cu_tokens``).  Whole sequences are read with
    ``cu_tokens`` the cumulative ``seq_lens``.  ``out``: a pair of contiguous
    tensors to write; rows that name no stored position are left as they were
    (undefined in fresh tensors).
    """
    what = "KvCacheRead"
    t = _float_type(dtype, f"{what}: dtype")
    if tokens is None:
        if cu_tokens is not None:
            raise IcxError(-1, f"{what}: tokens is needed with cu_tokens")
        tokens = page_table.shape[0]
    if tokens < 0:
        raise IcxError(-1, f"{what}: tokens must not be negative")
    arg, keep = _where(cache, page_table, seq_lens, cu_tokens, tokens, what)
    shape = (tokens, cache.kv_heads, cache.head_dim)
    if out is None:
        k = seq_lens.new_empty(shape, dtype=dtype)
        v = torch.empty_like(k)
    else:
        k, v = (_new_rows(o, shape, dtype, cache.device, f"{what}: out") for o in out)
    _on(cache.device, _lib.load().icx_kv_cache_read, cache._ref, ctypes.byref(arg), t,
        k.data_ptr(), v.data_ptr())
    return k, v


def gpu_kv_cache_attention(cache: KvCache, q: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor,
                           cu_tokens: torch.Tensor | None = None, scale: float | None = None,
                           out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of new tokens over the cache they were appended to.

    q: [tokens, q_heads, head_dim] Float32 / Float16 / BFloat16, any strides
    over tokens and heads; q_heads a multiple of kv_heads, consecutive query
    heads share a K/V head.  Each token attends to the positions 0 .. its own;
    ``scale`` (default 1 / sqrt(head_dim)) multiplies the scores.  Returns q's
    shape and type, contiguous.  A token without any position gives zeros;
    rows outside ``cu_tokens`` are left as they were in ``out`` (undefined in a
    fresh tensor).  Scores, softmax statistics and sums are f32.

    Which kernel runs follows the rows per K/V head and sequence on average
    over the call, ``tokens // batch * (q_heads // kv_heads)``: from 64 on, 16-bit
    queries with group 64 and head_dim up to 128 take those for prompt chunks, all
    else the one for few rows, which reads the cache once per 8 (16) rows.  A call
    that mixes a long chunk with many single tokens is right either way, but two
    calls, one for each, suit them better.

    BFloat16 prompt chunks meet K, V and the weights as f16 (2^-11 of a value),
    K and V in units of the largest of the positions a block of rows reads: values
    2^20 times smaller keep their bits, still smaller ones lose them.  Elsewhere
    the weights times the scales of V carry 22 bits where the scale is near the
    largest met, about 17 at 2^-13 of it and 10 at 2^-20.  Queries of 2^75 and
    more, and scores beyond 2^20, are more than f32 can tell apart: such rows may
    come out as NaN.
    """
    what = "KvCacheAttention"
    q = _rows(q, None, cache.head_dim, cache.device, f"{what}: q")
    t = _float_type(q.dtype, f"{what}: q")
    heads = q.shape[1]
    if heads == 0 or heads % cache.kv_heads:
        raise IcxError(-1, f"{what}: q_heads {heads} is no multiple of kv_heads {cache.kv_heads}")
    scale = 1.0 / math.sqrt(cache.head_dim) if scale is None else float(scale)
    if not math.isfinite(scale):
        raise IcxError(-1, f"{what}: scale must be finite")
    arg, keep = _where(cache, page_table, seq_lens, cu_tokens, q.shape[0], what)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    else:
        out = _new_rows(out, q.shape, q.dtype, cache.device, f"{what}: out")
    L = _lib.load()
    size = L.icx_kv_cache_attention_workspace_bytes(cache._ref, ctypes.byref(arg), heads, t)
    ws = q.new_empty(size, dtype=torch.uint8) if size else None
    _on(cache.device, L.icx_kv_cache_attention, cache._ref, ctypes.byref(arg),
        q.data_ptr(), t, heads, q.stride(0), q.stride(1), scale, out.data_ptr(), _ptr(ws), size)
    return out
