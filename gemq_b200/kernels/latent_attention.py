"""Latent attention (DeepSeek-V2's) over a paged cache.

The reference has no counterpart: it patches the MoE blocks of the host model and leaves its attention alone
(gemq/inference/patch.py:119-124); its static cache allows the two head sizes of that attention
(gemq/inference/kv_cache.py:10-76).

A token is cached as one row of ``rank + 64`` numbers that all heads share: the normalised latent vector and the rotated part
of the key.  A cache is ``[pages, page_size, rank + 64]``, fp16 or bf16, any stride between pages; ``page_size`` is 16, 32 or a
multiple of 64, ``rank`` 128, 256, 384 or 512.  Lengths, page tables and slots are device tensors that no call reads on the host,
so every call can be captured in a CUDA graph.  Entries out of range are reported in the device's error word
(``gemq_b200.kernels.latent_error``) and never used as an index.  That word is made by the first call of this package on a device, which
belongs outside a capture.  Serving only: the operators have no gradients.

The attention operators form scores, maxima, sums and results in 32 bits.  Each weight is rounded once to the type of the cache for the product
with the values (off by half a step of it at most, fp16 2^-11, bf16 2^-8, relative to the weight), their sum is not; results are
rounded once more.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple

import torch
from torch import Tensor

from .. import _capi
from ._ops import library_op
from ._runtime import host_latent_error_word, latent_error_word, require, require_cuda, stream_ptr

ROPE, NOPE, VALUE = 64, 128, 128
_HALF = (torch.float16, torch.bfloat16)


class _on:
    """The device of the tensors is the current one inside: the launches go to its streams."""

    def __init__(self, dev: torch.device):
        self.guard = None if dev.index == torch.cuda.current_device() else torch.cuda.device(dev)

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()

    def __exit__(self, *a):
        if self.guard is not None:
            self.guard.__exit__(*a)


def _native(name: str):
    """The call in native code (csrc/host.cpp); None where it does not take the arguments, which the checks here then name."""
    def fast(x, *rest):
        p = host_latent_error_word(x) if isinstance(x, Tensor) else None
        return None if p is None else getattr(_capi.host, name)(p, x, *rest)
    return fast


def latent_error(device=None) -> int:
    """The code of what the latent operators found out of range on the device since the last call of this, 0 for nothing:
    41 page, 42 length or offsets, 43 slot, 44 a wait inside a kernel; of several the latest.  Waits for all streams of the device (not
    while one of them is captured); the code is taken and cleared at once, so what calls that run meanwhile report is left for the next call."""
    dev = torch.device("cuda") if device is None else torch.device(device)
    require(dev.type == "cuda", f"the latent operators run on CUDA devices, not on {dev}")
    if dev.index is None:
        dev = torch.device(dev.type, torch.cuda.current_device())
    torch.cuda.synchronize(dev)
    code = torch.empty(1, dtype=torch.int32, device=dev)
    with _on(dev):
        _capi.check("gemq_latent_take_error", _capi.lib.gemq_latent_take_error(latent_error_word(dev).data_ptr(), code.data_ptr(), stream_ptr(dev)))
    return int(code.item())


def _strides(name: str, t: Tensor) -> list:
    """The strides of all but the last dimension, 0 where there is one of it (such a stride may be anything)."""
    s = [0 if n == 1 else s for n, s in zip(t.shape, t.stride())][:-1]
    require(t.data_ptr() % 16 == 0 and t.stride(-1) == 1 and all(v % 8 == 0 for v in s),
            f"{name} must be contiguous in its last dimension, its rows on 16-byte boundaries")
    return s


def _ints(name: str, t: Tensor, dtype: torch.dtype, shape) -> None:
    require(t.dtype == dtype and tuple(t.shape) == tuple(shape) and t.is_contiguous(), f"{name} must be contiguous {dtype} {list(shape)}")


def _check_cache(cache: Tensor, dtype: torch.dtype):
    """-> rank, elements from page to page."""
    require(cache.dim() == 3 and cache.dtype == dtype and dtype in _HALF, "cache must be [pages, page_size, rank + 64], fp16 or bf16 like the rest")
    pages, page, width = cache.shape
    rank = width - ROPE
    require(rank in (128, 256, 384, 512), f"latent rank must be 128, 256, 384 or 512, not {rank}")
    require(page in (16, 32) or (page > 0 and page % 64 == 0), f"page size must be 16, 32 or a multiple of 64, not {page}")
    require(pages > 0 and pages * page < 2 ** 31, "a cache has 1 to 2^31 - 1 rows")
    require(cache.stride(1) == width and (pages == 1 or cache.stride(0) >= page * width), "the rows of a page must lie one behind the other, pages apart")
    return rank, _strides("cache", cache)[0]


# ---- rows into the cache --------------------------------------------------------------------------
def _fake_append(kv, q_rope, norm_weight, eps, inv_freq, positions, slots, cache, rope_scale=1.0):
    return q_rope.new_empty(q_rope.shape), kv.new_empty(kv.shape)


@library_op("latent_append", _fake_append, _native("latent_append"), mutates=("cache",))
def latent_append(kv: Tensor, q_rope: Tensor, norm_weight: Tensor, eps: float, inv_freq: Tensor, positions: Tensor, slots: Tensor,
                  cache: Tensor, rope_scale: float = 1.0) -> Tuple[Tensor, Tensor]:
    """``kv [T, rank + 64]`` (what the compressing projection gives) -> cached rows, ``q_rope [T, H, 64]`` -> rotated queries.

    A row is ``RMSNorm(kv[:, :rank]) * norm_weight`` (rounded once, behind the weight) and ``kv[:, rank:]`` rotated at
    ``positions [T]``: pairs of neighbouring numbers, angle ``position * inv_freq [32]`` formed in 64 bits, cosine and sine times
    ``rope_scale``.  Row t is stored at row ``slots[t]`` of the cache seen as ``[pages * page_size, rank + 64]``; -1 is a padded
    token, which is stored nowhere.  Slots stored to must be distinct.  Returns the rotated queries ``[T, H, 64]`` and
    the rows ``[T, rank + 64]``, padded ones included."""
    dev = require_cuda(kv, q_rope, norm_weight, inv_freq, positions, slots, cache)
    rank, page_stride = _check_cache(cache, kv.dtype)
    require(kv.dim() == 2 and kv.shape[1] == rank + ROPE, f"kv must be [tokens, {rank + ROPE}]")
    T = kv.shape[0]
    require(q_rope.dim() == 3 and q_rope.shape[0] == T and q_rope.shape[2] == ROPE and q_rope.dtype == kv.dtype,
            "q_rope must be [tokens, heads, 64] of kv's type")
    require(tuple(norm_weight.shape) == (rank,) and norm_weight.dtype == kv.dtype, "norm_weight must be [rank] of kv's type")
    _ints("inv_freq", inv_freq, torch.float32, (ROPE // 2,))
    _ints("positions", positions, torch.int64, (T,))
    _ints("slots", slots, torch.int64, (T,))
    H = q_rope.shape[1]
    rows = torch.empty((T, rank + ROPE), dtype=kv.dtype, device=dev)
    q_out = torch.empty((T, H, ROPE), dtype=kv.dtype, device=dev)
    if T == 0:
        return q_out, rows
    kv_stride, = _strides("kv", kv)
    _strides("norm_weight", norm_weight)
    q_strides = _strides("q_rope", q_rope) if H else (0, 0)
    with _on(dev):
        _capi.check("gemq_latent_append", _capi.lib.gemq_latent_append(
            kv.data_ptr(), kv_stride, q_rope.data_ptr() if H else None, *q_strides, norm_weight.data_ptr(), eps, inv_freq.data_ptr(),
            rope_scale, positions.data_ptr(), slots.data_ptr(), cache.data_ptr(), page_stride, cache.shape[0], cache.shape[1], rows.data_ptr(),
            q_out.data_ptr() if H else None, T, H, rank, int(kv.dtype == torch.bfloat16), latent_error_word(dev).data_ptr(), stream_ptr(dev)))
    return q_out, rows


# ---- decoded tokens, absorbed form ------------------------------------------------------------------
def _decode(q_latent, q_rope, cache, table, lens, scale, prefix_table=None, prefix_lens=None, starts=None):
    shared = () if starts is None else (prefix_table, prefix_lens, starts)
    dev = require_cuda(q_latent, q_rope, cache, table, lens, *shared)
    rank, page_stride = _check_cache(cache, q_latent.dtype)
    require(q_latent.dim() == 4 and q_latent.shape[3] == rank, f"q_latent must be [batch, steps, heads, {rank}]")
    B, S, H, _ = q_latent.shape
    require(tuple(q_rope.shape) == (B, S, H, ROPE) and q_rope.dtype == q_latent.dtype, f"q_rope must be {[B, S, H, ROPE]} of q_latent's type")
    require(S > 0 and H > 0, "q_latent must have a step and a head")
    require(table.dim() == 2, "table must be [batch, pages of a sequence]")
    _ints("table", table, torch.int32, (B, table.shape[1]))
    _ints("lens", lens, torch.int32, (B,))
    out = torch.empty((B, S, H, rank), dtype=q_latent.dtype, device=dev)
    lse = torch.empty((B, S, H), dtype=torch.float32, device=dev)
    A = _capi.LatentDecode()
    if starts is not None:
        require(prefix_table.dim() == 2 and prefix_table.shape[0] > 0, "prefix_table must be [groups, pages of a prefix]")
        G = prefix_table.shape[0]
        _ints("prefix_table", prefix_table, torch.int32, (G, prefix_table.shape[1]))
        _ints("prefix_lens", prefix_lens, torch.int32, (G,))
        _ints("starts", starts, torch.int32, (G + 1,))
        A.prefix_table, A.prefix_pitch = prefix_table.data_ptr() or cache.data_ptr(), prefix_table.shape[1]
        A.prefix_lens = prefix_lens.data_ptr()
        A.starts, A.groups = starts.data_ptr(), G
    if B == 0:
        return out, lse
    A.q_latent, A.q_latent_stride[:] = q_latent.data_ptr(), _strides("q_latent", q_latent)
    A.q_rope, A.q_rope_stride[:] = q_rope.data_ptr(), _strides("q_rope", q_rope)
    A.cache, A.page_stride, A.n_pages, A.page_size = cache.data_ptr(), page_stride, cache.shape[0], cache.shape[1]
    A.table, A.table_pitch, A.lens = table.data_ptr() or cache.data_ptr(), table.shape[1], lens.data_ptr()
    A.batch, A.steps, A.heads, A.rank, A.scale, A.is_bf16 = B, S, H, rank, scale, int(q_latent.dtype == torch.bfloat16)
    A.out, A.lse, A.err = out.data_ptr(), lse.data_ptr(), latent_error_word(dev).data_ptr()
    with _on(dev):
        n = _capi.lib.gemq_latent_decode_scratch_bytes(C.byref(A))
        scratch = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
        _capi.check("gemq_latent_decode", _capi.lib.gemq_latent_decode(C.byref(A), scratch.data_ptr() if n else None, n, stream_ptr(dev)))
    return out, lse


def _fake_decode(q_latent, q_rope, cache, *rest):
    return q_latent.new_empty(q_latent.shape), q_latent.new_empty(q_latent.shape[:3], dtype=torch.float32)


@library_op("latent_decode", _fake_decode, _native("latent_decode"))
def latent_decode(q_latent: Tensor, q_rope: Tensor, cache: Tensor, table: Tensor, lens: Tensor, scale: float) -> Tuple[Tensor, Tensor]:
    """Attention of the last ``S`` tokens of every sequence over its cached rows, in the latent space.

    ``q_latent [B, S, H, rank]`` are the queries times the matrix that would expand the keys, ``q_rope [B, S, H, 64]`` the rotated
    part, any strides between their last dimensions.  Sequence b has ``lens[b]`` rows (the S new ones stored already) on the
    pages ``table[b]`` (int32, entries behind its last page are not read); its query i sees the positions before
    ``lens[b] - (S - 1 - i)``.  Returns the weighted latent vectors ``[B, S, H, rank]`` and the logarithm of the sum of
    exponentials ``[B, S, H]`` (fp32, natural); a query that sees nothing gives 0 and -inf.  What lies in a row behind what a query
    sees has no influence on it; one that sees a row with an infinity or a NaN may be NaN as a whole."""
    return _decode(q_latent, q_rope, cache, table, lens, scale)


def _native_shared(*a):
    if len(a) != 9:
        return None
    q_latent, q_rope, cache, table, lens, prefix_table, prefix_lens, starts, scale = a
    return _native("latent_decode")(q_latent, q_rope, cache, table, lens, scale, prefix_table, prefix_lens, starts)


@library_op("latent_decode_shared", _fake_decode, _native_shared)
def latent_decode_shared(q_latent: Tensor, q_rope: Tensor, cache: Tensor, table: Tensor, lens: Tensor, prefix_table: Tensor,
                         prefix_lens: Tensor, starts: Tensor, scale: float) -> Tuple[Tensor, Tensor]:
    """``latent_decode`` for a batch in which sequences ``starts[g] .. starts[g + 1] - 1`` begin with the same ``prefix_lens[g]``
    rows, the pages ``prefix_table[g]``; ``table`` and ``lens`` hold what each sequence has behind them.  The result is that of
    the joined sequences; a prefix is read and multiplied once for all its sequences.  ``starts [groups + 1]`` rises
    from 0 to the batch; where it does not, that is reported and all results are NaN."""
    return _decode(q_latent, q_rope, cache, table, lens, scale, prefix_table, prefix_lens, starts)


# ---- prompts, expanded form -------------------------------------------------------------------------
def _fake_prefill(q_nope, q_rope, kv, k_rope, cu_q, cu_k, scale, causal=True):
    return q_nope.new_empty(q_nope.shape), q_nope.new_empty(q_nope.shape[:2], dtype=torch.float32)


@library_op("latent_prefill", _fake_prefill, _native("latent_prefill"))
def latent_prefill(q_nope: Tensor, q_rope: Tensor, kv: Tensor, k_rope: Tensor, cu_q: Tensor, cu_k: Tensor, scale: float,
                   causal: bool = True) -> Tuple[Tensor, Tensor]:
    """Attention of prompts over expanded keys and values, sequences one behind the other.

    ``q_nope [Tq, H, 128]`` and ``q_rope [Tq, H, 64]`` are the two parts of the queries, ``kv [Tk, H, 256]`` the unrotated
    key part and the value as the expanding projection gives them, ``k_rope [Tk, 64]`` the rotated key part of all heads; any
    strides between the last dimensions.  Sequence b has the query rows ``cu_q[b] .. cu_q[b + 1] - 1`` and the key rows
    ``cu_k[b] .. cu_k[b + 1] - 1`` (int32, rising from 0); the last query sees the last key, one before it one key less, or
    all see all without ``causal``.  Returns ``[Tq, H, 128]`` and the logarithm of the sum of exponentials ``[Tq, H]``; rows that see
    nothing, and those behind the last sequence, are 0 and -inf."""
    dev = require_cuda(q_nope, q_rope, kv, k_rope, cu_q, cu_k)
    require(q_nope.dim() == 3 and q_nope.shape[2] == NOPE and q_nope.dtype in _HALF, "q_nope must be [rows, heads, 128], fp16 or bf16")
    Tq, H, _ = q_nope.shape
    require(tuple(q_rope.shape) == (Tq, H, ROPE), f"q_rope must be {[Tq, H, ROPE]}")
    require(kv.dim() == 3 and tuple(kv.shape[1:]) == (H, NOPE + VALUE), f"kv must be [rows, {H}, 256]")
    Tk = kv.shape[0]
    require(tuple(k_rope.shape) == (Tk, ROPE), f"k_rope must be {[Tk, ROPE]}")
    require(q_rope.dtype == kv.dtype == k_rope.dtype == q_nope.dtype, "queries, keys and values must have one type")
    require(cu_q.dim() == 1 and cu_q.shape[0] >= 1, "cu_q must be [sequences + 1]")
    _ints("cu_q", cu_q, torch.int32, cu_q.shape)
    _ints("cu_k", cu_k, torch.int32, cu_q.shape)
    require(H > 0, "q_nope must have a head")
    out = torch.empty((Tq, H, VALUE), dtype=q_nope.dtype, device=dev)
    lse = torch.empty((Tq, H), dtype=torch.float32, device=dev)
    if Tq == 0:
        return out, lse
    # a tiled copy has no stride of 0: what is expanded is laid out
    q_nope, q_rope, kv, k_rope = (t.contiguous() if any(n > 1 and s == 0 for n, s in zip(t.shape, t.stride())) else t
                                  for t in (q_nope, q_rope, kv, k_rope))
    A = _capi.LatentPrefill()
    A.q_nope, A.q_nope_stride[:] = q_nope.data_ptr(), _strides("q_nope", q_nope)
    A.q_rope, A.q_rope_stride[:] = q_rope.data_ptr(), _strides("q_rope", q_rope)
    if Tk:
        A.kv, A.kv_stride[:] = kv.data_ptr(), _strides("kv", kv)
        A.k_rope, A.k_rope_stride = k_rope.data_ptr(), _strides("k_rope", k_rope)[0]
    A.cu_q, A.cu_k, A.batch, A.q_rows, A.k_rows = cu_q.data_ptr(), cu_k.data_ptr(), cu_q.shape[0] - 1, Tq, Tk
    A.heads, A.causal, A.scale, A.is_bf16 = H, int(causal), scale, int(q_nope.dtype == torch.bfloat16)
    A.out, A.lse, A.err = out.data_ptr(), lse.data_ptr(), latent_error_word(dev).data_ptr()
    with _on(dev):
        _capi.check("gemq_latent_prefill", _capi.lib.gemq_latent_prefill(C.byref(A), stream_ptr(dev)))
    return out, lse


# ---- pages ------------------------------------------------------------------------------------------
@library_op("copy_pages", lambda cache, src, dst: None, mutates=("cache",))
def copy_pages(cache: Tensor, src: Tensor, dst: Tensor) -> None:
    """Page ``dst[i]`` becomes a copy of page ``src[i]`` (int64), in one launch for all layers: ``cache`` is ``[pages, ..]`` or, with
    four dimensions and more, ``[layers, pages, ..]``; the pages themselves contiguous, of any type, a multiple of 16 bytes.
    The destinations must be distinct, and no page may be both a source and a destination, but for ``src[i] == dst[i]``, which
    is left alone.  Ids outside the cache are reported and skipped."""
    if _native("copy_pages")(cache, src, dst):
        return
    dev = require_cuda(cache, src, dst)
    require(cache.dim() >= 2, "cache must be [pages, ..] or [layers, pages, ..]")
    layers = cache.shape[0] if cache.dim() >= 4 else 1
    page = cache[0, 0] if cache.dim() >= 4 and cache.numel() else cache[0] if cache.numel() else cache
    require(src.dim() == 1, "src must be [copies]")
    _ints("src", src, torch.int64, src.shape)
    _ints("dst", dst, torch.int64, src.shape)
    if src.numel() == 0:
        return
    require(cache.numel() > 0, "an empty cache has no pages to copy")
    require(page.is_contiguous(), "the pages must be contiguous")
    size, lead = cache.element_size(), cache.stride()
    page_stride, layer_stride = (lead[1], lead[0]) if cache.dim() >= 4 else (lead[0], 0)
    nbytes = page.numel() * size
    require(cache.data_ptr() % 16 == 0 and nbytes % 16 == 0 and page_stride * size % 16 == 0 and layer_stride * size % 16 == 0,
            "pages must lie on 16-byte boundaries and be a multiple of 16 bytes")
    with _on(dev):
        _capi.check("gemq_copy_pages", _capi.lib.gemq_copy_pages(
            cache.data_ptr(), layer_stride * size, page_stride * size, layers, cache.shape[-page.dim() - 1], nbytes, src.data_ptr(), dst.data_ptr(),
            src.numel(), latent_error_word(dev).data_ptr(), stream_ptr(dev)))
