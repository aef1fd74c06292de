"""A paged key/value cache in FP8, the append to it and attention over it, on sm_100a.

The reference stops at the linears (src/python/mambo/kernels/iq3_s_fp8.py:364-399);
this is what stands between its caller's qkv and output projections. The cache
uses the framework's number format: E4M3 values with power-of-two scales, one
for each page (16 to 128 tokens) of a head, keys and values apart. A step is

    q = launch_rotary(q, positions, rope)
    launch_fp8_kv_append(cache, k, v, page_table, lengths, offsets=offsets, rope=rope)
    out = fp8_paged_attention(q, cache, page_table, lengths + new, offsets=offsets)

Page table, lengths and offsets are in device memory and are not read on the
host, so that a step captures into one CUDA graph.
"""

from __future__ import annotations

import functools
from typing import TypedDict

import torch

from .. import _lib, _runtime
from .fp8_block import _DTYPES, _device_guard
from .rotary import RotaryFields, _check_rope, _head_strides

PAGE_TOKENS = (16, 32, 64, 128)
MAX_HEAD_DIM = 128


class Fp8KvCache(TypedDict):
    keys: torch.Tensor  # uint8 [pages, kv_heads, page_tokens, head_dim], E4M3
    values: torch.Tensor
    key_scales: torch.Tensor  # uint8 [pages, kv_heads], UE8M0: 2^(code - 127), codes 63 .. 254, 255: NaN
    value_scales: torch.Tensor


@_runtime.with_stream
def prepare_fp8_kv_cache(pages: int, kv_heads: int, page_tokens: int, head_dim: int, *, device="cuda",
                         stream=None) -> Fp8KvCache:
    """An empty cache: zero codes with the smallest scale."""
    if page_tokens not in PAGE_TOKENS:
        raise ValueError(f"a page has {PAGE_TOKENS} tokens")
    if head_dim < 16 or head_dim % 16 or head_dim > MAX_HEAD_DIM:
        raise ValueError(f"the head size must be a multiple of 16, at most {MAX_HEAD_DIM}")
    if pages < 1 or kv_heads < 1:
        raise ValueError("a cache has pages and heads")
    device = torch.device(device)
    if device.type != "cuda":
        raise ValueError("expected a CUDA device (this build has no CPU path)")
    shape = (pages, kv_heads, page_tokens, head_dim)
    keys, values = (torch.zeros(shape, dtype=torch.uint8, device=device) for _ in range(2))
    _runtime.require_device(keys.device)
    key_scales, value_scales = (torch.full(shape[:2], 63, dtype=torch.uint8, device=device) for _ in range(2))
    return {"keys": keys, "values": values, "key_scales": key_scales, "value_scales": value_scales}


def _cache_view(cache: Fp8KvCache) -> _lib.MamboKvCache:
    try:
        keys, values, ks, vs = cache["keys"], cache["values"], cache["key_scales"], cache["value_scales"]
    except (KeyError, TypeError, IndexError):
        raise TypeError("cache must have keys, values, key_scales and value_scales (prepare_fp8_kv_cache)") from None
    shape, dev = keys.shape, keys.get_device()
    if len(shape) != 4 or values.shape != shape or ks.shape != shape[:2] or vs.shape != shape[:2]:
        raise ValueError("cache must be [pages, kv_heads, page_tokens, head_dim] with scales [pages, kv_heads]")
    u8 = torch.uint8
    if keys.dtype != u8 or values.dtype != u8 or ks.dtype != u8 or vs.dtype != u8:
        raise ValueError("cache codes and scales must be uint8")
    if not (keys.is_contiguous() and values.is_contiguous() and ks.is_contiguous() and vs.is_contiguous()):
        raise ValueError("cache tensors must be contiguous")
    if dev < 0 or values.get_device() != dev or ks.get_device() != dev or vs.get_device() != dev:
        raise ValueError("cache tensors must be on one CUDA device")
    return _lib.MamboKvCache(keys.data_ptr(), values.data_ptr(), ks.data_ptr(), vs.data_ptr(), *shape)


def _sequences(page_table, lengths, offsets, tokens: int, device: int) -> tuple[_lib.MamboKvSequences, tuple]:
    """The C ABI's view of a call's sequences, and the tensors that it points to."""
    table, lengths = _runtime.as_cuda_tensor(page_table), _runtime.as_cuda_tensor(lengths)
    if table.ndim != 2 or table.dtype is not torch.int32 or table.shape[1] < 1 or table.get_device() != device:
        raise ValueError("page_table must be int32 [B, pages of a sequence] on the cache's device")
    batch, columns = table.shape
    if lengths.dtype is not torch.int32 or lengths.shape != (batch,) or lengths.get_device() != device:
        raise ValueError("lengths must be int32 [B] on the cache's device")
    if not lengths.is_contiguous():
        lengths = lengths.contiguous()
    stride, unit = table.stride()
    if (unit != 1 and columns > 1) or (stride < columns and batch > 1):  # also rows that share memory (expanded)
        table = table.contiguous()
        stride = columns
    at = None
    if offsets is not None:
        offsets = _runtime.as_cuda_tensor(offsets)
        if offsets.dtype is not torch.int32 or offsets.shape != (batch + 1,) or offsets.get_device() != device:
            raise ValueError("offsets must be int32 [B+1] on the cache's device")
        if not offsets.is_contiguous():
            offsets = offsets.contiguous()
        at = offsets.data_ptr()
    elif tokens != batch:
        raise ValueError("without offsets there is one token for each sequence")
    return (_lib.MamboKvSequences(table.data_ptr(), stride if batch > 1 else columns, columns, lengths.data_ptr(), at, batch),
            (table, lengths, offsets))


@_runtime.with_stream
def launch_fp8_kv_append(cache: Fp8KvCache, k, v, page_table, lengths, *, offsets=None, rope: RotaryFields | None = None,
                         stream=None) -> None:
    """Appends keys and values [T,H,D] (float32 or bfloat16) to their sequences' pages.

    ``page_table``: int32 [B, pages of a sequence], ``lengths``: int32 [B], the
    tokens that each sequence has in the cache before the call. Tokens
    ``offsets[b]`` .. ``offsets[b+1]-1`` (int32 [B+1]; None: token b) go to the
    positions from ``lengths[b]`` on; with ``rope`` the keys are turned by
    their positions first, in float32.

    A page's scale is the smallest power of two (2^-64 at least) with which its
    new values fit E4M3, or the page's own if that is larger and the page was
    begun by an earlier call; where it grows, the older codes are rounded anew.
    A page of a head that gets NaN or infinity is NaN until it is begun again.
    Tokens without a page (behind the table's end, or an entry outside the
    cache) are dropped. A page that is appended to belongs to one sequence.
    """
    view, dev = _cache_view(cache), cache["keys"].device
    k, v = _runtime.as_cuda_tensor(k), _runtime.as_cuda_tensor(v)
    if k.ndim != 3 or k.dtype not in _DTYPES or k.shape[1] != view.kv_heads or k.shape[2] != view.head_dim:
        raise ValueError("k must be float32 or bfloat16 [T,H,D] with the cache's heads and head size")
    if v.shape != k.shape or v.dtype is not k.dtype or k.get_device() != dev.index or v.get_device() != dev.index:
        raise ValueError("v must have k's shape and type, both on the cache's device")
    tokens = k.shape[0]
    seq, held = _sequences(page_table, lengths, offsets, tokens, dev.index)
    if rope is not None:
        _check_rope(rope, view.head_dim, dev)
    _runtime.require_device(dev)
    if not tokens:
        return
    if k.stride(2) != 1:
        k = k.contiguous()
    if v.stride(2) != 1:
        v = v.contiguous()
    with _device_guard(dev):
        _lib.check(_lib.load().mambo_kv_append(
            view, k.data_ptr(), *_head_strides(k), v.data_ptr(), *_head_strides(v), _DTYPES[k.dtype], tokens, seq,
            None if rope is None else rope["rotary"], _runtime.stream_handle(None, dev)), "launch_fp8_kv_append")


def _rows_aligned(t: torch.Tensor) -> bool:
    """Whether every head of [T,H,D] is 16-byte aligned with unit stride."""
    st, sh, unit = t.stride()
    return unit == 1 and not (st % 8 or sh % 8 or t.data_ptr() % 16)


@functools.lru_cache(maxsize=1024)
def _attention_workspace_bytes(heads: int, kv_heads: int, ragged: bool) -> int:
    return _lib.load().mambo_kv_attention_workspace_bytes(heads, kv_heads, int(ragged))


@_runtime.with_stream
def fp8_paged_attention(q, cache: Fp8KvCache, page_table, lengths, *, offsets=None, window: int = 0,
                        scale: float | None = None, return_lse: bool = False, stream=None,
                        out: torch.Tensor | None = None):
    """Causal attention of queries q [T,Hq,D] (bfloat16) over the cache -> out [T,Hq,D] (bfloat16).

    ``lengths``: int32 [B], the tokens of each sequence in the cache, the
    call's own among them: the n queries of a sequence (``offsets`` as in
    ``launch_fp8_kv_append``; None: one each) stand at its last n positions.
    A query sees the positions up to its own, with ``window`` the last
    ``window`` of them. Query head h reads key head h // (Hq / H). ``scale``
    (1/sqrt(D)) multiplies the scores. A query that sees nothing has zeros.
    Positions of a page outside the cache do not exist. ``out`` may be q; tokens
    that no sequence has keep what it holds (without it, and in the logarithms,
    anything).

    Scores and sums are float32. A position's weight times its page's value
    scale is rounded by 2^-11 of itself or 2^-24 of the row's largest such
    product, whichever is more: 8 bits are left of one that is 2^-16 of the
    largest, and nothing behind 2^-24. So where a query sees pages whose value
    scales are further apart than that, dimensions in which those of the large
    scale hold zeros lose what the others hold. The logarithms are right with
    scales up to 2^100 apart.

    ``return_lse``: also the float32 [T,Hq] logarithms of the sums of the
    exponentials (minus infinity where a query sees nothing), with which
    results over parts of a context are joined.
    """
    view, dev = _cache_view(cache), cache["keys"].device
    q = _runtime.as_cuda_tensor(q)
    if q.ndim != 3 or q.dtype is not torch.bfloat16 or q.shape[2] != view.head_dim or q.get_device() != dev.index:
        raise ValueError("q must be bfloat16 [T,Hq,D] with the cache's head size on its device")
    tokens, heads, dim = q.shape
    if heads < 1 or heads % view.kv_heads:
        raise ValueError("the query heads must be a multiple of the cache's heads")
    if window < 0:
        raise ValueError("window must not be negative")
    seq, held = _sequences(page_table, lengths, offsets, tokens, dev.index)
    _runtime.require_device(dev)
    if not _rows_aligned(q):
        q = q.clone(memory_format=torch.contiguous_format)
    given = out
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif tuple(out.shape) != (tokens, heads, dim) or out.dtype != torch.bfloat16 or out.device != dev:
        raise ValueError("out must be bfloat16 of q's shape on its device")
    elif not _rows_aligned(out):
        out = out.clone(memory_format=torch.contiguous_format)  # rows that no sequence covers keep what they hold
    lse = torch.empty((tokens, heads), dtype=torch.float32, device=dev) if return_lse else None
    if tokens:
        need = _attention_workspace_bytes(heads, view.kv_heads, offsets is not None)
        with _device_guard(dev):
            with _runtime.workspace(dev, None, need) as ws:
                _lib.check(_lib.load().mambo_kv_attention(
                    q.data_ptr(), *_head_strides(q), tokens, heads, view, seq, window,
                    dim ** -0.5 if scale is None else scale, out.data_ptr(), *_head_strides(out),
                    None if lse is None else lse.data_ptr(), heads, 1, ws.ptr, ws.size, ws.stream),
                    "fp8_paged_attention")
    if given is not None and given is not out:
        given.copy_(out)
        out = given
    return (out, lse) if return_lse else out
