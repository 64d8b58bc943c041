"""The quantized, paged key / value cache and the attention of new tokens over it, on the gfx950 kernels (no counterpart in
the reference, which quantizes all keys and values anew in every call, src/rdna4_sage/_attention.py:115-133).

    cache = cdna4_sage.new_cache(pages, 16, kv_heads, head_dim)               # int8, or dtype=torch.float8_e4m3fn
    slots = cdna4_sage.cache_slots(block_table, lengths, T, 16)               # lengths with the T new tokens counted
    cdna4_sage.cache_write(cache, k, v, slots)
    out = cdna4_sage.cache_attention(q, cache, block_table, lengths)          # q [B, H, T, D]

Nothing here reads device memory back, allocates outside torch's caching allocator or keeps state between calls, so
every call can be captured into a graph.
"""
from __future__ import annotations

import functools
from typing import NamedTuple

import torch

from . import _capi, ops
from ._attention import (_I32_MAX, ARCHS, DTYPES, HEAD_DIMS, Unsupported, _bsh, _packed, _plain_eager, gpu_arch,
                         refuse_tangents)
from ._rope import rope

_F32_NORMAL, _F32_MAX = torch.finfo(torch.float32).smallest_normal, torch.finfo(torch.float32).max
CACHE_DTYPES = {torch.int8: _capi.CACHE_INT8, torch.float8_e4m3fn: _capi.CACHE_E4M3}


class KVCache(NamedTuple):
    """Codes [pages, kv_heads, page_size, head_dim] (int8 or float8_e4m3fn) and scales [pages, kv_heads, page_size]
    (float32) of the keys and the values, contiguous: a key is code * scale.  Slot s is row s % page_size of page
    s // page_size.  page_size is a power of two from 16 to 1024.  float32 holds what the kernels derive from cached
    values of magnitude up to 2^100; E4M3 codes are finite (cache_write keeps a NaN in the scale)."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor


def new_cache(pages, page_size, kv_heads, head_dim, dtype=torch.int8, device=None):
    """An empty KVCache (all zeros)."""
    shape = (int(pages), int(kv_heads), int(page_size))
    _check_page(shape[2])
    if dtype not in CACHE_DTYPES:
        raise Unsupported(f"cache dtype {dtype} (int8 or float8_e4m3fn)")
    if head_dim not in HEAD_DIMS:
        raise Unsupported(f"head_dim {head_dim} (supported {HEAD_DIMS})")
    if shape[0] <= 0 or shape[1] <= 0:
        raise Unsupported("a cache needs pages and kv heads")
    device = torch.device("cuda" if device is None else device)
    codes = [torch.zeros(shape + (int(head_dim),), dtype=torch.int8, device=device).view(dtype) for _ in range(2)]
    return KVCache(*codes, *(torch.zeros(shape, dtype=torch.float32, device=device) for _ in range(2)))


def _check_page(page_size):
    if not 16 <= page_size <= 1024 or page_size & (page_size - 1):
        raise Unsupported(f"page_size {page_size} (a power of two from 16 to 1024)")


def check_cache(cache, gpu=None):
    """(pages, kv_heads, page_size, head_dim) of a usable cache (on GPU `gpu`); raises Unsupported with the reason."""
    k, v, ks, vs = cache
    shape = k.shape
    pages, heads, page_size, D = shape if len(shape) == 4 else (0, 0, 0, 0)
    rows = (pages, heads, page_size)
    if len(shape) != 4 or v.shape != shape or ks.shape != rows or vs.shape != rows:
        raise Unsupported("cache codes [pages, kv_heads, page_size, head_dim] and scales [pages, kv_heads, page_size] required")
    dtype = k.dtype
    if dtype not in CACHE_DTYPES or v.dtype != dtype:
        raise Unsupported(f"cache dtype {dtype}/{v.dtype} (int8 or float8_e4m3fn)")
    if ks.dtype != torch.float32 or vs.dtype != torch.float32:
        raise Unsupported("cache scales must be float32")
    _check_page(page_size)
    if D not in HEAD_DIMS:
        raise Unsupported(f"head_dim {D} (supported {HEAD_DIMS})")
    if pages == 0 or heads == 0 or pages > _I32_MAX:
        raise Unsupported("a cache needs pages and kv heads")
    if not (k.is_contiguous() and v.is_contiguous() and ks.is_contiguous() and vs.is_contiguous()):
        raise Unsupported("cache tensors must be contiguous")
    at = k.get_device()
    if at < 0 or not at == v.get_device() == ks.get_device() == vs.get_device() or (gpu is not None and gpu != at):
        raise Unsupported("tensors must be on one ROCm GPU")
    if gpu_arch(at) not in ARCHS:
        raise Unsupported("not a CDNA4 GPU")
    return pages, heads, page_size, D


def _addresses(cache):
    """Addresses of the codes and scales, k's first, as the C entries take them."""
    k, v, ks, vs = cache
    at = k.data_ptr(), ks.data_ptr(), v.data_ptr(), vs.data_ptr()
    if (at[0] | at[1] | at[2] | at[3]) % 16:
        raise Unsupported("cache tensors must start on 16-byte boundaries")
    return at


def cache_slots(block_table, lengths, count, page_size):
    """Slots of the last `count` of lengths[b] tokens of every sequence, int64 [B, count], for cache_write and cache_read;
    -1 where there is no such token or its page is missing (an entry below 0 or a column past the table)."""
    _check_page(page_size)
    pos = lengths.to(torch.int64)[:, None] - count + torch.arange(count, device=lengths.device)[None, :]
    column = torch.div(pos, page_size, rounding_mode="floor")
    if block_table.shape[1] == 0:
        return torch.full_like(pos, -1)
    page = block_table.to(torch.int64).gather(1, column.clamp(0, block_table.shape[1] - 1))
    there = (pos >= 0) & (column < block_table.shape[1]) & (page >= 0)
    return torch.where(there, page * page_size + pos % page_size, -1)


def _check_slots(slots, gpu, shape):
    if slots.dtype != torch.int64 and slots.dtype != torch.int32:
        raise Unsupported(f"slots {slots.dtype} (int32 or int64)")
    if slots.get_device() != gpu:
        raise Unsupported("tensors must be on one ROCm GPU")
    if slots.shape != shape:
        raise Unsupported(f"slots of shape {tuple(slots.shape)} for tokens {tuple(shape)}")
    return slots.contiguous()


def _rows_args(t, layout):
    """A packed [tokens, heads, D] or a 4D tensor as the kernels address it: tensor, (b, s, h) strides."""
    if t.dim() == 4:
        return _bsh(t, layout)
    t, s = _packed(t)
    return t, (0, *s)


def write_launch(cache, k, v, slots, layout):
    if layout != "HND" and layout != "NHD":
        raise Unsupported(f"layout {layout!r}")
    shape = k.shape
    if len(shape) not in (3, 4) or v.shape != shape:
        raise Unsupported("k and v of one shape, 4D or packed [tokens, kv_heads, head_dim], required")
    if k.dtype not in DTYPES or v.dtype != k.dtype:
        raise Unsupported(f"dtype {k.dtype}/{v.dtype} (fp16 or bf16 required)")
    gpu = k.get_device()
    if v.get_device() != gpu:
        raise Unsupported("tensors must be on one ROCm GPU")
    pages, Hkv, page_size, D = check_cache(cache, gpu)
    if len(shape) == 3:
        (S, h, d), B = shape, 1
        tokens = shape[:1]
    else:
        (B, h, S, d) = shape if layout == "HND" else (shape[0], shape[2], shape[1], shape[3])
        tokens = (B, S)
    if h != Hkv or d != D:
        raise Unsupported(f"{h} heads of {d} channels for a cache of {Hkv} heads of {D}")
    slots = _check_slots(slots, gpu, tokens)
    n = k.numel()
    if n == 0:
        return
    if n > _I32_MAX:
        raise Unsupported("tensor too large for 32-bit indexing")
    k, sk = _rows_args(k, layout)
    v, sv = _rows_args(v, layout)
    _capi.call_on(gpu, "sage_cache_write", k.data_ptr(), *sk, v.data_ptr(), *sv, B, S, DTYPES[k.dtype],
                  slots.data_ptr(), slots.dtype == torch.int64, *_addresses(cache), pages, page_size, Hkv, D,
                  CACHE_DTYPES[cache.k.dtype])


def read_launch(cache, slots, dtype, layout):
    if layout != "HND" and layout != "NHD":
        raise Unsupported(f"layout {layout!r}")
    if dtype not in DTYPES:
        raise Unsupported(f"dtype {dtype} (fp16 or bf16 required)")
    pages, Hkv, page_size, D = check_cache(cache)
    shape = slots.shape
    if len(shape) not in (1, 2):
        raise Unsupported("slots [tokens] or [B, tokens] required")
    gpu = cache.k.get_device()
    slots = _check_slots(slots, gpu, shape)
    k = cache.k.new_empty((*shape, Hkv, D), dtype=dtype)
    v = torch.empty_like(k)
    n = k.numel()
    if n:
        if n > _I32_MAX:
            raise Unsupported("tensor too large for 32-bit indexing")
        # (both outputs are contiguous: the batch needs no stride of its own)
        st = (0, Hkv * D, D)
        _capi.call_on(gpu, "sage_cache_read", k.data_ptr(), *st, v.data_ptr(), *st, 1, slots.numel(), DTYPES[dtype],
                      slots.data_ptr(), slots.dtype == torch.int64, *_addresses(cache), pages, page_size, Hkv, D,
                      CACHE_DTYPES[cache.k.dtype])
    if len(shape) == 2 and layout == "HND":
        return k.transpose(1, 2), v.transpose(1, 2)
    return k, v


def cache_write(cache, k, v, slots, tensor_layout="HND"):
    """Quantizes rows of k and v into the cache: per token and kv head one scale, max |x| / 127 (int8) or / 448 (E4M3), and
    the nearest codes of x / scale, ties to even; a row with an infinity or a NaN is kept as NaN (by its scale).
    k / v: [B, kv_heads, tokens, head_dim] ("HND") or [B, tokens, kv_heads, head_dim] ("NHD") with slots [B, tokens], or packed
    [tokens, kv_heads, head_dim] with slots [tokens]; slots int32 or int64.  Tokens whose slot is outside the cache (-1) are
    left out; two tokens of a call may not share a slot (that slot's row then holds parts of both).  Codes have no
    derivative: gradients and tangents of k and v end here."""
    if _plain_eager(k, v, slots, *cache, grad=True):   # (codes have no derivative: autograd sees nothing of the write)
        write_launch(cache, k, v, slots, tensor_layout)
    else:
        ops.cache_write(cache.k, cache.v, cache.k_scale, cache.v_scale, k, v, slots, tensor_layout)


def cache_read(cache, slots, dtype=torch.bfloat16, tensor_layout="HND"):
    """(k, v) of the slots as code * scale, rounded to dtype: packed [tokens, kv_heads, head_dim] for slots [tokens] (as
    sageattn_varlen takes them), 4D in tensor_layout for slots [B, tokens].  Slots outside the cache (-1) give zeros.  No derivative in the scales: a
    backward pass and tangents raise."""
    refuse_tangents("cache_read", *cache)
    if _plain_eager(slots, *cache):
        return read_launch(cache, slots, dtype, tensor_layout)
    return ops.cache_read(*cache, slots, dtype, tensor_layout)


@functools.lru_cache(maxsize=4096)
def _workspace(gpu, B, H, Hkv, T, D, page_size, max_pages):
    """Workspace bytes of a call of these sizes on GPU `gpu`."""
    if max_pages * page_size > 2**30 or B * -(-max_pages * page_size // 128) > 2**30:
        raise Unsupported(f"block_table of {max_pages} pages of {page_size} keys for batch {B} (at most 2^30 keys per sequence, 2^37 "
                          "in all)")
    with torch.cuda.device(gpu):
        return _capi.cache_attn_workspace(B, H, Hkv, T, D, page_size, max_pages)


def attention_launch(q, cache, block_table, lengths, layout, sm_scale, is_causal, tree_mask, return_lse):
    """Output in q's layout and dtype, contiguous as (B, T, H, D), and the logsumexp [B, H, T] or None."""
    if layout != "HND" and layout != "NHD":
        raise Unsupported(f"layout {layout!r}")
    shape = q.shape
    if len(shape) != 4:
        raise Unsupported("4D q required")
    if q.dtype not in DTYPES:
        raise Unsupported(f"dtype {q.dtype} (fp16 or bf16 required)")
    gpu = q.get_device()
    pages, Hkv, page_size, D = check_cache(cache, gpu)
    (B, H, T, d) = shape if layout == "HND" else (shape[0], shape[2], shape[1], shape[3])
    if d != D or H % Hkv:
        raise Unsupported(f"{H} heads of {d} channels for a cache of {Hkv} heads of {D}")
    if block_table.dim() != 2 or block_table.shape[0] != B or lengths.shape != (B,):
        raise Unsupported("block_table [B, max_pages] and lengths [B] required")
    if block_table.get_device() != gpu or lengths.get_device() != gpu:
        raise Unsupported("tensors must be on one ROCm GPU")
    if block_table.dtype != torch.int32:
        block_table = _as_int32(block_table)
    if lengths.dtype != torch.int32:
        lengths = _as_int32(lengths)
    mask, ms = None, (0, 0, 0)
    if tree_mask is not None:
        if not is_causal:
            raise Unsupported("tree_mask stands in the place of the causal rule: is_causal=False has none")
        if tree_mask.dtype != torch.bool or tree_mask.get_device() != gpu:
            raise Unsupported("tree_mask must be a bool tensor on q's device")
        if tuple(tree_mask.shape) not in ((T, T), (1, T, T), (B, T, T)):
            raise Unsupported(f"tree_mask of shape {tuple(tree_mask.shape)} for batch {B} and {T} new tokens")
        ms = tree_mask.stride()
        if len(ms) == 2 or tree_mask.shape[0] == 1:
            ms = (0, *ms[-2:])
        if T == 1:   # (strides that are never taken)
            ms = (ms[0], 0, 0)
        elif max(ms[1], ms[2]) * (T - 1) >= 2**30:
            raise Unsupported("a tree mask whose rows or columns reach over 2^30 bytes")
        mask = tree_mask.data_ptr()
    # (one allocation call each: the host's time is most of a small call's)
    out = q.new_empty_strided(shape, (T * H * D, D, H * D, 1) if layout == "HND" else (T * H * D, H * D, D, 1))
    lse = q.new_empty((B, H, T), dtype=torch.float32) if return_lse else None
    max_pages, n = block_table.shape[1], q.numel()
    if n == 0 or max_pages == 0:   # no query rows, or no keys
        return out.zero_(), None if lse is None else lse.fill_(float("-inf"))
    if n > _I32_MAX:
        raise Unsupported("tensor too large for 32-bit indexing")
    ws_bytes = _workspace(gpu, B, H, Hkv, T, D, page_size, max_pages)
    q, sq = _bsh(q, layout)
    ts = block_table.stride()
    if ts[1] != 1 and max_pages > 1:
        block_table = block_table.contiguous()
        ts = block_table.stride()
    lengths = lengths.contiguous()
    ws = q.new_empty(ws_bytes // 2) if ws_bytes else None   # (q's elements are of 2 bytes, the workspace's of 4)
    _capi.call_on(gpu, "sage_cache_attn", q.data_ptr(), *sq, out.data_ptr(), T * H * D, H * D, D,
                  None if lse is None else lse.data_ptr(), *_addresses(cache), block_table.data_ptr(), ts[0], lengths.data_ptr(),
                  mask, *ms, B, H, Hkv, T, D, DTYPES[q.dtype], CACHE_DTYPES[cache.k.dtype], pages, page_size, max_pages,
                  bool(is_causal), sm_scale, None if ws is None else ws.data_ptr(), ws_bytes)
    return out, lse


def _as_int32(t):
    """Lengths and page numbers of another integer type as the kernels read them (beyond 32 bits: at its ends, so that
    a number out of range stays out of range)."""
    if t.dtype != torch.int64:
        raise Unsupported("block_table and lengths must be int32 or int64")
    return t.clamp(-2**31, _I32_MAX).to(torch.int32)


def cache_attention(q, cache, block_table, lengths, tensor_layout="HND", sm_scale=None, is_causal=True, tree_mask=None,
                    return_lse=False):
    """Attention of the T new tokens of every sequence over the cache: q [B, H, T, D] ("HND") or [B, T, H, D] ("NHD"), H a
    multiple of the cache's kv heads.  lengths [B]: the cached keys of each sequence, the T new tokens' (already
    written, the last T of them) counted; block_table [B, max_pages]: key j is row j % page_size of page
    block_table[b, j // page_size], and a page outside the cache (-1) hides its keys.  A query sees every key before the new
    ones and, of those, its own and the earlier ones (is_causal), all (is_causal=False), or those its row of tree_mask
    shows: bool [T, T] or [B, T, T], True at (i, j) where new token i sees new token j (a tree of drafted tokens: its
    ancestors and itself).  A query that sees no key gives 0 (lengths[b] = 0, say), one that sees some and holds an infinity
    or a NaN gives NaN.  Returns the output in q's layout and dtype; return_lse adds the fp32 natural logsumexp [B, H, T], -inf
    where no key is seen.  sm_scale: a positive normal number of float32; None or a non-positive one stands for 1 / sqrt(D).
    Launch and workspace are planned for the table's width, the lengths being on the device: where they are known to stay
    below a bound, block_table[:, :pages] says so and copies nothing (too wide a table costs short prompts up to 1.4 times
    their time).  There is no derivative: a backward pass and inputs with forward-mode tangents raise.  Raises Unsupported
    for what the kernel does not take."""
    sm = float(sm_scale) if sm_scale is not None and sm_scale > 0 else 0.0
    if sm and not _F32_NORMAL <= sm <= _F32_MAX:
        raise Unsupported(f"sm_scale {sm} (float32's normal numbers)")
    ts = (q, *cache, block_table, lengths)
    refuse_tangents("cache_attention", *ts)
    if _plain_eager(*ts) and (tree_mask is None or type(tree_mask) is torch.Tensor):
        out, lse = attention_launch(q, cache, block_table, lengths, tensor_layout, sm, is_causal, tree_mask, return_lse)
    elif return_lse:
        out, lse = ops.cache_attention_lse(q, *cache, block_table, lengths, tree_mask, tensor_layout, sm, bool(is_causal))
        out = out.transpose(1, 2) if tensor_layout == "HND" else out
    else:
        out = ops.cache_attention(q, *cache, block_table, lengths, tree_mask, tensor_layout, sm, bool(is_causal))
        out = out.transpose(1, 2) if tensor_layout == "HND" else out
    return (out, lse) if return_lse else out


def cache_step(q, k, v, cache, slots, block_table, lengths, positions=None, freqs=None, tensor_layout="HND",
               interleaved=False, factor=1.0, sm_scale=None, tree_mask=None):
    """One decoding step of an attention layer: turns q and k by their positions (rope; where freqs is None they are
    taken as they are), writes k and v into the cache (cache_write) and attends over it (cache_attention).  lengths
    count the new tokens; positions: int [T] or [B, T], by default the tokens' places in their sequence (those of drafted
    tokens follow from their depth in the tree)."""
    if freqs is not None:
        if positions is None:
            T = q.shape[2] if tensor_layout == "HND" else q.shape[1]
            positions = lengths[:, None] - T + torch.arange(T, device=lengths.device, dtype=lengths.dtype)
        q, k = rope(q, k, positions, freqs, tensor_layout, interleaved, factor)
    cache_write(cache, k, v, slots, tensor_layout)
    return cache_attention(q, cache, block_table, lengths, tensor_layout, sm_scale, True, tree_mask)
