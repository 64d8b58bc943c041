"""torch.library registration: torch.ops.cdna4_sage.attention (and attention_masked, rope, cache_write, cache_read,
cache_attention, attention_train, relative_bias), traceable by torch.compile.

Same schema as the reference's rdna4_sage::attention (src/rdna4_sage/ops.py:7-17); the rdna4_sage package of this
repo registers that name too, for callers that use it directly.
"""
from typing import List, Optional, Tuple

import torch

from . import _attention


def _impl(q, k, v, layout, sm_scale, is_causal):
    return _attention.attention(q, k, v, layout, sm_scale if sm_scale > 0 else None, is_causal)


def _fake(q, k, v, layout, sm_scale, is_causal):
    B = q.shape[0]
    H, Sq = (q.shape[1], q.shape[2]) if layout == "HND" else (q.shape[2], q.shape[1])
    return q.new_empty((B, Sq, H, q.shape[3]))


@torch.library.custom_op("cdna4_sage::attention", mutates_args=())
def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, layout: str, sm_scale: float, is_causal: bool) -> torch.Tensor:
    """Output [batch, q_len, heads, head_dim], contiguous, whatever the input layout; a non-positive sm_scale stands
    for the default 1 / sqrt(head_dim)."""
    return _impl(q, k, v, layout, sm_scale, is_causal)


attention.register_fake(_fake)


@torch.library.custom_op("cdna4_sage::attention_masked", mutates_args=())
def attention_masked(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, attn_mask: torch.Tensor, layout: str,
                     sm_scale: float, is_causal: bool) -> torch.Tensor:
    """attention with an attn_mask as torch SDPA takes it (bool True = attend, or additive of q's dtype; broadcastable
    to [B, H, q_len, kv_len]); no counterpart in the reference, which sends masked calls to SDPA.  Returns
    (B, Sq, H, D) contiguous."""
    return _attention.attention(q, k, v, layout, sm_scale if sm_scale > 0 else None, is_causal, attn_mask=attn_mask)


@attention_masked.register_fake
def _fake_masked(q, k, v, attn_mask, layout, sm_scale, is_causal):
    return _fake(q, k, v, layout, sm_scale, is_causal)


# ---- rotary positions and the quantized key / value cache (no counterparts in the reference) --------------------------
# The implementations live in modules that import this one, so they are looked up at the call.

@torch.library.custom_op("cdna4_sage::rope", mutates_args=())
def rope(x: torch.Tensor, positions: Optional[torch.Tensor], freqs: torch.Tensor, layout: str, interleaved: bool,
         factor: float, inverse: bool) -> torch.Tensor:
    """x with the first 2 * freqs.numel() channels of every head turned (back, where inverse) by positions * freqs."""
    from . import _rope

    return _rope.rope_launch(x, None, positions, freqs, layout, interleaved, factor, inverse)[0]


@rope.register_fake
def _fake_rope(x, positions, freqs, layout, interleaved, factor, inverse):
    from . import _rope

    return _rope.out_like(x)


@torch.library.custom_op("cdna4_sage::rope_qk", mutates_args=())
def rope_qk(q: torch.Tensor, k: torch.Tensor, positions: Optional[torch.Tensor], freqs: torch.Tensor, layout: str,
            interleaved: bool, factor: float, inverse: bool) -> Tuple[torch.Tensor, torch.Tensor]:
    """rope of q and k in one launch."""
    from . import _rope

    return _rope.rope_launch(q, k, positions, freqs, layout, interleaved, factor, inverse)


@rope_qk.register_fake
def _fake_rope_qk(q, k, positions, freqs, layout, interleaved, factor, inverse):
    from . import _rope

    return _rope.out_like(q), _rope.out_like(k)


def _rope_setup(ctx, inputs, output):
    *_, positions, freqs, layout, interleaved, factor, inverse = inputs
    ctx.save_for_backward(positions, freqs)
    ctx.how = layout, interleaved, factor, not inverse


def _rope_backward(ctx, dx):
    return rope(dx, *ctx.saved_tensors, *ctx.how), None, None, None, None, None, None


def _rope_qk_backward(ctx, dq, dk):
    return (*rope_qk(dq, dk, *ctx.saved_tensors, *ctx.how), None, None, None, None, None, None)


rope.register_autograd(_rope_backward, setup_context=_rope_setup)
rope_qk.register_autograd(_rope_qk_backward, setup_context=_rope_setup)


@torch.library.custom_op("cdna4_sage::cache_write", mutates_args=("k8", "v8", "k_scale", "v_scale"))
def cache_write(k8: torch.Tensor, v8: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor, k: torch.Tensor,
                v: torch.Tensor, slots: torch.Tensor, layout: str) -> None:
    """k and v quantized into the rows `slots` of the cache (k8, v8, k_scale, v_scale)."""
    from . import _cache

    _cache.write_launch(_cache.KVCache(k8, v8, k_scale, v_scale), k, v, slots, layout)


@cache_write.register_fake
def _fake_cache_write(k8, v8, k_scale, v_scale, k, v, slots, layout):
    return None


@torch.library.custom_op("cdna4_sage::cache_read", mutates_args=())
def cache_read(k8: torch.Tensor, v8: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor, slots: torch.Tensor,
               dtype: torch.dtype, layout: str) -> Tuple[torch.Tensor, torch.Tensor]:
    """The rows `slots` of the cache in dtype."""
    from . import _cache

    return _cache.read_launch(_cache.KVCache(k8, v8, k_scale, v_scale), slots, dtype, layout)


@cache_read.register_fake
def _fake_cache_read(k8, v8, k_scale, v_scale, slots, dtype, layout):
    out = [k8.new_empty((*slots.shape, k8.shape[1], k8.shape[3]), dtype=dtype) for _ in range(2)]
    return tuple(t.transpose(1, 2) for t in out) if slots.dim() == 2 and layout == "HND" else tuple(out)


@torch.library.custom_op("cdna4_sage::cache_attention", mutates_args=())
def cache_attention(q: torch.Tensor, k8: torch.Tensor, v8: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                    block_table: torch.Tensor, lengths: torch.Tensor, tree_mask: Optional[torch.Tensor], layout: str,
                    sm_scale: float, is_causal: bool) -> torch.Tensor:
    """Attention of the new tokens over the cache, [batch, tokens, heads, head_dim]; a sm_scale of 0 stands for
    1 / sqrt(head_dim)."""
    from . import _cache

    out, _ = _cache.attention_launch(q, _cache.KVCache(k8, v8, k_scale, v_scale), block_table, lengths, layout, sm_scale,
                                     is_causal, tree_mask, False)
    return out.transpose(1, 2) if layout == "HND" else out


@cache_attention.register_fake
def _fake_cache_attention(q, k8, v8, k_scale, v_scale, block_table, lengths, tree_mask, layout, sm_scale, is_causal):
    return _fake(q, None, None, layout, sm_scale, is_causal)


@torch.library.custom_op("cdna4_sage::cache_attention_lse", mutates_args=())
def cache_attention_lse(q: torch.Tensor, k8: torch.Tensor, v8: torch.Tensor, k_scale: torch.Tensor,
                        v_scale: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor,
                        tree_mask: Optional[torch.Tensor], layout: str, sm_scale: float,
                        is_causal: bool) -> Tuple[torch.Tensor, torch.Tensor]:
    """cache_attention and the logsumexp of its rows, fp32 [batch, heads, tokens]."""
    from . import _cache

    out, lse = _cache.attention_launch(q, _cache.KVCache(k8, v8, k_scale, v_scale), block_table, lengths, layout, sm_scale,
                                       is_causal, tree_mask, True)
    return out.transpose(1, 2) if layout == "HND" else out, lse


@cache_attention_lse.register_fake
def _fake_cache_attention_lse(q, k8, v8, k_scale, v_scale, block_table, lengths, tree_mask, layout, sm_scale, is_causal):
    out = _fake(q, None, None, layout, sm_scale, is_causal)
    return out, q.new_empty((out.shape[0], out.shape[2], out.shape[1]), dtype=torch.float32)


# ---- attention for training and the relative position bias (no counterparts in the reference) --------------------------------

def _mask_axes(attn_mask, q, k, layout):
    """Whether the mask differs along batch, heads and rows; empty without one."""
    if attn_mask is None:
        return []
    a = 2 if layout == "HND" else 1
    shape = (q.shape[0], q.shape[3 - a], q.shape[a], k.shape[a])
    s = attn_mask.expand(shape).stride()
    return [int(n > 1 and x != 0) for n, x in zip(shape[:3], s)]


def _state_bytes(packed, B, H, Sq, Skv, D, axes, reach, keep):
    """The bytes of the state, as sage_train_workspace has them, of sizes that may be symbols."""
    def up(*n):
        return sum((x + 255) // 256 * 256 for x in n)

    n = 0
    if packed:      # bounds, tiles of queries and of keys
        n += up(16, 8 * (Sq // 128 + B), 8 * (Skv // 128 + B))
    if axes:        # a mask's bits, what its blocks show, that both ways, the keys seen (twice)
        bh = (B if axes[0] else 1) * (H if axes[1] else 1)
        rows, blocks = ((Sq + 63) // 64 * 64, (Sq + 63) // 64) if axes[2] else (1, 1)
        chunks = (Skv + 63) // 64
        wide, high = (chunks + 63) // 64, (blocks + 63) // 64
        n += up(bh * rows * chunks * 8, bh * blocks * chunks, bh * blocks * wide * 8, bh * chunks * high * 8)
        if keep:
            n += up(bh * blocks * chunks * 8, bh * chunks * high * 8)
    if reach:       # the bias by distance
        n += up(4 * H * (2 * reach + 1))
    if keep:        # what the rounding of out took away
        n += up(2 * (1 if packed else B) * H * Sq * D)
    return n


@torch.library.custom_op("cdna4_sage::attention_train", mutates_args=())
def attention_train(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, attn_mask: Optional[torch.Tensor],
                    table: Optional[torch.Tensor], cu_q: Optional[torch.Tensor], cu_k: Optional[torch.Tensor], layout: str,
                    sm_scale: float, is_causal: bool, bidirectional: bool, max_distance: int,
                    keep: bool) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Attention on 16-bit inputs: (out, lse, the state that the backward pass reads, where `keep` says that one comes); packed
    sequences where cu_q is given."""
    from . import _train

    return _train.forward_launch(q, k, v, attn_mask, table, cu_q, cu_k, layout, sm_scale, is_causal, bidirectional,
                                 max_distance, keep)[:3]


@attention_train.register_fake
def _fake_attention_train(q, k, v, attn_mask, table, cu_q, cu_k, layout, sm_scale, is_causal, bidirectional, max_distance, keep):
    from . import _capi, _rope

    packed = cu_q is not None
    if packed:
        out, (Sq, H, D), Skv, B = q.new_empty(q.shape), q.shape, k.shape[0], cu_q.shape[0] - 1
        lse = q.new_empty((H, Sq), dtype=torch.float32)
    else:
        out, (B, H, Sq, D) = _rope.out_like(q), q.shape if layout == "HND" else [q.shape[i] for i in (0, 2, 1, 3)]
        Skv = k.shape[2 if layout == "HND" else 1]
        lse = q.new_empty((B, H, Sq), dtype=torch.float32)
    state = 0
    if q.numel() != 0 and k.numel() != 0:
        reach = 0 if table is None else _capi.bias_borders(int(table.shape[0]), bidirectional, max_distance)[-1]
        state = _state_bytes(packed, B, H, Sq, Skv, D, _mask_axes(attn_mask, q, k, layout), reach, keep)
    return out, lse, q.new_empty((state,), dtype=torch.uint8)


@torch.library.custom_op("cdna4_sage::attention_train_backward", mutates_args=())
def attention_train_backward(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor,
                             lse: torch.Tensor, state: torch.Tensor, table: Optional[torch.Tensor],
                             cu_q: Optional[torch.Tensor], cu_k: Optional[torch.Tensor], layout: str, sm_scale: float,
                             is_causal: bool, bidirectional: bool, max_distance: int,
                             mask_axes: List[int]) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dq, dk, dv, dtable), the last one empty without a table; mask_axes: whether the mask had a batch, head and row axis."""
    from . import _train

    plan = _train.backward_plan(dout, q, k, v, out, lse, state, layout, table, cu_q, cu_k, bidirectional, max_distance,
                                tuple(mask_axes) or None)
    dq, dk, dv, dt = _train.backward_launch(dout, q, k, v, out, lse, state, table, cu_q, cu_k, layout, sm_scale, is_causal,
                                            plan, (True, True, table is not None))
    return dq, dk, dv, q.new_empty(0) if dt is None else dt


@attention_train_backward.register_fake
def _fake_attention_train_backward(dout, q, k, v, out, lse, state, table, cu_q, cu_k, layout, sm_scale, is_causal,
                                   bidirectional, max_distance, mask_axes):
    from . import _rope

    like = _rope.out_like if cu_q is None else (lambda t: t.new_empty(t.shape))
    return like(q), like(k), like(v), q.new_empty(0) if table is None else table.new_empty(table.shape)


def _train_setup(ctx, inputs, output):
    q, k, v, attn_mask, table, cu_q, cu_k, *ctx.how, keep = inputs
    if not keep:
        raise RuntimeError("cdna4_sage::attention_train: keep=True is needed for a backward pass")
    ctx.axes = _mask_axes(attn_mask, q, k, ctx.how[0])
    ctx.save_for_backward(q, k, v, *output, table, cu_q, cu_k)
    ctx.mark_non_differentiable(output[1], output[2])


def _train_backward(ctx, dout, *_):
    saved = ctx.saved_tensors   # (once: a checkpoint's unpacking may not be asked for twice)
    dq, dk, dv, dt = attention_train_backward(dout, *saved, *ctx.how, ctx.axes)
    return (dq, dk, dv, None, dt if saved[6] is not None else None) + (None,) * 8


attention_train.register_autograd(_train_backward, setup_context=_train_setup)


@torch.library.custom_op("cdna4_sage::relative_bias", mutates_args=())
def relative_bias(table: torch.Tensor, q_len: int, kv_len: int, bidirectional: bool, max_distance: int, dtype: torch.dtype,
                  offset: int, offset_at: Optional[torch.Tensor]) -> torch.Tensor:
    """The bias [heads, q_len, kv_len] of a table [buckets, heads] by relative position."""
    from . import _train

    return _train.bias_launch(table, q_len, kv_len, bidirectional, max_distance, dtype, offset, offset_at)


@relative_bias.register_fake
def _fake_relative_bias(table, q_len, kv_len, bidirectional, max_distance, dtype, offset, offset_at):
    return table.new_empty((table.shape[1], q_len, kv_len), dtype=dtype)


@torch.library.custom_op("cdna4_sage::relative_bias_backward", mutates_args=())
def relative_bias_backward(dbias: torch.Tensor, buckets: int, dtype: torch.dtype, bidirectional: bool, max_distance: int,
                           offset: int, offset_at: Optional[torch.Tensor]) -> torch.Tensor:
    """The gradient [buckets, heads] of relative_bias' table."""
    from . import _train

    return _train.bias_grad_launch(dbias, buckets, dtype, bidirectional, max_distance, offset, offset_at)


@relative_bias_backward.register_fake
def _fake_relative_bias_backward(dbias, buckets, dtype, bidirectional, max_distance, offset, offset_at):
    return dbias.new_empty((buckets, dbias.shape[0]), dtype=dtype)


def _bias_setup(ctx, inputs, output):
    table, _, _, bidirectional, max_distance, _, offset, offset_at = inputs
    ctx.how = table.shape[0], table.dtype, bidirectional, max_distance, offset
    ctx.save_for_backward(offset_at)


def _bias_backward(ctx, dbias):
    return (relative_bias_backward(dbias, *ctx.how, *ctx.saved_tensors),) + (None,) * 7


relative_bias.register_autograd(_bias_backward, setup_context=_bias_setup)
