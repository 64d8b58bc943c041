"""torch.library registration: torch.ops.cdna4_sage.attention (and attention_masked, rope, cache_write, cache_read,
cache_attention), traceable by torch.compile.

Same schema as the reference's rdna4_sage::attention (src/rdna4_sage/ops.py:7-17); the rdna4_sage package of this
repo registers that name too, for callers that use it directly.
"""
from typing import Optional, Tuple

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
