"""Attention on 16-bit inputs with its backward pass, and a learned relative position bias by buckets, on the gfx950 kernels (no
counterparts in the reference: its attention has no derivative, and its callers bring masks of their own).

The 8-bit attention of this package is for inference; a model is trained, or its text scored, with attention_train.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _capi, ops
from ._attention import (_ALIGN, ARCHS, DTYPES, HEAD_DIMS, Unsupported, _bsh, _packed, _plain_eager, gpu_arch,
                         refuse_tangents)
from ._rope import out_like

TABLE_DTYPES = {**DTYPES, torch.float32: _capi.DTYPE_F32}
BIAS_BUCKETS = 256
LEAST_SCALE = 2.0 ** -100   # with a backward pass


# ---- checks ---------------------------------------------------------------------------------------------------------------

def _bias(table, heads, bidirectional, max_distance, gpu):
    """(buckets, two-sided, max_distance) of a table of learned values [buckets, heads]."""
    if table.dim() != 2 or table.dtype not in TABLE_DTYPES:
        raise Unsupported(f"a bias table [buckets, heads] of fp32, bf16 or fp16 is required (got {tuple(table.shape)}, {table.dtype})")
    if heads is not None and table.shape[1] != heads:
        raise Unsupported(f"bias table of {table.shape[1]} heads for {heads}")
    if table.get_device() != gpu:
        raise Unsupported("tensors must be on one ROCm GPU")
    n = table.shape[0]
    if n < 2 or n > BIAS_BUCKETS or (bidirectional and (n % 2 or n < 4)):
        raise Unsupported(f"{n} buckets (2 to {BIAS_BUCKETS}; bidirectional an even number from 4)")
    near = (n // 2 if bidirectional else n) // 2
    if not near < max_distance <= 0x3FFFFFFF:
        raise Unsupported(f"max_distance {max_distance} (more than {near}, half of one side's buckets)")
    return n, bool(bidirectional), int(max_distance)


def _check(q, k, v, layout, packed):
    """(B, H, Hkv, Sq, Skv, D, GPU index); B is 0 where packed."""
    qs, ks = q.shape, k.shape
    if packed:
        if len(qs) != 3 or len(ks) != 3 or v.dim() != 3:
            raise Unsupported("3D tensors required")
        (Sq, H, D), (Skv, Hkv, _), B = qs, ks, 0
    else:
        if layout != "HND" and layout != "NHD":
            raise Unsupported(f"layout {layout!r}")
        if len(qs) != 4 or len(ks) != 4 or v.dim() != 4:
            raise Unsupported("4D tensors required")
        if layout == "HND":
            (B, H, Sq, D), (Bk, Hkv, Skv, _) = qs, ks
        else:
            (B, Sq, H, D), (Bk, Skv, Hkv, _) = qs, ks
        if Bk != B:
            raise Unsupported("q and k must have the same batch")
    if q.dtype not in DTYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise Unsupported(f"dtype {q.dtype}/{k.dtype}/{v.dtype} (fp16 or bf16 required)")
    if ks != v.shape or ks[-1] != D:
        raise Unsupported("k and v of one shape, and of q's head_dim, required")
    if D not in HEAD_DIMS:
        raise Unsupported(f"head_dim {D} (supported {HEAD_DIMS})")
    if H and (Hkv == 0 or H % Hkv):
        raise Unsupported(f"heads {H} not a multiple of kv heads {Hkv}")
    gpu = q.get_device()
    if gpu < 0 or k.get_device() != gpu or v.get_device() != gpu:
        raise Unsupported("tensors must be on one ROCm GPU")
    if gpu_arch(gpu) not in ARCHS:
        raise Unsupported("not a CDNA4 GPU")
    return B, H, Hkv, Sq, Skv, D, gpu


def _mask(attn_mask, shape):
    """The mask expanded to [B, H, Sq, Skv], with its (batch, head, row, key) strides, 0 where it is the same along an axis."""
    B, H, _, Sq, Skv, _, gpu = shape
    if not isinstance(attn_mask, torch.Tensor) or attn_mask.dtype != torch.bool:
        raise Unsupported("attn_mask must be a boolean tensor (learned biases: bias_table)")
    if attn_mask.get_device() != gpu:
        raise Unsupported("attn_mask must be on the device of q")
    if attn_mask.dim() > 4:
        raise Unsupported(f"attn_mask with {attn_mask.dim()} dims")
    try:
        m = attn_mask.expand(B, H, Sq, Skv)
    except RuntimeError as e:
        raise Unsupported(f"attn_mask of shape {tuple(attn_mask.shape)} does not broadcast to {(B, H, Sq, Skv)}") from e
    s = m.stride()
    return m, (s[0] if B > 1 else 0, s[1] if H > 1 else 0, s[2] if Sq > 1 else 0, s[3])


def _scale(sm_scale):
    """0 stands for 1 / sqrt(head_dim): None, non-positive values and NaN, as everywhere in this package."""
    if sm_scale is None or not sm_scale > 0:
        return 0.0
    sm = float(sm_scale)
    if not 2.0 ** -126 <= sm <= 2.0 ** 127:
        raise Unsupported(f"sm_scale {sm_scale} (2^-126 to 2^127)")
    return sm


def _check_offsets(cu_q, cu_k, gpu):
    """(For callers of the op: attention_train_varlen makes them so.)"""
    for c in (cu_q, cu_k):
        if c is None or c.dtype != torch.int32 or c.dim() != 1 or c.get_device() != gpu or not c.is_contiguous():
            raise Unsupported("cu_q and cu_k: contiguous int32 offsets on the GPU of q")
    if cu_q.shape != cu_k.shape or cu_q.numel() < 2:
        raise Unsupported("cu_q and cu_k must be of one length batch + 1 >= 2")


# ---- launches -------------------------------------------------------------------------------------------------------------

def _strides(t, layout, packed):
    """t as the kernels load it, and its (batch, token, head) strides."""
    if packed:
        t, s = _packed(t)
        return t, (0, *s)
    return _bsh(t, layout)


def _table_args(table, bias):
    if bias is None:
        return None, 0, 0, 0, 0, 0, None
    n, two, far = bias
    return table.data_ptr(), TABLE_DTYPES[table.dtype], *table.stride(), n, int(two), _capi.bias_borders(n, two, far)


def _sizes(shape, bias, axes, cu_q, keep):
    """(state bytes, workspace bytes, batch); raises Unsupported for a bias that reaches too far for the kernels."""
    B, H, Hkv, Sq, Skv, D, _ = shape
    if cu_q is not None:
        B = cu_q.shape[0] - 1
    try:
        return (*_capi.train_workspace(cu_q is not None, B, H, Hkv, Sq, Skv, D, axes, bias, keep), B)
    except _capi.SageError as e:
        raise Unsupported(str(e)) from e


def forward_launch(q, k, v, attn_mask, table, cu_q, cu_k, layout, sm_scale, causal, bidirectional, max_distance, keep):
    """(out, lse, state, what the kernels loaded of q, k and v, the call's plan for the backward pass); keep: one comes."""
    packed = cu_q is not None
    if keep and 0.0 < sm_scale < LEAST_SCALE:
        raise Unsupported(f"sm_scale {sm_scale} (where inputs require gradients at least 2^-100)")
    shape = _check(q, k, v, layout, packed)
    B, H, Hkv, Sq, Skv, D, gpu = shape
    if packed or cu_k is not None:
        if attn_mask is not None:
            raise Unsupported("packed sequences take no attn_mask")
        _check_offsets(cu_q, cu_k, gpu)
    bias = None if table is None else _bias(table, H, bidirectional, max_distance, gpu)
    mask, ms, axes = None, (0, 0, 0, 0), None
    if attn_mask is not None:
        mask, ms = _mask(attn_mask, shape)
        axes = (int(ms[0] != 0), int(ms[1] != 0), int(ms[2] != 0))
    out = torch.empty((Sq, H, D), dtype=q.dtype, device=q.device) if packed else out_like(q)
    lse = torch.empty((H, Sq) if packed else (B, H, Sq), dtype=torch.float32, device=q.device)
    if q.numel() == 0 or k.numel() == 0:
        out.zero_()
        lse.fill_(float("-inf"))
        return out, lse, torch.empty(0, dtype=torch.uint8, device=q.device), (q, k, v), (shape, bias, axes, 0, 0, 0)
    state_bytes, ws_bytes, nb = _sizes(shape, bias, axes, cu_q, keep)
    state = torch.empty(state_bytes, dtype=torch.uint8, device=q.device)
    q, sq = _strides(q, layout, packed)
    k, sk = _strides(k, layout, packed)
    v, sv = _strides(v, layout, packed)
    so = _strides(out, layout, packed)[1]
    _capi.call_on(gpu, "sage_train_fwd", q.data_ptr(), *sq, k.data_ptr(), *sk, v.data_ptr(), *sv, out.data_ptr(), *so,
                  lse.data_ptr(), nb, H, Hkv, Sq, Skv, D, DTYPES[q.dtype], causal, sm_scale,
                  None if cu_q is None else cu_q.data_ptr(), None if cu_k is None else cu_k.data_ptr(),
                  None if mask is None else mask.data_ptr(), *ms, *_table_args(table, bias), keep,
                  state.data_ptr() if state_bytes else None, state_bytes)
    return out, lse, state, (q, k, v), (shape, bias, axes, state_bytes, ws_bytes, nb)


def backward_launch(dout, q, k, v, out, lse, state, table, cu_q, cu_k, layout, sm_scale, causal, plan, need):
    """(dq, dk, dv, dtable); need: of q, of k or v, of the table.  table: any of the shape and type."""
    packed = cu_q is not None
    (B, H, Hkv, Sq, Skv, D, gpu), bias, axes, state_bytes, ws_bytes, nb = plan
    want_q, want_kv, want_table = need
    want_q = want_q or want_table   # (the table's gradient comes from the kernel of dq)
    like = (lambda t: torch.empty(t.shape, dtype=t.dtype, device=t.device)) if packed else out_like
    dq = like(q) if want_q else None
    dk, dv = (like(k), like(v)) if want_kv else (None, None)
    dtable = torch.empty(table.shape, dtype=table.dtype, device=table.device) if want_table else None
    if q.numel() == 0 or k.numel() == 0:
        for t in (dq, dk, dv, dtable):
            if t is not None:
                t.zero_()
        return dq, dk, dv, dtable
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device)
    args, keep = [], []
    for t in (dout, q, k, v, out):
        t, s = _strides(t, layout, packed)
        keep.append(t)
        args += (t.data_ptr(), *s)
    args.append(lse.data_ptr())
    for t in (dq, dk, dv):
        args += (None, 0, 0, 0) if t is None else (t.data_ptr(), *_strides(t, layout, packed)[1])
    if bias is None:
        ta = (None, 0, 0, 0, 0, 0, None)
    elif want_table:
        ta = _table_args(dtable, bias)
    else:
        ta = (None, _capi.DTYPE_F32, 0, 0, *bias[:2], _capi.bias_borders(*bias))
    _capi.call_on(gpu, "sage_train_bwd", *args, nb, H, Hkv, Sq, Skv, D, DTYPES[q.dtype], causal, sm_scale,
                  None if cu_q is None else cu_q.data_ptr(), None if cu_k is None else cu_k.data_ptr(),
                  axes is not None, *(axes or (0, 0, 0)), *ta, state.data_ptr() if state_bytes else None,
                  state_bytes, ws.data_ptr(), ws_bytes)
    return dq, dk, dv, dtable


def backward_plan(dout, q, k, v, out, lse, state, layout, table, cu_q, cu_k, bidirectional, max_distance, axes):
    """forward_launch's plan, from the same tensors, which are checked (they may come from a caller of the op)."""
    packed = cu_q is not None
    shape = _check(q, k, v, layout, packed)
    if packed or cu_k is not None:
        _check_offsets(cu_q, cu_k, shape[6])
    for t in (dout, out):
        if t.shape != q.shape or t.dtype != q.dtype or t.get_device() != shape[6]:
            raise Unsupported("dout and out must be like q")
    rows = (shape[1], shape[3]) if packed else (shape[0], shape[1], shape[3])
    if lse.shape != rows or lse.dtype != torch.float32 or lse.get_device() != shape[6] or not lse.is_contiguous():
        raise Unsupported(f"lse must be fp32 {rows}, contiguous, on the GPU of q")
    if axes is not None and len(axes) != 3:
        raise Unsupported("mask_axes: none, or one for each of batch, heads and rows")
    bias = None if table is None else _bias(table, shape[1], bidirectional, max_distance, shape[6])
    if q.numel() == 0 or k.numel() == 0:
        return shape, bias, axes, 0, 0, 0
    sizes = _sizes(shape, bias, axes, cu_q, True)
    if state.dtype != torch.uint8 or state.numel() < sizes[0] or state.get_device() != shape[6] or not state.is_contiguous():
        raise Unsupported(f"state: the {sizes[0]} bytes of attention_train with keep")
    return (shape, bias, axes, *sizes)


class _Train(torch.autograd.Function):
    """forward_launch with its backward pass, for eager calls."""

    @staticmethod
    def forward(ctx, q, k, v, table, attn_mask, cu_q, cu_k, *how):
        out, lse, state, used, ctx.plan = forward_launch(q, k, v, attn_mask, table, cu_q, cu_k, *how, True)
        ctx.save_for_backward(*used, out, lse, state, table, cu_q, cu_k)
        ctx.how = how[:3]
        ctx.mark_non_differentiable(lse)
        ctx.set_materialize_grads(False)
        return out, lse

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, _):
        if dout is None:
            return (None,) * 12
        nq, nk, nv, nt = ctx.needs_input_grad[:4]
        dq, dk, dv, dt = backward_launch(dout, *ctx.saved_tensors, *ctx.how, ctx.plan, (nq, nk or nv, nt))
        return dq if nq else None, dk if nk else None, dv if nv else None, dt, *(None,) * 8


def _attention(q, k, v, table, attn_mask, cu_q, cu_k, layout, sm_scale, causal, bidirectional, max_distance, return_lse):
    ts = [t for t in (q, k, v, table) if t is not None]
    how = (layout, _scale(sm_scale), bool(causal), bool(bidirectional), int(max_distance))
    recording = torch.is_grad_enabled() and any(t.requires_grad for t in ts)
    if _plain_eager(*ts, grad=True):
        if recording:
            out, lse = _Train.apply(q, k, v, table, attn_mask, cu_q, cu_k, *how)
        else:
            out, lse = forward_launch(q, k, v, attn_mask, table, cu_q, cu_k, *how, False)[:2]
    else:
        refuse_tangents("attention_train", *ts)
        out, lse, _ = ops.attention_train(q, k, v, attn_mask, table, cu_q, cu_k, *how, recording)
    return (out, lse) if return_lse else out


def attention_train(q, k, v, tensor_layout="HND", sm_scale=None, is_causal=False, attn_mask=None, bias_table=None,
                    bidirectional=True, max_distance=128, return_lse=False):
    """Attention on 16-bit inputs, differentiable in q, k, v and bias_table: softmax(q k^T * sm_scale + bias) v with scores,
    statistics and sums in float32, the weights (and in the backward pass the scores' gradients) rounded to the inputs' type
    where they enter a product.  q: [B, H, q_len, D] for "HND", [B, q_len, H, D] for "NHD", k / v alike with kv heads of
    which H is a multiple; bf16 or fp16, head dims 64, 96, 128, 256.  sm_scale: None for D ** -0.5, at most 2^127 and at least
    2^-100 (2^-126 where nothing requires a gradient).  Returns out like q, or (out, lse) with the rows'
    logsumexp, fp32 [B, H, q_len], which has no gradient.

    is_causal: query i sees the keys up to i + kv_len - q_len (bottom-right), any lengths.  attn_mask: boolean (True =
    attend), broadcastable to [B, H, q_len, kv_len].  bias_table: learned values [buckets, H] (fp32, bf16 or fp16), added by the
    relative position as relative_bias does, without a [H, q_len, kv_len] tensor; its last bucket has to begin at a distance of
    at most 760 (values of -inf hide their pairs).  A query that sees no key gives 0 (lse -inf) and has no gradient, whatever it holds, and so do keys that no
    query sees; a query that sees an infinity or a NaN gives NaN.  Equal inputs give equal bits, gradients too.

    Gradients are of first order, in reverse mode; under torch.compile too.  Before a backward pass is captured into a graph,
    drop the eager graphs of the same leaves: torch would wait for their streams, which ends the capture.  Raises
    Unsupported for what the kernels do not take."""
    return _attention(q, k, v, bias_table, attn_mask, None, None, tensor_layout, sm_scale, is_causal, bidirectional,
                      max_distance, return_lse)


def _offsets(cu, device):
    """Token offsets as the kernels read them; int64 ones that int32 cannot hold stay too large or too small."""
    if cu.dtype == torch.int64:
        cu = cu.clamp(-1, 2**31 - 1)
    elif cu.dtype != torch.int32:
        raise Unsupported(f"cu_seqlens of {cu.dtype} (int32 or int64)")
    return cu.to(device=device, dtype=torch.int32).contiguous()


def attention_train_varlen(q, k, v, cu_seqlens_q, cu_seqlens_k, max_seqlen_q=None, max_seqlen_k=None, sm_scale=None,
                           is_causal=False, bias_table=None, bidirectional=True, max_distance=128, return_lse=False):
    """attention_train of packed sequences: q [total_q, H, D], k / v [total_k, Hkv, D], cu_seqlens_q / cu_seqlens_k
    [batch + 1] token offsets (int32 or int64).  Each sequence attends to itself alone, with its own diagonal and positions;
    sequences may be empty.  Nothing is read back: rows outside every sequence are 0 (gradients too), and so is everything
    where offsets fall or pass the totals; max_seqlen_q and max_seqlen_k are not needed.  lse: fp32 [H, total_q], unspecified
    outside the sequences."""
    if cu_seqlens_q.dim() != 1 or cu_seqlens_q.shape != cu_seqlens_k.shape or cu_seqlens_q.numel() < 2:
        raise Unsupported("cu_seqlens_q / cu_seqlens_k must be 1-D of one length batch + 1 >= 2")
    cu_q, cu_k = (_offsets(c, q.device) for c in (cu_seqlens_q, cu_seqlens_k))
    return _attention(q, k, v, bias_table, None, cu_q, cu_k, "NHD", sm_scale, is_causal, bidirectional, max_distance, return_lse)


# ---- the bias alone -------------------------------------------------------------------------------------------------------

def _offset_args(offset, gpu):
    if isinstance(offset, torch.Tensor):
        if offset.numel() != 1 or offset.dtype not in (torch.int64, torch.int32) or offset.get_device() != gpu:
            raise Unsupported("q_offset must be an int, or one int32 / int64 value on the table's GPU")
        return 0, offset.data_ptr(), int(offset.dtype == torch.int64)
    if not -2**62 < offset < 2**62:
        raise Unsupported(f"q_offset {offset}")
    return int(offset), None, 0


def _bias_check(table, q_len, kv_len, bidirectional, max_distance, dtype):
    gpu = table.get_device()
    if gpu < 0:
        raise Unsupported("tensors must be on one ROCm GPU")
    if gpu_arch(gpu) not in ARCHS:
        raise Unsupported("not a CDNA4 GPU")
    bias = _bias(table, None, bidirectional, max_distance, gpu)
    if dtype not in TABLE_DTYPES:
        raise Unsupported(f"dtype {dtype} (fp32, bf16 or fp16)")
    if not (0 <= q_len <= 0x3FFFFFFF and 0 <= kv_len <= 0x3FFFFFFF and table.shape[1] <= 65535):
        raise Unsupported(f"bias of {table.shape[1]} heads, {q_len} queries and {kv_len} keys")
    return gpu, bias


def bias_launch(table, q_len, kv_len, bidirectional, max_distance, dtype, offset, offset_at):
    gpu, bias = _bias_check(table, q_len, kv_len, bidirectional, max_distance, dtype)
    H = table.shape[1]
    oa = _offset_args(offset if offset_at is None else offset_at, gpu)
    out = torch.empty((H, q_len, kv_len), dtype=dtype, device=table.device)
    if out.numel():
        t = _table_args(table, bias)
        _capi.call_on(gpu, "sage_relative_bias", *t[:4], H, *t[4:], q_len, kv_len, *oa, out.data_ptr(), TABLE_DTYPES[dtype])
    return out


def bias_grad_launch(dbias, buckets, table_dtype, bidirectional, max_distance, offset, offset_at):
    """The gradient [buckets, H] of a table from that of its bias [H, q_len, kv_len]."""
    H, q_len, kv_len = dbias.shape
    dtable = torch.empty((buckets, H), dtype=table_dtype, device=dbias.device)
    if dbias.numel() == 0:
        return dtable.zero_()
    gpu, bias = _bias_check(dtable, q_len, kv_len, bidirectional, max_distance, dbias.dtype)
    if kv_len > 1 and dbias.stride(2) != 1:
        dbias = dbias.contiguous()
    dt = TABLE_DTYPES[dbias.dtype]
    n = _capi.bias_grad_workspace(H, buckets, q_len, kv_len, dt)
    ws = torch.empty(n, dtype=torch.uint8, device=dbias.device)
    t = _table_args(dtable, bias)
    _capi.call_on(gpu, "sage_relative_bias_grad", dbias.data_ptr(), dbias.stride(0), dbias.stride(1), dt, H, *t[4:], q_len,
                  kv_len, *_offset_args(offset if offset_at is None else offset_at, gpu), *t[:4], ws.data_ptr(), n)
    return dtable


class _Bias(torch.autograd.Function):
    """bias_launch with its table's gradient, for eager calls."""

    @staticmethod
    def forward(ctx, table, q_len, kv_len, bidirectional, max_distance, dtype, offset, offset_at):
        ctx.how = table.shape[0], table.dtype, bidirectional, max_distance, offset
        ctx.save_for_backward(offset_at)
        return bias_launch(table, q_len, kv_len, bidirectional, max_distance, dtype, offset, offset_at)

    @staticmethod
    @once_differentiable
    def backward(ctx, dbias):
        return (bias_grad_launch(dbias, *ctx.how, *ctx.saved_tensors),) + (None,) * 7


def relative_bias(table, q_len, kv_len, bidirectional=True, max_distance=128, dtype=None, q_offset=None):
    """A learned bias by relative position: [H, q_len, kv_len] of `dtype` (table's where None), for attention's attn_mask, from
    learned values [buckets, H] (fp32, bf16 or fp16).  Key j is at position j, query i at q_offset + i; q_offset: an int
    (None: kv_len - q_len, the last query at the last key), or one int32 / int64 value on the GPU, so that a captured decoding
    step can move on.

    bidirectional: half of the buckets for keys ahead of the query; otherwise those share the bucket of distance 0.  Of one
    side's buckets the first half hold a distance each, the others ranges whose borders grow evenly in the logarithm up to
    max_distance; borders are exact.  Differentiable in table (first order, reverse mode), its gradient summed in float32.
    Raises Unsupported for what the kernels do not take."""
    dtype = table.dtype if dtype is None else dtype
    at = q_offset if isinstance(q_offset, torch.Tensor) else None
    offset = 0 if at is not None else kv_len - q_len if q_offset is None else int(q_offset)
    args = (int(q_len), int(kv_len), bool(bidirectional), int(max_distance), dtype, offset, at)
    if _plain_eager(table, grad=True):
        if torch.is_grad_enabled() and table.requires_grad:
            return _Bias.apply(table, *args)
        return bias_launch(table, *args)
    refuse_tangents("relative_bias", table)
    return ops.relative_bias(table, *args)
