"""Rotary positions on the gfx950 kernel (no counterpart in the reference, whose callers rotate q and k with torch).

One launch turns q and k; gradients turn back by the same kernel.  Frequencies are float64 tensors made once per model by
rope_frequencies, so that positions of 10^6 and more keep their angle.
"""
from __future__ import annotations

import math

import torch
from torch.autograd import forward_ad

from . import _capi, ops
from ._attention import (_I32_MAX, ARCHS, DTYPES, HEAD_DIMS, Unsupported, _bsh, _plain_tensors, gpu_arch,
                         refuse_tangents)


def rope_frequencies(rot_dim, base=10000.0, scaling=None, device=None):
    """(freqs, factor) for rope: radians per position of the rot_dim / 2 channel pairs, float64 on `device`, and the
    factor of the rotated channels.  freqs[i] = base^(-2 i / rot_dim).  scaling, for contexts longer than the one a model
    was trained on, is None or a dict:

    {"type": "linear", "factor": s}: positions interpolated, every frequency divided by s.
    {"type": "ntk", "factor": s}: the base raised to base * s^(rot_dim / (rot_dim - 2)), which divides the slowest
        frequency by s and leaves the fastest.
    {"type": "yarn", "factor": s, "original_length": n, "slow": 1, "fast": 32, "attention_factor": None}: pairs that turn
        less than `slow` times over n positions divided by s, those of more than `fast` turns kept, linear in the pair's
        index in between; the rotated channels times attention_factor (0.1 ln s + 1 where None)."""
    if rot_dim <= 0 or rot_dim % 2:
        raise ValueError(f"rot_dim {rot_dim} (positive and even)")
    if not base > 0:
        raise ValueError(f"base {base}")
    i = torch.arange(rot_dim // 2, dtype=torch.float64)
    factor = 1.0
    if scaling is None:
        f = base ** (-2.0 * i / rot_dim)
    else:
        kind, s = scaling.get("type"), float(scaling.get("factor", 0.0))
        if not s >= 1.0:
            raise ValueError(f"scaling factor {s} (at least 1)")
        if kind == "linear":
            f = base ** (-2.0 * i / rot_dim) / s
        elif kind == "ntk":
            if rot_dim == 2:
                raise ValueError("ntk scaling needs rot_dim > 2")
            f = (base * s ** (rot_dim / (rot_dim - 2))) ** (-2.0 * i / rot_dim)
        elif kind == "yarn":
            n, slow, fast = (float(scaling[x]) if x in scaling else d for x, d in
                             (("original_length", 0.0), ("slow", 1.0), ("fast", 32.0)))
            if not n > 0 or not fast > slow > 0:
                raise ValueError("yarn scaling needs original_length > 0 and fast > slow > 0")
            # the (fractional) index of the pair that turns t times over n positions
            at = [rot_dim * math.log(n / (2.0 * math.pi * t)) / (2.0 * math.log(base)) for t in (fast, slow)]
            lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rot_dim - 1)
            ramp = ((i - lo) / max(hi - lo, 1e-3)).clamp(0.0, 1.0)
            f = base ** (-2.0 * i / rot_dim)
            f = f * (1.0 - ramp) + f / s * ramp
            factor = scaling.get("attention_factor")
            factor = 0.1 * math.log(s) + 1.0 if factor is None else float(factor)
        else:
            raise ValueError(f"scaling type {kind!r} ('linear', 'ntk' or 'yarn')")
    return f.to(device=device), factor


def check_rope(q, k, positions, freqs, layout):
    """(batch, tokens, heads, head_dim) of q and the GPU's index; raises Unsupported with the reason."""
    if layout != "HND" and layout != "NHD":
        raise Unsupported(f"layout {layout!r}")
    shape = q.shape
    if len(shape) != 4 or (k is not None and k.dim() != 4):
        raise Unsupported("4D tensors required")
    if q.dtype not in DTYPES or (k is not None and k.dtype != q.dtype):
        raise Unsupported(f"dtype {q.dtype} (fp16 or bf16 required, the same for q and k)")
    (B, H, S, D) = shape if layout == "HND" else (shape[0], shape[2], shape[1], shape[3])
    if D not in HEAD_DIMS:
        raise Unsupported(f"head_dim {D} (supported {HEAD_DIMS})")
    gpu, big = q.get_device(), q.numel()
    if k is not None:
        ks = k.shape
        if ks[0] != B or ks[3] != D or ks[2 if layout == "HND" else 1] != S:
            raise Unsupported("q and k must have the same batch, length and head_dim")
        if k.get_device() != gpu:
            raise Unsupported("tensors must be on one ROCm GPU")
        big = max(big, k.numel())
    if freqs.dim() != 1 or freqs.dtype != torch.float64:
        raise Unsupported("freqs must be a 1D float64 tensor (rope_frequencies)")
    rot = 2 * freqs.shape[0]
    if rot == 0 or rot > D or rot % 8:
        raise Unsupported(f"{rot} rotated channels (a positive multiple of 8 up to head_dim {D})")
    if positions is not None:
        if positions.dtype != torch.int64 and positions.dtype != torch.int32:
            raise Unsupported(f"positions {positions.dtype} (int32 or int64)")
        ps = positions.shape
        if ps != (B, S) and ps != (S,) and ps != (1, S):
            raise Unsupported(f"positions of shape {tuple(ps)} for batch {B} and length {S}")
        if positions.get_device() != gpu:
            raise Unsupported("tensors must be on one ROCm GPU")
    if gpu < 0 or freqs.get_device() != gpu:
        raise Unsupported("tensors must be on one ROCm GPU")
    if gpu_arch(gpu) not in ARCHS:
        raise Unsupported("not a CDNA4 GPU")
    if big > _I32_MAX:
        raise Unsupported("tensor too large for 32-bit indexing")
    return B, S, H, D, gpu


def rope_launch(q, k, positions, freqs, layout, interleaved, factor, inverse):
    """The rotated q (and k), in new tensors (out_like)."""
    B, S, H, D, gpu = check_rope(q, k, positions, freqs, layout)
    oq = out_like(q)
    ok = None if k is None else out_like(k)
    if q.numel() == 0:   # no tokens, or no query heads: k alone
        if k is None or k.numel() == 0:
            return oq, ok
        return oq, rope_launch(k, None, positions, freqs, layout, interleaved, factor, inverse)[0]
    q, sq = _bsh(q, layout)
    so = _bsh(oq, layout)[1]
    pos, p64, pb, ps = None, 0, 0, 0
    if positions is not None:
        st = positions.stride()
        pos, p64, ps = positions.data_ptr(), positions.dtype == torch.int64, st[-1]
        if len(st) == 2 and positions.shape[0] > 1:
            pb = st[0]
    freqs = freqs.contiguous()
    rest = (B, S, D, DTYPES[q.dtype], pos, p64, pb, ps, freqs.data_ptr(), 2 * freqs.shape[0], bool(interleaved), factor,
            bool(inverse))
    Hk = 0 if k is None else k.shape[1 if layout == "HND" else 2]
    if Hk:
        k, sk = _bsh(k, layout)
        sko = _bsh(ok, layout)[1]
        _capi.call_on(gpu, "sage_rope", q.data_ptr(), *sq, oq.data_ptr(), *so, H, k.data_ptr(), *sk, ok.data_ptr(), *sko,
                      Hk, *rest)
    else:
        _capi.call_on(gpu, "sage_rope", q.data_ptr(), *sq, oq.data_ptr(), *so, H, None, 0, 0, 0, None, 0, 0, 0, 0, *rest)
    return oq, ok


def out_like(t):
    """An output for t: in t's memory order, or contiguous where the kernel cannot store 16-byte vectors in that order (the
    ops' fake implementations promise the same)."""
    out = torch.empty_like(t)
    s = out.stride()
    if len(s) == 4 and (s[3] != 1 or s[0] % 8 or s[1] % 8 or s[2] % 8):
        out = torch.empty(t.shape, dtype=t.dtype, device=t.device)
    return out


_transform = torch._C._functorch.peek_interpreter_stack   # the innermost of torch.func's transforms, or None


def _derived(*args):
    """rope_launch under autograd, in forward-mode levels and torch.func's transforms."""
    return (_Rope if _transform() is None else _RopeTransformed).apply(*args)


class _Rope(torch.autograd.Function):
    """rope_launch with its derivatives.  The rotation is linear: tangents turn as the inputs do, gradients turn back, and
    each is an application of its own, so that derivatives have derivatives."""

    @staticmethod
    def forward(ctx, *args):
        out = rope_launch(*args)
        _, k, positions, freqs, *ctx.how = args
        ctx.save_for_backward(positions, freqs)
        if forward_ad._current_level >= 0:
            ctx.save_for_forward(positions, freqs)
        elif k is not None:
            # the output of an input that needs no gradient needs none either (one of the two does)
            if not ctx.needs_input_grad[0]:
                ctx.mark_non_differentiable(out[0])
            elif not ctx.needs_input_grad[1]:
                ctx.mark_non_differentiable(out[1])
        return out

    @staticmethod
    def backward(ctx, dq, dk):
        *how, inverse = ctx.how
        need_q, need_k = ctx.needs_input_grad[:2]
        back = (*ctx.saved_tensors, *how, not inverse)
        # (create_graph: the gradients have gradients of their own)
        turn = _derived if torch.is_grad_enabled() or forward_ad._current_level >= 0 or _transform() is not None else rope_launch
        if need_q and need_k:
            dq, dk = turn(dq, dk, *back)
        elif need_q:
            dq, dk = turn(dq, None, *back)[0], None
        else:
            dq, dk = None, turn(dk, None, *back)[0] if need_k else None
        return dq, dk, None, None, None, None, None, None

    @staticmethod
    def jvp(ctx, tq, tk, *_):
        # (an input without a tangent comes with one of zeros)
        return _derived(tq, tk, *ctx.saved_tensors, *ctx.how)


class _RopeTransformed(_Rope):
    """_Rope in the form that torch.func's transforms take, which takes longer a call."""

    @staticmethod
    def forward(q, k, positions, freqs, layout, interleaved, factor, inverse):
        return rope_launch(q, k, positions, freqs, layout, interleaved, factor, inverse)

    @staticmethod
    def setup_context(ctx, inputs, output):
        _, _, positions, freqs, *ctx.how = inputs
        ctx.save_for_backward(positions, freqs)
        ctx.save_for_forward(positions, freqs)

    @staticmethod
    def vmap(info, in_dims, q, k, positions, freqs, *how):
        n = info.batch_size
        most = max(t.numel() // (1 if d is None else n) for t, d in zip((q, k), in_dims) if t is not None)
        if in_dims[3] is not None or n * most > _I32_MAX:   # frequencies of each entry's own, or too large: one launch each
            outs = [_derived(*(t if d is None else t.select(d, i) for t, d in zip((q, k, positions, freqs), in_dims)), *how)
                    for i in range(n)]
            return (torch.stack([o[0] for o in outs]), None if k is None else torch.stack([o[1] for o in outs])), \
                (0, None if k is None else 0)

        def first(t, d):
            return t.expand(n, *t.shape) if d is None else t.movedim(d, 0)

        # the mapped dimension joins the batch
        q, k = first(q, in_dims[0]), None if k is None else first(k, in_dims[1])
        B = q.shape[1]
        if positions is not None and (in_dims[2] is not None or positions.dim() > 1):
            positions = first(positions, in_dims[2])
            if positions.dim() == 2:
                positions = positions[:, None]
            if positions.dim() != 3 or positions.shape[1] not in (1, B):
                raise Unsupported(f"positions of shape {tuple(positions.shape[1:])} for batch {B}")
            positions = positions.expand(n, B, positions.shape[2]).flatten(0, 1)
        oq, ok = _derived(q.flatten(0, 1), None if k is None else k.flatten(0, 1), positions, freqs, *how)
        return (oq.unflatten(0, (n, B)), None if k is None else ok.unflatten(0, (n, B))), (0, None if k is None else 0)


def rope(q, k=None, positions=None, freqs=None, tensor_layout="HND", interleaved=False, factor=1.0):
    """Rotary positions: the first 2 * freqs.numel() channels of every head are pairs, (i, i + rot_dim / 2) or, interleaved,
    (2 i, 2 i + 1), and pair i of a token at position p turns by p * freqs[i] radians, times `factor`; the other
    channels are copied.  q: [B, heads, tokens, head_dim] for "HND", [B, tokens, heads, head_dim] for "NHD", k alike with
    heads of its own, bf16 or fp16.  positions: int32 / int64 [tokens] or [B, tokens] (None: 0, 1, ..).  freqs, factor:
    rope_frequencies.  Returns q, or (q, k), in new tensors, of the inputs' memory order where head_dim is innermost there.
    Differentiable in q and k (to any order, in reverse and forward mode, by torch.func's transforms too; under torch.compile
    in reverse mode, forward mode raises); float32 arithmetic, rounded once.  Before a backward pass is captured into a graph,
    drop the eager graphs of the same leaves: torch would wait for their streams, which ends the capture.  Raises
    Unsupported for what the kernel does not take."""
    if freqs is None:
        raise Unsupported("freqs are required (rope_frequencies)")
    ts = (q,) if k is None else (q, k)
    args = (positions, freqs, tensor_layout, interleaved, factor, False)
    if _plain_tensors(*ts):
        if _transform() is not None:
            out = _RopeTransformed.apply(q, k, *args)
        elif ((q.requires_grad or (k is not None and k.requires_grad)) and torch.is_grad_enabled()) or forward_ad._current_level >= 0:
            out = _Rope.apply(q, k, *args)
        else:
            out = rope_launch(q, k, *args)
        return out[0] if k is None else out
    refuse_tangents("rope under a tracer", *ts)
    if k is None:
        return ops.rope(q, positions, freqs, tensor_layout, bool(interleaved), float(factor), False)
    return ops.rope_qk(q, k, positions, freqs, tensor_layout, bool(interleaved), float(factor), False)
