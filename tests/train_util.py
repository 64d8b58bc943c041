"""The attention for training and the relative position bias in float64, and the distances that the kernels' arithmetic allows."""
from __future__ import annotations

import math

import torch

F32 = 2.0 ** -24          # half a step of float32, relative


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def bucket_of(away, buckets, reach, two_sided):
    """The bucket of a key `away` tokens ahead of its query, by whole numbers."""
    side = buckets // 2 if two_sided else buckets
    near = side // 2
    m = side - near
    n = abs(away) if two_sided else max(-away, 0)
    if n < near:
        b = n
    else:
        t = 0
        while t + 1 < m and n ** m >= near ** (m - t - 1) * reach ** (t + 1):
            t += 1
        b = near + t
    return b + side if two_sided and away > 0 else b


def bucket_map(Sq, Skv, buckets, reach, two_sided, offset=None):
    """[Sq, Skv] buckets; query i at position offset + i (default: the last query at the last key)."""
    offset = Skv - Sq if offset is None else offset
    of = {}
    rows = []
    for i in range(Sq):
        row = []
        for j in range(Skv):
            d = j - i - offset
            if d not in of:
                of[d] = bucket_of(max(-4 * reach, min(4 * reach, d)), buckets, reach, two_sided)
            row.append(of[d])
        rows.append(row)
    return torch.tensor(rows)


class Exact:
    """Attention of q [B, H, Sq, D] over k, v [B, Hkv, Skv, D] with its gradients in float64, and bounds of the kernels' distance:
    products and sums in float32 (each term's error counted at its largest), the weights p and the scores' gradients ds rounded to
    the inputs' type, results rounded once."""

    def __init__(self, q, k, v, causal=False, seen=None, bias=None, dout=None, sm_scale=None):
        u = half_step(q.dtype)
        self.dtype = q.dtype
        q, k, v = (t.double() for t in (q, k, v))
        B, H, Sq, D = q.shape
        Hkv, Skv = k.shape[1], k.shape[2]
        G = H // Hkv
        scale = sm_scale or D ** -0.5
        k, v = (t.repeat_interleave(G, dim=1) for t in (k, v))
        vis = torch.ones(1, 1, Sq, Skv, dtype=torch.bool)
        if causal:
            vis = vis.tril(Skv - Sq)
        if seen is not None:
            vis = vis & seen.cpu()
        vis = vis.expand(B, H, Sq, Skv)
        self.seen = vis
        x = q @ k.transpose(2, 3) * scale
        ax = q.abs() @ k.abs().transpose(2, 3) * scale
        if bias is not None:
            x = x + bias
            ax = ax + bias.abs()
        x = x.masked_fill(~vis, -math.inf)
        self.lse = torch.logsumexp(x, dim=-1)
        empty = self.lse == -math.inf
        top = torch.where(empty, 0.0, self.lse)
        p = torch.exp(x - top[..., None])
        self.p = p
        self.out = p @ v
        # a score's error in float32, its sum of D products at worst, the exponent's and the statistics'; twice: of p and of lse
        ax = ax.masked_fill(~vis, 0.0).amax(dim=-1) + top.abs() + 4.0
        ep = 2.0 * F32 * (D + 8) * ax[..., None]
        n = Skv * F32
        tiny = 2.0 ** -30 if self.dtype == torch.float16 else 0.0   # fp16's smallest steps, of weights scaled by 2^6 and more
        vmax = float(v.abs().max()) if v.numel() else 0.0
        # fp16 results below 2^-14 are multiples of 2^-24: they are off by up to half of that, however small they are
        least = 2.0 ** -25 if self.dtype == torch.float16 else 0.0
        self.room_out = least + u * self.out.abs() + (p * (u + 2 * ep + n)) @ v.abs() + tiny * Skv * vmax
        self.room_lse = F32 * (D + 16) * ax + n
        if dout is None:
            return
        do = dout.double()
        do = torch.where(empty[..., None], 0.0, do)
        dp = do @ v.transpose(2, 3)
        delta = (do * self.out).sum(dim=-1, keepdim=True)
        ds = p * (dp - delta)
        self.ds = ds
        back = lambda t: t.unflatten(1, (Hkv, G)).sum(2)  # noqa: E731
        self.dq = ds @ k * scale
        self.dk = back(ds.transpose(2, 3) @ q) * scale
        self.dv = back(p.transpose(2, 3) @ do)
        off_dp = F32 * (D + 8) * (do.abs() @ v.abs().transpose(2, 3) + (do * self.out).abs().sum(-1, keepdim=True))
        # of delta, by the rounding of out's weights; out itself is known to 2 u^2 (fp16: to half of its smallest step)
        kept = self.room_out - u * self.out.abs() + 2 * u * u * self.out.abs()
        off_d = (do.abs() * kept).sum(dim=-1, keepdim=True)
        self.sums = 3 * ep * ds.abs() + p * off_dp                      # of ds in float32, delta's error apart
        domax = float(do.abs().max())
        small = 2.0 ** -34 * domax * vmax if self.dtype == torch.float16 else 0.0   # fp16's smallest steps of scaled ds
        self.p_off_d = p * off_d
        room_ds = u * ds.abs() + self.sums + self.p_off_d + small
        N = (Sq * G + Skv) * F32
        self.room_dq = least + u * self.dq.abs() + (room_ds + N * ds.abs()) @ k.abs() * scale
        self.room_dk = least + u * self.dk.abs() + back((room_ds + N * ds.abs()).transpose(2, 3) @ q.abs()) * scale
        self.room_dv = least + u * self.dv.abs() + back((p * (u + 4 * ep + N)).transpose(2, 3) @ do.abs()) + \
            (2.0 ** -38 * domax * Sq * G if self.dtype == torch.float16 else 0.0)

    def table(self, bucket, buckets, reach_out, dtype):
        """(gradient [buckets, H] of the bias' table, its room).  reach_out: the pairs of the two outermost buckets, whose sums are
        freed of delta's error."""
        H = self.ds.shape[1]

        def by(t):
            out = torch.zeros(buckets, H, dtype=torch.float64)
            return out.index_add_(0, bucket.flatten(), t.sum(0).flatten(1).t().contiguous())

        d = by(self.ds)
        far = reach_out.double()
        freed = self.p * self.sums.sum(-1, keepdim=True)
        room = by(self.sums + (1 - far) * self.p_off_d + far * freed)
        count = by(self.ds.abs())
        least = 2.0 ** -25 if dtype == torch.float16 else 0.0
        return d, least + half_step(dtype) * d.abs() + room + 64 * F32 * count


def close(got, want, room):
    off = (got.detach().double().cpu() - want).abs()
    bad = ~(off <= room + 1e-30)
    assert not bool(bad.any()), (float((off / (room + 1e-30)).max()), int(bad.sum()), bad.nonzero()[:4].tolist())
