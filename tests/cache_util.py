"""Plain float64 forms of the decoding operators, on the CPU, and the distances that their kernels' arithmetic allows."""
from __future__ import annotations

import math

import torch

Q_MAX = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def step(dtype):
    """Half a step of dtype, relative to the value."""
    return torch.finfo(dtype).eps / 2


def quantize(x, dtype):
    """(codes, scales) of the rows of x [..., D] by the cache's definition."""
    x = x.double()
    a = x.abs().amax(dim=-1)
    bad = ~torch.isfinite(x).all(dim=-1)
    a = torch.where(bad, 0.0, a)
    y = torch.where(bad.unsqueeze(-1), 0.0, x) * Q_MAX[dtype] / torch.where(a > 0, a, 1.0).unsqueeze(-1)
    codes = torch.round(y).to(torch.int8) if dtype == torch.int8 else y.float().to(dtype)
    scale = a.float() / Q_MAX[dtype]          # float32 division, rounded once
    return codes, torch.where(bad, float("nan"), scale)


def random_cache(g, pages, page_size, heads, D, dtype, spread=0.0):
    """(k, v, k_scale, v_scale) of normal rows, row magnitudes spread by 10^(spread * N(0, 1))."""
    out = []
    for _ in range(2):
        x = torch.randn(pages, heads, page_size, D, generator=g, dtype=torch.float64)
        x *= 10.0 ** (spread * torch.randn(pages, heads, page_size, 1, generator=g, dtype=torch.float64))
        out.append(quantize(x.float(), dtype))
    return out[0][0], out[1][0], out[0][1], out[1][1]


def as_int8(t):
    return t if t.dtype == torch.int8 else t.view(torch.int8)


def attention(q, cache, table, lengths, sm_scale=None, is_causal=True, tree=None):
    """q [B, H, T, D] float64; returns out, lse, and for the tolerances per output the weighted magnitudes sum_j p_j |v_j|
    + 2^-19 max_j (p_j s_j) sum_j |code_j| (s: the values' scales) and per row the largest sum_c |q_c k_c| * scale over its
    visible keys."""
    k8, v8, ks, vs = cache
    B, H, T, D = q.shape
    pages, Hkv, n, _ = k8.shape
    scale = D ** -0.5 if sm_scale is None else sm_scale
    out = torch.zeros(B, H, T, D, dtype=torch.float64)
    mag = torch.zeros_like(out)
    lse = torch.full((B, H, T), -math.inf, dtype=torch.float64)
    big = torch.zeros(B, H, T, dtype=torch.float64)
    for b in range(B):
        length = min(max(int(lengths[b]), 0), table.shape[1] * n)
        keys = torch.arange(length)
        page = table[b][keys // n].long()
        ok = (page >= 0) & (page < pages)
        keys, page = keys[ok], page[ok]
        node = keys - (length - T)
        for i in range(T):
            seen = torch.ones_like(ok[ok])
            if tree is not None:
                t = tree if tree.dim() == 2 else tree[b if tree.shape[0] > 1 else 0]
                seen = (node < 0) | t[i][node.clamp(min=0)]
            elif is_causal:
                seen = node <= i
            pg, row = page[seen], keys[seen] % n
            if not pg.numel():
                continue
            for h in range(H):
                hk = h // (H // Hkv)
                K = k8[pg, hk, row].double() * ks[pg, hk, row].double()[:, None]
                C, s = v8[pg, hk, row].double(), vs[pg, hk, row].double()
                V = C * s[:, None]
                x = K @ q[b, h, i] * scale
                p = torch.softmax(x, 0)
                out[b, h, i] = p @ V
                mag[b, h, i] = p @ V.abs() + 2.0 ** -19 * (p * s).max() * C.abs().sum(0)
                lse[b, h, i] = torch.logsumexp(x, 0)
                big[b, h, i] = (K.abs() @ q[b, h, i].abs()).max() * scale
    return out, lse, mag, big


def score_slack(big, D):
    """How far a score may be off: D products summed in float32 (each partial sum within their magnitudes' sum), two
    scale factors and the exponential's argument, each off by half a step."""
    return big * (D + 8) * 2.0 ** -24


def attention_slack(mag, big, out, D, dtype):
    """Bound of |kernel - exact|: weights off by twice the score's slack (numerator and sum) and by a float16 rounding
    (2^-11), the float32 sums and exponentials (a few steps of 2^-24 each: 2^-20), and the output's own rounding.  The
    products p_j s_j are rounded to float16 with the row's largest at 2^6 or more, so those below 2^-14 there, float16's
    subnormals, are off by up to 2^-25, that is 2^-31 of the largest; each is multiplied by its code, so together by at
    most 2^-31 max_j (p_j s_j) sum_j |code_j|.  No multiple of sum_j p_j |v_j| bounds that: in a channel where the keys of
    large products have code 0 the sum can be as small as one likes.  attention's second term of mag times 2^-11 is twice
    that.  A float16 output below 2^-14 lies between multiples of 2^-24 and is rounded by up to 2^-25, more than half a step
    relative to it (9.5017e-06, the value of a single visible key, has the neighbours 9.4771e-06 and 9.5367e-06)."""
    tiny = 2.0 ** -25 if dtype == torch.float16 else 1e-30
    return mag * (2.0 ** -11 + 2.0 ** -20 + 2.0 * score_slack(big, D).unsqueeze(-1)) + out.abs() * step(dtype) + tiny


def lse_slack(big, lse, D):
    return score_slack(big, D) + (lse.abs() + 2.0) * 2.0 ** -21


def rotate(x, positions, freqs, interleaved, factor=1.0, back=False):
    """x [B, S, H, D] float64 (NHD), positions [B, S]; returns the rotated x and |a| + |b| of each element's pair."""
    R = 2 * freqs.numel()
    ang = positions.double()[:, :, None] * freqs.double()
    c, s = (torch.cos(ang) * factor).unsqueeze(2), (torch.sin(ang) * factor).unsqueeze(2)
    if back:
        s = -s
    y, m = x.clone(), torch.zeros_like(x)
    ia = slice(0, R, 2) if interleaved else slice(0, R // 2)
    ib = slice(1, R, 2) if interleaved else slice(R // 2, R)
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    m[..., ia] = m[..., ib] = a.abs() + b.abs()
    return y, m


def rotate_slack(y, m, factor, dtype):
    """Sine and cosine off by 2^-21 (the rest of the turn rounded to 2^-25 turns, 2^-22.3 radians, and their evaluation to a
    few steps of 2^-24), two float32 products and a sum, and the output's rounding (float16 has a smallest step of
    2^-24)."""
    return m * factor * 2.0 ** -20 + y.abs() * step(dtype) + (2.0 ** -25 if dtype == torch.float16 else 0.0)
