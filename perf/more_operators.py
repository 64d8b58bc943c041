"""The training operators of this package as cases that can be prepared, run, timed and checked: attention on 16-bit inputs
with its backward pass, dense and packed (``cdna4_sage.attention_train``, ``cdna4_sage.attention_train_varlen``), and a
learned relative position bias by buckets with its gradient (``cdna4_sage.relative_bias``, and inside the attention).

``run`` computes their plain form from elementary torch operations, or calls the package where ``own`` is true.  Head
counts and head dims are those of cdna4_sage.configs and of the tests; lengths and batches are theirs or generic.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _package():
    packages = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rdna4-sageattention_amd")
    if packages not in sys.path:
        sys.path.insert(0, packages)
    import cdna4_sage

    return cdna4_sage


# ---- the cases ------------------------------------------------------------------------------------------------------

def _attend(B, H, Hkv, Sq, Skv, D, layout, dtype, causal=False, mask="", buckets=0, reach=128, train=True, lse=False):
    """mask: "" for none, "keys" for padded keys, "docs" for documents one after the other in every row, with padding behind
    the last one that sees nothing.  buckets: of the relative position bias, 0 for none; two-sided unless causal."""
    return {"op": "attend", "B": B, "H": H, "Hkv": Hkv, "Sq": Sq, "Skv": Skv, "D": D, "layout": layout, "dtype": dtype,
            "causal": causal, "mask": mask, "buckets": buckets, "reach": reach, "train": train, "lse": lse}


def _packed(B, H, Hkv, shortest, longest, D, dtype, causal=True):
    """B sequences of shortest to longest tokens, one behind the other."""
    return {"op": "packed", "B": B, "H": H, "Hkv": Hkv, "shortest": shortest, "longest": longest, "D": D, "dtype": dtype,
            "causal": causal}


def _bias(H, Sq, Skv, buckets, reach, two_sided, dtype, table, train=False):
    """dtype: of the bias; table: of the learned values."""
    return {"op": "bias", "H": H, "Sq": Sq, "Skv": Skv, "buckets": buckets, "reach": reach, "two_sided": two_sided,
            "dtype": dtype, "table": table, "train": train}


def listed():
    return [
        # a training step of a small model on short sequences: where launches and the host's work count
        dict(_attend(4, 8, 8, 128, 128, 64, "HND", "bf16", causal=True), name="train_small"),
        # fine-tuning an image model: the joint attention of configuration 2
        dict(_attend(1, 24, 24, 4608, 4608, 128, "HND", "bf16"), name="train_joint"),
        # a language model with shared key / value heads: configuration 5a
        dict(_attend(2, 32, 8, 8192, 8192, 128, "HND", "bf16", causal=True), name="train_causal"),
        # the widest heads, an odd length
        dict(_attend(2, 12, 12, 2180, 2180, 256, "HND", "f16"), name="train_wide"),
        # the end of a longer sequence, of odd lengths, behind a prefix
        dict(_attend(3, 10, 5, 1777, 2049, 96, "NHD", "f16", causal=True), name="train_suffix"),
        # documents one after the other in padded rows, which see nothing at their ends
        dict(_attend(6, 16, 4, 1250, 1250, 64, "NHD", "bf16", causal=True, mask="docs"), name="train_docs"),
        # a packed batch of uneven sequences
        dict(_packed(14, 32, 8, 77, 3001, 128, "bf16"), name="train_packed"),
        # scoring: image tokens over a padded prompt, no gradients, with the logsumexp
        dict(_attend(2, 10, 10, 4096, 77, 64, "NHD", "f16", mask="keys", train=False, lse=True), name="score_cross"),
        # an encoder with a learned bias by distance, its table's gradient with the others
        dict(_attend(4, 16, 16, 1024, 1024, 64, "HND", "bf16", buckets=32), name="train_biased"),
        # the bias of one new token over its context
        dict(_bias(32, 1, 8192, 32, 128, False, "bf16", "bf16"), name="bias_token"),
        # the bias of a prompt, as a mask for the quantized attention
        dict(_bias(24, 4352, 4352, 32, 128, True, "bf16", "f32"), name="bias_prompt"),
        # the bias and its table's gradient from the gradient of every element, odd sizes
        dict(_bias(16, 2047, 2511, 64, 800, True, "f16", "f32", train=True), name="bias_train"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        kind = rng.choice(["train", "train", "train", "causal", "causal", "mask", "packed", "score", "biased", "bias", "bias"])
        dtype, layout = rng.choice(["bf16", "bf16", "f16"]), rng.choice(["HND", "NHD"])
        D, Hkv = rng.choice([64, 64, 96, 128, 128, 256]), rng.choice([1, 2, 4, 5, 8, 8, 10, 12, 16, 24])
        H = Hkv * rng.choice([1, 1, 2, 4])
        if H > 40:
            continue
        if kind == "bias":
            Skv = _log_int(rng, 3, 9000)
            Sq = 1 if rng.random() < 0.25 else _log_int(rng, 2, 6000)
            two = rng.random() < 0.5
            c = _bias(H, Sq, Skv, rng.choice([8, 16, 32, 32, 64]), rng.choice([64, 128, 128, 500, 2000]), two,
                      rng.choice(["bf16", "f16", "f32"]), rng.choice(["f32", dtype]), train=rng.random() < 0.5)
            if H * Sq * Skv > 1 << 28:
                continue
        elif kind == "packed":
            B, longest = rng.randint(2, 40), _log_int(rng, 16, 3000)
            c = _packed(B, H, Hkv, rng.randint(1, longest), longest, D, dtype, causal=rng.random() < 0.7)
            if B * H * longest * longest > 1 << 31:
                continue
        else:
            B, Skv = rng.randint(1, 6), _log_int(rng, 2, 8000)
            Sq = Skv if rng.random() < 0.5 else _log_int(rng, 1, 8000)
            causal = kind == "causal" or (kind in ("biased", "mask") and rng.random() < 0.5)
            if causal and Sq > Skv:
                Sq, Skv = Skv, Sq
            mask = "" if kind in ("train", "causal", "biased") else "keys" if rng.random() < 0.5 or Sq != Skv else "docs"
            c = _attend(B, H, Hkv, Sq, Skv, D, layout, dtype, causal=causal, mask=mask,
                        buckets=rng.choice([16, 32, 64]) if kind == "biased" else 0, reach=rng.choice([100, 128, 256]),
                        train=kind != "score", lse=kind == "score")
            # the plain form holds its scores in 32 bits
            if B * H * Sq * Skv > 1 << 31:
                continue
        w, most = work(c), work(_attend(2, 32, 8, 8192, 8192, 128, "HND", "bf16", causal=True))
        if max(w["bytes"], w["flops"] / 50) <= max(most["bytes"], most["flops"] / 50):
            return c


def _lengths(case):
    """Tokens of every packed sequence: spread from the shortest to the longest, in no order."""
    B, lo, hi = case["B"], case["shortest"], case["longest"]
    return [lo + (hi - lo) * ((b * 5 + 3) % B) // (B - 1) for b in range(B)]


def _visible_keys(case):
    """Of a "keys" mask: how many keys each batch entry shows, the last entry all of them."""
    B, n = case["B"], case["Skv"]
    return [max(1, n - (B - 1 - b) * n // (2 * B)) for b in range(B)]


def _documents(case):
    """Of a "docs" mask: every token's document, -1 for padding, as a row for each batch entry."""
    B, n = case["B"], case["Skv"]
    rows = []
    for b in range(B):
        size, pad = max(1, n // (2 + b % 3)), n * (b % 4) // 20
        rows.append([i // size if i < n - pad else -1 for i in range(n)])
    return rows


def _pairs(case):
    """Visible (query, key) pairs of one head, over the batch."""
    def triangle(q, k):  # the last q of k tokens, each up to itself
        return q * (k - q) + q * (q + 1) // 2

    if case["op"] == "packed":
        return sum(triangle(n, n) if case["causal"] else n * n for n in _lengths(case))
    B, Sq, Skv = case["B"], case["Sq"], case["Skv"]
    if case["mask"] == "docs":
        total = 0
        for row in _documents(case):
            sizes = {}
            for d in row:
                if d >= 0:
                    sizes[d] = sizes.get(d, 0) + 1
            total += sum(triangle(n, n) if case["causal"] else n * n for n in sizes.values())
        return total
    if case["mask"] == "keys":
        if not case["causal"]:
            return sum(Sq * n for n in _visible_keys(case))
        return sum(sum(min(n, i + 1 + Skv - Sq) for i in range(Sq)) for n in _visible_keys(case))
    return B * (triangle(Sq, Skv) if case["causal"] else Sq * Skv)


def _size(dtype):
    return 4 if dtype == "f32" else 2


def work(case):
    """Inputs read once and outputs written once; the products of the visible (query, key) pairs: two forward, and five
    backward (the scores once more, the gradient of the probabilities, and those of q, k and v)."""
    if case["op"] == "bias":
        n = case["H"] * case["Sq"] * case["Skv"]
        t = case["buckets"] * case["H"] * _size(case["table"])
        return {"bytes": n * _size(case["dtype"]) * (2 if case["train"] else 1) + t * (2 if case["train"] else 1),
                "flops": n if case["train"] else 0}
    H, Hkv, D = case["H"], case["Hkv"], case["D"]
    if case["op"] == "packed":
        tq = tk = sum(_lengths(case))
    else:
        tq, tk = case["B"] * case["Sq"], case["B"] * case["Skv"]
    train = case.get("train", True)
    q, kv = 2 * tq * H * D, 2 * 2 * tk * Hkv * D
    nbytes = 2 * q + kv
    if train:
        nbytes += 2 * q + kv  # the output's gradient, and dq, dk, dv
    if case.get("lse"):
        nbytes += 4 * tq * H
    if case.get("mask") == "docs":
        nbytes += case["B"] * case["Sq"] * case["Skv"]
    elif case.get("mask") == "keys":
        nbytes += tk
    if case.get("buckets"):
        nbytes += 2 * 2 * case["buckets"] * H
    return {"bytes": nbytes, "flops": (14 if train else 4) * H * _pairs(case) * D}


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _heads(g, dev, shape, dtype, offset_seed=None):
    """Activations [.., D]: normal, with a few channels offset for all tokens (as keys have them)."""
    x = torch.randn(shape, generator=g, device=dev, dtype=torch.float32)
    if offset_seed is not None:
        o = torch.Generator(device=dev).manual_seed(offset_seed)
        off = torch.zeros(shape[-1], device=dev)
        off[torch.randperm(shape[-1], generator=o, device=dev)[:8]] = torch.randn(8, generator=o, device=dev)
        x += off
    return x.to(DTYPES[dtype])


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(seed)
    s = {"case": case}
    if case["op"] == "bias":
        table = torch.randn((case["buckets"], case["H"]), generator=g, device=dev, dtype=torch.float32)
        s["table"] = table.to(DTYPES[case["table"]])
        if case["train"]:
            s["table"].requires_grad_(True)
            s["dbias"] = torch.randn((case["H"], case["Sq"], case["Skv"]), generator=g, device=dev,
                                     dtype=torch.float32).to(DTYPES[case["dtype"]])
        return s
    H, Hkv, D = case["H"], case["Hkv"], case["D"]
    if case["op"] == "packed":
        lens = torch.tensor([0] + _lengths(case), dtype=torch.int64)
        s["cu"] = torch.cumsum(lens, 0).to(device=dev, dtype=torch.int32)
        total = sum(_lengths(case))
        qs, ks = (total, H, D), (total, Hkv, D)
    else:
        B, Sq, Skv = case["B"], case["Sq"], case["Skv"]
        qs, ks = ((B, H, Sq, D), (B, Hkv, Skv, D)) if case["layout"] == "HND" else ((B, Sq, H, D), (B, Skv, Hkv, D))
        if case["mask"] == "keys":
            n = torch.tensor(_visible_keys(case), device=dev)
            s["mask"] = (torch.arange(Skv, device=dev) < n[:, None])[:, None, None, :]
        elif case["mask"] == "docs":
            d = torch.tensor(_documents(case), device=dev)
            s["mask"] = ((d[:, :, None] == d[:, None, :]) & (d >= 0)[:, :, None])[:, None]
        if case["buckets"]:
            table = torch.randn((case["buckets"], H), generator=g, device=dev, dtype=torch.float32)
            s["table"] = table.to(DTYPES[case["dtype"]])
    s["q"], s["k"] = _heads(g, dev, qs, case["dtype"]), _heads(g, dev, ks, case["dtype"], seed + 1)
    s["v"] = _heads(g, dev, ks, case["dtype"])
    if case.get("train", True):
        s["dout"] = _heads(g, dev, qs, case["dtype"])
        for name in ("q", "k", "v", "table"):
            if name in s:
                s[name].requires_grad_(True)
    return s


# ---- one pass -------------------------------------------------------------------------------------------------------

def _bucket(away, buckets, reach, two_sided):
    """The bucket of a key `away` tokens ahead of its query (int64): one for each small distance, then ranges whose borders
    grow evenly in the logarithm up to `reach`; two-sided, keys ahead have the second half of the buckets."""
    side = buckets // 2 if two_sided else buckets
    n = away.abs() if two_sided else (-away).clamp(min=0)
    near = side // 2
    # 64 bits, and a margin, as distances lie on the borders
    t = torch.log(n.clamp(min=1).double() / near) / math.log(reach / near) * (side - near)
    far = (near + torch.floor(t + 1e-9).long()).clamp(max=side - 1)
    b = torch.where(n < near, n, far)
    return b + (away > 0) * side if two_sided else b


def _away(Sq, Skv, dev):
    """Key position minus query position, the last query at the last key's."""
    return torch.arange(Skv, device=dev)[None, :] - (torch.arange(Sq, device=dev) + (Skv - Sq))[:, None]


def _plain_core(q, k, v, seen, bias, dout):
    """Attention of q [B, H, Sq, D] over k, v [B, Hkv, Skv, D] in 32 bits; seen: the visible pairs [B or 1, 1, Sq, Skv] or
    None; bias [H, Sq, Skv] or None.  (out, logsumexp) and, with dout, also (dq, dk, dv, dscores)."""
    B, H, Sq, D = q.shape
    Hkv, Skv = k.shape[1], k.shape[2]
    scale = D ** -0.5
    q, k, v = q.float().reshape(B, Hkv, -1, D), k.float(), v.float()  # the heads that share keys: rows behind each other
    p = (torch.matmul(q, k.transpose(2, 3)) * scale).view(B, H, Sq, Skv)
    if bias is not None:
        p += bias
    if seen is not None:
        p.masked_fill_(~seen, float("-inf"))
    top = p.amax(dim=-1, keepdim=True)
    top.masked_fill_(top == float("-inf"), 0.0)  # rows that see nothing
    p = p.sub_(top).exp_()
    total = p.sum(dim=-1, keepdim=True)
    lse = (top + torch.log(total)).squeeze(-1)
    p /= torch.where(total > 0, total, 1.0)
    rows = p.view(B, Hkv, -1, Skv)
    out = torch.matmul(rows, v).view(B, H, Sq, D)
    if dout is None:
        return out, lse
    do = dout.float().reshape(B, Hkv, -1, D)
    dv = torch.matmul(rows.transpose(2, 3), do)
    ds = torch.matmul(do, v.transpose(2, 3))
    ds -= (rows * ds).sum(dim=-1, keepdim=True)
    ds *= rows
    dq = torch.matmul(ds, k).view(B, H, Sq, D) * scale
    dk = torch.matmul(ds.transpose(2, 3), q) * scale
    return out, lse, dq, dk, dv, ds.view(B, H, Sq, Skv)


def _by_bucket(d, buckets, reach, two_sided):
    """[buckets, H]: the sums of d [H, Sq, Skv] over each bucket's pairs: along the diagonals, each in one bucket, then over
    those.  64 bits, for millions of values of both signs cancel."""
    H, Sq, Skv = d.shape
    wide = Sq + Skv - 1
    # rows last to first, each one place further right: column c holds the pairs of key - query = c - (Sq - 1)
    skewed = torch.nn.functional.pad(d.double().flip(1), (0, Sq)).flatten(1)[:, :Sq * wide].view(H, Sq, wide)
    bucket = _bucket(torch.arange(wide, device=d.device) - (Skv - 1), buckets, reach, two_sided)
    chosen = bucket[:, None] == torch.arange(buckets, device=d.device)
    return torch.mm(skewed.sum(dim=1), chosen.double()).t()


def _plain_attend(s):
    c = s["case"]
    bring = (lambda t: t) if c["layout"] == "HND" else (lambda t: t.transpose(1, 2))
    Sq, Skv = c["Sq"], c["Skv"]
    dev = s["q"].device
    seen, bias = s.get("mask"), None
    away = _away(Sq, Skv, dev) if c["causal"] or c["buckets"] else None
    if c["causal"]:
        seen = (away <= 0)[None, None] if seen is None else seen & (away <= 0)
    if c["buckets"]:
        bucket = _bucket(away, c["buckets"], c["reach"], not c["causal"])
        bias = s["table"].detach().float()[bucket].permute(2, 0, 1)
    dt = s["q"].dtype
    r = _plain_core(bring(s["q"].detach()), bring(s["k"].detach()), bring(s["v"].detach()), seen, bias,
                    bring(s["dout"]) if c["train"] else None)
    out = {"out": bring(r[0].to(dt))}
    if c["lse"]:
        out["lse"] = r[1]
    if c["train"]:
        out.update(dq=bring(r[2].to(dt)), dk=bring(r[3].to(dt)), dv=bring(r[4].to(dt)))
        if c["buckets"]:
            d = r[5].sum(dim=0, dtype=torch.float64)
            out["dtable"] = _by_bucket(d, c["buckets"], c["reach"], not c["causal"]).to(s["table"].dtype)
    return out


def _plain_packed(s):
    """The sequences side by side, padded to the longest."""
    c = s["case"]
    cu, n = s["cu"].long(), c["longest"]
    at = torch.arange(n, device=cu.device)
    real = at < (cu[1:] - cu[:-1])[:, None]
    index = (cu[:-1, None] + at).clamp(max=int(s["q"].shape[0]) - 1)
    seen = real[:, None, None, :]
    if c["causal"]:
        seen = seen & (at[None, :] <= at[:, None])

    def pad(t):
        return t.detach()[index].transpose(1, 2)

    do = pad(s["dout"]).masked_fill(~real[:, None, :, None], 0.0)  # rows behind a sequence are none
    out, _, dq, dk, dv, _ = _plain_core(pad(s["q"]), pad(s["k"]), pad(s["v"]), seen, None, do)
    dt = s["q"].dtype
    return {name: t.transpose(1, 2)[real].to(dt) for name, t in (("out", out), ("dq", dq), ("dk", dk), ("dv", dv))}


def _plain_bias(s):
    c = s["case"]
    t = s["table"].detach()
    bucket = _bucket(_away(c["Sq"], c["Skv"], t.device), c["buckets"], c["reach"], c["two_sided"])
    out = {"bias": t.float()[bucket].permute(2, 0, 1).to(DTYPES[c["dtype"]]).contiguous()}
    if c["train"]:
        out["dtable"] = _by_bucket(s["dbias"], c["buckets"], c["reach"], c["two_sided"]).to(t.dtype)
    return out


def run(state):
    s, c = state, state["case"]
    if not own:
        return {"attend": _plain_attend, "packed": _plain_packed, "bias": _plain_bias}[c["op"]](s)
    sage = _package()
    if c["op"] == "bias":
        bias = sage.relative_bias(s["table"], c["Sq"], c["Skv"], bidirectional=c["two_sided"], max_distance=c["reach"],
                                  dtype=DTYPES[c["dtype"]])
        if not c["train"]:
            return {"bias": bias}
        return {"bias": bias, "dtable": torch.autograd.grad(bias, s["table"], s["dbias"])[0]}
    if c["op"] == "packed":
        out = sage.attention_train_varlen(s["q"], s["k"], s["v"], s["cu"], s["cu"], c["longest"], c["longest"],
                                          is_causal=c["causal"])
        dq, dk, dv = torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["dout"])
        return {"out": out, "dq": dq, "dk": dk, "dv": dv}
    out = sage.attention_train(s["q"], s["k"], s["v"], tensor_layout=c["layout"], is_causal=c["causal"],
                               attn_mask=s.get("mask"), bias_table=s.get("table"), bidirectional=not c["causal"],
                               max_distance=c["reach"], return_lse=c["lse"])
    if c["lse"]:
        out, lse = out
    result = {"out": out}
    if c["lse"]:
        result["lse"] = lse
    if c["train"]:
        names = [n for n in ("q", "k", "v", "table") if n in s]
        grads = torch.autograd.grad(out, [s[n] for n in names], s["dout"])
        result.update(("d" + n, d) for n, d in zip(names, grads))
    return result


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------

def _exact_buckets(Sq, Skv, buckets, reach, two_sided):
    """By whole numbers alone: a distance n is past the t-th border where n^m >= near^(m - t) reach^t."""
    side = buckets // 2 if two_sided else buckets
    near = side // 2
    m = side - near

    def one(n):
        if n < near:
            return n
        t = 0
        while t + 1 < m and n ** m >= near ** (m - t - 1) * reach ** (t + 1):
            t += 1
        return near + t

    of = []
    for away in range(-(Skv - 1), Sq):
        n = abs(away) if two_sided else max(-away, 0)
        b = one(n) if n <= reach else side - 1
        of.append(b + side if two_sided and away > 0 else b)
    return torch.tensor(of).unfold(0, Skv, 1).flip(0)  # the last query's row comes first in `of`


def _exact_one(q, k, v, hidden, bias, dout):
    """One head: q [Sq, D], k, v [Skv, D], 64 bits."""
    x = torch.mm(q, k.t()) / math.sqrt(q.shape[1])
    if bias is not None:
        x = x + bias
    if hidden is not None:
        x = x.masked_fill(hidden, -math.inf)
    lse = torch.logsumexp(x, dim=1)
    p = torch.exp(x - torch.where(torch.isinf(lse), torch.zeros_like(lse), lse)[:, None])
    out = torch.mm(p, v)
    if dout is None:
        return out, lse
    delta = (dout * out).sum(dim=1, keepdim=True)
    ds = p * (torch.mm(dout, v.t()) - delta)
    return out, lse, torch.mm(ds, k) / math.sqrt(q.shape[1]), torch.mm(ds.t(), q) / math.sqrt(q.shape[1]), torch.mm(p.t(), dout), ds


def _exact_attend(case, s):
    lay = case["layout"]
    q, k, v, do = (None if s.get(n) is None else s[n].detach() if lay == "HND" else s[n].detach().transpose(1, 2)
                   for n in ("q", "k", "v", "dout"))
    B, H, Hkv, Sq, Skv = (case[x] for x in ("B", "H", "Hkv", "Sq", "Skv"))
    dev = q.device
    res = {"out": torch.zeros(q.shape, dtype=torch.float64, device=dev)}
    if case["lse"]:
        res["lse"] = torch.zeros(q.shape[:3], dtype=torch.float64, device=dev)
    if case["train"]:
        for n, t in (("dq", q), ("dk", k), ("dv", v)):
            res[n] = torch.zeros(t.shape, dtype=torch.float64, device=dev)
    later = torch.ones((Sq, Skv), dtype=torch.bool, device=dev).triu(Skv - Sq + 1) if case["causal"] else None
    bucket = None
    if case["buckets"]:
        bucket = _exact_buckets(Sq, Skv, case["buckets"], case["reach"], not case["causal"]).to(dev)
        table = s["table"].detach().double()
        if case["train"]:
            res["dtable"] = torch.zeros(table.shape, dtype=torch.float64, device=dev)
    for b in range(B):
        hidden = later
        if case["mask"]:
            hidden = ~s["mask"][b, 0].expand(Sq, Skv)
            if later is not None:
                hidden = hidden | later
        for h in range(H):
            j = h // (H // Hkv)
            r = _exact_one(q[b, h].double(), k[b, j].double(), v[b, j].double(), hidden,
                           None if bucket is None else table[:, h][bucket], None if do is None else do[b, h].double())
            res["out"][b, h] = r[0]
            if case["lse"]:
                res["lse"][b, h] = r[1]
            if case["train"]:
                res["dq"][b, h] = r[2]
                res["dk"][b, j] += r[3]
                res["dv"][b, j] += r[4]
                if bucket is not None:
                    res["dtable"][:, h] += torch.bincount(bucket.flatten(), weights=r[5].flatten(), minlength=case["buckets"])
    return {n: t if lay == "HND" or t.dim() != 4 else t.transpose(1, 2) for n, t in res.items()}


def _exact_packed(case, s):
    q, k, v, do = (s[n].detach() for n in ("q", "k", "v", "dout"))
    res = {n: torch.zeros(t.shape, dtype=torch.float64, device=q.device) for n, t in (("out", q), ("dq", q), ("dk", k), ("dv", v))}
    at = 0
    for n in _lengths(case):
        rows = slice(at, at + n)
        later = torch.ones((n, n), dtype=torch.bool, device=q.device).triu(1) if case["causal"] else None
        for h in range(case["H"]):
            j = h // (case["H"] // case["Hkv"])
            out, _, dq, dk, dv, _ = _exact_one(q[rows, h].double(), k[rows, j].double(), v[rows, j].double(), later, None,
                                               do[rows, h].double())
            res["out"][rows, h], res["dq"][rows, h] = out, dq
            res["dk"][rows, j] += dk
            res["dv"][rows, j] += dv
        at += n
    return res


def _exact_bias(case, s):
    table = s["table"].detach().double()
    bucket = _exact_buckets(case["Sq"], case["Skv"], case["buckets"], case["reach"], case["two_sided"]).to(table.device)
    res = {"bias": torch.stack([table[:, h][bucket] for h in range(case["H"])])}
    if case["train"]:
        res["dtable"] = torch.stack([torch.bincount(bucket.flatten(), weights=s["dbias"][h].double().flatten(),
                                                    minlength=case["buckets"]) for h in range(case["H"])], dim=1)
    return res


def exact(case, seed):
    return {"attend": _exact_attend, "packed": _exact_packed, "bias": _exact_bias}[case["op"]](case, prepare(case, seed))
