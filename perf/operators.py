"""The decoding operators of this package as cases that can be prepared, run, timed and checked: rotary positions
(``cdna4_sage.rope``, forward and backward), the quantized key / value cache (``cdna4_sage.cache_write`` and
``cdna4_sage.cache_read``) and the attention of new tokens over it (``cdna4_sage.cache_attention``).

``run`` computes their plain form from elementary torch operations, or calls the package where ``own`` is true.  Head
counts and head dims are those of cdna4_sage.configs and of the tests; lengths and batches are generic.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
LARGEST = {"int8": 127.0, "e4m3": 448.0}  # the code of a row's largest magnitude


def _package():
    packages = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rdna4-sageattention_amd")
    if packages not in sys.path:
        sys.path.insert(0, packages)
    import cdna4_sage

    return cdna4_sage


# ---- the cases ------------------------------------------------------------------------------------------------------

def _rope(B, S, H, Hk, D, rot, layout, dtype, interleaved=False, far=0, stretch=1.0, train=False):
    """far: the first position; stretch: the factor by which the low frequencies are slowed (long contexts)."""
    return {"op": "rope", "B": B, "S": S, "H": H, "Hk": Hk, "D": D, "rot": rot, "layout": layout, "dtype": dtype,
            "interleaved": interleaved, "far": far, "stretch": stretch, "train": train}


def _write(tokens, Hkv, D, page, code, dtype, padding=0):
    """padding: of the tokens, how many have no slot."""
    return {"op": "write", "tokens": tokens, "Hkv": Hkv, "D": D, "page": page, "code": code, "dtype": dtype,
            "padding": padding}


def _read(tokens, Hkv, D, page, code, dtype):
    return {"op": "read", "tokens": tokens, "Hkv": Hkv, "D": D, "page": page, "code": code, "dtype": dtype}


def _attend(B, T, H, Hkv, D, shortest, longest, page, code, layout, dtype, tree=False, lse=False):
    """B sequences of shortest to longest cached tokens (the T new ones among them)."""
    return {"op": "attend", "B": B, "T": T, "H": H, "Hkv": Hkv, "D": D, "shortest": shortest, "longest": longest,
            "page": page, "code": code, "layout": layout, "dtype": dtype, "tree": tree, "lse": lse}


def listed():
    return [
        # one decoding step of a few sequences far into a long context: where launches and the host's work count
        dict(_rope(4, 1, 32, 8, 128, 128, "NHD", "bf16", far=131072, stretch=8.0), name="rope_step"),
        # two prompts before the causal attention of configuration 5a
        dict(_rope(2, 8192, 32, 8, 128, 128, "HND", "bf16"), name="rope_prompt"),
        # a training step: half of every head rotated in interleaved pairs, forward and backward, odd length
        dict(_rope(3, 2047, 16, 4, 64, 32, "NHD", "f16", interleaved=True, train=True), name="rope_train"),
        # the new token of every sequence of a batch
        dict(_write(24, 8, 128, 16, "int8", "bf16"), name="write_step"),
        # padded prompts, some tokens without a slot
        dict(_write(18002, 8, 128, 64, "e4m3", "bf16", padding=1777), name="write_prompt"),
        # the prefix of one sequence, for a prompt chunk's attention
        dict(_read(1501, 4, 96, 32, "e4m3", "f16"), name="read_prefix"),
        # every key of a long context
        dict(_read(130000, 8, 128, 16, "int8", "bf16"), name="read_long"),
        # one sequence, one token: the latency of decoding
        dict(_attend(1, 1, 32, 8, 128, 1000, 1000, 16, "int8", "HND", "bf16"), name="decode_one"),
        # a ragged batch of the smaller heads, with the logsumexp
        dict(_attend(48, 1, 16, 4, 64, 77, 8192, 32, "e4m3", "NHD", "f16", lse=True), name="decode_batch"),
        # few sequences with long contexts: the cache is gigabytes
        dict(_attend(6, 1, 32, 8, 128, 100001, 131072, 64, "int8", "NHD", "bf16"), name="decode_long"),
        # a small tree of drafted tokens, every head with keys of its own
        dict(_attend(1, 7, 12, 12, 256, 4360, 4360, 128, "e4m3", "HND", "f16", tree=True), name="tree_one"),
        # a batch with a larger tree each, ragged lengths
        dict(_attend(16, 33, 32, 8, 128, 501, 9001, 16, "int8", "NHD", "bf16", tree=True), name="tree_batch"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        kind = rng.choice(["rope", "rope", "write", "read", "decode", "decode", "tree", "tree", "chunk"])
        dtype, code = rng.choice(["bf16", "bf16", "f16"]), rng.choice(["int8", "e4m3"])
        layout, page = rng.choice(["HND", "NHD"]), rng.choice([16, 16, 32, 64, 128, 256])
        D, Hkv = rng.choice([64, 96, 128, 128, 256]), rng.choice([1, 2, 4, 8, 8, 10, 12, 24])
        H = Hkv * rng.choice([1, 2, 4, 4, 5, 8])
        if H > 64:
            continue
        if kind == "rope":
            rot = rng.choice([D, D, D // 2, D // 4])
            B, S = (rng.randint(1, 64), 1) if rng.random() < 0.3 else (rng.randint(1, 4), _log_int(rng, 5, 9000))
            c = _rope(B, S, H, Hkv, D, rot, layout, dtype, interleaved=rng.random() < 0.5,
                      far=rng.choice([0, 0, 4096, 500000]), stretch=rng.choice([1.0, 1.0, 4.0, 16.0]),
                      train=S > 1 and rng.random() < 0.5)
        elif kind == "write":
            tokens = _log_int(rng, 1, 40000)
            c = _write(tokens, Hkv, D, page, code, dtype, padding=rng.choice([0, tokens // 9]))
        elif kind == "read":
            c = _read(_log_int(rng, 17, 100000), Hkv, D, page, code, dtype)
        else:
            B = _log_int(rng, 1, 64)
            T = 1 if kind == "decode" else rng.randint(2, 64) if kind == "tree" else _log_int(rng, 2, 200)
            longest = _log_int(rng, max(64, T), 60000)
            c = _attend(B, T, H, Hkv, D, rng.randint(T, longest), longest, page, code, layout, dtype,
                        tree=kind == "tree", lse=rng.random() < 0.3)
            # the plain form holds its scores and unpacked keys in 32 bits
            if B * H * T * longest > 1 << 30 or B * Hkv * longest * D > 1 << 29:
                continue
        w, most = work(c), work(_attend(6, 1, 32, 8, 128, 100001, 131072, 64, "int8", "NHD", "bf16"))
        if max(w["bytes"], w["flops"] / 50) <= max(most["bytes"], most["flops"] / 50):
            return c


def _lengths(case):
    """Cached tokens of every sequence: spread from the shortest to the longest, in no order."""
    B, lo, hi = case["B"], case["shortest"], case["longest"]
    if B == 1:
        return [hi]
    return [lo + (hi - lo) * ((b * 7 + 3) % B) // (B - 1) for b in range(B)]


def work(case):
    """Inputs read once and outputs written once; the products of the visible (query, key) pairs."""
    if case["op"] == "rope":
        n = case["B"] * case["S"] * (case["H"] + case["Hk"])
        passes = 2 if case["train"] else 1
        pairs = case["B"] * case["S"] * case["rot"] // 2
        return {"bytes": passes * (4 * n * case["D"] + 8 * case["B"] * case["S"]),
                "flops": passes * (3 * n * case["rot"] + 2 * pairs)}
    if case["op"] in ("write", "read"):
        # (16-bit values, codes and a scale) of K and V, and a slot for every token
        rows = 2 * (case["tokens"] - case.get("padding", 0)) * case["Hkv"]
        return {"bytes": rows * (3 * case["D"] + 4) + 8 * case["tokens"], "flops": 3 * rows * case["D"]}
    T, lens = case["T"], _lengths(case)
    pairs = sum(T * (n - T) + T * (T + 1) // 2 for n in lens)
    nbytes = sum(lens) * case["Hkv"] * (2 * case["D"] + 8) + 4 * case["B"] * T * case["H"] * case["D"]
    nbytes += sum(-(-n // case["page"]) for n in lens) * 4 + 4 * case["B"]
    if case["tree"]:
        nbytes += case["B"] * T * T
    if case["lse"]:
        nbytes += 4 * case["B"] * T * case["H"]
    return {"bytes": nbytes, "flops": 4 * case["H"] * pairs * case["D"]}


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _frequencies(case, dev):
    """Radians per position of every channel pair.  Pairs that turn less than once over the first 4096 positions are
    slowed by the stretch, those that turn more than 32 times are kept, in between a blend."""
    i = torch.arange(case["rot"] // 2, device=dev, dtype=torch.float64)
    f = 10000.0 ** (-2.0 * i / case["rot"])
    turns = 4096.0 * f / (2.0 * math.pi)
    keep = ((turns - 1.0) / 31.0).clamp(0.0, 1.0)
    return f * keep + f / case["stretch"] * (1.0 - keep), 0.1 * math.log(case["stretch"]) + 1.0


def _heads(g, dev, shape, dtype, offset_seed=None):
    """Activations [.., D]: normal, with a few channels offset for all tokens (as keys have them)."""
    x = torch.randn(shape, generator=g, device=dev, dtype=torch.float32)
    if offset_seed is not None:
        o = torch.Generator(device=dev).manual_seed(offset_seed)
        off = torch.zeros(shape[-1], device=dev)
        off[torch.randperm(shape[-1], generator=o, device=dev)[:8]] = torch.randn(8, generator=o, device=dev) * 1.7
        x += off
    return x.to(dtype)


def _quantized(x, code):
    """Codes and scales of the rows of x: the largest magnitude of a row takes the largest code."""
    a = x.abs().amax(dim=-1, keepdim=True).double()
    y = x.double() * LARGEST[code] / torch.where(a > 0, a, 1.0)  # 64 bits: rows hold quotients on a rounding border
    y = torch.round(y).to(torch.int8) if code == "int8" else y.float().to(torch.float8_e4m3fn)
    return y, (a / LARGEST[code]).float().squeeze(-1)


def _pool(case, seed, pages, dev, g):
    """A cache of random keys and values, quantized page by page."""
    shape = (pages, case["Hkv"], case["page"])
    out = {"code": case["code"]}
    for name in ("k", "v"):
        codes = torch.empty(shape + (case["D"],), device=dev, dtype=CODES[case["code"]])
        scale = torch.empty(shape, device=dev, dtype=torch.float32)
        step = max(1, (1 << 27) // (shape[1] * shape[2] * case["D"]))
        for p in range(0, pages, step):
            n = min(step, pages - p)
            x = _heads(g, dev, (n,) + shape[1:] + (case["D"],), torch.bfloat16, seed + 1 if name == "k" else None)
            codes[p:p + n], scale[p:p + n] = _quantized(x, case["code"])
        out[name], out[name + "s"] = codes, scale
    return out


def _slots(case, g, dev, pages):
    """A slot of its own for every token: consecutive rows of pages in no order."""
    order = torch.randperm(pages, generator=g, device=dev)
    t = torch.arange(case["tokens"], device=dev)
    return order[t // case["page"]] * case["page"] + t % case["page"]


def _tree(case, seed):
    """Which of the new tokens each one sees: itself and its ancestors in a random tree per sequence."""
    T = case["T"]
    g = torch.Generator().manual_seed(seed)
    r = torch.rand((case["B"], T), generator=g)
    m = torch.zeros((case["B"], T, T), dtype=torch.bool)
    rows = torch.arange(case["B"])
    for i in range(T):
        if i:
            m[:, i] = m[rows, (r[:, i] * i).long()]
        m[:, i, i] = True
    return m


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(seed)
    s = {"case": case}
    if case["op"] == "rope":
        B, S, D, dt = case["B"], case["S"], case["D"], DTYPES[case["dtype"]]
        for name, H in (("q", case["H"]), ("k", case["Hk"])):
            shape = (B, H, S, D) if case["layout"] == "HND" else (B, S, H, D)
            s[name] = _heads(g, dev, shape, dt)
            if case["train"]:
                s["d" + name] = _heads(g, dev, shape, dt)
                s[name].requires_grad_(True)
        start = torch.randint(0, 64, (B, 1), generator=g, device=dev) + case["far"]
        s["positions"] = start + torch.arange(S, device=dev)[None, :]
        s["freqs"], s["factor"] = _frequencies(case, dev)
    elif case["op"] == "write":
        pages = -(-case["tokens"] // case["page"]) + 3
        shape = (pages, case["Hkv"], case["page"])
        for name in ("k", "v"):
            s[name] = _heads(g, dev, (case["tokens"], case["Hkv"], case["D"]), DTYPES[case["dtype"]],
                             seed + 1 if name == "k" else None)
            s["c" + name] = torch.zeros(shape + (case["D"],), device=dev, dtype=CODES[case["code"]])
            s["s" + name] = torch.zeros(shape, device=dev, dtype=torch.float32)
        s["slots"] = _slots(case, g, dev, pages)
        if case["padding"]:
            s["slots"][torch.randperm(case["tokens"], generator=g, device=dev)[:case["padding"]]] = -1
    elif case["op"] == "read":
        pages = -(-case["tokens"] // case["page"]) + 3
        s["pool"] = _pool(case, seed, pages, dev, g)
        s["slots"] = _slots(case, g, dev, pages)
    else:
        B, T, H, D = case["B"], case["T"], case["H"], case["D"]
        lens = _lengths(case)
        need = [-(-n // case["page"]) for n in lens]
        pages = sum(need) + 3
        s["pool"] = _pool(case, seed, pages, dev, g)
        order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
        table = torch.full((B, max(need)), -1, dtype=torch.int32)
        at = 0
        order = order.cpu()
        for b, n in enumerate(need):
            table[b, :n] = order[at:at + n]
            at += n
        s["table"] = table.to(dev)
        s["lengths"] = torch.tensor(lens, dtype=torch.int32, device=dev)
        s["q"] = _heads(g, dev, (B, H, T, D) if case["layout"] == "HND" else (B, T, H, D), DTYPES[case["dtype"]])
        s["tree"] = _tree(case, seed).to(dev) if case["tree"] else None
    return s


# ---- one pass -------------------------------------------------------------------------------------------------------

def _rotate(x, cos, sin, interleaved, rot):
    """cos / sin [B, .., rot / 2] against x [B, .., D], in 32 bits, rounded once."""
    y = x.float()
    if interleaved:
        a, b = y[..., 0:rot:2], y[..., 1:rot:2]
        r = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = y[..., :rot // 2], y[..., rot // 2:rot]
        r = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((r, y[..., rot:]), dim=-1).to(x.dtype)


def _plain_rope(s):
    c = s["case"]
    angle = s["positions"].double()[:, :, None] * s["freqs"]  # 64 bits: far positions turn many times
    cos, sin = (torch.cos(angle) * s["factor"]).float(), (torch.sin(angle) * s["factor"]).float()
    axis = 1 if c["layout"] == "HND" else 2
    cos, sin = cos.unsqueeze(axis), sin.unsqueeze(axis)
    out = {"q": _rotate(s["q"].detach(), cos, sin, c["interleaved"], c["rot"]),
           "k": _rotate(s["k"].detach(), cos, sin, c["interleaved"], c["rot"])}
    if c["train"]:
        # the rotation's transpose turns back
        out["dq"] = _rotate(s["dq"], cos, -sin, c["interleaved"], c["rot"])
        out["dk"] = _rotate(s["dk"], cos, -sin, c["interleaved"], c["rot"])
    return out


def _plain_write(s):
    c = s["case"]
    at = torch.nonzero(s["slots"] >= 0).squeeze(1)
    page, row = s["slots"][at] // c["page"], s["slots"][at] % c["page"]
    kc, ks = _quantized(s["k"][at], c["code"])
    vc, vs = _quantized(s["v"][at], c["code"])
    s["ck"].view(torch.int8)[page, :, row] = kc.view(torch.int8)
    s["cv"].view(torch.int8)[page, :, row] = vc.view(torch.int8)
    s["sk"][page, :, row] = ks
    s["sv"][page, :, row] = vs
    return {"ck": s["ck"], "cv": s["cv"], "sk": s["sk"], "sv": s["sv"]}


def _values(codes, scale, page, row, dtype):
    x = codes.view(torch.int8)[page, :, row].view(codes.dtype)
    return (x.float() * scale[page, :, row].unsqueeze(-1)).to(dtype)


def _plain_read(s):
    c, p = s["case"], s["pool"]
    page, row = s["slots"] // c["page"], s["slots"] % c["page"]
    return {"k": _values(p["k"], p["ks"], page, row, DTYPES[c["dtype"]]),
            "v": _values(p["v"], p["vs"], page, row, DTYPES[c["dtype"]])}


def _gathered(codes, scale, table):
    """[B, Hkv, keys, D] in 32 bits."""
    x = codes.view(torch.int8)[table].view(codes.dtype).float() * scale[table].unsqueeze(-1)
    B, P, H, n, D = x.shape
    return x.transpose(1, 2).reshape(B, H, P * n, D)


def _plain_attend(s):
    c, p = s["case"], s["pool"]
    q = s["q"] if c["layout"] == "HND" else s["q"].transpose(1, 2)
    B, H, T, D = q.shape
    Hkv, table = c["Hkv"], s["table"].clamp(min=0).long()
    k, v = _gathered(p["k"], p["ks"], table), _gathered(p["v"], p["vs"], table)
    score = torch.matmul(q.float().reshape(B, Hkv, H // Hkv * T, D), k.transpose(2, 3)) * D ** -0.5
    score = score.view(B, H, T, -1)
    key = torch.arange(score.shape[-1], device=q.device)
    node = key[None, :] - (s["lengths"][:, None] - T)  # of a key among the new tokens
    if s["tree"] is None:
        seen = node[:, None, :] <= torch.arange(T, device=q.device)[None, :, None]
    else:
        inside = (node >= 0) & (node < T)
        at = node.clamp(0, T - 1)[:, None, :].expand(B, T, key.numel())
        seen = (node < 0)[:, None, :] | (inside[:, None, :] & torch.gather(s["tree"], 2, at))
    score.masked_fill_(~seen[:, None], float("-inf"))
    top = score.amax(dim=-1, keepdim=True)
    e = torch.exp(score - top)
    total = e.sum(dim=-1, keepdim=True)
    out = torch.matmul(e.view(B, Hkv, -1, key.numel()), v).view(B, H, T, D) / total
    out = out.to(q.dtype)
    out = {"out": out if c["layout"] == "HND" else out.transpose(1, 2)}
    if c["lse"]:
        out["lse"] = (top + torch.log(total)).squeeze(-1)
    return out


def run(state):
    s, c = state, state["case"]
    if not own:
        return {"rope": _plain_rope, "write": _plain_write, "read": _plain_read, "attend": _plain_attend}[c["op"]](s)
    sage = _package()
    if c["op"] == "rope":
        q, k = sage.rope(s["q"], s["k"], s["positions"], s["freqs"], tensor_layout=c["layout"],
                         interleaved=c["interleaved"], factor=s["factor"])
        if not c["train"]:
            return {"q": q, "k": k}
        dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
        return {"q": q, "k": k, "dq": dq, "dk": dk}
    if c["op"] == "write":
        sage.cache_write(sage.KVCache(s["ck"], s["cv"], s["sk"], s["sv"]), s["k"], s["v"], s["slots"])
        return {"ck": s["ck"], "cv": s["cv"], "sk": s["sk"], "sv": s["sv"]}
    p = s["pool"]
    cache = sage.KVCache(p["k"], p["v"], p["ks"], p["vs"])
    if c["op"] == "read":
        k, v = sage.cache_read(cache, s["slots"], DTYPES[c["dtype"]])
        return {"k": k, "v": v}
    out = sage.cache_attention(s["q"], cache, s["table"], s["lengths"], tensor_layout=c["layout"],
                               tree_mask=s["tree"], return_lse=c["lse"])
    return {"out": out[0], "lse": out[1]} if c["lse"] else {"out": out}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------

def _exact_rope(case, s):
    """Every pair as a complex number, turned by e^(i angle)."""
    angle = s["positions"].to(torch.float64).unsqueeze(-1) * s["freqs"]
    turn = torch.polar(torch.full_like(angle, s["factor"]), angle)
    turn = turn.unsqueeze(1 if case["layout"] == "HND" else 2)
    half = case["rot"] // 2

    def turned(x, w):
        x = x.detach().double()
        out = x.clone()
        a = x[..., :case["rot"]]
        if case["interleaved"]:
            z = torch.view_as_complex(a.unflatten(-1, (half, 2)).contiguous()) * w
            out[..., 0:case["rot"]:2], out[..., 1:case["rot"]:2] = z.real, z.imag
        else:
            z = torch.complex(a[..., :half].contiguous(), a[..., half:].contiguous()) * w
            out[..., :half], out[..., half:case["rot"]] = z.real, z.imag
        return out

    out = {"q": turned(s["q"], turn), "k": turned(s["k"], turn)}
    if case["train"]:
        out["dq"], out["dk"] = turned(s["dq"], turn.conj()), turned(s["dk"], turn.conj())
    return out


def _nearest(y, code):
    """The nearest code's value to y in [-largest, largest], ties to the even one."""
    if code == "int8":
        return torch.round(y)
    # e4m3: steps of an eighth of the power of two below, of 2^-9 below 2^-6
    power = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6)))
    step = torch.exp2(power - 3.0)
    return torch.round(y / step) * step


def _exact_write(case, s):
    top = LARGEST[case["code"]]
    out = {"ck": torch.zeros(s["ck"].shape, dtype=torch.float64, device=s["ck"].device),
           "cv": torch.zeros(s["cv"].shape, dtype=torch.float64, device=s["cv"].device),
           "sk": s["sk"].double(), "sv": s["sv"].double()}
    has = s["slots"] >= 0
    for name in ("k", "v"):
        x = s[name][has].to(torch.float64)
        a = torch.linalg.vector_norm(x, ord=float("inf"), dim=2)
        page = torch.div(s["slots"][has], case["page"], rounding_mode="floor")
        row = s["slots"][has] - page * case["page"]
        out["c" + name][page, :, row] = _nearest(x * top / a.unsqueeze(2), case["code"])
        out["s" + name][page, :, row] = a / top
    if case["code"] == "int8":
        out["ck"], out["cv"] = out["ck"].to(torch.int8), out["cv"].to(torch.int8)
    return out


def _exact_read(case, s):
    out, p = {}, s["pool"]
    for name in ("k", "v"):
        rows = p[name].view(torch.int8).transpose(1, 2).flatten(0, 1)  # [slot, head, channel]
        scale = p[name + "s"].transpose(1, 2).flatten(0, 1)
        x = rows.index_select(0, s["slots"]).view(p[name].dtype).to(torch.float64)
        out[name] = x * scale.index_select(0, s["slots"]).double().unsqueeze(2)
    return out


def _exact_attend(case, s):
    """Sequence by sequence and kv head by kv head."""
    B, T, H, Hkv, D, n = (case[x] for x in ("B", "T", "H", "Hkv", "D", "page"))
    q = s["q"] if case["layout"] == "HND" else s["q"].transpose(1, 2)
    p, dev = s["pool"], s["q"].device
    out = torch.empty((B, H, T, D), dtype=torch.float64, device=dev)
    lse = torch.empty((B, H, T), dtype=torch.float64, device=dev)
    for b, length in enumerate(_lengths(case)):
        pages = s["table"][b, :-(-length // n)].long()
        new = torch.ones((T, T), dtype=torch.bool, device=dev).tril() if s["tree"] is None else s["tree"][b]
        bias = torch.zeros((T, length), dtype=torch.float64, device=dev)
        bias[:, length - T:].masked_fill_(~new, float("-inf"))
        for h in range(Hkv):
            kv = []
            for name in ("k", "v"):
                codes = p[name][:, h].view(torch.int8)[pages].view(p[name].dtype).to(torch.float64)
                kv.append((codes * p[name + "s"][:, h][pages].double().unsqueeze(-1)).reshape(-1, D)[:length])
            for i in range(h * (H // Hkv), (h + 1) * (H // Hkv)):
                x = torch.mm(q[b, i].double(), kv[0].t()) / math.sqrt(D) + bias
                out[b, i] = torch.mm(torch.softmax(x, dim=1), kv[1])
                lse[b, i] = torch.logsumexp(x, dim=1)
    out = {"out": out if case["layout"] == "HND" else out.transpose(1, 2)}
    if case["lse"]:
        out["lse"] = lse
    return out


def exact(case, seed):
    state = prepare(case, seed)
    return {"rope": _exact_rope, "write": _exact_write, "read": _exact_read, "attend": _exact_attend}[case["op"]](
        case, state)
