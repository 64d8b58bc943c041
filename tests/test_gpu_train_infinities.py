"""A query of attention_train that sees an infinity or a NaN, in itself, in a key, a value or its gradient, is NaN, whatever sign the
scores get by it: not a query that sees nothing, and no number.  The others keep their bits."""
import math

import pytest
import torch

import cdna4_sage
from test_gpu_train import _draw, _run

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16
BAD = [math.nan, math.inf, -math.inf]


def _signs(q, k, channel):
    """Queries and keys of one sign each in a channel, so that an infinity there gives all scores one sign."""
    q[..., channel] = q[..., channel].abs() + 0.5
    k[..., channel] = -k[..., channel].abs() - 0.5


def _check(want, got, rows, out_rows, seen, exact):
    """rows: those with NaN gradients; out_rows: with NaN outputs; seen [Sq, Skv]: what they see."""
    assert bool(torch.isnan(got[0][:, :, out_rows]).all()) and torch.equal(got[0][:, :, ~out_rows], want[0][:, :, ~out_rows])
    assert bool(torch.isnan(got[1][:, :, out_rows]).all()) and torch.equal(got[1][:, :, ~out_rows], want[1][:, :, ~out_rows])
    touched = (seen & rows[:, None]).any(0)
    for a, b, nan in ((got[2][0], want[2][0], rows), (got[2][1], want[2][1], touched), (got[2][2], want[2][2], touched)):
        assert bool(torch.isnan(a[:, :, nan]).all())
        a, b = a[:, :, ~nan], b[:, :, ~nan]
        if exact:
            assert torch.equal(a, b)
        else:      # (fp16's gradients are held times a power of two of the largest finite rows, which may be others now)
            assert bool(torch.isfinite(a).all())
            assert not a.numel() or float((a.float() - b.float()).abs().max()) <= 2.0 ** -9 * float(b.abs().max())


@pytest.mark.parametrize("value", BAD)
@pytest.mark.parametrize("D,dtype,form", [(64, BF, "causal"), (96, HF, "causal"), (128, BF, "mask"), (128, HF, "bias"), (256, BF, "causal"),
                                          (256, HF, "mask")])
def test_one_infinity(dev, D, dtype, form, value):
    S, H = 200, 2
    seen = torch.ones(S, S, dtype=torch.bool).tril()
    if form == "mask":
        seen[:, 5] = False
        seen[150] = False
    for at in (0, 64, 127, S - 1):
        for signed in (True, False):
            q, k, v, do = _draw(1, H, H, S, S, D, dtype, seed=17)
            channel = 11
            if signed:
                _signs(q, k, channel)
            kw = {"is_causal": True}
            if form == "mask":
                kw = {"attn_mask": seen.to(dev)}
            if form == "bias":
                kw["table"] = torch.randn(16, H, generator=torch.Generator().manual_seed(18)).to(dtype)
                kw["max_distance"] = 40
            want = _run(dev, q, k, v, do, **kw)
            for where in ("q", "k", "v", "do"):
                ts = {n: t.clone() for n, t in dict(q=q, k=k, v=v, do=do).items()}
                ts[where][:, :, at, channel] = value
                got = _run(dev, *ts.values(), **kw)
                rows = torch.zeros(S, dtype=torch.bool)
                if where in ("q", "do"):
                    rows[at] = True
                else:
                    rows = seen[:, at].clone()
                out_rows = rows if where != "do" else torch.zeros(S, dtype=torch.bool)
                _check(want, got, rows, out_rows, seen, dtype == BF or where in ("q", "k"))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("Skv", [1, 65])
def test_a_single_query(dev, dtype, Skv):
    """Also over one key, where a score of -inf is all that there is."""
    for value in BAD:
        for where in range(4):
            ts = _draw(2, 3, 3, 1, Skv, 64, dtype, seed=19)
            _signs(ts[0], ts[1], 3)
            ts[where][0, 1, 0, 3] = value
            out, lse, grads = _run(dev, *ts)
            one = torch.zeros(2, 3, 1, dtype=torch.bool)
            one[0, 1] = True
            if where < 3:
                assert torch.equal(torch.isnan(lse.cpu()), one) and torch.equal(torch.isnan(out.cpu()).all(-1), one)
                assert torch.equal(torch.isnan(out.cpu()).any(-1), one)
            for g in grads:
                nan = torch.isnan(g.cpu())
                assert bool(nan[0, 1].all()) and not bool(nan[1].any()) and not bool(nan[0, [0, 2]].any())


@pytest.mark.parametrize("D,dtype", [(64, BF), (128, HF), (256, BF)])
def test_keys_of_either_infinity_in_packed_sequences(dev, D, dtype):
    """A key whose scores are -inf for every query, and one that gives both signs: a query's result is its own either way."""
    lens = [3, 130, 77]
    cu = torch.tensor([0, 3, 133, 210], dtype=torch.int32, device=dev)
    T, H = 210, 2
    for both in (False, True):
        q, k, v, do = (t[0].transpose(0, 1).contiguous() for t in _draw(1, H, H, T, T, D, dtype, seed=23))
        q[..., 7] = q[..., 7].abs() + 0.5
        if both:
            q[100, :, 7] = -1.0
        k[40, :, 7] = -math.inf                  # of the second sequence
        leaves = [t.to(dev).requires_grad_() for t in (q, k, v)]
        out = cdna4_sage.attention_train_varlen(*leaves, cu, cu)
        grads = torch.autograd.grad(out, leaves, do.to(dev))
        second = torch.zeros(T, dtype=torch.bool)
        second[lens[0]:lens[0] + lens[1]] = True
        for t in (out, *grads):
            assert bool(torch.isnan(t[second.to(dev)]).all()) and bool(torch.isfinite(t[~second.to(dev)]).all())


def test_scores_that_overflow(dev):
    """Finite inputs whose scores pass float32 downwards: beside other keys their weight is 0; where nothing else is seen, NaN."""
    S, D = 100, 64
    q, k, v, do = _draw(1, 1, 1, S, S, D, BF, seed=29)
    q[..., 0], k[..., 0] = 0.0, 0.0
    far = torch.arange(S) % 3 == 1
    q[:, :, :, 0] = 2.0 ** 80
    hide = [t.clone() for t in (q, k)]
    k[:, :, far, 0] = -(2.0 ** 80)
    mask = ~far.expand(S, S)
    want = _run(dev, *hide, v, do, attn_mask=mask.to(dev))
    got = _run(dev, q, k, v, do, attn_mask=torch.ones_like(mask).to(dev))      # (by the same kernel)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    assert bool(torch.isfinite(_run(dev, q, k, v, do)[0]).all())
    k[:, :, :, 0] = -(2.0 ** 80)
    for kw in ({}, {"is_causal": True}, {"attn_mask": mask.to(dev)}):
        out, lse, _ = _run(dev, q, k, v, do, **kw)
        sees = torch.ones(S, dtype=torch.bool)
        assert bool(torch.isnan(out[:, :, sees]).all()) and bool(torch.isnan(lse[:, :, sees]).all())


def test_a_bias_of_minus_infinity_hides(dev):
    """Learned values of -inf leave their pairs out, as a mask does, and rows of nothing else are 0."""
    S, H = 150, 2
    q, k, v, do = _draw(1, H, H, S, S, 64, BF, seed=31)
    table = torch.zeros(8, H)
    table[4:] = -math.inf                        # keys ahead of their query
    out, lse, grads = _run(dev, q, k, v, do, table=table, max_distance=20)
    want = _run(dev, q, k, v, do, is_causal=True)
    assert bool(torch.isfinite(out).all()) and torch.equal(out, want[0])
    for a, b in zip(grads[:3], want[2]):
        assert bool(torch.isfinite(a).all()) and float((a.float() - b.float()).abs().max()) <= 2.0 ** -7 * float(b.abs().max())
    out, lse, grads = _run(dev, q, k, v, do, table=torch.full((8, H), -math.inf), max_distance=20)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all()) and all(bool((g == 0).all()) for g in grads)
