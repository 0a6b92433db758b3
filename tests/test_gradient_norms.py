"""bf16 gradients of attention over selected blocks, head by head: the 2-norm of their error is what the documented roundings make it.

The bounds of single values have to allow the worst case of every rounding at once, which a gradient without part of a term can stay within.  Here roundings
are what they are, independent: one is uniform over a step of the type, at most 2^-8 of the value to either side, so that its square is 2^-16 / 3 of
the value's on average, or less.  Rounded are the results, out among them, from which delta is made; P and dS as factors of the products.  What float32 adds is a thousandth of
that.  The error's norm over a head, thousands of values of hundreds of rows, is near its mean, so 1.25 times the mean is a limit; steps of
values below a power of two being finer, about 0.75 of it is expected."""
import math

import pytest
import torch

from tests.helpers import dev
from tests.test_selected_attention import _mask, _run

SHAPES = [  # B, Lq, Lkv, H, Hkv, D, block, S, ragged
    (1, 300, 500, 8, 2, 128, 64, 6, False), (1, 1170, 390, 12, 4, 128, 128, 4, False), (2, 300, 500, 4, 4, 128, 128, 4, False), (1, 1000, 1100, 12, 12, 128, 64, 9, True),
    (1, 1500, 1400, 24, 24, 128, 64, 22, True), (1, 700, 2100, 6, 3, 128, 128, 9, True), (1, 400, 500, 4, 2, 64, 64, 5, False), (1, 400, 500, 4, 4, 128, 32, 9, True),
]


def _case(shape, device):
    B, Lq, Lkv, H, Hkv, D, block, S, ragged = shape
    g = torch.Generator(device=device).manual_seed(Lq + Lkv)
    r = lambda n, h: torch.randn(B, n, h, D, generator=g, device=device)  # noqa: E731
    q, k, v, dout = r(Lq, H).bfloat16(), (r(Lkv, Hkv) + 0.3).bfloat16(), r(Lkv, Hkv).bfloat16(), r(Lq, H).bfloat16()
    nq, nkv = -(-Lq // block), -(-Lkv // block)
    index = torch.rand(B, H, nq, nkv, generator=g, device=device).argsort(-1)[..., :S].to(torch.int32).contiguous()
    num = torch.full((B, H, nq), min(S, nkv), dtype=torch.int32, device=device)
    if ragged:
        num = torch.randint(0, min(S, nkv) + 1, (B, H, nq), generator=g, device=device).to(torch.int32)
    return q, k, v, dout, index, num, _mask(index, num, block, Lq, Lkv)


def _norms(q, k, v, mask, dout, delta_part=1.0):
    """Gradients in 64 bits and, for each, the mean square of what the roundings add: `[B, L, H, D]`.  `delta_part`: of delta that is subtracted, one where there is no mistake."""
    g, scale, c = q.shape[2] // k.shape[2], q.shape[-1] ** -0.5, 2.0 ** -16 / 3
    q, k, v, do = (x.double().transpose(1, 2) for x in (q, k, v, dout))
    kk, vv = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
    s = (q @ kk.transpose(-1, -2) * scale).masked_fill(~mask, -math.inf)
    p = torch.where(mask, (s - torch.logsumexp(s, -1, keepdim=True).clamp(min=-1e300)).exp(), 0.0)
    out, dp = p @ vv, do @ vv.transpose(-1, -2)
    ds = p * (dp - delta_part * (do * out).sum(-1, keepdim=True)) * scale
    sums = lambda x: x.unflatten(1, (-1, g)).sum(2)  # noqa: E731
    t = lambda x: x.transpose(-1, -2)  # noqa: E731
    dq, dk, dv = ds @ kk, sums(t(ds) @ q), sums(t(p) @ do)
    # delta: one error for a row, from out's rounding and, through out, from those of P
    e_delta = c * ((do * out).square().sum(-1, keepdim=True) + (p * dp).square().sum(-1, keepdim=True)) * scale ** 2
    e_dq = c * dq.square() + c * ds.square() @ kk.square() + e_delta * (p @ kk).square()
    e_dk = c * dk.square() + sums(t(c * ds.square() + e_delta * p.square()) @ q.square())
    e_dv = c * dv.square() + sums(t(c * p.square()) @ do.square())
    return {n: (_t12(x), _t12(e)) for n, x, e in (("dq", dq, e_dq), ("dk", dk, e_dk), ("dv", dv, e_dv))}


def _t12(x):
    return x.transpose(1, 2)


def _ratios(got, want):
    """Of each gradient, sample and head: the error's norm over its limit."""
    return {n: ((got[n].double() - x).square().sum((1, 3)) / (1.25 ** 2 * e.sum((1, 3)) + 1e-300)).sqrt() for n, (x, e) in want.items()}


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES)
def test_errors_are_what_the_roundings_make_them(shape):
    q, k, v, dout, index, num, mask = _case(shape, dev())
    got = _run(q, k, v, index, num, shape[6], dout)
    for name, ratio in _ratios(got, _norms(q, k, v, mask, dout)).items():
        assert float(ratio.max()) <= 1, (name, float(ratio.max()))


@pytest.mark.parametrize("shape", [s for s in SHAPES if s[1] * s[2] < 600000])
def test_the_limits_see_mistakes(shape):
    """Planted in the oracle: delta left out, or a half or a fifth of it; a few percent of scale; and the roundings themselves stay within."""
    q, k, v, dout, index, num, mask = _case(shape, "cpu")
    want = _norms(q, k, v, mask, dout)
    exact = {n: x.bfloat16() for n, (x, _) in want.items()}
    assert all(float(r.max()) < 1 for r in _ratios(exact, want).values())
    for part in (0.0, 0.5, 0.8):
        wrong = {n: x.bfloat16() for n, (x, _) in _norms(q, k, v, mask, dout, part).items()}
        ratio = _ratios(wrong, want)
        assert float(ratio["dq"].min()) > 1 and float(ratio["dk"].min()) > 1, (part, float(ratio["dq"].min()), float(ratio["dk"].min()))
    for scale in (0.97, 1.02, 1.05, 1.2):
        ratio = _ratios({n: x * scale for n, (x, _) in want.items()}, want)
        assert all(float(r.min()) > 1 for r in ratio.values()), scale
