"""Attention over selected blocks where something that IS attended to is no finite number: it shows in exactly the results that depend on it."""
import math

import pytest
import torch

from tests.helpers import dev
from tests.test_selected_attention import _exact, _inputs, _lists, _mask, _run


def _by_lists(q, k, v, mask, dout):
    """The formulas in 64 bits over the attended keys of each row alone, so that what a row does not attend to takes no part in its products.
    The softmax is e^(s - max) over its sum: a score that is no number, or +inf, leaves none in its row, one of -inf is a probability of zero."""
    g, scale = q.shape[2] // k.shape[2], q.shape[-1] ** -0.5
    q, k, v, dout, mask = (x.cpu() for x in (q.double(), k.double(), v.double(), dout.double(), mask))
    out, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    lse = torch.full((q.shape[0], q.shape[2], q.shape[1]), -math.inf, dtype=torch.float64)
    for b in range(q.shape[0]):
        for h in range(q.shape[2]):
            rows, which = torch.unique(mask[b, h], dim=0, return_inverse=True)       # rows that attend to the same keys
            for r in range(len(rows)):
                i, j = (which == r).nonzero()[:, 0], rows[r].nonzero()[:, 0]
                if len(j) == 0:
                    continue
                qi, kj, vj, do = q[b, i, h], k[b, j, h // g], v[b, j, h // g], dout[b, i, h]
                s = qi @ kj.T * scale
                e = (s - s.amax(-1, keepdim=True)).exp()
                p = e / e.sum(-1, keepdim=True)
                lse[b, h, i] = s.amax(-1) + e.sum(-1).log()
                out[b, i, h] = p @ vj
                ds = p * (do @ vj.T - (do * out[b, i, h]).sum(-1, keepdim=True)) * scale
                dq[b, i, h] = ds @ kj
                dk[b, :, h // g] = dk[b, :, h // g].index_add(0, j, ds.T @ qi)
                dv[b, :, h // g] = dv[b, :, h // g].index_add(0, j, p.T @ do)
    return {n: x.to(dev()) for n, x in (("out", out), ("lse", lse), ("dq", dq), ("dk", dk), ("dv", dv))}


def _agree(got, want, bounds):
    """The same places are finite, the same results are no numbers; finite ones are as near as `bounds` has it."""
    for name, w in want.items():
        x, finite = got[name].double(), torch.isfinite(w)
        assert torch.equal(torch.isfinite(x), finite), (name, int((torch.isfinite(x) & ~finite).sum()), int((~torch.isfinite(x) & finite).sum()))
        if name in ("out", "lse"):
            assert torch.equal(torch.isnan(x), torch.isnan(w)), name
        value, bound = bounds[name]
        far = ((x - value).abs() - bound - 1e-30)[finite]
        assert far.numel() == 0 or float(far.max()) <= 0, (name, float(far.max()))


def _where(index, num, block, B, H, row_block):
    """A block that this query block lists."""
    return int(index[0, 0, row_block, 0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D,block,sizes", [(torch.bfloat16, 128, 64, False), (torch.bfloat16, 128, 128, False), (torch.float32, 128, 64, False), (torch.float32, 48, 16, False),
                                                 (torch.bfloat16, 128, 32, False), (torch.bfloat16, 128, 64, True), (torch.float32, 128, 64, True), (torch.bfloat16, 96, 64, True)])
@pytest.mark.parametrize("Lq,H", [(1, 4), (8, 4), (9, 4), (333, 4), (333, 48)])
@pytest.mark.parametrize("what", ["key nan", "key +inf", "key -inf", "value nan", "value inf", "query nan", "query inf", "dout nan"])
def test_what_is_attended_to_and_no_number_shows(dtype, D, block, sizes, Lq, H, what):
    g = torch.Generator(device=dev()).manual_seed(block + Lq)
    Lkv, Hkv = 9 * block - 7, H // 2
    q, k, v, dout = _inputs(g, 1, Lq, Lkv, H, Hkv, D, dtype)
    q[..., 5] = q[..., 5].abs() + 0.25                        # so that an infinity in channel 5 of a key has one sign in all scores
    nq, nkv = -(-Lq // block), 9
    index, num = _lists(g, 1, H, nq, nkv, 4, "ragged" if nq > 1 else "full")
    row = nq - 1                                              # a query block, and a token of one of the blocks that it lists first
    num[0, 0, row] = 3
    more = {"block_sizes": torch.full((nkv,), block - 2, dtype=torch.int32, device=dev())} if sizes else {}
    mask = _mask(index, num, block, Lq, Lkv, more.get("block_sizes"))
    at = int(index[0, 0, row, 1]) * block + 3
    token = Lq - 1
    q2, k2, v2, dout2 = q.clone(), k.clone(), v.clone(), dout.clone()
    clean = mask
    kind, _, value = what.partition(" ")
    value = float(value)
    if kind == "key":
        k2[0, at, 0, 5] = value
        if value == -math.inf:                                # a probability of zero: as if it were not attended to
            clean = mask.clone()
            clean[0, :H // Hkv, :, at] = False
    elif kind == "value":
        v2[0, at, 0, 3] = value
    elif kind == "query":
        q2[0, token, 0, 5] = value
    else:
        dout2[0, token, 0, 5] = value
    want = _by_lists(q2, k2, v2, mask, dout2)
    assert kind == "dout" or not bool(torch.isfinite(want["out"]).all()) or what == "key -inf"
    _agree(_run(q2, k2, v2, index, num, block, dout2, **more), want, _exact(q, k, v, clean, dout))


@pytest.mark.gpu
@pytest.mark.parametrize("block", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_scores_of_minus_infinity_before_finite_ones(dtype, block):
    """Whole blocks whose scores are all -inf, first, last and in the middle of a list: the others are what is attended to.  A row that has nothing else is as
    one without a key."""
    g = torch.Generator(device=dev()).manual_seed(block)
    Lq, Lkv, H = 4 * block + 3, 6 * block, 4
    q, k, v, dout = _inputs(g, 1, Lq, Lkv, H, H, 128, dtype)
    q[..., 5] = q[..., 5].abs() + 0.25
    index = torch.tensor([[0, 2, 3], [2, 0, 3], [2, 3, 0], [0, 1, 0], [1, 0, 4]], dtype=torch.int32, device=dev()).expand(1, H, 5, 3).contiguous()
    num = torch.tensor([3, 3, 3, 2, 1], dtype=torch.int32, device=dev()).expand(1, H, 5).contiguous()
    mask = _mask(index, num, block, Lq, Lkv)
    k2 = k.clone()
    k2[:, :2 * block, :, 5] = -math.inf                        # blocks 0 and 1
    clean = mask.clone()
    clean[..., :2 * block] = False
    want = _exact(q, k, v, clean, dout)
    got = _run(q, k2, v, index, num, block, dout)
    touched = mask[..., :2 * block].any(-1).transpose(1, 2)    # dS of zero times an infinity in the rows that list those keys
    assert bool(torch.isnan(got["dq"][..., 5][touched & (want["lse"][0] > -math.inf).transpose(1, 2)]).all())
    for x in (got["dq"], want["dq"][0], want["dq"][1]):
        x[..., 5] = 0
    for name, (value, bound) in want.items():
        x = got[name].double()
        assert torch.equal(torch.isfinite(x), torch.isfinite(value)), name
        far = ((x - value).abs() - bound - 1e-30)[torch.isfinite(value)]
        assert float(far.max()) <= 0, (name, float(far.max()))
