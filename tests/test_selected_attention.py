"""Attention over selected blocks and its gradient, against dense masked attention in 64 bits."""
import math

import pytest
import torch
import torch.nn.functional as F

from tests.helpers import dev

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def _picked(index, num, nkv):
    """[B, H, Nq, Nkv]: which block counts; repeated ids once, ids that are no block not at all."""
    B, H, nq, S = index.shape
    picked = torch.zeros(B, H, nq, nkv + 1, dtype=torch.bool, device=index.device)
    counts = torch.arange(S, device=index.device) < num.clamp(0, S)[..., None]
    ids = torch.where(counts & (index >= 0) & (index < nkv), index, nkv).long()
    picked.scatter_(-1, ids, True)
    return picked[..., :nkv]


def _mask(index, num, block, Lq, Lkv, block_sizes=None):
    nkv = -(-Lkv // block)
    picked = _picked(index, num, nkv)
    q_of, k_at = torch.arange(Lq, device=index.device) // block, torch.arange(Lkv, device=index.device)
    mask = picked[:, :, q_of][..., k_at // block]
    if block_sizes is not None:
        mask = mask & (k_at % block < block_sizes[k_at // block])
    return mask


def _exact(q, k, v, mask, dout=None):
    """Results in 64 bits, and with them how much the documented roundings may move each: half a step of the type for the result, and in bf16
    for the probabilities and dS that are factors of products; `out` enters the gradient as it was rounded.  float32: a sum of n terms
    may be n 2^-24 of the sum of their absolute values off, and a score's error e is a relative error e of its probability."""
    kind, (D, g) = q.dtype, (q.shape[-1], q.shape[2] // k.shape[2])
    u, scale = HALF_STEP[kind], q.shape[-1] ** -0.5
    p_u = u if kind == torch.bfloat16 else 0.0
    q, k, v = (x.double().transpose(1, 2) for x in (q, k, v))
    kk, vv = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
    s = (q @ kk.transpose(-1, -2) * scale).masked_fill(~mask, -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.where(mask, (s - lse.clamp(min=-1e300)[..., None]).exp(), 0.0)
    # a score: D products and sums, the scale, the difference to the normaliser, and an exponential good to a few steps
    score = ((D + 4) * 2.0 ** -24 * (q.abs() @ kk.abs().transpose(-1, -2) * scale) + 2.0 ** -21 + 2.0 ** -23 * s.masked_fill(~mask, 0).abs()).masked_fill(~mask, 0)
    n = float(mask.sum(-1).max())
    rel = p_u + 2 * score.amax(-1, keepdim=True) + (n + 8) * 2.0 ** -24        # of a probability, its normaliser's error included
    out = p @ vv
    e_out = u * out.abs() + (rel * p) @ vv.abs() + (n + 4) * 2.0 ** -24 * (p @ vv.abs())
    e_lse = score.amax(-1) + (n + 8) * 2.0 ** -24 + 2.0 ** -22 * lse.clamp(min=-1e3).abs()
    got = {"out": (out, e_out), "lse": (lse, e_lse)}
    if dout is not None:
        do = dout.double().transpose(1, 2)
        dp, delta = do @ vv.transpose(-1, -2), (do * out).sum(-1, keepdim=True)
        ds = p * (dp - delta) * scale
        e_dp = (D + 2) * 2.0 ** -24 * (do.abs() @ vv.abs().transpose(-1, -2))
        e_delta = (do.abs() * e_out).sum(-1, keepdim=True) + (D + 2) * 2.0 ** -24 * (do.abs() * out.abs()).sum(-1, keepdim=True)
        e_ds = (rel + p_u) * ds.abs() + p * (e_dp + e_delta) * scale + 4 * 2.0 ** -24 * ds.abs()
        m = max(n, float(mask.sum(-2).max()) * g) + 8
        sums = lambda x: x.unflatten(1, (-1, g)).sum(2)  # noqa: E731
        dq, dk, dv = ds @ kk, sums(ds.transpose(-1, -2) @ q), sums(p.transpose(-1, -2) @ do)
        many = m * 2.0 ** -24
        got["dq"] = dq, u * dq.abs() + (e_ds + many * ds.abs()) @ kk.abs()
        got["dk"] = dk, u * dk.abs() + sums((e_ds + many * ds.abs()).transpose(-1, -2) @ q.abs())
        got["dv"] = dv, u * dv.abs() + sums(((rel + many) * p).transpose(-1, -2) @ do.abs())
    return {n: tuple(x if n == "lse" else x.transpose(1, 2) for x in pair) for n, pair in got.items()}


def _check(got, want):
    for name, (value, bound) in want.items():
        x = got[name].double()
        assert torch.equal(torch.isfinite(x), torch.isfinite(value)), name
        far = ((x - value).abs() - bound - 1e-30)[torch.isfinite(value)]
        assert far.numel() == 0 or float(far.max()) <= 0, (name, float(far.max()), float(bound.max()))


def _lists(g, B, H, nq, nkv, S, how):
    index = torch.rand(B, H, nq, nkv, generator=g, device=dev()).argsort(-1).to(torch.int32)
    index = index[..., :S] if S <= nkv else torch.cat([index, torch.full((B, H, nq, S - nkv), -1, dtype=torch.int32, device=dev())], -1)
    num = torch.full((B, H, nq), min(S, nkv), dtype=torch.int32, device=dev())
    if how != "full":
        num = torch.randint(0, min(S, nkv) + 1, (B, H, nq), generator=g, device=dev()).to(torch.int32)
        num[0, 0, 0] = 0
    if how == "dirty":          # ids twice, ids that are no block, counts beyond the row and below zero
        index = index.clone()
        index[..., 1::3] = index[..., 0:1].expand_as(index[..., 1::3])
        index[..., 2::5] = nkv + 3
        index[..., 3::7] = -5
        num = num + 1
        num[-1, -1, -1], num[0, -1, 0] = S + 100, -3
    return index.contiguous(), num


def _inputs(g, B, Lq, Lkv, H, Hkv, D, dtype, big=1.0):
    r = lambda n, h: torch.randn(B, n, h, D, generator=g, device=dev())  # noqa: E731
    return (r(Lq, H) * big).to(dtype), (r(Lkv, Hkv) * big + 0.3).to(dtype), r(Lkv, Hkv).to(dtype), r(Lq, H).to(dtype)


def _run(q, k, v, index, num, block, dout, **more):
    from worldattention_b200.hsa import selected_attention
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    out, lse = selected_attention(*leaves, index, num, block, return_lse=True, **more)
    assert not lse.requires_grad and out.dtype == q.dtype
    dq, dk, dv = torch.autograd.grad(out, leaves, dout)
    with torch.no_grad():
        again = selected_attention(*leaves, index, num, block, **more)
    assert torch.equal(again, out) or bool(torch.isnan(out).any())
    return {"out": out.detach(), "lse": lse, "dq": dq, "dk": dk, "dv": dv}


SHAPES = [  # B, Lq, Lkv, H, Hkv, D, block, S
    (1, 1, 1, 1, 1, 128, 64, 1), (1, 1, 64, 2, 2, 128, 64, 1), (2, 1, 1000, 4, 2, 128, 64, 5), (3, 1, 3000, 12, 12, 128, 128, 24), (1, 3, 700, 4, 1, 128, 64, 11),
    (2, 8, 333, 6, 3, 128, 128, 3), (1, 9, 129, 2, 1, 128, 128, 2), (1, 64, 65, 2, 2, 128, 64, 2), (2, 65, 200, 4, 2, 128, 64, 3), (1, 127, 129, 3, 1, 128, 128, 2),
    (1, 300, 500, 8, 2, 128, 64, 6), (2, 300, 500, 4, 4, 128, 128, 4), (1, 1000, 1100, 12, 12, 128, 64, 9), (1, 1170, 390, 12, 4, 128, 128, 4), (1, 1500, 1400, 24, 24, 128, 64, 22),
]
ODD_SHAPES = [(1, 100, 130, 2, 1, 64, 64, 2), (2, 33, 70, 4, 2, 24, 16, 3), (1, 40, 41, 3, 3, 16, 7, 4), (1, 150, 260, 2, 2, 192, 64, 3), (1, 70, 90, 2, 1, 256, 100, 1),
              (1, 20, 300, 2, 2, 128, 32, 6), (2, 5, 9, 2, 2, 1, 4, 2), (1, 200, 200, 2, 1, 100, 128, 2)]


@pytest.mark.gpu
@pytest.mark.parametrize("how", ["full", "ragged", "dirty"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES + ODD_SHAPES)
def test_values_and_gradients(shape, dtype, how):
    B, Lq, Lkv, H, Hkv, D, block, S = shape
    g = torch.Generator(device=dev()).manual_seed(Lq * 7 + Lkv)
    q, k, v, dout = _inputs(g, B, Lq, Lkv, H, Hkv, D, dtype)
    index, num = _lists(g, B, H, -(-Lq // block), -(-Lkv // block), S, how)
    _check(_run(q, k, v, index, num, block, dout), _exact(q, k, v, _mask(index, num, block, Lq, Lkv), dout))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_large_scores(dtype):
    """Probabilities close to one and to zero, and normalisers far from zero."""
    g = torch.Generator(device=dev()).manual_seed(3)
    q, k, v, dout = _inputs(g, 1, 200, 300, 2, 2, 128, dtype, big=4.0)
    k[:, 100:140] -= 8.0
    index, num = _lists(g, 1, 2, 4, 5, 4, "full")
    _check(_run(q, k, v, index, num, 64, dout), _exact(q, k, v, _mask(index, num, 64, 200, 300), dout))


@pytest.mark.gpu
@pytest.mark.parametrize("D,block", [(128, 64), (128, 128), (32, 16)])
def test_nan_and_infinity_where_nothing_is_attended_to(D, block):
    """Blocks that nobody lists, tokens behind a block's size, rows that list nothing: what lies there does not reach any result."""
    from worldattention_b200.hsa import selected_attention
    g = torch.Generator(device=dev()).manual_seed(4)
    Lq, Lkv = 3 * block + 5, 6 * block - 3
    for dtype in (torch.bfloat16, torch.float32):
        q, k, v, dout = _inputs(g, 1, Lq, Lkv, 2, 1, D, dtype)
        index = torch.tensor([0, 2, 5, 3], dtype=torch.int32, device=dev()).expand(1, 2, 4, 4).contiguous()
        num = torch.tensor([[[3, 2, 0, 3], [3, 3, 0, 1]]], dtype=torch.int32, device=dev())
        mask = _mask(index, num, block, Lq, Lkv)
        want = _exact(q, k, v, mask, dout)
        k2, v2, q2, dout2 = k.clone(), v.clone(), q.clone(), dout.clone()
        for x in (k2, v2):
            x[:, block:2 * block] = math.nan                    # block 1, and 3 and 4
            x[:, 3 * block:5 * block] = math.inf
        for x in (q2, dout2):
            x[:, 2 * block:3 * block] = math.nan                # the rows that list nothing
        got = _run(q2, k2, v2, index, num, block, dout2)
        _check(got, want)
        assert not bool(got["out"][:, 2 * block:3 * block].any()) and not bool(got["dq"][:, 2 * block:3 * block].any())
        sizes = torch.tensor([block - 3, 0, block, 0, 0, 1], dtype=torch.int32, device=dev())
        mask = _mask(index, num, block, Lq, Lkv, sizes)
        want = _exact(q, k, v, mask, dout)
        k2, v2 = k.clone(), v.clone()
        for x in (k2, v2):
            x[:, block - 3:block] = math.nan
            x[:, 5 * block + 1:] = math.inf
        _check(_run(q, k2, v2, index, num, block, dout, block_sizes=sizes), want)
    with torch.no_grad():
        out, lse = selected_attention(q, k, v, index, torch.zeros_like(num), block, return_lse=True)
    assert not bool(out.any()) and bool((lse == -math.inf).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides_shared_inputs_and_gradients_without_memory(dtype):
    g = torch.Generator(device=dev()).manual_seed(5)
    index, num = _lists(g, 2, 4, 3, 4, 3, "ragged")
    both = torch.randn(2, 200, 2, 2, 128, generator=g, device=dev()).to(dtype)                 # keys and values side by side
    heads_first = torch.randn(2, 4, 150, 128, generator=g, device=dev()).to(dtype)             # [B, H, L, D]
    q, k, v = heads_first.transpose(1, 2), both[:, :, 0], both[:, :, 1]
    dout = torch.ones((), dtype=dtype, device=dev()).expand(2, 150, 4, 128)
    want = _exact(q, k, v, _mask(index, num, 64, 150, 200), dout)
    _check(_run(q, k, v, index, num, 64, dout), want)
    wide = torch.randn(2, 150, 4, 256, generator=g, device=dev()).to(dtype)
    q = wide[..., ::2]                                                                        # last axis with a stride
    _check(_run(q, k, v, index, num, 64, dout), _exact(q, k, v, _mask(index, num, 64, 150, 200), dout))
    q = wide[..., 1:129]                                                                      # rows at odd addresses
    _check(_run(q, k, v, index, num, 64, dout), _exact(q, k, v, _mask(index, num, 64, 150, 200), dout))
    # one key head given to all query heads, one sample's keys to both samples: the gradients of the copies add up
    from worldattention_b200.hsa import selected_attention
    base = torch.randn(1, 200, 1, 128, generator=g, device=dev()).to(dtype).requires_grad_()
    q = heads_first.transpose(1, 2)
    full = base.expand(2, 200, 4, 128)
    out = selected_attention(q, full, full, index, num, 64)
    dbase, = torch.autograd.grad(out, base, torch.ones_like(out))
    w = _exact(q, full.detach(), full.detach(), _mask(index, num, 64, 150, 200), torch.ones_like(out))
    total = sum(w[n][0].sum((0, 2)) for n in ("dk", "dv"))
    bound = sum(w[n][1].sum((0, 2)) for n in ("dk", "dv")) + 16 * HALF_STEP[dtype] * sum(w[n][0].abs().sum((0, 2)) for n in ("dk", "dv"))      # (summed in the type: 16 terms)
    assert bool(((dbase[0, :, 0].double() - total).abs() <= bound).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_equal_calls_equal_bits_streams_and_graphs(dtype):
    from worldattention_b200.hsa import selected_attention
    g = torch.Generator(device=dev()).manual_seed(6)
    q, k, v, dout = _inputs(g, 1, 700, 900, 4, 2, 128, dtype)
    index, num = _lists(g, 1, 4, 11, 15, 8, "ragged")
    want = _run(q, k, v, index, num, 64, dout)
    for _ in range(3):
        got = _run(q, k, v, index, num, 64, dout)
        assert all(torch.equal(got[n], want[n]) for n in want)
    # two calls side by side on two streams
    streams, results = [torch.cuda.Stream() for _ in range(2)], []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            results.append(_run(q, k, v, index, num, 64, dout))
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(r[n], want[n]) for r in results for n in want)
    # two captured steps replayed in turn, on other inputs than they were captured with
    with torch.cuda.stream(streams[0]):
        static = [x.clone() for x in (q, k, v, dout)]
        graphs = []
        for _ in range(2):
            leaves = [x.requires_grad_() for x in (y.detach() for y in static[:3])]
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=streams[0]):
                out = selected_attention(*leaves, index, num, 64)
                grads = torch.autograd.grad(out, leaves, static[3])
            graphs.append((graph, out, grads))
        for x, y in zip(static, _inputs(g, 1, 700, 900, 4, 2, 128, dtype)):
            x.copy_(y)
        for graph, _, _ in graphs + graphs[:1]:
            graph.replay()
    torch.cuda.current_stream().wait_stream(streams[0])
    other = _run(*static[:3], index, num, 64, static[3])
    for _, out, grads in graphs:
        assert torch.equal(out, other["out"]) and all(torch.equal(x, other[n]) for x, n in zip(grads, ("dq", "dk", "dv")))


@pytest.mark.gpu
@pytest.mark.parametrize("block", [64, 128])
@pytest.mark.parametrize("q_len,kv_len,S", [(128, 8192, 60), (1, 20000, 30), (256, 4000, 31), (4096, 256, 2), (2500, 130, 1)])
def test_items_of_one_step_and_items_of_many(block, q_len, kv_len, S):
    """Key blocks that one query block lists, or none, and query blocks with one: every hand-over between items, on repeated calls."""
    g = torch.Generator(device=dev()).manual_seed(q_len + block)
    q, k, v, dout = _inputs(g, 1, q_len, kv_len, 6, 3, 128, torch.bfloat16)
    index, num = _lists(g, 1, 6, -(-q_len // block), -(-kv_len // block), S, "ragged")
    first = _run(q, k, v, index, num, block, dout)
    _check(first, _exact(q, k, v, _mask(index, num, block, q_len, kv_len), dout))
    for _ in range(4):
        again = _run(q, k, v, index, num, block, dout)
        assert all(torch.equal(again[n], first[n]) for n in first)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("block", [64, 128])
def test_what_follows_the_gradients_sees_all_of_them(dtype, block):
    """The second launch of the gradient is short here and begins before the first one's end: a copy behind it, on this stream, on another one or in a graph."""
    from worldattention_b200.hsa import selected_attention
    g = torch.Generator(device=dev()).manual_seed(15)
    q, k, v, dout = _inputs(g, 1, 70, 20000, 6, 3, 128, dtype)
    index, num = _lists(g, 1, 6, -(-70 // block), -(-20000 // block), -(-20000 // block), "full")
    leaves = [x.requires_grad_() for x in (q, k, v)]
    side = torch.cuda.Stream()

    def step():
        grads = torch.autograd.grad(selected_attention(*leaves, index, num, block), leaves, dout)
        return grads, [x.clone() for x in grads]
    for _ in range(3):
        grads, copies = step()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            far = [x.clone() for x in grads]
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) and torch.equal(x, z) for x, y, z in zip(grads, copies, far))
    want = [x.clone() for x in grads]
    del grads, copies, far
    leaves = [x.detach().requires_grad_() for x in leaves]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grads, copies = step()
    for _ in range(2):
        for x in (*grads, *copies):
            x.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) and torch.equal(y, z) for x, y, z in zip(want, grads, copies))


@pytest.mark.gpu
def test_gradient_against_differences():
    from worldattention_b200.hsa import selected_attention
    g = torch.Generator(device=dev()).manual_seed(7)
    q, k, v, dout = _inputs(g, 1, 90, 140, 4, 2, 32, torch.float32)
    index, num = _lists(g, 1, 4, 3, 5, 3, "ragged")
    got = _run(q, k, v, index, num, 32, dout)
    f = lambda q, k, v: float((selected_attention(q, k, v, index, num, 32).double() * dout).sum())  # noqa: E731
    at, eps = [q, k, v], 2.0 ** -7
    for i, name in enumerate(("dq", "dk", "dv")):
        step = torch.randn(at[i].shape, generator=g, device=dev())
        there = lambda t: f(*[x + t * step if j == i else x for j, x in enumerate(at)])  # noqa: B023, E731
        # fourth-order differences; 90 * 4 * 32 outputs with errors of about 2^-22 each, divided by the step, and what is left of the fifth derivative
        slope = (8 * (there(eps) - there(-eps)) - (there(2 * eps) - there(-2 * eps))) / (12 * eps)
        assert abs(slope - float((got[name].double() * step).sum())) < 90 * 4 * 32 * 2 ** -22 / eps * 0.2 + 0.02, name


@pytest.mark.gpu
def test_nothing_to_do_and_part_of_the_gradients():
    from worldattention_b200.hsa import selected_attention
    g = torch.Generator(device=dev()).manual_seed(8)
    q, k, v, dout = _inputs(g, 2, 70, 130, 4, 2, 128, torch.bfloat16)
    index, num = _lists(g, 2, 4, 2, 3, 2, "full")
    ids = lambda B, nq, S: (index[:B, :, :nq, :S].contiguous(), num[:B, :, :nq].contiguous())  # noqa: E731
    for qq, kk, (ii, nn) in ((q[:, :0], k, ids(2, 0, 2)), (q, k[:, :0], ids(2, 2, 2)), (q[:0], k[:0], ids(0, 2, 2)), (q, k, ids(2, 2, 0))):
        leaves = [x.detach().requires_grad_() for x in (qq, kk, kk)]
        out, lse = selected_attention(*leaves, ii, nn, 64, return_lse=True)
        assert out.shape == qq.shape and not bool(out.any()) and bool((lse == -math.inf).all())
        assert all(not bool(x.any()) for x in torch.autograd.grad(out.sum(), leaves))
    full = _run(q, k, v, index, num, 64, dout)
    for needs in ((True, False, False), (False, True, False), (False, False, True)):
        leaves = [x.detach().requires_grad_(n) for x, n in zip((q, k, v), needs)]
        grad, = torch.autograd.grad(selected_attention(*leaves, index, num, 64), [x for x, n in zip(leaves, needs) if n], dout)
        assert torch.equal(grad, full[("dq", "dk", "dv")[needs.index(True)]])


@pytest.mark.gpu
def test_a_layer_of_operators_trains():
    """Routing by pooled scores, rotary positions, attention over what was selected, pages moved: as they are used together."""
    from worldattention_b200.causal_dit import rope_table
    from worldattention_b200.hkv import move_pages
    from worldattention_b200.hsa import block_attention_map, block_mean_pool, build_block_routing, selected_attention
    from worldattention_b200.rope import axial_rope
    g = torch.Generator(device=dev()).manual_seed(9)
    B, L, H, Hkv, D, block = 2, 390, 4, 2, 128, 64
    x = torch.randn(B, L, 256, generator=g, device=dev())
    w = {n: (torch.randn(256, h * D, generator=g, device=dev()) / 16).requires_grad_() for n, h in (("q", H), ("k", Hkv), ("v", Hkv))}
    t = torch.arange(L, device=dev())
    pos = torch.stack([t // 30 % 13, t // 6 % 5, t % 6], -1).int()
    table = rope_table(D).to(dev())

    def step(dtype):
        q, k, v = ((x.to(dtype) @ w[n].to(dtype)).view(B, L, -1, D) for n in ("q", "k", "v"))
        q, k = axial_rope((q, k), pos, table)
        with torch.no_grad():
            pooled = [block_mean_pool(F.pad(y, (0, 0, 0, 0, 0, -L % block)).transpose(1, 2), L, -(-L // block), block) for y in (q, k)]
            routing = build_block_routing(block_attention_map(pooled[0], pooled[1].repeat_interleave(H // Hkv, 1)), tau_min=0.5, tau_max=0.9)
        index, num = routing.index, routing.num
        out = selected_attention(q, k, v, index, num, block)
        return q, k, v, index, num, out

    for dtype in (torch.float32, torch.bfloat16):
        q, k, v, index, num, out = step(dtype)
        dout = torch.randn(out.shape, generator=g, device=dev()).to(dtype)
        grads = torch.autograd.grad(out, (q, k, v), dout, retain_graph=True)
        _check(dict(zip(("out", "dq", "dk", "dv"), (out.detach(), *grads))), {n: e for n, e in _exact(q.detach(), k.detach(), v.detach(), _mask(index, num, block, L, L), dout).items() if n != "lse"})
        assert all(bool(torch.isfinite(d).all()) and bool(d.any()) for d in torch.autograd.grad(out, tuple(w.values()), dout))
    # the keys move to other pages of a cache, and the lists follow them
    with torch.no_grad():
        caches = [torch.zeros(B, 10 * block, Hkv, D, device=dev(), dtype=torch.bfloat16) for _ in range(2)]
        for c, y in zip(caches, (k, v)):
            c[:, :L] = y
        move_pages(caches, [9, 4, 0, 1, 2, 3], [0, 1, None, 2, 3, 4], block)
        where = torch.tensor([9, 4, 1, 2, 3, 5, 6], dtype=torch.int32, device=dev())      # page 5 and the short page 6 stay
        sizes = torch.full((10,), block, dtype=torch.int32, device=dev())
        sizes[6] = L - 6 * block
        moved = selected_attention(q, *caches, where[index.long()].contiguous(), num, block, block_sizes=sizes)
        _check({"out": moved}, {n: e for n, e in _exact(q, k, v, _mask(index, num, block, L, L)).items() if n == "out"})


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D", [16, 128])
def test_block_sparse_attention_carries_gradients(dtype, D):
    """The reference's names and layout (`[B, H, N, D]`, padded blocks), from a map and from lists; the values are those without gradients."""
    from worldattention_b200.hsa import block_sparse_attention_reference
    from worldattention_b200.hsa.block_sparse_triton import block_sparse_attention, map_to_index
    g = torch.Generator(device=dev()).manual_seed(D)
    B, H, nq, nk, block = 2, 3, 2, 4, 64
    q, k, v, dout = (x.transpose(1, 2).contiguous() for x in _inputs(g, B, nq * block, nk * block, H, H, D, dtype))
    sizes = torch.tensor([64, 64, 64, 10], dtype=torch.int32, device=dev())
    block_map = torch.rand(B, H, nq, nk, generator=g, device=dev()) < 0.5
    block_map[0, 1, 1] = False
    index, num = map_to_index(block_map)
    with torch.no_grad():
        want = block_sparse_attention(q, k, v, block_sizes=sizes, block_map=block_map)
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    out = block_sparse_attention(*leaves, block_sizes=sizes, block_map=block_map)
    assert torch.equal(out.detach(), want) and out.requires_grad
    grads = torch.autograd.grad(out, leaves, dout)
    t = lambda x: x.transpose(1, 2)  # noqa: E731
    exact = _exact(t(q), t(k), t(v), _mask(index, num, block, nq * block, nk * block, sizes), t(dout))
    _check({n: t(x) for n, x in zip(("out", "dq", "dk", "dv"), (out.detach(), *grads))}, {n: e for n, e in exact.items() if n != "lse"})
    out, lse = block_sparse_attention_reference(leaves[0], k, v, index.long(), num.long(), sizes.long(), block, return_lse=True)
    assert torch.equal(out.detach(), want) and torch.equal(torch.autograd.grad(out, leaves[0], dout)[0], grads[0]) and lse.shape == (B, H, nq * block)
    assert not block_sparse_attention_reference(q, k, v, index, num, sizes, block).requires_grad


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D,block", [(torch.bfloat16, 128, 64), (torch.bfloat16, 128, 128), (torch.float32, 128, 64), (torch.float32, 48, 64)])
def test_rows_that_list_only_blocks_without_a_key(dtype, D, block):
    g = torch.Generator(device=dev()).manual_seed(14)
    q, k, v, dout = _inputs(g, 1, 3 * block, 4 * block, 2, 2, D, dtype)
    index = torch.tensor([[0, 0], [1, 0], [2, 3]], device=dev(), dtype=torch.int32).expand(1, 2, 3, 2).contiguous()
    num = torch.full((1, 2, 3), 2, device=dev(), dtype=torch.int32)
    sizes = torch.tensor([0, block, block // 2, 5], device=dev(), dtype=torch.int32)
    want = _exact(q, k, v, _mask(index, num, block, 3 * block, 4 * block, sizes), dout)
    dout[:, :block], dout[:, 1] = math.nan, math.inf          # the first rows see no key: they have no part in the gradients
    got = _run(q, k, v, index, num, block, dout, block_sizes=sizes)
    _check(got, want)
    assert not bool(got["dq"][:, :block].any()) and not bool(got["dk"][:, :block].any()) and not bool(got["dv"][:, :block].any())


@pytest.mark.gpu
def test_a_step_is_not_captured_over_an_eager_graph_of_its_leaves():
    from worldattention_b200.hsa import selected_attention
    from worldattention_b200.rope import axial_rope
    g = torch.Generator(device=dev()).manual_seed(13)
    q, k, v, dout = _inputs(g, 1, 70, 130, 4, 4, 128, torch.bfloat16)
    index, num = _lists(g, 1, 4, 2, 3, 2, "full")
    pos, table = torch.zeros(70, 1, dtype=torch.int32, device=dev()), torch.ones(1, 64, 2, device=dev())
    q.requires_grad_()
    attend, turn = lambda q: selected_attention(q, k, v, index, num, 64), lambda q: axial_rope(q, pos, table)  # noqa: E731
    for call in (attend, lambda q: attend(q.view(q.shape)), turn, lambda q: turn(q[:, :])):
        for eager in (attend, turn, lambda q: q * 2):
            alive = eager(q)
            with pytest.raises(RuntimeError, match="eager graph"):
                with torch.cuda.graph(torch.cuda.CUDAGraph()):
                    call(q)
            del alive
    want = torch.autograd.grad(attend(q), q, dout)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        alive = attend(q)                             # on a side stream it may be alive
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        attend(q).backward(dout)
    graph.replay()
    assert torch.equal(q.grad, want)
    del alive


@pytest.mark.gpu
def test_a_gradient_tells_of_an_earlier_launch_that_gave_up():
    from worldattention_b200 import _lib
    from worldattention_b200.hsa import selected_attention
    g = torch.Generator(device=dev()).manual_seed(12)
    q, k, v, dout = _inputs(g, 1, 70, 130, 4, 2, 128, torch.bfloat16)
    index, num = _lists(g, 1, 4, 2, 3, 2, "full")
    q.requires_grad_()
    out = selected_attention(q, k, v, index, num, 64)
    torch.cuda.synchronize()
    word = _lib.status_word(dev())
    word.fill_(455)                                   # as a launch would have left it; the engine's thread does not hold the interpreter lock
    with pytest.raises(RuntimeError, match="wait site 455"):
        out.backward(dout)
    assert int(word) == 0
    out = selected_attention(q, k, v, index, num, 64)
    out.backward(dout)
    assert bool(q.grad.any())


@pytest.mark.gpu
def test_refusals():
    from worldattention_b200.hsa import selected_attention
    g = torch.Generator(device=dev()).manual_seed(10)
    q, k, v, dout = _inputs(g, 1, 70, 130, 4, 2, 16, torch.float32)
    index, num = _lists(g, 1, 4, 2, 3, 2, "full")
    call = lambda q=q, k=k, v=v, index=index, num=num, block=64, **more: selected_attention(q, k, v, index, num, block, **more)  # noqa: E731
    for bad, word in [(lambda: call(k=k[:, :100]), "Lkv"), (lambda: call(k=k[..., :8], v=v[..., :8]), "D"), (lambda: call(k=k.bfloat16(), v=v.bfloat16()), "dtype"),
                      (lambda: call(q=q[:, :, :3]), "divide"), (lambda: call(index=index[:, :, :1]), "Nq"), (lambda: call(num=num[..., :1]), "Nq"),
                      (lambda: call(index=index.long()), "int32"), (lambda: call(num=num.long()), "int32"), (lambda: call(block=0), "positive"), (lambda: call(block=32), "Nq"),
                      (lambda: call(q=q[0]), "B, L, H, D"), (lambda: call(q=q.half(), k=k.half(), v=v.half()), "float32 or bfloat16"),
                      (lambda: call(block_sizes=torch.ones(2, dtype=torch.int32, device=dev())), "block_sizes"), (lambda: call(block_sizes=torch.ones(3, device=dev())), "block_sizes")]:
        with pytest.raises(ValueError, match=word):
            bad()
    with pytest.raises(NotImplementedError, match="256"):
        call(q=q.repeat(1, 1, 1, 17), k=k.repeat(1, 1, 1, 17), v=v.repeat(1, 1, 1, 17))
    leaf = q.detach().requires_grad_()
    out = call(q=leaf)
    grad, = torch.autograd.grad(out, leaf, torch.ones_like(out).requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        grad.sum().backward()


def test_no_cpu_path_and_arguments_without_a_device():
    import ctypes

    from worldattention_b200 import _lib
    from worldattention_b200.hsa import selected_attention
    x, ids = torch.zeros(1, 4, 1, 16), torch.zeros(1, 1, 1, 1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        selected_attention(x, x, x, ids, ids[..., 0], 64)
    lib = _lib.lib()
    assert lib.wa_selected_params_size() == ctypes.sizeof(_lib.SelectedParams)
    t = lambda: _lib.Tensor4(4096, 1, 0, 8192, 128, 128)  # noqa: E731

    def params(**change):
        p = _lib.SelectedParams(B=1, H=2, Hkv=1, D=128, Lq=64, Lkv=64, block_size=64, index_stride=1, index=4096, num=4096, lse=4096)
        for n in ("q", "k", "v", "out", "dout", "dq", "dk", "dv"):
            setattr(p, n, t())
        for n, x in change.items():
            setattr(p, n, x)
        return p
    for change, rc in [(dict(B=0), -1), (dict(H=3, Hkv=2), -1), (dict(D=257), -2), (dict(block_size=0), -1), (dict(index=None), -1), (dict(k=_lib.Tensor4(4096, 0, 0, 1, 1, 1)), -1),
                       (dict(q=_lib.Tensor4(None, 1, 0, 1, 1, 1)), -1), (dict(Lkv=2 ** 31 - 1), -2), (dict(H=70000, Hkv=1), -2), (dict(), -3), (dict(workspace=4096, workspace_bytes=8), -3)]:
        p = params(**change)
        assert lib.wa_selected_forward(ctypes.byref(p), None) == rc, change
        assert lib.wa_selected_backward(ctypes.byref(p), None) == rc, change
        assert (lib.wa_selected_workspace_bytes(ctypes.byref(p), 1) == 0) == (rc not in (-3,))
    assert lib.wa_selected_backward(ctypes.byref(params(lse=None)), None) == -1
    big = params(workspace=4096 + 8, workspace_bytes=1 << 40)
    assert lib.wa_selected_forward(ctypes.byref(big), None) == _lib.WA_ERR_ALIGN
