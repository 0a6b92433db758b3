"""What the speed of the trainable and cache-keeping operators is measured on.

Three operators around a layer that attends over selected key blocks:

* `attend` -- attention over the key blocks that a routing selected for each query block, with its gradient
  (`hsa.selected_attention`).  Forward alone: a chunk of a rollout, and single tokens against a long cache.  With
  gradients: the training step of such a layer, one sequence or a ragged batch, in bf16 and in float32.
* `rotary` -- the rotary embedding of q and k in front of it, for tokens with a position of their own on several axes
  (`rope.axial_rope`): samples of different grids side by side, text between pictures; with its gradient where it trains.
* `pages`  -- what happens to the caches that it reads: pages copied, forked, moved together and cleared in place, in all
  tensors of a call at once (`hkv.move_pages`).

Sizes are those of the repository's benchmark configurations (12 heads of 128, frames of 1560 tokens, windows of 21
frames, chunks of 3, blocks of 64 and 128 tokens), and, in `draw`, everything between them and the smallest calls.
"""
import math

import torch
import torch.nn.functional as F

own = False

DEV = torch.device("cuda", 0)
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp32": 4}
TABLE_ROWS = 1024


# ------------------------------------------------------------------------------------------------
# the cases
# ------------------------------------------------------------------------------------------------
def listed():
    attend = dict(kind="attend", batch=1, heads=12, kv_heads=12, dim=128, block=64, dtype="bf16", train=False, ragged=False)
    return [
        # One new token for each of four sequences against a window of 21 frames: the call whose latency counts.
        dict(attend, name="attend single tokens", batch=4, q_len=1, kv_len=32760, select=32),
        # A chunk of three frames over the window, 128-token blocks: the headline configuration's shapes, forward alone.
        dict(attend, name="attend chunk", q_len=4680, kv_len=32760, block=128, select=16),
        # A training step on the first frames of a rollout, three frames of a small latent, float32: the accuracy configuration.
        dict(attend, name="train small fp32", q_len=1170, kv_len=1170, select=6, dtype="fp32", train=True, ragged=True),
        # A training step on a batch with heads that share keys, an odd length, and counts that differ from row to row (zero
        # among them), as the routing by cumulative mass gives them.
        dict(attend, name="train shared heads", batch=2, heads=16, kv_heads=4, q_len=2031, kv_len=4111, select=16, train=True, ragged=True),
        # A training step of a chunk over the window that it attends to, 128-token blocks.
        dict(attend, name="train chunk", q_len=4680, kv_len=32760, block=128, select=32, train=True),
        # The training step of a whole window over itself, 64-token blocks (the layer's default).
        dict(attend, name="train window", q_len=32760, kv_len=32760, select=32, train=True),
        # Single tokens with a position each: latency.
        dict(kind="rotary", name="rotary single tokens", batch=4, length=1, heads=12, kv_heads=12, dim=128, dtype="bf16", interleaved=True, train=False),
        # The chunk's q and k, positions in time, height and width.
        dict(kind="rotary", name="rotary chunk", batch=1, length=4680, heads=12, kv_heads=12, dim=128, dtype="bf16", interleaved=True, train=False),
        # A training batch of packed samples, shared key heads, pairs half a head apart, an odd length; forward and gradient.
        dict(kind="rotary", name="rotary train", batch=2, length=16383, heads=16, kv_heads=4, dim=128, dtype="bf16", interleaved=False, train=True),
        # Pages of a small paged cache forked for a second continuation: latency.
        dict(kind="pages", name="pages fork", tensors=8, pages=64, page=16, row=1536, moves=6, how="fork", dtype="bf16"),
        # The window of one layer rolls by three frames: keys and values.
        dict(kind="pages", name="pages roll", tensors=2, pages=21, page=1560, row=1536, moves=18, how="roll", dtype="bf16"),
        # Scattered pages of the whole model's caches are moved together, and what they leave is cleared.
        dict(kind="pages", name="pages compact", tensors=60, pages=21, page=1560, row=1536, moves=12, how="compact", dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the same ranges; half of them are attention calls."""
    kind = rng.choice(["attend"] * 4 + ["rotary", "rotary", "pages", "pages"])
    kv_heads = rng.choice([2, 4, 6, 12])
    heads = kv_heads * rng.choice([1, 1, 2, 4]) if kv_heads < 12 else 12
    if kind == "attend":
        dtype = rng.choice(["bf16"] * 4 + ["fp32"])
        train = rng.random() < 0.6
        block = rng.choice([64, 128])
        kv_len = _log_int(rng, 40, 32760 if dtype == "bf16" else 3000)
        if train:
            q_len = min(kv_len, _log_int(rng, 30, 16000 if dtype == "bf16" else 1500))
        else:
            q_len = rng.choice([1, rng.randint(2, 9), _log_int(rng, 10, 4680 if dtype == "bf16" else 1500)])
        blocks = -(-kv_len // block)
        return dict(kind=kind, batch=rng.choice([1, 1, 2, 3]) if kv_len * q_len < 2 ** 25 else 1, heads=heads, kv_heads=kv_heads,
                    dim=128 if dtype == "bf16" else rng.choice([64, 128]), block=block, dtype=dtype, train=train,
                    ragged=rng.random() < 0.5, q_len=q_len, kv_len=kv_len, select=min(blocks, _log_int(rng, 1, 48 * 64 // block)))
    if kind == "rotary":
        return dict(kind=kind, batch=rng.randint(1, 4), length=_log_int(rng, 1, 8000), heads=heads, kv_heads=kv_heads, dim=rng.choice([64, 96, 128]),
                    dtype=rng.choice(["bf16", "bf16", "fp32"]), interleaved=rng.random() < 0.5, train=rng.random() < 0.5)
    pages, page = rng.randint(6, 200), _log_int(rng, 7, 1560)
    how = rng.choice(["fork", "roll", "compact"])
    row = rng.choice([256, 768, 1536])
    tensors = max(1, min(rng.randint(1, 60), 4_000_000_000 // (pages * page * row * 2)))
    return dict(kind=kind, tensors=tensors, pages=pages, page=page, row=row, moves=rng.randint(1, pages // 2), how=how, dtype=rng.choice(["bf16", "fp32"]))


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _tokens(g, batch, n, heads, dim, dtype, spread=0.0):
    """`[batch, n, heads, dim]`: unit normal values plus an offset shared by 130 neighbouring tokens (a patch of the picture)."""
    x = torch.randn((batch, n, heads, dim), generator=g, device=DEV)
    if spread:
        x += (torch.randn((batch, -(-n // 130), heads, dim), generator=g, device=DEV) * spread).repeat_interleave(130, dim=1)[:, :n]
    return x.to(DTYPES[dtype])


def _selection(g, case):
    """Ids and counts as a router gives them: the best blocks of a noisy score that prefers near ones, best first."""
    B, H, S = case["batch"], case["heads"], case["select"]
    nq, nk = -(-case["q_len"] // case["block"]), -(-case["kv_len"] // case["block"])
    near = -(torch.arange(nq, device=DEV)[:, None] * (nk / nq) - torch.arange(nk, device=DEV)[None]).abs() * (4.0 / nk)
    score = torch.randn((B, H, nq, nk), generator=g, device=DEV) + near
    index = score.topk(S, dim=-1).indices.to(torch.int32).contiguous()
    num = torch.full((B, H, nq), S, dtype=torch.int32, device=DEV)
    if case["ragged"]:
        num = torch.randint(0, S + 1, (B, H, nq), generator=g, device=DEV).to(torch.int32)
    return index, num


def _axes(dim):
    """Rotated pairs of the time, height and width axes."""
    half = dim // 2
    return half - 2 * (half // 3), half // 3, half // 3


def _table(dim):
    """Cosines and sines `[rows, dim / 2, 2]`, a band of frequencies for each axis."""
    inv = torch.cat([10000.0 ** (-torch.arange(n, dtype=torch.float64, device=DEV) / n) for n in _axes(dim)])
    angle = torch.arange(TABLE_ROWS, dtype=torch.float64, device=DEV)[:, None] * inv
    return torch.stack([angle.cos(), angle.sin()], dim=-1)


def prepare(case, seed):
    g = _gen(seed)
    if case["kind"] == "attend":
        shape = lambda n, heads: (g, case["batch"], n, heads, case["dim"], case["dtype"])  # noqa: E731
        index, num = _selection(g, case)
        s = dict(case=case, index=index, num=num, q=_tokens(*shape(case["q_len"], case["heads"]), 0.7),
                 k=_tokens(*shape(case["kv_len"], case["kv_heads"]), 0.7), v=_tokens(*shape(case["kv_len"], case["kv_heads"])))
        if case["train"]:
            s["dout"] = _tokens(*shape(case["q_len"], case["heads"]))
            for name in ("q", "k", "v"):
                s[name].requires_grad_()
        return s
    if case["kind"] == "rotary":
        B, L = case["batch"], case["length"]
        # samples of several grids one behind the other: time, height and width of every token
        token = torch.arange(L, device=DEV)[None] + torch.randint(0, 500, (B, 1), generator=g, device=DEV)
        width = torch.randint(10, 60, (B, 1), generator=g, device=DEV)
        height = torch.randint(10, 40, (B, 1), generator=g, device=DEV)
        pos = torch.stack([(token // (width * height)) % TABLE_ROWS, (token // width) % height, token % width], dim=-1).to(torch.int32)
        s = dict(case=case, positions=pos.contiguous(), table=_table(case["dim"]).float(),
                 q=_tokens(g, B, L, case["heads"], case["dim"], case["dtype"]), k=_tokens(g, B, L, case["kv_heads"], case["dim"], case["dtype"]))
        if case["train"]:
            s["dq"], s["dk"] = (_tokens(g, B, L, case[n], case["dim"], case["dtype"]) for n in ("heads", "kv_heads"))
            s["q"].requires_grad_()
            s["k"].requires_grad_()
        return s
    n, m = case["pages"], case["moves"]
    r = torch.randperm(n, generator=torch.Generator().manual_seed(seed))
    if case["how"] == "fork":            # free pages become copies of pages in use
        dst, src = sorted(r[:m].tolist()), r[m:2 * m].tolist()
    elif case["how"] == "roll":          # everything moves to the front
        dst, src = list(range(m)), list(range(n - m, n))
    else:                                # kept pages move together, what lies behind them is cleared
        dst, src = list(range(n)), sorted(r[:m].tolist()) + [None] * (n - m)
    caches = [torch.randint(-2 ** 15, 2 ** 15, (1, n * case["page"], case["row"] * SIZE[case["dtype"]] // 2), generator=g, device=DEV, dtype=torch.int16)
              for _ in range(case["tensors"])]
    # any bits that are a number: moved, never computed with
    caches = [torch.where((c & 0x7f00) == 0x7f00, 0, c).view(DTYPES[case["dtype"]]).view(1, n * case["page"], -1, 128 if case["row"] % 128 == 0 else case["row"]) for c in caches]
    return dict(case=case, caches=caches, dst=dst, src=src)


# ------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------
def _blocks(x, block):
    """`[B, L, H, D]` -> `[B, H, blocks, block, D]`, zeros behind the last token."""
    x = F.pad(x, (0, 0, 0, 0, 0, -x.shape[1] % block))
    return x.unflatten(1, (-1, block)).permute(0, 3, 1, 2, 4)


def _tokens_of(x, length):
    return x.permute(0, 2, 3, 1, 4).flatten(1, 2)[:, :length]


def _attend_plain(q, k, v, index, num, block, dout=None):
    """Softmax attention of every query block over its selected key blocks and, with `dout`, its gradients; in q's type."""
    B, Lq, H, D = q.shape
    Lkv, Hkv = k.shape[1], k.shape[2]
    qb, kb, vb = _blocks(q, block), _blocks(k, block), _blocks(v, block)
    nq, nk, S = qb.shape[2], kb.shape[2], index.shape[-1]
    ids = index.long()
    row = (torch.arange(B, device=q.device)[:, None] * Hkv + torch.arange(H, device=q.device) // (H // Hkv))[..., None, None] * nk + ids
    kg, vg = kb.reshape(B * Hkv * nk, block, D)[row].flatten(3, 4), vb.reshape(B * Hkv * nk, block, D)[row].flatten(3, 4)
    real = (ids[..., None] * block + torch.arange(block, device=q.device) < Lkv) & (torch.arange(S, device=q.device) < num[..., None])[..., None]
    real = real.flatten(3, 4)[..., None, :]                                # [B, H, nq, 1, S * block]
    scale = D ** -0.5
    s = (qb @ kg.transpose(-1, -2) * scale).masked_fill(~real, -math.inf)
    top = s.amax(-1, keepdim=True).clamp(min=torch.finfo(s.dtype).min)
    p = (s - top).exp()
    total = p.sum(-1, keepdim=True)
    lse = (top + total.log()).flatten(2)[..., :Lq]
    p = p / total.clamp(min=torch.finfo(s.dtype).tiny)
    out = p @ vg
    if dout is None:
        return _tokens_of(out, Lq), lse
    do = _blocks(dout, block)
    ds = p * (do @ vg.transpose(-1, -2) - (do * out).sum(-1, keepdim=True)) * scale
    flat = row.flatten()
    sums = lambda x: torch.zeros((B * Hkv * nk, block * D), dtype=x.dtype, device=x.device).index_add_(  # noqa: E731
        0, flat, x.reshape(-1, block * D)).view(B, Hkv, nk, block, D)
    dq, dk, dv = ds @ kg, sums(ds.transpose(-1, -2) @ qb), sums(p.transpose(-1, -2) @ do)
    return _tokens_of(out, Lq), lse, _tokens_of(dq, Lq), _tokens_of(dk, Lkv), _tokens_of(dv, Lkv)


def _rotate(x, cos, sin, interleaved):
    """Pairs of `x [B, L, H, D]` turned by angles given as `cos`, `sin` `[B, L, 1, D / 2]`."""
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else x.chunk(2, dim=-1)
    u, w = a * cos - b * sin, a * sin + b * cos
    return torch.stack([u, w], dim=-1).flatten(-2) if interleaved else torch.cat([u, w], dim=-1)


def _angles(table, positions, dim):
    ends = [sum(_axes(dim)[:i + 1]) for i in range(3)]
    parts = [table[positions[..., i].long(), e - n:e] for i, (e, n) in enumerate(zip(ends, _axes(dim)))]
    return torch.cat(parts, dim=-2)[:, :, None]                            # [B, L, 1, D / 2, 2]


def _rotary_plain(x, angles, interleaved, back=False):
    return _rotate(x, angles[..., 0], -angles[..., 1] if back else angles[..., 1], interleaved)


def run(s):
    case = s["case"]
    if case["kind"] == "attend":
        if own:
            from worldattention_b200.hsa import selected_attention
            out, lse = selected_attention(s["q"], s["k"], s["v"], s["index"], s["num"], case["block"], return_lse=True)
            if not case["train"]:
                return dict(out=out, lse=lse)
            dq, dk, dv = torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["dout"])
            return dict(out=out.detach(), lse=lse.detach(), dq=dq, dk=dk, dv=dv)
        kind = DTYPES[case["dtype"]]
        names = ("out", "lse", "dq", "dk", "dv")
        with torch.no_grad():
            got = _attend_plain(s["q"].float(), s["k"].float(), s["v"].float(), s["index"], s["num"], case["block"],
                                s["dout"].float() if case["train"] else None)
            return {n: x if n == "lse" else x.to(kind) for n, x in zip(names, got)}
    if case["kind"] == "rotary":
        if own:
            from worldattention_b200.rope import axial_rope
            q, k = axial_rope((s["q"], s["k"]), s["positions"], s["table"], axes=_axes(case["dim"]), interleaved=case["interleaved"])
            if not case["train"]:
                return dict(q=q, k=k)
            dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
            return dict(q=q.detach(), k=k.detach(), dq=dq, dk=dk)
        with torch.no_grad():
            angles = _angles(s["table"], s["positions"], case["dim"])
            turn = lambda x, back: _rotary_plain(x.float(), angles, case["interleaved"], back).to(x.dtype)  # noqa: E731
            got = dict(q=turn(s["q"], False), k=turn(s["k"], False))
            if case["train"]:
                got.update(dq=turn(s["dq"], True), dk=turn(s["dk"], True))
            return got
    if own:
        from worldattention_b200.hkv import move_pages
        move_pages(s["caches"], s["dst"], s["src"], case["page"])
        return s["caches"]
    to = torch.tensor([d for d, p in zip(s["dst"], s["src"]) if p is not None], device=DEV)
    at = torch.tensor([p for p in s["src"] if p is not None], device=DEV)
    free = torch.tensor([d for d, p in zip(s["dst"], s["src"]) if p is None], device=DEV, dtype=torch.long)
    for c in s["caches"]:
        paged = c.unflatten(1, (-1, case["page"]))
        paged[:, to] = paged[:, at]
        paged[:, free] = 0
    return s["caches"]


# ------------------------------------------------------------------------------------------------
# what a pass cannot do without, and what it gives in 64 bits
# ------------------------------------------------------------------------------------------------
def work(case):
    if case["kind"] == "attend":
        B, Lq, Lkv, H, Hkv, D, e = (case[n] for n in ("batch", "q_len", "kv_len", "heads", "kv_heads", "dim", "dtype"))
        e = SIZE[e]
        rows, share = B * Lq * H, 0.5 if case["ragged"] else 1.0
        nq = -(-Lq // case["block"])
        keys = min(Lkv, case["select"] * case["block"] * share)             # that a row attends to
        # keys and values that some row attends to, as far as the call's rows can reach
        reached = B * min(Lkv * Hkv, H * nq * keys) * D * e
        queries = rows * D * e
        if case["train"]:                       # q, k, v, dout in; out, lse, dq, dk, dv out; two products forward, five back
            return {"bytes": 4 * queries + 4 * rows + 2 * reached + 2 * B * Lkv * Hkv * D * e, "flops": 14.0 * D * rows * keys}
        return {"bytes": 2 * queries + 4 * rows + 2 * reached, "flops": 4.0 * D * rows * keys}
    if case["kind"] == "rotary":
        n = case["batch"] * case["length"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        passes = 2 if case["train"] else 1
        return {"bytes": 2.0 * n * SIZE[case["dtype"]] * passes + 12 * case["batch"] * case["length"], "flops": 3.0 * n * passes}
    page = case["page"] * case["row"] * SIZE[case["dtype"]] * case["tensors"]
    if case["how"] == "compact":                # every page is written, the kept ones are read
        return {"bytes": page * (case["pages"] + case["moves"]), "flops": 0}
    return {"bytes": 2.0 * page * case["moves"], "flops": 0}


def exact(case, seed):
    """The definition in 64 bits, a (batch, head) at a time; moved pages are not computed, so they have none."""
    if case["kind"] == "pages" or case["kind"] == "attend" and case["q_len"] * case["select"] * case["block"] * case["heads"] > 2 ** 29:
        return None
    s = prepare(case, seed)
    with torch.no_grad():
        if case["kind"] == "rotary":
            table, pos = s["table"].double(), s["positions"].long()
            owner = torch.repeat_interleave(torch.arange(3, device=DEV), torch.tensor(_axes(case["dim"]), device=DEV))   # axis of each pair
            at = pos[..., owner]                                                                     # [B, L, D / 2]
            turn = torch.complex(table[..., 0], table[..., 1])[at, torch.arange(case["dim"] // 2, device=DEV)][:, :, None]

            def by(x, t):
                x = x.double().unflatten(-1, (-1, 2) if case["interleaved"] else (2, -1))
                x = x if case["interleaved"] else x.transpose(-1, -2)
                y = torch.view_as_real(torch.view_as_complex(x.contiguous()) * t)
                return (y if case["interleaved"] else y.transpose(-1, -2)).flatten(-2)
            got = dict(q=by(s["q"], turn), k=by(s["k"], turn))
            if case["train"]:
                got.update(dq=by(s["dq"], turn.conj()), dk=by(s["dk"], turn.conj()))
            return got
        B, Lq, H, D = s["q"].shape
        Lkv, Hkv, block = case["kv_len"], case["kv_heads"], case["block"]
        q, k, v = (s[n].double() for n in ("q", "k", "v"))
        got = dict(out=torch.zeros_like(q), lse=torch.full((B, H, Lq), -math.inf, dtype=torch.float64, device=DEV))
        if case["train"]:
            do = s["dout"].double()
            got.update(dq=torch.zeros_like(q), dk=torch.zeros_like(k), dv=torch.zeros_like(v))
        of_key = torch.arange(Lkv, device=DEV) // block
        picked = torch.zeros((B, H, -(-Lq // block), -(-Lkv // block)), dtype=torch.bool, device=DEV)
        for j in range(case["select"]):
            picked.scatter_(-1, s["index"][..., j:j + 1].long(), (s["num"] > j)[..., None] | picked.gather(-1, s["index"][..., j:j + 1].long()))
        step = max(block, 2 ** 27 // Lkv // block * block)
        for b in range(B):
            for h in range(H):
                kk, vv = k[b, :, h * Hkv // H], v[b, :, h * Hkv // H]
                for r in range(0, Lq, step):
                    rows = slice(r, min(Lq, r + step))
                    mask = picked[b, h][torch.arange(rows.start, rows.stop, device=DEV) // block][:, of_key]
                    z = (q[b, rows, h] @ kk.T / math.sqrt(D)).masked_fill(~mask, -math.inf)
                    lse = torch.logsumexp(z, dim=-1)
                    p = (z - lse.clamp(min=-1e300)[:, None]).exp()
                    got["lse"][b, h, rows] = lse
                    got["out"][b, rows, h] = o = p @ vv
                    if case["train"]:
                        g = do[b, rows, h]
                        dz = p * (g @ vv.T - (g * o).sum(-1, keepdim=True)) / math.sqrt(D)
                        got["dq"][b, rows, h] = dz @ kk
                        got["dk"][b, :, h * Hkv // H] += dz.T @ q[b, rows, h]
                        got["dv"][b, :, h * Hkv // H] += p.T @ g
        return got
