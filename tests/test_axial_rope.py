"""The rotary embedding of tokens with positions of their own on several axes, against the turn of complex numbers in 64 bits."""
import pytest
import torch

from tests.helpers import dev


def _table(rows, pairs, device):
    inv = 10000.0 ** (-torch.arange(pairs, dtype=torch.float64, device=device) / pairs)
    return torch.polar(torch.ones(rows, pairs, dtype=torch.float64, device=device), torch.arange(rows, dtype=torch.float64, device=device)[:, None] * inv)


def _want(x, pos, table, axes, interleaved):
    """Complex product in 64 bits; `table` complex [rows, pairs]."""
    pairs = sum(axes)
    owner = torch.repeat_interleave(torch.arange(len(axes), device=x.device), torch.tensor(axes, device=x.device))
    at = pos[..., owner].long()                                              # [(B,) L, pairs]
    turn = table[at, torch.arange(pairs, device=x.device)]
    turn = (turn if turn.dim() == 3 else turn[None])[:, :, None]
    x = x.double()
    a, b = (x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2]) if interleaved else (x[..., :pairs], x[..., pairs:2 * pairs])
    z = torch.complex(a, b) * turn
    head = torch.stack([z.real, z.imag], -1).flatten(-2) if interleaved else torch.cat([z.real, z.imag], -1)
    return torch.cat([head, x[..., 2 * pairs:]], -1)


def _close(got, want, angle_error):
    """Half a step of the result's type, and in float32 the table's rounding (2^-24 of cos and sin) and three more: each relative to
    the pair's length, which a turn keeps."""
    got, want = got.double(), want.double()
    length = want.abs().amax(-1, keepdim=True)          # of the longest pair, at most its channels' largest times sqrt(2)
    step = torch.finfo(torch.bfloat16).eps / 2 if angle_error == "bf16" else 0.0
    bound = step * want.abs() + 2 ** 0.5 * 2 * length * 5 * 2 ** -24
    assert bool(((got - want).abs() <= bound).all()), float(((got - want).abs() - bound).max())


CASES = [  # batch, length, heads of q and k, head_dim, axes, positions per sample
    (1, 1, (12, 12), 128, (22, 21, 21), True), (3, 5, (4, 1), 128, (22, 21, 21), True), (2, 257, (12, 4), 128, (22, 21, 21), False),
    (2, 33, (3, 2), 96, (16, 16, 16), True), (1, 40, (5, 5), 64, (32,), False), (2, 19, (2, 1), 80, (8, 8), True),       # 80: 2 * 16 turned, 48 copied
    (1, 7, (3, 1), 24, (4, 4, 4), True), (1, 9, (2, 2), 10, (1, 2, 1), True), (2, 6, (33, 1), 256, (64, 64), True), (1, 2100, (12, 12), 128, (64,), True),
    (1, 3, (1, 1), 2, (1,), True), (1, 12, (2, 2), 128, (8, 8, 8, 8, 8, 8, 8, 8), True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("case", CASES)
def test_values_and_gradients(case, interleaved, dtype):
    from worldattention_b200.rope import axial_rope
    B, L, heads, D, axes, own = case
    g = torch.Generator(device=dev()).manual_seed(L)
    rows = 700
    table = _table(rows, sum(axes), dev())
    pos = torch.randint(0, rows, (B, L, len(axes)) if own else (L, len(axes)), generator=g, device=dev(), dtype=torch.int32)
    xs = [torch.randn(B, L, h, D, generator=g, device=dev()).to(dtype).requires_grad_() for h in heads]
    ys = axial_rope(tuple(xs), pos, table, axes=axes, interleaved=interleaved)
    kind = "bf16" if dtype == torch.bfloat16 else "fp32"
    gs = [torch.randn(y.shape, generator=g, device=dev()).to(dtype) for y in ys]
    dxs = torch.autograd.grad(ys, xs, gs)
    for x, y, gy, dx in zip(xs, ys, gs, dxs):
        assert y.dtype == dtype and y.is_contiguous() and dx.dtype == dtype
        _close(y.detach(), _want(x.detach(), pos, table, axes, interleaved), kind)
        _close(dx, _want(gy, pos, table.conj().resolve_conj(), axes, interleaved), kind)
    with torch.no_grad():
        one = axial_rope(xs[1], pos, torch.view_as_real(table).float(), axes=axes, interleaved=interleaved)
    assert torch.equal(one, ys[1])


@pytest.mark.gpu
def test_gradient_against_differences():
    from worldattention_b200.rope import axial_rope
    g = torch.Generator(device=dev()).manual_seed(5)
    table, pos = _table(50, 12, dev()), torch.randint(0, 50, (2, 6, 3), generator=g, device=dev(), dtype=torch.int32)
    x = torch.randn(2, 6, 2, 28, generator=g, device=dev(), requires_grad=True)
    gy, step = torch.randn(2, 6, 2, 28, generator=g, device=dev()), torch.randn(2, 6, 2, 28, generator=g, device=dev())
    f = lambda t: float((axial_rope(t, pos, table).double() * gy).sum())  # noqa: E731
    dx, = torch.autograd.grad(axial_rope(x, pos, table), x, gy)
    with torch.no_grad():
        slope = (f(x + step) - f(x - step)) / 2          # a turn is linear: exact but for 672 roundings to float32 of values below about 6
    assert abs(slope - float((dx.double() * step).sum())) < 672 * 6 * 6 * 2 ** -22
    again, = torch.autograd.grad(axial_rope(x, pos, table), x, gy, create_graph=True)
    assert not again.requires_grad or again.grad_fn is not None
    w = gy.clone().requires_grad_()
    dx2, = torch.autograd.grad(axial_rope(x, pos, table), x, w, create_graph=True)
    back, = torch.autograd.grad(dx2, w, step)            # the gradient of the gradient is the turn itself
    assert torch.equal(back, axial_rope(step, pos, table))


@pytest.mark.gpu
def test_the_grid_of_causal_rope_apply_is_a_case():
    from worldattention_b200.causal_dit import rope_table
    from worldattention_b200.rope import axial_rope, causal_rope_apply
    x = torch.randn(1, 2 * 3 * 5, 4, 128, device=dev()).bfloat16()
    t, h, w = torch.meshgrid(torch.arange(7, 9), torch.arange(3), torch.arange(5), indexing="ij")
    pos = torch.stack([t, h, w], -1).flatten(0, 2).to(dev())
    table = rope_table(128).to(dev())
    got, want = axial_rope(x, pos, table).float(), causal_rope_apply(x, (2, 3, 5), table, 7).float()
    # both are within half a step of the exact value and float32's error of it: they differ only where that crosses a border
    assert float((got != want).float().mean()) < 1e-3 and bool(((got - want).abs() <= 2 ** -7 * want.abs() + 1e-6).all())


@pytest.mark.gpu
def test_strides_positions_outside_and_nothing():
    from worldattention_b200.rope import axial_rope
    table = _table(30, 64, dev())
    both = torch.randn(2, 11, 6, 2, 128, device=dev()).bfloat16()            # q and k side by side, heads before tokens
    q, k = both[:, :, :4, 0], both.permute(0, 2, 1, 3, 4).contiguous().permute(0, 2, 1, 3, 4)[:, :, 1:3, 1]
    pos = torch.randint(0, 30, (2, 11, 4), device=dev(), dtype=torch.int32)[..., 1:]      # rows with a gap
    for got, x in zip(axial_rope((q, k), pos, table, axes=(20, 22, 22)), (q, k)):
        _close(got, _want(x, pos, table, (20, 22, 22), True), "bf16")
    wide = torch.randn(2, 11, 3, 256, device=dev())
    x = wide[..., ::2]                                                          # last axis with a stride
    _close(axial_rope(x, pos, table), _want(x, pos, table, (22, 21, 21), True), "fp32")
    x = wide[..., 1:129]                                                        # rows that begin at an odd place
    _close(axial_rope(x, pos, table), _want(x, pos, table, (22, 21, 21), True), "fp32")
    e = torch.randn(2, 1, 3, 128, device=dev()).expand(2, 11, 3, 128).requires_grad_()
    y = axial_rope(e, pos, table)
    dx, = torch.autograd.grad(y, e, torch.ones((), device=dev()).expand(y.shape))         # a gradient without memory of its own
    _close(dx, _want(torch.ones(2, 11, 3, 128, device=dev()), pos, table.conj().resolve_conj(), (22, 21, 21), True), "fp32")
    bad = pos.clone()
    bad[0, 3, 1], bad[1, 4, 0], bad[1, 5, 2] = 30, -1, 2 ** 31 - 1
    y = axial_rope(q, bad, table)
    nan = torch.isnan(y)
    assert bool(nan[0, 3, :, 44:86].all()) and bool(nan[1, 4, :, :44].all()) and bool(nan[1, 5, :, 86:].all()) and int(nan.sum()) == 4 * (42 + 44 + 42)
    far = pos.long()
    far[0, 0, 0] = 2 ** 32                                                      # not row 0 once converted
    assert bool(torch.isnan(axial_rope(q, far, table)[0, 0, :, :44]).all())
    assert axial_rope(q[:, :0], pos[:, :0], table).shape == (2, 0, 4, 128) and axial_rope(q[:, :, :0], pos, table).shape == (2, 11, 0, 128)
    inf = torch.full((2, 11, 1, 132), float("inf"), device=dev())               # channels that are not turned are copies
    assert bool((axial_rope(inf, pos, table)[..., 128:] == float("inf")).all())


@pytest.mark.gpu
def test_captured_and_on_another_stream():
    from worldattention_b200.rope import axial_rope
    table = torch.view_as_real(_table(30, 64, dev())).float()
    x, gy = torch.randn(1, 50, 4, 128, device=dev()).bfloat16().requires_grad_(), torch.randn(1, 50, 4, 128, device=dev()).bfloat16()
    pos = torch.randint(0, 30, (50, 3), device=dev(), dtype=torch.int32)
    want = torch.autograd.grad(axial_rope(x, pos, table), x, gy)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        leaf = x.detach().clone().requires_grad_()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got, = torch.autograd.grad(axial_rope(leaf, pos, table), leaf, gy)
        got.zero_()
        graph.replay()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.int16, torch.int64, torch.uint16, torch.uint32, torch.uint64])
def test_positions_of_every_integer_type(dtype):
    from worldattention_b200.rope import axial_rope
    rows = 40000                                                                # more than 8 and 16 bits with a sign hold
    table = torch.view_as_real(_table(rows, 16, dev())).float()
    x = torch.randn(2, 9, 3, 32, device=dev())
    pos = torch.randint(0, 128, (2, 9, 1), device=dev(), dtype=torch.int32)
    assert torch.equal(axial_rope(x, pos.to(dtype), table), axial_rope(x, pos, table))


@pytest.mark.gpu
def test_refusals():
    from worldattention_b200.rope import axial_rope
    x, table = torch.randn(2, 5, 3, 16, device=dev()), _table(9, 8, dev())
    pos = torch.zeros(2, 5, 3, device=dev(), dtype=torch.int32)
    for call, word in [(lambda: axial_rope(x, pos[:, :4], table), "positions"), (lambda: axial_rope(x, pos[:1], table), "positions"),
                       (lambda: axial_rope(x, pos.float(), table), "integers"), (lambda: axial_rope(x, pos[..., :2], table), "axes"),
                       (lambda: axial_rope(x, pos, table, axes=(4, 4)), "positions"), (lambda: axial_rope(x, pos, table, axes=(4, 4, 4)), "pairs"),
                       (lambda: axial_rope(x, pos, _table(9, 9, dev())), "pairs"), (lambda: axial_rope(x[0], pos, table), "B, L, H, D"),
                       (lambda: axial_rope((x, x[:, :4]), pos, table), "share"), (lambda: axial_rope((x, x.bfloat16()), pos, table), "share"),
                       (lambda: axial_rope(x.half(), pos, table), "float32 or bfloat16"), (lambda: axial_rope((x,) * 5, pos, table), "four"),
                       (lambda: axial_rope(x, pos, table, axes=(9, -1, 0)), "pairs")]:
        with pytest.raises(ValueError, match=word):
            call()


@pytest.mark.gpu
def test_a_learned_table_is_refused_instead_of_left_without_its_gradient():
    from worldattention_b200.rope import axial_rope
    x, pos = torch.randn(2, 5, 3, 16, device=dev()), torch.zeros(5, 1, device=dev(), dtype=torch.int32)
    real = torch.randn(9, 8, 2, device=dev(), requires_grad=True)
    for table in (real, torch.view_as_complex(real), real.double()):
        for y in (x, x.detach().requires_grad_()):
            with pytest.raises(ValueError, match="gradient"):
                axial_rope(y, pos, table)
    with torch.no_grad():
        axial_rope(x, pos, real)


def test_no_cpu_path():
    from worldattention_b200.rope import axial_rope
    with pytest.raises(RuntimeError, match="CUDA"):
        axial_rope(torch.zeros(1, 2, 1, 8), torch.zeros(2, 1, dtype=torch.int32), torch.zeros(4, 4, 2))
