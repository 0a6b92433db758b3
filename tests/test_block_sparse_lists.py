"""`block_sparse_attention` under autograd: the values, layout and arguments of the call without gradients, whatever its lists hold."""
import pytest
import torch

from tests.helpers import dev
from tests.test_selected_attention import _check, _exact, _inputs, _mask


def _laid_out(q, k, v, dout, index, num, sizes, block):
    """The lists as they are -- an id that is named again counts again, one that is no block is the nearest one -- as lists of sets: every entry of
    every row has key blocks of its own.  -> what `_exact` gives, folded back to the keys, its bounds added up."""
    B, H, nq, S = index.shape
    n = k.shape[1] // block
    ids = index.clamp(0, n - 1).long().view(B, H, nq * S)
    at = (ids[..., None] * block + torch.arange(block, device=dev())).flatten(2)[..., None].expand(-1, -1, -1, k.shape[-1])     # [B, H, tokens, D]
    take = lambda x: x.transpose(1, 2).gather(2, at).transpose(1, 2)  # noqa: E731
    own = torch.arange(nq * S, dtype=torch.int32, device=dev()).view(1, 1, nq, S).expand(B, H, nq, S)
    mask = _mask(own, num.clamp(max=S), block, q.shape[1], nq * S * block)
    real = (torch.arange(block, device=dev()) < sizes[ids][..., None]).flatten(2)[:, :, None]
    want = _exact(q, take(k), take(v), mask & real, dout)
    fold = lambda x: torch.zeros(B, H, k.shape[1], k.shape[-1], dtype=x.dtype, device=dev()).scatter_add_(2, at, x.transpose(1, 2)).transpose(1, 2)  # noqa: E731
    return {n: (fold(x), fold(e)) if n in ("dk", "dv") else (x, e) for n, (x, e) in want.items()}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D,block", [(torch.bfloat16, 128, 64), (torch.float32, 128, 64), (torch.float32, 64, 32), (torch.bfloat16, 128, 128), (torch.bfloat16, 40, 16)])
@pytest.mark.parametrize("nq,nk", [(2, 4), (9, 7), (40, 3)])
def test_lists_count_as_they_do_without_gradients(dtype, D, block, nq, nk):
    from worldattention_b200.hsa import block_sparse_attention_reference
    g = torch.Generator(device=dev()).manual_seed(D + nq)
    B, H, S = 2, 3, 6
    q, k, v, dout = _inputs(g, B, nq * block, nk * block, H, H, D, dtype)
    index = torch.randint(-2, nk + 3, (B, H, nq, S), generator=g, device=dev()).to(torch.int32)
    index[..., 1::3] = index[..., 0:1]                                           # named again
    num = torch.randint(0, S + 3, (B, H, nq), generator=g, device=dev()).to(torch.int32)
    num[0, 0, 0], num[1, 0, 0] = -2, 0
    sizes = torch.randint(1, block + 1, (nk,), generator=g, device=dev()).to(torch.int32)
    sizes[1] = 0
    t = lambda x: x.transpose(1, 2)  # noqa: E731
    with torch.no_grad():
        want, lse = block_sparse_attention_reference(t(q), t(k), t(v), index, num, sizes, block, return_lse=True)
    leaves = [t(x).contiguous().requires_grad_() for x in (q, k, v)]
    out, lse2 = block_sparse_attention_reference(*leaves, index, num, sizes, block, return_lse=True)
    assert torch.equal(out.detach(), want) and torch.equal(lse2, lse) and out.requires_grad and not lse2.requires_grad
    assert out.is_contiguous() and out.detach().view(-1).shape == (q.numel(),)
    grads = torch.autograd.grad(out, leaves, t(dout))
    got = {"out": t(out.detach()), "lse": lse2, **{n: t(x) for n, x in zip(("dq", "dk", "dv"), grads)}}
    _check(got, _laid_out(q, k, v, dout, index, num, sizes, block))


@pytest.mark.gpu
def test_more_sizes_than_blocks_and_heads_side_by_side():
    """What the call without gradients takes: sizes of blocks behind the last one, inputs whose heads lie inside the tokens."""
    from worldattention_b200.hsa import block_sparse_attention_reference
    g = torch.Generator(device=dev()).manual_seed(2)
    q, k, v, dout = _inputs(g, 1, 128, 256, 2, 2, 128, torch.bfloat16)
    index = torch.tensor([[0, 3], [1, 2]], dtype=torch.int32, device=dev()).expand(1, 2, 2, 2).contiguous()
    num = torch.full((1, 2, 2), 2, dtype=torch.int32, device=dev())
    sizes = torch.tensor([64, 64, 60, 64, 7, 9], dtype=torch.int32, device=dev())
    t = lambda x: x.transpose(1, 2)  # noqa: E731
    with torch.no_grad():
        want = block_sparse_attention_reference(t(q), t(k), t(v), index, num, sizes, 64)
    leaves = [x.requires_grad_() for x in (q, k, v)]
    out = block_sparse_attention_reference(*map(t, leaves), index, num, sizes, 64)
    assert torch.equal(out, want) and out.is_contiguous()
    got = dict(zip(("dq", "dk", "dv"), torch.autograd.grad(out, leaves, t(dout))), out=t(out.detach()))
    exact = _exact(q.detach(), k.detach(), v.detach(), _mask(index, num, 64, 128, 256, sizes), dout)
    _check(got, {n: e for n, e in exact.items() if n != "lse"})
