"""Tangents of forward-mode derivatives: the operators that would lose them refuse the call."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from tests.helpers import dev


@pytest.mark.gpu
@pytest.mark.parametrize("grad", [False, True])
def test_a_tangent_is_refused(grad):
    from worldattention_b200.hkv import move_pages
    from worldattention_b200.hsa import selected_attention
    from worldattention_b200.rope import axial_rope
    g = torch.Generator(device=dev()).manual_seed(1)
    r = lambda *shape: torch.randn(*shape, generator=g, device=dev())  # noqa: E731
    q, k, v = r(1, 70, 4, 32), r(1, 130, 2, 32), r(1, 130, 2, 32)
    index, num = torch.zeros(1, 4, 2, 1, dtype=torch.int32, device=dev()), torch.ones(1, 4, 2, dtype=torch.int32, device=dev())
    pos, table = torch.zeros(70, 1, dtype=torch.int32, device=dev()), r(1, 16, 2)
    want = selected_attention(q, k, v, index, num, 64), axial_rope(q, pos, table)
    with forward_ad.dual_level():
        dual = lambda x: forward_ad.make_dual(x.clone().requires_grad_(grad), torch.randn_like(x))  # noqa: E731
        for call in (lambda: selected_attention(dual(q), k, v, index, num, 64), lambda: selected_attention(q, dual(k), v, index, num, 64),
                     lambda: selected_attention(q, k, dual(v), index, num, 64), lambda: axial_rope(dual(q), pos, table), lambda: axial_rope((q, dual(k[:, :70])), pos, table),
                     lambda: axial_rope(q, pos, forward_ad.make_dual(table, table))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        with pytest.raises((NotImplementedError, RuntimeError), match="forward-mode|in place"):
            move_pages([dual(q)], [0], [1], 10)
        # inside a level, what has no tangent is computed as ever
        assert torch.equal(selected_attention(q, k, v, index, num, 64), want[0]) and torch.equal(axial_rope(q, pos, table), want[1])
        leaf = q.clone().requires_grad_()
        assert torch.autograd.grad(selected_attention(leaf, k, v, index, num, 64).sum(), leaf)[0].shape == q.shape
    with pytest.raises(RuntimeError):      # a tensor that a function transform has wrapped has no memory
        torch.func.jvp(lambda x: selected_attention(x, k, v, index, num, 64), (q,), (torch.ones_like(q),))
