"""Training steps captured while an eager graph of their leaves is alive, where a leaf lies behind products of several inputs."""
import pytest
import torch

from tests.helpers import dev
from tests.test_selected_attention import _inputs, _lists


def _case():
    g = torch.Generator(device=dev()).manual_seed(1)
    q, k, v, dout = _inputs(g, 1, 70, 130, 4, 4, 128, torch.bfloat16)
    index, num = _lists(g, 1, 4, 2, 3, 2, "full")
    x, w = (torch.randn(n, 512, generator=g, device=dev()).bfloat16() for n in (70, 512))
    return q, k, v, dout, index, num, x, w


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["attend", "turn", "both"])
def test_a_leaf_behind_a_product(which):
    from worldattention_b200.hsa import selected_attention
    from worldattention_b200.rope import axial_rope
    _, k, v, dout, index, num, x, w = _case()
    pos, table = torch.zeros(70, 1, dtype=torch.int32, device=dev()), torch.ones(1, 64, 2, device=dev())
    w.requires_grad_()
    attend, turn = lambda q: selected_attention(q, k, v, index, num, 64), lambda q: axial_rope(q, pos, table)  # noqa: E731
    call = {"attend": attend, "turn": turn, "both": lambda q: attend(turn(q))}[which]
    q_of = lambda: (x @ w / 16).view(1, 70, 4, 128)  # noqa: E731
    want, = torch.autograd.grad(call(q_of()), w, dout)
    alive = q_of()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="eager graph"):
        with torch.cuda.graph(graph):
            call(q_of()).backward(dout)
    assert w.grad is None
    # a pass that ends before the leaf may be captured, and so may the forward pass
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q = q_of()
        dq, = torch.autograd.grad(call(q), q, dout)
    graph.replay()
    torch.cuda.synchronize()
    assert bool(torch.isfinite(dq).all()) and bool(dq.any())
    del alive, q, dq
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(q_of()).backward(dout)
    w.grad.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(w.grad, want)


@pytest.mark.gpu
def test_a_forward_pass_of_block_sparse_attention_is_captured_over_an_eager_graph():
    from worldattention_b200.hsa import block_sparse_attention_reference
    q, k, v, dout, index, num, _, _ = _case()
    q, k, v, dout = (x[:, :64].transpose(1, 2).contiguous() for x in (q, k, v, dout))
    index, num = torch.zeros(1, 4, 1, 1, dtype=torch.int32, device=dev()), torch.ones(1, 4, 1, dtype=torch.int32, device=dev())
    sizes = torch.tensor([50], dtype=torch.int32, device=dev())
    q.requires_grad_()
    call = lambda: block_sparse_attention_reference(q, k, v, index, num, sizes, 64)  # noqa: E731
    alive = call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out.detach(), alive.detach())
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="eager graph"):
        with torch.cuda.graph(graph):
            call().backward(dout)
    assert q.grad is None
