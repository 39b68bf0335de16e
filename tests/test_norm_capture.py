"""A differentiable call under graph capture is refused while an eager autograd graph of the same leaves lives that was made on the default
stream (the captured backward pass would end the process).  Where that is tested nothing is captured: the stream is said to be capturing."""
import gc

import pytest
import torch


class _Node(torch.autograd.Function):
    """holds what group_norm_act's node holds"""

    @staticmethod
    def forward(ctx, x, w, graph):
        ctx.graph = graph
        return x * w

    @staticmethod
    def backward(ctx, dy):
        return dy, dy, None


def test_a_leaf_is_held_as_long_as_its_graph(monkeypatch):
    from alphazero_amd import ops
    from alphazero_amd.engine import EngineError

    capturing, default = [False], [True]
    monkeypatch.setattr(ops, "_capturing", lambda: capturing[0])
    monkeypatch.setattr(ops, "_on_default_stream", lambda device: default[0])
    x, w, other = torch.ones(3), torch.ones(3, requires_grad=True), torch.ones(3, requires_grad=True)

    def enter(*ts):
        return ops._enter_graph([t for t in ts if t is not None])

    def refused(*ts):
        capturing[0] = True
        try:
            enter(*ts)
        except EngineError as e:
            assert "eager autograd graph" in str(e)
            return True
        finally:
            capturing[0] = False
        return False

    assert enter(x) is None and not refused(x, w)  # nothing to differentiate; no graph alive
    loss = _Node.apply(x, w, enter(x, w)).sum()
    assert refused(x, w) and refused(w) and not refused(other) and not refused(x)
    with torch.no_grad():
        assert not refused(w)
    loss.backward()
    assert refused(w)  # (a loss that is kept keeps its graph)
    del loss
    gc.collect()
    assert not refused(w)
    capturing[0] = True
    y = _Node.apply(x, w, enter(x, w))  # a graph made under capture does not stand in the way of the next
    capturing[0] = False
    assert not refused(w)
    hidden = w * 1  # not a leaf
    assert enter(hidden) is None
    del y, hidden
    default[0] = False
    side = _Node.apply(x, w, enter(x, w))  # nor does one made on a side stream,
    assert not refused(w)
    del side
    default[0] = True
    first = _Node.apply(x, w, enter(x, w))
    default[0] = False
    side = _Node.apply(x, w, enter(x, w))  # but for one that shares the node of a default-stream graph, which it keeps
    del first
    gc.collect()
    assert refused(w)
    del side
    gc.collect()
    assert not refused(w)


@pytest.mark.gpu
def test_group_norm_act_refuses_and_goes_on(monkeypatch):
    from alphazero_amd import ops
    from alphazero_amd.engine import EngineError
    from alphazero_amd.nets import GroupNormAct

    norm = GroupNormAct(2, 8).cuda()
    x = torch.randn(2, 8, 5, 5, device="cuda")
    kept = norm(x)
    want = kept.detach().clone()
    monkeypatch.setattr(ops, "_capturing", lambda: True)
    with pytest.raises(EngineError, match="eager autograd graph"):
        norm(x)
    with torch.no_grad():
        assert torch.equal(norm(x), want)
    kept.sum().backward()  # the eager graph is as it was
    del kept
    gc.collect()
    y = norm(x)
    assert torch.equal(y, want)
    y.sum().backward()


@pytest.mark.gpu
def test_make_graphed_callables():
    """forward and backward captured by torch's own means, which keeps the graph of its warm-up on a side stream"""
    from alphazero_amd.nets import GroupNormAct

    torch.manual_seed(0)
    norm = GroupNormAct(2, 8).cuda()
    plain = GroupNormAct(2, 8).cuda()
    last = lambda t: t.contiguous(memory_format=torch.channels_last)
    graphed = torch.cuda.make_graphed_callables(norm, (last(torch.randn(4, 8, 9, 9, device="cuda")).requires_grad_(True),))
    for seed in range(3):
        x = last(torch.randn(4, 8, 9, 9, device="cuda")).requires_grad_(True)
        xp = x.detach().clone().requires_grad_(True)
        dy = last(torch.randn(4, 8, 9, 9, device="cuda"))
        y, yp = graphed(x), plain(xp)
        assert torch.equal(y, yp)
        got = torch.autograd.grad(y, [x, *norm.parameters()], dy)
        want = torch.autograd.grad(yp, [xp, *plain.parameters()], dy)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        del y, yp, got, want
