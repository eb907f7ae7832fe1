"""Calls of layer norm and packed attention at the edge of what they promise: other kinds of derivatives."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch.device("cuda:0")


def calls(dev):
    """(operator, its tensors) for every differentiable call."""
    from gnn_amd import layer_norm, packed_attention, packed_segments, relative_buckets
    g = torch.Generator(device=dev)
    g.manual_seed(1)
    seg = packed_segments([5, 9], dev)
    codes = relative_buckets(seg, 4, 8)
    q, k, v = (torch.randn(14, h, 8, generator=g, device=dev) for h in (4, 2, 2))
    x, w, b = torch.randn(6, 8, generator=g, device=dev), torch.ones(8, device=dev), torch.zeros(8, device=dev)
    return [(lambda *t: layer_norm(*t), [x, w, b]), (lambda *t: packed_attention(*t, seg, causal=True), [q, k, v]),
            (lambda *t: packed_attention(*t[:3], seg, bias=t[3], buckets=codes),
             [q, k, v, torch.zeros(4, 4, device=dev)])]


def test_forward_mode_derivatives_are_refused(dev):
    """A tangent is never dropped in silence: not that of an input, with or without a graph, nor that of a gradient."""
    import torch.autograd.forward_ad as fwd
    for op, tensors in calls(dev):
        want = op(*tensors)
        for at in range(len(tensors)):
            for graph in (False, True):
                with fwd.dual_level(), torch.set_grad_enabled(graph):
                    dual = [fwd.make_dual(t, torch.ones_like(t)) if i == at else t for i, t in enumerate(tensors)]
                    if graph:
                        dual[at].requires_grad_()
                    with pytest.raises(RuntimeError):
                        op(*dual)
        with pytest.raises(RuntimeError):
            torch.func.jvp(lambda t: op(t, *tensors[1:]), (tensors[0],), (torch.ones_like(tensors[0]),))
        with fwd.dual_level():                                    # plain tensors are as welcome as ever
            assert torch.equal(op(*tensors), want)
            leaves = [t.clone().requires_grad_() for t in tensors]
            out = op(*leaves)
            torch.autograd.grad(out, leaves, torch.ones_like(out), retain_graph=True)
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(out, leaves, fwd.make_dual(torch.ones_like(out), torch.ones_like(out)))
