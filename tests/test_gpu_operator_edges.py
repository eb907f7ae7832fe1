"""Calls of layer norm and packed attention at the edge of what they promise."""
import math

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


def test_codes_made_on_another_stream_than_their_segments(dev):
    """Lists dropped while a stream that was not theirs still lays out codes from them: their memory stays."""
    from gnn_amd import packed_segments, pair_buckets, relative_buckets
    lengths = [700, 3, 90]
    flat = torch.randint(0, 9, (sum(n * n for n in lengths),), device=dev).to(torch.uint8)
    make = (lambda seg: pair_buckets(seg, flat), lambda seg: relative_buckets(seg, 8, 100))
    side = torch.cuda.Stream()
    for one in make:
        want = one(packed_segments(lengths, dev))
        seg = packed_segments(lengths, dev)
        at, size = seg._arrays.data_ptr(), seg._arrays.numel()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            busy = torch.randn(2048, 2048, device=dev)
            for _ in range(20):
                busy = busy @ busy * 1e-2
            got = one(seg)
        got.segments = want.segments
        del seg
        taken = [torch.empty(size, dtype=torch.int32, device=dev) for _ in range(20)]
        still = not side.query()
        assert not (still and at in [t.data_ptr() for t in taken])
        torch.cuda.synchronize()
        assert torch.equal(got._codes, want._codes) and torch.equal(got._by_key, want._by_key)


def test_hop_codes_of_segments_on_another_device(dev):
    from gnn_amd import hop_buckets, packed_segments
    seg = packed_segments([2], dev)
    seg.device = torch.device("cuda", 7)                          # stands for lists made there
    adj = torch.sparse_coo_tensor(torch.tensor([[0, 1], [1, 0]]), torch.ones(2), (2, 2)).to(dev)
    with pytest.raises(RuntimeError, match="same device"):
        hop_buckets(adj, torch.zeros(2, dtype=torch.long, device=dev), segments=seg)


@pytest.mark.parametrize("width", [2, 3, 7, 96, 130, 333, 1000, 2049, 4096, 8191, 8193, 20001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layer_norm_of_constant_rows(dev, dtype, width):
    """Equal values have no distance from their mean, whatever the rounding of their sum: the result is the bias, and
    what the backward pass makes of the rows is dy's sum in db and nothing in dw."""
    from gnn_amd import layer_norm
    values = torch.tensor([0.1, 1000.1, 12345.678, -7.3e-5, 3.0, 1e20], device=dev)
    x = values[:, None].expand(-1, width).to(dtype).contiguous().requires_grad_()
    w = torch.linspace(0.5, 2, width, device=dev).to(dtype).requires_grad_()
    b = torch.linspace(-1, 1, width, device=dev).to(dtype).requires_grad_()
    y = layer_norm(x, w, b)
    assert torch.equal(y, b.expand_as(y))
    dw = torch.autograd.grad(y, w, torch.ones_like(y))[0]
    assert not dw.any()


@pytest.mark.parametrize("width", [64, 333, 4097, 9001])
def test_layer_norm_of_rows_with_one_large_element(dev, width):
    """An element a million times the others, wherever it lies: its neighbours keep their digits relative to the row's
    deviation, a few fp32 roundings of the largest normalised value's share of the mean."""
    from gnn_amd import layer_norm
    g = torch.Generator(device=dev)
    g.manual_seed(width)
    x = torch.randn(8, width, generator=g, device=dev)
    x[torch.arange(8), torch.tensor([0, 1, 2, width // 2, width - 1, 0, 5, 9])] = 1e6
    ones = torch.ones(width, device=dev)
    d = x.double()
    mean, var = d.mean(1, keepdim=True), d.var(1, keepdim=True, unbiased=False)
    rstd = (var + 1e-5) ** -0.5
    want = (d - mean) * rstd
    # mean: the sum's roundings of at most a dozen partial sums that hold the large element, over the width, and one of
    # the mean; every distance one rounding; the deviation's own half a dozen
    chain = width / 64 + 80
    bound = 2.0 ** -24 * ((12e6 / width + mean.abs() + (d - mean).abs()) * rstd + (chain + 8) * want.abs())
    assert ((layer_norm(x, ones).double() - want).abs() <= bound).all()


def gradients(q, k, v, do, bias=None, code=None):
    """64-bit gradients of causal attention of one segment, and what the roundings of p and ds to the element type do to
    them: the errors of a sum's terms are independent and at most half a step each, so the error's standard deviation is
    at most half a step of the root of the terms' squares."""
    n, heads, dim = q.shape
    group = heads // k.shape[1]
    u = torch.finfo(q.dtype).eps / 2
    a, b, c, d = (t.double().transpose(0, 1) for t in (q, k, v, do))
    b, c = b.repeat_interleave(group, 0), c.repeat_interleave(group, 0)
    s = a @ b.transpose(1, 2) * dim ** -0.5
    off = torch.ones(n, n, dtype=torch.bool, device=q.device).triu(1)
    if bias is not None:
        s = s + bias.double()[:, code.long()]
    p = torch.softmax(s.masked_fill(off, -torch.inf), 2)
    dp = d @ c.transpose(1, 2)
    ds = p * (dp - (p * dp).sum(2, keepdim=True)) * dim ** -0.5
    ds[:, 0] = 0                                                  # a row of one pair
    pt, dst = p.transpose(1, 2), ds.transpose(1, 2)
    want = [ds @ b, dst @ a, pt @ d]
    noise = [u * (x.square() @ y.square()).sqrt() for x, y in ((ds, b), (dst, a), (pt, d))]

    def shared(x):
        return x.view(-1, group, n, dim).sum(1).transpose(0, 1)
    want = [want[0].transpose(0, 1), shared(want[1]), shared(want[2])]
    noise = [noise[0].transpose(0, 1), *(shared(x.square()).sqrt() for x in noise[1:])]
    return want, noise


def check_roundings(got, want, noise, dtype):
    for x, t, e, name in zip(got, want, noise, ("dq", "dk", "dv")):
        once = (t.to(dtype).double() - t).norm()                  # one rounding of the result
        # twice the noise: delta and the products' fp32 sums take part, too
        assert float((x.double() - t).norm()) <= float(1.1 * once + 2 * e.norm()), name


@pytest.mark.parametrize("size", [3e-5, 1e-4, 1e-3, 1.0, 2e3, "mixed"])
@pytest.mark.parametrize("dim,buckets", [(16, 0), (64, 0), (128, 0), (64, 4), (16, 4)])
def test_fp16_gradients_of_small_and_large_upstream_gradients(dev, size, dim, buckets):
    """The roundings of p and ds are relative to them, however small the upstream gradient and however many the keys."""
    from gnn_amd import packed_attention, packed_segments, pair_buckets
    g = torch.Generator(device=dev)
    g.manual_seed(dim + buckets)
    n = 1500
    q, k, v, do = (torch.randn(n, h, dim, generator=g, device=dev).half() for h in (4, 2, 2, 4))
    if size == "mixed":
        do = do * 10.0 ** torch.randint(-4, 3, (n, 1, 1), generator=g, device=dev)
    else:
        do = do * size
    do = do.half()
    seg = packed_segments([n], dev)
    leaves, kw, bias, code = [t.requires_grad_() for t in (q, k, v)], {}, None, None
    if buckets:
        bias = torch.randn(4, buckets, generator=g, device=dev).half()
        code = torch.randint(0, buckets, (n, n), generator=g, device=dev).to(torch.uint8)
        kw = dict(bias=bias, buckets=pair_buckets(seg, code))
    got = torch.autograd.grad(packed_attention(*leaves, seg, causal=True, **kw), leaves, do)
    want, noise = gradients(*(t.detach() for t in (q, k, v)), do, bias, code)
    check_roundings(got, want, noise, torch.float16)


@pytest.mark.parametrize("dim", [16, 64])
def test_fp16_weights_of_very_many_keys(dev, dim):
    """All scores alike: every weight is 1 / n, below the smallest normal number of fp16, and so is every ds."""
    from gnn_amd import packed_attention, packed_segments
    n = 40000
    g = torch.Generator(device=dev)
    g.manual_seed(3)
    v = torch.randn(n, 1, dim, generator=g, device=dev).half().requires_grad_()
    do = torch.randn(n, 1, dim, generator=g, device=dev).half()
    zero = torch.zeros(n, 1, dim, device=dev, dtype=torch.float16)
    k = torch.randn(n, 1, dim, generator=g, device=dev).half()
    q = zero.clone().requires_grad_()
    dq, dv = torch.autograd.grad(packed_attention(q, k, v, packed_segments([n], dev)), (q, v), do)
    vd, dd, kd = (t.detach().double()[:, 0] for t in (v, do, k))
    want_v = dd.mean(0)                                           # the same for all keys
    want_q = dim ** -0.5 * (dd @ (vd.t() @ kd) / n - (dd @ vd.mean(0))[:, None] * kd.mean(0))
    u = 2.0 ** -11
    # 40000 equal weights share their rounding's relative error, if it is no subnormal one; the result's own rounding
    assert float((dv[:, 0].double() - want_v).abs().max()) <= float((2.5 * u * want_v.abs()).max()) + 1e-6
    noise = u * dim ** -0.5 / n * (n ** 0.5) * float((dd @ vd.t()[:, :2000]).std() * kd.std())
    once = (want_q.half().double() - want_q).norm() / want_q.numel() ** 0.5
    assert float((dq[:, 0].double() - want_q).norm() / want_q.numel() ** 0.5) <= float(1.1 * once) + 2 * noise


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,buckets", [(16, 0), (64, 0), (128, 0), (16, 2), (64, 2)])
def test_thousands_of_keys_that_a_row_hardly_looks_at(dev, dtype, dim, buckets):
    """One key takes nearly all of every row's weight and has a value of zeros; what 4095 others of 2^-25.6 each add up to
    is the whole result.  fp16: half a step of its smallest numbers, 2^-25, against a weight of 2^-19.6; the others half
    a step of the type; besides a few fp32 roundings of the score."""
    from gnn_amd import packed_attention, packed_segments, pair_buckets
    n, high = 4096, 17.75
    q, k, v = (torch.zeros(n, 1, dim, device=dev, dtype=dtype) for _ in range(3))
    v[1:] = 100
    seg, kw = packed_segments([n], dev), {}
    if buckets:
        code = torch.ones(n, n, dtype=torch.uint8, device=dev)
        code[:, 0] = 0
        kw = dict(bias=torch.tensor([[high - 5, -5.0]], device=dev, dtype=dtype), buckets=pair_buckets(seg, code))
    else:
        q[:, 0, 3] = 1
        k[0, 0, 3] = high
    out = packed_attention(q, k, v, seg, scale=1.0, **kw)
    if buckets:
        high = float(kw["bias"][0, 0] - kw["bias"][0, 1])
    small = math.exp(-high) if dtype != torch.bfloat16 else math.exp(-float(torch.tensor(high).to(dtype)))
    want = 100 * 4095 * small / (1 + 4095 * small)
    tol = {torch.float16: 2.0 ** (-25 + 19.7), torch.bfloat16: 2.0 ** -7, torch.float32: 1e-4}[dtype]
    assert float((out.double() / want - 1).abs().max()) <= tol
