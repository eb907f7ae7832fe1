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


def reference(q, k, v, do, lengths, causal, bias=None, codes=None):
    """64-bit (out, dq, dk, dv), segment by segment; bias and codes as pair_buckets takes them, 255 masks."""
    group, dim, lo, at = q.shape[1] // k.shape[1], q.shape[2], 0, 0
    leaves = [t.detach().double().requires_grad_() for t in (q, k, v)]
    outs = []
    for n in lengths:
        a, b, c = (t[lo:lo + n].transpose(0, 1) for t in leaves)
        s = a @ b.repeat_interleave(group, 0).transpose(1, 2) * dim ** -0.5
        on = torch.ones(n, n, dtype=torch.bool, device=q.device)
        on = on.tril() if causal else on
        if bias is not None:
            code = codes[at:at + n * n].view(n, n).long()
            on = on & (code < bias.shape[1])
            s = s + bias.double()[:, code.clamp(max=bias.shape[1] - 1)]
        p = torch.softmax(s.masked_fill(~on, -torch.inf), 2).masked_fill(~on, 0.0)
        outs.append((p @ c.repeat_interleave(group, 0)).transpose(0, 1))
        lo, at = lo + n, at + n * n
    out = torch.cat(outs)
    return [out.detach(), *torch.autograd.grad(out, leaves, do.double())]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,buckets", [(16, 0), (24, 5), (64, 0), (64, 5), (128, 0), (100, 5)])
@pytest.mark.parametrize("parts,lengths", [(1, [300, 1, 77]), (3, [300, 1, 77]), (1, [33] * 12)],
                         ids=["whole", "parts", "short"])
def test_what_is_not_finite_reaches_what_attends_to_it_only(dev, dtype, dim, buckets, parts, lengths, monkeypatch):
    """Single elements of v and of d_out that are not finite, in causal segments, with masked pairs if there is a bias:
    the elements that weigh them are not finite, every other one is the result with zeros in their place."""
    from gnn_amd import packed_attention, packed_segments, pair_buckets
    from gnn_amd.attention import PackedSegments
    monkeypatch.setattr(PackedSegments, "key_parts", lambda *a: parts)
    g = torch.Generator(device=dev)
    g.manual_seed(dim)
    heads, kv, total = 6, 2, sum(lengths)
    rows = torch.randn(total, 2 * heads + 2 * kv, dim, generator=g, device=dev).to(dtype)
    q, k, v, do = (t.clone() if dim == 64 else t for t in rows.split([heads, kv, kv, heads], 1))     # or slices of one
    bias = codes = None
    kw = {}
    seg = packed_segments(lengths, dev)
    assert seg.block_rows == (32 if len(lengths) == 12 else 128)
    if buckets:
        bias = torch.randn(heads, buckets, generator=g, device=dev).to(dtype)
        codes = torch.randint(0, buckets, (sum(n * n for n in lengths),), generator=g, device=dev).to(torch.uint8)
        codes[torch.rand(codes.shape, generator=g, device=dev) < 0.3] = 255
        codes[0] = 0                                              # row 0 attends to itself
        kw = dict(bias=bias, buckets=pair_buckets(seg, codes))
    on = torch.zeros(total, total, dtype=torch.bool, device=dev)
    lo = at = 0
    for n in lengths:
        part = torch.ones(n, n, dtype=torch.bool, device=dev).tril()
        if buckets:
            part &= codes[at:at + n * n].view(n, n) < buckets
        on[lo:lo + n, lo:lo + n] = part
        lo, at = lo + n, at + n * n
    tol = {torch.float32: 2e-5, torch.float16: 6e-3, torch.bfloat16: 5e-2}[dtype]

    def check(got, want, spoilt, what):
        """What is spoilt is not finite; the rest is within a few roundings of terms as large as the largest."""
        assert not got[spoilt].isfinite().any(), what
        rest = ~spoilt
        assert got[rest].isfinite().all(), what
        assert float((got.double() - want)[rest].abs().max()) <= tol * float(want.abs().max()), what

    # values
    bad = torch.zeros_like(v, dtype=torch.bool)
    for row, head, d, x in ((5, 0, 3, math.inf), (64, 1, 0, math.nan), (150, 0, dim - 1, -math.inf), (151, 0, 1, math.inf),
                            (299, 1, 2, math.nan), (340, 1, 7, math.inf)):
        v[row, head, d], bad[row, head, d] = x, True
    clean = torch.where(bad, 0.0, v).to(dtype)
    want = reference(q, k, clean, do, lengths, True, bias, codes)
    out = packed_attention(q, k, v, seg, causal=True, **kw)
    spoilt = torch.einsum("ij,jhd->ihd", on.float(), bad.float()).repeat_interleave(heads // kv, 1) > 0
    check(out, want[0], spoilt, "out")
    # upstream gradients
    bad = torch.zeros_like(do, dtype=torch.bool)
    for row, head, d, x in ((0, 0, 3, math.inf), (40, 4, 0, math.nan), (41, 1, dim - 1, -math.inf), (290, 5, 1, math.inf),
                            (376, 2, 2, math.inf)):
        do[row, head, d], bad[row, head, d] = x, True
    leaves = [t.clone().requires_grad_() for t in (q, k, clean)]
    dq, dk, dv = torch.autograd.grad(packed_attention(*leaves, seg, causal=True, **kw), leaves, do)
    want = reference(q, k, clean, torch.where(bad, 0.0, do).to(dtype), lengths, True, bias, codes)
    rows = bad.any(2) & (on.sum(1) > 0)[:, None]                  # (row, head): delta is not finite
    spoilt = rows[..., None].expand_as(dq)
    check(dq, want[1], spoilt, "dq")
    reach = torch.einsum("ij,ih->jh", on.float(), rows.float())   # (key, query head)
    shared = reach.view(total, kv, -1).sum(2)[..., None].expand_as(dk) > 0
    check(dk, want[2], shared, "dk")
    some = torch.einsum("ij,ihd->jhd", on.float(), bad.float()).view(total, kv, -1, dim).sum(2) > 0
    check(dv, want[3], some, "dv")


@pytest.mark.parametrize("dtype,heads,kv,dim,buckets", [(torch.float16, 16, 4, 64, 0), (torch.bfloat16, 16, 4, 128, 0),
                                                      (torch.float16, 8, 8, 64, 32)])
def test_time_of_what_is_not_finite(dev, dtype, heads, kv, dim, buckets):
    """An overflowed step takes a bounded multiple of an ordinary one: twenty times as long at most where measured, several
    hundred if the pairs were taken one by one."""
    from gnn_amd import packed_attention, packed_segments, relative_buckets
    lengths = [1500] * 6
    n = sum(lengths)
    seg = packed_segments(lengths, dev)
    q, k, v, do = (torch.randn(n, h, dim, device=dev).to(dtype) for h in (heads, kv, kv, heads))
    kw = {}
    if buckets:
        kw = dict(bias=torch.randn(heads, buckets, device=dev).to(dtype), buckets=relative_buckets(seg, buckets, 128))
    places = torch.rand(n, device=dev) < 0.3

    def times(v, do):
        leaves = [t.clone().requires_grad_() for t in (q, k, v)]
        ends = [torch.cuda.Event(enable_timing=True) for _ in range(3)]
        for _ in range(2):                                        # the second counts
            ends[0].record()
            out = packed_attention(*leaves, seg, causal=True, **kw)
            ends[1].record()
            torch.autograd.grad(out, leaves, do)
            ends[2].record()
        torch.cuda.synchronize()
        return ends[0].elapsed_time(ends[1]), ends[1].elapsed_time(ends[2])
    usual = times(v, do)
    bad_v, bad_do, nan = v.clone(), do.clone(), torch.full_like(do, math.nan)
    bad_v[places, :, 3] = math.inf
    bad_do[places, :, 3] = math.inf
    for got in (times(bad_v, do), times(v, bad_do), times(v, nan)):
        for a, b in zip(got, usual):
            assert a <= 60 * b + 1
