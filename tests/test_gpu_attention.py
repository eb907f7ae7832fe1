"""``gnn_amd.packed_attention`` and its bucket codes against the definition in 64 bits, segment by segment.

Tolerances (``u`` = half a step of the element type, e = 2^-24, one fp32 rounding), worst case over the roundings:
  scores      (D + 6) e times the sum of the products' magnitudes, and 6 e of the score and the row's largest score
  p           twice the score's error (its own and the sum's), n e for the sum, and u for the 16-bit types, which
              round it before the second product (nothing for fp32)
  out         p's error against |v|, n e for the sum, u for the result
  delta       |do| against the error of out before its rounding (kept with its remainder), and D e
  ds          p's error against |dp - delta|, the errors of dp (D e) and delta against p, u as for p
  dq, dk, dv  the error of ds or p against the magnitudes of the other factor, n e, u; dk, dv summed over the group
  d_bias      the error of the unrounded ds summed, e per addition, u
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
E = 2.0 ** -24


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch.device("cuda:0")


def truth(q, k, v, do, lengths, causal, scale=None, bias=None, codes=None):
    """64-bit (out, dq, dk, dv[, d_bias]) and their tolerances; codes: one (n, n) tensor per segment."""
    dtype = q.dtype
    u = torch.finfo(dtype).eps / 2
    up = 0.0 if dtype == torch.float32 else u
    heads, kv, dim = q.shape[1], k.shape[1], q.shape[2]
    group = heads // kv
    scale = dim ** -0.5 if scale is None else scale
    q, k, v, do = (t.detach().double() for t in (q, k, v, do))
    out, dq, dk, dv = (torch.zeros_like(t) for t in (q, q, k, v))
    err = [torch.zeros_like(t) for t in (out, dq, dk, dv)]
    if bias is not None:
        bias = bias.detach().double()
        db, db_err, db_abs = (torch.zeros_like(bias) for _ in range(3))
    lo = 0
    for g, n in enumerate(lengths):
        if n == 0:
            continue
        r = slice(lo, lo + n)
        lo += n
        a, b, c, d = (t[r].transpose(0, 1) for t in (q, k, v, do))          # (heads, n, D)
        b, c = b.repeat_interleave(group, 0), c.repeat_interleave(group, 0)
        s = a @ b.transpose(1, 2) * scale
        ok = torch.ones(n, n, dtype=torch.bool, device=q.device)
        s_err = (dim + 6) * E * (a.abs() @ b.abs().transpose(1, 2)) * scale
        if causal:
            ok = ok.tril()
        if bias is not None:
            code = codes[g].long()
            ok = ok & (code < bias.shape[1])
            code = code.clamp(max=bias.shape[1] - 1)
            s = s + bias[:, code]
        ok = ok & (s > -math.inf)
        s = s.masked_fill(~ok, -math.inf)
        top = s.amax(2, keepdim=True)
        top = torch.where(top == -math.inf, 0.0, top)
        s_err = s_err + 6 * E * (torch.where(ok, s.abs(), 0.0) + top.abs())
        p = torch.exp(s - top)
        total = p.sum(2, keepdim=True)
        p = p / torch.where(total == 0, 1.0, total)
        rel = s_err + (s_err * p).sum(2, keepdim=True) + (n + 16) * E
        o = p @ c
        o_err = ((rel + up) * p) @ c.abs() + (n + 4) * E * (p @ c.abs())
        dp = d @ c.transpose(1, 2)
        delta = (d * o).sum(2, keepdim=True)
        de = (d.abs() * (o_err + u * u * o.abs() + torch.finfo(dtype).tiny)).sum(2, keepdim=True) + dim * E * (d.abs() * o.abs()).sum(2, keepdim=True)
        dpe = dim * E * (d.abs() @ c.abs().transpose(1, 2))
        ds = p * (dp - delta)
        ds_err = p * (rel * (dp - delta).abs() + dpe + de) * (1 + rel) + 4 * E * ds.abs()
        dsr = ds_err + up * (ds.abs() + ds_err)
        n_e = (n * group + 8) * E
        pr = p * (rel + up)
        parts = [(o, o_err), (scale * ds @ b, scale * (dsr @ b.abs() + n_e * (ds.abs() @ b.abs())))]
        for val, er, other in ((scale * ds, scale * dsr, a), (p, pr, d)):
            x = val.transpose(1, 2) @ other
            xe = er.transpose(1, 2) @ other.abs() + n_e * (val.abs().transpose(1, 2) @ other.abs())
            parts.append((x.view(kv, group, n, dim).sum(1), xe.view(kv, group, n, dim).sum(1)))
        for res, er, (x, xe) in zip((out, dq, dk, dv), err, parts):
            res[r], er[r] = x.transpose(0, 1), (xe + u * (x.abs() + xe)).transpose(0, 1)
        if bias is not None:
            for bucket in range(bias.shape[1]):
                hit = (code == bucket) & ok
                db[:, bucket] += (ds * hit).sum((1, 2))
                db_err[:, bucket] += (ds_err * hit).sum((1, 2))
                db_abs[:, bucket] += (ds.abs() * hit).sum((1, 2))
    res = [out, dq, dk, dv]
    if bias is not None:
        e = db_err + db_abs * E * (sum(lengths) / 32 + 64)
        res.append(db)
        err.append(e + u * (db.abs() + e))
    return res, err


def check(got, want, err, names=("out", "dq", "dk", "dv", "d_bias")):
    for x, t, e, name in zip(got, want, err, names):
        x = x.detach().double()
        worst = float(((x - t).abs() / (e + torch.finfo(got[0].dtype).tiny)).max()) if x.numel() else 0.0
        assert worst <= 1.0, (name, worst)


def make(dev, dtype, lengths, heads, kv, dim, tail=0, seed=0, buckets=0, holes=False):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    n = sum(lengths) + tail
    q, k, v, do = (torch.randn(n, h, dim, generator=g, device=dev).to(dtype) for h in (heads, kv, kv, heads))
    bias = codes = None
    if buckets:
        bias = torch.randn(heads, buckets, generator=g, device=dev).to(dtype)
        codes = [torch.randint(0, buckets, (m, m), generator=g, device=dev).to(torch.uint8) for m in lengths]
        if holes:                                   # padded nodes: rows and columns that do not attend, other gaps
            for c in codes:
                hole = torch.rand(c.shape[0], generator=g, device=dev) < 0.3
                c[hole] = 255
                c[:, hole] = buckets                # any code from n_buckets on
                c[torch.rand(c.shape, generator=g, device=dev) < 0.2] = 255
    return q, k, v, do, bias, codes


def run(q, k, v, do, lengths, causal, scale=None, bias=None, codes=None):
    from gnn_amd import packed_attention, packed_segments, pair_buckets
    seg = packed_segments(lengths, q.device)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    kw = {}
    if bias is not None:
        leaves.append(bias.detach().requires_grad_())
        flat = torch.cat([c.reshape(-1) for c in codes]) if codes else torch.empty(0, dtype=torch.uint8, device=q.device)
        kw = dict(bias=leaves[3], buckets=pair_buckets(seg, flat))
    out = packed_attention(*leaves[:3], seg, causal=causal, scale=scale, **kw)
    with torch.no_grad():                           # without a graph: the same numbers
        again = packed_attention(*leaves[:3], seg, causal=causal, scale=scale, **kw)
    assert ((out.detach() == again) | (out.detach().isnan() & again.isnan())).all()
    return [out, *torch.autograd.grad(out, leaves, do)]


# lengths on both sides of a wavefront's 32 rows, a workgroup's 128 and the key tiles of 32 and 64; one token; empty
RAGGED = [[1], [2, 0, 1, 33], [31, 32, 33, 0, 64, 65], [127, 128, 129], [300, 5, 257, 191], [40] * 20]
HEADS = [(1, 1, 64), (4, 2, 32), (6, 2, 128), (3, 3, 16)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lengths", RAGGED, ids=lambda x: "-".join(map(str, x[:6])))
@pytest.mark.parametrize("heads,kv,dim", HEADS)
def test_forward_and_backward(dev, dtype, causal, lengths, heads, kv, dim):
    q, k, v, do, _, _ = make(dev, dtype, lengths, heads, kv, dim, seed=dim)
    check(run(q, k, v, do, lengths, causal), *truth(q, k, v, do, lengths, causal))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lengths", RAGGED, ids=lambda x: "-".join(map(str, x[:6])))
@pytest.mark.parametrize("heads,kv,dim,buckets,holes", [(2, 2, 64, 7, False), (4, 2, 16, 32, True), (3, 1, 128, 1, True)])
def test_bias(dev, dtype, causal, lengths, heads, kv, dim, buckets, holes):
    q, k, v, do, bias, codes = make(dev, dtype, lengths, heads, kv, dim, seed=buckets, buckets=buckets, holes=holes)
    check(run(q, k, v, do, lengths, causal, bias=bias, codes=codes),
          *truth(q, k, v, do, lengths, causal, bias=bias, codes=codes))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [1, 3, 7, 8, 15, 17, 24, 31, 33, 40, 63, 65, 80, 96, 100, 127])
def test_head_widths(dev, dtype, dim):
    lengths = [50, 97]
    q, k, v, do, bias, codes = make(dev, dtype, lengths, 2, 1, dim, seed=dim, buckets=5)
    check(run(q, k, v, do, lengths, True), *truth(q, k, v, do, lengths, True))
    check(run(q, k, v, do, lengths, False, bias=bias, codes=codes),
          *truth(q, k, v, do, lengths, False, bias=bias, codes=codes))


@pytest.mark.parametrize("dtype", TYPES)
def test_a_long_segment_many_heads_and_a_scale(dev, dtype):
    lengths = [2300, 700]
    q, k, v, do, _, _ = make(dev, dtype, lengths, 12, 3, 64, seed=4)
    check(run(q, k, v, do, lengths, True, scale=0.3), *truth(q, k, v, do, lengths, True, scale=0.3))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", ["projection", "heads_first", "odd"])
def test_strides(dev, dtype, shape):
    """Slices of one projection's output, heads as the outer dimension, rows at odd elements, a shared key head
    expanded over the heads, a gradient of another layout."""
    lengths, heads, dim = [70, 33], 4, 40
    n = sum(lengths)
    g = torch.Generator(device=dev)
    g.manual_seed(3)
    if shape == "projection":
        q, k, v = torch.randn(n, 3 * heads, dim, generator=g, device=dev).to(dtype).split(heads, 1)
        do = torch.randn(n, heads, dim, generator=g, device=dev).to(dtype)
    elif shape == "heads_first":
        q, k, v, do = torch.randn(4, heads, n, dim, generator=g, device=dev).to(dtype).transpose(1, 2).unbind(0)
    else:
        buf = torch.randn(4, n, heads * 43 + 1, generator=g, device=dev).to(dtype)
        q, k, v, do = buf[:, :, 1:].reshape(4, n, heads, 43)[..., 1:41].unbind(0)
        k = k[:, :1].expand(n, heads, dim)
    check(run(q, k, v, do, lengths, True), *truth(q, k, v, do, lengths, True))
    t = torch.randn(n, dim, heads, generator=g, device=dev).to(dtype).transpose(1, 2)    # elements apart: copied
    check(run(t, k, v, do, lengths, False), *truth(t, k, v, do, lengths, False))


def test_rows_behind_the_last_segment_and_other_segments(dev):
    """Rows that belong to no segment may hold anything, give zeros and take no gradient; what is not finite in one
    segment does not reach another."""
    for dtype in TYPES:
        lengths = [40, 200, 17]
        q, k, v, do, _, _ = make(dev, dtype, lengths, 2, 2, 32, tail=61)
        total = sum(lengths)
        for t in (q, k, v, do):
            t[total:] = float("nan")
        got = run(q, k, v, do, lengths, False)
        want, err = truth(*(torch.where(t.isnan(), 0.0, t) for t in (q, k, v, do)), lengths, False)
        check(got, want, err)
        for t in got:
            assert not t[total:].any()
        for t in (q, k, v, do):
            t[40:240] = float("inf")
        dirty = run(q, k, v, do, lengths, False)
        for a, b in zip(dirty, got):
            assert torch.equal(a[:40], b[:40]) and torch.equal(a[240:], b[240:])


def test_keys_that_are_masked_may_hold_anything(dev):
    """Causal: a key that is not finite leaves the rows before it as they were; masked by its code: all rows."""
    lengths = [150]
    q, k, v, do, bias, codes = make(dev, torch.bfloat16, lengths, 2, 2, 32, buckets=3)
    clean = run(q, k, v, do, lengths, True)[0]
    bad = k.clone()
    bad[100] = float("nan")
    got = run(q, bad, v, do, lengths, True)[0]
    assert torch.equal(got[:100], clean[:100]) and got[100:].isnan().all()
    codes[0][:, 77] = 255
    clean = run(q, k, v, do, lengths, False, bias=bias, codes=codes)
    bad = k.clone()
    bad[77] = float("inf")
    got = run(q, bad, v, do, lengths, False, bias=bias, codes=codes)
    assert torch.equal(got[0], clean[0])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [16, 40, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_masked_pairs_may_hold_anything(dev, dtype, dim, bad):
    """Padded nodes whose codes do not attend hold values that are not finite in q, k and v: all other rows and all
    gradients are those of a batch with zeros there.  Causal: rows behind a row that is not finite in k and v."""
    lengths = [70, 200]
    q, k, v, do, bias, codes = make(dev, dtype, lengths, 4, 2, dim, buckets=4)
    holes = [3, 40, 64, 69, 71, 150, 269]
    for c, lo in zip(codes, (0, 70)):
        for x in holes:
            if lo <= x < lo + c.shape[0]:
                c[x - lo] = 255
                c[:, x - lo] = 255
    clean = []
    for t in (q, k, v):
        t[holes] = 0
        clean.append(t.clone())
        t[holes] = bad
    want, err = truth(*clean, do, lengths, False, bias=bias, codes=codes)
    check(run(q, k, v, do, lengths, False, bias=bias, codes=codes), want, err)
    q, k, v, do, _, _ = make(dev, dtype, lengths, 4, 2, dim)
    want, err = truth(q, k, v, do, lengths, True)
    k, v = k.clone(), v.clone()
    k[50:70] = bad
    v[50:70] = bad
    k[200:270:3] = bad
    v[200:270:3] = bad
    got = run(q, k, v, do, lengths, True)[0]
    keep = list(range(50)) + list(range(70, 200))
    check([got[keep]], [want[0][keep]], [err[0][keep]])
    assert not got[200:].isfinite().all(1).all(1).any()


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_without_pairs_and_extreme_biases(dev, dtype):
    lengths = [90, 33]
    q, k, v, do, bias, codes = make(dev, dtype, lengths, 2, 1, 24, buckets=4)
    codes[0][5] = 255
    codes[0][64:] = 9
    codes[1][:] = 255
    codes[0][7] = 2                                 # a row whose only bucket has -inf, for head 0
    bias[0, 2] = -math.inf
    codes[0][8] = 3                                 # a row all of whose pairs carry the type's lowest value
    bias[1, 3] = torch.finfo(dtype).min
    got = run(q, k, v, do, lengths, False, bias=bias, codes=codes)
    want, err = truth(q, k, v, do, lengths, False, bias=bias, codes=codes)
    # the lowest value of fp32 swallows the products: all 90 pairs of row 8, head 1 have the same score then, in 64
    # bits too (a step of 64-bit numbers there is 2^75); the tolerance's 6 e |score| says nothing about that row
    for x in err:
        x[torch.isinf(x)] = 0
    if dtype == torch.float32 or dtype == torch.bfloat16:
        assert torch.allclose(got[0][8, 1].double(), want[0][8, 1], rtol=2 * torch.finfo(dtype).eps, atol=1e-2)
        assert all(x.isfinite().all() for x in got)
        return_rows = [i for i in range(123) if i != 8]
        got0, want0, err0 = got[0][return_rows], want[0][return_rows], err[0][return_rows]
        check([got0], [want0], [err0])
    else:
        check(got, want, err)
    for row in [5] + list(range(64, 123)):
        assert not got[0][row].any() and not got[1][row].any()
    assert not got[0][7, 0].any() and got[0][7, 1].any()
    assert float(got[4][0, 2]) == 0.0


def test_no_segments_and_empty_segments(dev):
    for lengths in ([], [0], [0, 0, 0]):
        for buckets in (0, 3):
            q, k, v, do, bias, codes = make(dev, torch.float16, lengths, 2, 1, 16, tail=4, buckets=buckets)
            got = run(q, k, v, do, lengths, False, bias=bias, codes=codes)
            assert all(not t.any() for t in got)
    q, k, v, do, _, _ = make(dev, torch.float16, [], 2, 1, 16)
    assert run(q, k, v, do, [], True)[0].shape == (0, 2, 16)


def test_gradients_against_differences(dev):
    lengths = [13, 6]
    q, k, v, do, bias, codes = make(dev, torch.float32, lengths, 2, 1, 5, buckets=3)
    grads = run(q, k, v, do, lengths, False, bias=bias, codes=codes)[1:]
    args = [t.double() for t in (q, k, v, bias)]
    w = do.double()

    def loss(q, k, v, bias):
        total, lo = 0.0, 0
        for g, n in enumerate(lengths):
            for h in range(2):
                s = q[lo:lo + n, h] @ k[lo:lo + n, 0].T * 5 ** -0.5 + bias[h][codes[g].long()]
                total += float((torch.softmax(s, 1) @ v[lo:lo + n, 0] * w[lo:lo + n, h]).sum())
            lo += n
        return total
    for at, grad in enumerate(grads):
        for i in range(0, grad.numel(), 7):
            ends = []
            for step in (1e-5, -1e-5):              # central differences: error of the order of the step squared
                moved = [a.clone() for a in args]
                moved[at].view(-1)[i] += step
                ends.append(loss(*moved))
            diff = (ends[0] - ends[1]) / 2e-5
            assert abs(diff - float(grad.view(-1)[i])) <= 1e-4 * (1 + abs(diff))


def test_only_some_gradients_and_expanded_inputs(dev):
    """A key head expanded over the heads collects the gradients of all; inputs without a gradient cost nothing."""
    from gnn_amd import packed_attention, packed_segments
    lengths = [45]
    q, k, v, do, _, _ = make(dev, torch.float32, lengths, 4, 1, 16)
    shared = run(q, k, v, do, lengths, True)
    seg = packed_segments(lengths, dev)
    kl = k.clone().requires_grad_()
    out = packed_attention(q, kl.expand(45, 4, 16), v.expand(45, 4, 16), seg, causal=True)
    out.backward(do)
    assert torch.equal(out, shared[0])
    # four fp32 sums in another order: the terms' magnitudes are those of the gradient, up to cancellation
    assert torch.allclose(kl.grad, shared[2], rtol=1e-5, atol=1e-5)


def test_repeatable_on_any_stream_and_in_a_captured_graph(dev):
    from gnn_amd import packed_attention, packed_segments, pair_buckets
    lengths = [200, 64, 90]
    q, k, v, do, bias, codes = make(dev, torch.bfloat16, lengths, 4, 2, 64, buckets=6)
    first = run(q, k, v, do, lengths, True, bias=bias, codes=codes)
    assert all(torch.equal(a, b) for a, b in zip(first, run(q, k, v, do, lengths, True, bias=bias, codes=codes)))
    seg = packed_segments(lengths, dev)
    buckets = pair_buckets(seg, torch.cat([c.reshape(-1) for c in codes]))
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v, bias)]

    def once():
        out = packed_attention(*leaves[:3], seg, causal=True, bias=leaves[3], buckets=buckets)
        return [out, *torch.autograd.grad(out, leaves, do)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(s):
        other = once()
        for _ in range(2):                          # two captured graphs, replayed in turn
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s):
                got = once()
            graphs.append((graph, got))
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(first, other))
    for seed in range(3):
        nq, nk, nv, ndo, _, _ = make(dev, torch.bfloat16, lengths, 4, 2, 64, seed=20 + seed)
        with torch.no_grad():
            for old, new in zip((*leaves[:3], do), (nq, nk, nv, ndo)):
                old.copy_(new)
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        want = run(leaves[0], leaves[1], leaves[2], do, lengths, True, bias=leaves[3], codes=codes)
        for _, got in graphs:
            assert all(torch.equal(a, b) for a, b in zip(got, want))


# --- bucket codes -------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("value", ["lowest", -1e9, -3e4, 3e4, 1e30])
@pytest.mark.parametrize("dim", [16, 64])
def test_rows_whose_pairs_all_carry_one_large_bias(dev, dtype, value, dim):
    """Queries of zeros: every pair's score is the bias alone, and softmax knows differences only, so the results and
    gradients are those of a bias of zeros, however large it is."""
    q, k, v, do, bias, codes = make(dev, dtype, [70, 3, 131], 4, 2, dim, seed=5, buckets=3, holes=True)
    q.zero_()
    want, err = truth(q, k, v, do, [70, 3, 131], False, bias=torch.zeros_like(bias), codes=codes)
    lowest = torch.finfo(dtype).min
    bias.fill_(lowest if value == "lowest" else max(lowest, min(-lowest, value)))
    check(run(q, k, v, do, [70, 3, 131], False, bias=bias, codes=codes), want, err)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("parts", [1, 2, 3, 6])
@pytest.mark.parametrize("dim,buckets", [(37, 0), (128, 0), (16, 5), (64, 5)])
def test_query_heads_in_parts(dev, dtype, parts, dim, buckets, monkeypatch):
    """dK and dV summed by several workgroups per block of keys; once with a masked key that is not finite."""
    from gnn_amd.attention import PackedSegments
    assert PackedSegments.key_parts(_segments([4096, 100], dev), 6, 1, True) > 1
    assert PackedSegments.key_parts(_segments([20] * 8, dev), 6, 1, True) == 1
    monkeypatch.setattr(PackedSegments, "key_parts", lambda *a: parts)
    lengths = [70, 0, 3, 131]
    q, k, v, do, bias, codes = make(dev, dtype, lengths, 12, 2, dim, tail=5, seed=parts, buckets=buckets, holes=True)
    want, err = truth(q, k, v, do, lengths, True, bias=bias, codes=codes)
    got = run(q, k, v, do, lengths, True, bias=bias, codes=codes)
    check(got, want, err)
    for t in got[:4]:
        assert not t[sum(lengths):].any()
    do[100], want, err = math.inf, [t[:100] for t in want], [t[:100] for t in err]      # a row of the last segment
    later = run(q, k, v, do, lengths, True, bias=bias, codes=codes)
    assert torch.equal(later[0], got[0])
    assert buckets or not torch.isfinite(later[3][73:101]).all()            # with holes row 100 may attend to nothing
    for a, b in zip(later[1:4], got[1:4]):
        assert torch.equal(a[:73], b[:73]) and torch.allclose(a[101:204].double(), b[101:204].double(), rtol=0.1, atol=0.1)


def _segments(lengths, dev):
    from gnn_amd import packed_segments
    return packed_segments(lengths, dev)


@pytest.mark.parametrize("dim,heads", [(128, 1), (64, 2)])
def test_rows_gigabytes_apart(dev, dim, heads):
    """Rows of one tile lie further apart than 32-bit offsets reach."""
    q, k, v, do, _, _ = make(dev, torch.bfloat16, [128], heads, heads, dim, seed=3)
    apart = (1 << 24) - 8
    if torch.cuda.mem_get_info(dev)[0] < 16 << 30:
        pytest.skip("needs 16 GiB of free memory")
    want = run(q, k, v, do, [128], False)
    far = torch.empty(128 * apart, dtype=torch.bfloat16, device=dev)
    wide = [torch.as_strided(far, (128, heads, dim), (apart, dim, 1), at) for at in (0, 1024, 2048)]
    for x, t in zip(wide, (q, k, v)):
        x.copy_(t)
    from gnn_amd import packed_attention
    leaves = [x.detach().requires_grad_() for x in wide]
    out = packed_attention(*leaves, _segments([128], dev))
    for a, b in zip([out, *torch.autograd.grad(out, leaves, do)], want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dim,buckets", [(16, 4), (64, 4), (64, 32), (128, 9)])
def test_blocks_of_pairs_with_one_code(dev, dtype, causal, dim, buckets):
    """Codes that are alike over whole tiles: a far bucket, a mask over 64 columns (whose keys hold anything), one code
    everywhere; different ones per row."""
    lengths = [300, 77, 160]
    q, k, v, do, bias, codes = make(dev, dtype, lengths, 4, 2, dim, seed=buckets, buckets=buckets)
    i = torch.arange(300, device=dev)
    far = (i[:, None] - i[None, :]).abs()
    codes[0] = torch.where(far < 40, far % buckets, buckets - 1).to(torch.uint8)
    codes[0][:, 192:256] = 255
    codes[1].fill_(buckets - 2)
    codes[2] = (i[:160] % buckets)[:, None].expand(160, 160).contiguous().to(torch.uint8)
    want, err = truth(q, k, v, do, lengths, causal, bias=bias, codes=codes)
    check(run(q, k, v, do, lengths, causal, bias=bias, codes=codes), want, err)
    clean = run(q, k, v, do, lengths, causal, bias=bias, codes=codes)
    k[200], v[201] = math.nan, math.inf
    got = run(q, k, v, do, lengths, causal, bias=bias, codes=codes)
    rows = torch.ones(537, dtype=torch.bool, device=dev)
    rows[192:256] = False
    for a, b in zip(got[1:], clean[1:]):
        a, b = (t[rows] if t.shape[0] == 537 else t for t in (a, b))
        assert torch.allclose(a.double(), b.double(), rtol=0.02, atol=0.02 * float(b.abs().max()))
    check([got[0]], want[:1], err[:1])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,buckets", [(53, 0), (53, 8), (16, 8), (128, 3)])
def test_rows_of_one_pair_have_no_gradient(dev, dtype, dim, buckets):
    """Segments of one row, and the first row under a causal mask: softmax of one score is 1 whatever the score."""
    q, k, v, do, bias, codes = make(dev, dtype, [1] * 11, 6, 2, dim, buckets=buckets)
    got = run(q, k, v, do, [1] * 11, False, bias=bias, codes=codes)
    for t in got[1:3] + got[4:]:
        assert not t.any()
    assert torch.equal(got[0].view(11, 2, 3, dim), v[:, :, None].expand(11, 2, 3, dim))
    q, k, v, do, bias, codes = make(dev, dtype, [40, 140], 6, 2, dim, buckets=buckets)
    got = run(q, k, v, do, [40, 140], True, bias=bias, codes=codes)
    assert not got[1][0].any() and not got[1][40].any() and got[1][1:40].any()


def test_lists_that_outlive_or_leave_their_stream(dev):
    """Deep copies have memory of their own; lists made on one stream, used on another and dropped at once."""
    import copy
    from gnn_amd import packed_attention, packed_segments, relative_buckets
    q, k, v, do, bias, _ = make(dev, torch.float32, [300, 5, 90], 4, 2, 16, buckets=8)
    bias.requires_grad_()

    def once(buckets):
        out = packed_attention(q, k, v, buckets.segments, bias=bias, buckets=buckets)
        return [out, *torch.autograd.grad(out, [bias], do)]
    made = relative_buckets(packed_segments([300, 5, 90], dev), 8, 100)
    want = once(made)
    twin = copy.deepcopy(made)
    assert twin.segments is not made.segments and twin.segments._seg_ptr != made.segments._seg_ptr
    del made
    torch.zeros(1 << 20, dtype=torch.int32, device=dev)
    assert all(torch.equal(a, b) for a, b in zip(once(twin), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = once(twin)
    del twin
    junk = [torch.zeros(1 << n, dtype=torch.int32, device=dev) for n in range(4, 20)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and junk


def test_dense_and_relative_codes(dev):
    from gnn_amd import packed_segments, pair_buckets, relative_buckets
    lengths = [3, 0, 64, 131, 1]
    seg = packed_segments(torch.tensor(lengths), dev)
    assert seg.seg_ptr.tolist() == [0, 3, 3, 67, 198, 199]
    codes = [torch.randint(0, 256, (n, n), device=dev).to(torch.uint8) for n in lengths]
    b = pair_buckets(seg, torch.cat([c.reshape(-1) for c in codes]))
    assert all(torch.equal(b.dense(i), c) for i, c in enumerate(codes))
    b._codes = b._by_key                            # the copy with a row per key
    assert all(torch.equal(b.dense(i), c.t()) for i, c in enumerate(codes))
    for n_buckets, reach, both in ((32, 128, True), (8, 20, False), (2, 5, True), (1, 9, False)):
        got = relative_buckets(seg, n_buckets, reach, both)
        per = n_buckets // 2 if both else n_buckets
        exact = max(1, per // 2)
        for i, n in enumerate(lengths):
            want = np.zeros((n, n), np.uint8)
            for r in range(n):
                for c in range(n):
                    d = abs(c - r) if both else max(r - c, 0)
                    d = min(d, reach)
                    bucket = d if d < exact else min(per - 1, exact + int(math.floor(
                        math.log(d / exact) / math.log(reach / exact) * (per - exact))))
                    want[r, c] = bucket + (per if both and c > r else 0)
            assert np.array_equal(got.dense(i).cpu().numpy(), want), (n_buckets, i)
        got._codes = got._by_key
        assert np.array_equal(got.dense(3).cpu().numpy()[5, 7], relative_buckets(seg, n_buckets, reach, both).dense(
            3).cpu().numpy()[7, 5])


def test_relative_codes_of_a_reach_beyond_any_segment(dev):
    from gnn_amd import packed_segments, relative_buckets
    seg = packed_segments([9, 33], dev)
    got = relative_buckets(seg, 8, 2 ** 40, False)
    assert got.dense(1)[32, :].tolist() == [4] * 29 + [3, 2, 1, 0] and got.dense(1)[0, 1:].eq(0).all()
    assert torch.equal(got.dense(0), got.dense(1)[:9, :9])


@pytest.mark.parametrize("far", ["bucket", "mask"])
def test_hop_codes(dev, far):
    import os
    import sys
    sys.path.insert(0, os.path.join(os.path.dirname(__file__), ".."))
    from gnn_amd import hop_buckets
    from gnn_amd.synth import random_batch
    from oracle.distance_bias_oracle import hop_distances
    b = random_batch(9, 1, 60, 2.4, seed=3)
    adj, _, gi, _ = b.to_torch(dev)
    got = hop_buckets(adj, gi, max_distance=4, far=far)
    a = np.zeros((b.n_nodes, b.n_nodes), np.float32)
    a[b.indices[0], b.indices[1]] = b.values
    lo = 0
    for i, n in enumerate(b.sizes):
        want = hop_distances(a[lo:lo + n, lo:lo + n], 4).astype(np.int64)
        if far == "mask":
            want[want == 5] = 255
        assert np.array_equal(got.dense(i).cpu().numpy().astype(np.int64), want)
        lo += int(n)
    assert got.segments.lengths.tolist() == [int(n) for n in b.sizes]


# --- together -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("bits", [8, 32])
def test_a_graph_attention_block_trains(dev, bits):
    """Layer norm, attention over each graph's nodes with a bias by hop distance, and AdamW, as a model uses them:
    gradients against the same model in 64-bit torch operations, then steps of the optimiser."""
    from gnn_amd import AdamW, LayerNorm, hop_buckets, packed_attention
    from gnn_amd.synth import random_batch
    batch = random_batch(12, 4, 50, 3.0, seed=5, n_feat=24)
    adj, x, gi, _ = batch.to_torch(dev)
    buckets = hop_buckets(adj, gi, max_distance=3)
    torch.manual_seed(0)
    norm = LayerNorm(24, device=dev)
    proj = torch.nn.Linear(24, 3 * 32, device=dev)
    bias = torch.nn.Parameter(torch.randn(4, 5, device=dev) * 0.1)
    params = [norm.weight, norm.bias, proj.weight, proj.bias, bias]
    goal = torch.randn(x.shape[0], 32, device=dev)

    def loss():
        q, k, v = proj(norm(x)).view(-1, 3, 4, 8).unbind(1)
        out = packed_attention(q, k, v, buckets.segments, bias=bias, buckets=buckets)
        return (out.reshape(-1, 32) - goal).square().mean()

    def loss64(w, b, pw, pb, t):
        xd = x.double()
        h = torch.nn.functional.layer_norm(xd, (24,), w, b)
        q, k, v = (h @ pw.T + pb).view(-1, 3, 4, 8).unbind(1)
        outs, lo = [], 0
        for i, n in enumerate(int(s) for s in batch.sizes):
            s = torch.einsum("ihd,jhd->hij", q[lo:lo + n], k[lo:lo + n]) * 8 ** -0.5 + t[:, buckets.dense(i).long()]
            outs.append(torch.einsum("hij,jhd->ihd", torch.softmax(s, 2), v[lo:lo + n]))
            lo += n
        return (torch.cat(outs).reshape(-1, 32) - goal.double()).square().mean()
    grads = torch.autograd.grad(loss(), params)
    doubles = [p.detach().double().requires_grad_() for p in params]
    truths = torch.autograd.grad(loss64(*doubles), doubles)
    for g, t in zip(grads, truths):
        # fp32 throughout: a few hundred roundings of terms about as large as the gradient's largest entry
        assert float((g.double() - t).abs().max()) <= 1e-5 * float(t.abs().max() + 1e-3)
    opt = AdamW(params, lr=1e-3, state_bits=bits)
    for _ in range(3):
        opt.zero_grad()
        loss().backward()
        opt.step()
    assert all(p.isfinite().all() for p in params)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_saved_tensors_that_were_laid_anew(dev, dtype):
    """Hooks of saved tensors hand back the same values in a layout of their own."""
    from gnn_amd import packed_attention, packed_segments, pair_buckets
    lengths = [70, 33]
    n = sum(lengths)
    q, k, v, do, bias, codes = make(dev, dtype, lengths, 4, 2, 24, buckets=3)
    want = run(q, k, v, do, lengths, True, bias=bias, codes=codes)
    seg = packed_segments(lengths, dev)
    buckets = pair_buckets(seg, torch.cat([c.reshape(-1) for c in codes]))

    def apart(t):                                   # elements of a row far apart
        wide = torch.zeros(*t.shape, 3, dtype=t.dtype, device=t.device)
        wide[..., 1] = t
        return wide[..., 1]
    packed = torch.empty(n, 8, 24, device=dev, dtype=dtype)
    for part, t in zip(packed.split([4, 2, 2], 1), (q, k, v)):
        part.copy_(t)
    for hook in (torch.autograd.graph.save_on_cpu(), torch.autograd.graph.saved_tensors_hooks(lambda t: t, apart)):
        leaves = [t.detach().requires_grad_() for t in (*packed.split([4, 2, 2], 1), bias)]
        with hook:
            out = packed_attention(*leaves[:3], seg, causal=True, bias=leaves[3], buckets=buckets)
        got = [out, *torch.autograd.grad(out, leaves, do)]
        assert all(torch.equal(a, b) for a, b in zip(got, want))
