"""``gnn_amd.layer_norm`` against the definition in 64 bits.

Tolerances: u = half a step of the element type for the one rounding at the end, and for the fp32 arithmetic before it
2^-24 per operation along the longest chain of additions (a thread's share of a row, the tree over the threads) times
the sum of the magnitudes that are added."""
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
E24 = 2.0 ** -24


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch.device("cuda:0")


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def truth(x, w, b, dy, eps=1e-5):
    """64-bit results and their tolerances' fp32 part (without the final rounding)."""
    x, w, dy = x.double(), w.double(), dy.double()
    b = torch.zeros_like(w) if b is None else b.double()
    width = x.shape[1]
    mean = x.mean(1, keepdim=True)
    var = ((x - mean) ** 2).mean(1, keepdim=True)
    rstd = (var + eps) ** -0.5
    h = (x - mean) * rstd
    y = h * w + b
    chain = width / 64 + 80                                       # additions a partial sum goes through, at most
    h_err = E24 * (chain * x.abs().mean(1, keepdim=True) * rstd + chain * h.abs() + 4 * (x.abs() + mean.abs()) * rstd)
    y_err = h_err * w.abs() + E24 * 4 * (h.abs() * w.abs() + b.abs())
    t = dy * w
    a, c = t.mean(1, keepdim=True), (t * h).mean(1, keepdim=True)
    dx = rstd * (t - a - h * c)
    abs_sum = t.abs() + t.abs().mean(1, keepdim=True) + h.abs() * (t * h).abs().mean(1, keepdim=True)
    dx_err = rstd * (E24 * (2 * chain + 8) * abs_sum + h_err * (t * h).abs().mean(1, keepdim=True)
                     + h.abs() * (t.abs() * h_err).mean(1, keepdim=True))
    rows = x.shape[0]
    row_chain = rows / 64 + 100
    dw, db = (dy * h).sum(0), dy.sum(0)
    dw_err = (dy.abs() * h_err).sum(0) + E24 * row_chain * (dy * h).abs().sum(0)
    db_err = E24 * row_chain * dy.abs().sum(0)
    return (y, dx, dw, db), (y_err, dx_err, dw_err, db_err)


def check(got, want, err, dtype, what):
    got = got.detach().double()
    bound = err + half_step(dtype) * (want.abs() + err) + torch.finfo(dtype).tiny
    worst = float(((got - want).abs() / bound).max()) if got.numel() else 0.0
    assert worst <= 1.0, (what, worst)


def make(dev, rows, width, dtype, seed=0, offset=0.5):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    x = (2 * torch.randn(rows, width, generator=g, device=dev) + offset).to(dtype)
    w = (1 + 0.2 * torch.randn(width, generator=g, device=dev)).to(dtype)
    b = (0.2 * torch.randn(width, generator=g, device=dev)).to(dtype)
    dy = torch.randn(rows, width, generator=g, device=dev).to(dtype)
    return x, w, b, dy


def run(x, w, b, dy):
    from gnn_amd import layer_norm
    leaves = [t.detach().requires_grad_() for t in (x, w) + (() if b is None else (b,))]
    y = layer_norm(*leaves)
    return y, torch.autograd.grad(y, leaves, dy)


# widths on both sides of every change of launch shape, odd ones, one column, and rows too wide for registers
WIDTHS = [1, 3, 16, 17, 33, 64, 65, 127, 129, 256, 257, 511, 513, 1000, 1025, 2049, 4095, 4097, 8191, 8193, 10007]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", WIDTHS)
def test_forward_and_backward(dev, dtype, width):
    rows = 37 if width > 300 else 333
    x, w, b, dy = make(dev, rows, width, dtype, seed=width)
    y, grads = run(x, w, b, dy)
    want, err = truth(x, w, b, dy)
    for got, t, e, name in zip((y, *grads), want, err, ("y", "dx", "dw", "db")):
        assert got.dtype == dtype
        check(got, t, e, dtype, name)


@pytest.mark.parametrize("rows", [1, 2, 5, 1023, 70001])
@pytest.mark.parametrize("dtype,width", [(torch.float32, 24), (torch.bfloat16, 96)])
def test_row_counts(dev, rows, dtype, width):
    x, w, b, dy = make(dev, rows, width, dtype, seed=rows)
    y, grads = run(x, w, b, dy)
    want, err = truth(x, w, b, dy)
    for got, t, e, name in zip((y, *grads), want, err, ("y", "dx", "dw", "db")):
        check(got, t, e, dtype, name)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bias", [True, False])
def test_fp32_weights_and_no_bias(dev, dtype, bias):
    x, w, b, dy = make(dev, 129, 200, dtype)
    w, b = w.float() * 1.001, b.float() if bias else None
    y, grads = run(x, w, b, dy)
    assert y.dtype == dtype and all(g.dtype == torch.float32 for g in grads[1:]) and len(grads) == 2 + bias
    want, err = truth(x, w, b, dy)
    check(y, want[0], err[0], dtype, "y")
    check(grads[0], want[1], err[1], dtype, "dx")
    for i in range(1 + bias):
        check(grads[1 + i], want[2 + i], err[2 + i], torch.float32, ("dw", "db")[i])


def test_strided_rows_more_dimensions_and_expanded_gradients(dev):
    from gnn_amd import layer_norm
    wide, w, b, dy = make(dev, 60, 96, torch.bfloat16)
    x = wide[:, 7:71]                                             # rows 96 apart, beginning at odd elements
    w, b = w[:64], b[:64]
    y, grads = run(x, w, b, dy[:, 3:67])
    want, err = truth(x, w, b, dy[:, 3:67])
    for got, t, e, name in zip((y, *grads), want, err, ("y", "dx", "dw", "db")):
        check(got, t, e, torch.bfloat16, name)
    x3 = x.reshape(3, 4, 5, 64)
    assert torch.equal(layer_norm(x3, w, b), y.detach().view(3, 4, 5, 64))
    every_other = wide[:, ::2]                                    # elements apart: read as a copy
    assert torch.equal(layer_norm(every_other, w[:48], b[:48]), layer_norm(every_other.contiguous(), w[:48], b[:48]))
    xr = x.detach().requires_grad_()                              # the gradient of a sum is one number, expanded
    layer_norm(xr, w, b).float().sum().backward()
    ones = torch.ones(60, 64, device=dev, dtype=torch.bfloat16)
    want, err = truth(x, w, b, ones)
    check(xr.grad, want[1], err[1], torch.bfloat16, "dx of a sum")


def test_rows_far_from_zero_and_constant_rows(dev):
    """The variance comes from distances to the mean: an offset of 1000 standard deviations costs the digits of x
    itself (already in the tolerance's |x| / sigma), not the square of them."""
    x, w, b, dy = make(dev, 50, 300, torch.float32, offset=2000.0)
    y, grads = run(x, w, b, dy)
    want, err = truth(x, w, b, dy)
    for got, t, e, name in zip((y, *grads), want, err, ("y", "dx", "dw", "db")):
        check(got, t, e, torch.float32, name)
    from gnn_amd import layer_norm
    same = torch.full((4, 96), 3.0, device=dev)
    assert torch.equal(layer_norm(same, w[:96], b[:96]), b[:96].expand(4, 96))


def test_empty_batch_and_not_finite_rows(dev):
    from gnn_amd import layer_norm
    x, w, b, dy = make(dev, 9, 70, torch.float32)
    e = x[:0].requires_grad_()
    wl = w.clone().requires_grad_()
    y = layer_norm(e, wl, b)
    y.sum().backward()
    assert y.shape == (0, 70) and e.grad.shape == (0, 70) and not wl.grad.any()
    clean = layer_norm(x, w, b)
    x[4, 3] = float("inf")
    x[6, 0] = float("nan")
    got = layer_norm(x, w, b)
    keep = [0, 1, 2, 3, 5, 7, 8]
    assert torch.equal(got[keep], clean[keep]) and got[4].isnan().any() and got[6].isnan().all()


def test_module_streams_and_repeatability(dev):
    from gnn_amd import LayerNorm
    m = LayerNorm(130, device=dev, dtype=torch.bfloat16)
    assert [n for n, _ in m.named_parameters()] == ["weight", "bias"]
    assert LayerNorm(8, bias=False).bias is None
    x, _, _, dy = make(dev, 5000, 130, torch.bfloat16)

    def once():
        xl = x.detach().requires_grad_()
        y = m(xl)
        return [y] + list(torch.autograd.grad(y, [xl, m.weight, m.bias], dy))
    first = once()
    assert all(torch.equal(a, c) for a, c in zip(first, once()))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = once()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, c) for a, c in zip(first, other))


def test_captured_step_replays(dev):
    from gnn_amd import layer_norm
    x, w, b, dy = make(dev, 700, 96, torch.float32)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        for _ in range(2):
            y = layer_norm(*leaves)
            torch.autograd.grad(y, leaves, dy)
        with torch.cuda.graph(graph, stream=s):
            y = layer_norm(*leaves)
            grads = torch.autograd.grad(y, leaves, dy)
    torch.cuda.current_stream().wait_stream(s)
    for seed in range(3):
        nx, _, _, nd = make(dev, 700, 96, torch.float32, seed=10 + seed)
        with torch.no_grad():
            x.copy_(nx)
            dy.copy_(nd)
        graph.replay()
        torch.cuda.synchronize()
        ry, rg = run(x, w, b, dy)
        assert torch.equal(y, ry) and all(torch.equal(a, c) for a, c in zip(grads, rg))


def test_gradient_against_differences(dev):
    x, w, b, dy = make(dev, 3, 11, torch.float32)
    _, (dx, dw, db) = run(x, w, b, dy)

    def loss(x, w, b):
        x = x.double()
        h = (x - x.mean(1, keepdim=True)) / ((x - x.mean(1, keepdim=True)).square().mean(1, keepdim=True) + 1e-5).sqrt()
        return float(((h * w.double() + b.double()) * dy.double()).sum())
    step = 1e-5                       # central differences of a smooth function: error of the order of step^2
    for at, grad in enumerate((dx, dw, db)):
        for i in range(0, grad.numel(), 5):
            vals = []
            for sign in (1, -1):
                args = [x.double().clone(), w.double().clone(), b.double().clone()]
                args[at].view(-1)[i] += sign * step
                vals.append(loss(*args))
            diff = (vals[0] - vals[1]) / (2 * step)
            assert abs(diff - float(grad.view(-1)[i])) <= 1e-4 * (1 + abs(diff))


def test_one_derivative(dev):
    """Gradients may be asked for with a graph; their own derivative raises."""
    from gnn_amd import layer_norm
    x, w, b, dy = make(dev, 20, 33, torch.float32)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    plain = torch.autograd.grad(layer_norm(*leaves), leaves, dy)
    y = layer_norm(*leaves)
    again = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    graph = torch.autograd.grad(y, leaves, dy.requires_grad_(), create_graph=True)
    assert all(torch.equal(p, a) and torch.equal(p, g) for p, a, g in zip(plain, again, graph))
    with pytest.raises(RuntimeError, match="once"):
        graph[0].sum().backward()


def test_rows_of_two_elements(dev):
    """What is left of equal terms: the same numbers as the formula's steps in fp32, each rounded by itself."""
    from gnn_amd import layer_norm
    x, w, b, dy = make(dev, 200, 2, torch.float32)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = layer_norm(*leaves)
    dx = torch.autograd.grad(y, leaves, dy)[0]
    with torch.no_grad():
        centred = x - (x[:, :1] + x[:, 1:]) / 2
        square = centred * centred
        rstd = 1.0 / torch.sqrt((square[:, :1] + square[:, 1:]) / 2 + 1e-5)
        hat, t = centred * rstd, dy * w
        th = t * hat
        want = rstd * (t - (t[:, :1] + t[:, 1:]) / 2 - hat * ((th[:, :1] + th[:, 1:]) / 2))
        assert torch.equal(y, hat * w + b) and torch.equal(dx, want)


def test_saved_rows_that_were_laid_anew(dev):
    """Hooks of saved tensors hand back the same values in a layout of their own: a strided slice comes back packed,
    from host memory too, and the backward pass goes by the rows as they are."""
    from gnn_amd import layer_norm
    wide, w, b, dy = make(dev, 60, 96, torch.float32)
    w, b, dy = w[:64], b[:64], dy[:, :64]
    plain = run(wide[:, 7:71], w, b, dy)[1]

    def apart(t):                                                 # and packed rows come back strided
        if t.dim() != 2 or t.shape[1] != 64:
            return t
        return torch.nn.functional.pad(t, (3, 5))[:, 3:67]
    hooks = (torch.autograd.graph.save_on_cpu(), torch.autograd.graph.saved_tensors_hooks(lambda t: t, apart),
             torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.contiguous()))
    for hook in hooks:
        for x in (wide[:, 7:71], wide[:, 7:71].contiguous()):
            leaves = [t.detach().requires_grad_() for t in (x, w, b)]
            with hook:
                y = layer_norm(*leaves)
            grads = torch.autograd.grad(y, leaves, dy)
            assert all(torch.equal(g, p) for g, p in zip(grads, plain))
