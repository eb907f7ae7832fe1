"""``gnn_amd.AdamW`` against the formula in 64 bits (32-bit states) and, for the 8-bit states, against their definition
written out in numpy: every code and scale has to be equal, so a test that plants other rounding would fail."""
import copy

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
E24 = 2.0 ** -24
HYPER = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.02)
# chunk borders (4096 elements), block borders (256), vector borders (4), single elements
SIZES = [1, 3, 4, 255, 256, 257, 1023, 4095, 4096, 4097, 9001]


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch.device("cuda:0")


def make(dev, dtype, sizes, seed=0):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    params = [torch.nn.Parameter(torch.randn(n, generator=g, device=dev).to(dtype)) for n in sizes]
    grads = [[(torch.randn(n, generator=g, device=dev) * 10.0 ** (i % 4 - 2)).to(dtype) for i, n in enumerate(sizes)]
             for _ in range(4)]
    return params, grads


def formula(p, g, m, v, t, hyper):
    """One step in 64 bits."""
    b1, b2 = hyper["betas"]
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    up = hyper["lr"] * (m / (1 - b1 ** t)) / (torch.sqrt(v / (1 - b2 ** t)) + hyper["eps"])
    return p * (1 - hyper["lr"] * hyper["weight_decay"]) - up, m, v, up


@pytest.mark.parametrize("dtype", TYPES)
def test_32_bit_states_follow_the_formula(dev, dtype):
    """Per step from the kernel's own state: p, m and v each within their roundings - m and v three fp32 operations
    each, p the type's half step and a dozen fp32 operations on the update."""
    from gnn_amd import AdamW
    params, grads = make(dev, dtype, SIZES)
    opt = AdamW(params, **HYPER)
    u = torch.finfo(dtype).eps / 2
    for t, gs in enumerate(grads, 1):
        before = [(p.detach().double().clone(), opt.state[p]["exp_avg"].double().clone(),
                   opt.state[p]["exp_avg_sq"].double().clone()) for p in params]
        for p, g in zip(params, gs):
            p.grad = g
        opt.step()
        for p, g, (p0, m0, v0) in zip(params, gs, before):
            g = g.double()
            want, m, v, up = formula(p0, g, m0, v0, t, HYPER)
            got_m, got_v = opt.state[p]["exp_avg"].double(), opt.state[p]["exp_avg_sq"].double()
            assert ((got_m - m).abs() <= E24 * 4 * (m0.abs() + g.abs())).all()
            assert ((got_v - v).abs() <= E24 * 5 * v).all()
            bound = u * want.abs() + E24 * 4 * p0.abs() + E24 * 24 * up.abs() \
                + HYPER["lr"] * E24 * 8 * (m0.abs() + g.abs()) / (torch.sqrt(v) + 1e-8) + torch.finfo(dtype).tiny
            assert ((p.detach().double() - want).abs() <= bound * (1 + u)).all()
    assert float(opt.state_dict()["state"][0]["step"]) == 4


# --- 8-bit states: the definition in numpy ------------------------------------------------------------------------
def philox(n, tensor, step, seed):
    c = [np.arange(-(-n // 4), dtype=np.uint64), np.uint64(tensor), np.uint64(step), np.uint64(0)]
    c = [np.broadcast_to(x, c[0].shape).copy() for x in c]
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32
    low = np.uint64(0xFFFFFFFF)
    for _ in range(7):
        p0, p1 = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
        c = [(p1 >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), p1 & low, (p0 >> np.uint64(32)) ^ c[3] ^ np.uint64(k1), p0 & low]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return np.stack(c, 1).reshape(-1)[:n].astype(np.uint32)


def encode(x, bits, positive):
    """fp32 values in blocks of 256 -> (codes, scales), each operation rounded to fp32."""
    n = x.size
    f = np.float32
    blocks = np.zeros(-(-n // 256) * 256, f)
    blocks[:n] = np.abs(x)
    blocks = blocks.reshape(-1, 256)
    scale = blocks.max(1) * (f(1) / f(448))
    scale[scale < np.finfo(f).tiny] = 0
    with np.errstate(divide="ignore"):
        inverse = np.where(scale == 0, f(0), f(1) / scale)
    y = np.minimum(blocks * inverse[:, None], f(448)).reshape(-1)[:n]
    add = bits.astype(np.int64) << 4
    normal = ((y.view(np.uint32).astype(np.int64) + add) >> 20) - (120 << 3)
    small = ((y.astype(np.float64) * 2.0 ** 29).astype(np.int64) + add) >> 20
    code = np.where(y >= 2.0 ** -6, normal, small)
    if positive:
        code = np.where((code == 0) & (x > 0), 1, code)
    return (code | (np.signbit(x).astype(np.int64) << 7)).astype(np.uint8), scale


def decode(codes, scale):
    value = torch.from_numpy(codes.copy()).view(torch.float8_e4m3fn).float().numpy()
    return value * np.repeat(scale, 256)[:codes.size]


@pytest.mark.parametrize("dtype", TYPES)
def test_8_bit_states_are_the_defined_numbers(dev, dtype):
    from gnn_amd import AdamW
    params, grads = make(dev, dtype, SIZES, seed=1)
    seed = (7 << 32) + 12345
    opt = AdamW(params, state_bits=8, seed=seed, **HYPER)
    b1, b2 = HYPER["betas"]
    f = np.float32
    state = [[np.zeros(n, np.uint8), np.zeros(-(-n // 256), f), np.zeros(n, np.uint8), np.zeros(-(-n // 256), f)]
             for n in SIZES]
    u = torch.finfo(dtype).eps / 2
    for t, gs in enumerate(grads, 1):
        before = [p.detach().double().clone() for p in params]
        for p, g in zip(params, gs):
            p.grad = g
        opt.step()
        for i, (p, g, s) in enumerate(zip(params, gs, state)):
            gn = g.float().cpu().numpy()
            m = decode(s[0], s[1]) * f(b1) + gn * f(1 - b1)
            v = decode(s[2], s[3]) * f(b2) + (gn * f(1 - b2)) * gn
            bits = philox(gn.size, i, t, seed)
            s[0], s[1] = encode(m, bits & 0xFFFF, False)
            s[2], s[3] = encode(v, bits >> 16, True)
            st = opt.state[p]
            for name, mine in zip(("exp_avg", "exp_avg_scale", "exp_avg_sq", "exp_avg_sq_scale"), s):
                theirs = st[name].view(torch.uint8) if st[name].dtype == torch.float8_e4m3fn else st[name]
                assert np.array_equal(theirs.cpu().numpy(), mine), (name, gn.size, t)
            md, vd = (torch.from_numpy(z).double().to(dev) for z in (m, v))
            c1, c2 = 1 - b1 ** t, 1 - b2 ** t
            up = HYPER["lr"] * (md / c1) / (torch.sqrt(vd / c2) + HYPER["eps"])
            want = before[i] * (1 - HYPER["lr"] * HYPER["weight_decay"]) - up
            bound = u * want.abs() + E24 * (4 * before[i].abs() + 24 * up.abs()) + torch.finfo(dtype).tiny
            assert ((p.detach().double() - want).abs() <= bound * (1 + u)).all()


def test_8_bit_second_moment_keeps_moving(dev):
    """v of a gradient whose size drops a hundredfold follows the fp32 state down: its mean over many elements stays
    within the noise of the rounding (an eighth per value at most, averaged over 2^14 of them), where rounding to
    nearest would leave it where it was; and no positive v becomes zero."""
    from gnn_amd import AdamW
    g = torch.Generator(device=dev)
    g.manual_seed(3)
    n = 1 << 14
    p8, p32 = (torch.nn.Parameter(torch.zeros(n, device=dev)) for _ in range(2))
    o8, o32 = AdamW([p8], state_bits=8, betas=(0.9, 0.999)), AdamW([p32], betas=(0.9, 0.999))
    for t in range(1500):
        grad = torch.randn(n, generator=g, device=dev) * (1.0 if t < 500 else 0.01)
        p8.grad = p32.grad = grad
        o8.step()
        o32.step()
    st = o8.state[p8]
    v8 = st["exp_avg_sq"].float() * st["exp_avg_sq_scale"].repeat_interleave(256)
    v32 = o32.state[p32]["exp_avg_sq"]
    assert (st["exp_avg_sq"].float() > 0).all()
    # standard deviation of one value: about a quarter; of the mean: 0.25 / 128; five of them
    assert abs(float(v8.mean() / v32.mean()) - 1) < 0.01
    rms = float((p8 - p32).detach().square().mean().sqrt() / p32.detach().square().mean().sqrt())
    assert rms < 0.25


def test_zero_gradients_tiny_and_not_finite_values(dev):
    from gnn_amd import AdamW
    for bits in (8, 32):
        p = torch.nn.Parameter(torch.ones(1024, device=dev))
        opt = AdamW([p], lr=0.1, weight_decay=0.0, state_bits=bits)
        p.grad = torch.zeros(1024, device=dev)
        opt.step()
        assert torch.equal(p.detach(), torch.ones(1024, device=dev))          # 0 / (0 + eps)
        p.grad = torch.full((1024,), 1e-30, device=dev)                       # squares below the smallest number
        opt.step()
        assert p.isfinite().all()
        p.grad = torch.zeros(1024, device=dev)
        p.grad[300], p.grad[700] = float("inf"), float("nan")
        opt.step()
        opt.step()
        bad = ~p.isfinite()
        if bits == 32:
            assert bad.nonzero().flatten().tolist() == [300, 700]
        else:                                                                 # their blocks of 256
            assert bad[256:768].all() and not bad[:256].any() and not bad[768:].any()


def test_none_gradients_groups_and_unaligned_tensors(dev):
    """Two groups with their own rates, a tensor without gradient at one step (it does not age), tensors that begin at
    odd elements of a buffer, an empty one, more tensors than one launch holds; types mixed in a group."""
    from gnn_amd import AdamW
    base = torch.randn(30000, device=dev)
    at, ps = 1, []
    for i in range(300):
        n = 1 + (37 * i) % 91
        ps.append(torch.nn.Parameter(base[at:at + n]))
        at += n
    ps += [torch.nn.Parameter(torch.randn(513, device=dev).bfloat16()), torch.nn.Parameter(torch.empty(0, device=dev))]
    ref = [torch.nn.Parameter(p.detach().double()) for p in ps]
    groups = lambda q: [dict(params=q[:150], lr=1e-2), dict(params=q[150:], lr=3e-3, betas=(0.8, 0.95), weight_decay=0.1)]
    mine, theirs = AdamW(groups(ps)), torch.optim.AdamW(groups(ref), foreach=False)
    for t in range(3):
        for i, (p, r) in enumerate(zip(ps, ref)):
            skip = t == 1 and i % 7 == 0
            p.grad = None if skip else torch.randn_like(p)
            r.grad = None if skip else p.grad.double()
        if t == 2:
            for o in (mine, theirs):
                o.param_groups[0]["lr"] = 5e-3
        mine.step()
        theirs.step()
    for i, (p, r) in enumerate(zip(ps, ref)):
        # three steps: the type's half step each, and fp32 arithmetic on updates of at most a few rates
        tol = 3 * torch.finfo(p.dtype).eps / 2 * 4 + 1e-6
        assert ((p.detach().double() - r.detach()).abs() <= tol * (1 + r.detach().abs())).all(), i
    saved = mine.state_dict()["state"]
    assert float(saved[0]["step"]) == 2 and float(saved[1]["step"]) == 3
    rest = base[at:].clone()
    mine.step()
    assert torch.equal(base[at:], rest)                                       # nothing behind the last tensor


@pytest.mark.parametrize("bits", [8, 32])
def test_checkpoint_continues_bit_for_bit(dev, bits):
    from gnn_amd import AdamW
    params, grads = make(dev, torch.bfloat16, [700, 33], seed=5)

    def go(opt, ps, gs):
        for p, g in zip(ps, gs):
            p.grad = g
        opt.step()
    opt = AdamW(params, state_bits=bits, seed=9, **HYPER)
    for gs in grads[:2]:
        go(opt, params, gs)
    saved, weights = copy.deepcopy(opt.state_dict()), [p.detach().clone() for p in params]
    for gs in grads[2:]:
        go(opt, params, gs)
    fresh = [torch.nn.Parameter(w) for w in weights]
    other = AdamW(fresh, state_bits=bits, seed=9)
    other.load_state_dict(saved)
    assert other.param_groups[0]["lr"] == HYPER["lr"]
    for gs in grads[2:]:
        go(other, fresh, gs)
    for a, b in zip(params, fresh):
        assert torch.equal(a, b)
        for name, t in opt.state[a].items():
            if name != "step":
                assert torch.equal(t.view(torch.uint8) if t.dtype.itemsize == 1 else t,
                                   other.state[b][name].view(torch.uint8) if t.dtype.itemsize == 1 else other.state[b][name])
    assert all(t["exp_avg"].dtype == (torch.float8_e4m3fn if bits == 8 else torch.float32)
               for t in other.state_dict()["state"].values())
    with pytest.raises(ValueError):
        AdamW(fresh, state_bits=40 - bits).load_state_dict(saved)


def test_captured_step_replays_with_a_new_rate(dev):
    from gnn_amd import AdamW
    for bits in (8, 32):
        params, grads = make(dev, torch.float32, [5000, 77], seed=6)
        twin = [torch.nn.Parameter(p.detach().clone()) for p in params]
        a, b = AdamW(params, state_bits=bits, seed=2), AdamW(twin, state_bits=bits, seed=2)
        for q in (params, twin):
            for p, g in zip(q, grads[0]):
                p.grad = g.clone()
        a.step()                                                 # tables; the capture needs them
        b.step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            a.step()
        for k in range(4):
            if k == 2:
                for o in (a, b):
                    o.param_groups[0]["lr"] = 4e-4
                a.push_lr()
            for q in (params, twin):
                for p, g in zip(q, grads[k % 4]):
                    p.grad.copy_(g)
            graph.replay()
            torch.cuda.synchronize()
            b.step()
            for p, q in zip(params, twin):
                assert torch.equal(p, q), (bits, k)
        assert float(a.state_dict()["state"][0]["step"]) == 5


def test_parameters_that_move_and_strided_gradients(dev):
    from gnn_amd import AdamW
    p = torch.nn.Parameter(torch.randn(40, 30, device=dev))
    q = torch.nn.Parameter(p.detach().clone())
    a, b = AdamW([p]), AdamW([q])
    for t in range(3):
        g = torch.randn(30, 40, device=dev)
        p.grad, q.grad = g.t(), g.t().contiguous()
        a.step()
        b.step()
        if t == 0:
            p.data = p.data.clone()                              # another address: the tables follow
    assert torch.equal(p, q) and float(a.state_dict()["state"][0]["step"]) == 3


@pytest.mark.parametrize("bits", [8, 32])
def test_copies_go_on_by_themselves(dev, bits):
    """A deep copy has tensors of its own, the step counts of the original and the same numbers from then on."""
    from gnn_amd import AdamW
    params, grads = make(dev, torch.float32, SIZES)
    opt = AdamW(params, **HYPER, state_bits=bits, seed=7)
    for gs in grads[:2]:
        for p, g in zip(params, gs):
            p.grad = g.clone()
        opt.step()
    twin = copy.deepcopy(opt)
    copies = twin.param_groups[0]["params"]
    for o, ps in ((opt, params), (twin, copies)):
        for gs in grads[2:]:
            for p, g in zip(ps, gs):
                p.grad = g.clone()
            o.step()
    assert all(a.data_ptr() != b.data_ptr() and torch.equal(a, b) for a, b in zip(params, copies))
    a, b = (o.state_dict()["state"] for o in (opt, twin))
    assert all(int(a[i]["step"]) == 4 == int(b[i]["step"]) for i in a)


def test_a_refused_step_changes_nothing(dev):
    """Gradients are checked before the first launch, those of later groups and types too."""
    from gnn_amd import AdamW
    a, b = torch.nn.Parameter(torch.ones(300, device=dev)), torch.nn.Parameter(torch.ones(5, device=dev).half())
    opt = AdamW([{"params": [a]}, {"params": [b], "lr": 1.0}])
    a.grad, b.grad = torch.ones_like(a), torch.ones_like(b)
    opt.step()
    before = a.detach().clone()
    b.grad = torch.sparse_coo_tensor(torch.tensor([[0]], device=dev), torch.ones(1, device=dev).half(), (5,))
    with pytest.raises(RuntimeError, match="sparse"):
        opt.step()
    assert torch.equal(a, before) and int(opt.state_dict()["state"][0]["step"]) == 1


@pytest.mark.parametrize("bits", [8, 32])
def test_all_of_a_chunk_takes_one_step_count(dev, bits):
    """Elements that are alike stay alike, in every chunk of more than fit the device at once and in every quarter of
    one: no wavefront takes the count that another has advanced.  (With 8-bit states the same element of each tensor has
    bits of its own, so a twin with the same seed is compared instead.)"""
    from gnn_amd import AdamW
    n = 6 << 20
    params = [torch.nn.Parameter(torch.full((n,), 0.5, device=dev)) for _ in range(2)]
    opts = [AdamW([p], **HYPER, state_bits=bits, seed=3) for p in params]
    for t in range(40):
        for p, o in zip(params, opts):
            p.grad = torch.full((n,), (-0.9) ** t, device=dev)
            o.step()
    assert torch.equal(*params)
    if bits == 32:
        assert (params[0] == params[0][0]).all()
    counts = opts[0]._tables[0].steps
    assert counts.numel() == n // 4096 and (counts == 40).all()


@pytest.mark.parametrize("bits", [8, 32])
def test_states_that_a_caller_clears_or_replaces(dev, bits):
    """Cleared states begin anew, replaced ones are taken, and what was replaced is not written any more."""
    from collections import defaultdict
    from gnn_amd import AdamW
    for reset in ("clear", "replace", "assign", "count"):
        params, grads = make(dev, torch.float32, [700, 5000], seed=8)
        opt = AdamW(params, **HYPER, state_bits=bits, seed=4)

        def go(o, ps, gs):
            for p, g in zip(ps, gs):
                p.grad = g.clone()
            o.step()
        go(opt, params, grads[0])
        go(opt, params, grads[1])
        old = [dict(opt.state[p]) for p in params]
        before = [{n: t.clone() for n, t in st.items()} for st in old]
        fresh = [torch.nn.Parameter(p.detach().clone()) for p in params]
        other = AdamW(fresh, **HYPER, state_bits=bits, seed=4)
        if reset == "clear":
            opt.state.clear()
        elif reset == "assign":
            opt.state = defaultdict(dict)
        else:
            saved = copy.deepcopy(opt.state_dict())
            for p, s in zip(params, saved["state"].values()):
                if reset == "replace":                   # as after keeping them elsewhere for a while
                    for name, t in opt.state[p].items():
                        if name != "step":
                            opt.state[p][name] = t.cpu().to(dev)
                else:
                    opt.state[p]["step"] = torch.tensor(7.0)
                    s["step"] = torch.tensor(7.0)
            other.load_state_dict(saved)
        for gs in grads[2:]:
            go(opt, params, gs)
            go(other, fresh, gs)
        assert all(torch.equal(a, b) for a, b in zip(params, fresh)), reset
        a, b = (o.state_dict()["state"] for o in (opt, other))
        assert [float(s["step"]) for s in a.values()] == [float(s["step"]) for s in b.values()], reset
        if reset != "count":
            for was, now in zip(before, old):
                for name in was:
                    if name != "step":
                        assert torch.equal(was[name].view(torch.uint8), now[name].view(torch.uint8)), (reset, name)


@pytest.mark.parametrize("bits", [8, 32])
def test_parameters_and_states_that_no_longer_fit(dev, bits):
    """Same address, other elements: refused, with the step counts as they were."""
    from gnn_amd import AdamW

    def moved(change, kind, match):
        p = torch.nn.Parameter(torch.ones(32, 32, device=dev))
        opt = AdamW([p], state_bits=bits)
        p.grad = torch.ones_like(p)
        opt.step()
        change(p, opt)
        before = p.detach().clone()
        with pytest.raises(kind, match=match):
            opt.step()
        assert torch.equal(p, before) and int(opt.state_dict()["state"][0]["step"]) == 1

    def shrink(p, opt):
        p.grad = None
        p.data = p.data[:3]
        p.grad = torch.ones_like(p)

    def transpose(p, opt):
        p.data = p.data.t()

    def widen(p, opt):
        p.grad = None
        p.data = torch.ones(64, 64, device=dev)
        p.grad = torch.ones_like(p)

    def offload(p, opt):
        opt.state[p]["exp_avg"] = opt.state[p]["exp_avg"].cpu()

    def lose(p, opt):
        del opt.state[p]["exp_avg_sq"]

    def halve(p, opt):
        opt.state[p]["exp_avg"] = opt.state[p]["exp_avg"].half()
    moved(shrink, ValueError, "shape")
    moved(widen, ValueError, "shape")
    moved(transpose, ValueError, "contiguous")
    moved(offload, RuntimeError, "device")
    moved(lose, ValueError, "exp_avg_sq")
    moved(halve, ValueError, "float16")


def test_groups_that_a_caller_changes(dev):
    from gnn_amd import AdamW
    params, grads = make(dev, torch.float32, [300, 40, 9], seed=2)
    opt = AdamW(params[:2], lr=0.1, weight_decay=0.0)
    for p, g in zip(params, grads[0]):
        p.grad = g
    opt.step()
    kept = params[1].detach().clone()
    opt.param_groups[0]["params"] = [params[0], params[2]]
    before = params[2].detach().clone()
    opt.step()
    assert torch.equal(params[1], kept) and not torch.equal(params[2], before)
    assert float(opt.state.pop(params[1])["step"]) == 1.0            # torch saves no state of a parameter of no group
    assert [float(s["step"]) for s in opt.state_dict()["state"].values()] == [2.0, 1.0]


@pytest.mark.parametrize("strided", [False, True])
def test_gradients_are_freed_when_their_owner_frees_them(dev, strided):
    """Neither the gradients nor the copies of strided ones outlive the step."""
    from gnn_amd import AdamW
    n = 2048
    p = torch.nn.Parameter(torch.zeros(n, n, device=dev))
    opt = AdamW([p])
    for _ in range(3):
        before = torch.cuda.memory_allocated(dev)
        g = torch.ones(n, n, device=dev)
        p.grad = g.t() if strided else g
        del g
        opt.step()
        opt.zero_grad(set_to_none=True)
        torch.cuda.synchronize()
        assert torch.cuda.memory_allocated(dev) < before + 4 * n * n // 2
    assert (p == p[0, 0]).all() and float(p[0, 0]) < 0


def test_a_captured_step_outlives_its_tables(dev):
    """Replays after the states were loaded anew read and write what the capture did, which is still there."""
    from gnn_amd import AdamW
    params, grads = make(dev, torch.float32, [5000, 77], seed=6)
    opt = AdamW(params)
    for p, g in zip(params, grads[0]):
        p.grad = g.clone()
    opt.step()
    moments = [opt.state[p]["exp_avg"] for p in params]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    saved = copy.deepcopy(opt.state_dict())
    opt.load_state_dict(saved)
    at = [m.data_ptr() for m in moments]
    tables = [t.packed.data_ptr() for tables, _ in opt._captured for t in tables]
    del moments
    taken = [torch.empty(n, device=dev) for n in (5000, 77) for _ in range(40)]          # of the sizes given back
    assert not set(at) & {t.data_ptr() for t in taken} and len(tables) == 1
    for t in taken:
        t.zero_()
    new = [opt.state[p]["exp_avg"].clone() for p in params]
    graph.replay()
    torch.cuda.synchronize()
    assert all(not t.any() for t in taken)
    assert all(torch.equal(opt.state[p]["exp_avg"], n) for p, n in zip(params, new))
    assert int(opt.state_dict()["state"][0]["step"]) == 1


def test_tables_built_on_one_stream_and_dropped_on_another(dev):
    from gnn_amd import AdamW
    params, grads = make(dev, torch.float32, [5000, 77], seed=6)
    twin = [torch.nn.Parameter(p.detach().clone()) for p in params]
    a, b = AdamW(params), AdamW(twin)
    side = torch.cuda.Stream()
    for gs in grads:
        for p, q, g in zip(params, twin, gs):
            p.grad, q.grad = g.clone(), g.clone()
        b.step()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            a.step()
        torch.cuda.current_stream().wait_stream(side)
    a._drop_tables()
    assert all(torch.equal(p, q) for p, q in zip(params, twin)) and int(a.state[params[0]]["step"]) == 4


def test_options_that_would_be_another_optimiser(dev):
    """torch's checkpoints load where the steps are the same ones, and are refused, unchanged, where they are not."""
    from gnn_amd import AdamW
    p, q = (torch.nn.Parameter(torch.ones(40, device=dev)) for _ in range(2))
    for kind, options, good in ((torch.optim.AdamW, {}, True), (torch.optim.Adam, dict(weight_decay=0.0), True),
                                (torch.optim.AdamW, dict(amsgrad=True), False), (torch.optim.AdamW, dict(maximize=True), False),
                                (torch.optim.Adam, dict(weight_decay=0.1), False)):
        theirs = kind([q], lr=0.01, **options)
        q.grad = torch.ones_like(q)
        theirs.step()
        mine = AdamW([p], lr=0.5)
        if good:
            mine.load_state_dict(theirs.state_dict())
            assert torch.equal(mine.state[p]["exp_avg"], theirs.state[q]["exp_avg"]) and mine.param_groups[0]["lr"] == 0.01
        else:
            with pytest.raises(ValueError, match="gnn_amd.AdamW"):
                mine.load_state_dict(theirs.state_dict())
            assert mine.param_groups[0]["lr"] == 0.5 and not mine.state[p]["exp_avg"].any()
            if "weight_decay" not in options:
                with pytest.raises(ValueError, match="gnn_amd.AdamW"):
                    AdamW([dict(params=[p], **options)])


def test_8_bit_states_that_lie_in_one_buffer(dev):
    """A caller keeps the states packed, one behind the other: nothing is written behind a state's last element."""
    from gnn_amd import AdamW
    params, grads = make(dev, torch.float32, [300, 77, 512], seed=3)
    twin = [torch.nn.Parameter(p.detach().clone()) for p in params]
    a, b = AdamW(params, state_bits=8, seed=1), AdamW(twin, state_bits=8, seed=1)

    def go():
        for q in (params, twin):
            for p, g in zip(q, grads[0]):
                p.grad = g.clone()
        a.step()
        b.step()
    go()
    for name in ("exp_avg", "exp_avg_sq"):
        buffer, at = torch.full((4096,), 17, dtype=torch.uint8, device=dev), 0
        for p in params:
            view = buffer[at:at + p.numel()].view(torch.float8_e4m3fn)
            view.copy_(a.state[p][name])
            a.state[p][name] = view
            at += p.numel()
        kept = buffer.clone()
        go()
        assert torch.equal(buffer[at:], kept[at:])
    go()
    assert all(torch.equal(p, q) for p, q in zip(params, twin))
    for p, q in zip(params, twin):
        for name in ("exp_avg", "exp_avg_sq"):
            assert torch.equal(a.state[p][name].view(torch.uint8), b.state[q][name].view(torch.uint8))
