"""Measured calls of four operators for models over packed graphs, walks and prompts: layer norm, attention inside
packed segments, attention with a learned bias by position buckets, and the AdamW step over many tensors.

``run`` computes them in plain torch arithmetic (``own = False``) or with the framework's kernels (``own = True``);
``exact`` gives the same outputs from the definitions in 64 bits.
"""
import math
import random

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_MASKED = 255                  # bucket code of a pair that does not attend
_BLOCK = 256                   # elements of a tensor that share one scale of an 8-bit state
_F8_MAX = 448.0                # largest finite value of float8_e4m3fn
_HYPER = dict(lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01)
_STEPS_BEFORE = 100            # the optimiser's step count when the measured step begins
_SEED = 20240229               # key of the optimiser's rounding bits


def _device():
    return torch.device("cuda", torch.cuda.current_device()) if torch.cuda.is_available() else torch.device("cpu")


# ------------------------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one small batch's pooled rows before a classifier, forward only: launch latency
        dict(name="norm_rows_bf16", op="norm", dtype="bf16", rows=17, width=256, train=False),
        # node features of a batch of 4096 molecule-sized graphs at hidden width 64, one training step
        dict(name="norm_nodes_f32", op="norm", dtype="f32", rows=102400, width=64, train=True),
        # tokens of a large pretraining batch
        dict(name="norm_tokens_bf16", op="norm", dtype="bf16", rows=32768, width=4096, train=True),
        # the ten parameter tensors of RW_NN at the default hyper-parameters: launch latency
        dict(name="adamw_rwnn_f32_32", op="adamw", dtype="f32", shapes="rwnn", width=32, bits=32),
        # one transformer block, fp32 weights and states
        dict(name="adamw_block_f32_32", op="adamw", dtype="f32", shapes="block", width=2048, bits=32),
        # the same block in bf16 with 8-bit states
        dict(name="adamw_block_bf16_8", op="adamw", dtype="bf16", shapes="block", width=2048, bits=8),
        # an odd narrow block, fp32 weights with 8-bit states
        dict(name="adamw_odd_f32_8", op="adamw", dtype="f32", shapes="block", width=333, bits=8),
        # one short prompt, forward only: launch latency
        dict(name="attn_short_bf16", op="attention", dtype="bf16", heads=8, kv_heads=2, dim=64, segments=1, low=61,
             high=61, causal=True, train=False, buckets=0, kind="none", tail=0),
        # a ragged batch of walks and short prompts padded to a fixed row count, training
        dict(name="attn_ragged_f16", op="attention", dtype="f16", heads=16, kv_heads=4, dim=64, segments=48, low=1,
             high=1500, causal=True, train=True, buckets=0, kind="none", tail=177),
        # long prompts with grouped heads, training
        dict(name="attn_long_bf16", op="attention", dtype="bf16", heads=32, kv_heads=8, dim=128, segments=4, low=1000,
             high=8192, causal=True, train=True, buckets=0, kind="none", tail=0),
        # whole-graph attention over 1024 protein-sized graphs with a bias by hop distance, fp32 training
        dict(name="bias_graphs_f32", op="attention", dtype="f32", heads=4, kv_heads=4, dim=16, segments=1024, low=100,
             high=500, causal=False, train=True, buckets=8, kind="hops", tail=0),
        # causal attention over packed walks with a bias by relative position, training
        dict(name="bias_walks_bf16", op="attention", dtype="bf16", heads=8, kv_heads=8, dim=64, segments=64, low=16,
             high=1024, causal=True, train=True, buckets=32, kind="relative", tail=0),
    ]


def _spread(rng, low, high):
    """An integer spread over the logarithm of [low, high]."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    dtype = rng.choice(["f32", "f16", "bf16"])
    op = rng.choice(["norm", "adamw", "attention", "bias"])
    if op == "norm":
        width = _spread(rng, 1, 8192)
        rows = _spread(rng, 1, max(1, min(200000, 16384 * 4096 // width)))
        return dict(op="norm", dtype=dtype, rows=rows, width=width, train=rng.random() < 0.75)
    if op == "adamw":
        shapes = rng.choice(["block", "block", "rwnn"])
        return dict(op="adamw", dtype=dtype, shapes=shapes, width=_spread(rng, 1, 1400 if shapes == "block" else 4096),
                    bits=rng.choice([8, 32]))
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    heads = kv_heads * rng.choice([1, 1, 2, 3, 4])
    dim = rng.choice([rng.randint(1, 128), 8 * rng.randint(1, 16), 16, 64, 128])
    high = _spread(rng, 1, 3000)
    low = rng.choice([1, high, _spread(rng, 1, high)])
    # at most a quarter of the largest listed case's products, and of the graphs' pairs for fp32
    pairs = (4e8 if dtype != "f32" else 4e7) / (heads * max(dim, 16)) * 64
    segments = _spread(rng, 1, max(1, min(1024, int(pairs / max(high * high, 256)))))
    case = dict(op="attention", dtype=dtype, heads=heads, kv_heads=kv_heads, dim=dim, segments=segments, low=low,
                high=high, causal=rng.random() < 0.5, train=rng.random() < 0.75, buckets=0, kind="none",
                tail=rng.choice([0, 0, 1, 100]))
    if op == "bias":
        case["buckets"] = rng.randint(2, 32)
        case["kind"] = rng.choice(["hops", "relative", "holes"])
    return case


def _lengths(case):
    """Segment lengths: the longest first, the others uniform in [low, high], the same for every seed."""
    n, low, high = case["segments"], case["low"], case["high"]
    r = random.Random("%d %d %d" % (n, low, high))
    return [high] + [r.randint(low, high) for _ in range(n - 1)]


def _pairs(case):
    if case["causal"]:
        return sum(n * (n + 1) // 2 for n in _lengths(case))
    return sum(n * n for n in _lengths(case))


def _shapes(case):
    d = case["width"]
    if case["shapes"] == "rwnn":     # adj_hidden, features_hidden, fc, bn, fc1, fc2 of RW_NN; width = penultimate_dim
        return [(16, 10), (16, 5, 4), (4, 1), (4,), (32,), (32,), (d, 32), (d,), (2, d), (2,)]
    return [(d,), (d,), (3 * d, d), (3 * d,), (d, d), (d,), (d,), (d,), (4 * d, d), (4 * d,), (d, 4 * d), (d,)]


def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "norm":
        n = case["rows"] * case["width"]
        w = case["width"] * e
        if case["train"]:            # x, dy in; y, dx, dw, db out
            return {"bytes": 4 * n * e + 4 * w, "flops": 17 * n}
        return {"bytes": 2 * n * e + 2 * w, "flops": 7 * n}
    if case["op"] == "adamw":
        sizes = [math.prod(s) for s in _shapes(case)]
        n = sum(sizes)
        per = 3 * e + (16 if case["bits"] == 32 else 4)      # p in and out, g in, both states in and out
        scales = 0 if case["bits"] == 32 else 16 * sum(-(-s // _BLOCK) for s in sizes)
        return {"bytes": n * per + scales, "flops": 14 * n}
    rows = sum(_lengths(case)) + case["tail"]
    q, kv = rows * case["heads"] * case["dim"], rows * case["kv_heads"] * case["dim"]
    products = 2 * case["dim"] * case["heads"] * _pairs(case)
    codes = sum(n * n for n in _lengths(case)) if case["buckets"] else 0
    table = case["heads"] * case["buckets"] * e
    if case["train"]:                # q, k, v, d_out in; out, dq, dk, dv out
        return {"bytes": (4 * q + 4 * kv) * e + codes + 2 * table, "flops": 7 * products}
    return {"bytes": (2 * q + 2 * kv) * e + codes + table, "flops": 2 * products}


# ------------------------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------------------------
def _chunks(lengths, per_pair):
    """Segments of similar length together, so that their square score tensors, padded to the longest, stay below
    2^27 values: lists of segment numbers."""
    order = sorted(range(len(lengths)), key=lambda g: -lengths[g])
    chunks = []
    for g in order:
        if chunks and (len(chunks[-1]) + 1) * lengths[chunks[-1][0]] ** 2 * per_pair <= 2 ** 27 \
                and 2 * lengths[g] >= lengths[chunks[-1][0]]:
            chunks[-1].append(g)
        else:
            chunks.append([g])
    return [c for c in chunks if lengths[c[0]] > 0]


def _offsets(lengths):
    rows, pairs = [0], [0]
    for n in lengths:
        rows.append(rows[-1] + n)
        pairs.append(pairs[-1] + n * n)
    return rows, pairs


def _padded(lengths, chunk, device):
    """Row numbers (B, L) and pair numbers (B, L, L) of a chunk of segments, zero where there is none, and the mask
    of the rows that exist."""
    rows, pairs = _offsets(lengths)
    n = torch.tensor([lengths[g] for g in chunk], device=device)
    first = torch.tensor([rows[g] for g in chunk], device=device)
    pair = torch.tensor([pairs[g] for g in chunk], device=device)
    i = torch.arange(max(lengths[g] for g in chunk), device=device)
    there = i[None, :] < n[:, None]
    row = torch.where(there, first[:, None] + i[None, :], 0)
    both = there[:, :, None] & there[:, None, :]
    at = torch.where(both, pair[:, None, None] + i[None, :, None] * n[:, None, None] + i[None, None, :], 0)
    return row, at, there, both


def _codes(case, lengths, gen, device):
    """Bucket codes of all ordered pairs inside the segments, segment after segment, row-major, uint8."""
    flat = torch.zeros(sum(n * n for n in lengths), dtype=torch.uint8, device=device)
    top = case["buckets"] - 1
    for chunk in _chunks(lengths, 1):
        _, at, there, both = _padded(lengths, chunk, device)
        size = there.shape[1]
        if case["kind"] == "relative":
            # half of the buckets by exact distance, the others by its logarithm up to 128
            d = torch.arange(size, device=device)
            d = (d[:, None] - d[None, :]).abs()
            half = max(1, case["buckets"] // 2)
            far = half + (torch.log(d.clamp(min=half) / half) / math.log(max(2.0, 128 / half)) * half).long()
            code = torch.where(d < half, d, far).clamp(max=top)[None].expand(both.shape)
        else:
            # hop distances of random graphs with about four neighbours a node; unreached pairs in the last bucket
            near = torch.rand(both.shape, generator=gen, device=device) * there.sum(1)[:, None, None] < 2
            step = ((near | near.transpose(1, 2)) & both).float()
            reached = torch.eye(size, device=device).expand(both.shape).contiguous()
            code = torch.where(reached > 0, 0, top)
            for hop in range(1, min(top, 8)):
                grown = ((torch.matmul(reached, step) + reached) > 0).float()
                code = torch.where((grown > 0) & (reached == 0), hop, code)
                reached = grown
            if case["kind"] == "holes":      # one node in eight is padding: neither attends nor is attended
                hole = torch.rand(there.shape, generator=gen, device=device) < 0.125
                code = torch.where(hole[:, :, None] | hole[:, None, :], _MASKED, code)
        flat[at[both]] = code[both].to(torch.uint8)
    return flat


def _to_f8(x, up):
    """8-bit state of non-negative or signed x by blocks of 256: (values as float8, scales); round to nearest."""
    flat = torch.nn.functional.pad(x.reshape(-1), (0, -x.numel() % _BLOCK)).view(-1, _BLOCK)
    scale = flat.abs().amax(1) / _F8_MAX
    y = (flat / scale[:, None]).clamp(-_F8_MAX, _F8_MAX)
    if up:
        y = y.clamp(min=2.0 ** -9)
    return y.to(torch.float8_e4m3fn).view(-1)[:x.numel()].view(x.shape), scale


def _inputs(case, seed):
    device, dtype = _device(), _TYPES[case["dtype"]]
    gen = torch.Generator(device=device)
    gen.manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=device)

    if case["op"] == "norm":
        shape = (case["rows"], case["width"])
        return dict(x=(2.0 * normal(*shape) + 0.5).to(dtype), weight=(1.0 + 0.1 * normal(case["width"])).to(dtype),
                    bias=(0.1 * normal(case["width"])).to(dtype), dy=normal(*shape).to(dtype))
    if case["op"] == "adamw":
        got = dict(param=[], grad=[], state=[])
        for shape in _shapes(case):
            got["param"].append((0.05 * normal(*shape)).to(dtype))
            got["grad"].append((0.01 * normal(*shape)).to(dtype))
            m = 0.004 * normal(*shape)
            v = 1e-4 * (normal(*shape).square() * 0.3 + 0.05)
            if case["bits"] == 32:
                got["state"].append([m, v])
            else:
                got["state"].append([*_to_f8(m, False), *_to_f8(v, True)])
        return got
    lengths = _lengths(case)
    rows, heads, kv = sum(lengths) + case["tail"], case["heads"], case["kv_heads"]
    qkv = normal(rows, heads + 2 * kv, case["dim"]).to(dtype)      # one projection's output
    q, k, v = qkv.split([heads, kv, kv], dim=1)
    got = dict(q=q, k=k, v=v, d_out=normal(rows, heads, case["dim"]).to(dtype), lengths=lengths)
    if case["buckets"]:
        got["table"] = normal(heads, case["buckets"]).to(dtype)
        got["codes"] = _codes(case, lengths, gen, device)
    return got


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    if not own:
        if case["op"] == "adamw":
            state["step"] = _STEPS_BEFORE
        return state
    import gnn_amd
    if case["op"] == "norm":
        for name in ("x", "weight", "bias"):
            state[name].requires_grad_(case["train"])
    elif case["op"] == "adamw":
        params = [torch.nn.Parameter(p) for p in state["param"]]
        opt = gnn_amd.AdamW(params, state_bits=case["bits"], seed=_SEED, **_HYPER)
        names = ("exp_avg", "exp_avg_sq") if case["bits"] == 32 else ("exp_avg", "exp_avg_scale", "exp_avg_sq",
                                                                     "exp_avg_sq_scale")
        saved = opt.state_dict()
        saved["state"] = {i: dict(zip(names, s), step=torch.tensor(float(_STEPS_BEFORE)))
                          for i, s in enumerate(state["state"])}
        opt.load_state_dict(saved)           # a run continued from a checkpoint
        for p, g in zip(params, state["grad"]):
            p.grad = g
        state["optimizer"] = opt
        state["outputs"] = [[p.detach()] + [opt.state[p][n] for n in names] for p in params]
    else:
        state["segments"] = gnn_amd.packed_segments(state["lengths"], state["q"].device)
        for name in ("q", "k", "v"):
            state[name] = state[name].detach().requires_grad_(case["train"])
        if case["buckets"]:
            state["buckets"] = gnn_amd.pair_buckets(state["segments"], state["codes"])
            state["table"].requires_grad_(case["train"])
    return state


# ------------------------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if own:
        return _run_own(state, case)
    with torch.no_grad():
        return {"norm": _plain_norm, "adamw": _plain_adamw, "attention": _plain_attention}[case["op"]](state, case)


def _run_own(state, case):
    import gnn_amd
    if case["op"] == "norm":
        y = gnn_amd.layer_norm(state["x"], state["weight"], state["bias"], eps=1e-5)
        if not case["train"]:
            return [y]
        return [y, *torch.autograd.grad(y, (state["x"], state["weight"], state["bias"]), state["dy"])]
    if case["op"] == "adamw":
        state["optimizer"].step()
        return state["outputs"]
    leaves = [state["q"], state["k"], state["v"]]
    if case["buckets"]:
        out = gnn_amd.packed_attention(*leaves, state["segments"], causal=case["causal"], bias=state["table"],
                                       buckets=state["buckets"])
        leaves.append(state["table"])
    else:
        out = gnn_amd.packed_attention(*leaves, state["segments"], causal=case["causal"])
    if not case["train"]:
        return [out]
    return [out, *torch.autograd.grad(out, leaves, state["d_out"])]


def _plain_norm(state, case):
    dtype = state["x"].dtype
    x, w, b = state["x"].float(), state["weight"].float(), state["bias"].float()
    centred = x - x.mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt((centred * centred).mean(1, keepdim=True) + 1e-5)
    hat = centred * rstd
    y = (hat * w + b).to(dtype)
    if not case["train"]:
        return [y]
    dy = state["dy"].float()
    t = dy * w
    dx = rstd * (t - t.mean(1, keepdim=True) - hat * (t * hat).mean(1, keepdim=True))
    return [y, dx.to(dtype), (dy * hat).sum(0).to(dtype), dy.sum(0).to(dtype)]


def _plain_bits(n, tensor, step, device):
    """32 random bits for each of n elements: Philox4x32 with seven rounds, one call for four elements (counter =
    {element / 4, tensor, step, 0}, key = the seed's two words), word = element % 4."""
    low = 0xFFFFFFFF
    c0 = torch.arange(-(-n // 4), device=device, dtype=torch.int64)
    c1, c2, c3 = torch.full_like(c0, tensor), torch.full_like(c0, step), torch.zeros_like(c0)
    k0, k1 = _SEED & low, _SEED >> 32

    def product(a, b):                       # high and low words of a 32 by 32 bit product
        upper, lower = a * (b >> 16), a * (b & 0xFFFF)
        upper = upper + (lower >> 16)
        return upper >> 16, ((upper & 0xFFFF) << 16) | (lower & 0xFFFF)

    for _ in range(7):
        h0, l0 = product(0xD2511F53, c0)
        h1, l1 = product(0xCD9E8D57, c2)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack([c0, c1, c2, c3], 1).view(-1)[:n]


def _plain_decode(value, scale):
    each = scale.repeat_interleave(_BLOCK)[:value.numel()]
    return (value.reshape(-1).float() * each).view(value.shape)


def _plain_encode(x, bits, nonzero):
    """x by blocks of 256 as float8 and scale, rounded up or down at random in proportion to the distances; where
    ``nonzero``, a positive value does not become zero."""
    n = x.numel()
    flat = torch.nn.functional.pad(x.reshape(-1), (0, -n % _BLOCK)).view(-1, _BLOCK)
    scale = flat.abs().amax(1) / _F8_MAX
    scale = torch.where(scale < torch.finfo(torch.float32).tiny, 0.0, scale)
    inverse = torch.where(scale == 0, 0.0, 1.0 / scale)
    y = (flat.abs() * inverse[:, None]).clamp(max=_F8_MAX).view(-1)[:n]
    add = bits << 4
    normal = (y.view(torch.int32).long() + add >> 20) - (120 << 3)
    small = ((y * 2.0 ** 29).long() + add) >> 20
    code = torch.where(y >= 2.0 ** -6, normal, small)
    if nonzero:
        code = torch.where((code == 0) & (x.reshape(-1) > 0), 1, code)
    code = code | (torch.signbit(x.reshape(-1)).long() << 7)
    return code.to(torch.uint8).view(torch.float8_e4m3fn).view(x.shape), scale


def _plain_adamw(state, case):
    state["step"] += 1
    step = state["step"]
    lr, (b1, b2), eps, decay = _HYPER["lr"], _HYPER["betas"], _HYPER["eps"], _HYPER["weight_decay"]
    c1, c2 = 1.0 - b1 ** step, math.sqrt(1.0 - b2 ** step)
    outputs = []
    for i, (p, g, s) in enumerate(zip(state["param"], state["grad"], state["state"])):
        g = g.float()
        m, v = (s[0], s[1]) if case["bits"] == 32 else (_plain_decode(s[0], s[1]), _plain_decode(s[2], s[3]))
        m = m * b1 + g * (1.0 - b1)
        v = v * b2 + (g * (1.0 - b2)) * g
        p.copy_(p.float() * (1.0 - lr * decay) - (lr / c1) * (m / (torch.sqrt(v) / c2 + eps)))
        if case["bits"] == 32:
            new = [m, v]
        else:
            bits = _plain_bits(p.numel(), i, step, p.device)
            new = [*_plain_encode(m, bits & 0xFFFF, False), *_plain_encode(v, bits >> 16, True)]
        for old, now in zip(s, new):
            old.copy_(now)
        outputs.append([p, *s])
    return outputs


def _plain_attention(state, case):
    q, k, v = state["q"].float(), state["k"].float(), state["v"].float()
    dtype, device, lengths = state["q"].dtype, state["q"].device, state["lengths"]
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    scale, group = 1.0 / math.sqrt(dim), heads // kv
    out, dq = torch.zeros_like(q), torch.zeros_like(q)
    dk, dv = torch.zeros_like(k), torch.zeros_like(v)
    d_out = state["d_out"].float()
    if case["buckets"]:
        table = state["table"].float()
        d_table = torch.zeros_like(table)
    for chunk in _chunks(lengths, heads):
        row, at, there, both = _padded(lengths, chunk, device)
        size = row.shape[1]
        mask = both
        if case["causal"]:
            i = torch.arange(size, device=device)
            mask = mask & (i[None, None, :] <= i[None, :, None])

        def take(x, repeat):                 # (N, heads, D) -> (B, heads, L, D), zero rows where there is none
            x = torch.where(there[:, :, None, None], x[row], 0.0).transpose(1, 2)
            return x.repeat_interleave(group, 1) if repeat else x.contiguous()

        qs, ks, vs = take(q, False), take(k, True), take(v, True)
        scores = torch.matmul(qs, ks.transpose(2, 3).contiguous()) * scale
        if case["buckets"]:
            code = state["codes"][at].long()
            mask = mask & (code < case["buckets"])
            code = code.clamp(max=case["buckets"] - 1)
            scores = scores + table[:, code].transpose(0, 1)
        scores = scores.masked_fill(~mask[:, None], -math.inf)
        top = scores.amax(3, keepdim=True)
        top = torch.where(torch.isinf(top), 0.0, top)
        prob = torch.exp(scores - top)
        total = prob.sum(3, keepdim=True)
        prob = prob / torch.where(total == 0, 1.0, total)
        o = torch.matmul(prob, vs)
        out[row[there]] = o.transpose(1, 2)[there]
        if not case["train"]:
            continue
        do = take(d_out, False)
        dvs = torch.matmul(prob.transpose(2, 3).contiguous(), do)
        d_prob = torch.matmul(do, vs.transpose(2, 3).contiguous())
        d_score = prob * (d_prob - (d_prob * prob).sum(3, keepdim=True))
        dqs = torch.matmul(d_score, ks) * scale
        dks = torch.matmul(d_score.transpose(2, 3).contiguous(), qs) * scale
        dq[row[there]] = dqs.transpose(1, 2)[there]
        for grad, part in ((dk, dks), (dv, dvs)):
            part = part.view(part.shape[0], kv, group, size, dim).sum(2)
            grad[row[there]] = part.transpose(1, 2)[there]
        if case["buckets"]:
            for b in range(case["buckets"]):
                hit = ((code == b) & mask).float()
                d_table[:, b] += (d_score * hit[:, None]).sum((0, 2, 3))
    got = [out.to(dtype)]
    if case["train"]:
        got += [dq.to(dtype), dk.to(dtype), dv.to(dtype)]
        if case["buckets"]:
            got.append(d_table.to(dtype))
    return got


# ------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    given = _inputs(case, seed)
    return {"norm": _exact_norm, "adamw": _exact_adamw, "attention": _exact_attention}[case["op"]](given, case)


def _exact_norm(given, case):
    x, w, b = (given[n].double().requires_grad_(case["train"]) for n in ("x", "weight", "bias"))
    var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
    y = torch.addcmul(b, (x - mean) * torch.rsqrt(var + 1e-5), w)
    if not case["train"]:
        return [y]
    return [y.detach(), *torch.autograd.grad(y, (x, w, b), given["dy"].double())]


def _exact_bits(n, tensor, step, device):
    import numpy as np
    low, shift = np.uint64(0xFFFFFFFF), np.uint64(32)
    word = np.zeros((4, -(-n // 4)), np.uint64)
    word[0], word[1], word[2] = np.arange(word.shape[1], dtype=np.uint64), tensor, step
    key = [_SEED % 2 ** 32, _SEED // 2 ** 32]
    for r in range(7):
        if r:
            key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
        a, b = word[0] * np.uint64(0xD2511F53), word[2] * np.uint64(0xCD9E8D57)
        word = np.stack([(b >> shift) ^ word[1] ^ np.uint64(key[0]), b & low,
                         (a >> shift) ^ word[3] ^ np.uint64(key[1]), a & low])
    return torch.from_numpy(word.T.reshape(-1)[:n].astype(np.int64)).to(device)


def _exact_round(x, chance, nonzero):
    """(float8 values of x over its block's scale, scales) in 64 bits; chance in [0, 1) per element."""
    n = x.numel()
    blocks = torch.zeros(-(-n // _BLOCK) * _BLOCK, dtype=torch.float64, device=x.device)
    blocks[:n] = x.reshape(-1)
    blocks = blocks.view(-1, _BLOCK)
    scale = blocks.abs().max(1).values / _F8_MAX
    y = torch.where(scale[:, None] > 0, blocks.abs() / scale[:, None], 0.0).view(-1)[:n]
    unit = torch.exp2(torch.floor(torch.log2(y.clamp(min=2.0 ** -6))) - 3)
    down = torch.floor(y / unit)
    value = (down + (y / unit - down + chance >= 1).double()) * unit
    if nonzero:
        value = torch.where((value == 0) & (x.reshape(-1) > 0), 2.0 ** -9, value)
    return (torch.sign(x.reshape(-1)) * value.clamp(max=_F8_MAX)).view(x.shape), scale


def _exact_adamw(given, case):
    step = _STEPS_BEFORE + 1
    lr, (b1, b2), eps, decay = _HYPER["lr"], _HYPER["betas"], _HYPER["eps"], _HYPER["weight_decay"]
    outputs = []
    for i, (p, g, s) in enumerate(zip(given["param"], given["grad"], given["state"])):
        p, g, n = p.double(), g.double(), p.numel()
        if case["bits"] == 32:
            m, v = s[0].double(), s[1].double()
        else:
            block = torch.arange(n, device=p.device).div(_BLOCK, rounding_mode="floor").view(p.shape)
            m, v = s[0].double() * s[1].double()[block], s[2].double() * s[3].double()[block]
        m = torch.lerp(m, g, 1 - b1)
        v = b2 * v + (1 - b2) * g ** 2
        p = p - lr * decay * p - lr * (m / (1 - b1 ** step)) / ((v / (1 - b2 ** step)).sqrt() + eps)
        if case["bits"] == 32:
            outputs.append([p, m, v])
            continue
        bits = _exact_bits(n, i, step, p.device)
        outputs.append([p, *_exact_round(m, (bits % 65536).double() / 65536, False),
                        *_exact_round(v, torch.div(bits, 65536, rounding_mode="floor").double() / 65536, True)])
    return outputs


def _exact_attention(given, case):
    heads, group = case["heads"], case["heads"] // case["kv_heads"]
    q, k, v, d_out = (given[n].double() for n in ("q", "k", "v", "d_out"))
    out, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    table = given["table"].double() if case["buckets"] else None
    d_table = torch.zeros_like(table) if case["buckets"] else None
    first = pair = 0
    for n in given["lengths"]:
        rows = slice(first, first + n)
        allowed = torch.ones(n, n, dtype=torch.bool, device=q.device)
        if case["causal"]:
            allowed = allowed.tril()
        if case["buckets"]:
            code = given["codes"][pair:pair + n * n].view(n, n).long()
            allowed = allowed & (code < case["buckets"])
            code = torch.where(allowed, code, 0)
        some = allowed.any(1)
        # all heads of a short segment together, the heads of a long one in turn
        at_once = heads if n <= 512 else group
        for h in range(0, heads, at_once):
            hs, ks = slice(h, h + at_once), slice(h // group, (h + at_once) // group)
            a, b, c = (t.transpose(0, 1).contiguous().requires_grad_(case["train"])
                       for t in (q[rows, hs], k[rows, ks], v[rows, ks]))
            leaves = [a, b, c]
            logit = torch.matmul(a.view(b.shape[0], group * n, -1), b.transpose(1, 2).contiguous())
            logit = logit.view(at_once, n, n) * case["dim"] ** -0.5
            if case["buckets"]:
                leaves.append(table[hs].clone().requires_grad_(case["train"]))
                logit = logit + leaves[3][:, code]
            logit = logit.masked_fill(~allowed, float("-inf")).masked_fill(~some[:, None], 0.0)
            prob = torch.softmax(logit, -1).masked_fill(~some[:, None], 0.0)
            o = torch.matmul(prob.view(b.shape[0], group * n, n), c).view(at_once, n, -1)
            out[rows, hs] = o.detach().transpose(0, 1)
            if case["train"]:
                grads = torch.autograd.grad(o, leaves, d_out[rows, hs].transpose(0, 1).contiguous())
                dq[rows, hs], dk[rows, ks], dv[rows, ks] = (t.transpose(0, 1) for t in grads[:3])
                if case["buckets"]:
                    d_table[hs] += grads[3]
        first, pair = first + n, pair + n * n
    if not case["train"]:
        return [out]
    return [out, dq, dk, dv] + ([d_table] if case["buckets"] else [])
