"""What the layer norm, AdamW and attention entry points refuse: at the C entry on the host, before anything is launched
(no GPU is touched), and in Python."""
import ctypes

import numpy as np
import pytest
import torch

NULL, SIZE, UNSUPPORTED, ALIGN = -1, -2, -3, -4
A = 4096          # stands for a device address: every call below returns before it would be used


@pytest.fixture(scope="module")
def lib():
    from gnn_amd import _lib
    return _lib.load()


def test_layer_norm_entry_points(lib):
    from gnn_amd.layer_norm import _Args

    def call(entry, **k):
        a = _Args()
        good = {n: A for n in ("x", "weight", "y", "mean", "rstd", "dy", "dx", "partials", "dw")}
        for name, value in (good | dict(x_stride=64, dy_stride=64, rows=4, width=64) | k).items():
            setattr(a, name, value)
        return entry(ctypes.addressof(a), None)
    fwd, bwd = lib.rwk_layer_norm_forward, lib.rwk_layer_norm_backward
    assert fwd(None, None) == NULL and bwd(None, None) == NULL
    for entry, names in ((fwd, ("x", "weight", "y", "mean", "rstd")),
                         (bwd, ("x", "dy", "weight", "mean", "rstd", "dx", "partials", "dw"))):
        for name in names:
            assert call(entry, **{name: None}) == NULL, name
        for bad in (dict(rows=0), dict(rows=-1), dict(width=0), dict(width=1 << 40), dict(x_stride=63)):
            assert call(entry, **bad) == SIZE, bad
        for bad in (dict(type=3), dict(type=-1), dict(weight_type=1), dict(type=1, weight_type=2)):
            assert call(entry, **bad) == UNSUPPORTED, bad
    assert call(bwd, dy_stride=1) == SIZE
    blocks = lib.rwk_layer_norm_backward_blocks
    assert blocks(0, 8, 0) == 0 and blocks(8, 0, 0) == 0 and blocks(1, 8, 0) == 1
    for rows, width in ((10 ** 6, 64), (10 ** 6, 4096), (10 ** 6, 100000)):
        assert 1 <= blocks(rows, width, 0) <= 4096


def test_adamw_entry_point(lib):
    def step(n=1, **k):
        args = dict(chunks=A, n_chunks=1, size=1024, base=0, grads=(ctypes.c_void_p * n)(*[A] * n), n_grads=n, type=0, bits=32, lr=A, b1=0.9, b2=0.999, eps=1e-8, wd=0.0, seed=0, steps=A,
                    stream=None) | k
        return lib.rwk_adamw_step(*args.values())
    for name in ("chunks", "grads", "lr", "steps"):
        assert step(**{name: None}) == NULL, name
    for bad in (dict(n_chunks=0), dict(n_chunks=-3), dict(base=-1), dict(n_grads=0), dict(n_chunks=1 << 40)):
        assert step(**bad) == SIZE, bad
    for bad in (dict(type=3), dict(type=-1), dict(bits=16), dict(bits=0), dict(n=257), dict(size=0), dict(size=2048)):
        assert step(**bad) == UNSUPPORTED, bad
    assert {lib.rwk_adamw_chunk_size(n) for n in (0, 1, 10 ** 6, 10 ** 9)} == {1024, 4096}


def test_attention_entry_points(lib):
    from gnn_amd.attention import _Args

    def call(backward=False, **k):
        a = _Args()
        good = dict(heads=4, kv_heads=2, dim=64, rows=10, n_segments=1, n_items=1, scale=1.0, type=0, block_rows=32)
        for name in ("q", "k", "v", "out", "d_out", "dq", "dk", "dv", "seg_ptr", "stats", "delta", "q_items", "k_items"):
            good[name] = A
        for name, value in (good | k).items():
            setattr(a, name, value)
        return (lib.rwk_attention_backward if backward else lib.rwk_attention_forward)(ctypes.addressof(a), None)
    assert lib.rwk_attention_forward(None, None) == NULL and lib.rwk_attention_backward(None, None) == NULL
    biased = dict(n_buckets=4, table=A, codes=A, codes_by_key=A, code_start=A, d_table=A, d_table_partials=A)
    for backward in (False, True):
        names = ["q", "k", "v", "out", "seg_ptr", "q_items"]
        names += ["d_out", "dq", "dk", "dv", "stats", "delta", "k_items"] if backward else []
        for name in names:
            assert call(backward, **{name: None}) == NULL, name
        for name in ["table", "codes", "code_start"] + (["codes_by_key", "d_table", "d_table_partials"] if backward else []):
            assert call(backward, **(biased | {name: None})) == NULL, name
        for bad in (dict(heads=0), dict(kv_heads=0), dict(kv_heads=3), dict(dim=0), dict(rows=-1), dict(rows=1 << 31),
                    dict(n_segments=-1), dict(n_items=-1), dict(n_items=1 << 30), dict(scale=0.0), dict(scale=-1.0),
                    dict(scale=float("nan")), dict(n_buckets=-1)):
            assert call(backward, **bad) == SIZE, bad
        for bad in (dict(dim=129), dict(type=3), dict(type=-1), dict(block_rows=64), biased | dict(n_buckets=33)):
            assert call(backward, **bad) == UNSUPPORTED, bad
        assert call(backward, **(biased | dict(codes=A + 8))) == ALIGN
    assert call(n_items=0, q=None, seg_ptr=None) == 0          # nothing to do


def test_pair_bucket_entry_points(lib):
    def refused(entry, *front, outputs):
        good = [*front, A, A, A, 3, 32, *[A] * outputs, None]
        at = len(front)
        call = lambda i, v: entry(*[v if j == i else x for j, x in enumerate(good)])
        for i in (0, at, at + 1, at + 2, *range(at + 5, at + 5 + outputs)):
            assert call(i, None) == NULL, i
        assert call(at + 3, -1) == SIZE and call(at + 3, 1 << 31) == SIZE and call(at + 4, 64) == UNSUPPORTED
        for i in range(at + 5, at + 5 + outputs):
            assert call(i, A + 8) == ALIGN, i
        return call
    dense = refused(lib.rwk_pair_buckets_dense, A, A, outputs=2)
    assert dense(1, None) == NULL
    relative = refused(lib.rwk_pair_buckets_relative, A, 4, outputs=2)
    assert relative(1, -1) == SIZE and relative(1, 1 << 40) == SIZE
    hops = refused(lib.rwk_pair_buckets_hops, A, A, A, 4, outputs=1)
    assert hops(3, -1) == SIZE and hops(3, 256) == SIZE
    assert lib.rwk_pair_buckets_dense(None, None, None, None, None, 0, 32, None, None, None) == 0


def test_attention_scales_and_parts(lib):
    from gnn_amd.attention import _Args

    def call(**k):
        a = _Args()
        for name in ("q", "k", "v", "out", "d_out", "dq", "dk", "dv", "seg_ptr", "stats", "delta", "q_items", "k_items"):
            setattr(a, name, A)
        for name, value in (dict(heads=12, kv_heads=2, dim=64, rows=10, n_segments=1, n_items=1, scale=1.0, type=0,
                                 block_rows=32) | k).items():
            setattr(a, name, value)
        return lib.rwk_attention_backward(ctypes.addressof(a), None)
    for bad in (dict(scale=1e-31), dict(scale=1e31), dict(scale=float("inf")), dict(key_parts=-1), dict(key_parts=4),
                dict(key_parts=12), dict(key_parts=5)):
        assert call(**bad) == SIZE, bad
    assert call(key_parts=3) == NULL                           # no place for the parts' sums


def test_lengths_that_wrap_around():
    from gnn_amd import packed_segments
    for lengths in ([2 ** 62, 2 ** 62, 2 ** 62, 2 ** 62], [2 ** 31], torch.tensor([2 ** 30, 2 ** 30])):
        with pytest.raises(NotImplementedError, match="rows"):
            packed_segments(lengths)


def test_no_cpu_fallback():
    from gnn_amd import AdamW, layer_norm, packed_attention, packed_segments
    with pytest.raises(RuntimeError, match="HIP devices only"):
        layer_norm(torch.zeros(2, 4), torch.ones(4))
    with pytest.raises(RuntimeError, match="HIP devices only"):
        AdamW([torch.nn.Parameter(torch.zeros(3))])
    with pytest.raises(RuntimeError, match="HIP devices only"):
        packed_segments([3, 4], "cpu")
    x = torch.zeros(4, 2, 8)
    with pytest.raises(RuntimeError, match="HIP devices only"):
        packed_attention(x, x, x, None)


def test_optimiser_arguments():
    from gnn_amd import AdamW
    p = [torch.nn.Parameter(torch.zeros(3))]
    for bad in (dict(state_bits=16), dict(seed=-1), dict(seed=1 << 64), dict(lr=-1.0), dict(lr=float("nan")),
                dict(eps=-1e-8), dict(weight_decay=-0.1), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1))):
        with pytest.raises(ValueError):
            AdamW(p, **bad)


def test_segment_lengths():
    from gnn_amd import packed_segments
    for bad in ([1.5, 2.0], [[1, 2], [3, 4]], torch.tensor([1.0]), torch.tensor([True]), np.array(["a"]), "ab"):
        with pytest.raises(TypeError):
            packed_segments(bad, "cuda")
    with pytest.raises(ValueError):
        packed_segments([3, -1], "cuda")


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch.device("cuda:0")


@pytest.mark.gpu
def test_layer_norm_arguments(dev):
    from gnn_amd import layer_norm
    x, w = torch.zeros(3, 8, device=dev), torch.ones(8, device=dev)
    for args, kind in (((x, w[:7]), ValueError), ((x, w.view(2, 4)), ValueError), ((x, w, w[:7]), ValueError),
                       ((x[:, :0], w[:0]), ValueError), ((x[0, 0], w), ValueError), ((x, w, None, -1.0), ValueError),
                       ((x, w, None, float("nan")), ValueError), ((x.double(), w), TypeError), ((x.int(), w), TypeError),
                       ((x, w.half()), TypeError), ((x.half(), w.bfloat16()), TypeError),
                       ((x.half(), w.half(), w), TypeError), ((x, w.cpu()), RuntimeError)):
        with pytest.raises(kind):
            layer_norm(*args)


@pytest.mark.gpu
def test_adamw_arguments(dev):
    from gnn_amd import AdamW
    with pytest.raises(TypeError):
        AdamW([torch.nn.Parameter(torch.zeros(3, device=dev, dtype=torch.float64))])
    with pytest.raises(ValueError):
        AdamW([torch.nn.Parameter(torch.zeros(3, 4, device=dev).t())])
    p = torch.nn.Parameter(torch.zeros(4, device=dev))
    opt = AdamW([p])
    p.grad = torch.zeros(4, device=dev).to_sparse()
    with pytest.raises(RuntimeError, match="sparse"):
        opt.step()
    p.grad = None
    saved = opt.state_dict()
    saved["state"][0] = dict(saved["state"][0], exp_avg=torch.zeros(5, device=dev))
    with pytest.raises(ValueError):
        opt.load_state_dict(saved)
    with pytest.raises(ValueError):
        AdamW([p], state_bits=8).load_state_dict(opt.state_dict())


@pytest.mark.gpu
def test_attention_arguments(dev):
    from gnn_amd import packed_attention, packed_segments, pair_buckets, relative_buckets
    seg, other = packed_segments([3, 2], dev), packed_segments([3, 2], dev)
    q, k = torch.zeros(5, 4, 8, device=dev), torch.zeros(5, 2, 8, device=dev)
    bias, b = torch.zeros(4, 3, device=dev), pair_buckets(seg, torch.zeros(13, dtype=torch.uint8, device=dev))
    packed_attention(q, k, k, seg, bias=bias, buckets=b)
    cases = [((q[0], k, k, seg), {}, ValueError), ((q, k, k[:4], seg), {}, ValueError),
             ((q, k[:4], k[:4], seg), {}, ValueError), ((q, k[..., :7], k[..., :7], seg), {}, ValueError),
             ((q[:, :3], k, k, seg), {}, ValueError), ((q, k[:, :0], k[:, :0], seg), {}, ValueError),
             ((q[:4], k[:4], k[:4], seg), {}, ValueError), ((q.half(), k, k, seg), {}, TypeError),
             ((q.double(), k.double(), k.double(), seg), {}, TypeError), ((q, k.cpu(), k.cpu(), seg), {}, RuntimeError),
             ((q, k, k, seg), dict(scale=0.0), ValueError), ((q, k, k, seg), dict(scale=float("inf")), ValueError),
             ((q, k, k, seg), dict(bias=bias), ValueError), ((q, k, k, seg), dict(buckets=b), ValueError),
             ((q, k, k, seg), dict(bias=bias[:3], buckets=b), ValueError),
             ((q, k, k, seg), dict(bias=torch.zeros(4, 33, device=dev), buckets=b), ValueError),
             ((q, k, k, seg), dict(bias=bias.half(), buckets=b), TypeError),
             ((q, k, k, other), dict(bias=bias, buckets=b), ValueError)]
    for args, kw, kind in cases:
        with pytest.raises(kind):
            packed_attention(*args, **kw)
    wide = torch.zeros(5, 1, 129, device=dev)
    with pytest.raises(NotImplementedError):
        packed_attention(wide, wide, wide, seg)
    with pytest.raises(TypeError):
        pair_buckets(seg, torch.zeros(13, device=dev))
    with pytest.raises(ValueError):
        pair_buckets(seg, torch.zeros(12, dtype=torch.uint8, device=dev))
    with pytest.raises(RuntimeError):
        pair_buckets(seg, torch.zeros(13, dtype=torch.uint8))
    for bad in (dict(n_buckets=33), dict(n_buckets=0), dict(n_buckets=7), dict(n_buckets=32, max_distance=8)):
        with pytest.raises(ValueError):
            relative_buckets(seg, **bad)
