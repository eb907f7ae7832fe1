"""Attention inside the segments of a packed batch: the nodes of every graph of a block-diagonal batch, or the rows of
walks and prompts laid end to end.

The distance-biased walk models weigh all pairs of a graph's nodes by a fixed function of their hop distance, a softmax
of ``-alpha * dist`` per row (``rwgnn2/rwgnn_dis_bias6.py:222-250``; :mod:`gnn_amd.distance_bias` applies it).  Here
the weights are learned: ``softmax_j(scale * q_i . k_j + bias[h, bucket_ij]) v_j`` over the pairs of a segment, with a
trainable number per head and bucket of the pair - its hop distance (:func:`hop_buckets`), the rows' distance in a walk
(:func:`relative_buckets`) or any other code (:func:`pair_buckets`).

One launch forward and two backward (``csrc/rwk_attention_body.h``; one more for the bias gradient, and one where the
query heads of long blocks of keys are shared out); scores never reach memory and all sums run in a fixed order, so
results are bitwise reproducible.  HIP devices only.
"""
from __future__ import annotations

import ctypes
import math
from ctypes import c_float, c_int32, c_int64, c_void_p

import numpy as np
import torch

from . import _lib
from .structure import GraphStructure

__all__ = ["PackedSegments", "packed_segments", "PairBuckets", "pair_buckets", "relative_buckets", "hop_buckets",
           "packed_attention"]

_P, _I64 = c_void_p, c_int64


class _Args(ctypes.Structure):
    """``rwk_attention`` of ``rwk.h``."""
    _fields_ = [("q", _P), ("k", _P), ("v", _P), ("out", _P), ("out_low", _P), ("d_out", _P), ("dq", _P), ("dk", _P), ("dv", _P),
                ("q_row", _I64), ("q_head", _I64), ("k_row", _I64), ("k_head", _I64), ("v_row", _I64),
                ("v_head", _I64), ("do_row", _I64), ("do_head", _I64), ("seg_ptr", _P), ("n_segments", _I64),
                ("rows", _I64), ("heads", _I64), ("kv_heads", _I64), ("dim", _I64), ("scale", c_float),
                ("causal", c_int32), ("type", c_int32), ("block_rows", c_int32), ("stats", _P), ("delta", _P),
                ("codes", _P), ("codes_by_key", _P), ("code_start", _P), ("table", _P), ("n_buckets", _I64), ("d_table", _P),
                ("d_table_partials", _P), ("q_items", _P), ("k_items", _P), ("n_items", _I64), ("key_parts", c_int32), ("few_keys", c_int32),
                ("dkv_partials", _P)]


class PackedSegments:
    """Lengths of the segments of a packed batch and the launch lists made from them; build with
    :func:`packed_segments` once per batch."""

    def __init__(self, lengths: np.ndarray, device: torch.device):
        self.lengths, self.device = lengths, device
        starts = np.concatenate([[0], np.cumsum(lengths)])
        self.n_segments, self.total = int(lengths.size), int(starts[-1])
        self.starts = starts
        # Four wavefronts that share the tiles they read pay while most of their 32-row slots are filled; where
        # blocks of 128 rows would hold over half as much padding again as blocks of 32, a wavefront works alone.
        alone, shared = (int((-(-lengths // b) * b).sum()) for b in (32, 128))
        self.block_rows = 128 if 2 * shared <= 3 * alone else 32
        b = self.block_rows
        blocks = -(-lengths // b)
        seg = np.repeat(np.arange(self.n_segments), blocks)
        first = (np.arange(seg.size) - np.repeat(np.cumsum(blocks) - blocks, blocks)) * b
        n = lengths[seg]
        lists = [np.stack([seg, first], 1)[np.argsort(-work, kind="stable")]
                 for work in (n, np.minimum(n, first + b), n - first)]       # the longest blocks start first
        self.n_items = int(seg.size)
        # Weights in two numbers of a 16-bit type leave the result's own rounding as the only error, in one number its
        # 1.15 to 1.41 fold (from 32 to 2048 rows).  What they cost grows with the length: bf16, 16 heads of 64, 32768 rows in
        # segments of 64: 50 for 47 us, of 256: 76 for 58, of 2048: 435 for 314; heads of 128: 122 for 115, 229 for 126,
        # 1116 for 567.  One launch has one form, so the longest segment decides for all.
        self.few_keys = int(lengths.max(initial=0)) <= 256
        # rows that a block of keys meets: at most, and on average per place of 512 (two workgroups a compute unit)
        self._key_work = [(int(w.max(initial=0)), int(w.sum()) / 512) for w in (n, n - first)]
        packed = torch.from_numpy(np.ascontiguousarray(np.concatenate(
            [starts] + [x.reshape(-1) for x in lists]), dtype=np.int32)).to(device)
        self._arrays, self._stream = packed, _lib.current_stream(device)
        at = packed.data_ptr()
        self._seg_ptr = at
        self._items, self._q_causal, self._k_causal = (at + 4 * (starts.size + 2 * i * self.n_items) for i in range(3))

    def __reduce__(self):                                 # a copy has lists of its own
        return PackedSegments, (self.lengths, self.device)

    def key_parts(self, heads: int, kv_heads: int, causal: bool) -> int:
        """Workgroups that share a block of keys in the backward pass, each with its part of the query heads.  Whole,
        the longest block may be what all others wait for; every part has sums of its own that go through memory
        once more (a row's as long as 0.006 rows of products, measured) and the parts need a launch to add them.
        Backward passes: 4 prompts of up to 8192 tokens, 4 query heads to a key head, 128 elements in bf16, 3.43 ms
        whole, 3.10 in two parts, 3.17 in four; 48 of up to 1500, 64 elements in fp16, 495, 497 and 550 us."""
        group = heads // kv_heads
        most, share = self._key_work[causal]
        share *= heads

        def time(p):
            return max(most * (group // p), share) + (200 + 0.006 * p * self.total * kv_heads if p > 1 else 0)
        return min((p for p in range(1, group + 1) if group % p == 0), key=time)

    @property
    def seg_ptr(self) -> torch.Tensor:
        """int32 (n_segments + 1): first row of every segment."""
        return self._arrays[:self.n_segments + 1]


def packed_segments(lengths, device=None) -> PackedSegments:
    """``lengths``: rows of every segment in order (a sequence, array or tensor of integers; segments without rows
    are allowed), or a :class:`GraphStructure`, whose graphs are the segments.  ``device``: the HIP device, by default
    that of the tensor or structure, else the current one."""
    if isinstance(lengths, GraphStructure):
        if lengths.perm is not None:
            raise NotImplementedError("graph_indicator must be sorted (nodes of a graph contiguous)")
        device = lengths.device if device is None else device
        lengths = lengths.counts
    if isinstance(lengths, torch.Tensor):
        if device is None and lengths.is_cuda:
            device = lengths.device
        if lengths.is_floating_point() or lengths.is_complex() or lengths.dtype == torch.bool:
            raise TypeError("lengths must be integers")
        lengths = lengths.cpu().numpy()
    array = np.asarray(lengths)
    if array.size == 0:
        array = array.astype(np.int64)
    if array.ndim != 1 or array.dtype.kind not in "iu":
        raise TypeError("lengths must be a list of integers")
    if array.size and int(array.min()) < 0:
        raise ValueError("lengths must not be negative")
    if sum(array.tolist()) >= 2 ** 31:
        raise NotImplementedError("at most 2^31 - 1 rows")
    device = torch.device("cuda" if device is None else device)
    if device.type != "cuda":
        raise RuntimeError("gnn_amd runs on HIP devices only (no CPU fallback)")
    if device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    return PackedSegments(array.astype(np.int64), device)


class PairBuckets:
    """Bucket codes (uint8) of all pairs of a packed batch as the kernels read them: a row per query, and the same with
    a row per key for the pass that owns the keys.  Two bytes per pair, one if the codes are symmetric."""

    def __init__(self, segments: PackedSegments, symmetric: bool = False):
        self.segments = segments
        padded = -(-segments.lengths // 32) * 32
        sizes = segments.lengths * padded
        self._start = torch.from_numpy(np.concatenate([[0], np.cumsum(sizes)])).to(segments.device)
        self._codes = torch.empty(int(sizes.sum()), dtype=torch.uint8, device=segments.device)
        self._by_key = self._codes if symmetric else torch.empty_like(self._codes)
        self._stream = _lib.current_stream(segments.device)

    def dense(self, segment: int) -> torch.Tensor:
        """Codes of one segment, (n, n): query row, key row."""
        n = int(self.segments.lengths[segment])
        lengths = self.segments.lengths[:segment]
        start = int((lengths * (-(-lengths // 32) * 32)).sum())
        padded = -(-n // 32) * 32
        return self._codes[start:start + n * padded].view(n, padded)[:, :n]


def _fill(segments: PackedSegments, entry: str, *args, symmetric: bool = False) -> PairBuckets:
    buckets = PairBuckets(segments, symmetric)
    out = (buckets._codes.data_ptr(),) if symmetric else (buckets._codes.data_ptr(), buckets._by_key.data_ptr())
    _used_here(segments, None, buckets._stream)
    with _lib.device_guard(segments.device):
        _lib.check(getattr(_lib.load(), entry)(
            *args, segments._seg_ptr, buckets._start.data_ptr(), segments._items, segments.n_items,
            segments.block_rows, *out, _lib.current_stream(segments.device)), entry)
    return buckets


def pair_buckets(segments: PackedSegments, codes: torch.Tensor) -> PairBuckets:
    """``codes`` (uint8, on the segments' device): the bucket of every ordered pair, segment after segment, query row
    by query row (``sum(n * n)`` values).  A code of ``bias.shape[1]`` or more - 255, say - keeps the pair from
    attending."""
    if codes.dtype != torch.uint8:
        raise TypeError("codes must be uint8")
    if codes.device != segments.device:
        raise RuntimeError("codes and segments must be on the same device")
    squares = segments.lengths ** 2
    if codes.numel() != int(squares.sum()):
        raise ValueError(f"expected {int(squares.sum())} codes, got {codes.numel()}")
    flat = codes.reshape(-1).contiguous()
    start = torch.from_numpy(np.concatenate([[0], np.cumsum(squares)])).to(segments.device)
    return _fill(segments, "rwk_pair_buckets_dense", flat.data_ptr(), start.data_ptr())


def relative_buckets(segments: PackedSegments, n_buckets: int = 32, max_distance: int = 128,
                     bidirectional: bool = True) -> PairBuckets:
    """Buckets of the difference of two rows' places in their segment.  Half of a direction's buckets stand for the
    distances 0, 1, 2, ... one by one, the other half for ever wider ranges, growing geometrically up to
    ``max_distance``, from which on all share the last.  ``bidirectional``: keys behind the query have buckets of
    their own; otherwise they share bucket 0 (causal attention never looks there)."""
    per = n_buckets // 2 if bidirectional else n_buckets
    if not 1 <= int(n_buckets) <= 32 or per < 1 or (bidirectional and n_buckets % 2):
        raise ValueError("n_buckets must be in 1..32, even if bidirectional")
    exact = max(1, per // 2)
    if int(max_distance) <= exact:
        raise ValueError("max_distance must exceed the distances with a bucket of their own (%d)" % exact)
    reach = min(int(max_distance), int(segments.lengths.max(initial=1)))       # no rows lie further apart
    d = np.arange(-reach, reach + 1)                            # key row - query row
    dist = np.abs(d) if bidirectional else np.maximum(-d, 0)
    wide = exact + np.floor(np.log(np.maximum(dist, exact) / exact) / math.log(int(max_distance) / exact) * (per - exact))
    code = np.where(dist < exact, dist, np.minimum(wide, per - 1)).astype(np.int64)
    if bidirectional:
        code = code + np.where(d > 0, per, 0)
    table = torch.from_numpy(code.astype(np.uint8)).to(segments.device)
    return _fill(segments, "rwk_pair_buckets_relative", table.data_ptr(), reach)


def hop_buckets(adj: torch.Tensor, graph_indicator: torch.Tensor, max_distance: int = 3, far: str = "bucket",
                segments: PackedSegments = None) -> PairBuckets:
    """Buckets by hop distance on a block-diagonal batch (``adj``, ``graph_indicator`` as ``RW_NN.forward`` takes
    them, the matrix symmetric; ``rwgnn_dis_bias6.py:109-128``): 0 for a node itself, 1 .. ``max_distance`` for
    neighbourhoods, and every other pair of the graph in bucket ``max_distance + 1`` (``far="bucket"``) or kept from
    attending (``far="mask"``).  The result's ``segments`` are the graphs."""
    from .distance_bias import distance_bias_structure
    if far not in ("bucket", "mask"):
        raise ValueError('far must be "bucket" or "mask"')
    if segments is not None and segments.device != adj.device:
        raise RuntimeError("the matrix and segments must be on the same device")
    st = distance_bias_structure(adj, graph_indicator, max_distance=max_distance)
    if segments is None:
        segments = packed_segments(st.base)
    elif not np.array_equal(segments.lengths, st.base.counts.cpu().numpy()):
        raise ValueError("the segments are not the batch's graphs")
    return _fill(segments, "rwk_pair_buckets_hops", st.row_start.data_ptr(), _lib.ptr(st.col), _lib.ptr(st.dist),
                 st.max_distance + 1 if far == "bucket" else 255, symmetric=True)


def _used_here(segments: PackedSegments, buckets, stream: int):
    """Lists and codes that were made on another stream: their memory is not handed out again before this stream's
    work on them is done."""
    if segments._stream != stream:
        segments._arrays.record_stream(torch.cuda.current_stream(segments.device))
    if buckets is not None and buckets._stream != stream:
        for t in (buckets._codes, buckets._by_key, buckets._start):
            t.record_stream(torch.cuda.current_stream(segments.device))


def _heads(t: torch.Tensor) -> torch.Tensor:
    """The elements of a head have to be adjacent; rows and heads may lie anywhere."""
    return t if t.stride(2) == 1 or t.shape[2] == 1 else t.contiguous()


def _describe(q, k, v, segments, causal, scale, table, buckets):
    a = _Args()
    a.q, a.k, a.v = q.data_ptr(), k.data_ptr(), v.data_ptr()
    a.q_row, a.q_head, _ = q.stride()
    a.k_row, a.k_head, _ = k.stride()
    a.v_row, a.v_head, _ = v.stride()
    a.seg_ptr, a.n_segments = segments._seg_ptr, segments.n_segments
    a.rows, a.heads, a.dim = q.shape
    a.kv_heads = k.shape[1]
    a.scale, a.causal, a.type = scale, causal, _lib.element_type(q.dtype)
    a.block_rows, a.n_items, a.few_keys = segments.block_rows, segments.n_items, segments.few_keys
    a.q_items = segments._q_causal if causal else segments._items
    a.k_items = segments._k_causal if causal else segments._items
    if table is not None:
        a.codes, a.codes_by_key = buckets._codes.data_ptr(), buckets._by_key.data_ptr()
        a.code_start = buckets._start.data_ptr()
        a.table, a.n_buckets = table.data_ptr(), table.shape[1]
    return a


def _forward(q, k, v, segments, causal, scale, table, buckets, stats):
    a = _describe(q, k, v, segments, causal, scale, table, buckets)
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    if segments.total < a.rows:
        out[segments.total:].zero_()
    st = low = None
    a.out = out.data_ptr()
    if stats:
        st = torch.empty((a.heads, a.rows, 2), dtype=torch.float32, device=q.device)
        a.stats = st.data_ptr()
        if a.type:                                     # 16 bits: what the rounding of out leaves over
            low = torch.empty_like(out)
            a.out_low = low.data_ptr()
    dev = segments.device
    stream = _lib.current_stream(dev)
    _used_here(segments, buckets, stream)
    with _lib.device_guard(dev):
        _lib.check(_lib.load().rwk_attention_forward(ctypes.addressof(a), stream), "rwk_attention_forward")
    return out, st, low


class _PackedAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, table, segments, causal, scale, buckets):
        q, k, v = _heads(q.detach()), _heads(k.detach()), _heads(v.detach())
        table = None if table is None else table.detach().contiguous()
        out, stats, low = _forward(q, k, v, segments, causal, scale, table, buckets, True)
        ctx.save_for_backward(q, k, v, table, out, stats, low)
        ctx.rest = (segments, causal, scale, buckets)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_out):
        _lib.refuse_tangent(d_out)
        q, k, v, *rest = ctx.saved_tensors
        q, k, v = _heads(q), _heads(k), _heads(v)         # hooks of saved tensors may have laid them anew
        table, out, stats, low = (None if t is None else t.contiguous() for t in rest)
        segments, causal, scale, buckets = ctx.rest
        dev = q.device
        d_out = _heads(d_out)
        a = _describe(q, k, v, segments, causal, scale, table, buckets)
        dq = torch.empty(q.shape, dtype=q.dtype, device=dev)
        dk = torch.empty(k.shape, dtype=q.dtype, device=dev)
        dv = torch.empty(v.shape, dtype=q.dtype, device=dev)
        if segments.total < q.shape[0]:
            for t in (dq, dk, dv):
                t[segments.total:].zero_()
        delta = torch.empty((q.shape[1], q.shape[0]), dtype=torch.float32, device=dev)
        a.key_parts = segments.key_parts(q.shape[1], k.shape[1], causal)
        if a.key_parts > 1:
            parts = torch.empty((a.key_parts, 2, k.numel()), dtype=torch.float32, device=dev)
            a.dkv_partials = parts.data_ptr()
        a.out, a.out_low = out.data_ptr(), _lib.ptr(low)
        a.stats, a.delta = stats.data_ptr(), delta.data_ptr()
        a.d_out, a.dq, a.dk, a.dv = d_out.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr()
        a.do_row, a.do_head, _ = d_out.stride()
        d_table = None
        if table is not None:
            d_table = torch.empty(table.shape, dtype=table.dtype, device=dev)
            partials = torch.empty(table.numel() * segments.n_items, dtype=torch.float32, device=dev)
            a.d_table, a.d_table_partials = d_table.data_ptr(), partials.data_ptr()
        stream = _lib.current_stream(dev)
        _used_here(segments, buckets, stream)
        with _lib.device_guard(dev):
            _lib.check(_lib.load().rwk_attention_backward(ctypes.addressof(a), stream), "rwk_attention_backward")
        return dq, dk, dv, d_table, None, None, None, None


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, segments: PackedSegments,
                     causal: bool = False, scale: float = None, bias: torch.Tensor = None,
                     buckets: PairBuckets = None) -> torch.Tensor:
    """``q`` (N, H, D), ``k`` and ``v`` (N, H_kv, D) with H a multiple of H_kv (query heads ``h`` share key / value
    head ``h // (H / H_kv)``) and D at most 128, all float32, float16 or bfloat16; slices of one projection's output
    are read in place.  ``segments``: which rows belong together (:func:`packed_segments`); rows behind the last
    segment give zeros and take no gradient.  ``causal``: a row attends to itself and the rows before it.  ``scale``:
    factor of the products, positive, ``D ** -0.5`` by default.  ``bias`` (H, n_buckets <= 32) of the same type, with
    ``buckets``: added to the scaled products by the pair's bucket; an entry may be ``-inf``.

    Returns (N, H, D), contiguous.  A row that attends to nothing gives zeros.  Differentiable once with respect to
    q, k, v and bias.  Sums, softmax statistics and the bias gradient are fp32; for the 16-bit types probabilities
    are rounded to the type before they meet ``v`` (to two numbers of it for heads of up to 32 elements and in
    batches whose longest segment has at most 256 rows), and so are, in the backward pass, probabilities and the
    gradients of the scores before their products (to two numbers before ``k`` for heads of up to 32 elements).
    Errors are then up to 1.5 times those of rounding the results once (1.65 in segments of one or two rows).  fp16:
    these factors are scaled to the type's range first, so that small upstream gradients and many keys cost no
    digits.  Results repeat bit by bit; in another batch, whose longest segment or padding asks for another launch
    shape, the same segment may differ within these errors.  What a pair's rows hold counts for nothing where the
    pair does not attend, values that are not finite included: blocks of rows that such a value may have reached are
    computed a second time, which takes up to some twenty times as long (2 prompts of 2048 rows, 32 heads of 128:
    forward 0.1 ms, 1.9 with infinities all over ``v``).  Where it does attend, the elements it reaches are not
    finite, infinite or NaN."""
    if not q.is_cuda:
        raise RuntimeError("gnn_amd runs on HIP devices only (no CPU fallback)")
    shape, k_shape, dtype, device = q.shape, k.shape, q.dtype, q.device          # every look costs a small call time
    _lib.element_type(dtype)
    if len(shape) != 3 or len(k_shape) != 3 or k_shape != v.shape or shape[0] != k_shape[0] or shape[2] != k_shape[2]:
        raise ValueError(f"expected q (N, H, D), k and v (N, H_kv, D), got {tuple(shape)}, {tuple(k_shape)}, "
                         f"{tuple(v.shape)}")
    rows, heads, dim = shape
    kv_heads = k_shape[1]
    if heads < 1 or kv_heads < 1 or heads % kv_heads:
        raise ValueError(f"{heads} query heads cannot share {kv_heads} key / value heads")
    if not 1 <= dim <= 128:
        raise NotImplementedError("heads of 1 to 128 elements")
    if k.dtype is not dtype or v.dtype is not dtype:
        raise TypeError("q, k and v must have the same type")
    if k.device != device or v.device != device or segments.device != device:
        raise RuntimeError("q, k, v and segments must be on the same device")
    if segments.total > rows:
        raise ValueError(f"the segments cover {segments.total} rows of {rows}")
    if segments.n_items * heads >= 2 ** 31 or rows >= 2 ** 31:
        raise NotImplementedError("more blocks of rows than a launch holds")
    scale = dim ** -0.5 if scale is None else float(scale)
    if not 1e-30 <= scale <= 1e30:
        raise ValueError("scale must be in 1e-30 .. 1e30")
    if (bias is None) != (buckets is None):
        raise ValueError("bias and buckets go together")
    if bias is not None:
        if bias.dim() != 2 or bias.shape[0] != heads or not 1 <= bias.shape[1] <= 32:
            raise ValueError(f"bias has shape {tuple(bias.shape)}, expected ({heads}, 1..32)")
        if bias.dtype is not dtype:
            raise TypeError("bias must have the type of q")
        if bias.device != device:
            raise RuntimeError("q and bias must be on the same device")
        if buckets.segments is not segments:
            raise ValueError("the buckets were made for other segments")
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or (
            bias is not None and bias.requires_grad)) or _lib.forward_mode():
        return _PackedAttention.apply(q, k, v, bias, segments, bool(causal), scale, buckets)
    return _forward(_heads(q), _heads(k), _heads(v), segments, bool(causal), scale,
                    None if bias is None else bias.contiguous(), buckets, False)[0]
