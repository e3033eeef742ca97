"""Attention of serialised point clouds on B200.

The layer that transformers over serialised clouds put on top of the point
operations of this package: points are ordered along a space-filling curve,
the clouds of a batch lie one after another in flat rows (Pointcept offsets:
inclusive cumulative ends, mps_pointops/pointcept.py:46-56 of
gamzerA/mps-pointops, which has no such layer itself), and a point attends to
its neighbours along the order of its own cloud.

* ``norm_rotate``: norms of queries and keys for each head and the rotation by
  position, in one pass over both.
* ``window_attention``: softmax attention inside each cloud with a sliding
  window, a few first rows that stay visible to all (sinks), shared key heads
  and a learned relative position bias by buckets.  One call serves training
  (every input but the positions has a gradient), inference over whole clouds
  and single new rows over cached keys.
* ``Segments``: the layout of a ragged batch, made once for a batch and used by
  all of its layers (making it reads the offsets on the host).
* ``log_buckets``: the bucket map of logarithmic distances.

float32, float16 and bfloat16; scores, softmax, sums and norms are held in
float32, weights and score gradients of 16-bit inputs are rounded to the input
type as operands of the tensor cores (float16 score gradients below 2^-24 vanish:
scale the loss).  All results are bit-reproducible.
CUDA tensors only; other tensors raise ``RuntimeError`` after validation.
"""

from __future__ import annotations

import ctypes
import math

import torch
from torch import Tensor
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _native as N

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_MAX_ENTRIES = 256
_MAX_REACH = 1024
_MAX_POSITION = (1 << 30) - 1


def _ends(value: Tensor, name: str) -> list[int]:
    if not isinstance(value, Tensor) or value.ndim != 1 or value.dtype not in (torch.int32,
                                                                                 torch.int64):
        raise ValueError(f"{name} must be a one-dimensional int32/int64 tensor")
    return value.tolist()


class Segments:
    """The clouds of a ragged batch.

    ``offset`` holds the inclusive cumulative ends of each cloud's query rows
    (``[4, 9]`` = rows 0-3 and 4-8), ``key_offset`` those of its key rows when
    keys are others than the queries' own rows (cached keys, a chunk of new
    rows).  Query row i of a cloud of Lq query and Lk key rows stands at
    position ``i + Lk - Lq`` of its keys.  Offsets are read on the host once,
    here (a synchronisation); the object may be used by any number of calls,
    on any stream of its device.
    """

    def __init__(self, offset: Tensor, key_offset: Tensor | None = None):
        ends = _ends(offset, "offset")
        key_ends = ends if key_offset is None else _ends(key_offset, "key_offset")
        if len(ends) != len(key_ends):
            raise ValueError("offset and key_offset must have the same batch count")
        if key_offset is not None and key_offset.device != offset.device:
            raise ValueError("offset and key_offset must be on the same device")
        self.device = offset.device
        self.clouds = len(ends)
        self.rows = ends[-1] if ends else 0
        self.keys = key_ends[-1] if key_ends else 0
        self.query_tiles = self._plan(ends, key_ends, 0)
        self.key_tiles = self._plan(key_ends, ends, 1)
        self.max_rows = max((b - a for a, b in zip((0, *ends), ends)), default=0)
        self.max_keys = max((b - a for a, b in zip((0, *key_ends), key_ends)), default=0)
        self._stream = None
        if self.device.type == "cuda":
            # Blocking copies: the tiles are on the device when this returns.
            self.query_tiles = self.query_tiles.to(self.device)
            self.key_tiles = self.key_tiles.to(self.device)
            self._stream = torch.cuda.current_stream(self.device).cuda_stream

    @staticmethod
    def _plan(own: list[int], other: list[int], keys: int) -> Tensor:
        n = len(own)
        a, b = (ctypes.c_int64 * n)(*own), (ctypes.c_int64 * n)(*other)
        count = N.lib().mpo_attention_plan(a, b, n, keys, None, 0)
        if count < 0:
            raise ValueError(N.last_error())
        tiles = torch.empty((count, 8), dtype=torch.int32)
        N.lib().mpo_attention_plan(a, b, n, keys, N.ptr(tiles), count)
        return tiles

    def _use(self, stream: int) -> None:
        """Keep the tiles' memory until the work queued now on this stream, the
        current one, is done."""
        if stream != self._stream:
            current = torch.cuda.current_stream(self.device)
            self.query_tiles.record_stream(current)
            self.key_tiles.record_stream(current)


def log_buckets(buckets: int, max_distance: int, bidirectional: bool = True,
                device: torch.device | str | None = None) -> Tensor:
    """Bucket of each difference key - query in [-max_distance, max_distance]:
    an int32 map for ``window_attention(buckets=...)``.

    Of the buckets of one direction the first half holds one distance each, the
    second half spans logarithmically what is left up to ``max_distance``; all
    beyond shares the last.  ``bidirectional``: keys ahead of the query have the
    upper half of the buckets; otherwise they share bucket 0."""
    if buckets < (4 if bidirectional else 2):
        raise ValueError("too few buckets")
    if not 0 < max_distance <= _MAX_REACH:
        raise ValueError(f"max_distance must be in [1, {_MAX_REACH}]")
    per_side = buckets // 2 if bidirectional else buckets
    exact = per_side // 2
    if max_distance <= exact:
        raise ValueError("max_distance must exceed half of a direction's buckets")
    out = []
    for d in range(-max_distance, max_distance + 1):
        base = per_side if bidirectional and d > 0 else 0
        n = abs(d) if bidirectional else max(-d, 0)
        if n >= exact:
            step = math.log(n / exact) / math.log(max_distance / exact) * (per_side - exact)
            n = min(per_side - 1, exact + int(step))
        out.append(base + n)
    return torch.tensor(out, dtype=torch.int32, device=device)


# ----------------------------------------------------------------------------- checks

def _heads(value: Tensor, name: str, dim: int | None = None) -> None:
    if not isinstance(value, Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if value.ndim != 3:
        raise ValueError(f"{name} must have shape (N, heads, D), got {tuple(value.shape)}")
    if value.dtype not in _DTYPES:
        raise TypeError(f"{name} must be float32, float16 or bfloat16")
    if dim is not None and value.shape[2] != dim:
        raise ValueError(f"{name} must have head size {dim}, got {value.shape[2]}")


def _same(value: Tensor, like: Tensor, name: str) -> None:
    if value.dtype != like.dtype:
        raise TypeError(f"{name} must be {like.dtype} like q")
    if value.device != like.device:
        raise ValueError(f"{name} must be on {like.device}")


def _rows(x: Tensor, elements: int) -> Tensor:
    """``x`` itself where its innermost axis is dense, each row starts on a multiple
    of ``elements`` elements and no axis is broadcast, else a dense copy."""
    rows, heads, inner = x.stride()
    if (inner == 1 and rows > 0 and heads > 0 and rows % elements == 0 and heads % elements == 0
            and heads < 1 << 31 and x.data_ptr() % (elements * x.element_size()) == 0) or x.numel() == 0:
        return x
    return x.clone(memory_format=torch.contiguous_format)


def _dense(x: Tensor | None) -> Tensor | None:
    """A dense copy of ``x`` unless it is dense and starts on 16 bytes."""
    if x is None:
        return None
    x = x.contiguous()
    return x if x.data_ptr() % 16 == 0 else x.clone()


def _tracked(*tensors: Tensor | None) -> bool:
    """Whether a result has to know its inputs: some require gradients, or carry a
    forward-mode tangent (which the autograd functions refuse).  Calls without go past
    the functions, 7 to 10 us of host time each."""
    grad = torch.is_grad_enabled()
    return any(x is not None and ((grad and x.requires_grad) or
                                  forward_ad.unpack_dual(x).tangent is not None) for x in tensors)


def _address(x: Tensor | None) -> int:
    return 0 if x is None else x.data_ptr()


def _stream(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


# ----------------------------------------------------------------------------- norm and rotation

_pack_rotate = N.packer(N.RotateArgs)
_POSITIONS = {torch.int32: 0, torch.float32: 1, torch.int64: 2}


def _rotate_call(backward: bool, q, k, wq, wk, position, freqs, eps, interleaved, out_q, out_k,
                 grad_q=None, grad_k=None, grad_wq=None, grad_wk=None) -> None:
    device = q.device

    def pack(ws, nbytes):
        return _pack_rotate(
            q.data_ptr(), k.data_ptr(), q.stride(0), q.stride(1), k.stride(0), k.stride(1),
            _address(grad_q), _address(grad_k), out_q.data_ptr(), out_k.data_ptr(), _address(wq),
            _address(wk), _address(grad_wq), _address(grad_wk), _address(position),
            _address(freqs), _address(ws), nbytes, q.shape[0], q.shape[1], k.shape[1], q.shape[2],
            0 if freqs is None else freqs.shape[1], 0 if freqs is None else freqs.shape[0],
            0 if position is None else _POSITIONS[position.dtype], int(interleaved),
            _DTYPES[q.dtype], eps,
            int(freqs is not None and freqs.dtype == torch.float64))

    with N.on_device(device):
        lib = N.lib()
        if not backward:
            N.check(lib.mpo_norm_rotate(pack(None, 0), _stream(device)), "norm_rotate")
            return
        nbytes = int(lib.mpo_norm_rotate_workspace_bytes(pack(None, 0)))
        ws = N.workspace(nbytes, device)
        N.check(lib.mpo_norm_rotate_backward(pack(ws, nbytes), _stream(device)),
                "norm_rotate backward")


def _rotate_forward(q, k, *rest):
    out_q = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    out_k = torch.empty(k.shape, dtype=k.dtype, device=k.device)
    _rotate_call(False, q, k, *rest, out_q, out_k)
    return out_q, out_k


class _NormRotate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, wq, wk, position, freqs, eps, interleaved):
        q, k = _rows(q, 4), _rows(k, 4)
        ctx.save_for_backward(q, k, wq, wk, position, freqs)
        ctx.options = (eps, interleaved)
        return _rotate_forward(q, k, wq, wk, position, freqs, eps, interleaved)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_q, grad_k):
        q, k, wq, wk, position, freqs = ctx.saved_tensors
        grad_q, grad_k = _dense(grad_q), _dense(grad_k)
        dq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        dk = torch.empty(k.shape, dtype=k.dtype, device=k.device)
        dwq = torch.empty_like(wq) if wq is not None and ctx.needs_input_grad[2] else None
        dwk = torch.empty_like(wk) if wk is not None and ctx.needs_input_grad[3] else None
        _rotate_call(True, q, k, wq, wk, position, freqs, *ctx.options, dq, dk, grad_q, grad_k,
                     dwq, dwk)
        return dq, dk, dwq, dwk, None, None, None, None


def norm_rotate(q: Tensor, k: Tensor, position: Tensor | None, freqs: Tensor | None, *,
                q_weight: Tensor | None = None, k_weight: Tensor | None = None,
                eps: float = 1e-6, interleaved: bool = False) -> tuple[Tensor, Tensor]:
    """Root-mean-square norm of each head of q (N, H, D) and k (N, K, D), times
    ``q_weight`` / ``k_weight`` (D,), then the rotation by position.

    Pair t of the first 2P elements of a head, (t, P + t) or with
    ``interleaved`` (2t, 2t + 1), turns by ``sum_a position[n, a] * freqs[a, t]``;
    elements beyond 2P are left as they are.  ``position`` is (N, A) or (N,),
    int32, int64 or float32, A up to 3 (grid coordinates, say, or a row index);
    ``freqs`` is (A, P), P a multiple of 4, float32 or float64: positions go to its
    type and the angle is formed in it (float64 where positions are large).  Both None: no rotation.
    D is a multiple of 8 up to 256.  q and k may be strided views (of a packed
    projection); results are dense.  Gradients reach q, k and the weights, not
    the positions or frequencies.
    """
    _heads(q, "q")
    _heads(k, "k", q.shape[2])
    _same(k, q, "k")
    n, dim = q.shape[0], q.shape[2]
    if k.shape[0] != n:
        raise ValueError("q and k must have the same row count")
    if dim % 8 or not 8 <= dim <= 256:
        raise ValueError("the head size must be a multiple of 8 up to 256")
    if q.shape[1] < 1 or k.shape[1] < 1:
        raise ValueError("q and k must have at least one head")
    if (position is None) != (freqs is None):
        raise ValueError("position and freqs must be given together")
    if not (math.isfinite(eps) and eps >= 0):
        raise ValueError("eps must be finite and not negative")
    if freqs is not None:
        if not isinstance(freqs, Tensor) or freqs.ndim != 2 or freqs.dtype not in (torch.float32,
                                                                                   torch.float64):
            raise ValueError("freqs must be a float32 or float64 tensor of shape (A, P)")
        axes, pairs = freqs.shape
        if not 1 <= axes <= 3:
            raise ValueError("freqs must have 1 to 3 axes")
        if pairs % 4 or 2 * pairs > dim:
            raise ValueError("freqs must have a multiple of 4 pairs, at most half of the head size")
        if not isinstance(position, Tensor) or position.dtype not in _POSITIONS:
            raise ValueError("position must be an int32, int64 or float32 tensor")
        if position.ndim == 1:
            position = position.unsqueeze(1)
        if tuple(position.shape) != (n, axes):
            raise ValueError(f"position must have shape ({n}, {axes})")
        if position.device != q.device or freqs.device != q.device:
            raise ValueError(f"position and freqs must be on {q.device}")
    weights = []
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None:
            if not isinstance(w, Tensor) or tuple(w.shape) != (dim,) or w.dtype not in _DTYPES:
                raise ValueError(f"{name} must be a floating-point tensor of shape ({dim},)")
            if w.device != q.device:
                raise ValueError(f"{name} must be on {q.device}")
            w = _dense(w.float())
        weights.append(w)
    N.require_cuda(q, "attention.norm_rotate")
    if freqs is not None:
        position, freqs = position.detach().contiguous(), _dense(freqs.detach())
        if freqs.shape[1] == 0:
            position = freqs = None
    args = (*weights, position, freqs, float(eps), bool(interleaved))
    if _tracked(q, k, *weights):
        return _NormRotate.apply(q, k, *args)
    return _rotate_forward(_rows(q, 4), _rows(k, 4), *args)


# ----------------------------------------------------------------------------- attention

# (device index, stream) -> a word in pinned host memory, and the same as a ctypes integer.
_statuses: dict[tuple[int, int], tuple[Tensor | None, ctypes.c_int32]] = {}


def _ran_out(word: ctypes.c_int32) -> bool:
    """Whether a wait ran out since this was last asked."""
    if not word.value:
        return False
    word.value = 0
    return True


def _raise_ran_out() -> None:
    raise RuntimeError("mps_pointops: a wait inside an earlier window_attention kernel ran out; "
                       "its results are not valid")


def _status(device: torch.device, stream: int) -> int:
    """Address of the word that a kernel on this stream sets when a bounded wait runs
    out; it is read here without waiting for the GPU."""
    entry = _statuses.get((device.index, stream))
    if entry is None:
        pinned = torch.zeros(1, dtype=torch.int32).pin_memory()
        entry = _statuses.setdefault((device.index, stream),
                                     (pinned, ctypes.c_int32.from_address(pinned.data_ptr())))
    elif _ran_out(entry[1]):
        _raise_ran_out()
    return ctypes.addressof(entry[1])


def check(device: torch.device | str | None = None) -> None:
    """Raise if a wait inside a ``window_attention`` kernel on ``device`` (default: the
    current one) ran out, which makes its results invalid (synchronises).  The waits
    are for the kernel's own copies and products, two seconds each at most; the next ``window_attention`` call on the same stream raises as well, without waiting,
    if the word has been set by then."""
    device = torch.device("cuda" if device is None else device)
    index = torch.cuda.current_device() if device.index is None else device.index
    torch.cuda.synchronize(index)
    if any([_ran_out(word) for (owner, _), (_, word) in list(_statuses.items()) if owner == index]):
        _raise_ran_out()


class _Options:
    """What a call of ``window_attention`` fixes besides its tensors."""

    __slots__ = ("segments", "left", "right", "sinks", "causal", "scale", "reach", "want_lse")


_pack_attention = N.packer(N.AttentionArgs)


def _attention_call(backward: bool, o: _Options, q, k, v, bias, out, lse, grad=None,
                    delta=None, dq=None, dk=None, dv=None, dtable=None) -> None:
    """``bias``: the table, the positions of queries and keys and the bucket map (or None)."""
    seg, device = o.segments, q.device
    table, qpos, kpos, mapping = bias
    stream = _stream(device)
    shape = (0,) * 4 if table is None else (_DTYPES[table.dtype], table.shape[0], table.shape[1],
                                            o.reach)

    def pack(ws, nbytes):
        return _pack_attention(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), q.stride(0), q.stride(1), k.stride(0),
            k.stride(1), v.stride(0), v.stride(1), out.data_ptr(), _address(lse),
            _address(grad), _address(delta), _address(dq), _address(dk),
            _address(dv), _address(table), _address(dtable), _address(qpos), _address(kpos),
            _address(mapping), seg.query_tiles.data_ptr(), seg.key_tiles.data_ptr(),
            status, seg.query_tiles.shape[0], seg.key_tiles.shape[0], q.shape[0],
            k.shape[0], _address(ws), nbytes, q.shape[1], k.shape[1], q.shape[2],
            _DTYPES[q.dtype], *shape, o.left, o.right, o.sinks, o.causal, seg.max_rows,
            seg.max_keys, seg.clouds, o.scale, int(backward))

    with N.on_device(device):
        lib = N.lib()
        status = _status(device, stream)
        args = pack(None, 0)
        nbytes = int(lib.mpo_window_attention_workspace_bytes(args))
        ws = None
        if nbytes:
            ws = N.workspace(nbytes, device)
            args = pack(ws, nbytes)
        seg._use(stream)
        call = lib.mpo_window_attention_backward if backward else lib.mpo_window_attention
        N.check(call(args, stream), "window_attention backward" if backward else "window_attention")


def _forward(q, k, v, bias, o: _Options):
    out, lse = torch.empty(q.shape, dtype=q.dtype, device=q.device), None
    if o.want_lse:
        lse = torch.empty((q.shape[1], q.shape[0]), dtype=torch.float32, device=q.device)
    _attention_call(False, o, q, k, v, bias, out, lse)
    return out, lse


class _WindowAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, o: _Options, *bias):
        vec = 16 // q.element_size()
        q, k, v = _rows(q, vec), _rows(k, vec), _rows(v, vec)
        out, lse = _forward(q, k, v, bias, o)
        # Positions and map among them: the backward forms the bias again, and autograd
        # refuses it if the caller has changed them since.
        ctx.save_for_backward(q, k, v, out, lse, *bias)
        ctx.options = o
        ctx.mark_non_differentiable(lse)
        return out, lse

    @staticmethod
    @once_differentiable
    def backward(ctx, grad, _):
        q, k, v, out, lse, *bias = ctx.saved_tensors
        o, table = ctx.options, bias[0]
        device = q.device
        grad = _dense(grad)
        dq = torch.empty(q.shape, dtype=q.dtype, device=device)
        dk = torch.empty(k.shape, dtype=k.dtype, device=device)
        dv = torch.empty(v.shape, dtype=v.dtype, device=device)
        delta = torch.empty_like(lse)
        dtable = None
        if table is not None and ctx.needs_input_grad[4]:
            dtable = torch.empty(table.shape, dtype=torch.float32, device=device)
        _attention_call(True, o, q, k, v, bias, out, lse, grad, delta, dq, dk, dv, dtable)
        if dtable is not None:
            dtable = dtable.to(table.dtype)
        return dq, dk, dv, None, dtable, None, None, None


def _limit(value, name: str) -> int:
    if isinstance(value, bool) or not isinstance(value, int):
        raise ValueError(f"{name} must be an integer")
    return -1 if value < 0 else min(value, 1 << 30)


def _positions(value: Tensor | None, rows: int, axes: int, like: Tensor, name: str) -> Tensor:
    if not isinstance(value, Tensor) or value.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{name} must be an int32 or int64 tensor")
    if value.ndim == 1:
        value = value.unsqueeze(1)
    if tuple(value.shape) != (rows, axes):
        raise ValueError(f"{name} must have shape ({rows}, {axes}), got {tuple(value.shape)}")
    if value.device != like.device:
        raise ValueError(f"{name} must be on {like.device}")
    return value


def _int32(position: Tensor) -> Tensor:
    """Dense int32 positions; int64 ones end at the kernels' limits."""
    if position.dtype == torch.int64:
        position = position.clamp(-_MAX_POSITION, _MAX_POSITION).to(torch.int32)
    return position.contiguous()


def window_attention(q: Tensor, k: Tensor, v: Tensor, segments: Segments | Tensor, *,
                     window: tuple[int, int] = (-1, -1), sinks: int = 0, causal: bool = False,
                     scale: float | None = None, bias_table: Tensor | None = None,
                     position: Tensor | None = None, key_position: Tensor | None = None,
                     buckets: Tensor | None = None,
                     return_lse: bool = False) -> Tensor | tuple[Tensor, Tensor]:
    """Attention of q (N, H, D) over k and v (M, K, D) inside each cloud.

    ``segments``: a ``Segments``, or the offset of a self-attention batch.  H is
    a multiple of K (each K head serves H / K query heads); D is a multiple of
    8 up to 128.  q, k and v may be strided views of a packed projection.

    Key j of a cloud is visible to its query at position p when
    ``j < sinks or p - left <= j <= p + right`` (``window = (left, right)``,
    negative: no limit on that side) and, if ``causal``, ``j <= p``.  A query that
    sees no key gets zeros.  Scores are ``scale * q.k`` (default 1 / sqrt(D)) plus
    the bias ``sum_a bias_table[a, bucket_a, h]``: ``position`` (N, A) and
    ``key_position`` (M, A; default ``position``) are integers below 2^30 in
    magnitude (int64 ones beyond are taken as 2^30 - 1 of their sign; longer codes
    need an origin of their own), ``bias_table`` (A, buckets, H) is learned, and the bucket of an axis
    is the difference key - query clamped to [-R, R], plus R, where
    ``buckets = 2 R + 1``; or, with the map ``buckets`` (2 R + 1,), what the map
    names there (``log_buckets``; names are clamped to the table).  A * buckets
    is at most 256.  Positions may change after the call, but not between a forward
    and its backward, where autograd refuses the change.  16-bit types: a row more than
    2^15 on some axis from the middle one of its 128 is formed pair by pair, about a
    microsecond for each; keep such rows few.

    ``return_lse``: also the logarithm of each row's softmax denominator, (H, N)
    float32, -inf for a row that sees no key (no gradient through it).
    Gradients reach q, k, v and bias_table.
    """
    _heads(q, "q")
    _heads(k, "k", q.shape[2])
    _heads(v, "v", q.shape[2])
    _same(k, q, "k")
    _same(v, q, "v")
    if k.shape != v.shape:
        raise ValueError("k and v must have the same shape")
    if q.shape[2] % 8 or not 8 <= q.shape[2] <= 128:
        raise ValueError("the head size must be a multiple of 8 up to 128")
    if k.shape[1] < 1 or q.shape[1] < 1 or q.shape[1] % k.shape[1]:
        raise ValueError("q must have a multiple of k's heads")
    o = _Options()
    if not isinstance(window, (tuple, list)) or len(window) != 2:
        raise ValueError("window must be (left, right)")
    o.left, o.right = _limit(window[0], "window"), _limit(window[1], "window")
    if isinstance(sinks, bool) or not isinstance(sinks, int) or sinks < 0:
        raise ValueError("sinks must be a nonnegative integer")
    o.sinks, o.causal = min(sinks, 1 << 30), int(bool(causal))
    o.scale = 1.0 / math.sqrt(q.shape[2]) if scale is None else float(scale)
    if not math.isfinite(o.scale):
        raise ValueError("scale must be finite")
    if not isinstance(segments, Segments):
        segments = Segments(segments)
    if segments.rows != q.shape[0]:
        raise ValueError(f"segments must end at q's row count ({q.shape[0]})")
    if segments.keys != k.shape[0]:
        raise ValueError(f"segments must end at k's row count ({k.shape[0]})")
    if segments.device != q.device:
        raise ValueError(f"segments must be on {q.device}")
    o.segments = segments
    o.reach = 0
    if bias_table is None:
        if position is not None or key_position is not None or buckets is not None:
            raise ValueError("position, key_position and buckets need a bias_table")
    else:
        if not isinstance(bias_table, Tensor) or bias_table.ndim != 3 or \
                bias_table.dtype not in _DTYPES:
            raise ValueError("bias_table must be a floating-point tensor of shape (A, buckets, H)")
        axes, entries, heads = bias_table.shape
        if heads != q.shape[1] or not 1 <= axes <= 3 or entries < 1:
            raise ValueError(f"bias_table must have shape (A, buckets, {q.shape[1]}) with A in 1..3")
        if axes * entries > _MAX_ENTRIES:
            raise ValueError(f"bias_table must have at most {_MAX_ENTRIES} axes * buckets")
        if bias_table.device != q.device:
            raise ValueError(f"bias_table must be on {q.device}")
        if buckets is not None:
            if not isinstance(buckets, Tensor) or buckets.ndim != 1 or buckets.dtype != torch.int32:
                raise ValueError("buckets must be a one-dimensional int32 tensor")
            if buckets.device != q.device:
                raise ValueError(f"buckets must be on {q.device}")
        span = entries if buckets is None else buckets.shape[0]
        if span % 2 == 0 or span > 2 * _MAX_REACH + 1:
            raise ValueError("an axis must span 2 R + 1 differences, R at most 1024")
        o.reach = span // 2
        qpos = _positions(position, q.shape[0], axes, q, "position")
        if key_position is None:
            if q.shape[0] != k.shape[0]:
                raise ValueError("key_position is needed where keys are not the queries' rows")
            kpos = qpos
        else:
            kpos = _positions(key_position, k.shape[0], axes, q, "key_position")
    N.require_cuda(q, "attention.window_attention")
    bias = (None,) * 4
    if bias_table is not None:
        same = kpos is qpos
        qpos = _int32(qpos)
        kpos = qpos if same else _int32(kpos)
        bias = (bias_table.contiguous(), qpos, kpos, None if buckets is None else buckets.contiguous())
    tracked = _tracked(q, k, v, bias_table)
    o.want_lse = bool(return_lse) or tracked
    if tracked:
        out, lse = _WindowAttention.apply(q, k, v, o, *bias)
    else:
        vec = 16 // q.element_size()
        out, lse = _forward(_rows(q, vec), _rows(k, vec), _rows(v, vec), bias, o)
    return (out, lse) if return_lse else out


__all__ = ["Segments", "check", "log_buckets", "norm_rotate", "window_attention"]
