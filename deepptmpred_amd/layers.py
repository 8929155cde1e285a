"""Layer operators on whole proteins: attention over packed sequences with a sliding window, first tokens that stay
visible and a learned bias by relative position, and the per-head norm of queries and keys with the position rotation;
forward, backward, and the form that computes the rows of chosen sites only.

The classifier itself attends within windows of at most 51 residues (pred/train_PTM/model.py:43-85) with a position
table per window (model.py:16-41); these are the same layers for sequences of any length, so that the residue rows a
site is scored from (pred/train_PTM/predict.py:487-501) can be computed and trained on the device and handed to
``Scorer.score_protein_device`` without leaving it.

Tensors are torch tensors on one GPU, ``[rows, heads, head_dim]`` with the rows of all sequences one behind the other; any
strides of rows and heads do, if addresses and strides are multiples of 16 bytes, rows are less than 32 MiB apart and a head's
elements are adjacent.  What a call writes shares no memory with what it reads, except where it says so.  Types are float32,
bfloat16 and float16.  Calls go out on the current stream of the tensors' GPU and wait for nothing; what they need
besides their results they take from torch's allocator, so calls on several streams and captured graphs do not share
memory.  A plan may be dropped while calls on any stream still run; a captured graph needs its plans kept as it needs its
inputs.  Gradients are explicit calls, as everywhere in this package: a tensor that requires grad is refused while autograd
records, and so is one with a tangent of forward-mode differentiation.
"""
from __future__ import annotations

import ctypes as C
import struct
import threading
from typing import Optional, Sequence, Tuple

import numpy as np
import torch
import torch.autograd.forward_ad as _forward_ad

from . import _native

_TYPES = {torch.float32: _native.PRECISIONS["f32"], torch.bfloat16: _native.PRECISIONS["bf16"],
          torch.float16: _native.PRECISIONS["f16"]}

_SIZES = {_native.PRECISIONS["f32"]: 4, _native.PRECISIONS["bf16"]: 2, _native.PRECISIONS["f16"]: 2}

# The argument blocks of the C calls, packed in one go: a call's cost on the host counts where a protein is short.
_ROWS = "Qqqq"
_NO_ROWS = (0, 0, 0, 0)
_ATTENTION = struct.Struct("@QQ" + 4 * _ROWS + "QQQQQQ" + 4 * _ROWS + "Qiiiif")
_NORM_ROPE = struct.Struct("@" + 4 * _ROWS + "QQQQQQ" + 4 * _ROWS + "QQQQqiiiiiiif")


class _Block(threading.local):
    """Memory that a call's arguments are packed into, one per thread."""

    def __init__(self):
        self.attention = C.create_string_buffer(C.sizeof(_native.AttentionArgs))
        self.attention_at = C.addressof(self.attention)
        self.norm_rope = C.create_string_buffer(C.sizeof(_native.NormRopeArgs))
        self.norm_rope_at = C.addressof(self.norm_rope)


_block = _Block()
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(device: int) -> int:
    return _raw_stream(device) if _raw_stream is not None else torch.cuda.current_stream(device).cuda_stream


def _check(rc: int, what: str) -> int:
    if rc >= 0:
        return rc
    msg = f"{what}: {(_native.load_library().dptm_layer_last_error() or b'').decode('utf-8', 'replace')}"
    if rc == _native.DPTM_EINVAL:
        raise ValueError(msg)
    if rc == _native.DPTM_ENOMEM:
        raise MemoryError(msg)
    raise RuntimeError(msg)


def _device(device) -> torch.device:
    if isinstance(device, int):
        return torch.device("cuda", device)
    device = torch.device(device)
    if device.type == "cuda" and device.index is None:
        return torch.device("cuda", torch.cuda.current_device())
    return device


def _first(t, what: str):
    """Type code and GPU of a call's first tensor; the others have to agree."""
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{what}: expected torch tensors")
    code = _TYPES.get(t.dtype)
    if code is None:
        raise ValueError(f"{what}: dtype {t.dtype} is not float32, bfloat16 or float16")
    device = t.get_device()
    if device < 0:
        raise ValueError(f"{what}: tensors must be on a GPU")
    return code, device


def _refuse(t, what: str, name: str, dtype, device: int):
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{what}: {name} is not a torch tensor")
    if t.dtype != dtype:
        raise ValueError(f"{what}: {name} has dtype {t.dtype}, expected {dtype}")
    if t.get_device() != device:
        raise ValueError(f"{what}: {name} is on {t.device}, not on cuda:{device}")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{what}: {name} requires grad, and this call does not record; detach it or use no_grad")


def _refuse_tangents(what: str, **tensors):
    for name, t in tensors.items():
        if isinstance(t, torch.Tensor) and _forward_ad.unpack_dual(t).tangent is not None:
            raise ValueError(f"{what}: {name} carries a tangent of forward-mode differentiation, which this call would lose")


def _rows(t, what: str, name: str, dtype, device: int, heads: int, dim: int, rows: int):
    """Address, rows and strides of a tensor [rows or more, heads, dim]."""
    if not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.get_device() != device or t.requires_grad:
        _refuse(t, what, name, dtype, device)
    shape = t.shape
    if len(shape) != 3 or shape[1] != heads or shape[2] != dim:
        raise ValueError(f"{what}: {name} has shape {tuple(shape)}, expected [rows, {heads}, {dim}]")
    n = shape[0]
    if n < rows:
        raise ValueError(f"{what}: {name} has {n} rows, the call needs {rows}")
    row, head, one = t.stride()
    if one != 1 and n and heads:
        raise ValueError(f"{what}: the elements of a head of {name} are not adjacent")
    # the stride of a dimension of one entry says nothing
    return t.data_ptr(), n, row if n > 1 else heads * dim, head if heads > 1 else dim


def _flat(t, what: str, name: str, shape, dtype, device: int) -> int:
    if t is None:
        return 0
    if not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.get_device() != device or t.requires_grad:
        _refuse(t, what, name, dtype, device)
    if t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{what}: {name} must be contiguous of shape {tuple(shape)}, got {tuple(t.shape)}")
    return t.data_ptr()


def _result(t, like, what: str, name: str, device: int, heads: int, dim: int, rows: int):
    """A result tensor [rows, heads, dim], the caller's or a new one of ``like``'s type, and its address, rows and strides."""
    if t is not None:
        return t, _rows(t, what, name, like.dtype, device, heads, dim, rows)
    t = like.new_empty((rows, heads, dim))
    return t, (t.data_ptr(), rows, heads * dim, dim)


def _lengths(a, name: str) -> np.ndarray:
    a = np.asarray(a.cpu() if isinstance(a, torch.Tensor) else a)
    if a.size == 0:
        a = a.astype(np.int32)
    if a.ndim != 1 or a.dtype.kind not in "iu":
        raise ValueError(f"AttentionPlan: {name} must be a list of whole numbers")
    if a.size and (int(a.max()) > 2 ** 31 - 1 or int(a.min()) < -2 ** 31):
        raise ValueError(f"AttentionPlan: {name} does not fit 32 bits")
    return np.ascontiguousarray(a, dtype=np.int32)


def _whole(x, what: str, name: str, least: int = -2 ** 31, most: int = 2 ** 31 - 1) -> int:
    """``x`` as a whole number of 32 bits (a ctypes field would drop the bits above them)."""
    try:
        n = int(x)
    except (TypeError, ValueError, OverflowError):
        n = None
    if n is None or n != x or not least <= n <= most:
        raise ValueError(f"{what}: {name} must be a whole number in {least}..{most}, got {x!r}")
    return n


def _f32(x, what: str, name: str) -> float:
    """``x``, which an argument block holds in 32 bits."""
    if not abs(x) < 3.4e38:
        raise ValueError(f"{what}: {name} must be a number that float32 holds, got {x!r}")
    return x


class AttentionPlan:
    """The layout of one batch: lengths, window, heads, and the work list made from them.  Kept and used for every
    layer and step of that batch; it only holds what it was made with, so any number of calls may use it at once.

    ``q_lens`` / ``k_lens`` (default: the same): rows of every sequence, on the host.  Query ``i`` of a sequence stands at
    position ``i + k_len - q_len`` -- one new token behind a cache stands at its end -- or at ``q_positions`` (all
    sequences' rows one behind the other, in any order): the site rows of a protein are asked for by giving the sites as
    positions.  Key ``j`` is visible to a query at position ``p`` if ``j <= p + window[1]`` and (``j >= p - window[0]`` or
    ``j < sinks``); a negative side has no limit, ``window=(-1, 0)`` looks back only.  ``training=False`` leaves out what
    only ``attention_backward`` needs.  ``device=None`` keeps the plan on the host."""

    def __init__(self, q_lens: Sequence[int], k_lens: Optional[Sequence[int]] = None, *, heads: int, kv_heads: Optional[int] = None,
                 head_dim: int, window: Tuple[int, int] = (-1, -1), sinks: int = 0, q_positions=None, training: bool = True,
                 device=0):
        lib = _native.load_library()
        q = _lengths(q_lens, "q_lens")
        k = q if k_lens is None else _lengths(k_lens, "k_lens")
        if k.shape != q.shape:
            raise ValueError(f"AttentionPlan: {len(q)} query lengths and {len(k)} key lengths")
        pos = None
        if q_positions is not None:
            pos = _lengths(q_positions, "q_positions")
            if len(pos) != int(q.sum(dtype=np.int64)):
                raise ValueError(f"AttentionPlan: {len(pos)} positions for {int(q.sum(dtype=np.int64))} query rows")
        what, far = "AttentionPlan", 2 ** 31 - 1
        try:
            left, right = window
        except TypeError:
            raise ValueError(f"{what}: window must be a pair (left, right), got {window!r}") from None
        left, right = (max(-1, min(_whole(w, what, "window", -2 ** 63, 2 ** 63), far)) for w in (left, right))
        d = _native.AttentionDesc(_whole(heads, what, "heads"), _whole(heads if kv_heads is None else kv_heads, what, "kv_heads"),
                                  _whole(head_dim, what, "head_dim"), left, right, min(_whole(sinks, what, "sinks", most=2 ** 63), far), 1 if training else 0)
        if device is not None:
            device = _device(device)
            if device.type != "cuda":
                raise ValueError(f"{what}: device must be a GPU, or None for a plan that stays on the host, not {device}")
        words = np.empty(4096, dtype=np.int32)
        while True:
            n = _check(lib.dptm_attention_plan(C.byref(d), q.ctypes.data, k.ctypes.data, None if pos is None else pos.ctypes.data,
                                               len(q), words.ctypes.data, words.size), "AttentionPlan")
            if n <= words.size:
                break
            words = np.empty(n, dtype=np.int32)
        self.words = words[:n]
        self.heads, self.kv_heads, self.head_dim = d.heads, d.kv_heads, d.head_dim
        self.q_rows, self.k_rows = int(q.sum(dtype=np.int64)), int(k.sum(dtype=np.int64))
        self.training = bool(training)
        self.device = device
        self.device_words = None if device is None else torch.from_numpy(self.words).to(self.device)
        self._at = None if device is None else (self.words.ctypes.data, self.device_words.data_ptr())
        self._streams = set() if device is None else {_stream(self.device.index)}
        self._bytes: dict = {}

    def _words(self, what: str, device: int, stream: int):
        """Addresses of the plan's two copies, for a call on ``stream``."""
        if self._at is None:
            raise ValueError(f"{what}: the plan was made for the host only")
        if self.device.index != device:
            raise ValueError(f"{what}: the plan is on {self.device}, the tensors are on cuda:{device}")
        if stream not in self._streams:
            # the plan may be dropped while that stream still reads it
            self.device_words.record_stream(torch.cuda.current_stream(device))
            self._streams.add(stream)
        return self._at

    def _workspace(self, n_buckets: int, max_distance: int, backward: int) -> int:
        key = (n_buckets, max_distance, backward)
        n = self._bytes.get(key)
        if n is None:
            n = self._bytes[key] = _check(_native.load_library().dptm_attention_workspace(self.words.ctypes.data, *key), "AttentionPlan")
        return n


def relative_buckets(n_buckets: int, max_distance: int, bidirectional: bool = True, device=0):
    """Bucket of every relative position ``-max_distance .. max_distance`` (``j - p``), int32: half of a side's buckets one
    distance each, the others by the logarithm of the distance up to ``max_distance``; ``bidirectional``: the upper half of
    the buckets for keys behind the query, otherwise those count as distance 0.  Borders are found in whole numbers.
    ``device=None``: a NumPy array."""
    n_buckets, max_distance = (_whole(x, "relative_buckets", name) for x, name in ((n_buckets, "n_buckets"), (max_distance, "max_distance")))
    side = n_buckets // 2 if bidirectional else n_buckets
    near = side // 2
    if near < 1 or n_buckets > 64 or (bidirectional and n_buckets % 2):
        raise ValueError("relative_buckets: 2 to 64 buckets, a multiple of 2 and at least 4 if bidirectional")
    if not near < max_distance <= 1024:
        raise ValueError(f"relative_buckets: max_distance must be in {near + 1}..1024")
    of = np.arange(max_distance + 1, dtype=np.int32)
    steps = side - near
    for d in range(near, max_distance + 1):
        # the largest step with near (max_distance / near)^(step / steps) <= d
        k = 0
        while k + 1 < steps and d ** steps * near ** (k + 1) >= near ** steps * max_distance ** (k + 1):
            k += 1
        of[d] = near + k
    behind = of + side if bidirectional else np.zeros_like(of)
    behind[0] = 0
    m = np.concatenate([of[:0:-1], behind]).astype(np.int32)
    return m if device is None else torch.from_numpy(m).to(_device(device))


def rotary_table(n_positions: int, head_dim: int, base: float = 10000.0, device=0):
    """Cosine and sine of ``position * base^(-2 i / head_dim)``, float32 ``[n_positions, head_dim / 2]`` each; angles in 64 bits."""
    n_positions, head_dim = _whole(n_positions, "rotary_table", "n_positions"), _whole(head_dim, "rotary_table", "head_dim")
    if n_positions < 0 or head_dim < 2 or head_dim % 2 or not 0 < base < float("inf"):
        raise ValueError("rotary_table: bad sizes, or a base that is not positive and finite")
    angle = np.arange(n_positions, dtype=np.float64)[:, None] * float(base) ** (-np.arange(0, head_dim, 2, dtype=np.float64) / head_dim)
    cos, sin = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
    return torch.from_numpy(cos).to(_device(device)), torch.from_numpy(sin).to(_device(device))


def _bias(what: str, plan: AttentionPlan, table, buckets, dtype, device: int):
    """Addresses of table and buckets, number of buckets and largest distance."""
    if table is None and buckets is None:
        return 0, 0, 0, 0
    if table is None or buckets is None:
        raise ValueError(f"{what}: table and buckets go together")
    if not isinstance(table, torch.Tensor) or not isinstance(buckets, torch.Tensor):
        raise ValueError(f"{what}: table and buckets must be torch tensors")
    if table.dim() != 2 or table.shape[1] != plan.heads:
        raise ValueError(f"{what}: table has shape {tuple(table.shape)}, expected [buckets, {plan.heads}]")
    if buckets.dim() != 1 or buckets.shape[0] % 2 == 0:
        raise ValueError(f"{what}: buckets must hold an odd number of entries, one per distance")
    return (_flat(table, what, "table", table.shape, dtype, device), _flat(buckets, what, "buckets", buckets.shape, torch.int32, device),
            table.shape[0], buckets.shape[0] // 2)


def attention(q, k, v, plan: AttentionPlan, *, scale: Optional[float] = None, table=None, buckets=None, out=None, lse=None):
    """Softmax attention of ``plan``'s sequences: ``(out [q_rows, heads, head_dim], lse float32 [heads, q_rows])``.

    Scores are ``scale * q.k`` (default ``head_dim ** -0.5``) plus ``table[buckets[j - p], head]`` where a relative position
    bias is given (``relative_buckets``; ``table [buckets, heads]`` of the tensors' type).  A row that sees no key gets zeros and
    ``-inf``; a table entry at or below ``-2^100`` hides the pairs of its bucket.  ``out`` and ``lse`` may be given; rows of ``out`` behind the plan's are left as they are."""
    lib, what, dim = _native.load_library(), "attention", plan.head_dim
    code, device = _first(q, what)
    if _forward_ad._current_level >= 0:         # inside dual_level: asking every tensor takes microseconds
        _refuse_tangents(what, q=q, k=k, v=v, table=table, out=out, lse=lse)
    dtype, heads, nq, nk = q.dtype, plan.heads, plan.q_rows, plan.k_rows
    stream = _stream(device)
    host, dev = plan._words(what, device, stream)
    out, out_rows = _result(out, q, what, "out", device, heads, dim, nq)
    if lse is None:
        lse = q.new_empty((heads, nq), dtype=torch.float32)
    table_at, buckets_at, n_buckets, reach = _bias(what, plan, table, buckets, dtype, device)
    n = plan._workspace(0, 0, 0)
    hold = q.new_empty((n // _SIZES[code],)) if n else None
    block = _block
    _ATTENTION.pack_into(
        block.attention, 0, host, dev, *_rows(q, what, "q", dtype, device, heads, dim, nq),
        *_rows(k, what, "k", dtype, device, plan.kv_heads, dim, nk), *_rows(v, what, "v", dtype, device, plan.kv_heads, dim, nk),
        *out_rows, _flat(lse, what, "lse", (heads, nq), torch.float32, device),
        table_at, buckets_at, hold.data_ptr() if n else 0, n, stream, *_NO_ROWS, *_NO_ROWS, *_NO_ROWS, *_NO_ROWS, 0,
        code, device, n_buckets, reach, dim ** -0.5 if scale is None else _f32(scale, what, "scale"))
    rc = lib.dptm_attention_forward(block.attention_at)
    if rc:
        _check(rc, what)
    return out, lse


def attention_backward(dout, q, k, v, out, lse, plan: AttentionPlan, *, scale: Optional[float] = None, table=None, buckets=None,
                       dq=None, dk=None, dv=None):
    """Gradients of ``attention``: ``(dq, dk, dv, dtable)`` from the gradient of its ``out``; ``out`` and ``lse`` as it left
    them, ``dtable`` ``None`` without a bias.  ``dq`` / ``dk`` / ``dv`` may be given (views of one packed tensor, say).
    Nothing is added through atomics: equal calls give equal bits."""
    lib, what, dim = _native.load_library(), "attention_backward", plan.head_dim
    code, device = _first(q, what)
    if _forward_ad._current_level >= 0:
        _refuse_tangents(what, dout=dout, q=q, k=k, v=v, out=out, lse=lse, table=table, dq=dq, dk=dk, dv=dv)
    dtype, heads, kv_heads, nq, nk = q.dtype, plan.heads, plan.kv_heads, plan.q_rows, plan.k_rows
    stream = _stream(device)
    host, dev = plan._words(what, device, stream)
    dq, dq_rows = _result(dq, q, what, "dq", device, heads, dim, nq)
    dk, dk_rows = _result(dk, q, what, "dk", device, kv_heads, dim, nk)
    dv, dv_rows = _result(dv, q, what, "dv", device, kv_heads, dim, nk)
    table_at, buckets_at, n_buckets, reach = _bias(what, plan, table, buckets, dtype, device)
    dtable = q.new_empty((n_buckets, heads)) if n_buckets else None
    n = plan._workspace(n_buckets, reach, 1)
    hold = q.new_empty((n // _SIZES[code],)) if n else None
    block = _block
    _ATTENTION.pack_into(
        block.attention, 0, host, dev, *_rows(q, what, "q", dtype, device, heads, dim, nq),
        *_rows(k, what, "k", dtype, device, kv_heads, dim, nk), *_rows(v, what, "v", dtype, device, kv_heads, dim, nk),
        *_rows(out, what, "out", dtype, device, heads, dim, nq), _flat(lse, what, "lse", (heads, nq), torch.float32, device),
        table_at, buckets_at, hold.data_ptr() if n else 0, n, stream,
        *_rows(dout, what, "dout", dtype, device, heads, dim, nq), *dq_rows, *dk_rows, *dv_rows,
        dtable.data_ptr() if n_buckets else 0, code, device, n_buckets, reach, dim ** -0.5 if scale is None else _f32(scale, what, "scale"))
    rc = lib.dptm_attention_backward(block.attention_at)
    if rc:
        _check(rc, what)
    return dq, dk, dv, dtable


def _norm_rope(what: str, q, k, cos, sin, q_gain, k_gain, positions, code, device: int):
    """Sizes and the addresses that both directions share."""
    if not isinstance(k, torch.Tensor) or q.dim() != 3 or k.dim() != 3:
        raise ValueError(f"{what}: q and k must be tensors [rows, heads, head_dim]")
    n, heads, dim = q.shape
    if k.shape[0] != n or k.shape[2] != dim:
        raise ValueError(f"{what}: q {tuple(q.shape)} and k {tuple(k.shape)} differ in rows or head_dim")
    if not isinstance(cos, torch.Tensor) or cos.dim() != 2:
        raise ValueError(f"{what}: cos must be a tensor [positions, head_dim / 2]")
    table, f32 = (cos.shape[0], dim // 2), torch.float32
    return (n, heads, k.shape[1], dim, table[0],
            (_flat(q_gain, what, "q_gain", (dim,), f32, device), _flat(k_gain, what, "k_gain", (dim,), f32, device),
             _flat(cos, what, "cos", table, f32, device), _flat(sin, what, "sin", table, f32, device),
             _flat(positions, what, "positions", (n,), torch.int32, device)))


def qk_norm_rope(q, k, cos, sin, *, q_gain=None, k_gain=None, positions=None, eps: float = 1e-6, interleaved: bool = False,
                 q_out=None, k_out=None):
    """Norm of every head of ``q [rows, heads, head_dim]`` and ``k`` -- ``x / sqrt(mean x^2 + eps) * gain``, left out where the
    gain (float32 ``[head_dim]``) is ``None`` -- and the rotation by position in the same pass: ``(q_out, k_out)``.

    Row ``r`` stands at ``positions[r]`` (int32, default ``r``); ``cos`` / ``sin`` are ``rotary_table``'s.  The pairs ``(i, i +
    head_dim / 2)`` turn together, with ``interleaved`` the pairs ``(2 i, 2 i + 1)``.  A position outside the table makes its
    row NaN.  ``q_out`` / ``k_out`` may be given, also as the inputs themselves."""
    lib, what = _native.load_library(), "qk_norm_rope"
    code, device = _first(q, what)
    if _forward_ad._current_level >= 0:
        _refuse_tangents(what, q=q, k=k, cos=cos, sin=sin, q_gain=q_gain, k_gain=k_gain, q_out=q_out, k_out=k_out)
    dtype = q.dtype
    n, heads, kv_heads, dim, n_pos, shared = _norm_rope(what, q, k, cos, sin, q_gain, k_gain, positions, code, device)
    q_out, q_out_rows = _result(q_out, q, what, "q_out", device, heads, dim, n)
    k_out, k_out_rows = _result(k_out, q, what, "k_out", device, kv_heads, dim, n)
    block = _block
    _NORM_ROPE.pack_into(
        block.norm_rope, 0, *_rows(q, what, "q", dtype, device, heads, dim, n), *_rows(k, what, "k", dtype, device, kv_heads, dim, n),
        *q_out_rows, *k_out_rows, *shared, _stream(device), *_NO_ROWS, *_NO_ROWS, *_NO_ROWS, *_NO_ROWS, 0, 0, 0, 0, n, code, device, dim, heads, kv_heads, n_pos,
        1 if interleaved else 0, _f32(eps, what, "eps"))
    rc = lib.dptm_qk_norm_rope_forward(block.norm_rope_at)
    if rc:
        _check(rc, what)
    return q_out, k_out


def qk_norm_rope_backward(dq_out, dk_out, q, k, cos, sin, *, q_gain=None, k_gain=None, positions=None, eps: float = 1e-6,
                          interleaved: bool = False, dq=None, dk=None):
    """Gradients of ``qk_norm_rope``: ``(dq, dk, dq_gain, dk_gain)``; ``q`` and ``k`` as it read them, a gain's gradient (float32)
    is ``None`` where there is no gain.  ``dq`` / ``dk`` may be given, also as ``dq_out`` / ``dk_out`` or ``q`` / ``k``.  Padding
    rows need a position inside the table too: one outside makes the gains' gradients NaN with its row."""
    lib, what = _native.load_library(), "qk_norm_rope_backward"
    code, device = _first(q, what)
    if _forward_ad._current_level >= 0:
        _refuse_tangents(what, dq_out=dq_out, dk_out=dk_out, q=q, k=k, cos=cos, sin=sin, q_gain=q_gain, k_gain=k_gain, dq=dq, dk=dk)
    dtype = q.dtype
    n, heads, kv_heads, dim, n_pos, shared = _norm_rope(what, q, k, cos, sin, q_gain, k_gain, positions, code, device)
    dq, dq_rows = _result(dq, q, what, "dq", device, heads, dim, n)
    dk, dk_rows = _result(dk, q, what, "dk", device, kv_heads, dim, n)
    dq_gain = None if q_gain is None else cos.new_empty((dim,))
    dk_gain = None if k_gain is None else cos.new_empty((dim,))

    def pack(at, size):
        _NORM_ROPE.pack_into(
            _block.norm_rope, 0, *_rows(q, what, "q", dtype, device, heads, dim, n), *_rows(k, what, "k", dtype, device, kv_heads, dim, n),
            *_NO_ROWS, *_NO_ROWS, *shared, _stream(device),
            *_rows(dq_out, what, "dq_out", dtype, device, heads, dim, n), *_rows(dk_out, what, "dk_out", dtype, device, kv_heads, dim, n),
            *dq_rows, *dk_rows, 0 if dq_gain is None else dq_gain.data_ptr(), 0 if dk_gain is None else dk_gain.data_ptr(), at, size, n, code, device, dim,
            heads, kv_heads, n_pos, 1 if interleaved else 0, _f32(eps, what, "eps"))

    size, hold = 0, None
    if dq_gain is not None or dk_gain is not None:
        key = (n, heads + kv_heads, dim)
        size = _norm_rope_bytes.get(key)
        if size is None:
            pack(0, 0)
            size = _check(lib.dptm_qk_norm_rope_workspace(_block.norm_rope_at), what)
            if len(_norm_rope_bytes) < 4096:
                _norm_rope_bytes[key] = size
        hold = cos.new_empty((size // 4,))
    pack(hold.data_ptr() if size else 0, size)
    rc = lib.dptm_qk_norm_rope_backward(_block.norm_rope_at)
    if rc:
        _check(rc, what)
    return dq, dk, dq_gain, dk_gain


_norm_rope_bytes: dict = {}      # workspace sizes by row count, heads and head_dim
