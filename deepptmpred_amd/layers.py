"""Layer operators on whole proteins: attention over packed sequences with a sliding window, first tokens that stay
visible and a learned bias by relative position, and the per-head norm of queries and keys with the position rotation;
forward, backward, and the form that computes the rows of chosen sites only.

The classifier itself attends within windows of at most 51 residues (pred/train_PTM/model.py:43-85) with a position
table per window (model.py:16-41); these are the same layers for sequences of any length, so that the residue rows a
site is scored from (pred/train_PTM/predict.py:487-501) can be computed and trained on the device and handed to
``Scorer.score_protein_device`` without leaving it.

Tensors are torch tensors on one GPU, ``[rows, heads, head_dim]`` with the rows of all sequences one behind the other; any
strides of rows and heads do, if addresses and strides are multiples of 16 bytes and a head's elements are adjacent.  Types are
float32, bfloat16 and float16.  Calls go out on the current stream of the tensors' GPU and wait for nothing; what they need
besides their results they take from torch's allocator, so calls on several streams and captured graphs do not share
memory.  Gradients are explicit calls, as everywhere in this package: a tensor that requires grad is refused while autograd
records.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Sequence, Tuple

import numpy as np
import torch

from . import _native

_TYPES = {torch.float32: _native.PRECISIONS["f32"], torch.bfloat16: _native.PRECISIONS["bf16"],
          torch.float16: _native.PRECISIONS["f16"]}


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


class _Call:
    """Checks of the tensors of one call, and their C form."""

    def __init__(self, what: str, first: torch.Tensor, dim: int):
        self.what, self.dim = what, dim
        if not isinstance(first, torch.Tensor):
            raise ValueError(f"{what}: expected torch tensors")
        if first.dtype not in _TYPES:
            raise ValueError(f"{what}: dtype {first.dtype} is not float32, bfloat16 or float16")
        if first.device.type != "cuda":
            raise ValueError(f"{what}: tensors must be on a GPU")
        self.dtype, self.device = first.dtype, first.device

    def tensor(self, t, name: str, dtype=None):
        if not isinstance(t, torch.Tensor):
            raise ValueError(f"{self.what}: {name} is not a torch tensor")
        if t.device != self.device:
            raise ValueError(f"{self.what}: {name} is on {t.device}, not on {self.device}")
        if t.dtype != (dtype or self.dtype):
            raise ValueError(f"{self.what}: {name} has dtype {t.dtype}, expected {dtype or self.dtype}")
        if t.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{self.what}: {name} requires grad, and this call does not record; detach it or use no_grad")
        return t

    def rows(self, t, name: str, heads: int, rows: int) -> _native.Rows:
        self.tensor(t, name)
        if t.dim() != 3 or t.shape[1] != heads or t.shape[2] != self.dim:
            raise ValueError(f"{self.what}: {name} has shape {tuple(t.shape)}, expected [rows, {heads}, {self.dim}]")
        if t.shape[0] < rows:
            raise ValueError(f"{self.what}: {name} has {t.shape[0]} rows, the call needs {rows}")
        if t.stride(2) != 1 and t.numel():
            raise ValueError(f"{self.what}: the elements of a head of {name} are not adjacent")
        # the stride of a dimension of one entry says nothing
        head = t.stride(1) if heads > 1 else self.dim
        row = t.stride(0) if t.shape[0] > 1 else heads * self.dim
        return _native.Rows(t.data_ptr(), t.shape[0], row, head)

    def flat(self, t, name: str, shape, dtype) -> Optional[int]:
        if t is None:
            return None
        self.tensor(t, name, dtype)
        if tuple(t.shape) != tuple(shape) or not t.is_contiguous():
            raise ValueError(f"{self.what}: {name} must be contiguous of shape {tuple(shape)}, got {tuple(t.shape)}")
        return t.data_ptr()

    def empty(self, *shape, dtype=None):
        return torch.empty(shape, dtype=dtype or self.dtype, device=self.device)

    def stream(self) -> int:
        return torch.cuda.current_stream(self.device).cuda_stream

    def workspace(self, nbytes: int):
        t = torch.empty(max(0, nbytes), dtype=torch.uint8, device=self.device)
        return t, (t.data_ptr() if nbytes else None)


def _lengths(a, name: str) -> np.ndarray:
    a = np.asarray(a.cpu() if isinstance(a, torch.Tensor) else a)
    if a.size == 0:
        a = a.astype(np.int32)
    if a.ndim != 1 or a.dtype.kind not in "iu":
        raise ValueError(f"AttentionPlan: {name} must be a list of whole numbers")
    if a.size and (int(a.max()) > 2 ** 31 - 1 or int(a.min()) < -2 ** 31):
        raise ValueError(f"AttentionPlan: {name} does not fit 32 bits")
    return np.ascontiguousarray(a, dtype=np.int32)


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
        left, right = window
        d = _native.AttentionDesc(heads, kv_heads if kv_heads is not None else heads, head_dim, max(-1, min(int(left), 2 ** 31 - 1)),
                                  max(-1, min(int(right), 2 ** 31 - 1)), sinks, 1 if training else 0)
        words = np.empty(4096, dtype=np.int32)
        while True:
            n = _check(lib.dptm_attention_plan(C.byref(d), q.ctypes.data, k.ctypes.data, None if pos is None else pos.ctypes.data,
                                               len(q), words.ctypes.data, words.size), "AttentionPlan")
            if n <= words.size:
                break
            words = np.empty(n, dtype=np.int32)
        self.words = words[:n]
        self.heads, self.kv_heads, self.head_dim = d.heads, d.kv_heads, head_dim
        self.q_rows, self.k_rows = int(q.sum(dtype=np.int64)), int(k.sum(dtype=np.int64))
        self.training = bool(training)
        self.device = None if device is None else _device(device)
        self.device_words = None if device is None else torch.from_numpy(self.words).to(self.device)

    def _pair(self, call: _Call):
        if self.device_words is None:
            raise ValueError(f"{call.what}: the plan was made for the host only")
        if self.device != call.device:
            raise ValueError(f"{call.what}: the plan is on {self.device}, the tensors are on {call.device}")
        return self.words.ctypes.data, self.device_words.data_ptr()


def relative_buckets(n_buckets: int, max_distance: int, bidirectional: bool = True, device=0):
    """Bucket of every relative position ``-max_distance .. max_distance`` (``j - p``), int32: half of a side's buckets one
    distance each, the others by the logarithm of the distance up to ``max_distance``; ``bidirectional``: the upper half of
    the buckets for keys behind the query, otherwise those count as distance 0.  Borders are found in whole numbers.
    ``device=None``: a NumPy array."""
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
    if n_positions < 0 or head_dim < 2 or head_dim % 2:
        raise ValueError("rotary_table: bad sizes")
    angle = np.arange(n_positions, dtype=np.float64)[:, None] * float(base) ** (-np.arange(0, head_dim, 2, dtype=np.float64) / head_dim)
    cos, sin = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
    return torch.from_numpy(cos).to(_device(device)), torch.from_numpy(sin).to(_device(device))


def _bias(call: _Call, plan: AttentionPlan, table, buckets):
    if table is None and buckets is None:
        return None
    if table is None or buckets is None:
        raise ValueError(f"{call.what}: table and buckets go together")
    if table.dim() != 2 or table.shape[1] != plan.heads:
        raise ValueError(f"{call.what}: table has shape {tuple(table.shape)}, expected [buckets, {plan.heads}]")
    if buckets.dim() != 1 or buckets.numel() % 2 == 0:
        raise ValueError(f"{call.what}: buckets must hold an odd number of entries, one per distance")
    return _native.AttentionBias(call.flat(table, "table", table.shape, call.dtype), call.flat(buckets, "buckets", buckets.shape, torch.int32),
                                 table.shape[0], buckets.numel() // 2)


def _scale(plan: AttentionPlan, scale: Optional[float]) -> float:
    return plan.head_dim ** -0.5 if scale is None else float(scale)


def attention(q, k, v, plan: AttentionPlan, *, scale: Optional[float] = None, table=None, buckets=None, out=None, lse=None):
    """Softmax attention of ``plan``'s sequences: ``(out [q_rows, heads, head_dim], lse float32 [heads, q_rows])``.

    Scores are ``scale * q.k`` (default ``head_dim ** -0.5``) plus ``table[buckets[j - p], head]`` where a relative position
    bias is given (``relative_buckets``; ``table [buckets, heads]`` of the tensors' type).  A row that sees no key gets zeros and
    ``-inf``.  ``out`` and ``lse`` may be given; rows of ``out`` behind the plan's are left as they are."""
    lib = _native.load_library()
    call = _Call("attention", q, plan.head_dim)
    host, dev = plan._pair(call)
    if out is None:
        out = call.empty(plan.q_rows, plan.heads, plan.head_dim)
    if lse is None:
        lse = call.empty(plan.heads, plan.q_rows, dtype=torch.float32)
    b = _bias(call, plan, table, buckets)
    args = [call.rows(q, "q", plan.heads, plan.q_rows), call.rows(k, "k", plan.kv_heads, plan.k_rows),
            call.rows(v, "v", plan.kv_heads, plan.k_rows), call.rows(out, "out", plan.heads, plan.q_rows)]
    n = _check(lib.dptm_attention_workspace(host, 0, 0), "attention")
    hold, ws = call.workspace(n)
    _check(lib.dptm_attention_forward(host, dev, _TYPES[call.dtype], *[C.byref(x) for x in args],
                                      call.flat(lse, "lse", (plan.heads, plan.q_rows), torch.float32), _scale(plan, scale),
                                      None if b is None else C.byref(b), ws, n, call.device.index, call.stream()), "attention")
    return out, lse


def attention_backward(dout, q, k, v, out, lse, plan: AttentionPlan, *, scale: Optional[float] = None, table=None, buckets=None,
                       dq=None, dk=None, dv=None):
    """Gradients of ``attention``: ``(dq, dk, dv, dtable)`` from the gradient of its ``out``; ``out`` and ``lse`` as it left
    them, ``dtable`` ``None`` without a bias.  ``dq`` / ``dk`` / ``dv`` may be given (views of one packed tensor, say).
    Nothing is added through atomics: equal calls give equal bits."""
    lib = _native.load_library()
    call = _Call("attention_backward", q, plan.head_dim)
    host, dev = plan._pair(call)
    if dq is None:
        dq = call.empty(plan.q_rows, plan.heads, plan.head_dim)
    if dk is None:
        dk = call.empty(plan.k_rows, plan.kv_heads, plan.head_dim)
    if dv is None:
        dv = call.empty(plan.k_rows, plan.kv_heads, plan.head_dim)
    b = _bias(call, plan, table, buckets)
    dtable = None if b is None else call.empty(*table.shape)

    def rq(t, name):
        return call.rows(t, name, plan.heads, plan.q_rows)

    def rk(t, name):
        return call.rows(t, name, plan.kv_heads, plan.k_rows)

    ins = [rq(dout, "dout"), rq(q, "q"), rk(k, "k"), rk(v, "v"), rq(out, "out")]
    outs = [rq(dq, "dq"), rk(dk, "dk"), rk(dv, "dv")]
    n = _check(lib.dptm_attention_workspace(host, 0 if b is None else b.n_buckets, 1), "attention_backward")
    hold, ws = call.workspace(n)
    _check(lib.dptm_attention_backward(host, dev, _TYPES[call.dtype], *[C.byref(x) for x in ins],
                                       call.flat(lse, "lse", (plan.heads, plan.q_rows), torch.float32), _scale(plan, scale),
                                       None if b is None else C.byref(b), *[C.byref(x) for x in outs],
                                       None if dtable is None else dtable.data_ptr(), ws, n, call.device.index, call.stream()),
           "attention_backward")
    return dq, dk, dv, dtable


def _norm_rope(what: str, q, k, cos, sin, q_gain, k_gain, positions, eps, interleaved):
    if not isinstance(q, torch.Tensor) or not isinstance(k, torch.Tensor) or q.dim() != 3 or k.dim() != 3:
        raise ValueError(f"{what}: q and k must be tensors [rows, heads, head_dim]")
    if q.shape[0] != k.shape[0] or q.shape[2] != k.shape[2]:
        raise ValueError(f"{what}: q {tuple(q.shape)} and k {tuple(k.shape)} differ in rows or head_dim")
    call = _Call(what, q, q.shape[2])
    n = q.shape[0]
    if not isinstance(cos, torch.Tensor) or cos.dim() != 2:
        raise ValueError(f"{what}: cos must be a tensor [positions, head_dim / 2]")
    table = (cos.shape[0], call.dim // 2)
    d = _native.NormRopeDesc(_TYPES[call.dtype], call.dim, q.shape[1], k.shape[1], n, table[0], 1 if interleaved else 0, eps)
    shared = [call.flat(q_gain, "q_gain", (call.dim,), torch.float32), call.flat(k_gain, "k_gain", (call.dim,), torch.float32),
              call.flat(cos, "cos", table, torch.float32), call.flat(sin, "sin", table, torch.float32),
              call.flat(positions, "positions", (n,), torch.int32)]
    return call, d, shared


def qk_norm_rope(q, k, cos, sin, *, q_gain=None, k_gain=None, positions=None, eps: float = 1e-6, interleaved: bool = False,
                 q_out=None, k_out=None):
    """Norm of every head of ``q [rows, heads, head_dim]`` and ``k`` -- ``x / sqrt(mean x^2 + eps) * gain``, left out where the
    gain (float32 ``[head_dim]``) is ``None`` -- and the rotation by position in the same pass: ``(q_out, k_out)``.

    Row ``r`` stands at ``positions[r]`` (int32, default ``r``); ``cos`` / ``sin`` are ``rotary_table``'s.  The pairs ``(i, i +
    head_dim / 2)`` turn together, with ``interleaved`` the pairs ``(2 i, 2 i + 1)``.  A position outside the table makes its
    row NaN.  ``q_out`` / ``k_out`` may be given, also as the inputs themselves."""
    lib = _native.load_library()
    call, d, shared = _norm_rope("qk_norm_rope", q, k, cos, sin, q_gain, k_gain, positions, eps, interleaved)
    q_out = call.empty(*q.shape) if q_out is None else q_out
    k_out = call.empty(*k.shape) if k_out is None else k_out
    ins = [call.rows(q, "q", d.heads, d.rows), call.rows(k, "k", d.kv_heads, d.rows)]
    outs = [call.rows(q_out, "q_out", d.heads, d.rows), call.rows(k_out, "k_out", d.kv_heads, d.rows)]
    _check(lib.dptm_qk_norm_rope_forward(C.byref(d), *[C.byref(x) for x in ins], *shared, *[C.byref(x) for x in outs],
                                         call.device.index, call.stream()), "qk_norm_rope")
    return q_out, k_out


def qk_norm_rope_backward(dq_out, dk_out, q, k, cos, sin, *, q_gain=None, k_gain=None, positions=None, eps: float = 1e-6,
                          interleaved: bool = False, dq=None, dk=None):
    """Gradients of ``qk_norm_rope``: ``(dq, dk, dq_gain, dk_gain)``; ``q`` and ``k`` as it read them, a gain's gradient (float32)
    is ``None`` where there is no gain.  ``dq`` / ``dk`` may be given, also as ``dq_out`` / ``dk_out``."""
    lib = _native.load_library()
    call, d, shared = _norm_rope("qk_norm_rope_backward", q, k, cos, sin, q_gain, k_gain, positions, eps, interleaved)
    dq = call.empty(*q.shape) if dq is None else dq
    dk = call.empty(*k.shape) if dk is None else dk
    ins = [call.rows(dq_out, "dq_out", d.heads, d.rows), call.rows(dk_out, "dk_out", d.kv_heads, d.rows),
           call.rows(q, "q", d.heads, d.rows), call.rows(k, "k", d.kv_heads, d.rows)]
    outs = [call.rows(dq, "dq", d.heads, d.rows), call.rows(dk, "dk", d.kv_heads, d.rows)]
    dq_gain = None if q_gain is None else call.empty(call.dim, dtype=torch.float32)
    dk_gain = None if k_gain is None else call.empty(call.dim, dtype=torch.float32)
    n = _check(lib.dptm_qk_norm_rope_workspace(C.byref(d)), "qk_norm_rope_backward") if q_gain is not None or k_gain is not None else 0
    hold, ws = call.workspace(n)
    _check(lib.dptm_qk_norm_rope_backward(C.byref(d), *[C.byref(x) for x in ins], *shared, *[C.byref(x) for x in outs],
                                          None if dq_gain is None else dq_gain.data_ptr(), None if dk_gain is None else dk_gain.data_ptr(),
                                          ws, n, call.device.index, call.stream()), "qk_norm_rope_backward")
    return dq, dk, dq_gain, dk_gain
