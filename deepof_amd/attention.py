"""Sequence operators on packed recordings: what a transformer over whole recordings needs next to the windowed family.

The transformer family (/root/reference/deepof/clustering/models_new.py:832-1327) attends inside one window, in fp32, with
sinusoidal positions added to its input.  These operators take the same mathematics to recordings of any length: ``norm_rope``
(RMS norm of every query / key head and rotation by its position, one pass), ``attention`` (packed documents, grouped heads,
causal / prefix masks, tanh cap, distance bias) -- both with their backward pass -- and ``attention_step``, which takes the new
frames of live streams against a paged key / value cache.  Elements are float32, bfloat16 or float16; sums, norms and softmax
statistics are fp32.

Gradients are explicit: every ``*_backward`` takes the gradients at the outputs and returns those at the inputs; autograd does not
record these calls.  Tensors of the caller that a call writes to are marked as changed, as torch's own in-place operations mark them.

``AttentionOps`` issues the C-ABI calls (include/deepof_hip.h) on the current HIP stream of its device; product code obtains it
through :func:`create_attention_ops`, which requires a ROCm device and the compiled library and raises otherwise.  Workspaces and
outputs come from torch's allocator, one per call, so calls on different streams and captured graphs never share memory.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Sequence

import numpy as np
import torch
from torch.autograd.graph import increment_version

from . import _capi

DTYPES = {torch.float32: _capi.DTYPE_F32, torch.bfloat16: _capi.DTYPE_BF16, torch.float16: _capi.DTYPE_F16}


def rotary_frequencies(rot_dim: int, base: float = 10000.0, scale: float = 1.0, original_length: Optional[float] = None,
                       low_turns: float = 1.0, high_turns: float = 32.0, device=None) -> torch.Tensor:
    """Angles per position of the ``rot_dim / 2`` pairs, float64: ``base ** (-2 i / rot_dim)``.

    ``scale`` > 1 stretches the positions for recordings that many times longer than those trained on.  Without
    ``original_length`` every frequency is divided by it.  With it, only the slow pairs are: a pair that turns fewer than
    ``low_turns`` times over ``original_length`` positions is divided by ``scale``, one that turns more than ``high_turns`` times
    stays, and between the two the divisor's reciprocal runs linearly with the number of turns."""
    if rot_dim < 2 or rot_dim % 2:
        raise ValueError(f"rot_dim must be an even number from 2, got {rot_dim}")
    if not (base > 0.0 and scale > 0.0):
        raise ValueError("base and scale must be positive")
    f = float(base) ** (-torch.arange(rot_dim // 2, dtype=torch.float64) / (rot_dim // 2))
    if scale != 1.0:
        if original_length is None:
            f = f / scale
        else:
            if not 0.0 <= low_turns < high_turns:
                raise ValueError("need 0 <= low_turns < high_turns")
            turns = f * (original_length / (2.0 * np.pi))
            keep = ((turns - low_turns) / (high_turns - low_turns)).clamp(0.0, 1.0)
            f = f * (keep + (1.0 - keep) / scale)
    return f.to(device) if device is not None else f


def _rows(name: str, t: torch.Tensor, device, dtype=None, ndim: int = 3):
    """A (..., heads, head_dim) tensor whose heads are runs of memory; raises otherwise."""
    if not isinstance(t, torch.Tensor) or t.dim() != ndim:
        raise ValueError(f"{name} must be a tensor of {ndim} dimensions")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, these operators are on {device}")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{name} has dtype {t.dtype}, expected {dtype}")
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"the elements of a head of {name} must lie side by side (stride 1 in the last dimension)")
    return t


def _writable(name: str, t: torch.Tensor):
    """An output may not address one element twice (an expanded view)."""
    for n, s in zip(t.shape, t.stride()):
        if n > 1 and s == 0:
            raise ValueError(f"{name} is an expanded view; its elements must be distinct")
    return t


def _changed(*tensors: Optional[torch.Tensor]):
    """The caller's tensors that the call writes to: autograd then refuses a backward pass which needs what they held."""
    for t in tensors:
        if t is not None:
            increment_version(t)


def _vector(name: str, t: Optional[torch.Tensor], n: int, dtype, device):
    if t is None:
        return 0
    if t.shape != (n,) or t.dtype != dtype or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of {n} elements on {device}")
    return t.data_ptr()


def _st(t: torch.Tensor):
    """The strides but the last (which is 1): row and head, or stream, frame and head."""
    return t.stride()[:-1]


def _ptr(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _is_wide(t: torch.Tensor) -> bool:
    """Address and strides are multiples of 16 bytes (what the attention kernels load at once)."""
    e = t.element_size()
    bits = t.data_ptr()
    for s in t.stride()[:-1]:
        bits |= s * e
    return not bits & 15


def _apart(name: str, out: Optional[torch.Tensor], /, **inputs):
    """An output the caller gave may not share a byte with an input: other workgroups still read it.  Both may be slices of one
    buffer in any order (a packed q | k | v, heads side by side)."""
    if not isinstance(out, torch.Tensor):
        return
    for other, t in inputs.items():
        if isinstance(t, torch.Tensor) and _share(out, t):
            raise ValueError(f"{name} must not share memory with {other}")


def _share(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Do two tensors have a byte in common?  Exact for slices of one buffer; tensors whose strides have so little to do with
    each other that the search grows long count as sharing."""
    apart = b.data_ptr() - a.data_ptr()
    if apart < 0:
        a, b, apart = b, a, -apart
    if a.is_contiguous() and apart >= a.nbytes or a.numel() == 0 or b.numel() == 0:
        return False
    a, b = (t if t.dim() else t.reshape(1) for t in (a, b))
    ea, eb, sa, sb = a.element_size(), b.element_size(), a.stride(), b.stride()
    inner_a, inner_b = ea, eb  # bytes from the first to the last of one row
    for n, s in zip(a.shape[1:], sa[1:]):
        inner_a += (n - 1) * s * ea
    for n, s in zip(b.shape[1:], sb[1:]):
        inner_b += (n - 1) * s * eb
    if apart >= inner_a + (a.shape[0] - 1) * sa[0] * ea:
        return False
    pitch = sa[0] * ea
    if pitch == sb[0] * eb and pitch and inner_a <= apart % pitch <= pitch - inner_b:
        return False  # side by side in rows of one buffer
    # is `apart` a sum of i * stride over a's dimensions, less one over b's, plus the place of a byte in either's element?
    range_of = {1: [1 - eb, ea - 1]}
    for t, st, e, sign in ((a, sa, ea, 0), (b, sb, eb, 1)):
        for n, s in zip(t.shape, st):
            if n > 1 and s > 0:
                r = range_of.setdefault(s * e, [0, 0])
                r[1 - sign] += (1 - 2 * sign) * (n - 1)
    dims = sorted(((s, lo, hi) for s, (lo, hi) in range_of.items()), reverse=True)
    reach = [(0, 0)]  # what the dimensions from the k-th on can add up to
    for s, lo, hi in reversed(dims):
        reach.insert(0, (reach[0][0] + s * lo, reach[0][1] + s * hi))
    left = [10000]

    def found(k, want):
        if k == len(dims):
            return want == 0
        left[0] -= 1
        if left[0] < 0:
            return True
        (s, lo, hi), (least, most) = dims[k], reach[k + 1]
        return any(found(k + 1, want - i * s) for i in range(max(lo, -((most - want) // s)), min(hi, (want - least) // s) + 1))

    return found(0, apart)


def _wide(t: torch.Tensor) -> torch.Tensor:
    """The tensor itself, or a contiguous copy of one whose memory the kernels' 16-byte loads do not fit."""
    return t if _is_wide(t) else t.clone(memory_format=torch.contiguous_format)


class AttentionPlan:
    """The tiles of one packed batch on the device (:meth:`AttentionOps.attention_plan`): serves any number of heads, head sizes,
    dtypes and streams, forward and backward; never written after it is made.  It may be dropped while calls that use it still
    run; a captured graph reads it at every replay, so keep it as long as the graph."""

    def __init__(self, ops: "AttentionOps", q_lengths, k_lengths, causal, prefix):
        ql = self._host("q_lengths", q_lengths)
        kl = ql if k_lengths is None else self._host("k_lengths", k_lengths)
        if len(kl) != len(ql):
            raise ValueError(f"{len(ql)} query lengths and {len(kl)} key lengths")
        if prefix is not None and not causal:
            raise ValueError("a prefix is part of a causal mask: pass causal=True")
        pre = None
        if prefix is not None:
            pre = self._host("prefix", prefix)
            if len(pre) != len(ql):
                raise ValueError(f"{len(ql)} documents and {len(pre)} prefixes")
            pre = np.minimum(pre, 2 ** 31 - 1).astype(np.int32)
        q_off, k_off = (np.concatenate(([0], np.cumsum(x))).astype(np.int64) for x in (ql, kl))
        self.device, self.causal, self.n_docs = ops.device, bool(causal), len(ql)
        self.q_rows, self.k_rows = int(q_off[-1]), int(k_off[-1])
        self.record = _capi.AttnPlan()
        _capi.check(ops.lib, ops.lib.dof_attn_plan_size(len(ql), q_off.ctypes.data, k_off.ctypes.data, int(self.causal),
                                                        C.byref(self.record)), "dof_attn_plan_size")
        host = torch.empty(max(16, self.record.table_bytes), dtype=torch.uint8)
        _capi.check(ops.lib, ops.lib.dof_attn_plan_table(C.byref(self.record), q_off.ctypes.data, k_off.ctypes.data,
                                                         pre.ctypes.data if pre is not None else 0, host.data_ptr()),
                    "dof_attn_plan_table")
        self.table = host.to(self.device)

    @staticmethod
    def _host(name, lengths):
        if isinstance(lengths, torch.Tensor) and lengths.is_cuda:
            raise ValueError(f"{name} must be host data: the plan is made on the host")
        a = np.asarray(lengths)
        if a.ndim != 1 or (a.size and a.dtype.kind not in "iu"):
            raise ValueError(f"{name} must be a sequence of whole numbers")
        a = a.astype(np.int64)
        if a.size and a.min() < 0:
            raise ValueError(f"{name} must not be negative")
        return a


class AttentionOps:
    """The operators on one device.  Holds no state between calls; safe to share between streams and captured graphs."""

    def __init__(self, lib, device):
        self.lib = lib
        self.device = torch.device(device)
        if self.device.type == "cuda" and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())

    def _launch(self, name: str, *args, plan: Optional[AttentionPlan] = None):
        """The entry point on the current stream of this object's device; launches go to the current device, so another one is made
        current for the call.  The allocator is told that the plan's tiles are read there, so that a plan which is dropped gives its
        memory back only behind the call, also where another stream made it."""
        fn = getattr(self.lib, name)
        if self.device.type != "cuda":
            rc = fn(*args, 0)
        else:
            stream = torch.cuda.current_stream(self.device)
            if plan is not None:
                plan.table.record_stream(stream)
            if torch.cuda.current_device() == self.device.index:
                rc = fn(*args, stream.cuda_stream)
            else:
                with torch.cuda.device(self.device):
                    rc = fn(*args, stream.cuda_stream)
        if rc:
            _capi.check(self.lib, rc, name)

    def _dtype(self, name, t):
        if not isinstance(t, torch.Tensor) or t.dtype not in DTYPES:
            raise ValueError(f"{name} must be a float32, bfloat16 or float16 tensor")
        return t.dtype

    def _output(self, name, t, like):
        """The caller's output, or a new contiguous one of ``like``'s shape and dtype."""
        if t is None:
            return like.new_empty(like.shape)
        _rows(name, t, self.device, like.dtype, like.dim())
        if t.shape != like.shape:
            raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(like.shape)}")
        return _writable(name, t)

    # ---- norm + rotation ------------------------------------------------------------------------------------------
    def _norm_rope_args(self, q, k, positions, freqs, q_weight, k_weight, eps, interleaved):
        """The checked head of the record and the addresses of positions, freqs and weights."""
        dt = self._dtype("q", q)
        _rows("q", q, self.device, dt)
        _rows("k", k, self.device, dt)
        rows, hq, dim = q.shape
        if k.shape[0] != rows or k.shape[2] != dim:
            raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)} must have the same rows and head size")
        if not isinstance(freqs, torch.Tensor) or freqs.dim() != 1:
            raise ValueError("freqs must be a tensor of one angle per rotated pair")
        pairs = freqs.shape[0]
        if 2 * pairs > dim:
            raise ValueError(f"{pairs} rotated pairs do not fit a head of {dim}")
        if not eps >= 0.0:
            raise ValueError("eps must not be negative")
        head = (DTYPES[dt], dim, 2 * pairs, 1 if interleaved else 0, hq, k.shape[1], rows, eps, 0)
        return head, (_vector("positions", positions, rows, torch.int32, self.device),
                      _vector("freqs", freqs, pairs, torch.float64, self.device),
                      _vector("q_weight", q_weight, dim, torch.float32, self.device),
                      _vector("k_weight", k_weight, dim, torch.float32, self.device))

    def norm_rope(self, q, k, positions, freqs, q_weight=None, k_weight=None, eps: float = 1e-6, interleaved: bool = False,
                  q_out=None, k_out=None):
        """-> (q', k').  q (rows, query heads, head_dim) and k (rows, key heads, head_dim): every head divided by its root mean
        square and multiplied by ``q_weight`` / ``k_weight`` (fp32, None: no norm), then its first ``2 len(freqs)`` elements
        rotated by ``positions[row] * freqs[pair]`` (positions int32; freqs float64, see :func:`rotary_frequencies`).
        ``interleaved``: neighbouring elements are a pair; otherwise the pairs lie half the rotated part apart.  head_dim: even, up
        to 256.  ``q_out`` / ``k_out`` may be q / k themselves."""
        head, ptrs = self._norm_rope_args(q, k, positions, freqs, q_weight, k_weight, eps, interleaved)
        _apart("q_out", q_out, k=k)
        _apart("k_out", k_out, q=q)
        for name, out, x in (("q_out", q_out, q), ("k_out", k_out, k)):
            if out is not None and (out.data_ptr() != x.data_ptr() or out.stride() != x.stride()):
                _apart(name, out, **{name[0]: x})
        if q_out is not None and k_out is not None:
            _apart("q_out", q_out, k_out=k_out)
        given = q_out, k_out
        q_out = self._output("q_out", q_out, q)
        k_out = self._output("k_out", k_out, k)
        _changed(*given)
        rec = _capi.PACK_NORM_ROPE.pack(*head, *_st(q), *_st(k), *_st(q_out), *_st(k_out), 0, 0, 0, 0)
        self._launch("dof_norm_rope_forward", rec, q.data_ptr(), k.data_ptr(), *ptrs, q_out.data_ptr(), k_out.data_ptr())
        return q_out, k_out

    def norm_rope_backward(self, dq_out, dk_out, q, k, positions, freqs, q_weight=None, k_weight=None, eps: float = 1e-6,
                           interleaved: bool = False):
        """-> (dq, dk, dq_weight, dk_weight) from the gradients at :meth:`norm_rope`'s outputs and its inputs (the weight gradients
        are None without a weight; they are the same bits on every run)."""
        head, ptrs = self._norm_rope_args(q, k, positions, freqs, q_weight, k_weight, eps, interleaved)
        for name, g, x in (("dq_out", dq_out, q), ("dk_out", dk_out, k)):
            _rows(name, g, self.device, q.dtype)
            if g.shape != x.shape:
                raise ValueError(f"{name} has shape {tuple(g.shape)}, expected {tuple(x.shape)}")
        dq, dk = q.new_empty(q.shape), k.new_empty(k.shape)
        dwq = None if q_weight is None else torch.empty_like(q_weight)
        dwk = None if k_weight is None else torch.empty_like(k_weight)
        rec = _capi.PACK_NORM_ROPE.pack(*head, *_st(q), *_st(k), *_st(dq), *_st(dk), *_st(dq_out), *_st(dk_out))
        ws = None
        if dwq is not None or dwk is not None:
            ws = torch.empty(self._bytes("dof_norm_rope_workspace_bytes", rec), dtype=torch.uint8, device=self.device)
        self._launch("dof_norm_rope_backward", rec, dq_out.data_ptr(), dk_out.data_ptr(), q.data_ptr(), k.data_ptr(), *ptrs,
                     dq.data_ptr(), dk.data_ptr(), _ptr(dwq), _ptr(dwk), _ptr(ws))
        return dq, dk, dwq, dwk

    # ---- attention over packed documents ----------------------------------------------------------------------------
    def attention_plan(self, q_lengths: Sequence[int], k_lengths: Optional[Sequence[int]] = None, causal: bool = False,
                       prefix: Optional[Sequence[int]] = None) -> "AttentionPlan":
        """The packing of a batch: document d has ``q_lengths[d]`` query rows and ``k_lengths[d]`` key rows (default: the same),
        one behind the other in the tensors.  ``causal``: the last query row stands at the last key, every row sees the keys up to
        its own; ``prefix``: the first ``prefix[d]`` keys of a document are visible to all its rows besides.  Lengths are host
        data (lists, arrays, CPU tensors).  Build it once per batch, before any capture, and use it for every layer, forward and backward."""
        return AttentionPlan(self, q_lengths, k_lengths, causal, prefix)

    def _attention_args(self, plan, q, k, v, scale, cap, slopes):
        if not isinstance(plan, AttentionPlan) or plan.device != self.device:
            raise ValueError("plan must come from attention_plan() of these operators")
        dt = self._dtype("q", q)
        _rows("q", q, self.device, dt)
        _rows("k", k, self.device, dt)
        _rows("v", v, self.device, dt)
        if k.shape != v.shape or q.shape[2] != k.shape[2]:
            raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}: k and v must have one shape and q's head size")
        if q.shape[0] < plan.q_rows or k.shape[0] < plan.k_rows:
            raise ValueError(f"the plan covers {plan.q_rows} query and {plan.k_rows} key rows, the tensors have {q.shape[0]} and {k.shape[0]}")
        if k.shape[1] < 1 or q.shape[1] % k.shape[1] or q.shape[1] < 1:
            raise ValueError(f"{q.shape[1]} query heads are not a multiple of {k.shape[1]} key heads")
        head = (DTYPES[dt], q.shape[2], q.shape[1], k.shape[1], q.shape[2] ** -0.5 if scale is None else scale, cap)
        return head, _vector("slopes", slopes, q.shape[1], torch.float32, self.device)

    def _lse(self, lse, q):
        if not isinstance(lse, torch.Tensor) or lse.shape != q.shape[:2] or lse.dtype != torch.float32 or lse.device != self.device \
                or not lse.is_contiguous():
            raise ValueError(f"lse must be a contiguous float32 tensor of shape {tuple(q.shape[:2])} on {self.device}")
        return lse

    def attention(self, plan, q, k, v, scale: Optional[float] = None, cap: float = 0.0, slopes=None, out=None, lse=None):
        """-> (o, lse).  q (rows, query heads, head_dim), k and v (rows, key heads, head_dim); query head h reads key head
        ``h // (query heads / key heads)``.  Scores ``scale q.k`` (default ``head_dim ** -0.5``), ``cap``: ``cap tanh(score / cap)``,
        ``slopes`` (fp32 per query head): minus ``slope * distance``.  lse (rows, query heads), fp32, natural log.  A row that sees no
        key gives zeros and -inf.  Rows behind the last document are left as they were in ``out`` / ``lse`` and are zeros in tensors
        allocated here.  ``out`` and ``lse`` may not lie in q, k, v or each other.  head_dim: a multiple of 8 up to 128."""
        head, sl = self._attention_args(plan, q, k, v, scale, cap, slopes)
        _apart("out", out, q=q, k=k, v=v)
        tail, given = q.shape[0] > plan.q_rows, (out, lse)
        if out is None and tail:
            out = q.new_zeros(q.shape)
        o = self._output("out", out, q)
        if lse is None:
            lse = (torch.zeros if tail else torch.empty)(q.shape[:2], dtype=torch.float32, device=self.device)
        else:
            _apart("lse", lse, q=q, k=k, v=v, out=out)
        self._lse(lse, q)
        _changed(*given)
        q, k, v = _wide(q), _wide(k), _wide(v)
        ow = o if _is_wide(o) else o.clone(memory_format=torch.contiguous_format)
        rec = _capi.PACK_ATTENTION.pack(*head, *_st(q), *_st(k), *_st(v), *_st(ow), 0, 0, 0, 0, 0, 0, 0, 0)
        self._launch("dof_attention_forward", C.byref(plan.record), plan.table.data_ptr(), rec, q.data_ptr(), k.data_ptr(), v.data_ptr(),
                     sl, ow.data_ptr(), lse.data_ptr(), plan=plan)
        if ow is not o:
            o.copy_(ow)
        return o, lse

    def attention_backward(self, plan, do, q, k, v, o, lse, scale: Optional[float] = None, cap: float = 0.0, slopes=None):
        """-> (dq, dk, dv) from the gradient at ``o`` and the forward's inputs and results; zeros in rows of no document.  The same
        bits on every run.  ``slopes`` are constants: they get no gradient.  float16: the scores' gradients are carried with a power
        of two of their own, so that gradients of any size keep their precision; dq, dk and dv themselves are float16 numbers.  What a
        document's rows hold must be finite: an infinity or NaN of q, k, v or do reaches gradients of that document's other rows, those
        that do not see it among them (other documents' it does not reach)."""
        head, sl = self._attention_args(plan, q, k, v, scale, cap, slopes)
        for name, t in (("do", do), ("o", o)):
            _rows(name, t, self.device, q.dtype)
            if t.shape != q.shape:
                raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(q.shape)}")
        self._lse(lse, q)
        dq = q.new_zeros(q.shape) if q.shape[0] > plan.q_rows else q.new_empty(q.shape)
        new_k = k.new_zeros if k.shape[0] > plan.k_rows else k.new_empty
        dk, dv = new_k(k.shape), new_k(k.shape)
        q, k, v, do, o = _wide(q), _wide(k), _wide(v), _wide(do), _wide(o)
        rec = _capi.PACK_ATTENTION.pack(*head, *_st(q), *_st(k), *_st(v), *_st(o), *_st(do), *_st(dq), *_st(dk), *_st(dv))
        need = self._bytes("dof_attention_workspace_bytes", C.byref(plan.record), rec)
        ws = torch.empty(need, dtype=torch.uint8, device=self.device) if need else None
        self._launch("dof_attention_backward", C.byref(plan.record), plan.table.data_ptr(), rec, do.data_ptr(), q.data_ptr(), k.data_ptr(),
                     v.data_ptr(), sl, o.data_ptr(), lse.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), _ptr(ws), plan=plan)
        return dq, dk, dv

    # ---- the new frames of live streams ------------------------------------------------------------------------------
    def attention_step(self, q, k, v, k_cache, v_cache, page_table, lengths, scale: Optional[float] = None, cap: float = 0.0,
                       slopes=None, out=None):
        """-> o (streams, new, query heads, head_dim).  q (streams, new, query heads, head_dim), k and v (streams, new, key heads,
        head_dim): 1 to 16 new frames of every stream.  They are stored in ``k_cache`` / ``v_cache`` (pages, page size, key heads,
        head_dim) behind the ``lengths`` (streams, int32) frames already there, on the pages that ``page_table`` (streams, pages,
        int32) lists for the stream, and attend to everything up to themselves; the caller advances ``lengths``.  ``scale``, ``cap``
        and ``slopes`` as in :meth:`attention`.

        Streams may share pages that are full.  A negative length marks an idle stream: nothing of it is read or written (its rows
        of ``out`` stay; allocated here they are undefined).  Frames behind the table's last page and frames on a page index that the
        cache does not have are neither stored nor seen."""
        dt = self._dtype("q", q)
        _rows("q", q, self.device, dt, 4)
        _rows("k", k, self.device, dt, 4)
        _rows("v", v, self.device, dt, 4)
        _writable("k_cache", _rows("k_cache", k_cache, self.device, dt, 4))
        _writable("v_cache", _rows("v_cache", v_cache, self.device, dt, 4))
        b, new, hq, dim = q.shape
        hk = k.shape[2]
        if k.shape != v.shape or k.shape[:2] != q.shape[:2] or k.shape[3] != dim:
            raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)} do not go together")
        if k_cache.shape != v_cache.shape or k_cache.shape[2:] != (hk, dim):
            raise ValueError(f"caches {tuple(k_cache.shape)} / {tuple(v_cache.shape)} must be (pages, page size, {hk}, {dim})")
        if hk < 1 or hq % hk or hq < 1:
            raise ValueError(f"{hq} query heads are not a multiple of {hk} key heads")
        _apart("out", out, q=q, k=k, v=v, k_cache=k_cache, v_cache=v_cache)
        if _share(k_cache, v_cache):
            raise ValueError("k_cache and v_cache must be two tensors that share no memory")
        if not (_is_wide(k_cache) and _is_wide(v_cache)):
            raise ValueError("the caches' address and strides must be multiples of 16 bytes")
        if page_table.dim() != 2 or page_table.shape[0] != b or page_table.dtype != torch.int32 or page_table.device != self.device \
                or not page_table.is_contiguous():
            raise ValueError(f"page_table must be a contiguous int32 tensor ({b}, pages of a stream) on {self.device}")
        ln = _vector("lengths", lengths, b, torch.int32, self.device)
        sl = _vector("slopes", slopes, hq, torch.float32, self.device)
        o = self._output("out", out, q)
        _changed(k_cache, v_cache, out)
        ow = o if _is_wide(o) else o.clone(memory_format=torch.contiguous_format)
        q, k, v = _wide(q), _wide(k), _wide(v)
        rec = _capi.PACK_ATTN_STEP.pack(DTYPES[dt], dim, hq, hk, b, new, k_cache.shape[0], k_cache.shape[1], page_table.shape[1], 0,
                                        dim ** -0.5 if scale is None else scale, cap, *_st(q), *_st(k), *_st(v), *_st(ow),
                                        *_st(k_cache), *_st(v_cache))
        need = self._bytes("dof_attention_step_workspace_bytes", rec)
        ws = torch.empty(need, dtype=torch.uint8, device=self.device) if need else None
        self._launch("dof_attention_step", rec, q.data_ptr(), k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
                     page_table.data_ptr(), ln, sl, ow.data_ptr(), _ptr(ws))
        if ow is not o:
            o.copy_(ow)
        return o

    def _bytes(self, fn: str, *args) -> int:
        n = getattr(self.lib, fn)(*args)
        if n < 0:
            _capi.check(self.lib, n, fn)
        return n


def create_attention_ops(device=None) -> AttentionOps:
    """Product entry: requires a ROCm GPU and the compiled HIP library (no fallback)."""
    from ._lib import load_hip_library

    if not torch.cuda.is_available():
        raise RuntimeError("deepof_amd needs a ROCm GPU (torch.cuda.is_available() is False); there is no CPU path")
    lib = load_hip_library()
    dev = torch.device(device if device is not None else f"cuda:{torch.cuda.current_device()}")
    if dev.type != "cuda":
        raise RuntimeError(f"deepof_amd runs on ROCm devices only, got {dev}")
    return AttentionOps(lib, dev)
