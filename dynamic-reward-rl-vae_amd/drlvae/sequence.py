"""The sequence operators on torch tensors: attention, linear attention with a decaying state, group normalisation
(include/drlvae.h, "sequence operators over packed series").

WindowScorer inherits SequenceOps.  Unlike the scoring calls, which run on the scorer's stream, these run on torch's
current stream of the scorer's GPU, as torch's own operators do: their results and workspaces are torch allocations, so
they are ordered with what torch does before and after, also inside a captured graph.  They are forward only.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Sequence

import numpy as np

from . import _abi

_ACTS = {"linear": 0, "relu": 1, "sigmoid": 2, "silu": 3}
_torch = None
_dtypes = {}


_stream = None
_fw = None


def _t():
    global _torch, _stream, _fw
    if _torch is None:
        import torch
        import torch.autograd.forward_ad as _fw
        _dtypes.update({torch.float32: 0, torch.float16: 1, torch.bfloat16: 2})
        _stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda d: torch.cuda.current_stream(d).cuda_stream)
        _torch = torch
    return _torch


def _number(name, x):
    """x as what a float32 argument can hold."""
    if not -3.4e38 < x < 3.4e38:
        raise ValueError(f"{name} {x} is not a float32 number")
    return x


def _scale(scale, dim):
    return _number("scale", scale) if scale is not None else dim ** -0.5 if dim else 1.0


def _whole(offsets):
    a = np.asarray(offsets)
    if a.dtype.kind != "i":
        try:
            with np.errstate(invalid="ignore"):
                whole = a.astype(np.int64)
        except (OverflowError, TypeError, ValueError):
            whole = None
        if whole is None or not np.array_equal(whole, a):        # a fraction would be cut off without a word
            raise ValueError(f"offsets are whole numbers of 64 bits, not {offsets!r:.200}")
        a = whole
    return np.ascontiguousarray(a, dtype=np.int64)


class SeqLayout:
    """Which rows of packed tensors belong to which series: made once per batch layout with ``WindowScorer.seq_layout``
    and kept by the caller for as long as calls, or captured graphs, use it."""

    def __init__(self, scorer, q_offsets: Sequence[int], k_offsets: Optional[Sequence[int]] = None):
        q = _whole(q_offsets)
        k = q if k_offsets is None else _whole(k_offsets)
        if q.ndim != 1 or k.ndim != 1 or len(q) < 1 or len(q) != len(k):
            raise ValueError("offsets are one-dimensional, n_seg + 1 entries, as many for k as for q")
        self._lib, self._h = scorer._lib, None
        p64 = C.POINTER(C.c_int64)
        h = C.c_void_p()
        scorer._check(self._lib.drl_seq_layout_create(scorer._h, q.ctypes.data_as(p64), None if k_offsets is None else k.ctypes.data_as(p64),
                                                      len(q) - 1, C.byref(h)), "drl_seq_layout_create")
        self._h = h
        self._plans = {}              # scratch bytes that calls of given sizes need
        self.device = scorer.device
        self.n_seg = len(q) - 1
        self.q_first, self.q_rows = int(q[0]), int(q[-1])
        self.k_first, self.k_rows = int(k[0]), int(k[-1])

    def close(self):
        if getattr(self, "_h", None):
            self._lib.drl_seq_layout_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class SequenceOps:
    """Mixin of WindowScorer."""

    def seq_layout(self, q_offsets: Sequence[int], k_offsets: Optional[Sequence[int]] = None) -> SeqLayout:
        """The plan of a packed batch: series i owns rows q_offsets[i]:q_offsets[i+1] of q and of the outputs, and rows
        k_offsets[i]:k_offsets[i+1] of k and v (the same rows without k_offsets; a cache's slots for steps)."""
        return SeqLayout(self, q_offsets, k_offsets)

    # ------------------------------------------------------------------ checks and plumbing
    def _tensor(self, name, x, dtype, ndim):
        """x as a tensor of that many axes on this scorer's GPU; its shape."""
        torch = _torch or _t()
        if not isinstance(x, torch.Tensor) or (dtype is not None and x.dtype != dtype):
            raise ValueError(f"{name} must be a {ndim}-dimensional tensor" + (f" of {dtype}" if dtype is not None else ""))
        shape = x.shape
        if len(shape) != ndim:
            raise ValueError(f"{name} must be a {ndim}-dimensional tensor, not of shape {tuple(shape)}")
        if not x.is_cuda or x.get_device() != self.device:
            raise ValueError(f"{name} is on {x.device}, the scorer on GPU {self.device}")
        if x.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{name} requires a gradient: the sequence operators are forward only (use torch.no_grad())")
        # outside of a dual level (its number, -1 there, is cheaper to ask for) no tensor has a tangent
        if getattr(_fw, "_current_level", 0) >= 0 and _fw.unpack_dual(x).tangent is not None:
            raise ValueError(f"{name} has a forward-mode tangent: the sequence operators have no derivatives")
        return shape

    def _rows(self, name, x, dtype, rows, heads=None, dim=None):
        """(shape, strides) of a tensor of rows x heads x dim."""
        s = self._tensor(name, x, dtype, 3)
        if s[0] < rows or (heads is not None and s[1] != heads) or (dim is not None and s[2] != dim):
            raise ValueError(f"{name} has shape {tuple(s)}, expected at least {rows} rows x {heads or s[1]} heads x {dim or s[2]}")
        st = x.stride()
        if st[2] != 1 and s[2] != 1:
            raise ValueError(f"the last axis of {name} must be dense")
        return s, st

    def _flat(self, name, x, dtype, n):
        s = self._tensor(name, x, dtype, 1)
        if s[0] != n or (n > 1 and x.stride(0) != 1):
            raise ValueError(f"{name} must hold {n} dense values")
        return x.data_ptr()

    def _layout(self, layout):
        if not isinstance(layout, SeqLayout) or layout._h is None:
            raise ValueError("layout is what seq_layout returned, not closed")
        if layout.device != self.device:
            raise ValueError(f"the layout is GPU {layout.device}'s, the scorer GPU {self.device}'s")
        return layout

    def _output(self, out, like, shape, covered):
        """(output tensor, its strides): the caller's, or a new one, zero where no series writes."""
        if out is None:
            out = like.new_empty(shape) if covered else like.new_zeros(shape)
            return out, out.stride()
        s, st = self._rows("out", out, like.dtype, 0, shape[1], shape[2])
        if s[0] != shape[0]:
            raise ValueError(f"out has {s[0]} rows, q {shape[0]}")
        return out, st

    def _run(self, name, dtype, like, head, args, plan):
        """One call on torch's current stream.  ``plan``, a dictionary of the layout's (or None: no scratch), keeps how much
        scratch calls of these sizes need; the scratch itself is torch's, new for each call."""
        code = _dtypes.get(dtype)
        if code is None:
            raise ValueError(f"dtype {dtype}: float32, float16 or bfloat16")
        lib, stream = self._lib, _stream(self.device)
        need, ws = 0, None
        if plan is not None:
            need = plan[0].get(plan[1])
            if need is None:
                n = C.c_int64(0)
                call = _abi.pack_call(_abi.SEQ_CALL_SIZE, _abi.ABI_REVISION, code, 1, stream, 0, 0)
                self._check(getattr(lib, f"drl_{name}_workspace")(self._h, *head, call, args, C.byref(n)), f"drl_{name}_workspace")
                need = plan[0][plan[1]] = n.value
        if need:
            ws = like.new_empty(need, dtype=_torch.uint8)
            call = _abi.pack_call(_abi.SEQ_CALL_SIZE, _abi.ABI_REVISION, code, 1, stream, ws.data_ptr(), need)
        else:
            call = _abi.pack_call(_abi.SEQ_CALL_SIZE, _abi.ABI_REVISION, code, 1, stream, 0, 0)
        rc = getattr(lib, f"drl_{name}_dev")(self._h, *head, call, args)
        if rc:
            self._check(rc, f"drl_{name}_dev")

    # ------------------------------------------------------------------ attention
    def attention(self, q, k, v, layout: SeqLayout, *, scale: Optional[float] = None, causal: bool = True, window: int = 0,
                  key_mask=None, k_len=None, out=None, return_lse: bool = False):
        """Softmax attention over the layout's series: q [rows, heads, dim], k and v [rows, kv_heads, dim] (any row and
        head strides of 16 bytes; float32, float16 or bfloat16), heads a multiple of kv_heads, dim a multiple of 8 up to 128.

        Row i of a series with nq rows and nk keys sees key j when j <= i + nk - nq (``causal``), j > i + nk - nq -
        window (``window`` > 0) and ``key_mask``[j] (bool, one per row of k).  ``k_len`` (int32, one per series): how
        many of its rows of k are filled; values outside them are clamped.  A row that sees nothing gets 0 and a
        log-sum of -inf.  Returns out, or (out, lse [rows, heads] float32)."""
        layout = self._layout(layout)
        (rows, heads, dim), qs = self._rows("q", q, None, layout.q_rows)
        dtype = q.dtype
        (k_rows, kv, _), ks = self._rows("k", k, dtype, layout.k_rows, None, dim)
        _, vs = self._rows("v", v, dtype, layout.k_rows, kv, dim)
        covered = layout.q_first == 0 and layout.q_rows == rows
        out, os_ = self._output(out, q, (rows, heads, dim), covered)
        lse, mask, klen = None, 0, 0
        if return_lse:
            lse = (q.new_empty if covered else q.new_zeros)((rows, heads), dtype=_torch.float32)
        if key_mask is not None:
            mask = self._flat("key_mask", key_mask, None, k_rows)
            if key_mask.dtype not in (_torch.bool, _torch.uint8):
                raise ValueError("key_mask must be bool or uint8")
        if k_len is not None:
            klen = self._flat("k_len", k_len, _torch.int32, layout.n_seg)
        window = max(-1, min(int(window), 0x7fffffff))             # more than any series has rows
        args = _abi.pack_attn(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), 0 if lse is None else lse.data_ptr(), mask, klen,
                              qs[0], qs[1], ks[0], ks[1], vs[0], vs[1], os_[0], os_[1], heads, kv, dim, 1 if causal else 0, window,
                              _scale(scale, dim))
        self._run("attention", dtype, q, (layout._h,), args, (layout._plans, (0, dtype, heads, kv, dim, causal, window)))
        return out if lse is None else (out, lse)

    # ------------------------------------------------------------------ linear attention
    def _state(self, name, x, shape):
        if self._tensor(name, x, _torch.float32, 4) != shape or not x.is_contiguous():
            raise ValueError(f"{name} must be a dense tensor of shape {shape}")
        return x.data_ptr()

    def linear_attention(self, q, k, v, log_decay, layout: SeqLayout, *, scale: Optional[float] = None, state=None, out=None,
                         final_state=None):
        """Linear attention over whole series: S <- exp(min(log_decay[h], 0)) S + k_t v_t^T, out_t = scale S^T q_t.

        q [rows, heads, dim_k], k [rows, kv_heads, dim_k], v [rows, kv_heads, dim_v]; the states are float32
        [n_seg, heads, dim_k, dim_v]: ``state`` the first ones (None: zeros), the last ones are returned, in
        ``final_state`` if given (it may be ``state``).  Returns (out [rows, heads, dim_v], final_state)."""
        layout = self._layout(layout)
        (rows, heads, dk), qs = self._rows("q", q, None, layout.q_rows)
        dtype = q.dtype
        (_, kv, _), ks = self._rows("k", k, dtype, layout.q_rows, None, dk)
        (_, _, dv), vs = self._rows("v", v, dtype, layout.q_rows, kv)
        out, os_ = self._output(out, q, (rows, heads, dv), layout.q_first == 0 and layout.q_rows == rows)
        shape = (layout.n_seg, heads, dk, dv)
        first = 0 if state is None else self._state("state", state, shape)
        if final_state is None:
            final_state = q.new_empty(shape, dtype=_torch.float32)
            last = final_state.data_ptr()
        else:
            last = self._state("final_state", final_state, shape)
        args = _abi.pack_linear(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), self._flat("log_decay", log_decay, _torch.float32, heads),
                                first, last, qs[0], qs[1], ks[0], ks[1], vs[0], vs[1], os_[0], os_[1], heads, kv, dk, dv,
                                _scale(scale, dk), 0)
        self._run("linear_attention", dtype, q, (layout._h,), args, (layout._plans, (1, dtype, heads, kv, dk, dv)))
        return out, final_state

    def linear_attention_step(self, q, k, v, log_decay, state, *, scale: Optional[float] = None, out=None):
        """One new row of each of n series: q [n, heads, dim_k], k [n, kv_heads, dim_k], v [n, kv_heads, dim_v]; ``state``
        [n, heads, dim_k, dim_v] is updated in place.  Returns out [n, heads, dim_v]."""
        (n, heads, dk), qs = self._rows("q", q, None, 0)
        dtype = q.dtype
        (_, kv, _), ks = self._rows("k", k, dtype, n, None, dk)
        (_, _, dv), vs = self._rows("v", v, dtype, n, kv)
        out, os_ = self._output(out, q, (n, heads, dv), True)
        st = self._state("state", state, (n, heads, dk, dv))
        args = _abi.pack_linear(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), self._flat("log_decay", log_decay, _torch.float32, heads),
                                st, st, qs[0], qs[1], ks[0], ks[1], vs[0], vs[1], os_[0], os_[1], heads, kv, dk, dv,
                                _scale(scale, dk), 0)
        self._run("linear_attention_step", dtype, q, (n,), args, None)
        return out

    # ------------------------------------------------------------------ group norm
    def group_norm(self, x, groups: int, gamma=None, beta=None, *, layout: Optional[SeqLayout] = None, eps: float = 1e-5,
                   activation: str = "linear", out=None):
        """Group normalisation and an activation ("linear", "relu", "sigmoid", "silu") of x [rows, channels]: statistics
        over each group's channels in all rows of a series, or, without a layout, in each row.  gamma and beta are
        float32 [channels].  ``out`` may be x."""
        rows, c = self._tensor("x", x, None, 2)
        xs = x.stride()
        if xs[1] != 1 and c != 1:
            raise ValueError("the last axis of x must be dense")
        if layout is not None and self._layout(layout).q_rows > rows:
            raise ValueError(f"x has {rows} rows, the layout {layout.q_rows}")
        if out is None:
            out = (x.new_empty if layout is None or (layout.q_first == 0 and layout.q_rows == rows) else x.new_zeros)((rows, c))
            ys = (c, 1)
        else:
            if self._tensor("out", out, x.dtype, 2) != x.shape or (out.stride(1) != 1 and c != 1):
                raise ValueError("out must have x's shape and a dense last axis")
            ys = out.stride()
        act = _ACTS.get(activation)
        if act is None:
            raise ValueError(f"activation {activation!r}: one of {', '.join(_ACTS)}")
        groups = max(-1, min(int(groups), 0x7fffffff))             # more than any tensor has channels
        xp, yp = x.data_ptr(), out.data_ptr()
        xr, yr = (xs[0], ys[0]) if rows > 1 else (c, c)
        args = _abi.pack_norm(xp, yp, 0 if gamma is None else self._flat("gamma", gamma, _torch.float32, c),
                              0 if beta is None else self._flat("beta", beta, _torch.float32, c), xr, yr, c, groups, act, _number("eps", eps))
        if layout is None:
            self._run("group_norm", x.dtype, x, (None, rows), args, None)
        else:
            # the plan goes by what x and out, and their rows, are aligned to as well
            self._run("group_norm", x.dtype, x, (layout._h, rows), args,
                      (layout._plans, (2, x.dtype, c, groups, (xp | yp) & 15, (xr | yr) & 7)))
        return out
