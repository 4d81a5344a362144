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


def _t():
    global _torch
    if _torch is None:
        import torch
        _dtypes.update({torch.float32: 0, torch.float16: 1, torch.bfloat16: 2})
        _torch = torch
    return _torch


class SeqLayout:
    """Which rows of packed tensors belong to which series: made once per batch layout with ``WindowScorer.seq_layout``
    and kept by the caller for as long as calls, or captured graphs, use it."""

    def __init__(self, scorer, q_offsets: Sequence[int], k_offsets: Optional[Sequence[int]] = None):
        q = np.ascontiguousarray(q_offsets, dtype=np.int64)
        k = q if k_offsets is None else np.ascontiguousarray(k_offsets, dtype=np.int64)
        if q.ndim != 1 or k.ndim != 1 or len(q) < 1 or len(q) != len(k):
            raise ValueError("offsets are one-dimensional, n_seg + 1 entries, as many for k as for q")
        self._lib, self._h = scorer._lib, None
        p64 = C.POINTER(C.c_int64)
        h = C.c_void_p()
        scorer._check(self._lib.drl_seq_layout_create(scorer._h, q.ctypes.data_as(p64), None if k_offsets is None else k.ctypes.data_as(p64),
                                                      len(q) - 1, C.byref(h)), "drl_seq_layout_create")
        self._h = h
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
        torch = _t()
        if not isinstance(x, torch.Tensor) or x.dim() != ndim or (dtype is not None and x.dtype != dtype):
            raise ValueError(f"{name} must be a {ndim}-dimensional tensor" + (f" of {dtype}" if dtype is not None else ""))
        if not x.is_cuda or x.get_device() != self.device:
            raise ValueError(f"{name} is on {x.device}, the scorer on GPU {self.device}")
        if x.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{name} requires a gradient: the sequence operators are forward only (use torch.no_grad())")
        return x

    def _rows(self, name, x, dtype, rows, heads=None, dim=None):
        self._tensor(name, x, dtype, 3)
        s = x.shape
        if s[0] < rows or (heads is not None and s[1] != heads) or (dim is not None and s[2] != dim):
            raise ValueError(f"{name} has shape {tuple(s)}, expected at least {rows} rows x {heads or s[1]} heads x {dim or s[2]}")
        if x.stride(2) != 1 and s[2] != 1:
            raise ValueError(f"the last axis of {name} must be dense")
        return x

    def _flat(self, name, x, dtype, n):
        self._tensor(name, x, dtype, 1)
        if x.shape[0] != n or not x.is_contiguous():
            raise ValueError(f"{name} must hold {n} dense values")
        return x.data_ptr()

    def _layout(self, layout):
        if not isinstance(layout, SeqLayout) or layout._h is None:
            raise ValueError("layout is what seq_layout returned, not closed")
        if layout.device != self.device:
            raise ValueError(f"the layout is GPU {layout.device}'s, the scorer GPU {self.device}'s")
        return layout

    def _output(self, out, like, shape, covered):
        """The output tensor: the caller's, or a new one, zero where no series writes."""
        torch = _t()
        if out is None:
            return torch.empty(shape, dtype=like.dtype, device=like.device) if covered else torch.zeros(shape, dtype=like.dtype, device=like.device)
        self._rows("out", out, like.dtype, 0, shape[1], shape[2])
        if out.shape[0] != shape[0]:
            raise ValueError(f"out has {out.shape[0]} rows, q {shape[0]}")
        return out

    def _call(self, dtype):
        try:
            code = _dtypes[dtype]
        except KeyError:
            raise ValueError(f"dtype {dtype}: float32, float16 or bfloat16") from None
        return _abi.SeqCall(_abi.SEQ_CALL_SIZE, _abi.ABI_REVISION, code, 1, _torch.cuda.current_stream(self.device).cuda_stream, None, 0)

    def _workspace(self, fn, head, call, args, device):
        """Asks how much scratch the call needs and takes it from torch; returns the tensor that keeps it alive."""
        n = C.c_int64(0)
        self._check(fn(self._h, *head, C.byref(call), C.byref(args), C.byref(n)), fn.__name__)
        if n.value == 0:
            return None
        ws = _torch.empty(n.value, dtype=_torch.uint8, device=device)
        call.workspace, call.workspace_bytes = ws.data_ptr(), n.value
        return ws

    # ------------------------------------------------------------------ attention
    def attention(self, q, k, v, layout: SeqLayout, *, scale: Optional[float] = None, causal: bool = True, window: int = 0,
                  key_mask=None, k_len=None, out=None, return_lse: bool = False):
        """Softmax attention over the layout's series: q [rows, heads, dim], k and v [rows, kv_heads, dim] (any row and
        head strides; float32, float16 or bfloat16), heads a multiple of kv_heads, dim a multiple of 8 up to 128.

        Row i of a series with nq rows and nk keys sees key j when j <= i + nk - nq (``causal``), j > i + nk - nq -
        window (``window`` > 0) and ``key_mask``[j] (bool, one per row of k).  ``k_len`` (int32, one per series): how
        many of its rows of k are filled; values outside them are clamped.  A row that sees nothing gets 0 and a
        log-sum of -inf.  Returns out, or (out, lse [rows, heads] float32)."""
        torch = _t()
        layout = self._layout(layout)
        self._rows("q", q, None, layout.q_rows)
        rows, heads, dim = q.shape
        self._rows("k", k, q.dtype, layout.k_rows, None, dim)
        self._rows("v", v, q.dtype, layout.k_rows, k.shape[1], dim)
        covered = layout.q_first == 0 and layout.q_rows == rows
        out = self._output(out, q, (rows, heads, dim), covered)
        lse = None
        if return_lse:
            lse = torch.empty((rows, heads), dtype=torch.float32, device=q.device) if covered else torch.zeros((rows, heads), dtype=torch.float32, device=q.device)
        mask = None
        if key_mask is not None:
            if key_mask.dtype not in (torch.bool, torch.uint8):
                raise ValueError("key_mask must be bool or uint8")
            mask = self._flat("key_mask", key_mask, None, k.shape[0])
        klen = None if k_len is None else self._flat("k_len", k_len, torch.int32, layout.n_seg)
        call = self._call(q.dtype)
        qs, ks, vs, os_ = q.stride(), k.stride(), v.stride(), out.stride()
        a = _abi.AttnArgs(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), None if lse is None else lse.data_ptr(), mask, klen,
                          qs[0], qs[1], ks[0], ks[1], vs[0], vs[1], os_[0], os_[1], heads, k.shape[1], dim, 1 if causal else 0, int(window),
                          dim ** -0.5 if scale is None else float(scale))
        ws = self._workspace(self._lib.drl_attention_workspace, (layout._h,), call, a, q.device)
        self._check(self._lib.drl_attention_dev(self._h, layout._h, C.byref(call), C.byref(a)), "drl_attention_dev")
        del ws
        return (out, lse) if return_lse else out

    # ------------------------------------------------------------------ linear attention
    def _linear_args(self, q, k, v, log_decay, out, state_in, state_out, scale):
        qs, ks, vs, os_ = q.stride(), k.stride(), v.stride(), out.stride()
        return _abi.LinearArgs(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), self._flat("log_decay", log_decay, _torch.float32, q.shape[1]),
                               None if state_in is None else state_in.data_ptr(), None if state_out is None else state_out.data_ptr(),
                               qs[0], qs[1], ks[0], ks[1], vs[0], vs[1], os_[0], os_[1], q.shape[1], k.shape[1], q.shape[2], v.shape[2],
                               q.shape[2] ** -0.5 if scale is None else float(scale), 0)

    def _state(self, name, x, shape):
        self._tensor(name, x, _torch.float32, 4)
        if tuple(x.shape) != shape or not x.is_contiguous():
            raise ValueError(f"{name} must be a dense tensor of shape {shape}")
        return x

    def linear_attention(self, q, k, v, log_decay, layout: SeqLayout, *, scale: Optional[float] = None, state=None, out=None,
                         final_state=None):
        """Linear attention over whole series: S <- exp(min(log_decay[h], 0)) S + k_t v_t^T, out_t = scale S^T q_t.

        q [rows, heads, dim_k], k [rows, kv_heads, dim_k], v [rows, kv_heads, dim_v]; the states are float32
        [n_seg, heads, dim_k, dim_v]: ``state`` the first ones (None: zeros), the last ones are returned, in
        ``final_state`` if given (it may be ``state``).  Returns (out [rows, heads, dim_v], final_state)."""
        torch = _t()
        layout = self._layout(layout)
        self._rows("q", q, None, layout.q_rows)
        rows, heads, dk = q.shape
        self._rows("k", k, q.dtype, layout.q_rows, None, dk)
        self._rows("v", v, q.dtype, layout.q_rows, k.shape[1])
        dv = v.shape[2]
        out = self._output(out, q, (rows, heads, dv), layout.q_first == 0 and layout.q_rows == rows)
        shape = (layout.n_seg, heads, dk, dv)
        if state is not None:
            self._state("state", state, shape)
        if final_state is None:
            final_state = torch.empty(shape, dtype=torch.float32, device=q.device)
        else:
            self._state("final_state", final_state, shape)
        call = self._call(q.dtype)
        a = self._linear_args(q, k, v, log_decay, out, state, final_state, scale)
        ws = self._workspace(self._lib.drl_linear_attention_workspace, (layout._h,), call, a, q.device)
        self._check(self._lib.drl_linear_attention_dev(self._h, layout._h, C.byref(call), C.byref(a)), "drl_linear_attention_dev")
        del ws
        return out, final_state

    def linear_attention_step(self, q, k, v, log_decay, state, *, scale: Optional[float] = None, out=None):
        """One new row of each of n series: q [n, heads, dim_k], k [n, kv_heads, dim_k], v [n, kv_heads, dim_v]; ``state``
        [n, heads, dim_k, dim_v] is updated in place.  Returns out [n, heads, dim_v]."""
        _t()
        self._rows("q", q, None, 0)
        n, heads, dk = q.shape
        self._rows("k", k, q.dtype, n, None, dk)
        self._rows("v", v, q.dtype, n, k.shape[1])
        out = self._output(out, q, (n, heads, v.shape[2]), True)
        self._state("state", state, (n, heads, dk, v.shape[2]))
        call = self._call(q.dtype)
        a = self._linear_args(q, k, v, log_decay, out, state, state, scale)
        self._check(self._lib.drl_linear_attention_step_dev(self._h, n, C.byref(call), C.byref(a)), "drl_linear_attention_step_dev")
        return out

    # ------------------------------------------------------------------ group norm
    def group_norm(self, x, groups: int, gamma=None, beta=None, *, layout: Optional[SeqLayout] = None, eps: float = 1e-5,
                   activation: str = "linear", out=None):
        """Group normalisation and an activation ("linear", "relu", "sigmoid", "silu") of x [rows, channels]: statistics
        over each group's channels in all rows of a series, or, without a layout, in each row.  gamma and beta are
        float32 [channels].  ``out`` may be x."""
        torch = _t()
        self._tensor("x", x, None, 2)
        rows, c = x.shape
        if x.stride(1) != 1 and c != 1:
            raise ValueError("the last axis of x must be dense")
        if layout is not None and self._layout(layout).q_rows > rows:
            raise ValueError(f"x has {rows} rows, the layout {layout.q_rows}")
        if out is None:
            covered = layout is None or (layout.q_first == 0 and layout.q_rows == rows)
            out = (torch.empty if covered else torch.zeros)((rows, c), dtype=x.dtype, device=x.device)
        else:
            self._tensor("out", out, x.dtype, 2)
            if out.shape != x.shape or (out.stride(1) != 1 and c != 1):
                raise ValueError("out must have x's shape and a dense last axis")
        if activation not in _ACTS:
            raise ValueError(f"activation {activation!r}: one of {', '.join(_ACTS)}")
        call = self._call(x.dtype)
        a = _abi.NormArgs(x.data_ptr(), out.data_ptr(), None if gamma is None else self._flat("gamma", gamma, torch.float32, c),
                          None if beta is None else self._flat("beta", beta, torch.float32, c),
                          x.stride(0) if rows > 1 else c, out.stride(0) if rows > 1 else c, c, int(groups), _ACTS[activation], float(eps))
        h = None if layout is None else layout._h
        ws = self._workspace(self._lib.drl_group_norm_workspace, (h, rows), call, a, x.device)
        self._check(self._lib.drl_group_norm_dev(self._h, h, rows, C.byref(call), C.byref(a)), "drl_group_norm_dev")
        del ws
        return out
