"""Operators on activation rows for attention between two meshes: rows of one
graph (cells, or single probe points) read the states of an encoder that ran
over another graph of another size.

  rms_norm         root-mean-square norm with the residual's addition
  rotary           rotary positions over several axes (cell coordinates)
  cross_attention  softmax attention of query rows to another sequence's keys

Rows are fp32, bf16 or fp16; sums, softmax statistics and norms are fp32 and
each output is rounded once.  All three run and differentiate in HIP kernels
of libmignn.so (through _ops.so, csrc/torch_ops.cpp, which also checks the
arguments) on the tensors' device and its current stream; there is no CPU path.
Outputs and scratch come from PyTorch's allocator at every call, so calls on
several streams, or captured into several graphs, share nothing but the
read-only `RotaryAxes` / `CrossPlan`.  Gradients are first order and reverse mode only.

A graph batch is a list of lengths (one sequence a graph), rows back to back.
"""

from __future__ import annotations

import ctypes
import math
from typing import Optional, Sequence

import numpy as np
import torch
import torch.nn as nn

from . import _lib
from . import train_ops as T

_ROW = {torch.float32: _lib.ROW_F32, torch.bfloat16: _lib.ROW_BF16, torch.float16: _lib.ROW_F16}


def _on_device(what: str, ref: torch.Tensor, **others):
    """Raises unless `ref` is on a ROCm device and the others are with it."""
    if not ref.is_cuda:
        raise RuntimeError(f"mignn {what} runs on ROCm devices only (no CPU path)")
    for name, t in others.items():
        if t is not None and t.device != ref.device:
            raise RuntimeError(f"mignn {what}: {name} is on {t.device}, not on {ref.device}")


# ---------------------------------------------------------------------------
# Root-mean-square norm

def rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None,
             eps: float = 1e-6):
    """y = s / sqrt(mean(s^2) + eps) * weight over the columns of x [N, H].

    Without `residual`, s = x and y is returned; with it (x's shape and type)
    s = x + residual and (y, s) is returned, s being the stream that the next
    residual adds to.  y is formed from the unrounded s.  weight: [H], float32
    or x's type.  H <= 2048."""
    return _lib.ops().rms_norm(x, weight, residual, eps)


# ---------------------------------------------------------------------------
# Rotary positions

class RotaryAxes:
    """The rotated pairs of each position axis and their frequencies.

    pairs[a] column pairs of a head belong to axis a, in order; pair i of axis
    a turns by pos[a] * scales[a] * base^(-i / pairs[a]) radians.  Pair j of
    all is columns (j, j + sum(pairs)), or (2j, 2j + 1) when `interleaved`;
    further columns of a head pass through.  Immutable; one device."""

    __slots__ = ("pairs", "base", "scales", "interleaved", "device", "freq", "axis", "total")

    def __init__(self, pairs: Sequence[int], base: float = 10000.0,
                 scales: Optional[Sequence[float]] = None, interleaved: bool = False,
                 device="cuda"):
        self.pairs = tuple(int(m) for m in pairs)
        if not self.pairs or any(m < 0 for m in self.pairs) or sum(self.pairs) == 0:
            raise ValueError(f"RotaryAxes: pairs must be counts with a positive sum, got {pairs}")
        if sum(self.pairs) > _lib.ROTARY_MAX_PAIRS:
            raise ValueError(f"RotaryAxes: {sum(self.pairs)} pairs (at most "
                             f"{_lib.ROTARY_MAX_PAIRS})")
        if not (base > 0.0 and math.isfinite(base)):
            raise ValueError(f"RotaryAxes: base must be positive and finite, got {base}")
        self.scales = tuple(float(s) for s in scales) if scales is not None \
            else (1.0,) * len(self.pairs)
        if len(self.scales) != len(self.pairs) or not all(math.isfinite(s) for s in self.scales):
            raise ValueError(f"RotaryAxes: {len(self.pairs)} finite scales expected, got {scales}")
        self.base, self.interleaved = float(base), bool(interleaved)
        self.total = sum(self.pairs)
        freq = [s * self.base ** (-i / m) / (2.0 * math.pi)
                for m, s in zip(self.pairs, self.scales) for i in range(m)]
        axis = [a for a, m in enumerate(self.pairs) for _ in range(m)]
        self.freq = torch.tensor(freq, dtype=torch.float64).to(device)
        self.axis = torch.tensor(axis, dtype=torch.int32).to(device)
        self.device = self.freq.device


def rotary(x: torch.Tensor, pos: torch.Tensor, axes: RotaryAxes) -> torch.Tensor:
    """x [N, heads, d] with the pairs of every head turned by the row's
    position pos [N, len(axes.pairs)] (float32 / float64 coordinates or int32 /
    int64 indices; angles are formed in float64).  Positions get no gradient."""
    return _lib.ops().rotary(x, pos, axes.freq, axes.axis, len(axes.pairs), axes.interleaved)


# ---------------------------------------------------------------------------
# Cross attention

def _lengths(what: str, lens) -> np.ndarray:
    if torch.is_tensor(lens):
        if lens.device.type != "cpu":
            raise ValueError(f"CrossPlan: {what} must be on the host (they size the launches)")
        lens = lens.tolist()
    if isinstance(lens, (int, np.integer)):
        lens = [lens]
    a = np.asarray(lens)
    if a.size and (a.dtype.kind not in "iu"):
        raise ValueError(f"CrossPlan: {what} must be whole numbers")
    a = np.ascontiguousarray(a.reshape(-1), dtype=np.int64)
    if a.size and a.min() < 0:
        raise ValueError(f"CrossPlan: negative length in {what}")
    return a


class CrossPlan:
    """The work of cross attention for given lengths: q_lens[b] queries read
    k_lens[b] keys, the sequences' rows back to back (one int: a single
    sequence).  Lengths of 0 are allowed.  Holds the launches' work lists on
    `device`; immutable, so it may serve any number of calls, streams and
    captured graphs (which need it for as long as they are replayed).
    train=False leaves the backward's lists out."""

    __slots__ = ("q_lens", "k_lens", "queries", "keys", "heads", "kv_heads", "head_dim", "dtype",
                 "device", "train", "_call", "_lists", "_address")

    def __init__(self, q_lens, k_lens, *, heads: int, kv_heads: Optional[int] = None,
                 head_dim: int, dtype: torch.dtype = torch.float32, device="cuda",
                 train: bool = True):
        ql, kl = _lengths("q_lens", q_lens), _lengths("k_lens", k_lens)
        if ql.size != kl.size:
            raise ValueError(f"CrossPlan: {ql.size} query sequences but {kl.size} key sequences")
        kv_heads = heads if kv_heads is None else kv_heads
        if heads < 1 or kv_heads < 1 or heads % kv_heads:
            raise ValueError(f"CrossPlan: {heads} query heads over {kv_heads} key heads")
        if heads // kv_heads > _lib.CROSS_MAX_GROUP:
            raise ValueError(f"CrossPlan: more than {_lib.CROSS_MAX_GROUP} query heads a key head")
        if head_dim < 8 or head_dim % 8 or head_dim > _lib.CROSS_MAX_D:
            raise ValueError(f"CrossPlan: head_dim must be a multiple of 8 up to "
                             f"{_lib.CROSS_MAX_D}, got {head_dim}")
        if dtype not in _ROW:
            raise TypeError(f"CrossPlan: rows must be float32, bfloat16 or float16, got {dtype}")
        self.q_lens, self.k_lens = tuple(ql.tolist()), tuple(kl.tolist())
        self.heads, self.kv_heads, self.head_dim = int(heads), int(kv_heads), int(head_dim)
        self.dtype, self.train = dtype, bool(train)
        self.queries, self.keys = int(ql.sum()), int(kl.sum())
        L = _lib.lib()
        info = (ctypes.c_int64 * 8)()
        lengths = ql.ctypes.data, kl.ctypes.data
        lists, spans, at = [], [], 0
        size = _lib.CROSS_ITEM_BYTES
        for kind in range(3 if train else 1):
            def plan(items, joins):
                _lib.check(L.mignn_cross_plan(
                    *lengths, ql.size, self.heads, self.kv_heads, self.head_dim, _ROW[dtype],
                    kind, items, joins, info), "mignn_cross_plan")
            plan(None, None)
            n_items, n_joins, part = info[:3]
            buf = np.empty((n_items + n_joins) * size, np.uint8)
            base = buf.ctypes.data
            plan(base, base + n_items * size)
            spans.append((at, at + n_items * size, part, n_items, n_joins) + tuple(info[5:]))
            lists.append(buf)
            at += buf.size
        host = torch.from_numpy(np.concatenate(lists))
        self._lists = host.to(device)
        self.device = self._lists.device
        base = self._lists.data_ptr()
        call = _lib.CrossCall()
        call.heads, call.kv_heads, call.d = self.heads, self.kv_heads, self.head_dim
        call.dtype, call.n_keys = _ROW[dtype], self.keys
        for kind, (items, joins, part, n_items, n_joins, tile, rows, whole) in enumerate(spans):
            ps = call.passes[kind]
            ps.items, ps.joins, ps.part_bytes = base + items, base + joins, part
            ps.n_items, ps.n_joins, ps.n_whole = n_items, n_joins, whole
            ps.tile, ps.rows = tile, rows
        self._call = call
        self._address = ctypes.addressof(call)


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, plan: CrossPlan,
                    key_mask: Optional[torch.Tensor] = None,
                    scale: Optional[float] = None) -> torch.Tensor:
    """Attention of q [queries, heads, d] to k, v [keys, kv_heads, d], each
    sequence of `plan` to its own keys; query head h reads key head
    h // (heads // kv_heads).  key_mask: bool [keys], False leaves a key out,
    whatever its rows hold.  scale: > 0, default 1 / sqrt(d).  Returns
    [queries, heads, d]; a query without keys gets 0, and no gradient flows
    through it.

    fp32 rows are multiplied as three bf16 terms each, to fp32's own rounding;
    there an infinite key or value makes NaN of the queries that read it.  16-bit
    rows: the weights (and, in the backward, the scores' gradients) are rounded
    to the rows' type ahead of their product with the values, but for
    passes of few results (a key head's output, or its keys' gradient, of less
    than 16384 numbers, or no sequence above 32 rows), gradients over at most 64
    keys or rows, and queries' gradients of heads to 16 columns, which keep the
    remainders: what a row's last bits are depends on the plan that it is part of."""
    return _lib.ops().cross_attention(q, k, v, key_mask, scale, plan._lists, plan._address,
                                      plan.queries, plan.train)


# ---------------------------------------------------------------------------
# The block

def graph_lengths(batch: Optional[torch.Tensor], num_nodes: int, num_graphs: Optional[int] = None):
    """Rows of each graph of a `Batch` (its `batch` vector, sorted as
    `Batch.from_data_list` makes it); one graph without a vector.  Reads the
    vector on the host."""
    if batch is None:
        return [num_nodes]
    b = batch.detach().cpu()
    if b.numel() != num_nodes or (b.numel() > 1 and bool((b[1:] < b[:-1]).any())):
        raise ValueError("graph_lengths: batch must be a sorted vector, one entry a row")
    return torch.bincount(b, minlength=num_graphs or 0).tolist()


class CrossAttention(nn.Module):
    """Rows of one graph read the states of another:

        q = turn(Wq norm(x)),  k = turn(Wk norm(context)),  v = Wv norm(context)
        (y, s) = norm(Wo attend(q, k, v), residual=x)

    `turn` is `rotary` by the rows' positions (cell centres), so that scores
    depend on where the cells lie to each other.  Returns (y, s): the normed
    rows and the stream s = x + the attention's output.  fp32, on the device;
    differentiable in the rows, the context and the parameters."""

    def __init__(self, hidden_dim: int, heads: int = 4, kv_heads: Optional[int] = None,
                 axes: int = 3, base: float = 100.0, position_scale: float = 64.0,
                 eps: float = 1e-6):
        super().__init__()
        kv_heads = heads if kv_heads is None else kv_heads
        if heads < 1 or hidden_dim % heads or kv_heads < 1 or heads % kv_heads:
            raise ValueError(f"CrossAttention: hidden_dim {hidden_dim} over {heads} heads, "
                             f"{kv_heads} key heads")
        d = hidden_dim // heads
        if d % 8 or d > _lib.CROSS_MAX_D:
            raise ValueError(f"CrossAttention: head width {d} must be a multiple of 8 up to "
                             f"{_lib.CROSS_MAX_D}")
        if not 1 <= axes <= d // 2:
            raise ValueError(f"CrossAttention: {axes} position axes for heads of width {d}")
        self.hidden_dim, self.heads, self.kv_heads, self.head_dim = hidden_dim, heads, kv_heads, d
        self.axes, self.base, self.position_scale = axes, base, position_scale
        self.eps = eps
        self.norm_x = nn.Parameter(torch.ones(hidden_dim))
        self.norm_context = nn.Parameter(torch.ones(hidden_dim))
        self.norm_out = nn.Parameter(torch.ones(hidden_dim))
        self.lin_query = nn.Linear(hidden_dim, heads * d)
        self.lin_key = nn.Linear(hidden_dim, kv_heads * d)
        self.lin_value = nn.Linear(hidden_dim, kv_heads * d)
        self.lin_out = nn.Linear(heads * d, hidden_dim)
        self._axes = None

    def plan(self, q_lens, k_lens, train: bool = True, device="cuda") -> CrossPlan:
        """The work lists for rows and context rows per graph."""
        return CrossPlan(q_lens, k_lens, heads=self.heads, kv_heads=self.kv_heads,
                         head_dim=self.head_dim, device=device, train=train)

    def _rotary_axes(self, device) -> RotaryAxes:
        scales = (float(self.position_scale),) * self.axes
        if self._axes is None or self._axes.device != device \
                or (self._axes.base, self._axes.scales) != (self.base, scales):
            half = self.head_dim // 2
            pairs = [half // self.axes + (a < half % self.axes) for a in range(self.axes)]
            self._axes = RotaryAxes(pairs, base=self.base, scales=scales, device=device)
        return self._axes

    def keys_values(self, context: torch.Tensor, context_pos: torch.Tensor):
        """(k, v) of the context rows: computed once for many `attend` calls."""
        n = context.shape[0]
        h = rms_norm(context, self.norm_context, eps=self.eps)
        k = T.linear(h, self.lin_key.weight, self.lin_key.bias)
        v = T.linear(h, self.lin_value.weight, self.lin_value.bias)
        k = rotary(k.view(n, self.kv_heads, self.head_dim), context_pos[:, :self.axes],
                   self._rotary_axes(context.device))
        return k, v.view(n, self.kv_heads, self.head_dim)

    def attend(self, x: torch.Tensor, pos: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
               plan: CrossPlan, key_mask: Optional[torch.Tensor] = None):
        """(y, s) of rows x at positions pos [N, >= axes] over given keys and values."""
        n = x.shape[0]
        q = T.linear(rms_norm(x, self.norm_x, eps=self.eps), self.lin_query.weight,
                     self.lin_query.bias)
        q = rotary(q.view(n, self.heads, self.head_dim), pos[:, :self.axes],
                   self._rotary_axes(x.device))
        o = cross_attention(q, k, v, plan, key_mask=key_mask)
        o = T.linear(o.reshape(n, self.heads * self.head_dim), self.lin_out.weight,
                     self.lin_out.bias)
        return rms_norm(o, self.norm_out, residual=x, eps=self.eps)

    def forward(self, x, pos, context, context_pos, plan: CrossPlan,
                key_mask: Optional[torch.Tensor] = None):
        for name, t in (("x", x), ("context", context)):
            if t.dim() != 2 or t.shape[1] != self.hidden_dim or t.dtype != torch.float32:
                raise ValueError(f"CrossAttention: {name} must be float32 [N, {self.hidden_dim}], "
                                 f"got {t.dtype} {tuple(t.shape)}")
        _on_device("CrossAttention", x, context=context, parameters=self.norm_x)
        k, v = self.keys_values(context, context_pos)
        return self.attend(x, pos, k, v, plan, key_mask)
