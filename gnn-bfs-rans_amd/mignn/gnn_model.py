"""FlowGNN on MI355X: the reference's model API, executed by libmignn.so.

Drop-in for `gnn_model.FlowGNN` (reference gnn_model.py:14-220) and
`FlowGNNSurrogate` (:223-291):

* same constructor arguments, `forward(x, edge_index, edge_attr=None,
  batch=None) -> [N, output_dim]`, `predict_fields`, and the same
  `state_dict` keys as the PyG-built reference model, so a
  reference checkpoint's `model_state_dict` loads with `load_state_dict`
  (PyG 2.3/2.4 `lin_src/lin_dst` and 2.5+ `lin` GAT layouts both accepted);
* same errors: `ValueError("Unknown layer type ...")`, `ValueError` on a bad
  edge_index shape / edge_attr count, and any failure inside a layer becomes
  `RuntimeError("Message passing failed in layer i (type): ...")` with the
  reference's diagnostic lines (gnn_model.py:173-181); invalid indices are
  dropped silently (:133-141), on the device, without host syncs.

Every arithmetic step of `forward` runs in the HIP library (CSR build,
aggregation, MFMA transforms, fused epilogues); PyTorch only allocates device
memory and provides the stream.

Precision (`FlowGNN.precision`, default from $MIGNN_PRECISION, else
"f16x3"): "f32" runs the node transforms on the exact-fp32 MFMA
(v_mfma_f32_16x16x4_f32, a k-ordered fmaf chain); "f16x3" runs them as three
fp16 MFMAs on power-of-two-scaled hi/lo splits of both operands with fp32
accumulation (relative error per product ~2^-22, 16x the f32 MFMA rate),
where a kernel exists for the shape (fused GCN layer, H in {64, 128}); the
measured field error stays well inside the north star's 1e-5 either way.  There is no CPU path: tensors must be on a
ROCm device and the library must be built.  model.train() runs the
training path (mignn.train_ops): exact-fp32 kernels with
batch-statistics BN, dropout and a HIP backward for every layer type.

Weight re-association (one-time per weight version, float64 on the device):
* GAT: logits a_src = x . (W_h^T att_src_h) -> an [N, 2*heads] GEMV-GEMM;
  out = mean_h (sum_j alpha x_j) W_h^T -> one [N, heads*H] x [heads*H, H] GEMM.
* TransformerConv: q~_h = Wk_h^T q_h, so q_h . k_j = q~_h . x_j + q_h . bk_h;
  value / skip projections are applied after aggregation by one GEMM.
  The [N, heads*C] Q/K/V tensors of the reference are never materialised.
"""

from __future__ import annotations

import math
import os
from typing import Dict, Optional, Tuple

import torch
import torch.nn as nn

from . import _lib
from . import train_ops as T
from .attention import CrossAttention, graph_lengths
from ._lib import (CSR_ONE_SELF_LOOP, CSR_TRANSPOSE, CSR_VERBATIM, EPI_AFFINE, EPI_BIAS, EPI_RELU,
                   EPI_RESIDUAL)

HEADS = 4  # gnn_model.py:67, :79
# the split-fp16 GCN layer kernel of FlowGNN.gcn_kernel = "auto", per hidden
# width: the fastest measured on the bench mesh: the
# window kernel at both widths (10M-row layer, same box: H = 64 1.24 ms vs the
# ring kernel's 1.32; H = 128 2.84 ms vs the producer / consumer kernel's 3.02
# -- 0.7 ms per 4-layer forward against its 0.46 ms plan per graph).  A
# block-ordered CSR (a shard's range) takes the ring kernel at H = 64 and the
# producer / consumer kernel at H = 128 (FlowGNN._gcn_kernel).
GCN_KERNEL_AUTO = {64: "win", 128: "win"}
GCN_BLOCK_ORDER = {64: "ring", 128: "pc"}


# ---------------------------------------------------------------------------
# PyG-named parameter containers (state_dict layout of the reference model)
# ---------------------------------------------------------------------------

class GCNConv(nn.Module):
    """Parameters of PyG GCNConv(H, H): `lin.weight` [H,H] (no bias), `bias` [H]."""

    def __init__(self, in_channels: int, out_channels: int):
        super().__init__()
        self.lin = nn.Linear(in_channels, out_channels, bias=False)
        self.bias = nn.Parameter(torch.zeros(out_channels))


class GATConv(nn.Module):
    """Parameters of PyG GATConv(H, H, heads=4, concat=False)."""

    def __init__(self, in_channels: int, out_channels: int, heads: int = HEADS,
                 concat: bool = False, dropout: float = 0.0, negative_slope: float = 0.2):
        super().__init__()
        self.heads, self.out_channels = heads, out_channels
        self.dropout, self.negative_slope = dropout, negative_slope
        self.lin = nn.Linear(in_channels, heads * out_channels, bias=False)
        self.att_src = nn.Parameter(torch.zeros(1, heads, out_channels))
        self.att_dst = nn.Parameter(torch.zeros(1, heads, out_channels))
        self.bias = nn.Parameter(torch.zeros(out_channels))

    def _load_from_state_dict(self, state_dict, prefix, *args, **kwargs):
        # PyG 2.3/2.4 registered the shared projection as lin_src (== lin_dst).
        src, dst, new = prefix + "lin_src.weight", prefix + "lin_dst.weight", prefix + "lin.weight"
        if src in state_dict and new not in state_dict:
            state_dict[new] = state_dict.pop(src)
            state_dict.pop(dst, None)
        super()._load_from_state_dict(state_dict, prefix, *args, **kwargs)


class GINConv(nn.Module):
    """Parameters of PyG GINConv(nn=Seq(Lin, ReLU, Lin), eps=0, train_eps=False)."""

    def __init__(self, nn_module: nn.Module, eps: float = 0.0):
        super().__init__()
        self.nn = nn_module
        self.register_buffer("eps", torch.tensor([float(eps)]))


class TransformerConv(nn.Module):
    """Parameters of PyG TransformerConv(H, H, heads=4, concat=False)."""

    def __init__(self, in_channels: int, out_channels: int, heads: int = HEADS,
                 concat: bool = False, dropout: float = 0.0):
        super().__init__()
        self.heads, self.out_channels, self.dropout = heads, out_channels, dropout
        self.lin_key = nn.Linear(in_channels, heads * out_channels)
        self.lin_query = nn.Linear(in_channels, heads * out_channels)
        self.lin_value = nn.Linear(in_channels, heads * out_channels)
        self.lin_skip = nn.Linear(in_channels, out_channels)


class BatchNorm(nn.Module):
    """PyG BatchNorm: `module` = BatchNorm1d(H, eps=1e-5, momentum=0.1)."""

    def __init__(self, in_channels: int, eps: float = 1e-5, momentum: float = 0.1):
        super().__init__()
        self.module = nn.BatchNorm1d(in_channels, eps=eps, momentum=momentum)


# ---------------------------------------------------------------------------
# Graph structure cache
# ---------------------------------------------------------------------------

class Csr:
    """Destination-major CSR.  With a locality order (`perm`, `inv` set), node
    ids inside the CSR are the internal ids: internal row p is caller node
    perm[p], caller node v is internal row inv[v]."""
    __slots__ = ("row_ptr", "col", "dinv", "ew", "info", "num_nodes", "num_edges", "edge_index",
                 "perm", "inv", "pos", "key_tensor", "plans", "order_info")

    def __init__(self, row_ptr, col, dinv, info, num_nodes, num_edges, edge_index, ew=None):
        self.row_ptr, self.col, self.dinv, self.info = row_ptr, col, dinv, info
        self.num_nodes, self.num_edges, self.edge_index = num_nodes, num_edges, edge_index
        self.ew = ew
        self.perm = self.inv = self.pos = None
        self.order_info = None   # int32[4] of the column order (mignn_locality_order_cols)
        self.key_tensor = None   # the caller's edge_index the cache key was made from
        self.plans: Dict[Tuple[str, int, int, int, int], torch.Tensor] = {}

    def ring_plan(self, h: int, row_begin: int, row_end: int) -> torch.Tensor:
        """The ring kernel's plan of rows [row_begin, row_end) for hidden
        width h (mignn_gcn_ring_plan: per-tile records, ext-row lists and the
        schedule of this device), built on first use and kept with the CSR."""
        # (the plan's schedule is for the device current at build time: its
        # CU count sets the grid -- a launch from another device must not reuse it)
        key = ("ring", h, row_begin, row_end, torch.cuda.current_device())
        plan = self.plans.get(key)
        if plan is None:
            L = _lib.lib()
            nb = L.mignn_gcn_ring_plan_bytes(row_begin, row_end, h)
            plan = torch.empty(max(nb, 16), dtype=torch.uint8, device=self.col.device)
            _lib.check(L.mignn_gcn_ring_plan(_lib.ptr(self.row_ptr), _lib.ptr(self.col),
                                             _lib.ptr(self.ew), row_begin, row_end, h,
                                             _lib.ptr(plan), nb, None,
                                             _lib.stream(self.col.device)), "mignn_gcn_ring_plan")
            self.plans[key] = plan
        return plan

    def win_plan(self, h: int, row_begin: int, row_end: int) -> torch.Tensor:
        """The window kernel's plan of rows [row_begin, row_end) for hidden
        width h (mignn_gcn_win_plan: header with this device's grid and the
        schedule -- the column schedule when the CSR is in the column order
        and the plan's rows start at row 0 (a shard's interior range: the
        plane count per column taken from the CSR, mignn_gcn_win_plan) --
        and a 16-B record per row: neighbour codes and degree classes, the
        weights rebuilt in LDS from the header's class table -- a row whose
        ew are not exactly those products takes the CSR path), built on first
        use and kept with the CSR (it reads ew once, at build time)."""
        key = ("win", h, row_begin, row_end, torch.cuda.current_device())
        plan = self.plans.get(key)
        if plan is None:
            L = _lib.lib()
            nb = L.mignn_gcn_win_plan_bytes(row_begin, row_end, h)
            plan = torch.empty(max(nb, 16), dtype=torch.uint8, device=self.col.device)
            info = self.order_info if row_begin == 0 else None
            _lib.check(L.mignn_gcn_win_plan(_lib.ptr(self.row_ptr), _lib.ptr(self.col),
                                            _lib.ptr(self.ew), row_begin, row_end, h,
                                            _lib.ptr(info), _lib.ptr(plan), nb, None,
                                            _lib.stream(self.col.device)), "mignn_gcn_win_plan")
            self.plans[key] = plan
        return plan

    def compute_gcn_weights(self, row_begin: int = 0, row_end: Optional[int] = None):
        """Per-entry PyG gcn_norm weights (mignn_gcn_norm); call again after the
        halo dinv exchange of a sharded graph."""
        re = self.num_nodes if row_end is None else row_end
        if self.ew is None:
            self.ew = torch.empty_like(self.col, dtype=torch.float32)
        self.plans.clear()
        _lib.check(_lib.lib().mignn_gcn_norm(_lib.ptr(self.row_ptr), _lib.ptr(self.col),
                                             _lib.ptr(self.dinv), row_begin, re, _lib.ptr(self.ew),
                                             _lib.stream(self.col.device)), "mignn_gcn_norm")


def locality_order(pos: torch.Tensor, edge_index: torch.Tensor, cols: bool = False):
    """(perm, inv) of mignn_locality_order: 4x4x4-cell blocks (one 64-row tile
    of the fused layer each) in panels of 4x4 block columns swept along the
    third axis, from the cell centres `pos` [N, >=3]; perm[new] = old id,
    inv[old] = new.  cols=True: the column order of the window GCN kernel
    (mignn_locality_order_cols: 8x8-cell columns, z inside) and its info,
    (perm, inv, info)."""
    dev = pos.device
    n = int(pos.shape[0])
    p = pos if (pos.dtype == torch.float32 and pos.stride(1) == 1) else pos.float().contiguous()
    ei = edge_index
    if ei.dtype != torch.int64 or not ei.is_contiguous():
        ei = ei.to(torch.int64).contiguous()
    perm = torch.empty(max(n, 1), dtype=torch.int32, device=dev)
    inv = torch.empty(max(n, 1), dtype=torch.int32, device=dev)
    L = _lib.lib()
    nbytes = L.mignn_locality_order_scratch_bytes(n)
    if nbytes == 0:
        raise _lib.MignnError("locality order scratch query failed: " + _lib.last_error())
    scratch = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    if cols:
        info = torch.zeros(4, dtype=torch.int32, device=dev)
        _lib.check(L.mignn_locality_order_cols(_lib.ptr(p), p.stride(0), n, _lib.ptr(ei),
                                               int(ei.shape[1]), _lib.ptr(perm), _lib.ptr(inv),
                                               _lib.ptr(info), _lib.ptr(scratch), nbytes,
                                               _lib.stream(dev)), "mignn_locality_order_cols")
        return perm[:n], inv[:n], info
    _lib.check(L.mignn_locality_order(_lib.ptr(p), p.stride(0), n, _lib.ptr(ei), int(ei.shape[1]),
                                      _lib.ptr(perm), _lib.ptr(inv), _lib.ptr(scratch), nbytes,
                                      _lib.stream(dev)), "mignn_locality_order")
    return perm[:n], inv[:n]


def build_csr(edge_index: torch.Tensor, num_nodes: int, mode: int,
              relabel: Optional[torch.Tensor] = None) -> Csr:
    """Destination-major CSR on the device (mignn_csr_build); no host sync.
    `relabel` (int32 [N], a permutation): node ids mapped through it."""
    dev = edge_index.device
    ei = edge_index
    if ei.dtype != torch.int64 or not ei.is_contiguous():
        ei = ei.to(torch.int64).contiguous()
    E = int(ei.shape[1])
    N = int(num_nodes)
    row_ptr = torch.empty(N + 1, dtype=torch.int32, device=dev)
    col = torch.empty(max(E + N, 1), dtype=torch.int32, device=dev)
    dinv = torch.empty(max(N, 1), dtype=torch.float32, device=dev) if mode == CSR_ONE_SELF_LOOP else None
    info = torch.zeros(4, dtype=torch.int64, device=dev)
    L = _lib.lib()
    nbytes = L.mignn_csr_scratch_bytes(E, N)
    if nbytes == 0:
        raise _lib.MignnError("csr scratch query failed: " + _lib.last_error())
    scratch = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    # ONE_SELF_LOOP: the gcn_norm weights come out of the same pass
    ew = torch.empty_like(col, dtype=torch.float32) if mode == CSR_ONE_SELF_LOOP else None
    _lib.check(L.mignn_csr_build_gcn(_lib.ptr(ei), E, N, mode, _lib.ptr(relabel),
                                     _lib.ptr(row_ptr), _lib.ptr(col), _lib.ptr(dinv), _lib.ptr(ew),
                                     _lib.ptr(info), _lib.ptr(scratch), nbytes,
                                     _lib.stream(dev)), "mignn_csr_build")
    return Csr(row_ptr, col, dinv, info, N, E, ei, ew=ew)


def build_csr_range(edge_index: torch.Tensor, num_nodes: int, lo: int, hi: int,
                    inv: torch.Tensor, ghost_rank: torch.Tensor, n_local: int, mode: int) -> Csr:
    """A node-range shard's CSR straight from its global-id in-edges
    (mignn_csr_build_range): ids mapped to the shard's local ids inside the
    build as mignn_range_relabel maps them (`inv` int64 [hi - lo],
    `ghost_rank` int64 [num_nodes + 1], mignn.dist.RangeLayout's) -- the same
    CSR as build_csr(<the relabelled list>, n_local, mode), bit for bit."""
    dev = edge_index.device
    ei = edge_index
    if ei.dtype != torch.int64 or not ei.is_contiguous():
        ei = ei.to(torch.int64).contiguous()
    E = int(ei.shape[1])
    N = int(n_local)
    row_ptr = torch.empty(N + 1, dtype=torch.int32, device=dev)
    col = torch.empty(max(E + N, 1), dtype=torch.int32, device=dev)
    dinv = torch.empty(max(N, 1), dtype=torch.float32, device=dev) if mode == CSR_ONE_SELF_LOOP else None
    info = torch.zeros(4, dtype=torch.int64, device=dev)
    L = _lib.lib()
    nbytes = L.mignn_csr_scratch_bytes(E, N)
    if nbytes == 0:
        raise _lib.MignnError("csr scratch query failed: " + _lib.last_error())
    scratch = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    ew = torch.empty_like(col, dtype=torch.float32) if mode == CSR_ONE_SELF_LOOP else None
    _lib.check(L.mignn_csr_build_range(_lib.ptr(ei), E, int(num_nodes), int(lo), int(hi),
                                       _lib.ptr(inv), _lib.ptr(ghost_rank), N, mode,
                                       _lib.ptr(row_ptr), _lib.ptr(col), _lib.ptr(dinv),
                                       _lib.ptr(ew), _lib.ptr(info), _lib.ptr(scratch), nbytes,
                                       _lib.stream(dev)), "mignn_csr_build_range")
    return Csr(row_ptr, col, dinv, info, N, E, None, ew=ew)


class _CsrCache:
    """Keyed by (edge_index storage, version, shape, N, mode, device) -- plus
    the positions' storage / version when a locality order is requested;
    holds references to the keyed tensors themselves (Csr.key_tensor,
    Csr.pos) so their storage cannot be recycled while cached."""

    def __init__(self, capacity: int = 4):
        self.capacity = capacity
        self.entries: Dict[Tuple, Csr] = {}

    @staticmethod
    def _build(edge_index, num_nodes, mode, pos, cols=False):
        if pos is None:
            return build_csr(edge_index, num_nodes, mode)
        info = None
        if cols:
            perm, inv, info = locality_order(pos, edge_index, cols=True)
        else:
            perm, inv = locality_order(pos, edge_index)
        csr = build_csr(edge_index, num_nodes, mode, relabel=inv)
        csr.perm, csr.inv, csr.pos, csr.order_info = perm, inv, pos, info
        return csr

    def get(self, edge_index: torch.Tensor, num_nodes: int, mode: int,
            pos: Optional[torch.Tensor] = None, cols: bool = False) -> Csr:
        """cols: the column order (the window GCN kernel's) instead of the
        block order, when a locality order is requested (pos given)."""
        if self.capacity <= 0:        # caching off: rebuild every forward
            return self._build(edge_index, num_nodes, mode, pos, cols)
        key = (edge_index.data_ptr(), edge_index._version, tuple(edge_index.shape),
               tuple(edge_index.stride()), edge_index.dtype, int(num_nodes), mode,
               str(edge_index.device))
        if pos is not None:
            key += (pos.data_ptr(), pos._version, tuple(pos.shape), tuple(pos.stride()), bool(cols))
        hit = self.entries.get(key)
        if hit is not None:
            return hit
        csr = self._build(edge_index, num_nodes, mode, pos, cols)
        # the key holds the caller's storage address: keep that tensor (not
        # only the int64 copy build_csr may have made of an int32 or strided
        # edge_index) alive so the allocator cannot hand its address to the
        # next graph while this entry exists
        csr.key_tensor = edge_index
        if len(self.entries) >= self.capacity:
            self.entries.pop(next(iter(self.entries)))
        self.entries[key] = csr
        return csr


# ---------------------------------------------------------------------------
# Native op wrappers
# ---------------------------------------------------------------------------

def _stream(t: torch.Tensor) -> int:
    return _lib.stream(t.device)


def linear(a: torch.Tensor, w: torch.Tensor, bias=None, *, relu=False, residual=None,
           scale=None, shift=None, a2: Optional[torch.Tensor] = None,
           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """out = epi([a | a2] @ w.T) on MFMA (mignn_linear)."""
    M, K1 = a.shape
    K2 = 0 if a2 is None else a2.shape[1]
    N = w.shape[0]
    if out is None:
        out = torch.empty((M, N), dtype=torch.float32, device=a.device)
    flags = (EPI_BIAS if bias is not None else 0) | (EPI_RESIDUAL if residual is not None else 0) \
        | (EPI_AFFINE if scale is not None else 0) | (EPI_RELU if relu else 0)
    _lib.check(_lib.lib().mignn_linear(
        _lib.ptr(a), a.stride(0), M, K1, _lib.ptr(a2), 0 if a2 is None else a2.stride(0), K2,
        _lib.ptr(w), N, _lib.ptr(bias), _lib.ptr(residual),
        0 if residual is None else residual.stride(0), _lib.ptr(scale), _lib.ptr(shift), flags,
        _lib.ptr(out), out.stride(0), _stream(a)), "mignn_linear")
    return out


def f16x3_image(w: torch.Tensor) -> torch.Tensor:
    """Split-fp16 image of W [n, k] for linear_f16x3 (mignn_linear_f16x3_prep)."""
    L = _lib.lib()
    w = w.detach().float().contiguous()
    n, k = w.shape
    img = torch.empty(L.mignn_linear_f16x3_prep_bytes(n, k), dtype=torch.uint8, device=w.device)
    _lib.check(L.mignn_linear_f16x3_prep(_lib.ptr(w), n, k, _lib.ptr(img), img.numel(),
                                         _stream(w)), "mignn_linear_f16x3_prep")
    return img


def gin_fused_image(w: torch.Tensor) -> torch.Tensor:
    """k-permuted split-fp16 image of GIN's nn.2 weight [256, 256] for
    mignn_gin_layer_fused (mignn_gin_fused_prep)."""
    L = _lib.lib()
    w = w.detach().float().contiguous()
    img = torch.empty(L.mignn_gin_fused_prep_bytes(w.shape[1]), dtype=torch.uint8, device=w.device)
    _lib.check(L.mignn_gin_fused_prep(_lib.ptr(w), w.shape[1], _lib.ptr(img), img.numel(),
                                      _stream(w)), "mignn_gin_fused_prep")
    return img


def linear_f16x3(a: torch.Tensor, img: torch.Tensor, n: int, bias=None, *, relu=False,
                 residual=None, scale=None, shift=None, a2: Optional[torch.Tensor] = None,
                 out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """out = epi([a | a2] @ w.T) in split-fp16 MFMA arithmetic (mignn_linear_f16x3);
    `img` = f16x3_image(w), w [n, a.shape[1] + a2.shape[1]]."""
    M, K1 = a.shape
    K2 = 0 if a2 is None else a2.shape[1]
    if out is None:
        out = torch.empty((M, n), dtype=torch.float32, device=a.device)
    flags = (EPI_BIAS if bias is not None else 0) | (EPI_RESIDUAL if residual is not None else 0) \
        | (EPI_AFFINE if scale is not None else 0) | (EPI_RELU if relu else 0)
    _lib.check(_lib.lib().mignn_linear_f16x3(
        _lib.ptr(a), a.stride(0), M, K1, _lib.ptr(a2), 0 if a2 is None else a2.stride(0), K2,
        _lib.ptr(img), n, _lib.ptr(bias), _lib.ptr(residual),
        0 if residual is None else residual.stride(0), _lib.ptr(scale), _lib.ptr(shift), flags,
        _lib.ptr(out), out.stride(0), _stream(a)), "mignn_linear_f16x3")
    return out


def bn_fold(bn: nn.BatchNorm1d) -> Tuple[torch.Tensor, torch.Tensor]:
    h = bn.num_features
    dev = bn.running_mean.device
    scale = torch.empty(h, dtype=torch.float32, device=dev)
    shift = torch.empty(h, dtype=torch.float32, device=dev)
    _lib.check(_lib.lib().mignn_bn_fold(
        _lib.ptr(bn.weight), _lib.ptr(bn.bias), _lib.ptr(bn.running_mean),
        _lib.ptr(bn.running_var), float(bn.eps), h, _lib.ptr(scale), _lib.ptr(shift),
        _lib.stream(dev)), "mignn_bn_fold")
    return scale, shift


def _value_plus_edge_attr_check(a, b):
    """Shape semantics of `value_j + edge_attr` in PyG TransformerConv.message
    (ATen infer_size, same message text)."""
    ndim = max(len(a), len(b))
    for i in range(ndim - 1, -1, -1):
        off = ndim - 1 - i
        da = a[len(a) - 1 - off] if off < len(a) else 1
        db = b[len(b) - 1 - off] if off < len(b) else 1
        if da != db and da != 1 and db != 1:
            raise RuntimeError(f"The size of tensor a ({da}) must match the size of tensor b "
                               f"({db}) at non-singleton dimension {i}")
    raise NotImplementedError("TransformerConv with a broadcastable edge_attr (edge_dim=None) "
                              "is not supported")


def _versions(*ts) -> Tuple:
    return tuple((t.data_ptr(), t._version) for t in ts)


# ---------------------------------------------------------------------------
# FlowGNN
# ---------------------------------------------------------------------------

class FlowGNN(nn.Module):
    """MI355X-native FlowGNN (reference gnn_model.py:14-220)."""

    def __init__(self, input_dim: int = 3, hidden_dim: int = 128, output_dim: int = 8,
                 num_layers: int = 4, layer_type: str = "GCN", use_edge_attr: bool = True,
                 dropout: float = 0.1, use_batch_norm: bool = True):
        super().__init__()
        self.input_dim = input_dim
        self.hidden_dim = hidden_dim
        self.output_dim = output_dim
        self.num_layers = num_layers
        self.layer_type = layer_type
        self.use_edge_attr = use_edge_attr
        self.use_batch_norm = use_batch_norm
        self.input_proj = nn.Linear(input_dim, hidden_dim)
        self.gnn_layers = nn.ModuleList()
        self.batch_norms = nn.ModuleList() if use_batch_norm else None
        for _ in range(num_layers):
            if layer_type == "GCN":
                layer = GCNConv(hidden_dim, hidden_dim)
            elif layer_type == "GAT":
                layer = GATConv(hidden_dim, hidden_dim, heads=HEADS, concat=False, dropout=dropout)
            elif layer_type == "GIN":
                layer = GINConv(nn.Sequential(nn.Linear(hidden_dim, hidden_dim), nn.ReLU(),
                                              nn.Linear(hidden_dim, hidden_dim)))
            elif layer_type == "Transformer":
                layer = TransformerConv(hidden_dim, hidden_dim, heads=HEADS, concat=False,
                                        dropout=dropout)
            else:
                raise ValueError(f"Unknown layer type: {layer_type}")
            self.gnn_layers.append(layer)
            if use_batch_norm:
                self.batch_norms.append(BatchNorm(hidden_dim))
        self.output_proj = nn.Sequential(
            nn.Linear(hidden_dim, hidden_dim), nn.ReLU(), nn.Dropout(dropout),
            nn.Linear(hidden_dim, hidden_dim), nn.ReLU(), nn.Dropout(dropout),
            nn.Linear(hidden_dim, hidden_dim // 2), nn.ReLU(),
            nn.Linear(hidden_dim // 2, output_dim))
        self.dropout = nn.Dropout(dropout)
        self.precision = os.environ.get("MIGNN_PRECISION", "f16x3")
        # internal locality order of the nodes: "auto" (meshes of >= 2^20
        # nodes with 3-D cell-centre features), "1" always, "0" never
        self.reorder = os.environ.get("MIGNN_REORDER", "auto")
        # split-fp16 GCN layer kernel at H in {64, 128}: "win" (the window
        # kernel over the column order, csrc/gcn_win.hip), "ring" (the
        # persistent ring kernel, csrc/gcn_ring.hip), "pc" (the producer /
        # consumer kernel, csrc/gcn_f16x3.hip: any node order, no plan) or
        # "auto" (GCN_KERNEL_AUTO per H); read once here, not per forward
        self.gcn_kernel = os.environ.get("MIGNN_GCN_KERNEL", "auto")
        if self.gcn_kernel not in ("ring", "pc", "win", "auto"):
            raise ValueError(
                f"MIGNN_GCN_KERNEL must be auto, win, ring or pc, got {self.gcn_kernel!r}")
        # kernel-route switches (A/B studies; the defaults are the measured
        # fastest routes), read once at construction -- plain attributes after
        # that, never environment lookups inside forward:
        #   fuse_layer0     input_proj composed into layer 0 (MIGNN_FUSE_LAYER0)
        #   gat_coords      GAT layer 0 collapsed to 3-vectors (MIGNN_GAT_COORDS)
        #   gat_next_logits a GAT layer's epilogue forms the next layer's
        #                   logits (MIGNN_GAT_NEXT_LOGITS)
        #   fused256        H = 256 fused layer / head kernels: "1", "0",
        #                   "layer" or "head" (MIGNN_FUSED256)
        self.fuse_layer0 = os.environ.get("MIGNN_FUSE_LAYER0", "1") == "1"
        #   gcn_codes       GCN H = 128 on the window kernel: layer 0 writes 32-B
        #                   row codes and layer 1 expands them (MIGNN_GCN_CODES)
        self.gcn_codes = os.environ.get("MIGNN_GCN_CODES", "1") == "1"
        # after every eval forward, read the device's sticky in-kernel error word
        # and raise if a bounded wait ran out (costs a device sync; off by
        # default -- bench.py and the tests check it themselves)
        self.check_device_errors = os.environ.get("MIGNN_CHECK_ERRORS", "0") == "1"
        self.gat_coords = os.environ.get("MIGNN_GAT_COORDS", "1") == "1"
        self.gat_next_logits = os.environ.get("MIGNN_GAT_NEXT_LOGITS", "1") == "1"
        self.fused256 = os.environ.get("MIGNN_FUSED256", "1")
        if self.fused256 not in ("0", "1", "layer", "head"):
            raise ValueError(f"MIGNN_FUSED256 must be 0, 1, layer or head, got {self.fused256!r}")
        self._csr = _CsrCache()
        self._prep: Dict[Tuple, object] = {}

    # ------------------------------------------------------------------ API
    def predict_fields(self, output: torch.Tensor) -> dict:
        """gnn_model.py:199-220."""
        fields = {"U": output[:, :3], "p": output[:, 3:4], "k": output[:, 4:5],
                  "epsilon": output[:, 5:6], "nut": output[:, 6:7]}
        if output.shape[1] > 7:
            fields["residual"] = output[:, 7:8]
        return fields

    def forward(self, x: torch.Tensor, edge_index: torch.Tensor,
                edge_attr: Optional[torch.Tensor] = None,
                batch: Optional[torch.Tensor] = None) -> torch.Tensor:
        num_nodes = x.shape[0]
        # gnn_model.py:126-127
        if edge_index.dim() != 2 or edge_index.shape[0] != 2:
            raise ValueError(f"edge_index must have shape [2, num_edges], got {edge_index.shape}")
        self._check_runtime(x, edge_index)
        E = edge_index.shape[1]
        # gnn_model.py:152-156 (shape-only: invalid-edge filtering keeps counts aligned)
        if edge_attr is not None and E > 0 and edge_attr.shape[0] != E:
            raise ValueError(f"edge_attr must have {E} entries, got {edge_attr.shape[0]}")
        H = self.hidden_dim
        if self.training:
            return self._forward_train(x, edge_index, edge_attr)
        out = torch.empty((num_nodes, self.output_dim), dtype=torch.float32, device=x.device)
        if num_nodes == 0:
            return out
        xin = x.contiguous().float() if (x.dtype != torch.float32 or not x.is_contiguous()) else x
        buf_a = torch.empty((num_nodes, H), dtype=torch.float32, device=x.device)
        buf_b = torch.empty_like(buf_a)
        mode = CSR_ONE_SELF_LOOP if self.layer_type in ("GCN", "GAT") else CSR_VERBATIM
        pos = xin if self._use_reorder(xin) else None
        csr = self._csr.get(edge_index, num_nodes, mode, pos, cols=self._column_order())
        self._prepare_plans(csr, 0, num_nodes)
        cur, nxt = buf_a, buf_b
        first = 0
        kind = self._layer0_kind(edge_attr)
        if kind == "gcn" and self._use_gcn_codes(csr):
            # layers 0 and 1 through the row codes: layer 0's [N, H] rows are
            # never written (mignn_gcn_layer0_codes + mignn_gcn_layer_win_codes)
            try:
                self._gcn_layers01_codes(csr, self._coords(xin, csr), num_nodes, cur)
            except RuntimeError as e:
                raise self._layer_error(0, e, num_nodes, edge_index, xin, edge_attr) from e
            first = 2
        elif kind is not None:
            # input_proj composed into layer 0, from the coordinates
            try:
                self._layer0(kind, csr, self._coords(xin, csr), 0, num_nodes, cur)
            except RuntimeError as e:
                raise self._layer_error(0, e, num_nodes, edge_index, xin, edge_attr) from e
            first = 1
        else:
            # input_proj (gnn_model.py:159), gathered into the CSR's node order
            self._input_proj(xin, cur, rows=csr.perm)
        # GAT: a layer's epilogue forms the next layer's logits (no logit GEMV launch)
        chain = self.layer_type == "GAT" and self.precision == "f16x3" and self.gat_next_logits
        lg_cur = None
        for i, layer in enumerate(self.gnn_layers):
            if i < first:
                continue
            try:
                if self.layer_type == "Transformer" and edge_attr is not None:
                    # PyG TransformerConv.message adds a non-None edge_attr to value_j
                    # ([E, heads, C] + [E, d]); reproduce the resulting torch error.
                    _value_plus_edge_attr_check((E, HEADS, H), tuple(edge_attr.shape))
                lg_next = None
                if chain and i + 1 < len(self.gnn_layers):
                    lg_next = torch.empty((num_nodes, 2 * HEADS), dtype=torch.float32,
                                          device=x.device)
                self._layer(i, layer, csr, cur, nxt, 0, num_nodes, logits=lg_cur,
                            logits_next=lg_next)
                lg_cur = lg_next
            except RuntimeError as e:
                raise self._layer_error(i, e, num_nodes, edge_index, cur, edge_attr) from e
            cur, nxt = nxt, cur
        self._output_mlp(cur, nxt, out, rows=csr.perm, inv=csr.inv)
        if self.check_device_errors:
            _lib.check_device_errors("FlowGNN.forward")
        return out

    # ------------------------------------------------------------- internals
    def _check_runtime(self, x, edge_index):
        if x.device.type != "cuda" or edge_index.device.type != "cuda":
            raise RuntimeError(
                "mignn FlowGNN runs on ROCm devices only (no CPU path): move the model and the "
                "graph to 'cuda' (HIP).")
        if self.input_proj.weight.device != x.device:
            raise RuntimeError(f"model is on {self.input_proj.weight.device}, input on {x.device}")
        # every forward (a few attribute reads): parameters swapped in by
        # load_state_dict(assign=True) or direct assignment bypass _apply
        for p in self.parameters():
            if p.dtype != torch.float32:
                raise RuntimeError("mignn FlowGNN computes in fp32; parameters must be float32")
        if self.hidden_dim % 8 != 0:
            raise RuntimeError("mignn FlowGNN requires hidden_dim % 8 == 0")
        if self.precision not in ("f32", "f16x3"):
            raise ValueError(f"precision must be 'f32' or 'f16x3', got {self.precision!r}")

    def _forward_train(self, x, edge_index, edge_attr):
        """model.train() forward (gnn_model.py:159-195) as autograd ops over HIP
        kernels (mignn.train_ops): batch-statistics BN with running-stat updates,
        dropout, and a backward for every parameter."""
        num_nodes = x.shape[0]
        if num_nodes == 0:
            raise ValueError("training forward on an empty graph")
        H = self.hidden_dim
        if self.layer_type in ("GAT", "Transformer") and H > 256:
            raise NotImplementedError(
                f"mignn training path: {self.layer_type} layers support hidden_dim <= 256 "
                f"(got {H}); eval mode has no such limit")
        if self.use_batch_norm and H > 512:
            raise NotImplementedError(
                f"mignn training path: BatchNorm statistics support hidden_dim <= 512 (got {H})")
        try:
            return self._forward_train_impl(x, edge_index, edge_attr)
        finally:
            # the BN kernels update running_mean / running_var in place through
            # raw pointers (their _version does not move): drop every eval
            # image derived from them (BN folds, layer-0 coefficients)
            if self.use_batch_norm:
                self._prep = {k: v for k, v in self._prep.items() if k[0] not in ("bn", "layer0")}

    def _forward_train_impl(self, x, edge_index, edge_attr):
        num_nodes = x.shape[0]
        xin = x.contiguous().float() if (x.dtype != torch.float32 or not x.is_contiguous()) else x
        mode = CSR_ONE_SELF_LOOP if self.layer_type in ("GCN", "GAT") else CSR_VERBATIM
        csr = self._csr.get(edge_index, num_nodes, mode)
        csr_t = self._csr.get(edge_index, num_nodes, mode | CSR_TRANSPOSE)
        h = T.linear(xin, self.input_proj.weight, self.input_proj.bias)
        p = float(self.dropout.p)
        for i, layer in enumerate(self.gnn_layers):
            try:
                if self.layer_type == "GCN":
                    z = T.gcn_residual(h, layer.lin.weight, layer.bias, csr, csr_t)
                elif self.layer_type == "GAT":
                    # per-step weight images (O(heads H^2), differentiable):
                    # wlog = [W_k^T att_src_k | W_k^T att_dst_k], wcat = head-mean blocks
                    heads, C = layer.heads, layer.out_channels
                    W = layer.lin.weight.view(heads, C, -1)
                    wlog = torch.cat([torch.einsum("hck,hc->hk", W, layer.att_src.view(heads, C)),
                                      torch.einsum("hck,hc->hk", W, layer.att_dst.view(heads, C))])
                    wcat = W.permute(1, 0, 2).reshape(C, heads * W.shape[2]) / heads
                    z = T.gat_residual(h, wlog, wcat, layer.bias, csr, csr_t, heads,
                                       layer.negative_slope, float(layer.dropout))
                elif self.layer_type == "Transformer":
                    if edge_attr is not None:   # PyG adds edge_attr to value_j (see eval)
                        _value_plus_edge_attr_check((edge_index.shape[1], HEADS, self.hidden_dim),
                                                    tuple(edge_attr.shape))
                    wqkv = torch.cat([layer.lin_query.weight, layer.lin_key.weight,
                                      layer.lin_value.weight])
                    bqkv = torch.cat([layer.lin_query.bias, layer.lin_key.bias,
                                      layer.lin_value.bias])
                    z = T.transformer_residual(h, wqkv, bqkv, layer.lin_skip.weight,
                                               layer.lin_skip.bias, csr, csr_t, layer.heads,
                                               float(layer.dropout))
                else:   # GIN: nn = Seq(Linear, ReLU, Linear), eps buffer
                    l1, l2 = layer.nn[0], layer.nn[2]
                    eps = self._cached("eps", i, (layer.eps,),
                                       lambda: float(layer.eps.reshape(-1)[0]))
                    z = T.gin_residual(h, l1.weight, l1.bias, l2.weight, l2.bias, eps, csr,
                                       csr_t)
            except RuntimeError as e:
                raise self._layer_error(i, e, num_nodes, edge_index, h, edge_attr) from e
            bn = self.batch_norms[i].module if self.use_batch_norm else None
            h = T.bn_relu_dropout(z, bn, p)
        mods = list(self.output_proj)
        k = 0
        while k < len(mods):
            m = mods[k]
            if isinstance(m, nn.Linear):
                relu = k + 1 < len(mods) and isinstance(mods[k + 1], nn.ReLU)
                h = T.linear(h, m.weight, m.bias, relu=relu)
                k += 2 if relu else 1
            elif isinstance(m, nn.Dropout):
                h = T.dropout(h, float(m.p))
                k += 1
            else:
                raise NotImplementedError(f"output_proj module {type(m).__name__}")
        return h

    def _layer_error(self, i, e, num_nodes, edge_index, x, edge_attr):
        """gnn_model.py:175-181, reporting the edge list the convs saw: after
        the silent filtering of invalid indices (:133-141) and the all-invalid
        self-loop fallback (:144-149), as the reference does."""
        ei = edge_index
        if ei.shape[1] > 0:
            valid = (ei[0] >= 0) & (ei[0] < num_nodes) & (ei[1] >= 0) & (ei[1] < num_nodes)
            if not bool(valid.all()):
                ei = ei[:, valid]
                if edge_attr is not None and edge_attr.shape[0] > 0:
                    edge_attr = edge_attr[valid]
            if ei.shape[1] == 0:
                ei = torch.arange(num_nodes, device=ei.device).repeat(2, 1)
                if edge_attr is not None:
                    edge_attr = torch.zeros((num_nodes, edge_attr.shape[1]),
                                            dtype=edge_attr.dtype, device=edge_attr.device)
        E = ei.shape[1]
        if E > 0:
            rng = f"[{ei.min().item()}, {ei.max().item()}]"
        else:
            rng = "[N/A, N/A]"
        return RuntimeError(
            f"Message passing failed in layer {i} ({self.layer_type}): {str(e)}\n"
            f"  num_nodes: {num_nodes}, num_edges: {E if E > 0 else 0}\n"
            f"  edge_index range: {rng}\n"
            f"  x shape: {x.shape}, edge_attr shape: "
            f"{edge_attr.shape if edge_attr is not None else 'None'}")

    def _layer0_kind(self, edge_attr=None) -> Optional[str]:
        """The composition of input_proj into layer 0 that runs from the
        node coordinates (no [N, H] input_proj output, no layer-0 halo when
        sharded), or None: input_proj writes [N, H] and layer 0 runs as the
        others.  gcn: mignn_gcn_layer0_coords; transformer:
        mignn_transformer_layer0_coords; gat: mignn_gat_layer0_coords
        (collapsed to 3-vectors), gat_mfma: mignn_gat_layer0_fused; gin (H =
        256): mignn_gin_layer0_fused."""
        if self._fuse_layer0():
            return "gcn"
        if self._fuse_tf_layer0(edge_attr):
            return "transformer"
        if self._fuse_gat_layer0():
            return "gat" if self.gat_coords else "gat_mfma"
        if self._fuse_gin_layer0():
            return "gin"
        return None

    def _layer0(self, kind: str, csr: Csr, pos: torch.Tensor, rb: int, re: int, out,
                logits_next=None):
        """Layer 0 (input_proj composed in) for rows [rb, re) of the CSR from
        pos [rows, input_dim] (coordinates of every row the CSR references, in
        its node order).  logits_next (kind gat only): also the next GAT
        layer's logits of the rows, from the same kernel."""
        if kind == "gcn":
            self._gcn_layer0(csr, pos, rb, re, out)
        elif kind == "transformer":
            self._tf_layer0(csr, pos, rb, re, out)
        elif kind == "gat":
            self._gat_layer0(csr, pos, rb, re, out, logits_next)
        elif kind == "gat_mfma":
            self._gat_layer0_mfma(csr, pos, rb, re, out)
        elif kind == "gin":
            self._gin_layer0(csr, pos, rb, re, out)
        else:
            raise ValueError(f"unknown layer-0 composition {kind!r}")

    def _fuse_layer0(self) -> bool:
        return (self.fuse_layer0 and self.layer_type == "GCN"
                and self.num_layers > 0 and 1 <= self.input_dim <= 4
                and self.hidden_dim in (4, 8, 16, 32, 64, 128, 256))

    def _fuse_tf_layer0(self, edge_attr) -> bool:
        return (self.fuse_layer0 and self.layer_type == "Transformer"
                and edge_attr is None and self.num_layers > 0 and 1 <= self.input_dim <= 3
                and self.hidden_dim in (64, 128, 256) and self.precision == "f16x3")

    def _tf_layer0_tables(self):
        """fp64 composition of input_proj into TransformerConv layer 0
        (mignn_transformer_layer0_coords): GT [4][12] = G_h | g_h and T [H][20]
        = A_0..A_3 | e_0..e_3 | B | d, bias, residual and BN folded in."""
        layer = self.gnn_layers[0]
        ts = [layer.lin_query.weight, layer.lin_query.bias, layer.lin_key.weight,
              layer.lin_key.bias, layer.lin_value.weight, layer.lin_value.bias,
              layer.lin_skip.weight, layer.lin_skip.bias, self.input_proj.weight,
              self.input_proj.bias]
        if self.use_batch_norm:
            bn = self.batch_norms[0].module
            ts += [bn.weight, bn.bias, bn.running_mean, bn.running_var]

        def make():
            d64 = lambda t: t.detach().double()  # noqa: E731
            heads, C = layer.heads, layer.out_channels
            H, D = self.hidden_dim, self.input_dim
            Wq = d64(layer.lin_query.weight).view(heads, C, -1)
            Wk = d64(layer.lin_key.weight).view(heads, C, -1)
            Wv = d64(layer.lin_value.weight).view(heads, C, -1)
            bq = d64(layer.lin_query.bias).view(heads, C)
            bv = d64(layer.lin_value.bias).view(heads, C)
            M = torch.einsum("hck,hcq->hkq", Wk, Wq)                    # qt_h = M_h x + m_h
            mb = torch.einsum("hck,hc->hk", Wk, bq)
            Win = torch.zeros(H, 3, dtype=torch.float64, device=Wq.device)
            Win[:, :D] = d64(self.input_proj.weight)
            bin_ = d64(self.input_proj.bias)
            G = torch.einsum("ka,hkq,qb->hab", Win, M, Win)               # [h, 3, 3]
            g = torch.einsum("ka,hk->ha", Win, torch.einsum("hkq,q->hk", M, bin_) + mb)
            gt = torch.cat([G.reshape(heads, 9), g], 1)                    # [4, 12]
            A = torch.einsum("chk,ka->hca", Wv.permute(1, 0, 2), Win) / heads   # [h, C, 3]
            e = (torch.einsum("chk,k->hc", Wv.permute(1, 0, 2), bin_) + bv) / heads
            Ws = d64(layer.lin_skip.weight)
            B = Ws @ Win + Win
            dd = Ws @ bin_ + d64(layer.lin_skip.bias) + bin_
            if self.use_batch_norm:
                bn = self.batch_norms[0].module
                sc = d64(bn.weight) / torch.sqrt(d64(bn.running_var) + bn.eps)
                sh = d64(bn.bias) - d64(bn.running_mean) * sc
                A = A * sc[None, :, None]
                e = e * sc[None, :]
                B = B * sc[:, None]
                dd = dd * sc + sh
            T = torch.cat([A.permute(1, 0, 2).reshape(C, 3 * heads), e.t(), B, dd[:, None]], 1)
            return T.float().contiguous(), gt.float().contiguous()
        return self._cached("tf0", 0, ts, make)

    def _tf_layer0(self, csr: Csr, pos, rb, re, out):
        T, gt = self._tf_layer0_tables()
        P = _lib.ptr
        _lib.check(_lib.lib().mignn_transformer_layer0_coords(
            P(csr.row_ptr), P(csr.col), P(pos), pos.stride(0), self.input_dim, rb, re,
            self.hidden_dim, HEADS, 1.0 / math.sqrt(self.hidden_dim), P(T), P(gt), 1, P(out),
            out.stride(0), _stream(pos)), "mignn_transformer_layer0_coords")

    def _fuse_gat_layer0(self) -> bool:
        # (the MFMA form, gat_coords off, has kernels for H in {64, 128} only;
        # at H = 256 it is the two-step route then)
        return (self.fuse_layer0 and self.layer_type == "GAT"
                and self.num_layers > 0 and 1 <= self.input_dim <= 3
                and (self.hidden_dim in (64, 128) or (self.hidden_dim == 256 and self.gat_coords))
                and self.precision == "f16x3")

    def _gat_layer0(self, csr: Csr, pos, rb, re, out, logits_next=None):
        """input_proj + GAT layer 0 + residual + BN + ReLU collapsed to
        3-vectors (mignn_gat_layer0_coords): logits through lw = [wlog W_in |
        wlog b_in], per head P = sum alpha pos_j and S = sum alpha, output
        sum_k (Wcat_k W_in P_k + S_k Wcat_k b_in) + bias + x_i, BN folded
        (fp64 composition)."""
        layer = self.gnn_layers[0]
        H, D = self.hidden_dim, self.input_dim
        ts = [layer.lin.weight, layer.att_src, layer.att_dst, layer.bias,
              self.input_proj.weight, self.input_proj.bias]
        if self.use_batch_norm:
            bn = self.batch_norms[0].module
            ts += [bn.weight, bn.bias, bn.running_mean, bn.running_var]

        def make():
            d64 = lambda t: t.detach().double()  # noqa: E731
            heads, C = layer.heads, layer.out_channels
            W = d64(layer.lin.weight).view(heads, C, -1)                    # [h, c, k]
            vs = torch.einsum("hck,hc->hk", W, d64(layer.att_src).view(heads, C))
            vd = torch.einsum("hck,hc->hk", W, d64(layer.att_dst).view(heads, C))
            wlog = torch.cat([vs, vd], 0)                                   # [8, H]
            Win = torch.zeros(H, 3, dtype=torch.float64, device=W.device)
            Win[:, :D] = d64(self.input_proj.weight)
            bin_ = d64(self.input_proj.bias)
            lw = torch.zeros(2 * heads, 4, dtype=torch.float64, device=W.device)
            lw[:, :3] = wlog @ Win
            lw[:, 3] = wlog @ bin_
            A = torch.einsum("hck,ka->hca", W, Win) / heads                 # [h, C, 3]
            e = torch.einsum("hck,k->hc", W, bin_) / heads                   # [h, C]
            B = Win.clone()                                                 # residual x_i
            dd = d64(layer.bias) + bin_
            if self.use_batch_norm:
                bn = self.batch_norms[0].module
                sc = d64(bn.weight) / torch.sqrt(d64(bn.running_var) + bn.eps)
                sh = d64(bn.bias) - d64(bn.running_mean) * sc
                A = A * sc[None, :, None]
                e = e * sc[None, :]
                B = B * sc[:, None]
                dd = dd * sc + sh
            T = torch.cat([A.permute(1, 0, 2).reshape(C, 3 * heads), e.t(), B, dd[:, None]], 1)
            return T.float().contiguous(), lw.float().contiguous()
        T, lw = self._cached("gat0c", 0, ts, make)
        wlog_n = None
        if logits_next is not None:
            nl = self.gnn_layers[1]
            wlog_n, _ = self._cached("gat", 1, (nl.lin.weight, nl.att_src, nl.att_dst),
                                     lambda: self._gat_weights(nl))
        P = _lib.ptr
        _lib.check(_lib.lib().mignn_gat_layer0_coords(
            P(csr.row_ptr), P(csr.col), P(pos), pos.stride(0), D, rb, re, H, HEADS,
            float(layer.negative_slope), P(T), P(lw), 1, P(out), out.stride(0), P(wlog_n),
            P(logits_next), _stream(pos)), "mignn_gat_layer0_coords")

    def _gat_layer0_mfma(self, csr: Csr, pos, rb, re, out):
        """input_proj + GAT layer 0 + residual + BN + ReLU in one kernel: logits
        through [wlog W_in | wlog b_in], per head P = sum alpha pos_j and S =
        sum alpha, weighted sums W_in P + S b_in (fp64-composed weights)."""
        layer = self.gnn_layers[0]
        H, D = self.hidden_dim, self.input_dim
        ts = (layer.lin.weight, layer.att_src, layer.att_dst, self.input_proj.weight,
              self.input_proj.bias)

        def make():
            heads, C = layer.heads, layer.out_channels
            W = layer.lin.weight.detach().double().view(heads, C, -1)
            vs = torch.einsum("hck,hc->hk", W, layer.att_src.detach().double().view(heads, C))
            vd = torch.einsum("hck,hc->hk", W, layer.att_dst.detach().double().view(heads, C))
            wlog = torch.cat([vs, vd], 0)                                   # [8, H]
            lw = torch.zeros(2 * heads, 4, dtype=torch.float64, device=W.device)
            lw[:, :D] = wlog @ self.input_proj.weight.detach().double()
            lw[:, 3] = wlog @ self.input_proj.bias.detach().double()
            return lw.float().contiguous()
        lw = self._cached("gat0", 0, ts, make)
        _, wcat = self._cached("gat", 0, (layer.lin.weight, layer.att_src, layer.att_dst),
                               lambda: self._gat_weights(layer))
        img = self._img("w_gat", 0, (layer.lin.weight,), wcat)
        scale, shift = self._bn(0)
        epi = EPI_BIAS | EPI_RESIDUAL | (EPI_AFFINE if scale is not None else 0) | EPI_RELU
        P = _lib.ptr
        _lib.check(_lib.lib().mignn_gat_layer0_fused(
            P(csr.row_ptr), P(csr.col), P(pos), pos.stride(0), D, rb, re, H,
            float(layer.negative_slope), P(self.input_proj.weight), P(self.input_proj.bias), P(lw),
            P(img), P(layer.bias), P(scale), P(shift), epi, P(out), out.stride(0), _stream(pos)),
            "mignn_gat_layer0_fused")

    def _fuse_gin_layer0(self) -> bool:
        return (self.fuse_layer0 and self.layer_type == "GIN"
                and self.num_layers > 0 and 1 <= self.input_dim <= 3 and self.hidden_dim == 256
                and self._fused256())

    def _gin_layer0(self, csr: Csr, pos, rb, re, out):
        """input_proj + GIN layer 0 + residual + BN + ReLU in one kernel:
        a_i = W_in (sum_j pos_j + (1+eps) pos_i) + (deg_i + 1 + eps) b_in."""
        layer = self.gnn_layers[0]
        nn0, nn2 = layer.nn[0], layer.nn[2]
        eps = self._cached("eps", 0, (layer.eps,), lambda: float(layer.eps.reshape(-1)[0]))
        img1 = self._cached("w_gin0", 0, (nn0.weight,), lambda: f16x3_image(nn0.weight))
        img2 = self._cached("w_gin2p", 0, (nn2.weight,), lambda: gin_fused_image(nn2.weight))
        scale, shift = self._bn(0)
        epi = EPI_BIAS | EPI_RESIDUAL | (EPI_AFFINE if scale is not None else 0) | EPI_RELU
        P = _lib.ptr
        _lib.check(_lib.lib().mignn_gin_layer0_fused(
            P(csr.row_ptr), P(csr.col), P(pos), pos.stride(0), self.input_dim, rb, re,
            256, eps, P(self.input_proj.weight), P(self.input_proj.bias), P(img1), P(nn0.bias),
            P(img2), P(nn2.bias), P(scale), P(shift), epi, P(out), out.stride(0), _stream(pos)),
            "mignn_gin_layer0_fused")

    def _layer0_coef(self):
        """A = diag(sc) W_in, B = diag(sc) W W_in, d = sc*(W b_in), e = sc*(b_in + b) + sh
        per output column, fp64-composed (gcn_layer0.hip)."""
        layer = self.gnn_layers[0]
        ts = [self.input_proj.weight, self.input_proj.bias, layer.lin.weight, layer.bias]
        if self.use_batch_norm:
            bn = self.batch_norms[0].module
            ts += [bn.weight, bn.bias, bn.running_mean, bn.running_var]

        def make():
            Win, bin_ = (t.detach().double() for t in ts[:2])
            W, b = (t.detach().double() for t in ts[2:4])
            if self.use_batch_norm:
                bn = self.batch_norms[0].module
                sc = bn.weight.double() / torch.sqrt(bn.running_var.double() + bn.eps)
                sh = bn.bias.double() - bn.running_mean.double() * sc
            else:
                sc = torch.ones_like(b)
                sh = torch.zeros_like(b)
            A = sc[:, None] * Win
            B = sc[:, None] * (W @ Win)
            d = sc * (W @ bin_)
            e = sc * (bin_ + b) + sh
            return torch.cat([A, B, d[:, None], e[:, None]], 1).float().contiguous()
        return self._cached("layer0", 0, ts, make)

    def _coords(self, x, csr: Csr):
        """The node features (coordinates) in the CSR's node order."""
        if csr.perm is None:
            return x
        D = self.input_dim
        # (3-D coordinates into 16-B rows: the layer-0 kernels gather a
        # neighbour's coordinates with one 16-B load; the 4th column unread)
        ld = 4 if D == 3 else D
        pos = torch.empty((x.shape[0], ld), dtype=torch.float32, device=x.device)
        _lib.check(_lib.lib().mignn_rows_gather(
            _lib.ptr(x), x.stride(0), _lib.ptr(csr.perm), x.shape[0], D, _lib.ptr(pos), ld,
            _stream(x)), "mignn_rows_gather")
        return pos[:, :D]

    def _gcn_layer0(self, csr: Csr, pos, rb, re, out):
        _lib.check(_lib.lib().mignn_gcn_layer0_coords(
            _lib.ptr(csr.row_ptr), _lib.ptr(csr.col), _lib.ptr(csr.ew), _lib.ptr(pos),
            pos.stride(0), self.input_dim, rb, re, _lib.ptr(self._layer0_coef()), self.hidden_dim,
            _lib.ptr(out), out.stride(0), _stream(pos)), "mignn_gcn_layer0_coords")

    def _use_gcn_codes(self, csr: Csr) -> bool:
        """Layers 0 and 1 of a GCN stack through layer 0's row codes: the
        window kernel at H = 128 on this CSR, 3-D coordinates, >= 2 layers."""
        return (self.gcn_codes and self.layer_type == "GCN" and self.hidden_dim == 128
                and self.input_dim == 3 and self.num_layers >= 2 and self.precision == "f16x3"
                and self._gcn_kernel(128, csr) == "win")

    def _gcn_layers01_codes(self, csr: Csr, pos, n: int, out):
        """Layer 0 as row codes (c_i, C_i, s_i) [n, 8], then layer 1 by the
        window kernel expanding every row it reads from them with layer 0's
        coefficients -- the same rows, bitwise, without layer 0's [n, H]
        write and layer 1's re-read of it."""
        codes = torch.empty((n, 8), dtype=torch.float32, device=pos.device)
        self._gcn_layer0_codes(csr, pos, 0, n, codes)
        self._gcn_layer1_codes(csr, codes, 0, n, out)

    def _gcn_layer0_codes(self, csr: Csr, pos, rb: int, re: int, codes):
        """Layer 0's row codes (c_i, C_i, s_i) of rows [rb, re) into codes [*, 8]."""
        _lib.check(_lib.lib().mignn_gcn_layer0_codes(
            _lib.ptr(csr.row_ptr), _lib.ptr(csr.col), _lib.ptr(csr.ew), _lib.ptr(pos),
            pos.stride(0), self.input_dim, rb, re, _lib.ptr(codes), codes.stride(0),
            _stream(pos)), "mignn_gcn_layer0_codes")

    def _gcn_layer1_codes(self, csr: Csr, codes, rb: int, re: int, out):
        """Layer 1 of rows [rb, re) by the window kernel's codes form: every
        row it reads expanded from `codes` (the rows of every referenced node
        present, a shard's ghosts included)."""
        P = _lib.ptr
        layer = self.gnn_layers[1]
        scale, shift = self._bn(1)
        epi = EPI_BIAS | EPI_RESIDUAL | (EPI_AFFINE if scale is not None else 0) | EPI_RELU
        plan = csr.win_plan(128, rb, re)
        _lib.check(_lib.lib().mignn_gcn_layer_win_codes(
            P(plan), P(csr.row_ptr), P(csr.col), P(csr.ew), P(codes), codes.stride(0), rb, re, 128,
            P(self._layer0_coef()), P(layer.lin.weight), P(layer.bias), P(scale), P(shift), epi,
            P(out), out.stride(0), _stream(codes)), "mignn_gcn_layer_win_codes")

    def _gcn_kernel(self, H: int, csr: Optional["Csr"] = None) -> str:
        """The GCN layer kernel at width H; with `csr`: the kernel for that
        graph -- under "auto" the window kernel only on a CSR in the column
        order (a shard's block-ordered range takes GCN_BLOCK_ORDER instead)."""
        k = self.gcn_kernel if self.gcn_kernel != "auto" else GCN_KERNEL_AUTO.get(H, "pc")
        if k == "win" and self.gcn_kernel == "auto" and csr is not None and csr.order_info is None:
            k = GCN_BLOCK_ORDER.get(H, "pc")
        return k

    def _column_order(self) -> bool:
        """The locality order of this model's graphs: the column order when
        its GCN layers run the window kernel (one z-plane of an 8x8 column
        per tile), the block order otherwise."""
        H = self.hidden_dim
        return (self.layer_type == "GCN" and H in (64, 128) and self.precision == "f16x3"
                and self._gcn_kernel(H) == "win")

    def _prepare_plans(self, csr: "Csr", row_begin: int, row_end: int):
        """Build the per-graph plan of the GCN layer kernel before the layer
        loop (part of the graph setup, with the CSR; not inside a layer)."""
        H = self.hidden_dim
        if self.layer_type != "GCN" or H not in (64, 128) or self.precision != "f16x3":
            return
        kern = self._gcn_kernel(H, csr)
        if kern == "win":
            csr.win_plan(H, row_begin, row_end)
        elif kern == "ring":
            csr.ring_plan(H, row_begin, row_end)

    def _use_reorder(self, x) -> bool:
        if self.reorder not in ("auto", "0", "1"):
            raise ValueError(f"MIGNN_REORDER must be auto, 0 or 1, got {self.reorder!r}")
        if self.reorder == "0" or x.shape[1] < 3:
            return False
        return self.reorder == "1" or x.shape[0] >= (1 << 20)

    def _input_proj(self, x, out, rows=None):
        w, b = self.input_proj.weight, self.input_proj.bias
        if self.input_dim <= 8:
            _lib.check(_lib.lib().mignn_input_proj_rows(
                _lib.ptr(x), x.shape[0], self.input_dim, _lib.ptr(rows), _lib.ptr(w), _lib.ptr(b),
                self.hidden_dim, _lib.ptr(out), out.stride(0), _stream(x)), "mignn_input_proj")
        else:
            linear(x if rows is None else x[rows.long()], w, b, out=out)

    def _bn(self, i):
        if not self.use_batch_norm:
            return None, None
        bn = self.batch_norms[i].module
        key = ("bn", i) + _versions(bn.weight, bn.bias, bn.running_mean, bn.running_var)
        hit = self._prep.get(key)
        if hit is None:
            self._prep = {k: v for k, v in self._prep.items() if k[:2] != ("bn", i)}
            hit = self._prep[key] = bn_fold(bn)
        return hit

    def _cached(self, tag, i, tensors, make):
        key = (tag, i) + _versions(*tensors)
        hit = self._prep.get(key)
        if hit is None:
            self._prep = {k: v for k, v in self._prep.items() if k[:2] != (tag, i)}
            with torch.no_grad():
                hit = self._prep[key] = make()
        return hit

    def _img(self, tag, i, srcs, w):
        """The split-fp16 image of W = w (derived from the parameters `srcs`,
        cached per parameter version) when the transform runs in split fp16
        (precision "f16x3" and a shape the fused kernels leave over: k or n >
        128, n >= 64); None: exact fp32 MFMA."""
        n, k = w.shape
        if self.precision == "f16x3" and n >= 64 and (n > 128 or k > 128):
            return self._cached(tag, i, srcs, lambda: f16x3_image(w))
        return None

    def _fused256(self, part: str = "layer") -> bool:
        """The H = 256 fused kernels (split-fp16 arithmetic) -- the default in
        f16x3 precision: GIN / GCN / TransformerConv layers (mignn_gin_layer_fused,
        mignn_gcn_layer_fused, mignn_transformer_layer_fused; part "layer") and
        the output head (mignn_mlp_head at h = 256; part "head").
        MIGNN_FUSED256=0 runs the aggregate + GEMM launches for both, "layer" /
        "head" keeps only that part fused."""
        v = self.fused256
        return self.precision == "f16x3" and (v == "1" or v == part)

    def _mm(self, tag, i, srcs, w, a, bias=None, **kw):
        """Node transform by W = w: split-fp16 GEMM (mignn_linear_f16x3) or
        exact fp32 MFMA (mignn_linear), as _img decides."""
        img = self._img(tag, i, srcs, w)
        if img is not None:
            return linear_f16x3(a, img, w.shape[0], bias, **kw)
        return linear(a, w, bias, **kw)

    def _layer(self, i, layer, csr: Csr, x, out, rb: int, re: int, logits=None,
               logits_next=None):
        """One conv + residual + BN + ReLU (gnn_model.py:162-192) for rows [rb, re).
        `x` holds every row the CSR references (own rows + halo rows).  GAT:
        `logits` [rows, 2*heads] of every referenced row, precomputed by a
        sharded caller (mignn.dist); None: computed here for all rows of x."""
        H = self.hidden_dim
        L = _lib.lib()
        st = _stream(x)
        scale, shift = self._bn(i)
        epi = EPI_BIAS | EPI_RESIDUAL | (EPI_AFFINE if scale is not None else 0) | EPI_RELU
        P = _lib.ptr
        n = re - rb
        if n <= 0:
            return
        if self.layer_type == "GCN":
            w, b = layer.lin.weight, layer.bias
            kern = self._gcn_kernel(H, csr)
            if H in (64, 128) and self.precision == "f16x3" and kern == "win":
                # the hot kernel: window walk over the CSR's window plan
                plan = csr.win_plan(H, rb, re)
                _lib.check(L.mignn_gcn_layer_win(
                    P(plan), P(csr.row_ptr), P(csr.col), P(csr.ew), P(x), x.stride(0), rb, re, H,
                    P(w), P(b), P(scale), P(shift), epi, P(out), out.stride(0), st),
                    "mignn_gcn_layer_win")
            elif H in (64, 128) and self.precision == "f16x3" and kern == "ring":
                # the hot kernel: persistent ring over the CSR's ring plan
                plan = csr.ring_plan(H, rb, re)
                _lib.check(L.mignn_gcn_layer_ring(
                    P(plan), P(csr.row_ptr), P(csr.col), P(csr.ew), P(x), x.stride(0), rb, re, H,
                    P(w), P(b), P(scale), P(shift), epi, P(out), out.stride(0), st),
                    "mignn_gcn_layer_ring")
            elif H in (64, 128):
                fn = L.mignn_gcn_layer_f16x3 if self.precision == "f16x3" else L.mignn_gcn_layer
                _lib.check(fn(P(csr.row_ptr), P(csr.col), P(csr.ew), P(x), x.stride(0), rb, re, H,
                              P(w), P(b), P(scale), P(shift), epi, P(out), out.stride(0), st),
                           "mignn_gcn_layer")
            elif H == 256 and self._fused256():
                # aggregate + split-fp16 transform in one kernel (csrc/agg_gemm.hip)
                img = self._cached("w_gcn", i, (w,), lambda: f16x3_image(w))
                _lib.check(L.mignn_gcn_layer_fused(P(csr.row_ptr), P(csr.col), P(csr.ew), P(x),
                                                   x.stride(0), rb, re, H, P(img), P(b), P(scale),
                                                   P(shift), epi, P(out), out.stride(0), st),
                           "mignn_gcn_layer_fused")
            else:
                agg = torch.empty((n, H), dtype=torch.float32, device=x.device)
                _lib.check(L.mignn_gcn_aggregate(P(csr.row_ptr), P(csr.col), P(csr.dinv), P(x),
                                                 x.stride(0), rb, re, H,
                                                 P(agg) - rb * agg.stride(0) * 4, agg.stride(0),
                                                 st), "mignn_gcn_aggregate")
                self._mm("w_gcn", i, (w,), w, agg, b, relu=True, residual=x[rb:re], scale=scale,
                         shift=shift, out=out[rb:re])
        elif self.layer_type == "GIN":
            nn0, nn2 = layer.nn[0], layer.nn[2]
            eps = self._cached("eps", i, (layer.eps,), lambda: float(layer.eps.reshape(-1)[0]))
            if H == 256 and self._fused256():
                # sum aggregate + nn.0 + ReLU + nn.2 in one kernel (csrc/agg_gemm.hip):
                # neither the aggregate nor the hidden layer reaches memory
                img1 = self._cached("w_gin0", i, (nn0.weight,), lambda: f16x3_image(nn0.weight))
                img2 = self._cached("w_gin2p", i, (nn2.weight,), lambda: gin_fused_image(nn2.weight))
                _lib.check(L.mignn_gin_layer_fused(P(csr.row_ptr), P(csr.col), P(x), x.stride(0),
                                                   rb, re, H, eps, P(img1), P(nn0.bias), P(img2),
                                                   P(nn2.bias), P(scale), P(shift), epi, P(out),
                                                   out.stride(0), st), "mignn_gin_layer_fused")
                return
            agg = torch.empty((n, H), dtype=torch.float32, device=x.device)
            if H in (64, 128):
                _lib.check(L.mignn_gin_layer(P(csr.row_ptr), P(csr.col), P(x), x.stride(0), rb, re,
                                             H, eps, P(nn0.weight), P(nn0.bias), P(nn2.weight),
                                             P(nn2.bias), P(scale), P(shift), epi, P(agg),
                                             agg.stride(0), P(out), out.stride(0), st),
                           "mignn_gin_layer")
                return
            _lib.check(L.mignn_sum_aggregate(P(csr.row_ptr), P(csr.col), P(x), x.stride(0),
                                             1.0 + eps, rb, re, H,
                                             P(agg) - rb * agg.stride(0) * 4, agg.stride(0), st),
                       "mignn_sum_aggregate")
            h1 = self._mm("w_gin0", i, (nn0.weight,), nn0.weight, agg, nn0.bias, relu=True)
            self._mm("w_gin2", i, (nn2.weight,), nn2.weight, h1, nn2.bias, relu=True,
                     residual=x[rb:re], scale=scale, shift=shift, out=out[rb:re])
        elif self.layer_type == "GAT":
            # one C-ABI call (csrc/attn_layers.hip): logits (unless given by
            # a sharded caller), softmax aggregation, head-mean transform
            wlog, wcat = self._cached("gat", i, (layer.lin.weight, layer.att_src, layer.att_dst),
                                      lambda: self._gat_weights(layer))
            img = self._img("w_gat", i, (layer.lin.weight,), wcat)
            if logits is not None:
                logits = logits.contiguous()
            n_x = x.shape[0]
            nb = L.mignn_gat_layer_scratch_bytes(0 if logits is not None else n_x, n, H, HEADS)
            scratch = torch.empty(max(nb, 1), dtype=torch.uint8, device=x.device)
            if logits_next is not None:
                # this layer's epilogue also forms the next GAT layer's logits
                nl = self.gnn_layers[i + 1]
                wlog_n, _ = self._cached("gat", i + 1, (nl.lin.weight, nl.att_src, nl.att_dst),
                                         lambda: self._gat_weights(nl))
                _lib.check(L.mignn_gat_layer_next(
                    P(csr.row_ptr), P(csr.col), P(x), x.stride(0), n_x, rb, re, H, HEADS,
                    float(layer.negative_slope), P(wlog), P(logits), 2 * HEADS, P(wcat), P(img),
                    P(layer.bias), P(scale), P(shift), epi, P(scratch), nb, P(out), out.stride(0),
                    P(wlog_n), P(logits_next), st), "mignn_gat_layer_next")
                return
            _lib.check(L.mignn_gat_layer(
                P(csr.row_ptr), P(csr.col), P(x), x.stride(0), n_x, rb, re, H, HEADS,
                float(layer.negative_slope), P(wlog), P(logits), 2 * HEADS, P(wcat), P(img),
                P(layer.bias), P(scale), P(shift), epi, P(scratch), nb, P(out), out.stride(0), st),
                "mignn_gat_layer")
        elif self.layer_type == "Transformer":
            ts = (layer.lin_query.weight, layer.lin_query.bias, layer.lin_key.weight,
                  layer.lin_key.bias, layer.lin_value.weight, layer.lin_value.bias,
                  layer.lin_skip.weight, layer.lin_skip.bias)
            wqk, bqk, wout, bout = self._cached("tf", i, ts, lambda: self._tf_weights(layer))
            # one C-ABI call (csrc/attn_layers.hip): Q~K transform, softmax
            # aggregation, output transform over [agg | x]
            img_q = self._img("w_tfq", i, ts, wqk)
            nb = L.mignn_transformer_layer_scratch_bytes(n, H, HEADS)
            scratch = torch.empty(max(nb, 1), dtype=torch.uint8, device=x.device)
            if H == 256 and HEADS == 4 and self._fused256():
                # aggregation + output transform in one kernel (agg_gemm.hip)
                def make():
                    img = torch.empty(L.mignn_transformer_fused_prep_bytes(H, HEADS),
                                      dtype=torch.uint8, device=x.device)
                    _lib.check(L.mignn_transformer_fused_prep(P(wout), H, HEADS, P(img),
                                                              img.numel(), st),
                               "mignn_transformer_fused_prep")
                    return img
                fimg = self._cached("w_tff", i, ts, make)
                _lib.check(L.mignn_transformer_layer_fused(
                    P(csr.row_ptr), P(csr.col), P(x), x.stride(0), rb, re, H, HEADS,
                    1.0 / math.sqrt(H), P(img_q), P(bqk), P(fimg), P(bout), P(scale), P(shift),
                    epi, P(scratch), nb, P(out), out.stride(0), st), "mignn_transformer_layer_fused")
                return
            img_o = self._img("w_tfo", i, ts, wout)
            _lib.check(L.mignn_transformer_layer(
                P(csr.row_ptr), P(csr.col), P(x), x.stride(0), rb, re, H, HEADS,
                1.0 / math.sqrt(H), P(wqk), P(img_q), P(bqk), P(wout), P(img_o), P(bout),
                P(scale), P(shift), epi, P(scratch), nb, P(out), out.stride(0), st),
                "mignn_transformer_layer")
        else:
            raise ValueError(f"Unknown layer type: {self.layer_type}")

    @staticmethod
    def _gat_weights(layer: GATConv):
        heads, C = layer.heads, layer.out_channels
        W = layer.lin.weight.double().view(heads, C, -1)              # [h, c, k]
        vs = torch.einsum("hck,hc->hk", W, layer.att_src.double().view(heads, C))
        vd = torch.einsum("hck,hc->hk", W, layer.att_dst.double().view(heads, C))
        wlog = torch.cat([vs, vd], 0).float().contiguous()            # [2*heads, H]
        wcat = (W.permute(1, 0, 2).reshape(C, heads * W.shape[2]) / heads).float().contiguous()
        return wlog, wcat

    @staticmethod
    def _tf_weights(layer: TransformerConv):
        heads, C = layer.heads, layer.out_channels
        d = lambda t: t.detach().double()  # noqa: E731
        Wq = d(layer.lin_query.weight).view(heads, C, -1)   # [h, c, k]
        Wk = d(layer.lin_key.weight).view(heads, C, -1)
        Wv = d(layer.lin_value.weight).view(heads, C, -1)
        bq = d(layer.lin_query.bias).view(heads, C)
        bk = d(layer.lin_key.bias).view(heads, C)
        bv = d(layer.lin_value.bias).view(heads, C)
        Hin = Wq.shape[2]
        # score_ij = q_i . k_j = (Wk^T q_i) . x_j + q_i . bk; the second term is
        # the same for every j of row i (per head) and cancels in the softmax
        M = torch.einsum("hck,hcq->hkq", Wk, Wq).reshape(heads * Hin, Hin)   # rows h*H+kk
        mb = torch.einsum("hck,hc->hk", Wk, bq).reshape(heads * Hin)
        wqk = M.float().contiguous()                                          # [h*H, H]
        bqk = mb.float().contiguous()
        wv = Wv.permute(1, 0, 2).reshape(C, heads * Hin) / heads             # [C, h*H]
        wbv = bv.t() / heads                                                  # [C, h]
        wout = torch.cat([wv, wbv, d(layer.lin_skip.weight)], 1).float().contiguous()
        bout = layer.lin_skip.bias.detach().float().contiguous()
        return wqk, bqk, wout, bout

    def _output_mlp(self, x, tmp, out, rows=None, inv=None):
        """output_proj (gnn_model.py:90-100, :195): Lin-ReLU-Lin-ReLU-Lin-ReLU-Lin.
        precision "f16x3" with H in {64, 128} (or 256 with the fused H = 256 kernels
        on) and output_dim <= 8: one fused launch (mignn_mlp_head, split-fp16
        MFMA); otherwise four launches."""
        l0, l3, l6, l8 = (self.output_proj[i] for i in (0, 3, 6, 8))
        H = self.hidden_dim
        if (self.precision == "f16x3" and self.output_dim <= 8
                and (H in (64, 128) or (H == 256 and self._fused256("head")))):
            L = _lib.lib()
            P = _lib.ptr
            ts = (l0.weight, l0.bias, l3.weight, l3.bias, l6.weight, l6.bias, l8.weight,
                  l8.bias)

            def make():
                img = torch.empty(L.mignn_mlp_head_prep_bytes(H), dtype=torch.uint8,
                                  device=x.device)
                _lib.check(L.mignn_mlp_head_prep(*(P(t) for t in ts), H, self.output_dim,
                                                 P(img), img.numel(), _stream(x)),
                           "mignn_mlp_head_prep")
                return img
            img = self._cached("head", 0, ts, make)
            _lib.check(L.mignn_mlp_head(P(x), x.stride(0), x.shape[0], H, P(img), self.output_dim,
                                        P(out), out.stride(0), P(rows), _stream(x)),
                       "mignn_mlp_head")
            return
        mm = lambda j, l, a, **kw: self._mm("w_head", j, (l.weight,), l.weight, a, l.bias, **kw)  # noqa: E731
        h1 = mm(0, l0, x, relu=True, out=tmp)
        h2 = mm(1, l3, h1, relu=True, out=x)
        h3 = mm(2, l6, h2, relu=True)
        if inv is None:
            mm(3, l8, h3, out=out)
            return
        y = mm(3, l8, h3)                           # internal order -> caller order
        _lib.check(_lib.lib().mignn_rows_gather(
            _lib.ptr(y), y.stride(0), _lib.ptr(inv), y.shape[0], y.shape[1], _lib.ptr(out),
            out.stride(0), _stream(y)), "mignn_rows_gather")


class FlowGNNSurrogate(nn.Module):
    """Encoder/decoder composition of FlowGNN (reference gnn_model.py:223-291).

    cross_heads > 0 adds, between encoder and decoder, cross attention to the
    encoder's states of a second graph (`context` of the forward: a coarser or
    wider mesh of the same flow, any size): every node reads every context node
    of its graph, where the convolutions carry information one edge a layer.
    With the default 0 the model and its state_dict are the reference's."""

    def __init__(self, input_dim: int = 3, hidden_dim: int = 128, num_layers: int = 4,
                 layer_type: str = "GCN", use_edge_attr: bool = True, dropout: float = 0.1,
                 cross_heads: int = 0):
        super().__init__()
        self.encoder = FlowGNN(input_dim=input_dim, hidden_dim=hidden_dim, output_dim=hidden_dim,
                               num_layers=num_layers // 2, layer_type=layer_type,
                               use_edge_attr=use_edge_attr, dropout=dropout)
        self.decoder = FlowGNN(input_dim=hidden_dim, hidden_dim=hidden_dim, output_dim=8,
                               num_layers=num_layers // 2, layer_type=layer_type,
                               use_edge_attr=use_edge_attr, dropout=dropout)
        self.cross = CrossAttention(hidden_dim, cross_heads, axes=min(3, input_dim)) \
            if cross_heads else None

    def __setstate__(self, state):
        super().__setstate__(state)
        if "cross" not in self._modules:    # a model pickled before there was one
            self.__dict__.setdefault("cross", None)

    def forward(self, x, edge_index, edge_attr=None, boundary_conditions=None, context=None,
                batch=None, plan=None):
        """context (only with cross_heads > 0, and then required): the second
        graph, a `Data` / `Batch` whose x has the nodes' features; batch: the
        nodes' graph of each row when there are several (context.batch then
        too); plan: `self.cross.plan(...)` of the two graphs' sizes, built here
        when not given."""
        if (context is None) != (self.cross is None):
            raise ValueError("FlowGNNSurrogate: context is for cross_heads > 0, which needs it")
        encoded = self.encoder(x, edge_index, edge_attr)
        if context is not None:
            states = self.encoder(context.x, context.edge_index, context.edge_attr)
            if plan is None:
                context_batch = getattr(context, "batch", None)
                if (batch is None) != (context_batch is None):
                    raise ValueError("FlowGNNSurrogate: batch and context.batch go together")
                kl = graph_lengths(context_batch, context.x.shape[0])
                ql = graph_lengths(batch, x.shape[0], len(kl))
                kl += [0] * (len(ql) - len(kl))
                plan = self.cross.plan(ql, kl, train=torch.is_grad_enabled(), device=x.device)
            encoded, _ = self.cross(encoded, x.detach(), states, context.x.detach(), plan)
        if boundary_conditions is not None:
            encoded = encoded + boundary_conditions
        return self.decoder(encoded, edge_index, edge_attr)
