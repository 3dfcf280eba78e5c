"""Row operators (mignn.attention) on the host: refusals of bad arguments
before any device work, the cross-attention plan's coverage, and the C entry
points' argument checks.  No GPU needed."""

import ctypes

import numpy as np
import pytest
import torch

from mignn import _lib
from mignn import attention as A
from oracle import attention_oracle as orc


def test_rms_norm_refusals():
    x, w = torch.zeros(4, 16), torch.ones(16)
    for args, exc, msg in [
            ((torch.zeros(4), w), ValueError, "x must be"),
            ((torch.zeros(4, 16, dtype=torch.float64), w), TypeError, "rows must be"),
            ((torch.zeros(4, 16, dtype=torch.int32), w), TypeError, "rows must be"),
            ((torch.zeros(4, 0), torch.ones(0)), ValueError, "width 0"),
            ((torch.zeros(1, 2049), torch.ones(2049)), ValueError, "width 2049"),
            ((x, torch.ones(15)), ValueError, "weight must be"),
            ((x, torch.ones(1, 16)), ValueError, "weight must be"),
            ((x, w.half()), TypeError, "weight must be float32"),
            ((x, w, torch.zeros(3, 16)), ValueError, "residual must be"),
            ((x, w, x.half()), ValueError, "residual must be"),
            ((x, w, None, -1e-6), ValueError, "eps"),
            ((x, w, None, float("nan")), ValueError, "eps"),
            ((x, w), RuntimeError, "ROCm devices only")]:
        with pytest.raises(exc, match=msg):
            A.rms_norm(*args)


def test_rotary_refusals():
    ax = A.RotaryAxes((3, 3, 2), device="cpu")
    x, pos = torch.zeros(5, 2, 16), torch.zeros(5, 3)
    for args, exc, msg in [
            ((torch.zeros(5, 16), pos, ax), ValueError, "x must be"),
            ((x.double(), pos, ax), TypeError, "rows must be"),
            ((x, torch.zeros(5, 2), ax), ValueError, "pos must be"),
            ((x, torch.zeros(4, 3), ax), ValueError, "pos must be"),
            ((x, pos.half(), ax), TypeError, "pos must be"),
            ((torch.zeros(5, 2, 14), pos, ax), ValueError, "do not fit"),
            ((x, pos.clone().requires_grad_(), ax), NotImplementedError, "no gradient"),
            ((x, pos, ax), RuntimeError, "ROCm devices only")]:
        with pytest.raises(exc, match=msg):
            A.rotary(*args)
    for pairs, kw in [((), {}), ((0, 0), {}), ((4097,), {}), ((2, -1), {}), ((2,), {"base": 0.0}),
                      ((2,), {"base": float("inf")}), ((2, 2), {"scales": (1.0,)}),
                      ((2,), {"scales": (float("nan"),)})]:
        with pytest.raises(ValueError):
            A.RotaryAxes(pairs, device="cpu", **kw)


def test_cross_plan_refusals():
    ok = dict(heads=4, kv_heads=2, head_dim=32, device="cpu")
    for ql, kl, kw, exc, msg in [
            ([1, 2], [3], ok, ValueError, "2 query sequences but 1"),
            ([1, -2], [3, 4], ok, ValueError, "negative length in q_lens"),
            ([1], [-1], ok, ValueError, "negative length in k_lens"),
            ([1.5], [2], ok, ValueError, "whole numbers"),
            ([1], [1], dict(ok, kv_heads=3), ValueError, "4 query heads over 3"),
            ([1], [1], dict(ok, heads=0), ValueError, "0 query heads"),
            ([1], [1], dict(ok, heads=33, kv_heads=1), ValueError, "more than 32"),
            ([1], [1], dict(ok, head_dim=12), ValueError, "head_dim"),
            ([1], [1], dict(ok, head_dim=136), ValueError, "head_dim"),
            ([1], [1], dict(ok, head_dim=0), ValueError, "head_dim"),
            ([1], [1], dict(ok, dtype=torch.float64), TypeError, "rows must be"),
            ([2 ** 31], [1], ok, _lib.MignnError, "too long"),
            ([2 ** 30, 2 ** 30, 2 ** 30], [1, 1, 1], dict(ok, heads=1, kv_heads=1),
             _lib.MignnError, "2\\^31")]:
        with pytest.raises(exc, match=msg):
            A.CrossPlan(ql, kl, **kw)


def test_cross_attention_refusals():
    plan = A.CrossPlan([3, 2], [4, 1], heads=4, kv_heads=2, head_dim=16, device="cpu", train=False)
    q, k = torch.zeros(5, 4, 16), torch.zeros(5, 2, 16)
    for args, kw, exc, msg in [
            ((q[:4], k, k), {}, ValueError, "plan's q"),
            ((q, k[:4], k), {}, ValueError, "plan's k"),
            ((q, k, k[..., :8]), {}, ValueError, "plan's v"),
            ((q.half(), k, k), {}, TypeError, "plan's rows"),
            ((q, k, k.bfloat16()), {}, TypeError, "plan's rows"),
            ((q, k, k), {"key_mask": torch.ones(4, dtype=torch.bool)}, ValueError, "key_mask"),
            ((q, k, k), {"key_mask": torch.ones(5)}, ValueError, "key_mask"),
            ((q, k, k), {"scale": 0.0}, ValueError, "scale"),
            ((q, k, k), {"scale": -1.0}, ValueError, "scale"),
            ((q, k, k), {"scale": float("inf")}, ValueError, "scale"),
            ((q, k, k), {"scale": float("nan")}, ValueError, "scale"),
            ((q, k, k), {}, RuntimeError, "ROCm devices only")]:
        with pytest.raises(exc, match=msg):
            A.cross_attention(*args, plan, **kw)


def _lists(plan, kind):
    ps = plan._call.passes[kind]
    raw = plan._lists.numpy().view(np.int32).reshape(-1, 8)
    base = plan._lists.data_ptr()
    a, b = ((ps.items or 0) - base) // 32, ((ps.joins or 0) - base) // 32
    return raw[a:a + ps.n_items], raw[b:b + ps.n_joins], ps.part_bytes


@pytest.mark.parametrize("ql,kl,heads,kv", [
    ([1], [1], 1, 1), ([5], [0], 4, 4), ([0], [9], 4, 2), ([0, 0], [0, 0], 2, 1), ([], [], 2, 2),
    ([1], [20000], 8, 2), ([40000], [33], 4, 1), ([129, 0, 1, 4000], [1, 700, 0, 5000], 6, 3),
    ([1] * 64, list(range(0, 64 * 97, 97)), 8, 2),
    ([33000], [3000], 4, 2), ([9000, 70, 30000], [300, 9000, 2000], 4, 4)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_cross_plan_covers_every_pair_once(ql, kl, heads, kv, dtype):
    """Every (row, key) pair of every sequence is in exactly one item of each
    pass, every tile row in one item or in one join whose slots are its own and
    fit the scratch."""
    plan = A.CrossPlan(ql, kl, heads=heads, kv_heads=kv, head_dim=32, dtype=dtype, device="cpu")
    g = heads // kv
    for kind in range(3):
        items, joins, part = _lists(plan, kind)
        dkv = kind == _lib.CROSS_DKV
        seen, slots, tiles = {}, {}, {}
        for qb, kb, r0, r1, c0, c1, slot, _ in items.tolist():
            assert 0 <= r0 < r1 and 0 <= c0 <= c1
            seen.setdefault((qb, kb, r0, r1), []).append((c0, c1, slot))
            if slot >= 0:
                assert slot not in slots
                slots[slot] = (qb, kb, r0, r1)
        qb = kb = 0
        for lq, lk in zip(ql, kl):
            rn, cn = (lk, lq * g) if dkv else (lq * g, lk)
            spans = sorted((r0, r1) for a, b, r0, r1 in seen
                           if (a, b) == (qb, kb) and rn > r0 and (a, b, r0, r1) not in tiles)
            at = 0
            for r0, r1 in spans:
                assert r0 == at
                at = r1
                cs = sorted(seen[(qb, kb, r0, r1)])
                tiles[(qb, kb, r0, r1)] = cs
                c = 0
                for c0, c1, slot in cs:
                    assert c0 == c and (slot >= 0) == (len(cs) > 1)
                    c = c1
                assert c == cn
            assert at == rn
            qb, kb = qb + lq, kb + lk
        assert len(tiles) == len(seen)
        joined = {}
        for begin, r0, r1, slot, parts, *_ in joins.tolist():
            for s in range(slot, slot + parts):
                a, b, t0, t1 = slots.pop(s)
                assert (b if dkv else a) == begin and (t0, t1) == (r0, r1)
                joined[s] = True
        assert not slots
        rows = max([r1 - r0 for _, _, r0, r1 in seen] or [0])
        if joined:
            assert part >= (max(joined) + 1) * kv * rows * 32 * 4


def test_c_entry_points_check_arguments():
    L = _lib.lib()
    buf = (ctypes.c_float * 64)()
    p = (ctypes.addressof(buf) + 15) & ~15      # never dereferenced

    def norm(dtype=0, n=2, h=8, ldx=8, x=p, eps=1e-6, ldy=8):
        return L.mignn_rms_norm(x, ldx, None, 0, p, 1, n, h, eps, dtype, p, ldy, None, 0, None)
    assert norm(n=0) == 0
    for kw, msg in [({"dtype": 3}, "row type"), ({"h": 0}, "h = 0"), ({"h": 2049}, "h = 2049"),
                    ({"n": -1}, "n = -1"), ({"x": None}, "null"), ({"ldx": 7}, "stride"),
                    ({"eps": -1.0}, "eps"), ({"ldy": 7}, "output")]:
        assert norm(**kw) == 1 and msg in _lib.last_error(), (kw, _lib.last_error())
    need = L.mignn_rms_norm_backward_scratch_bytes(1000, 8, 0)
    assert need > 0 and L.mignn_rms_norm_backward_scratch_bytes(-1, 8, 0) == 0
    assert L.mignn_rms_norm_backward_scratch_bytes(100, 8, 0) == 0     # one block's

    def norm_backward(n, w, nbytes):
        return L.mignn_rms_norm_backward(p, 8, None, 0, w, 1, n, 8, 1e-6, 0, p, 8, None, 0, p, 8, p,
                                         p, nbytes, None)
    assert norm_backward(1000, p, need - 1) == 4
    assert norm_backward(0, None, need) == 1 and "null" in _lib.last_error()

    def rot(n=1, heads=1, d=8, pos_type=0, pairs=4, dtype=0, freq=p):
        return L.mignn_rotary(p, 8, 8, n, heads, d, p, pos_type, 1, freq, p, pairs, 0, 0, dtype, p,
                              8, 8, None)
    assert rot(n=0) == 0 and rot(heads=0) == 0
    for kw, msg in [({"dtype": -1}, "row type"), ({"pos_type": 4}, "position type"),
                    ({"pairs": 5}, "pairs = 5"), ({"pairs": 0}, "pairs = 0"),
                    ({"freq": None}, "null")]:
        assert rot(**kw) == 1 and msg in _lib.last_error(), kw

    plan = A.CrossPlan([3], [9], heads=2, head_dim=16, device="cpu")

    def fwd(q=p, ldq=32, ldkh=16, scale=1.0, d=16, out=p, k=p):
        c = _lib.CrossCall.from_buffer_copy(plan._call)
        c.q, c.k, c.v, c.ldq, c.ldqh, c.ldk, c.ldkh = q, k, p, ldq, 16, 32, ldkh
        c.ldv, c.ldvh, c.scale, c.d = 32, 16, scale, d
        return L.mignn_cross_attn_forward(ctypes.addressof(c), out, None, None, None)
    for kw, msg in [({"q": p + 4}, "q needs"), ({"ldq": 33}, "q needs"), ({"ldkh": 2}, "k needs"),
                    ({"k": None}, "k needs"), ({"scale": 0.0}, "scale"), ({"d": 20}, "head width"),
                    ({"out": p + 4}, "output")]:
        assert fwd(**kw) == 1 and msg in _lib.last_error(), (kw, _lib.last_error())
    assert L.mignn_cross_attn_forward(None, p, None, None, None) == 1


def test_call_struct_layout_matches_header():
    """The ctypes mirror of mignn_cross_call has the C layout (x86-64)."""
    assert ctypes.sizeof(_lib.CrossPass) == 48
    assert _lib.CrossCall.ldq.offset == 32 and _lib.CrossCall.n_keys.offset == 80
    assert _lib.CrossCall.scale.offset == 104 and _lib.CrossCall.scratch.offset == 112
    assert ctypes.sizeof(_lib.CrossCall) == 128 + 3 * 48


def test_oracle_gradients_match_differences():
    """The oracle's gradient formulas against central differences of its own
    forward, in float64."""
    gen = torch.Generator().manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64)  # noqa: E731
    ql, kl = [3, 0, 2], [5, 2, 0]
    q, k, v, do = r(5, 4, 8), r(7, 2, 8), r(7, 2, 8), r(5, 4, 8)
    mask = torch.tensor([1, 0, 1, 1, 1, 1, 1], dtype=torch.bool)
    ref = orc.cross_attention(q, k, v, ql, kl, mask, None, do)
    e = 1e-5
    for name, t in (("dq", q), ("dk", k), ("dv", v)):
        way = r(*t.shape)
        args = {"dq": q, "dk": k, "dv": v}
        hi, lo = (orc.cross_attention(*[args[m] + (s * e * way if m == name else 0)
                                        for m in ("dq", "dk", "dv")], ql, kl, mask)["out"]
                  for s in (1, -1))
        num = ((hi - lo) * do).sum() / (2 * e)
        assert abs(num - (ref[name] * way).sum()) < 1e-7
    x, res, w, dy, ds = r(6, 9), r(6, 9), r(9), r(6, 9), r(6, 9)
    dx, dw, _, _ = orc.rms_norm_grads(x, w, res, 1e-6, dy, ds)

    def loss(x, w):
        y, s, _ = orc.rms_norm(x, w, res, 1e-6)
        return (y * dy).sum() + (s * ds).sum()
    wx, ww = r(6, 9), r(9)
    assert abs((loss(x + e * wx, w) - loss(x - e * wx, w)) / (2 * e) - (dx * wx).sum()) < 1e-7
    assert abs((loss(x, w + e * ww) - loss(x, w - e * ww)) / (2 * e) - (dw * ww).sum()) < 1e-7
    # a rotation's gradient is its transpose, the rotation back
    pos, u = torch.randint(0, 50, (4, 2), generator=gen), r(4, 3, 14)
    for il in (False, True):
        back = orc.rotary(orc.rotary(u, pos, (3, 2), interleaved=il), pos, (3, 2), interleaved=il,
                          inverse=True)
        assert (back - u).abs().max() < 1e-12


def test_block_and_surrogate_refusals():
    from mignn import Data, FlowGNNSurrogate
    for args in [(30, 4), (64, 0), (64, 3), (512, 2), (64, 16)]:
        with pytest.raises(ValueError, match="CrossAttention"):
            A.CrossAttention(*args)
    with pytest.raises(ValueError, match="position axes"):
        A.CrossAttention(32, 4, axes=5)
    blk = A.CrossAttention(64, 4)
    plan = blk.plan([3], [2], device="cpu")
    x, c = torch.zeros(3, 64), torch.zeros(2, 64)
    with pytest.raises(ValueError, match="context must be"):
        blk(x, x[:, :3], c[:, :32], c[:, :3], plan)
    with pytest.raises(RuntimeError, match="ROCm devices only"):
        blk(x, x[:, :3], c, c[:, :3], plan)
    ei = torch.zeros(2, 1, dtype=torch.long)
    ctx = Data(x=torch.zeros(2, 3), edge_index=ei)
    with pytest.raises(ValueError, match="context is for"):
        FlowGNNSurrogate(hidden_dim=32)(torch.zeros(3, 3), ei, context=ctx)
    with pytest.raises(ValueError, match="context is for"):
        FlowGNNSurrogate(hidden_dim=32, cross_heads=4)(torch.zeros(3, 3), ei)
    # the default model has the reference's parameters and no more
    assert not [k for k in FlowGNNSurrogate(hidden_dim=32).state_dict() if k.startswith("cross")]


def test_graph_lengths():
    assert A.graph_lengths(None, 7) == [7]
    assert A.graph_lengths(torch.tensor([0, 0, 2]), 3, 4) == [2, 0, 1, 0]
    assert A.graph_lengths(torch.zeros(0, dtype=torch.long), 0, 2) == [0, 0]
    for bad in (torch.tensor([1, 0]), torch.tensor([0])):
        with pytest.raises(ValueError, match="sorted"):
            A.graph_lengths(bad, 2)


def test_ops_module_is_bound_to_the_product_library():
    """_ops.so loads, its table has the entry points that it calls, and a wrong
    table is an error, not a jump."""
    ops = _lib.ops()
    assert ops is _lib.ops()
    assert all(n in _lib.SIGNATURES for n in _lib.OPS_ENTRIES)
    with pytest.raises(ValueError, match="entry points"):
        ops.bind([0])


def test_block_axes_follow_its_settings():
    blk = A.CrossAttention(64, 4)
    cpu = torch.device("cpu")
    first = blk._rotary_axes(cpu)
    assert blk._rotary_axes(cpu) is first
    blk.position_scale = 8.0
    assert blk._rotary_axes(cpu).scales == (8.0,) * 3
    blk.base = 50.0
    assert blk._rotary_axes(cpu).base == 50.0


def test_more_blocks_than_a_launch_holds_are_refused():
    n = 2 ** 22
    with pytest.raises(_lib.MignnError, match="too many tiles"):
        A.CrossPlan(np.ones(n, np.int64), np.ones(n, np.int64), heads=4, head_dim=8, device="cpu",
                    train=False)
    L = _lib.lib()
    buf = (ctypes.c_float * 64)()
    p = (ctypes.addressof(buf) + 15) & ~15      # never dereferenced
    assert L.mignn_rotary(p, 8192, 8192, 1 << 24, 1, 8192, p, 0, 1, p, p, 4096, 0, 0, 1, p, 8192, 8192,
                          None) == 1 and "too many rows" in _lib.last_error()


def test_block_and_axes_copy_and_pickle():
    import copy
    import pickle
    blk = A.CrossAttention(64, 4)
    axes = blk._rotary_axes(torch.device("cpu"))
    for other in (copy.deepcopy(blk), pickle.loads(pickle.dumps(blk))):
        assert other._axes.pairs == axes.pairs and torch.equal(other._axes.freq, axes.freq)
        assert all(torch.equal(a, b) for a, b in zip(blk.state_dict().values(),
                                                     other.state_dict().values()))


@pytest.mark.parametrize("ql,kl", [([1], [20000]), ([300, 5], [900, 4000]), ([0], [9])])
def test_backward_s_work_lists_follow_the_lists_it_holds(ql, kl):
    """The backward forms the addresses of its work lists from the list tensor
    in its hands, not from where the forward found the plan's."""
    plan = A.CrossPlan(ql, kl, heads=4, kv_heads=2, head_dim=32, device="cpu")
    other = plan._lists.clone()
    assert other.data_ptr() != plan._lists.data_ptr()

    def places(at):
        return _lib.ops().plan_places(plan._address, plan._lists, at)
    own = [p or 0 for ps in plan._call.passes for p in (ps.items, ps.joins)]
    assert places(plan._lists) == own
    assert [p - other.data_ptr() for p in places(other)] == \
        [p - plan._lists.data_ptr() for p in own]


def test_forward_mode_tangents_are_refused_by_name():
    """A dual tensor, with or without requires_grad: no output without its tangent."""
    import torch.autograd.forward_ad as fwd
    w, axes, pos = torch.ones(16), A.RotaryAxes((3, 3, 2), device="cpu"), torch.zeros(5, 3)
    plan = A.CrossPlan([5], [5], heads=2, head_dim=16, device="cpu")
    h = torch.zeros(5, 2, 16)
    calls = {
        "rms_norm: x": lambda d: A.rms_norm(d(torch.zeros(4, 16)), w),
        "rms_norm: weight": lambda d: A.rms_norm(torch.zeros(4, 16), d(w)),
        "rms_norm: residual": lambda d: A.rms_norm(torch.zeros(4, 16), w, d(torch.zeros(4, 16))),
        "rotary: x": lambda d: A.rotary(d(h), pos, axes),
        "rotary: pos": lambda d: A.rotary(h, d(pos), axes),
        "cross_attention: q": lambda d: A.cross_attention(d(h), h, h, plan),
        "cross_attention: k": lambda d: A.cross_attention(h, d(h), h, plan),
        "cross_attention: v": lambda d: A.cross_attention(h, h, d(h), plan)}
    for name, call in calls.items():
        for leaf in (False, True):
            with fwd.dual_level():
                def dual(t):
                    return fwd.make_dual(t.clone().requires_grad_(leaf and name != "rotary: pos"),
                                         torch.ones_like(t))
                for grad in (True, False):
                    with torch.set_grad_enabled(grad), \
                            pytest.raises(NotImplementedError, match=name + " carries a tangent"):
                        call(dual)
                # forward mode switched off, or the primal alone: an ordinary call
                with fwd._set_fwd_grad_enabled(False), \
                        pytest.raises(RuntimeError, match="ROCm devices only"):
                    call(dual)
                with pytest.raises(RuntimeError, match="ROCm devices only"):
                    call(lambda t: fwd.unpack_dual(dual(t)).primal)


def test_surrogate_pickled_before_cross_attention_still_runs():
    """A model saved whole when FlowGNNSurrogate had no `cross`, and one with it."""
    import pickle
    from mignn import Data, FlowGNNSurrogate
    x, ei = torch.zeros(2, 3), torch.zeros(2, 0, dtype=torch.long)
    m = FlowGNNSurrogate(hidden_dim=32, num_layers=2)
    del m.__dict__["cross"]
    old = pickle.loads(pickle.dumps(m))
    assert old.cross is None and list(old.state_dict()) == list(FlowGNNSurrogate(
        hidden_dim=32, num_layers=2).state_dict())
    with pytest.raises(RuntimeError, match="ROCm devices only"):
        old(x, ei)
    with pytest.raises(ValueError, match="context is for"):
        old(x, ei, context=Data(x=x, edge_index=ei))
    new = pickle.loads(pickle.dumps(FlowGNNSurrogate(hidden_dim=32, num_layers=2, cross_heads=2)))
    assert isinstance(new.cross, A.CrossAttention) and "cross" not in new.__dict__
