"""The row operators' backward (mignn.attention) where autograd hands its saved
tensors through other hands: checkpointing, saved-tensor hooks, tensors kept in
host memory.  The arithmetic is the plain step's, so every gradient has its
bits."""

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from mignn import _lib
from mignn import attention as A

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU")
    _lib.lib()


def rnd(*shape, seed=0, dt=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(dt).to(DEV)


class Copies:
    """Saved-tensor hooks that keep a copy and let the saved tensor go."""

    def __enter__(self):
        self.hooks = torch.autograd.graph.saved_tensors_hooks(
            lambda t: t.detach().clone(), lambda t: t)
        return self.hooks.__enter__()

    def __exit__(self, *a):
        return self.hooks.__exit__(*a)


def run(f, way):
    """f() under a way of keeping what the backward needs."""
    if way == "plain":
        return f()
    if way == "checkpoint":
        return checkpoint(f, use_reentrant=False)
    with Copies() if way == "copies" else torch.autograd.graph.save_on_cpu(pin_memory=way == "pinned"):
        return f()


WAYS = ["checkpoint", "copies", "host", "pinned"]


@pytest.mark.parametrize("way", WAYS)
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("ql,kl", [([300, 5], [900, 4000]), ([2], [5000]), ([700], [9])])
def test_plan_dropped_ahead_of_the_backward(ql, kl, dt, way):
    """The plan lives in the forward alone, and its memory goes to others
    before the backward runs."""
    q, k, v = (rnd(sum(n), h, 32, seed=i, dt=dt).requires_grad_()
               for i, (n, h) in enumerate(((ql, 4), (kl, 2), (kl, 2))))
    mask = (torch.rand(sum(kl), generator=torch.Generator().manual_seed(7)) < 0.7).to(DEV)
    do = rnd(*q.shape, seed=5, dt=dt)
    size = []

    def forward():
        plan = A.CrossPlan(ql, kl, heads=4, kv_heads=2, head_dim=32, dtype=dt)
        size.append(plan._lists.numel())
        return A.cross_attention(q, k, v, plan, key_mask=mask)
    want = torch.autograd.grad(forward(), (q, k, v), do)
    out = run(forward, way)
    others = [torch.zeros(size[0], dtype=torch.uint8, device=DEV) for _ in range(16)]
    got = torch.autograd.grad(out, (q, k, v), do)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(int(t.count_nonzero()) == 0 for t in others)


@pytest.mark.parametrize("way", WAYS)
def test_surrogate_that_makes_its_own_plan(way):
    """A training step of FlowGNNSurrogate without plan=."""
    from mignn import Data, FlowGNNSurrogate
    from mignn.synthetic import grid_graph
    torch.manual_seed(0)
    m = FlowGNNSurrogate(hidden_dim=64, num_layers=4, dropout=0.0, cross_heads=4).to(DEV).train()
    x, ei = grid_graph(8, 6, 5, device=DEV, permute_seed=0)
    cx, cei = grid_graph(4, 3, 3, device=DEV, permute_seed=1)
    ctx = Data(x=cx, edge_index=cei)
    params = list(m.parameters())

    def same(a, b):
        return all(x is y or torch.equal(x, y) for x, y in zip(a, b))

    def step(how):
        out = run(lambda: m(x, ei, context=ctx), how)
        junk = [torch.zeros(n, dtype=torch.uint8, device=DEV) for n in range(64, 4096, 64)]
        grads = torch.autograd.grad(out.square().mean(), params, allow_unused=True)
        del junk
        return grads
    want = step("plain")
    assert same(step("plain"), want)
    assert same(step(way), want)


@pytest.mark.parametrize("spoil", ["host", "type", "rows"])
def test_hooks_that_give_back_other_tensors_are_refused(spoil):
    """Each saved tensor in turn comes back on the host, in another type or a row
    short: an error by name ahead of any launch."""
    x, w = rnd(20, 64, seed=1).requires_grad_(), rnd(64, seed=2).requires_grad_()
    q, k = rnd(20, 4, 32, seed=3).requires_grad_(), rnd(90, 2, 32, seed=4).requires_grad_()
    mask = torch.ones(90, dtype=torch.bool, device=DEV)
    pos = torch.rand(20, 2, device=DEV)
    axes = A.RotaryAxes((4, 4))
    plan = A.CrossPlan([20], [90], heads=4, kv_heads=2, head_dim=32)
    change = {"host": lambda t: t.cpu(), "type": lambda t: t.to(torch.float64),
              "rows": lambda t: t[:-1]}[spoil]
    for what, f, leaf in [
            ("rms_norm", lambda: A.rms_norm(x, w), x),
            ("rms_norm", lambda: A.rms_norm(x, w, residual=x)[0], w),
            ("rms_norm", lambda: A.rms_norm(x.half(), w, residual=x.half())[0], x),
            ("rotary", lambda: A.rotary(q, pos, axes), q),
            ("cross_attention", lambda: A.cross_attention(q, k, k, plan, key_mask=mask), k)]:
        turn, kept = 0, [1]
        while turn < kept[0]:
            kept[0] = 0

            def pack(t):
                kept[0] += 1
                return kept[0] - 1, t

            def unpack(p):
                return change(p[1]) if p[0] == turn else p[1]
            with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
                y = f()
            with pytest.raises(RuntimeError, match=f"{what} backward: saved"):
                torch.autograd.grad(y.float().square().sum(), leaf)
            turn += 1
        assert turn == {"rms_norm": 3 if y.dtype == torch.float16 else 2, "rotary": 1,
                        "cross_attention": 6}[what]
