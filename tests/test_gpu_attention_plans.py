"""Cross attention where the plan mixes what the smaller cases take one by one:
tiles of 128 rows that carry the remainders of the 16-bit roundings, and passes
of whole and split tiles.  Against the float64 restatement in
oracle/attention_oracle.py; bounds as in test_gpu_attention.py (u = 2^-24, h the
half step of the rows' type), but where the remainders are carried P and dS are
off by h^2 (the rounding of the remainder), not by h.
"""

import pytest
import torch

from mignn import _lib
from mignn import attention as A
from oracle import attention_oracle as orc

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
EXACT = 1 << 16        # MIGNN_CROSS_EXACT, in a pass's tile


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU")
    _lib.lib()


def half_step(dt):
    return torch.finfo(dt).eps / 2


def rnd(*shape, seed=0, dt=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(dt).to(DEV)


def close(got, ref, bound, dt, what):
    """|got - ref| <= bound + the store's rounding (and fp16's subnormal step)."""
    got, ref = got.detach().double().cpu(), ref.double().cpu()
    tiny = 2.0 ** -25 if dt == torch.float16 else 2.0 ** -140
    lim = bound + half_step(dt) * (ref.abs() + bound) + tiny
    err = (got - ref).abs()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    assert not (err > lim).any(), f"{what}: worst {(err / lim).max().item():.2f} of the bound"


def left_by_rounding(plan, dt):
    """What the rounding of P or dS leaves in the forward, dq and dk / dv: nothing
    in fp32, h^2 where the remainders are carried (all tiles but plain ones of 128)."""
    h = half_step(dt)
    return [0.0 if dt == torch.float32 else h if p.tile == 128 else h * h
            for p in plan._call.passes]


def check(ql, kl, heads, kv, d, dt, masked=False):
    """Outputs and gradients (dS carries the forward's rounding in <do, o>)."""
    q, k, v = (rnd(sum(n), m, d, seed=i, dt=dt)
               for i, (n, m) in enumerate(((ql, heads), (kl, kv), (kl, kv))))
    do = rnd(sum(ql), heads, d, seed=5, dt=dt)
    mask = None
    if masked:
        mask = (torch.rand(sum(kl), generator=torch.Generator().manual_seed(9)) < 0.8).to(DEV)
    ref = orc.cross_attention(q, k, v, ql, kl, mask, None, do)
    plan = A.CrossPlan(ql, kl, heads=heads, kv_heads=kv, head_dim=d, dtype=dt)
    for t in (q, k, v):
        t.requires_grad_()
    out = A.cross_attention(q, k, v, plan, key_mask=mask)
    grads = torch.autograd.grad(out, (q, k, v), do)
    lk, lr = max(kl), max(ql) * (heads // kv)
    hf, hq, hk = left_by_rounding(plan, dt)
    base = 2 * (d + 6) * U * ref["score_mag"].max().item()
    r = base + (lk + 16) * U
    bound = {"out": r + hf, "dq": 2 * (r + (lk + d + 16) * U) + hf + hq,
             "dk": 2 * (r + (lr + lk + d + 16) * U) + hf + hk, "dv": base + (lr + lk + 16) * U + hk}
    for name, g in zip(("out", "dq", "dk", "dv"), (out,) + grads):
        close(g, ref[name], bound[name] * ref[name + "_mag"], dt, name)
    return plan


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("ql,kl,heads,kv,d,kinds", [
    ([120], [9000], 2, 2, 128, "fq"), ([2300], [120], 2, 1, 128, "k"),
    ([160], [9000], 2, 2, 96, "fq"), ([4000], [101], 2, 2, 96, "k"),
    ([70, 55], [34000, 33700], 2, 1, 64, "q"), ([2500], [230], 2, 2, 64, "k"),
    ([33, 260], [11, 65000], 2, 2, 32, "q"), ([3000, 5], [400, 90], 3, 1, 32, ""),
    ([250], [68000], 1, 1, 64, "fq"), ([505], [67000], 1, 1, 32, "fq"),
    ([20000, 40], [500, 1], 2, 1, 32, "k"),
    ([1] * 35, [75 * i for i in range(35)], 2, 2, 24, "k"), ([9, 16], [3000, 1], 8, 2, 64, "k"),
    ([700, 300], [64, 1], 4, 2, 128, "q"), ([32], [2000], 2, 1, 96, "k")])
def test_few_results_and_short_gradients_carry_the_remainders(ql, kl, heads, kv, d, kinds, dt):
    """128-row tiles with the remainders, at every width, ragged and grouped."""
    plan = check(ql, kl, heads, kv, d, dt, masked=True)
    for kind, name in enumerate("fqk"):
        if name in kinds:
            assert plan._call.passes[kind].tile == 128 | EXACT, name


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("ql,kl,heads,kv,d,kinds", [
    ([33000, 70], [600, 50], 4, 2, 32, "fq"), ([600], [66000], 4, 2, 32, "k"),
    ([17000], [600], 4, 4, 64, "fq"), ([260], [66000], 4, 2, 64, "k"),
    ([16512], [600], 4, 4, 128, "fq")])
def test_whole_and_split_tiles_in_one_pass(ql, kl, heads, kv, d, kinds, dt):
    """More tiles than the card holds at a time, the last round's split and
    joined: both ranges of a launch's workgroups, joins of some tiles only."""
    plan = check(ql, kl, heads, kv, d, dt, masked=True)
    for kind, name in enumerate("fqk"):
        p = plan._call.passes[kind]
        if name in kinds:
            assert p.tile == 128 and 0 < p.n_whole < p.n_items and p.n_joins > 0, name


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [8, 16, 24])
def test_dq_of_narrow_heads_carries_the_remainders(d, dt):
    plan = check([2100, 300], [700, 1234], 4, 2, d, dt, masked=True)
    assert plan._call.passes[1].tile == (128 | EXACT if d <= 16 else 128)
