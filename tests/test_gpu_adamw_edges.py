"""The AdamW step and the gradient norm at the ends of f32."""
from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")
from test_gpu_adamw import F32, HYPER, decode, lists, rand, state_8  # noqa: E402
from train_ref import U, assert_within  # noqa: E402

pytestmark = pytest.mark.gpu

NAMES = ("exp_avg", "exp_avg_sq")


@pytest.mark.parametrize("bad,v_only", [(1e20, True), (-1e20, True), (math.inf, False), (-math.inf, False)])
def test_step_8_bits_overflow_makes_the_block_nan(kernels, bad, v_only):
    """A square past f32 makes its block's v NaN, an infinite gradient its m too; the next step shows it in every
    parameter of the block and in no other."""
    n = 2000
    p, g = [rand(n, F32, 1)], [rand(n, F32, 2)]
    s, clean = state_8([n], 3), state_8([n], 3)
    q, spoilt = [p[0].clone()], [g[0].clone()]
    spoilt[0][700] = bad
    keep = torch.ones(n, dtype=torch.bool, device="cuda")
    keep[512:768] = False
    kernels.adamw(p, g, **clean, **HYPER)
    kernels.adamw(q, spoilt, **s, **HYPER)
    others = torch.ones(n, dtype=torch.bool, device="cuda")
    others[700] = False
    assert torch.equal(p[0][others], q[0][others])
    for name in NAMES:
        assert torch.equal(s[name][0].float()[keep], clean[name][0].float()[keep])
        value = decode(s[name][0], s[name + "_scales"][0])
        assert bool(value[keep].isfinite().all())
        assert bool(value[~keep].isfinite().all() if name == "exp_avg" and v_only else value[~keep].isnan().all()), name
    kernels.adamw(p, g, **clean, **{**HYPER, "step": 8})
    kernels.adamw(q, g, **s, **{**HYPER, "step": 8})
    assert torch.equal(p[0][keep], q[0][keep]) and bool(q[0][~keep].isnan().all())


@pytest.mark.parametrize("n", [100, 256, 4096, 70001])
@pytest.mark.parametrize("eps", [1e-38, 1e-40, 1e-45])
def test_step_8_bits_subnormal_eps(kernels, eps, n):
    """An element whose gradient and states are zero only decays, however small eps is."""
    p, g = [rand(n, F32, 1)], [rand(n, F32, 2)]
    g[0][::3] = 0.0
    s = kernels.adamw_state(p, bits=8)
    before = p[0].clone()
    kernels.adamw(p, g, **s, **{**HYPER, "step": 1, "eps": eps})
    want = before[::3].double() * (1 - 1e-3)
    assert_within(p[0][::3], want, 4 * U * want.abs(), "decayed only")
    assert bool(p[0].isfinite().all())
    moved = torch.ones(n, dtype=torch.bool, device="cuda")
    moved[::3] = False
    # From zeroed states the first step moves by lr: 12 roundings bound the quotient's.
    want = before.double() * (1 - 1e-3) - 1e-2 * torch.sign(g[0].double())
    assert_within(p[0][moved], want[moved], (4 * U * before.double().abs() + 12 * U * 1e-2 + 2 * U * want.abs())[moved], "moved")


def test_norm_past_f32(kernels):
    """A norm that f32 does not hold is infinite, its scale NaN, and the step leaves everything as it was."""
    p, g, m, v = lists([1000, 70], F32, F32)
    g = [torch.full_like(t, 3e38) for t in g]
    norm, scale = kernels.grad_norm(g, 1.0)
    assert math.isinf(norm.item()) and math.isnan(scale.item())
    before = [t.clone() for t in p + m + v]
    kernels.adamw(p, g, m, v, grad_scale=scale, **HYPER)
    assert all(torch.equal(a, b) for a, b in zip(before, p + m + v))
    # The largest norms that f32 holds are finite, and clipped.
    norm, scale = kernels.grad_norm([torch.full((4,), 1.5e38, device="cuda")], 1.0)
    assert norm.item() == pytest.approx(3e38, rel=4 * U) and scale.item() == pytest.approx(1 / 3e38, rel=4 * U, abs=2.0 ** -150)
