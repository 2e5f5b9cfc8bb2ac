"""The AdamW step and the gradient norm at the ends of f32."""
from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")
from test_gpu_adamw import F32, HYPER, decode, rand, state_8  # noqa: E402

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
