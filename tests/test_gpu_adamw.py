"""The gradient norm and the AdamW step against 64-bit formulas, with bounds
counted in roundings (train_ref.py)."""
from __future__ import annotations

import math

import pytest

from conftest import spmd_mod

torch = pytest.importorskip("torch")
from train_ref import U, adam_ref, assert_within, norm_back_ref, norm_ref, rounded  # noqa: E402

pytestmark = pytest.mark.gpu

F32, F16, BF16, E4M3 = torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn
SIZES = [1, 2, 255, 256, 257, 1000, 2047, 2048, 2049, 65537, 0, 300001]
HYPER = {"step": 7, "lr": 1e-2, "betas": (0.9, 0.95), "eps": 1e-8, "weight_decay": 0.1}


def rand(n, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(n, generator=g, device="cuda") * scale).to(dtype)


def lists(sizes, p_t, g_t, seed=1):
    p = [rand(n, p_t, seed + k, 0.5) for k, n in enumerate(sizes)]
    g = [rand(n, g_t, seed + 100 + k, 0.01) for k, n in enumerate(sizes)]
    m = [rand(n, F32, seed + 200 + k, 0.01) for k, n in enumerate(sizes)]
    v = [rand(n, F32, seed + 300 + k, 0.01).square() for k, n in enumerate(sizes)]
    return p, g, m, v


def ref_args(h, k=0):
    wd = h["weight_decay"]
    return {"step": h["step"], "lr": h["lr"], "betas": h["betas"], "eps": h["eps"],
            "decay": wd[k] if isinstance(wd, list) else wd}


def check_32(kernels, p, g, m, v, copies=None, scale=None, **h):
    want = [adam_ref(*t, **ref_args(h, k), scale=1.0 if scale is None else scale.item())
            for k, t in enumerate(zip(p, g, m, v))]
    kernels.adamw(p, g, m, v, copies=copies, grad_scale=scale, **h)
    for k, (p1, m1, v1, e_p, e_m, e_v) in enumerate(want):
        assert_within(m[k], m1, e_m, f"m of {k}")
        assert_within(v[k], v1, e_v, f"v of {k}")
        assert_within(p[k], p1, e_p + rounded(p1.abs() + e_p, p[k].dtype), f"p of {k}")
        if copies is not None and copies[k] is not None:
            assert_within(copies[k], p1, e_p + rounded(p1.abs() + e_p, copies[k].dtype), f"copy of {k}")
            if p[k].dtype == F32:
                assert torch.equal(copies[k], p[k].to(copies[k].dtype))


@pytest.mark.parametrize("p_t", [F32, F16, BF16])
@pytest.mark.parametrize("g_t", [F32, F16, BF16])
def test_step_types_and_sizes(kernels, p_t, g_t):
    p, g, m, v = lists(SIZES, p_t, g_t)
    check_32(kernels, p, g, m, v, **HYPER)


def test_step_mixed_types_in_one_call(kernels):
    types = [(F32, BF16), (BF16, BF16), (F16, F32), (F32, F32), (F32, BF16)]
    p, g, m, v = ([lists([1000 + 17 * k], *t, seed=k)[i][0] for k, t in enumerate(types)] for i in range(4))
    copies = [torch.zeros_like(p[0], dtype=BF16), None, None, torch.zeros_like(p[3], dtype=F16), None]
    check_32(kernels, p, g, m, v, copies=copies, **{**HYPER, "weight_decay": [0.0, 0.1, 0.2, 0.0, 1.0]})


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("shift", [1, 3, 4])
def test_step_at_unaligned_addresses(kernels, bits, shift):
    """Tensors that start `shift` elements into their buffers; what lies around them stays as it was."""
    n = 5000
    bufs = [rand(n + 16, t, k) for k, t in enumerate((F32, BF16))]
    p, g = ([b[shift:shift + n]] for b in bufs)
    edges = [b.clone() for b in bufs]
    copy_buf = torch.zeros(n + 16, device="cuda", dtype=BF16)
    copies = [copy_buf[shift:shift + n]]
    if bits == 32:
        mb, vb = rand(n + 16, F32, 3, 0.01), rand(n + 16, F32, 4, 0.01).square()
        edges += [mb.clone(), vb.clone()]
        check_32(kernels, p, g, [mb[shift:shift + n]], [vb[shift:shift + n]], copies=copies, **HYPER)
        bufs += [mb, vb]
    else:
        s = state_8([n], 5)
        mb, vb = torch.zeros(2, n + 16, device="cuda").to(E4M3)
        mb[shift:shift + n].copy_(s["exp_avg"][0])
        vb[shift:shift + n].copy_(s["exp_avg_sq"][0])
        s["exp_avg"], s["exp_avg_sq"] = [mb[shift:shift + n]], [vb[shift:shift + n]]
        check_8(kernels, p, g, s, copies=copies, **HYPER)
        mb, vb = mb.float(), vb.float()
        bufs += [mb, vb]
        edges += [torch.zeros_like(mb), torch.zeros_like(vb)]
    edges.append(torch.zeros_like(copy_buf))
    for b, e in zip(bufs + [copy_buf], edges):
        assert torch.equal(b[:shift], e[:shift]) and torch.equal(b[shift + n:], e[shift + n:])


@pytest.mark.parametrize("count", [31, 32, 33, 384, 385, 800])
def test_step_over_many_tensors(kernels, count):
    sizes = [1 + (k * 37) % 301 for k in range(count)]
    p, g, m, v = lists([sum(sizes)], F32, F32)
    parts = [[t for t in torch.split(a[0], sizes)] for a in (p, g, m, v)]
    whole = [a[0].clone() for a in (p, g, m, v)]
    kernels.adamw(*parts, **HYPER)
    kernels.adamw(*([t] for t in whole), **HYPER)
    assert all(torch.equal(a[0], b) for a, b in zip((p, m, v), (whole[0], whole[2], whole[3])))


def test_step_first_steps_and_zero_gradients(kernels):
    """From zeroed states; an element whose gradient and states are zero only decays."""
    p, g, m, v = lists([3000], F32, F32)
    state = kernels.adamw_state(p)
    g[0][::3] = 0.0
    before = p[0].clone()
    check_32(kernels, p, g, state["exp_avg"], state["exp_avg_sq"], **{**HYPER, "step": 1})
    want = before[::3].double() * (1 - 1e-3)
    assert_within(p[0][::3], want, 4 * U * want.abs(), "decayed only")
    check_32(kernels, p, g, state["exp_avg"], state["exp_avg_sq"], **{**HYPER, "step": 2})


def test_step_numbers_on_the_device(kernels):
    p, g, m, v = lists([777, 4096], F32, BF16)
    q, n, w = ([t.clone() for t in ts] for ts in (p, m, v))
    kernels.adamw(p, g, m, v, **HYPER)
    more = {**HYPER, "step": torch.tensor([7], device="cuda"), "lr": torch.tensor([1e-2], device="cuda")}
    kernels.adamw(q, g, n, w, **more)
    for a, b in zip(p + m + v, q + n + w):
        assert_within(a, b.double(), 4 * U * b.double().abs() + 1e-9, "device numbers")
    assert all(torch.equal(a, b) for a, b in zip(m + v, n + w))


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_a_bad_factor_changes_nothing(kernels, bits, bad):
    p, g, m, v = lists([1000, 70], F32, F32)
    kw = {"exp_avg": m, "exp_avg_sq": v} if bits == 32 else state_8([1000, 70], 3)
    flat = [t for ts in ([p] + list(kw.values())) for t in ts]
    before = [t.float().clone() for t in flat]
    kernels.adamw(p, g, grad_scale=torch.tensor([bad], device="cuda"), **kw, **HYPER)
    assert all(torch.equal(a, b.float()) for a, b in zip(before, flat))


def test_a_bad_gradient_stays_in_its_element(kernels):
    p, g, m, v = lists([5000], F32, F32)
    g[0][1234] = math.nan
    check_32(kernels, p, g, m, v, **HYPER)
    assert int(p[0].isnan().sum()) == 1


# ---- 8-bit states -----------------------------------------------------------------
def blocks(t):
    return torch.nn.functional.pad(t, (0, -t.numel() % 256)).view(-1, 256)


def encode(t, floor):
    b = blocks(t)
    s = (b.abs().amax(1) / 448).clamp(min=2.0 ** -120)
    u = b / s[:, None]
    if floor:
        u = torch.where(u > 0, u.clamp(min=2.0 ** -9), u)
    return u.to(E4M3).view(-1)[:t.numel()].clone(), s


def decode(code, scale):
    return code.double() * scale.double().repeat_interleave(256)[:code.numel()]


def state_8(sizes, seed):
    out = {"exp_avg": [], "exp_avg_sq": [], "exp_avg_scales": [], "exp_avg_sq_scales": []}
    for k, n in enumerate(sizes):
        for name, t, floor in (("exp_avg", rand(n, F32, seed + k, 0.01), False),
                               ("exp_avg_sq", rand(n, F32, seed + 50 + k, 0.01).abs(), True)):
            c, s = encode(t, floor)
            out[name].append(c)
            out[name + "_scales"].append(s)
    return out


def check_codes(code, scale, want, bound, floor, what):
    """Scales within their roundings; each code is the value's nearest, up to
    the error of the value before it is rounded."""
    w, e = blocks(want), blocks(bound)
    top = w.abs().amax(1)
    s = (top / 448).clamp(min=2.0 ** -120)
    assert_within(scale, s, e.amax(1) / 448 + 3 * U * s, what + " scale")
    unit = (w / s[:, None]).view(-1)[:code.numel()]
    off = ((e + 5 * U * w.abs()) / s[:, None] + w.abs() / s[:, None] * (e.amax(1) / top.clamp(min=1e-300))[:, None]).view(-1)[:code.numel()]
    step = torch.exp2((unit.abs().clamp(min=2.0 ** -6)).log2().floor() - 3)
    # A value within its error of a power of two may be rounded at the larger step beyond it.
    step = torch.maximum(step, torch.exp2(((unit.abs() + off).clamp(min=2.0 ** -6)).log2().floor() - 3))
    target = torch.where((want > 0) & (unit < 2.0 ** -9), torch.full_like(unit, 2.0 ** -9), unit) if floor else unit
    assert_within(code, target, step / 2 + off, what)
    if floor:
        # v is held in f32, whose smallest value is 2^-149: a product or sum below half of that is zero there and has
        # no root.  v above 2^-146 is a sum of at most two terms of which one is above 2^-147, so it is not zero.
        assert bool((code.float()[want > 2.0 ** -73] > 0).all()), what


def check_8(kernels, p, g, s, copies=None, scale=None, **h):
    want = []
    for k in range(len(p)):
        m, r = decode(s["exp_avg"][k], s["exp_avg_scales"][k]), decode(s["exp_avg_sq"][k], s["exp_avg_sq_scales"][k])
        p1, m1, v1, e_p, e_m, e_v = adam_ref(p[k], g[k], m, r * r, **ref_args(h, k), scale=1.0 if scale is None else scale.item())
        # The decoded values themselves carry a rounding (m) and three (v).
        e_m, e_v = e_m + 2 * U * m.abs(), e_v + 4 * U * r * r
        den = (v1 / (1 - h["betas"][1] ** h["step"])).sqrt() + h["eps"]
        e_p = e_p + h["lr"] / (1 - h["betas"][0] ** h["step"]) / den * (2 * U * m.abs() + 8 * U * m1.abs())
        want.append((p1, m1, v1, e_p, e_m, e_v))
    kernels.adamw(p, g, copies=copies, grad_scale=scale, **s, **h)
    for k, (p1, m1, v1, e_p, e_m, e_v) in enumerate(want):
        if not p1.numel():
            continue
        assert_within(p[k], p1, e_p + rounded(p1.abs() + e_p, p[k].dtype), f"p of {k}")
        check_codes(s["exp_avg"][k], s["exp_avg_scales"][k], m1, e_m, False, f"m of {k}")
        root = v1.sqrt()
        e_r = torch.minimum(e_v / root.clamp(min=1e-300), e_v.sqrt()) + 2 * U * root
        check_codes(s["exp_avg_sq"][k], s["exp_avg_sq_scales"][k], root, e_r, True, f"root of {k}")
        if copies is not None and copies[k] is not None:
            assert_within(copies[k], p1, e_p + rounded(p1.abs() + e_p, copies[k].dtype), f"copy of {k}")


@pytest.mark.parametrize("p_t", [F32, F16, BF16])
@pytest.mark.parametrize("g_t", [F32, F16, BF16])
def test_step_8_bits(kernels, p_t, g_t):
    p, g, _, _ = lists(SIZES, p_t, g_t)
    copies = [torch.zeros_like(t, dtype=BF16) for t in p] if p_t == F32 else None
    check_8(kernels, p, g, state_8(SIZES, 9), copies=copies, scale=torch.tensor([0.5], device="cuda"), **HYPER)


def test_step_8_bits_spread_values(kernels):
    """Blocks whose values span many decades, blocks of zeros, tiny blocks, first steps from zeroed states."""
    n = 256 * 9 + 100
    p, g = [rand(n, F32, 1)], [rand(n, F32, 2)]
    g[0] *= torch.logspace(-9, 3, n, device="cuda")
    g[0][256:512] = 0.0
    g[0][512:768] *= 1e-18
    s = kernels.adamw_state(p, bits=8)
    for step in (1, 2, 3):
        check_8(kernels, p, g, s, **{**HYPER, "step": step})
    assert bool((s["exp_avg"][0][256:512].float() == 0).all()) and bool((s["exp_avg_sq"][0][256:512].float() == 0).all())


def test_step_8_bits_bad_gradient_stays_in_its_block(kernels):
    n = 2000
    p, g = [rand(n, F32, 1)], [rand(n, F32, 2)]
    s, clean = state_8([n], 3), state_8([n], 3)
    q, bad = [p[0].clone()], [g[0].clone()]
    bad[0][700] = math.nan
    kernels.adamw(p, g, **clean, **HYPER)
    kernels.adamw(q, bad, **s, **HYPER)
    keep = torch.ones(n, dtype=torch.bool, device="cuda")
    keep[700] = False
    assert torch.equal(p[0][keep], q[0][keep]) and bool(q[0][700].isnan())
    keep[512:768] = False
    for name in ("exp_avg", "exp_avg_sq"):
        assert torch.equal(s[name][0].float()[keep], clean[name][0].float()[keep])
        assert bool(s[name + "_scales"][0][2].isnan()) and int(s[name + "_scales"][0].isnan().sum()) == 1


def test_long_tensors(kernels):
    """More than 2^31 elements: the far end of a step and of a norm."""
    n = (1 << 31) + 1027
    p, g = [torch.zeros(n, device="cuda", dtype=BF16)], [torch.zeros(n, device="cuda", dtype=BF16)]
    s = kernels.adamw_state(p, bits=8)
    at = [5, (1 << 31) - 1, 1 << 31, n - 1]
    g[0][at] = torch.tensor([3.0, 4.0, 12.0, 84.0], device="cuda", dtype=BF16)
    norm, scale = kernels.grad_norm(g, 17.0)
    assert norm.item() == 85.0 and scale.item() == pytest.approx(0.2, rel=2 * U)  # 3 4 12 84 85
    kernels.adamw(p, g, **s, **{**HYPER, "step": 1, "weight_decay": 0.0})
    # From zeroed states the first step moves by lr where there is a gradient.
    got = p[0][at].double()
    assert_within(got, torch.full_like(got, -1e-2), torch.full_like(got, 1e-2 * (2.0 ** -8 + 1e-6)), "p")
    assert int((p[0] != 0).sum()) == 4
    assert float(s["exp_avg"][0][n - 1].float() * s["exp_avg_scales"][0][-1]) == pytest.approx(8.4, rel=1e-6)


# ---- gradient norm ----------------------------------------------------------------
def check_norm(kernels, grads, max_norm):
    norm, scale = kernels.grad_norm(grads, max_norm)
    exact = math.sqrt(math.fsum(float(g.double().square().sum()) for g in grads))
    # Four roundings of each square and of the short sums at most, halved by the root, and the last one.
    assert abs(norm.item() - exact) <= 3.001 * U * exact
    assert scale.item() == pytest.approx(min(1.0, max_norm / exact) if exact else 1.0, rel=4 * U)
    return norm, scale


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_norm_sizes(kernels, dtype):
    for sizes in ([1], [7], [8192], [8193, 0, 1, 3], SIZES, [1 + k % 50 for k in range(1500)]):
        check_norm(kernels, [rand(n, dtype, k) for k, n in enumerate(sizes)], 0.5)


def test_norm_mixed_unaligned_and_rank(kernels):
    a = rand(5000, F32, 1)[1:4001].view(40, 100)
    b = rand(5000, BF16, 2)[3:]
    c = rand(1 << 20, F16, 3)[1:]
    check_norm(kernels, [a, b, c], 1e9)
    check_norm(kernels, [a, a, a], 1.0)  # the same tensor may be listed again


def test_norm_extremes(kernels):
    big = torch.full((1000,), 1e30, device="cuda")
    check_norm(kernels, [big], 1.0)
    check_norm(kernels, [big * 1e-60, torch.full((9,), 1e-30, device="cuda")], 1.0)
    tiny = torch.full((70,), 2.0 ** -140, device="cuda")
    norm, _ = kernels.grad_norm([tiny], 1.0)
    assert norm.item() == pytest.approx(math.sqrt(70) * 2.0 ** -140, abs=2.0 ** -150)
    check_norm(kernels, [torch.cat([tiny, rand(100000, F32, 1, 1e-20), big])], 1.0)
    zero, one = kernels.grad_norm([torch.zeros(100, device="cuda")], 1.0)
    assert zero.item() == 0.0 and one.item() == 1.0
    none, one = kernels.grad_norm([], 1.0)
    assert none.item() == 0.0 and one.item() == 1.0
    only, no_scale = kernels.grad_norm([big])
    assert no_scale is None and only.item() > 0
    for bad in (math.inf, math.nan):
        g = rand(3000, F32, 1)
        g[1700] = bad
        norm, scale = kernels.grad_norm([rand(10, BF16, 2), g], 1.0)
        assert (math.isinf(norm.item()) if math.isinf(bad) else math.isnan(norm.item())) and math.isnan(scale.item())


def test_norm_same_bits_every_time(kernels):
    g = [rand(n, BF16, n) for n in (3_000_001, 77, 500_000)]
    first = kernels.grad_norm(g, 1.0)
    for _ in range(4):
        assert all(torch.equal(a, b) for a, b in zip(kernels.grad_norm(g, 1.0), first))


# ---- the operators together -------------------------------------------------------
def train(kernels, steps, bits, captured):
    """y = layer_norm(x) over a learned weight and bias and a second norm after
    a fixed map; loss = sum(y * c) / rows: gradients, clip, step, all on the device."""
    rows, n = 96, 200
    x, c = rand(rows * n, F32, 1).view(rows, n), rand(rows * n, F32, 2).view(rows, n) / rows
    params = [torch.ones(n, device="cuda"), torch.zeros(n, device="cuda"), torch.ones(n, device="cuda"), torch.zeros(n, device="cuda")]
    copies = [torch.zeros(n, device="cuda", dtype=BF16) for _ in params]
    state = kernels.adamw_state(params, bits=bits)
    step, lr = torch.zeros(1, dtype=torch.int64, device="cuda"), torch.full((1,), 1e-2, device="cuda")
    norms = []

    def one():
        h, m1, r1 = kernels.layer_norm(x, params[0], params[1])
        _, m2, r2 = kernels.layer_norm(h, params[2], params[3])
        dh, dw2, db2 = kernels.layer_norm_backward(c, h, m2, r2, params[2])
        _, dw1, db1 = kernels.layer_norm_backward(dh, x, m1, r1, params[0], dx=dh)
        grads = [dw1, db1, dw2, db2]
        norm, scale = kernels.grad_norm(grads, 0.05)
        step.add_(1)
        kernels.adamw(params, grads, **state, step=step, lr=lr, betas=(0.9, 0.99), weight_decay=0.0, copies=copies,
                      grad_scale=scale)
        return norm

    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = one()
        for _ in range(steps):
            graph.replay()
            norms.append(out.item())
    else:
        for _ in range(steps):
            norms.append(one().item())
    assert all(torch.equal(a, b.to(BF16)) for a, b in zip(copies, params))
    return [p.clone() for p in params], norms, (x, c)


@pytest.mark.parametrize("bits", [8, 32])
def test_training_steps_eager_and_captured(kernels, bits):
    a, na, _ = train(kernels, 4, bits, False)
    b, nb, _ = train(kernels, 4, bits, True)
    assert na == nb and all(torch.equal(p, q) for p, q in zip(a, b))


def test_gradients_of_the_run(kernels):
    """The chain's gradients against autograd of the formula in 64 bits."""
    rows, n = 96, 200
    _, norms, (x, c) = train(kernels, 1, 32, False)
    w = [torch.ones(n, device="cuda", dtype=torch.float64, requires_grad=True) for _ in range(2)]
    b = [torch.zeros(n, device="cuda", dtype=torch.float64, requires_grad=True) for _ in range(2)]
    h = x.double()
    for k in range(2):
        off = h - h.mean(-1, keepdim=True)
        h = off / (off.square().mean(-1, keepdim=True) + 1e-5).sqrt() * w[k] + b[k]
    (h * c.double()).sum().backward()
    exact = torch.stack([t.grad.square().sum() for t in (*w, *b)]).sum().sqrt().item()
    # Every element of the gradients is a sum over 96 rows of terms a few dozen roundings off: 200 roundings bound them all.
    total = torch.stack([(t.grad.abs().sum()) for t in (*w, *b)]).sum().item()
    assert abs(norms[0] - exact) <= 200 * U * (exact + total)
    _, m, r, *_ = norm_ref(x, None, None, 1e-5)
    assert norm_back_ref(c, x, m, r, None)[0].shape == (rows, n)


def test_other_stream(kernels):
    p, g, m, v = lists([1000, 5], F32, F32)
    q, n, w = ([t.clone() for t in ts] for ts in (p, m, v))
    norm, scale = kernels.grad_norm(g, 0.1)
    kernels.adamw(p, g, m, v, grad_scale=scale, **HYPER)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    norm2, scale2 = kernels.grad_norm(g, 0.1, stream=side)
    kernels.adamw(q, g, n, w, grad_scale=scale2, stream=side, **HYPER)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(p + m + v + [norm, scale], q + n + w + [norm2, scale2]))


def test_refusals(kernels):
    err = spmd_mod("_lib").SpmdError
    p, g, m, v = lists([100, 300], F32, F32)
    s = state_8([100, 300], 3)
    go = lambda **kw: kernels.adamw(**{**{"params": p, "grads": g, "exp_avg": m, "exp_avg_sq": v}, **HYPER, **kw})  # noqa: E731
    for call, kind in (
        (lambda: go(grads=g[:1]), ValueError),
        (lambda: go(grads=[g[0], g[1].cpu()]), ValueError),
        (lambda: go(grads=[g[0], g[1].view(3, 100)]), ValueError),
        (lambda: go(grads=[g[0], g[1].double()]), TypeError),
        (lambda: go(grads=[g[0], rand(600, F32, 1)[::2]]), ValueError),
        (lambda: go(exp_avg=[m[0], m[1].half()]), TypeError),
        (lambda: go(exp_avg=s["exp_avg"], exp_avg_sq=s["exp_avg_sq"]), TypeError),
        (lambda: go(**{**s, "exp_avg_scales": None}), ValueError),
        (lambda: go(**{**s, "exp_avg_scales": s["exp_avg_scales"][::-1]}), ValueError),
        (lambda: go(copies=[None]), ValueError),
        (lambda: go(copies=[None, torch.zeros(300, device="cuda")]), TypeError),
        (lambda: go(weight_decay=[0.1]), ValueError),
        (lambda: go(weight_decay=-0.1), err),
        (lambda: go(step=0), err),
        (lambda: go(lr=-1.0), err),
        (lambda: go(lr=math.nan), err),
        (lambda: go(lr=torch.tensor([1e-3, 1e-3], device="cuda")), ValueError),
        (lambda: go(step=torch.tensor([1.0], device="cuda")), ValueError),
        (lambda: go(grad_scale=torch.ones(1)), ValueError),
        (lambda: go(betas=(1.0, 0.9)), err),
        (lambda: go(betas=(0.9, -0.1)), err),
        (lambda: go(eps=-1e-8), err),
        (lambda: go(exp_avg_sq=m), err),
        (lambda: go(params=[p[0], p[0]], grads=[g[0], g[0]], exp_avg=[m[0], m[1][:100]], exp_avg_sq=[v[0], v[1][:100]]), err),
        (lambda: go(grads=p), err),
        (lambda: kernels.grad_norm([g[0].double()], 1.0), TypeError),
        (lambda: kernels.grad_norm([g[0].cpu()], 1.0), ValueError),
        (lambda: kernels.grad_norm([rand(600, F32, 1)[::2]], 1.0), ValueError),
        (lambda: kernels.grad_norm(g, -1.0), err),
        (lambda: kernels.grad_norm(g, math.nan), err),
        (lambda: kernels.grad_norm(g, 1.0, ws=torch.empty(4, device="cuda")), err),
        (lambda: kernels.adamw_state(p, bits=4), ValueError),
    ):
        with pytest.raises(kind):
            call()
    # A gradient may serve two parameters; nothing above changed a tensor.
    q, gg, n, w = lists([100, 300], F32, F32)
    assert all(torch.equal(a, b) for a, b in zip(p + g + m + v, q + gg + n + w))
    half = [g[0][:100], g[1][:100]]
    kernels.adamw([p[0], p[1][:100]], [half[0], half[0]], [m[0], m[1][:100]], [v[0], v[1][:100]], **HYPER)
