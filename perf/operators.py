"""The training-step operators measured on a GPU: layer norm forward and backward, the gradient norm over many tensors,
and the AdamW step over many tensors with states in 32 or in 8 bits.

`own` chooses between the plain form (elementary torch operations) and the library's kernels.
"""
import functools
import importlib
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-5
BLOCK = 256  # elements that share one scale of an 8-bit state
ALIGN = 256  # every tensor of a flat buffer starts at a multiple of this many elements
TOP = 448.0  # the largest e4m3 value
LEAST = 2.0 ** -120  # the smallest scale of a block
TINY = 2.0 ** -9  # the smallest e4m3 value above zero
OPT = {"lr": 3e-4, "betas": (0.9, 0.95), "eps": 1e-8, "weight_decay": 0.1, "step": 1000}
MAX_NORM = 1.0


def listed():
    return [
        # One new token of one request on its way through a served layer: latency alone.
        norm("norm of one token", 1, 4096, "bf16", "bf16", "bf16", stats=False),
        # A packed batch whose row length is odd: no row but the first begins on a 16-byte boundary.
        norm("norm of odd rows", 16384, 1001, "f16", "f16", "f32"),
        # A training batch: the residual stream in 32 bits, the layer's input in 16, the statistics kept for the way back.
        norm("norm of a training batch", 65536, 4096, "f32", "bf16", "f32"),
        # The same layer's gradients at 16 bits throughout, weights included.
        back("norm gradient of a batch", 32768, 4096, "bf16", "bf16", "bf16"),
        # Norms over single heads: very many short rows, where the weight's gradient is a long sum over few columns.
        back("norm gradient of heads", 262144, 64, "f16", "f16", "f32"),
        # A few very long rows (whole images or feature maps normalised at once).
        back("norm gradient of long rows", 24, 262144, "f32", "f32", "f32"),
        # The norm of a small model's gradients before clipping: many tensors of very different, odd sizes.
        grads("gradient norm, small tensors", 96, 1 << 20, "f32"),
        # The norm of a large model's 16-bit gradients.
        grads("gradient norm, large", 48, 1 << 28, "bf16"),
        # A small model or a set of adapters: many little tensors in 32 bits, where launches and the host count.
        adamw("step, small tensors", 96, 1 << 20, "f32", "f32", "none", 32),
        # Mixed-precision training: 32-bit parameters, 16-bit gradients and the 16-bit copy that the next forward pass reads.
        adamw("step, mixed precision", 48, 1 << 28, "f32", "bf16", "bf16", 32),
        # Fine-tuning in 16 bits with states in 8 bits, to fit a larger model.
        adamw("step, 8-bit states", 40, 1 << 27, "bf16", "bf16", "none", 8),
        # One odd-sized 32-bit tensor with 8-bit states.
        adamw("step, one tensor in 8 bits", 1, 1000003, "f32", "f32", "none", 8),
    ]


def norm(name, rows, cols, x, y, w, pitch=0, stats=True):
    return {"name": name, "op": "norm", "rows": rows, "cols": cols, "x": x, "y": y, "w": w, "pitch": pitch, "stats": stats}


def back(name, rows, cols, x, y, w, pitch=0):
    return {"name": name, "op": "back", "rows": rows, "cols": cols, "x": x, "y": y, "w": w, "pitch": pitch}


def grads(name, tensors, elements, g):
    return {"name": name, "op": "grads", "tensors": tensors, "elements": elements, "g": g, "sizes": 1}


def adamw(name, tensors, elements, p, g, copy, bits):
    return {"name": name, "op": "adamw", "tensors": tensors, "elements": elements, "p": p, "g": g, "copy": copy, "bits": bits, "sizes": 1}


def between(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["norm", "norm", "back", "back", "grads", "adamw", "adamw"])
    if op in ("norm", "back"):
        cols = between(rng, 8, 1 << 18)
        rows = between(rng, 1, max(1, min(1 << 18, (1 << 27) // cols)))
        x, y = rng.choice([("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "bf16"), ("f32", "f16"), ("bf16", "f32"), ("f16", "f32")])
        w = rng.choice(["f32", x, "none"])
        pitch = rng.choice([0, 0, cols + between(rng, 1, 500)])
        c = norm("", rows, cols, x, y, w, pitch, rng.random() < 0.7) if op == "norm" else back("", rows, cols, x, y, w, pitch)
    elif op == "grads":
        tensors = between(rng, 1, 400)
        c = grads("", tensors, between(rng, tensors, 1 << 28), rng.choice(["f32", "bf16", "f16"]))
    else:
        tensors, bits = between(rng, 1, 400), rng.choice([32, 8])
        p, g, copy = rng.choice([("f32", "f32", "none"), ("f32", "bf16", "bf16"), ("f32", "f16", "f16"), ("bf16", "bf16", "none"), ("f32", "f32", "bf16"), ("f16", "f16", "none"), ("bf16", "f32", "none")])
        c = adamw("", tensors, between(rng, tensors, 1 << 27), p, g, copy, bits)
    if "sizes" in c:
        c["sizes"] = rng.randrange(1 << 20)
    del c["name"]
    return c


def sizes_of(case):
    """Sizes of the case's tensors: they differ by up to a factor of a thousand, are mostly odd, and sum to about `elements`."""
    rng, n = random.Random(case["sizes"]), case["tensors"]
    shares = [math.exp(rng.uniform(0, math.log(1000))) for _ in range(n)]
    return [max(1, int(case["elements"] * s / sum(shares))) for s in shares] if n > 1 else [case["elements"]]


def work(case):
    if case["op"] in ("norm", "back"):
        r, n, sx, sy, sw = case["rows"], case["cols"], SIZE[case["x"]], SIZE[case["y"]], SIZE.get(case["w"], 0)
        if case["op"] == "norm":
            return {"bytes": r * n * (sx + sy) + 2 * n * sw + 8 * r * case["stats"], "flops": 8 * r * n}
        return {"bytes": r * n * (2 * sx + sy) + 8 * r + 3 * n * sw, "flops": 15 * r * n}
    sizes = sizes_of(case)
    n = sum(sizes)
    if case["op"] == "grads":
        return {"bytes": n * SIZE[case["g"]] + 8, "flops": 2 * n}
    state = 16 * n if case["bits"] == 32 else 4 * n + 16 * sum(-(-s // BLOCK) for s in sizes)
    return {"bytes": n * (2 * SIZE[case["p"]] + SIZE[case["g"]] + SIZE.get(case["copy"], 0)) + state, "flops": 16 * n}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    if case["op"] in ("norm", "back"):
        return {"case": case, **prepare_norm(case, normal)}
    return {"case": case, **prepare_tensors(case, normal)}


def prepare_norm(case, normal):
    rows, cols, width = case["rows"], case["cols"], max(case["cols"], case["pitch"])

    def wide(kind, shift=0.0):
        t = normal(rows, width)
        return (t if not shift else t.add_(shift * normal(rows, 1))).to(TYPES[kind])[:, :cols]

    x = wide(case["x"], 0.5)  # rows whose mean is not zero
    w = b = None
    if case["w"] != "none":
        w, b = (1 + 0.2 * normal(cols)).to(TYPES[case["w"]]), (0.2 * normal(cols)).to(TYPES[case["w"]])
    state = {"x": x, "w": w, "b": b}
    if case["op"] == "back":
        parts = [part.double() for part in x.split(max(1, (1 << 25) // cols))]
        mean, var = torch.cat([t.mean(1) for t in parts]), torch.cat([t.var(1, unbiased=False) for t in parts])
        state.update(dy=wide(case["y"]), mean=mean.float(), rstd=(var + EPS).rsqrt().float())
    return state


def prepare_tensors(case, normal):
    sizes = sizes_of(case)
    starts, total = [], 0
    for n in sizes:
        starts.append(total)
        total += -(-n // ALIGN) * ALIGN
    views = [(a, a + n) for a, n in zip(starts, sizes)]

    def flat(values, kind):
        t = values.to(kind)
        return t, [t[a:b] for a, b in views]

    # Gradients of every tensor have a level of their own, from 1e-5 to 1e-2, as layers do.
    level = torch.repeat_interleave((10 ** (-3.5 + normal(len(sizes)).clamp(-1.5, 1.5))), torch.tensor([-(-n // ALIGN) * ALIGN for n in sizes], device="cuda"))
    g, gs = flat(normal(total) * level, TYPES[case["g"]])
    state = {"g": g, "gs": gs}
    if case["op"] == "grads":
        return state
    state["p"], state["ps"] = flat(0.05 * normal(total), TYPES[case["p"]])
    state["copy"], state["copies"] = flat(state["p"], TYPES[case["copy"]]) if case["copy"] != "none" else (None, None)
    m, v = 0.3 * normal(total) * level, (0.5 + normal(total).square()) * level.square()
    if case["bits"] == 32:
        state["m"], state["ms"] = flat(m, torch.float32)
        state["v"], state["vs"] = flat(v, torch.float32)
    else:
        keep = torch.zeros(total, dtype=torch.bool, device="cuda")
        for a, b in views:
            keep[a:b] = True
        for name, t in (("m", m), ("v", v.sqrt())):
            code, scale = to_8_bits(t * keep)
            state[name], state[name + "s"] = flat(code, torch.float8_e4m3fn)
            state[name + "_scale"] = scale
            state[name + "_scales"] = [scale[a // BLOCK:-(-b // BLOCK)] for a, b in views]
    state["grad_scale"] = torch.full((1,), 0.75, device="cuda")
    return state


def to_8_bits(t, floor=False):
    """Codes and scales of a tensor whose length is a multiple of BLOCK; with `floor` values above zero keep the smallest code at least."""
    blocks = t.view(-1, BLOCK)
    scale = (blocks.abs().amax(1) / TOP).clamp(min=LEAST)
    units = blocks / scale[:, None]
    if floor:
        units = torch.where(units > 0, units.clamp(min=TINY), units)
    return units.to(torch.float8_e4m3fn).view(-1), scale


@functools.cache
def kernels():
    return importlib.import_module("spmd-dialect_b200.kernels")


def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        return RUN_OWN[op](state, case)
    return RUN_PLAIN[op](state, case)


def own_norm(s, case):
    y, mean, rstd = kernels().layer_norm(s["x"], s["w"], s["b"], eps=EPS, dtype=TYPES[case["y"]], stats=case["stats"])
    return {"y": y, "mean": mean, "rstd": rstd}


def own_back(s, case):
    dx, dw, db = kernels().layer_norm_backward(s["dy"], s["x"], s["mean"], s["rstd"], s["w"])
    return {"dx": dx, "dw": dw, "db": db}


def own_grads(s, case):
    length, scale = kernels().grad_norm(s["gs"], MAX_NORM)
    return {"norm": length, "scale": scale}


def own_adamw(s, case):
    more = {"exp_avg_scales": s["m_scales"], "exp_avg_sq_scales": s["v_scales"]} if case["bits"] == 8 else {}
    kernels().adamw(s["ps"], s["gs"], s["ms"], s["vs"], copies=s["copies"], grad_scale=s["grad_scale"], **OPT, **more)
    return updated(s)


def updated(s):
    return {k: s[k] for k in ("p", "copy", "m", "v", "m_scale", "v_scale") if s.get(k) is not None}


def plain_norm(s, case):
    x = s["x"].float()
    mean = x.mean(1, keepdim=True)
    off = x - mean
    rstd = (off.square().mean(1, keepdim=True) + EPS).rsqrt()
    y = off * rstd
    if s["w"] is not None:
        y = y * s["w"].float() + s["b"].float()
    y = y.to(TYPES[case["y"]])
    return {"y": y, "mean": mean[:, 0] if case["stats"] else None, "rstd": rstd[:, 0] if case["stats"] else None}


def plain_back(s, case):
    dy, x, rstd = s["dy"].float(), s["x"].float(), s["rstd"][:, None]
    xh = (x - s["mean"][:, None]) * rstd
    a = dy if s["w"] is None else dy * s["w"].float()
    dx = (a - a.mean(1, keepdim=True) - xh * (a * xh).mean(1, keepdim=True)) * rstd
    dx = dx.to(s["x"].dtype)
    if s["w"] is None:
        return {"dx": dx, "dw": None, "db": None}
    return {"dx": dx, "dw": (dy * xh).sum(0).to(s["w"].dtype), "db": dy.sum(0).to(s["w"].dtype)}


def plain_grads(s, case):
    total = torch.stack([g.double().square().sum() for g in s["gs"]]).sum()
    length = total.sqrt()
    return {"norm": length.float().view(1), "scale": (MAX_NORM / length).clamp(max=1).float().view(1)}


def plain_adamw(s, case):
    m_scales, v_scales = (s["m_scales"], s["v_scales"]) if case["bits"] == 8 else (s["ms"], s["vs"])
    step = plain_step_8 if case["bits"] == 8 else plain_step_32
    copies = s["copies"] or s["ps"]
    [step(*tensors, s["grad_scale"]) for tensors in zip(s["ps"], s["gs"], s["ms"], s["vs"], m_scales, v_scales, copies)]
    return updated(s)


def plain_update(p, g, m, v, grad_scale):
    b1, b2 = OPT["betas"]
    g = g.float() * grad_scale
    m = m * b1 + g * (1 - b1)
    v = v * b2 + g * g * (1 - b2)
    p = p.float() * (1 - OPT["lr"] * OPT["weight_decay"])
    root = (v / (1 - b2 ** OPT["step"])).sqrt() + OPT["eps"]
    return p - OPT["lr"] / (1 - b1 ** OPT["step"]) * m / root, m, v


def plain_step_32(p, g, m, v, _, __, copy, grad_scale):
    new, m1, v1 = plain_update(p, g, m, v, grad_scale)
    m.copy_(m1)
    v.copy_(v1)
    p.copy_(new)
    copy.copy_(new)


def plain_step_8(p, g, m, v, m_scale, v_scale, copy, grad_scale):
    n = p.numel()
    each = lambda t: t.repeat_interleave(BLOCK)[:n]  # noqa: E731
    full = lambda t: torch.nn.functional.pad(t, (0, -n % BLOCK))  # noqa: E731
    new, m1, v1 = plain_update(p, g, m.float() * each(m_scale), (v.float() * each(v_scale)).square(), grad_scale)
    for code, scale, value, floor in ((m, m_scale, m1, False), (v, v_scale, v1.sqrt(), True)):
        c, s = to_8_bits(full(value), floor)
        code.copy_(c[:n])
        scale.copy_(s)
    p.copy_(new)
    copy.copy_(new)


RUN_OWN = {"norm": own_norm, "back": own_back, "grads": own_grads, "adamw": own_adamw}
RUN_PLAIN = {"norm": plain_norm, "back": plain_back, "grads": plain_grads, "adamw": plain_adamw}


def exact(case, seed):
    """The operators' definitions in 64 bits, on the same inputs."""
    s = prepare(case, seed)
    return {"norm": exact_norm, "back": exact_back, "grads": exact_grads, "adamw": exact_adamw}[case["op"]](s, case)


def exact_norm(s, case):
    x = s["x"].to(torch.float64)
    n = x.shape[1]
    mean = x.sum(dim=1) / n
    x -= mean.unsqueeze(1)
    deviation = torch.sqrt(torch.linalg.vector_norm(x, dim=1).square() / n + EPS)
    x /= deviation.unsqueeze(1)
    if s["w"] is not None:
        x *= s["w"].to(torch.float64).unsqueeze(0)
        x += s["b"].to(torch.float64).unsqueeze(0)
    return {"y": x, "mean": mean if case["stats"] else None, "rstd": deviation.reciprocal() if case["stats"] else None}


def exact_back(s, case):
    """dx as the product of dy w with the Jacobian (I - 1/n - xh xh'/n) rstd, the sums as matrix products."""
    x, n = s["x"].to(torch.float64), s["x"].shape[1]
    rstd = s["rstd"].to(torch.float64).unsqueeze(1)
    xh = (x - s["mean"].to(torch.float64).unsqueeze(1)).mul_(rstd)
    del x
    dy = s["dy"].to(torch.float64)
    ones = torch.ones(1, dy.shape[0], dtype=torch.float64, device=dy.device)
    dw = db = None
    if s["w"] is not None:
        db = (ones @ dy)[0]
        dw = (ones @ (dy * xh))[0]
        dy *= s["w"].to(torch.float64)
    along = torch.einsum("rn,rn->r", dy, xh) / n
    dy -= dy.sum(dim=1, keepdim=True) / n
    dy -= xh.mul_(along.unsqueeze(1))
    return {"dx": dy.mul_(rstd), "dw": dw, "db": db}


def exact_grads(s, case):
    parts = [torch.linalg.vector_norm(g.to(torch.float64)) for g in s["gs"]]
    length = math.sqrt(math.fsum(float(t) ** 2 for t in parts))
    out = torch.tensor([length, min(1.0, MAX_NORM / length) if length else 1.0], dtype=torch.float64)
    return {"norm": out[:1], "scale": out[1:]}


def exact_adamw(s, case):
    """Each tensor's step in 64 bits; the buffers' padding as it was."""
    out = {k: (t.clone() if t.dtype == torch.float8_e4m3fn else t.to(torch.float64)) for k, t in updated(s).items()}
    (b1, b2), t, at = OPT["betas"], OPT["step"], 0
    for k, n in enumerate(sizes_of(case)):
        g = s["gs"][k].to(torch.float64) * s["grad_scale"].item()
        b0, b9 = at // BLOCK, at // BLOCK + -(-n // BLOCK)
        if case["bits"] == 8:
            spread = torch.arange(n, device=g.device) // BLOCK
            m = s["ms"][k].to(torch.float64) * s["m_scale"][b0:b9].to(torch.float64)[spread]
            v = (s["vs"][k].to(torch.float64) * s["v_scale"][b0:b9].to(torch.float64)[spread]) ** 2
        else:
            m, v = s["ms"][k].to(torch.float64), s["vs"][k].to(torch.float64)
        m = torch.lerp(g, m, b1)
        v = torch.lerp(g.square(), v, b2)
        p = s["ps"][k].to(torch.float64)
        change = m / (1 - math.pow(b1, t)) / (torch.sqrt(v / (1 - math.pow(b2, t))) + OPT["eps"]) + OPT["weight_decay"] * p
        p = p - OPT["lr"] * change
        out["p"][at:at + n] = p
        if "copy" in out:
            out["copy"][at:at + n] = p
        if case["bits"] == 8:
            for name, value in (("m", m), ("v", torch.sqrt(v))):
                scale = torch.zeros((b9 - b0) * BLOCK, dtype=torch.float64, device=g.device)
                scale[:n] = value.abs()
                scale = torch.clamp(scale.view(-1, BLOCK).max(dim=1).values / TOP, min=LEAST)
                units = value / scale[spread]
                if name == "v":
                    units = torch.where(value > 0, torch.clamp(units, min=TINY), units)
                out[name][at:at + n] = units.to(torch.float8_e4m3fn)
                out[name + "_scale"][b0:b9] = scale
        else:
            out["m"][at:at + n], out["v"][at:at + n] = m, v
        at += -(-n // ALIGN) * ALIGN
    return out
