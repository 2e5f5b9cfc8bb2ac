"""Calls that write given tensors raise their version counters: autograd refuses a graph that saved them before."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")
from conftest import spmd_mod  # noqa: E402

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def test_a_step_between_forward_and_backward_is_refused(kernels):
    p = torch.ones(1000, device="cuda", requires_grad=True)
    g = torch.ones(1000, device="cuda")
    state = kernels.adamw_state([p])
    loss = (p * p).sum()
    kernels.adamw([p], [g], **state, step=1, lr=0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    (p * p).sum().backward()  # and a graph built after the step is fine
    assert torch.equal(p.grad, 2 * p.detach())


def versions(ts):
    return [t._version for t in ts]


@pytest.mark.parametrize("bits", [8, 32])
def test_a_step_raises_parameters_and_copies_and_no_gradient(kernels, bits):
    p = [torch.ones(n, device="cuda") for n in (300, 7)]
    g = [torch.ones(n, device="cuda") for n in (300, 7)]
    copies = [torch.zeros(300, device="cuda", dtype=BF16), None]
    state = kernels.adamw_state(p, bits=bits)
    written = [*p, copies[0]]
    before, grads = versions(written), versions(g)
    norm, scale = kernels.grad_norm(g, 1.0)
    kernels.adamw(p, g, **state, copies=copies, grad_scale=scale, step=1, lr=0.1)
    assert all(b > a for a, b in zip(before, versions(written))) and versions(g) == grads and norm._version == 0
    before = versions(written)
    with pytest.raises(spmd_mod("_lib").SpmdError):
        kernels.adamw(p, g, **state, step=0, lr=0.1)
    assert versions(written) == before  # a refused call writes nothing


def test_layer_norm_raises_given_outputs(kernels):
    x, w = torch.randn(8, 64, device="cuda"), torch.ones(64, device="cuda")
    y, mean, rstd = kernels.layer_norm(x, w)
    assert versions([x, w, y, mean, rstd]) == [0] * 5
    out, dx, dw, db = torch.empty_like(x), torch.empty_like(x), torch.empty_like(w), torch.empty_like(w)
    kernels.layer_norm(x, w, out=out)
    kernels.layer_norm_backward(y, x, mean, rstd, w, dx=dx, dweight=dw, dbias=db)
    assert versions([out, dx, dw, db]) == [1] * 4 and versions([x, w, y, mean, rstd]) == [0] * 5
    leaf = torch.randn(8, 64, device="cuda", requires_grad=True)
    loss = leaf.square().sum()
    kernels.layer_norm(leaf, out=leaf)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_inference_tensors_have_no_counter(kernels):
    with torch.inference_mode():
        p, g = [torch.ones(300, device="cuda")], [torch.ones(300, device="cuda")]
        state = kernels.adamw_state(p)
        x = torch.randn(4, 32, device="cuda")
        kernels.adamw(p, g, **state, step=1, lr=0.1)
    kernels.adamw(p, g, **state, step=2, lr=0.1)
    kernels.layer_norm(x, out=x)
    assert bool((p[0] < 1).all())
