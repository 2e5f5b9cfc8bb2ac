"""Views that torch negates lazily (the imaginary part of a conjugate): their memory holds other values than they do,
so that the operators of a training step refuse them."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


def test_negated_views_are_refused(kernels):
    c = torch.randn(6, 40, device="cuda", dtype=torch.complex64)
    x, plain = c.conj().imag, c.imag
    assert x.is_neg() and x.dtype == torch.float32 and torch.equal(x, -plain)
    y, mean, rstd = kernels.layer_norm(x.resolve_neg())
    state = kernels.adamw_state([mean])
    flat = torch.view_as_complex(torch.zeros(6, 2, device="cuda")).conj().imag
    whole = torch._neg_view(torch.ones(6, device="cuda"))
    for call in (lambda: kernels.layer_norm(x), lambda: kernels.layer_norm(y, out=x),
                 lambda: kernels.layer_norm_backward(x, y, mean, rstd), lambda: kernels.layer_norm_backward(y, x, mean, rstd),
                 lambda: kernels.layer_norm_backward(y, y, mean, rstd, dx=x),
                 lambda: kernels.grad_norm([flat]), lambda: kernels.grad_norm([whole]),
                 lambda: kernels.adamw([mean.clone()], [whole], **state, step=1, lr=0.1),
                 lambda: kernels.adamw([whole], [mean], **state, step=1, lr=0.1)):
        with pytest.raises(ValueError):
            call()
    # The plain part of the same memory is a strided view like any other.
    got = kernels.layer_norm(plain)[0]
    # A norm of the negated rows, by other lanes: 40 roundings of 2^-24 at the most on values below 40 ** 0.5.
    assert float((got + y).abs().max()) <= 40 * 2.0 ** -24 * 40 ** 0.5
