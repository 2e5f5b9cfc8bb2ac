"""Layer norm on rows whose values lie far from zero, NaN and infinity in long
and in strided rows: where one share of a row's sums is empty, or a value
outside the row takes part with a factor of zero, the products have to stay
finite."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")
from test_gpu_layer_norm import BF16, F32, check_forward, make, weights  # noqa: E402
from train_ref import assert_within, norm_back_ref, rounded  # noqa: E402

pytestmark = pytest.mark.gpu

# (columns, view): two passes over runs, the same with rows that start within a vector, strided columns that a
# cluster's blocks read, and those of a row of several runs.
ROWS = [(70000, "whole"), (70001, "whole"), (60000, "shifted"), (5000, "strided"), (70000, "strided")]


def view(t, kind):
    """`t` as a view of a wider buffer."""
    rows, cols = t.shape
    if kind == "whole":
        return t
    if kind == "shifted":
        out = t.new_zeros(rows, cols + 5)[:, 3:cols + 3]
    else:
        out = t.new_zeros(rows, 2 * cols)[:, ::2]
    out.copy_(t)
    return out


@pytest.mark.parametrize("x_t,y_t", [(F32, F32), (BF16, BF16), (F32, BF16)])
@pytest.mark.parametrize("cols,kind", ROWS)
def test_far_means_of_long_and_strided_rows(kernels, cols, kind, x_t, y_t):
    """Means of 2^64 and more, whose square leaves f32, while the variance does not."""
    x = make((6, cols), F32, 1)
    x[0] = 1e20
    x[1] = 1e20 + 4e16 * x[1]  # squares' sum 1.1e38 at 70000 columns
    x[2] = -3e25
    x[4] = 1e20 * torch.sign(x[4]) * 1e-6
    x = view(x.to(x_t), kind)
    w, b = weights(cols, F32, 3)
    # bf16 holds 1e20 to 2^58, so that row 1 is off its mean by some 2.4e17 there: 70000 squares are 4e39, which is past
    # f32's 3.4e38.  Such a sum is infinite, rstd zero and y the bias.
    past = (x.double() - x.double().mean(-1, keepdim=True)).square().sum(-1) > 2.0 ** 128 * 1.1
    assert past.tolist() == [False, x_t == BF16 and cols > 6000, False, False, False, False]
    for rows in (x[:1], x[2:]) if bool(past[1]) else (x,):
        check_forward(kernels, rows, w, b, ydtype=y_t)
    y, mean, rstd = kernels.layer_norm(x, w, b, dtype=y_t)
    assert bool((rstd[past] == 0).all()) and torch.equal(y[past], b.to(y_t).expand_as(y)[past])
    assert bool(y.isfinite().all()) and bool(mean.isfinite().all()) and bool(rstd.isfinite().all())


@pytest.mark.parametrize("cols,kind", ROWS)
def test_a_bad_row_stays_alone_in_long_and_strided_rows(kernels, cols, kind):
    x, dy = make((9, cols), F32, 1), make((9, cols), F32, 2)
    bad = x.clone()
    bad[4, cols // 2] = float("nan")
    bad[6, 0] = float("inf")
    bad[7, cols - 1] = float("-inf")
    x, bad, dy = view(x, kind), view(bad, kind), view(dy, kind)
    w, b = weights(cols, F32, 3)
    y, mean, rstd = kernels.layer_norm(x, w, b)
    y1, mean1, rstd1 = kernels.layer_norm(bad, w, b)
    dx, _, _ = kernels.layer_norm_backward(dy, x, mean, rstd, w, wgrad=False)
    dx1, _, _ = kernels.layer_norm_backward(dy, bad, mean1, rstd1, w, wgrad=False)
    good = [0, 1, 2, 3, 5, 8]
    for p, q in ((y, y1), (mean, mean1), (rstd, rstd1), (dx, dx1)):
        assert torch.equal(p[good], q[good])
    for t in (y1, dx1):
        assert all(bool(t[k].isnan().all()) for k in (4, 6, 7))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("apart", [False, True])
@pytest.mark.parametrize("cols", [5, 37, 100, 1001, 4096, 5003, 8200, 20001, 60001])
def test_gradients_of_constant_far_rows(kernels, cols, apart, dtype):
    """A constant row has xh = 0 and a finite gradient, also where mean * rstd leaves f32."""
    x, dy = torch.full((5, cols), 1e33, device="cuda"), make((5, cols), dtype, 2)
    x[1] = 0.0
    x[2] = -1e36
    x = x.to(dtype)
    mean, rstd = x[:, 0].float().contiguous(), torch.full((5,), 1e6, device="cuda")
    if apart:
        x, dy = (torch.nn.functional.pad(t, (at, 9 - at))[:, at:at + cols] for t, at in ((x, 3), (dy, 2)))
    w, _ = weights(cols, F32, 3)
    want = norm_back_ref(dy, x, mean, rstd, w)
    dx, _, _ = kernels.layer_norm_backward(dy, x, mean, rstd, w, wgrad=False)
    assert_within(dx, want[0], want[3] + rounded(want[0].abs() + want[3], dtype), "dx")
