"""Long rows where the work is cut: an element at every place around a cut has to
count once.  Each row has one value far above the others, at a place of its own,
so that losing it, or taking it twice, moves the row's statistics and gradients
far past the bounds; and the bounds count the additions that the kernels make."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")
import train_ref  # noqa: E402
from train_ref import assert_within, norm_back_ref, norm_ref, rounded  # noqa: E402

F32, BF16 = torch.float32, torch.bfloat16
EPS = 1e-5
RUN, LONG_RUN = 4096, 16384  # columns of a run; of a block's turn at a strided row going forward
SPIKE = 2.0 ** 14


def additions(n: int) -> int:
    """Roundings on the longest way of an element into a row's sums.  A thread adds 16 elements, as 8 pairs and their two
    halves (9); a warp's shuffles are 5 more, a block's or a cluster's warps at most 16 one after another, then 5: 35.  Rows
    past a cluster join moments instead."""
    return 40 if n <= 49152 - 8 else additions_of_joins(n)


def additions_of_joins(n: int) -> int:
    """A join of two sets' moments rounds 8 times at most.  A thread's 16 elements one after another (18 with the mean's
    division), 5 shuffles, 7 joins of a block's warps or 10 by shuffles, a lane's or a block's runs (n / 4096 / 32 or
    n / 16384 / 8), 10 by shuffles: 18 + 5 + 27 * 8 = 239, and 8 for each of n / 131072."""
    return 240 + n // 16384


@pytest.fixture(autouse=True)
def bounds_of_the_kernels(monkeypatch):
    monkeypatch.setattr(train_ref, "chain", additions)


def places(cols: int, cut: int) -> list[int]:
    """Columns around every cut, for any start within a vector, and the row's ends."""
    around = [c + o for c in range(0, cols + cut, cut) for o in range(-9, 10)]
    ends = [cols - 1 - o for o in range(10)]
    return sorted({c for c in around + ends if 0 <= c < cols})


def spikes(cols: int, cut: int, dtype, seed: int, device="cuda"):
    at = places(cols, cut)
    g = torch.Generator(device=device).manual_seed(seed)
    t = torch.randn((len(at), cols), generator=g, device=device).to(dtype)
    t[torch.arange(len(at)), at] = SPIKE
    return t


def as_view(t, kind, start):
    if kind == "strided":
        out = t.new_zeros(t.shape[0], 2 * t.shape[1])[:, ::2]
    else:
        out = t.new_full((t.shape[0], (t.shape[1] + 15) // 8 * 8), float("nan"))[:, start:start + t.shape[1]]
    out.copy_(t)
    return out


def check(kernels, x, dy, w, b, out, dx):
    """Both directions into given views; the spike is in x going forward, and in dy and x going back."""
    y, mean, rstd = kernels.layer_norm(x, w, b, out=out, dtype=out.dtype)
    want, m, r, e_m, e_r, e_y = norm_ref(x, w, b, EPS)
    assert_within(mean, m, e_m, "mean")
    assert_within(rstd, r, e_r, "rstd")
    assert_within(y, want, e_y + rounded(want.abs() + e_y, y.dtype), "y")
    _, dw, db = kernels.layer_norm_backward(dy, x, mean, rstd, w, dx=dx)
    gx, gw, gb, e_x, e_w, e_b = norm_back_ref(dy, x, mean, rstd, w)
    assert_within(dx, gx, e_x + rounded(gx.abs() + e_x, dx.dtype), "dx")
    assert_within(dw, gw, e_w + rounded(gw.abs() + e_w, dw.dtype), "dweight")
    assert_within(db, gb, e_b + rounded(gb.abs() + e_b, db.dtype), "dbias")


def operands(cols, cut, x_t, y_t):
    x, dy = spikes(cols, cut, x_t, 1), spikes(cols, cut, y_t, 2)
    plain = torch.randn(x.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)).to(x_t)
    g = torch.Generator(device="cuda").manual_seed(4)
    return x, dy, plain, 1 + 0.2 * torch.randn(cols, generator=g, device="cuda"), torch.randn(cols, generator=g, device="cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("start", range(8))
@pytest.mark.parametrize("x_t,y_t", [(F32, F32), (BF16, BF16), (F32, BF16)])
@pytest.mark.parametrize("cols", [49153, 57344, 70000])
def test_elements_around_a_cut(kernels, cols, x_t, y_t, start):
    """All views start alike, `start` elements into a vector; then the outputs start elsewhere."""
    x, dy, plain, w, b = operands(cols, RUN, x_t, y_t)
    for shift in (0, 3):
        # (dy's spike against an x without one: the sums of a and of a xh both hang on it.)
        for source in (x, plain):
            view_x = as_view(source, "whole", start)
            view_dy = as_view(dy, "whole", start)
            out = as_view(torch.zeros_like(dy), "whole", (start + shift) % 8)
            dx = as_view(torch.zeros_like(x), "whole", (start + shift) % 8)
            check(kernels, view_x, view_dy, w, b, out, dx)


@pytest.mark.gpu
@pytest.mark.parametrize("x_t,y_t", [(F32, F32), (BF16, BF16)])
@pytest.mark.parametrize("cols,cut", [(70000, RUN), (70000, LONG_RUN), (150001, LONG_RUN), (20000, LONG_RUN), (9000, RUN)])
def test_elements_around_a_cut_of_strided_rows(kernels, monkeypatch, cols, cut, x_t, y_t):
    monkeypatch.setattr(train_ref, "chain", additions_of_joins)
    x, dy, plain, w, b = operands(cols, cut, x_t, y_t)
    for source in (x, plain):
        check(kernels, *(as_view(t, "strided", 0) for t in (source, dy)), w, b,
              *(as_view(torch.zeros_like(t), "strided", 0) for t in (dy, x)))


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [131072, 300001])
def test_long_rows_within_the_additions_made(kernels, cols):
    g = torch.Generator(device="cuda").manual_seed(cols)
    x, dy = (torch.randn((5, cols), generator=g, device="cuda") for _ in range(2))
    w, b = 1 + 0.2 * torch.randn(cols, generator=g, device="cuda"), torch.randn(cols, generator=g, device="cuda")
    for kind in ("whole", "strided"):
        check(kernels, *(as_view(t, kind, 1) for t in (x, dy)), w, b, *(as_view(torch.zeros_like(t), kind, 2) for t in (x, dy)))


# ---- the bounds themselves, on the CPU ----------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("times", [0, 2])
@pytest.mark.parametrize("cols", [49153, 70000, 150001])
def test_the_bounds_see_a_lost_or_doubled_element(cols, times, dtype):
    """An oracle whose sums take each row's spike `times` times falls outside the bounds in every row."""
    x, dy = spikes(cols, LONG_RUN, dtype, 1, "cpu"), spikes(cols, LONG_RUN, dtype, 2, "cpu")
    at = torch.tensor(places(cols, LONG_RUN))
    rows = torch.arange(len(at))
    xd, gd = x.double(), dy.double()
    _, m, r, e_m, e_r, _ = norm_ref(x, None, None, EPS)
    extra = (times - 1) * xd[rows, at]
    mean = (xd.sum(-1) + extra) / cols
    off = (xd - mean[:, None]).square()
    rstd = 1 / ((off.sum(-1) + (times - 1) * off[rows, at]) / cols + EPS).sqrt()
    assert bool(((mean - m).abs() > 10 * e_m).all()) and bool(((rstd - r).abs() > 10 * e_r).all())
    plain = torch.randn(x.shape, generator=torch.Generator().manual_seed(3)).to(dtype)
    stats = norm_ref(plain, None, None, EPS)[1:3]
    gx, _, _, e_x, _, _ = norm_back_ref(dy, plain, *stats, None)
    xh = (plain.double() - stats[0][:, None]) * stats[1][:, None]
    c1 = (gd.sum(-1) + (times - 1) * gd[rows, at]) / cols
    c2 = ((gd * xh).sum(-1) + (times - 1) * (gd * xh)[rows, at]) / cols
    wrong = (gd - c1[:, None] - xh * c2[:, None]) * stats[1][:, None]
    outside = (wrong - gx).abs() > e_x + rounded(gx.abs() + e_x, dtype)
    assert bool(outside.any(-1).all()) and float(outside.double().mean()) > 0.5
