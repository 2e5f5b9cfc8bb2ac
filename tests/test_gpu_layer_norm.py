"""Layer norm and its gradients against 64-bit formulas, with bounds counted in
roundings (train_ref.py)."""
from __future__ import annotations

import pytest

from conftest import spmd_mod

torch = pytest.importorskip("torch")
from train_ref import U, assert_within, norm_back_ref, norm_ref, rounded  # noqa: E402

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
PAIRS = [(F32, F32), (F16, F16), (BF16, BF16), (F32, F16), (F32, BF16), (F16, F32), (BF16, F32)]
COLS = [1, 2, 3, 7, 8, 31, 64, 100, 128, 257, 512, 1000, 1001, 1024, 2040, 4096, 5003, 8192, 8200, 12288, 16385, 20000,
        32768, 40001, 70000, 131072, 300001]
EPS = 1e-5


def make(shape, dtype, seed, shift=0.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = torch.randn(shape, generator=g, device="cuda")
    if len(shape) > 1 and shift:
        t = t + shift * torch.randn((*shape[:-1], 1), generator=g, device="cuda")
    return t.to(dtype)


def weights(cols, dtype, seed):
    if dtype is None:
        return None, None
    return (1 + 0.2 * make((cols,), F32, seed)).to(dtype), (0.2 * make((cols,), F32, seed + 1)).to(dtype)


def check_forward(k, x, w, b, eps=EPS, ydtype=None, **kw):
    y, mean, rstd = k.layer_norm(x, w, b, eps=eps, dtype=ydtype, **kw)
    want, m, r, e_m, e_r, e_y = norm_ref(x, w, b, eps)
    assert y.dtype == (ydtype or x.dtype) and y.shape == x.shape
    assert_within(mean, m, e_m, "mean")
    assert_within(rstd, r, e_r, "rstd")
    assert_within(y, want, e_y + rounded(want.abs() + e_y, y.dtype), "y")
    return y, mean, rstd


def check_backward(k, dy, x, w, eps=EPS, stats=None, **kw):
    n = x.shape[-1]
    if stats is None:
        xd = x.double()
        stats = xd.mean(-1).float(), (1 / (xd.var(-1, unbiased=False) + eps).sqrt()).float()
    want = norm_back_ref(dy, x, *stats, w)  # before dx may overwrite an input
    kind = x.dtype
    dx, dw, db = k.layer_norm_backward(dy, x, *stats, w, **kw)
    assert dx.dtype == kind and dx.shape == dy.shape
    assert_within(dx, want[0], want[3] + rounded(want[0].abs() + want[3], kind), "dx")
    if dw is not None:
        assert dw.shape == db.shape == (n,)
        assert_within(dw, want[1], want[4] + rounded(want[1].abs() + want[4], dw.dtype), "dweight")
        assert_within(db, want[2], want[5] + rounded(want[2].abs() + want[5], db.dtype), "dbias")
    return dx, dw, db


@pytest.mark.parametrize("cols", COLS)
def test_row_lengths(kernels, cols):
    """Every row length class with f32 and 16-bit rows, odd row counts."""
    rows = 5 if cols > 20000 else 37
    for x_t, y_t, w_t in ((F32, F32, F32), (BF16, BF16, F32), (F16, F16, F16), (F32, BF16, F32), (BF16, F32, None)):
        x, dy = make((rows, cols), x_t, cols), make((rows, cols), y_t, cols + 1)
        w, b = weights(cols, w_t, cols + 2)
        _, mean, rstd = check_forward(kernels, x, w, b, ydtype=y_t)
        check_backward(kernels, dy, x, w, stats=(mean, rstd))


@pytest.mark.parametrize("rows", [1, 2, 3, 148, 149, 1000, 4099])
@pytest.mark.parametrize("cols", [24, 1001, 4096])
def test_row_counts(kernels, rows, cols):
    x, dy = make((rows, cols), BF16, rows), make((rows, cols), BF16, rows + 1)
    w, b = weights(cols, BF16, rows + 2)
    _, mean, rstd = check_forward(kernels, x, w, b)
    check_backward(kernels, dy, x, w, stats=(mean, rstd))


@pytest.mark.parametrize("rows,cols", [(700, 60001), (1500, 20000), (9, 4000001), (40, 1500000), (5000, 8190)])
def test_long_rows_in_batches(kernels, rows, cols):
    """More long rows than one batch holds: statistics and sums go on from batch to batch."""
    x, dy = make((rows, cols), BF16, rows), make((rows, cols), BF16, rows + 1)
    w, b = weights(cols, F32, 2)
    y, mean, rstd = kernels.layer_norm(x, w, b)
    dx, dw, db = kernels.layer_norm_backward(dy, x, mean, rstd, w)
    tw, tb = (torch.zeros(cols, device="cuda", dtype=torch.float64) for _ in range(2))
    aw, ab = torch.zeros_like(tw), torch.zeros_like(tb)
    for i in range(0, rows, 64):
        s = slice(i, i + 64)
        want, m, r, e_m, e_r, e_y = norm_ref(x[s], w, b, EPS)
        assert_within(mean[s], m, e_m, "mean")
        assert_within(rstd[s], r, e_r, "rstd")
        assert_within(y[s], want, e_y + rounded(want.abs() + e_y, BF16), "y")
        ref = norm_back_ref(dy[s], x[s], mean[s], rstd[s], w)
        assert_within(dx[s], ref[0], ref[3] + rounded(ref[0].abs() + ref[3], BF16), "dx")
        tw += ref[1]
        tb += ref[2]
        aw += ref[4] / (min(64, rows - i) + 20)
        ab += ref[5] / (min(64, rows - i) + 16)
    assert_within(dw, tw, (rows + 20) * aw + rounded(tw.abs(), F32), "dweight")
    assert_within(db, tb, (rows + 16) * ab + rounded(tb.abs(), F32), "dbias")


@pytest.mark.parametrize("x_t,y_t", PAIRS)
@pytest.mark.parametrize("rows,cols", [(700, 8193), (501, 12289), (150, 28672), (301, 40968), (77, 49145), (75, 49152), (75, 49153)])
def test_rows_spread_over_blocks(kernels, rows, cols, x_t, y_t):
    """Rows held by two to twelve blocks, more of them than are resident at once."""
    x, dy = make((rows, cols), x_t, 1), make((rows, cols), y_t, 2)
    w, b = weights(cols, F32, 3)
    _, mean, rstd = check_forward(kernels, x, w, b, ydtype=y_t)
    check_backward(kernels, dy, x, w, stats=(mean, rstd))


@pytest.mark.parametrize("x_t,y_t", PAIRS)
@pytest.mark.parametrize("w_t", [None, F32, F16, BF16])
def test_types(kernels, x_t, y_t, w_t):
    for rows, cols in ((33, 320), (9, 1026)):
        x, dy = make((rows, cols), x_t, 1), make((rows, cols), y_t, 2)
        w, b = weights(cols, w_t, 3)
        check_forward(kernels, x, w, b, ydtype=y_t)
        _, dw, _ = check_backward(kernels, dy, x, w)
        assert (dw is None) == (w is None) and (w is None or dw.dtype == w_t)


def layouts(t_wide):
    """Views of one buffer [12, 30, 700]: (name, view)."""
    return [
        ("pitched", t_wide[:, 0, :640]),
        ("shifted by one element", t_wide[:, 3, 1:601]),
        ("rank 3 slice", t_wide[:, 2:9, :512]),
        ("rank 3, odd", t_wide[1:, 5:, 3:404]),
        ("every second column", t_wide[:, :4, ::2]),
        ("columns as rows", t_wide[:, 0, :].t()),
        ("swapped leading dimensions", t_wide[:, :, :96].transpose(0, 1)),
        ("one row", t_wide[0, 0]),
        ("rank 4", t_wide.view(3, 4, 30, 700)),
    ]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("at", range(9))
def test_layouts(kernels, dtype, at):
    name, x = layouts(make((12, 30, 700), dtype, 5))[at]
    _, dy = layouts(make((12, 30, 700), dtype, 6))[at]
    w, b = weights(x.shape[-1], F32, 7)
    check_forward(kernels, x, w, b)
    check_backward(kernels, dy, x, w)
    # Into views of the same layout: what lies between the rows stays as it was.
    buf = torch.full((12, 30, 700), 7.0, device="cuda", dtype=dtype)
    out = layouts(buf)[at][1]
    # (A layout may sum in an order of its own: every one is within the bound, not of one bit pattern.)
    y, mean, rstd = check_forward(kernels, x, w, b, out=out)
    assert y is out
    mask = torch.zeros(12, 30, 700, device="cuda", dtype=torch.bool)
    layouts(mask)[at][1].fill_(True)
    assert bool((buf[~mask] == 7.0).all()), name
    buf.fill_(7.0)
    dx, _, _ = check_backward(kernels, dy, x, w, stats=(mean, rstd), dx=out)
    assert dx is out and bool((buf[~mask] == 7.0).all()), name


def within_nan(t, pitch, at):
    """t's values as a view of a buffer of NaN: rows `pitch` apart, from column `at` on; and the buffer."""
    *lead, cols = t.shape
    buf = torch.full((*lead, pitch), float("nan"), device="cuda", dtype=t.dtype)
    view = buf[..., at:at + cols]
    view.copy_(t)
    return view, buf


@pytest.mark.parametrize("x_t,y_t", [(F32, F32), (BF16, BF16), (F16, F32), (F32, BF16)])
@pytest.mark.parametrize("cols", [1, 3, 8, 15, 33, 100, 257, 1001, 2047, 4090, 4096, 5003, 8185, 8192, 9001, 20001, 49150, 70000])
def test_rows_that_start_apart(kernels, x_t, y_t, cols):
    """Inputs and outputs whose rows start at different places within a vector, all with NaN around them."""
    for seed, (rows, px, ax, py, ay, pd, ad) in enumerate((
            ((3,), 5, 1, 0, 0, 0, 0), ((41,), 0, 0, 7, 3, 2, 1), ((2, 21), 9, 2, 3, 0, 8, 5), ((1,), 9, 7, 9, 1, 9, 3))):
        x, dy = make((*rows, cols), x_t, seed), make((*rows, cols), y_t, seed + 9)
        w, b = weights(cols, F32, seed + 5)
        x, _ = within_nan(x, cols + px, ax)
        dy, _ = within_nan(dy, cols + py, ay)
        out, out_buf = within_nan(torch.zeros_like(dy), cols + py + 4, ay + 1)
        dx, dx_buf = within_nan(torch.zeros_like(x), cols + pd, ad)
        _, mean, rstd = check_forward(kernels, x, w, b, ydtype=y_t, out=out)
        _, dw, db = check_backward(kernels, dy, x, w, stats=(mean, rstd), dx=dx)
        for view, buf in ((out, out_buf), (dx, dx_buf)):
            view.fill_(float("nan"))
            assert bool(buf.isnan().all())
        again = kernels.layer_norm_backward(dy, x, mean, rstd, w, dx=dx)
        assert torch.equal(dw, again[1]) and torch.equal(db, again[2])


@pytest.mark.parametrize("rows,cols", [(20011, 1001), (40009, 60), (3001, 4099), (2500, 9001)])
def test_many_rows_that_start_apart(kernels, rows, cols):
    """More rows than blocks: a thread's rows come one after another."""
    x, _ = within_nan(make((rows, cols), BF16, 1), cols + 5, 3)
    dy, _ = within_nan(make((rows, cols), BF16, 2), cols + 6, 1)
    w, b = weights(cols, F32, 3)
    _, mean, rstd = check_forward(kernels, x, w, b)
    check_backward(kernels, dy, x, w, stats=(mean, rstd))


@pytest.mark.parametrize("cols", [64, 1001, 4096, 20000, 100000])
def test_broadcast_inputs(kernels, cols):
    """Inputs of stride 0: one row for all, one value for a whole row."""
    x, dy = make((1, cols), F32, 1).expand(6, cols), make((6, cols), F32, 2)
    w, b = weights(cols, F32, 3)
    check_forward(kernels, x, w, b)
    check_backward(kernels, dy, x, w)
    check_backward(kernels, make((6, 1), F32, 4).expand(6, cols), make((6, cols), F32, 5), w)
    check_backward(kernels, torch.ones((), device="cuda").expand(6, cols), make((6, cols), F32, 5), w)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("cols", [40, 1001, 4096, 9000, 20000, 100000])
def test_in_place(kernels, dtype, cols):
    x, dy = make((11, cols), dtype, 1), make((11, cols), dtype, 2)
    w, b = weights(cols, F32, 3)
    want, mean, rstd = kernels.layer_norm(x, w, b)
    dx, dw, db = kernels.layer_norm_backward(dy, x, mean, rstd, w)
    for target in ("dy", "x"):
        a, c = dy.clone(), x.clone()
        got = kernels.layer_norm_backward(a, c, mean, rstd, w, dx=a if target == "dy" else c)
        assert all(torch.equal(p, q) for p, q in zip(got, (dx, dw, db))), target
    y = x.clone()
    assert torch.equal(kernels.layer_norm(y, w, b, out=y)[0], want)


def test_partial_arguments(kernels):
    x, dy = make((40, 300), F32, 1), make((40, 300), F32, 2)
    w, b = weights(300, F32, 3)
    full, mean, rstd = kernels.layer_norm(x, w, b)
    y, none1, none2 = kernels.layer_norm(x, w, b, stats=False)
    assert torch.equal(y, full) and none1 is None and none2 is None
    check_forward(kernels, x, w, None)
    check_forward(kernels, x, None, b)
    check_forward(kernels, x, None, None, eps=0.0)
    dx, dw, db = kernels.layer_norm_backward(dy, x, mean, rstd, w)
    only, n1, n2 = kernels.layer_norm_backward(dy, x, mean, rstd, w, wgrad=False)
    assert torch.equal(only, dx) and n1 is None and n2 is None
    # Sums without a weight, and sums in a type of their own.
    _, dw1, db1 = check_backward(kernels, dy, x, None, stats=(mean, rstd), wgrad=True)
    assert torch.equal(dw1, dw) and torch.equal(db1, db)
    kind = torch.empty(300, device="cuda", dtype=BF16)
    _, dw2, db2 = check_backward(kernels, dy, x, w, stats=(mean, rstd), dweight=kind)
    assert dw2 is kind and db2.dtype == BF16 and torch.equal(dw2, dw.bfloat16())


def test_no_rows(kernels):
    x = torch.empty((0, 100), device="cuda")
    w, b = weights(100, F32, 1)
    y, mean, rstd = kernels.layer_norm(x, w, b)
    assert y.shape == (0, 100) and mean.shape == rstd.shape == (0,)
    dx, dw, db = kernels.layer_norm_backward(x, x, mean, rstd, w)
    assert dx.shape == (0, 100) and bool((dw == 0).all()) and bool((db == 0).all())
    y, _, _ = kernels.layer_norm(torch.empty((3, 0, 100), device="cuda"), w, b)
    assert y.shape == (3, 0, 100)
    x, (w, b) = torch.empty((0, 30000), device="cuda"), weights(30000, F32, 1)
    y, mean, rstd = kernels.layer_norm(x, w, b)
    _, dw, db = kernels.layer_norm_backward(x, x, mean, rstd, w)
    assert y.shape == (0, 30000) and bool((dw == 0).all()) and bool((db == 0).all())


@pytest.mark.parametrize("cols", [8, 1001, 4096, 40000])
def test_far_means_and_constant_rows(kernels, cols):
    """Rows whose mean is far above their spread, constant rows, rows of zeros and rows of large values."""
    x = make((8, cols), F32, 1)
    x[0] += 1000.0
    x[1] = 3.25
    x[2] = 0.0
    x[3] *= 1e15
    x[4] *= 1e-15
    w, b = weights(cols, F32, 3)
    _, mean, rstd = check_forward(kernels, x, w, b)
    assert bool((rstd[2] - EPS ** -0.5).abs() <= 4 * U * EPS ** -0.5)
    check_backward(kernels, make((8, cols), F32, 2), x, w, stats=(mean, rstd))


@pytest.mark.parametrize("cols", [16, 1001, 4096, 20000])
def test_a_bad_row_stays_alone(kernels, cols):
    """NaN and infinity spoil their own row, and the sums over rows; other rows keep their bits."""
    x, dy = make((9, cols), F32, 1), make((9, cols), F32, 2)
    w, b = weights(cols, F32, 3)
    y, mean, rstd = kernels.layer_norm(x, w, b)
    dx, dw, db = kernels.layer_norm_backward(dy, x, mean, rstd, w)
    bad = x.clone()
    bad[4, cols // 2] = float("nan")
    bad[6, 0] = float("inf")
    y1, mean1, rstd1 = kernels.layer_norm(bad, w, b)
    dx1, dw1, db1 = kernels.layer_norm_backward(dy, bad, mean1, rstd1, w)
    good = [0, 1, 2, 3, 5, 7, 8]
    for a, c in ((y, y1), (mean, mean1), (rstd, rstd1), (dx, dx1)):
        assert torch.equal(a[good], c[good])
    assert bool(y1[4].isnan().all()) and bool(y1[6].isnan().all()) and bool(dx1[4].isnan().all())
    assert bool(dw1.isnan().all()) and torch.equal(db1, db)


def test_same_bits_every_time(kernels):
    for rows, cols in ((5000, 64), (700, 1001), (300, 4096), (40, 30000)):
        x, dy = make((rows, cols), BF16, 1), make((rows, cols), BF16, 2)
        w, b = weights(cols, F32, 3)
        _, mean, rstd = kernels.layer_norm(x, w, b)
        first = kernels.layer_norm_backward(dy, x, mean, rstd, w)
        for _ in range(3):
            assert all(torch.equal(p, q) for p, q in zip(kernels.layer_norm_backward(dy, x, mean, rstd, w), first))


@pytest.mark.parametrize("cols", [48, 1001])
def test_differences(kernels, cols):
    """dx, dweight and dbias against central differences of the forward kernel
    along random directions: they differ by the roundings of both sides and by
    what the difference itself is off, which 64 bits give."""
    rows, h = 6, 1 / 64
    x, w, b, c = make((rows, cols), F32, 1), *weights(cols, F32, 2), make((rows, cols), F32, 4)
    _, mean, rstd = kernels.layer_norm(x, w, b)
    grads = kernels.layer_norm_backward(c, x, mean, rstd, w)
    ref = norm_back_ref(c, x, mean, rstd, w)
    true = norm_back_ref(c, x, *norm_ref(x, w, b, EPS)[1:3], w)
    for k, t in enumerate((x, w, b)):
        d = make(tuple(t.shape), F32, 10 + k)
        sides, exact, off = [], [], 0.0
        for sign in (1, -1):
            a = [x, w, b]
            a[k] = t + sign * h * d
            y = kernels.layer_norm(*a)[0]
            want, *_, e_y = norm_ref(*a, EPS)
            sides.append((y.double() * c).sum())
            exact.append((want * c).sum())
            off += float(((e_y + rounded(want.abs() + e_y, F32)) * c.abs()).sum()) / (2 * h)
        moved = (a[k].double() - t) / (-h)  # the step that was taken, rounding included
        got = (sides[0] - sides[1]) / (2 * h)
        along = (true[k] * d).sum()
        off += float((((exact[0] - exact[1]) / (2 * h)) - along).abs())
        off += float(((ref[k] - true[k]).abs() * d.abs()).sum() + ((ref[3 + k] + rounded(ref[k].abs() + ref[3 + k], F32)) * d.abs()).sum())
        assert abs(float((grads[k].double() * d).sum() - got)) <= off, k
        assert moved.shape == d.shape


def test_offsets_past_32_bits(kernels):
    """Rows 2^31 + 8 elements apart."""
    pitch, cols = (1 << 31) + 8, 1000
    buf = torch.empty(2 * pitch + cols, device="cuda", dtype=F16)
    x = buf.as_strided((3, cols), (pitch, 1))
    x.copy_(make((3, cols), F16, 1))
    w, b = weights(cols, F32, 2)
    y = kernels.layer_norm(x, w, b, out=x)[0]
    want = kernels.layer_norm(make((3, cols), F16, 1), w, b)[0]
    assert torch.equal(y, want)
    dy = make((3, cols), F16, 3)
    x.copy_(make((3, cols), F16, 1))
    got = check_backward(kernels, dy, x, w)
    assert got[0].shape == (3, cols)


def test_other_stream_and_capture(kernels):
    """A side stream, and a captured pair of calls replayed on new inputs."""
    x, dy = make((257, 768), BF16, 1), make((257, 768), BF16, 2)
    w, b = weights(768, F32, 3)
    want = kernels.layer_norm(x, w, b)
    grads = kernels.layer_norm_backward(dy, x, *want[1:], w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = kernels.layer_norm(x, w, b, stream=side)
    back = kernels.layer_norm_backward(dy, x, *got[1:], w, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip((*want, *grads), (*got, *back)))
    sx, sdy = torch.zeros_like(x), torch.zeros_like(dy)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a = kernels.layer_norm(sx, w, b)
        g = kernels.layer_norm_backward(sdy, sx, *a[1:], w)
    for seed in (1, 7):
        sx.copy_(make((257, 768), BF16, seed))
        sdy.copy_(make((257, 768), BF16, seed + 1))
        graph.replay()
        e = kernels.layer_norm(sx, w, b)
        eg = kernels.layer_norm_backward(sdy, sx, *e[1:], w)
        assert all(torch.equal(p, q) for p, q in zip((*a, *g), (*e, *eg)))


@pytest.mark.parametrize("rows,cols", [(40, 12289), (500, 30000), (300, 200000), (1500, 60000)])
def test_long_rows_captured_and_on_two_streams(kernels, rows, cols):
    """Rows over several blocks and in batches, whose kernels overlap: captured, replayed back to
    back, and on two streams at once, each call gives the bits that it gives alone."""
    args = []
    for seed in (1, 5):
        x, dy = make((rows, cols), BF16, seed), make((rows, cols), BF16, seed + 1)
        w, b = weights(cols, F32, seed + 2)
        y, mean, rstd = kernels.layer_norm(x, w, b)
        args.append((x, dy, w, b, (y, mean, rstd, *kernels.layer_norm_backward(dy, x, mean, rstd, w))))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(3):
        for k, (x, dy, w, b, _) in enumerate(args):
            with torch.cuda.stream(streams[k]):
                y, mean, rstd = kernels.layer_norm(x, w, b)
                got[k].append((y, mean, rstd, *kernels.layer_norm_backward(dy, x, mean, rstd, w)))
    torch.cuda.synchronize()
    for k in range(2):
        for g in got[k]:
            assert all(torch.equal(p, q) for p, q in zip(g, args[k][4]))
    got.clear()
    x, dy, w, b, want = args[0]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, mean, rstd = kernels.layer_norm(x, w, b)
        grads = kernels.layer_norm_backward(dy, x, mean, rstd, w)
    for _ in range(3):
        for t in (y, mean, rstd, *grads):
            t.fill_(float("nan"))
        graph.replay()
        graph.replay()
        assert all(torch.equal(p, q) for p, q in zip((y, mean, rstd, *grads), want))


def test_refusals(kernels):
    err = spmd_mod("_lib").SpmdError
    x, w = make((4, 32), F32, 1), make((32,), F32, 2)
    _, mean, rstd = kernels.layer_norm(x)
    for call, kind in (
        (lambda: kernels.layer_norm(x.double()), TypeError),
        (lambda: kernels.layer_norm(x.half(), dtype=BF16), TypeError),
        (lambda: kernels.layer_norm(x.cpu()), ValueError),
        (lambda: kernels.layer_norm(x, w.cpu()), ValueError),
        (lambda: kernels.layer_norm(x, w[:16]), ValueError),
        (lambda: kernels.layer_norm(x, make((64,), F32, 2)[::2]), ValueError),
        (lambda: kernels.layer_norm(x, w, w.half()), TypeError),
        (lambda: kernels.layer_norm(x, out=make((4, 16), F32, 1)), ValueError),
        (lambda: kernels.layer_norm(x, dtype=F16, out=torch.empty_like(x)), TypeError),
        (lambda: kernels.layer_norm(x, out=x[:1].expand(4, 32)), err),
        (lambda: kernels.layer_norm(x, eps=-1.0), err),
        (lambda: kernels.layer_norm(x, eps=float("nan")), err),
        (lambda: kernels.layer_norm(torch.empty((4, 0), device="cuda")), err),
        (lambda: kernels.layer_norm(torch.ones((), device="cuda")), ValueError),
        (lambda: kernels.layer_norm(make((2, 3, 4, 8), F32, 1).transpose(0, 2)), ValueError),
        (lambda: kernels.layer_norm_backward(x[:2], x, mean, rstd), ValueError),
        (lambda: kernels.layer_norm_backward(x, x, mean[:2], rstd), ValueError),
        (lambda: kernels.layer_norm_backward(x, x, mean.half(), rstd), TypeError),
        (lambda: kernels.layer_norm_backward(x, x, mean, rstd, dx=x.half()), TypeError),
        (lambda: kernels.layer_norm_backward(x, x, mean, rstd, w, ws=torch.empty(16, device="cuda")), err),
        (lambda: kernels.layer_norm_backward(x, x, mean, rstd, w, wgrad=False, dbias=w), ValueError),
    ):
        with pytest.raises(kind):
            call()
