"""Operators on device buffers against plain implementations in 64 bits."""
import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
U = 2.0 ** -24  # half a step of fp32
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
TINY = {"f32": 2.0 ** -149, "bf16": 2.0 ** -133, "f16": 2.0 ** -24}  # smallest subnormals


def code(g, t):
    return {"f32": g.F32, "bf16": g.BF16, "f16": g.F16}[t]


def stream():
    return torch.cuda.current_stream().cuda_stream


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def matrix(rows, n, ld, t, offset=0, fill=float("nan")):
    """A [rows][n] view of pitch ld that begins `offset` elements into its buffer; what lies around it holds `fill`."""
    buf = torch.full((offset + rows * ld + 64,), fill, dtype=TYPES[t], device=DEV)
    return buf, buf[offset:offset + rows * ld].view(rows, ld)[:, :n]


def untouched(buf, view, fill):
    """True where everything of buf but the view still holds fill."""
    keep = buf.clone()
    rows, n = view.shape
    off = (view.data_ptr() - buf.data_ptr()) // buf.element_size()
    keep[off:off + rows * view.stride(0)].view(rows, view.stride(0))[:, :n] = fill
    return bool((torch.isnan(keep) if math.isnan(fill) else keep == fill).all())


def chain(n):
    """Additions that a value goes through in a row sum: a lane's own, then the lanes' tree."""
    return (32 if n <= 512 * 32 else -(-n // 512)) + 10


def norm_inputs(rows, n, t, ld, offset, seed, kind):
    r = gen(seed)
    x = torch.randn(rows, n, generator=r, device=DEV) * torch.exp(0.5 * torch.randn(rows, 1, generator=r, device=DEV))
    if kind == "offset":
        x = x + 100.0
    elif kind == "relu":
        x = torch.relu(x)
        x[::3] = 0.0
    buf, v = matrix(rows, n, ld, t, offset)
    v.copy_(x)
    gain = 1.0 + 0.3 * torch.randn(n, generator=r, device=DEV)
    shift = 0.2 * torch.randn(n, generator=r, device=DEV)
    return buf, v, gain, shift, r


def norm_exact(x, gain, shift, eps):
    x = x.double()
    mean = x.mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + eps)
    y = (x - mean) * rstd * (1.0 if gain is None else gain.double()) + (0.0 if shift is None else shift.double())
    return y, mean, rstd


def norm_tolerance(x, gain, shift, eps, t):
    """|y - exact|: the mean's rounding (d additions of |x|, one division), its effect on every difference; the variance's (d + 4
    roundings, and the mean's error squared), half of it on rstd with its root and reciprocal; then four roundings of y."""
    x = x.double()
    d = chain(x.shape[1])
    mean = x.mean(1, keepdim=True)
    dm = U * ((d + 2) * x.abs().mean(1, keepdim=True))
    var = ((x - mean) ** 2).mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt(var + eps)
    # the differences that are squared carry one rounding each of the larger of x and mean, and the mean's error
    dd = U * (x - mean).abs() + dm
    dvar = (d + 4) * U * var + 2 * ((x - mean).abs() * U * (x - mean).abs()).mean(1, keepdim=True) + dm ** 2
    drstd = rstd * (0.5 * dvar / (var + eps) + 3 * U)
    ga = 1.0 if gain is None else gain.double().abs()
    y = norm_exact(x, gain, shift, eps)[0]
    tol = ga * (dd * rstd + (x - mean).abs() * drstd + 2 * U * (x - mean).abs() * rstd) + U * y.abs()
    return tol * 1.01 + HALF[t] * (y.abs() + tol) + TINY[t], dm, drstd


def run_norm(g, x, gain, shift, y, t, eps=1e-5):
    rows, n = x.shape
    mean, rstd = torch.full((rows,), 7.0, device=DEV), torch.full((rows,), 7.0, device=DEV)
    g.layer_norm(x.data_ptr(), x.stride(0), None if gain is None else gain.data_ptr(), None if shift is None else shift.data_ptr(),
                 y.data_ptr(), y.stride(0), mean.data_ptr(), rstd.data_ptr(), rows, n, eps=eps, dtype=code(g, t), stream=stream())
    return mean, rstd


def check_norm(g, rows, n, t, ldx, ldy, offset, kind, seed=1, eps=1e-5, plain=False):
    _, x, gain, shift, _ = norm_inputs(rows, n, t, ldx, offset, seed, kind)
    if plain:
        gain = shift = None
    ybuf, y = matrix(rows, n, ldy, t, offset, fill=3.0)
    mean, rstd = run_norm(g, x, gain, shift, y, t, eps)
    ey, em, er = norm_exact(x, gain, shift, eps)
    tol, dm, drstd = norm_tolerance(x, gain, shift, eps, t)
    assert bool(((y.double() - ey).abs() <= tol).all()), float(((y.double() - ey).abs() / tol).max())
    assert bool(((mean.double() - em[:, 0]).abs() <= dm[:, 0] + TINY["f32"]).all())
    assert bool(((rstd.double() - er[:, 0]).abs() <= 1.01 * drstd[:, 0]).all())
    assert untouched(ybuf, y, 3.0)


WIDTHS = [1, 2, 3, 7, 8, 16, 17, 31, 32, 33, 64, 100, 255, 256, 257, 511, 512, 513, 520, 1000, 1024, 1025, 1032, 2048, 4096, 4104, 5001, 8192,
          8200, 8193, 16384, 16392, 20001, 40000]


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n", WIDTHS)
def test_layer_norm_widths(g, n, t):
    for rows in (1, 5, 37):
        check_norm(g, rows, n, t, n, n, 0, "plain", seed=n + rows)


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("kind", ["plain", "offset", "relu"])
def test_layer_norm_values_pitches_and_offsets(g, t, kind):
    for n, ldx, ldy, offset in ((256, 256, 264, 0), (256, 257, 256, 0), (256, 256, 256, 1), (1000, 1008, 1000, 8), (1000, 1002, 1004, 2),
                                (77, 80, 99, 3), (4096, 4096, 4098, 0), (20000, 20008, 20001, 5)):
        check_norm(g, 19, n, t, ldx, ldy, offset, kind, seed=n)


@pytest.mark.parametrize("n", [3, 16, 96, 1024])
def test_layer_norm_many_rows(g, n):
    check_norm(g, 30011, n, "f32", n, n, 0, "plain")
    check_norm(g, 30011, n, "bf16", n, n, 0, "relu", plain=True)


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,n,pad", [(700, 4096, 0), (593, 4096, 8), (5001, 1025, 0), (6007, 500, 0), (20011, 257, 0), (601, 9001, 0),
                                        (1203, 2050, 0), (4099, 1000, 0), (30001, 264, 0), (9000, 255, 0)])
def test_layer_norm_walks(g, t, rows, n, pad):
    """More rows than lanes hold at a time: rows of whole 16-byte pieces, rows that begin anywhere, a last turn that is cut."""
    check_norm(g, rows, n, t, n + pad, n + 2 * pad, 0, "relu", seed=rows)
    check_norm(g, rows, n, t, n + pad, n + pad, 0, "offset", seed=n, plain=True)


def test_layer_norm_in_place_and_without_statistics(g):
    for n, t, rows in ((300, "f32", 50), (4096, "bf16", 50), (20000, "f16", 50), (4096, "f32", 700), (1025, "bf16", 5000)):
        _, x, gain, shift, _ = norm_inputs(rows, n, t, n, 0, 3, "plain")
        y = torch.empty_like(x)
        run_norm(g, x, gain, shift, y, t)
        g.layer_norm(x.data_ptr(), n, gain.data_ptr(), shift.data_ptr(), x.data_ptr(), n, None, None, rows, n, dtype=code(g, t),
                     stream=stream())
        assert torch.equal(x, y)


def test_layer_norm_rows_that_are_constant_or_not_finite(g):
    n = 500
    x = torch.randn(8, n, generator=gen(1), device=DEV)
    x[0] = 0.0
    x[1] = 3.0          # (exactly representable: the mean is exact, every difference zero)
    x[2, 17] = float("nan")
    x[3, 5] = float("inf")
    x[4] = 1e18         # squares of differences stay in range
    gain, shift = torch.full((n,), 2.0, device=DEV), torch.linspace(-1, 1, n, device=DEV)
    y = torch.empty_like(x)
    mean, rstd = run_norm(g, x, gain, shift, y, "f32")
    assert torch.equal(y[0], shift) and torch.equal(y[1], shift)
    assert abs(float(rstd[0]) - 1e-5 ** -0.5) <= 4 * U * 1e-5 ** -0.5
    assert bool(torch.isnan(y[2]).all()) and bool(torch.isnan(y[3]).all())
    ey, _, _ = norm_exact(x[5:], gain, shift, 1e-5)
    tol = norm_tolerance(x[5:], gain, shift, 1e-5, "f32")[0]
    assert bool(((y[5:].double() - ey).abs() <= tol).all())


def back_exact(dy, x, gain, mean, rstd):
    """From the saved statistics, as the operator is defined."""
    dy, x = dy.double(), x.double()
    xh = (x - mean.double()[:, None]) * rstd.double()[:, None]
    v = dy if gain is None else dy * gain.double()
    dx = rstd.double()[:, None] * (v - v.mean(1, keepdim=True) - xh * (v * xh).mean(1, keepdim=True))
    return dx, (dy * xh).sum(0), dy.sum(0)


def check_back(g, rows, n, t, lddy, ldx, lddx, offset, kind="plain", seed=1, plain=False, want=(True, True, True)):
    _, x, gain, _, r = norm_inputs(rows, n, t, ldx, offset, seed, kind)
    if plain:
        gain = None
    _, dy = matrix(rows, n, lddy, t, offset)
    dy.copy_(1e-2 * torch.randn(rows, n, generator=r, device=DEV))
    _, em, er = norm_exact(x, None, None, 1e-5)
    mean, rstd = em[:, 0].float(), er[:, 0].float()
    dxbuf, dx = matrix(rows, n, lddx, t, offset, fill=3.0)
    dgain, dshift = torch.full((n + 1,), 5.0, device=DEV), torch.full((n + 1,), 5.0, device=DEV)
    bytes_ = g.layer_norm_backward_workspace(rows, n)
    work = torch.full((bytes_ + 256,), 0xFF, dtype=torch.uint8, device=DEV)

    def call(work_at):
        g.layer_norm_backward(dy.data_ptr(), lddy, x.data_ptr(), ldx, None if gain is None else gain.data_ptr(), mean.data_ptr(),
                              rstd.data_ptr(), dx.data_ptr() if want[0] else None, lddx, dgain.data_ptr() if want[1] else None,
                              dshift.data_ptr() if want[2] else None, rows, n, work.data_ptr() + work_at, bytes_, dtype=code(g, t),
                              stream=stream())
    call(0)
    first = (dx.clone(), dgain.clone(), dshift.clone())
    call(3)  # a workspace on no boundary; the same bits
    assert torch.equal(first[0], dx) and torch.equal(first[1], dgain) and torch.equal(first[2], dshift)
    assert bool((work[bytes_ + 3:] == 255).all()) and float(dgain[n]) == 5.0 and float(dshift[n]) == 5.0
    ex, eg, es = back_exact(dy, x, gain, mean, rstd)
    d = chain(n)
    xd, dyd = x.double(), dy.double()
    rd = rstd.double()[:, None]
    xh = ((xd - mean.double()[:, None]) * rd).abs()
    dxh = 2 * U * xh
    v = (dyd if gain is None else dyd * gain.double()).abs()
    if want[0]:
        # row sums: d additions over |v| and |v xh|, products' roundings; dx itself: five roundings of its terms
        a, b = v.mean(1, keepdim=True), (v * xh).mean(1, keepdim=True)
        tol = rd * ((d + 4) * U * (a + xh * b) + dxh * b + 6 * U * (v + a + xh * b))
        tol = 1.01 * tol + HALF[t] * (ex.abs() + tol) + TINY[t]
        assert bool(((dx.double() - ex).abs() <= tol).all()), float(((dx.double() - ex).abs() / tol).max())
        assert untouched(dxbuf, dx, 3.0)
    # column sums: a lane adds its rows one by one, then groups, CTAs and slices
    depth = rows / 32 + 400 if rows > 4096 or n > 8192 else rows + 20
    if want[1]:
        tol = 1.01 * U * ((depth + 3) * (dyd.abs() * xh).sum(0)) + TINY["f32"]
        assert bool(((dgain[:n].double() - eg).abs() <= tol).all()), float(((dgain[:n].double() - eg).abs() / tol).max())
    else:
        assert bool((dgain == 5.0).all())
    if want[2]:
        tol = 1.01 * U * (depth * dyd.abs().sum(0)) + TINY["f32"]
        assert bool(((dshift[:n].double() - es).abs() <= tol).all())
    else:
        assert bool((dshift == 5.0).all())


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n", WIDTHS)
def test_layer_norm_backward_widths(g, n, t):
    for rows in (1, 6, 41):
        check_back(g, rows, n, t, n, n, n, 0, seed=n + rows)


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
def test_layer_norm_backward_pitches_and_outputs(g, t):
    for n, lddy, ldx, lddx, offset in ((256, 256, 264, 256, 0), (256, 257, 256, 300, 0), (1000, 1000, 1000, 1000, 1), (77, 80, 99, 81, 3),
                                       (4096, 4098, 4096, 4096, 2), (20000, 20000, 20008, 20001, 5)):
        check_back(g, 23, n, t, lddy, ldx, lddx, offset, kind="relu", seed=n)
        for want in ((True, False, False), (False, True, True), (False, False, True), (True, True, False)):
            check_back(g, 9, n, t, lddy, ldx, lddx, offset, seed=n, want=want, plain=True)


@pytest.mark.parametrize("n", [2, 24, 257, 1024])
def test_layer_norm_backward_many_rows(g, n):
    check_back(g, 30011, n, "f32", n, n, n, 0)
    check_back(g, 9001, n, "bf16", n, n, n, 0, kind="offset")


@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("n,ld,offset", [(1, 2, 0), (1, 2, 1), (2, 2, 1), (3, 4, 0), (17, 18, 1), (50, 50, 0), (100, 100, 0), (101, 102, 3),
                                         (255, 258, 1), (511, 512, 1), (1025, 1025, 0), (2050, 2050, 1), (8191, 8191, 0)])
def test_layer_norm_backward_of_rows_of_words(g, t, n, ld, offset):
    """16-bit rows that begin on an even or an odd element, several or one of them per warp, more of them than groups."""
    for rows in (3, 149, 9001 if n < 600 else 701):
        check_back(g, rows, n, t, ld, ld, ld, offset, seed=rows + n)


def test_layer_norm_backward_in_place(g):
    for n, t in ((300, "f32"), (4096, "bf16"), (20000, "f16")):
        rows = 33
        _, x, gain, _, r = norm_inputs(rows, n, t, n, 0, 3, "plain")
        dy = (torch.randn(rows, n, generator=r, device=DEV)).to(TYPES[t])
        _, em, er = norm_exact(x, None, None, 1e-5)
        mean, rstd = em[:, 0].float(), er[:, 0].float()
        bytes_ = g.layer_norm_backward_workspace(rows, n)
        work = torch.empty(bytes_, dtype=torch.uint8, device=DEV)

        def call(dy, x, dx):
            dg, ds = torch.empty(n, device=DEV), torch.empty(n, device=DEV)
            g.layer_norm_backward(dy.data_ptr(), n, x.data_ptr(), n, gain.data_ptr(), mean.data_ptr(), rstd.data_ptr(), dx.data_ptr(), n,
                                  dg.data_ptr(), ds.data_ptr(), rows, n, work.data_ptr(), bytes_, dtype=code(g, t), stream=stream())
            return dx, dg, ds
        want = call(dy, x, torch.empty_like(x))
        d2 = dy.clone()
        x2 = x.clone()
        for got in (call(d2, x, d2), call(dy, x2, x2)):
            for a, b in zip(want, got):
                assert torch.equal(a, b)


def test_layer_norm_backward_of_no_rows(g):
    dg, ds = torch.ones(9, device=DEV), torch.ones(9, device=DEV)
    g.layer_norm_backward(None, 9, None, 9, None, None, None, None, 9, dg.data_ptr(), ds.data_ptr(), 0, 9, None, 0, stream=stream())
    assert not dg.any() and not ds.any()


def test_layer_norm_gradient_against_differences(g):
    """d(sum(dy * y)) / dx by central differences of the forward pass in 64 bits, at the values that the kernels were given."""
    rows, n, eps = 3, 11, 1e-5
    _, x, gain, shift, r = norm_inputs(rows, n, "f32", n, 0, 5, "plain")
    dy = torch.randn(rows, n, generator=r, device=DEV)
    y = torch.empty_like(x)
    mean, rstd = run_norm(g, x, gain, shift, y, "f32")
    dx, dg, ds = torch.empty(rows, n, device=DEV), torch.empty(n, device=DEV), torch.empty(n, device=DEV)
    bytes_ = g.layer_norm_backward_workspace(rows, n)
    work = torch.empty(bytes_, dtype=torch.uint8, device=DEV)
    g.layer_norm_backward(dy.data_ptr(), n, x.data_ptr(), x.stride(0), gain.data_ptr(), mean.data_ptr(), rstd.data_ptr(), dx.data_ptr(), n,
                          dg.data_ptr(), ds.data_ptr(), rows, n, work.data_ptr(), bytes_, stream=stream())

    def loss(x_, gain_, shift_):
        return float((norm_exact(x_, gain_, shift_, eps)[0] * dy.double()).sum())
    h = 2.0 ** -17  # truncation about h^2 times third derivatives (below 100 here), rounding 2^-52 / h: both below 1e-7
    xs, gs, ss = x.double().contiguous(), gain.double(), shift.double()
    for i in range(rows):
        for j in range(n):
            up, dn = xs.clone(), xs.clone()
            up[i, j] += h
            dn[i, j] -= h
            assert abs((loss(up, gs, ss) - loss(dn, gs, ss)) / (2 * h) - float(dx[i, j])) <= 1e-5 * (1 + float(dx[i].abs().max()))
    for j in range(n):
        e = torch.zeros(n, dtype=torch.float64, device=DEV)
        e[j] = h
        assert abs((loss(xs, gs + e, ss) - loss(xs, gs - e, ss)) / (2 * h) - float(dg[j])) <= 1e-5 * (1 + float(dg.abs().max()))
        assert abs((loss(xs, gs, ss + e) - loss(xs, gs, ss - e)) / (2 * h) - float(ds[j])) <= 1e-5 * (1 + float(ds.abs().max()))


# ---- orthogonalisation --------------------------------------------------------------------------------------
QUINTIC = (3.4445, -4.7750, 2.0315)


def iterate(u, steps, coef, eps, dtype):
    x = u.to(dtype)
    x = x / (u.double().norm().to(dtype) + eps)
    tall = x.shape[0] > x.shape[1]
    if tall:
        x = x.t()
    for k in range(steps):
        a, b, c = coef[k]
        gram = x @ x.t()
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.t() if tall else x


def gradient(m, n, seed, kind="mixed"):
    r = gen(seed)
    if kind == "noise":
        return torch.randn(m, n, generator=r, device=DEV)
    k = min(6, m, n)
    g_ = torch.randn(m, k, generator=r, device=DEV) @ torch.randn(k, n, generator=r, device=DEV)
    g_ = g_ + 0.3 * torch.randn(m, n, generator=r, device=DEV)
    return 1e-3 * g_ * torch.exp(torch.randn(m, 1, generator=r, device=DEV))


def ortho_tolerance(u, steps, coef, eps, exact):
    """Two bounds, in the largest element.  The error of a product, relative to the norms of what is multiplied: 2^-22 for the
    parts, 24 truncations and the drains' roundings of an accumulator, the epilogue's four; at most half of it in a mean.
    A step passes an error on by no more than its slope at zero (that is where the steps are steepest) or 1, and adds three
    products' worth.  And, as a bound that follows the data: 16 times what fp32 products without parts are off by."""
    p, q = min(u.shape), max(u.shape)
    per = (4 + 24 + 4 + math.ceil(q / 128)) * U
    err = 0.0
    for k in range(steps):
        err = err * max(1.0, abs(coef[k][0])) + 3 * per
    plain = float((iterate(u, steps, coef, eps, torch.float32).double() - exact).abs().max())
    return min(err, 16 * plain + 8 * U * float(exact.abs().max()))


def coefs(steps, coef=QUINTIC):
    return [coef] * steps


def run_ortho(g, ins, outs, t, steps=5, coefficients=None, eps=1e-7, dirty=0xFF):
    items = g.ortho_items([dict(rows=a.shape[0], cols=a.shape[1], d_in=a.data_ptr(), ld_in=a.stride(0), d_out=b.data_ptr(),
                                ld_out=b.stride(0)) for a, b in zip(ins, outs)])
    bytes_ = g.orthogonalize_workspace(items)
    work = torch.full((bytes_ + 64,), dirty, dtype=torch.uint8, device=DEV)
    g.orthogonalize(items, work.data_ptr(), bytes_, coefficients=coefficients, steps=steps, eps=eps, dtype=code(g, t), stream=stream())
    g.orthogonalize_status(work.data_ptr(), stream=stream())
    assert bool((work[bytes_:] == dirty).all())
    return work


def check_ortho(g, shapes, t="f32", steps=5, coefficients=None, kind="mixed", seed=1, pad=0, offset=0):
    ins, outs, bufs = [], [], []
    for i, (m, n) in enumerate(shapes):
        _, a = matrix(m, n, n + pad, t, offset)
        a.copy_(gradient(m, n, seed + i, kind))
        buf, b = matrix(m, n, n + 2 * pad, t, offset, fill=3.0)
        ins.append(a), outs.append(b), bufs.append(buf)
    run_ortho(g, ins, outs, t, steps, coefficients)
    coef = coefficients or coefs(steps)
    for a, b, buf in zip(ins, outs, bufs):
        exact = iterate(a.double(), steps, coef, 1e-7, torch.float64)
        tol = ortho_tolerance(a, steps, coef, 1e-7, exact)
        tol = tol + HALF[t] * (exact.abs() + tol)
        err = (b.double() - exact).abs()
        assert bool((err <= tol).all()), (tuple(a.shape), float(err.max()), float((err / tol).max()))
        assert untouched(buf, b, 3.0)


@pytest.mark.parametrize("shape", [(1, 1), (1, 2), (2, 1), (3, 5), (16, 4), (1, 256), (256, 1), (31, 33), (64, 64), (65, 63), (100, 128),
                                   (127, 129), (128, 128), (129, 128), (200, 300), (256, 256), (256, 32), (257, 511), (500, 1000),
                                   (1000, 784), (1024, 640), (640, 2000), (1100, 1300),
                                   # around the sizes that one CTA takes: 128 by about 320 at most, longer where narrower
                                   (16, 16), (17, 64), (48, 65), (10, 2048), (16, 3400), (16, 3500), (30, 1000), (64, 600), (64, 900), (112, 320),
                                   (128, 320), (128, 321), (320, 128), (64, 512), (64, 513), (513, 20), (120, 340), (2000, 33), (7, 5000), (5000, 12), (60000, 2), (1, 70000)])
def test_orthogonalize_shapes(g, shape):
    check_ortho(g, [shape])


def test_orthogonalize_small_matrices_alone_and_beside_large_ones(g):
    """The same matrices on one CTA each and riding along with a large one."""
    shapes = [(33, 90), (100, 128), (12, 700), (1, 9)]
    check_ortho(g, shapes)
    check_ortho(g, shapes + [(300, 400)])
    check_ortho(g, [(3 + i, 40 + 13 * i) for i in range(21)])  # more than one launch takes


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
def test_orthogonalize_types_pitches_and_lists(g, t):
    check_ortho(g, [(300, 200), (64, 777), (5, 5)], t, pad=3, offset=5)
    check_ortho(g, [(20, 10), (10, 30), (1, 7)], t, pad=1, offset=3)
    check_ortho(g, [(130, 40 + i) for i in range(19)], t)  # more than one launch takes


@pytest.mark.parametrize("steps,coef", [(1, None), (2, None), (8, None), (16, (1.5, -0.5, 0.0)), (12, (1.875, -1.25, 0.375)), (3, (1.0, 0.0, 0.0))])
def test_orthogonalize_steps_and_coefficients(g, steps, coef):
    check_ortho(g, [(200, 260), (24, 18)], steps=steps, coefficients=None if coef is None else coefs(steps, coef), kind="noise")


def test_orthogonalize_converging_coefficients_give_orthogonal_rows(g):
    """The rows of what converging coefficients give are orthonormal to the products' error."""
    a = torch.randn(96, 400, generator=gen(3), device=DEV)
    b = torch.empty_like(a)
    run_ortho(g, [a], [b], "f32", steps=16, coefficients=coefs(16, (1.875, -1.25, 0.375)))
    gram = b.double() @ b.double().t()
    # 16 steps bring singular values of 1/96 and more to 1 within rounding; three products per step, of which only the last counts
    assert float((gram - torch.eye(96, device=DEV)).abs().max()) <= 2 * 3 * 36 * U


def test_orthogonalize_matrices_that_are_zero_tiny_huge_or_not_finite(g):
    shapes = [(40, 70), (40, 70), (40, 70), (40, 70), (40, 70), (300, 70)]
    ins = [gradient(m, n, 7) for m, n in shapes]
    ins[0].zero_()
    ins[1].mul_(1e-30)       # below eps: scaled by 1 / eps
    ins[2].mul_(1e30)        # squares beyond fp32
    ins[3][3, 4] = float("nan")
    ins[4][3, 4] = float("inf")
    ins[5][50:].zero_()      # nodes without a gradient
    outs = [torch.empty_like(a) for a in ins]
    run_ortho(g, ins, outs, "f32")
    assert not outs[0].any()
    for i in (1, 2, 5):
        exact = iterate(ins[i].double(), 5, coefs(5), 1e-7, torch.float64)
        assert float((outs[i].double() - exact).abs().max()) <= ortho_tolerance(gradient(*shapes[i], 7) if i < 3 else ins[i], 5, coefs(5), 1e-7, exact) + 1e-30
    assert bool(torch.isnan(outs[3]).all()) and bool(torch.isnan(outs[4]).all())
    assert not outs[5][50:].any()


def test_orthogonalize_in_place_and_repeatable(g):
    ins = [gradient(150, 420, 1), gradient(60, 20, 2), gradient(700, 300, 3)]
    outs = [torch.empty_like(a) for a in ins]
    run_ortho(g, ins, outs, "f32")
    again = [torch.empty_like(a) for a in ins]
    run_ortho(g, ins, again, "f32", dirty=0x7B)
    for a, b in zip(outs, again):
        assert torch.equal(a, b)
    run_ortho(g, ins, ins, "f32")
    for a, b in zip(outs, ins):
        assert torch.equal(a, b)


def vector_exact(u, steps=5, off=0.0):
    """O of a single row or column with the coefficients as fp32 holds them; off: its norm's relative error."""
    u = u.double()
    norm = u.norm() * (1.0 + off)
    x = u / (norm + 1e-7)
    factor, gram = 1.0, (x * x).sum()
    for a, b, c in coefs(steps):
        a, b, c = (float(torch.tensor(v, dtype=torch.float32)) for v in (a, b, c))
        f = a + gram * (b + gram * c)
        factor, gram = factor * f, gram * f * f
    return x * factor


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("beside", [None, (40, 30), (300, 260)])
def test_orthogonalize_single_rows_and_columns(g, t, beside):
    """The only roundings are the norm's (half a step of fp32, and what the steps make of it) and the result's two."""
    ins, outs, bufs = [], [], []
    for i, (m, n, pad) in enumerate([(1, 1, 0), (1, 256, 0), (256, 1, 0), (256, 1, 6), (1, 545, 3), (40001, 1, 2), (1, 131072, 0)]):
        _, a = matrix(m, n, n + pad, t, i % 2)
        a.copy_(torch.randn(m, n, generator=gen(i), device=DEV))
        buf, b = matrix(m, n, n + 2 * pad, t, i % 3, fill=3.0)
        ins.append(a), outs.append(b), bufs.append(buf)
    ins[4][0, 7] = float("nan")
    if beside:
        ins.append(gradient(*beside, 9).to(TYPES[t])), outs.append(torch.empty_like(ins[-1]))
    run_ortho(g, ins, outs, t)
    for a, b, buf in zip(ins, outs, bufs):
        assert untouched(buf, b, 3.0)
        if a is ins[4]:
            assert bool(torch.isnan(b).all())
            continue
        exact = vector_exact(a)
        tol = sum((vector_exact(a, off=o) - exact).abs() for o in (1.01 * U, -1.01 * U)) + 1e-12 * exact.abs()
        tol = tol + (U + HALF[t]) * exact.abs() * 1.01 + TINY[t]
        assert bool(((b.double() - exact).abs() <= tol).all()), (tuple(a.shape), float(((b.double() - exact).abs() / tol).max()))


def test_single_rows_beside_a_matrix_in_order_and_in_a_graph(g):
    """What comes before and behind the call on the stream sees it as one: the row's input is made in front of it, its output
    and the matrix's are used behind it, eager and replayed."""
    big, row = gradient(400, 300, 1), torch.randn(1, 300, generator=gen(2), device=DEV)
    src, out = [torch.empty_like(big), torch.empty_like(row)], [torch.empty_like(big), torch.empty_like(row)]
    items = g.ortho_items([dict(rows=a.shape[0], cols=a.shape[1], d_in=a.data_ptr(), ld_in=a.shape[1], d_out=b.data_ptr(), ld_out=a.shape[1])
                           for a, b in zip(src, out)])
    bytes_ = g.orthogonalize_workspace(items)
    work = torch.empty(bytes_, dtype=torch.uint8, device=DEV)
    got = [torch.empty_like(big), torch.empty_like(row)]

    def call():
        for a, b in zip(src, (big, row)):
            a.copy_(b)
        g.orthogonalize(items, work.data_ptr(), bytes_, stream=stream())
        for a, b in zip(got, out):
            a.copy_(b)
        for a in src + out:
            a.fill_(float("nan"))

    call()
    want = [a.clone() for a in got]
    assert bool(((want[1].double() - vector_exact(row)).abs() <= 1e-6).all()) and bool(torch.isfinite(want[0]).all())
    for _ in range(20):
        call()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        call()
    for _ in range(20):
        for a in got:
            a.zero_()
        graph.replay()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_orthogonalize_lists_of_several_launches_of_all_kinds(g):
    check_ortho(g, [(1, 50), (200, 150), (70, 1)] + [(20, 30 + i) for i in range(14)] + [(1, 90), (12, 12), (1, 1)])
    check_ortho(g, [(1, 60 + i) for i in range(17)] + [(3, 9)])
    check_ortho(g, [(1, 60 + i) for i in range(17)] + [(300, 140), (9, 1)], "bf16")


def test_orthogonalize_long_and_moving_single_columns(g):
    """Those that the kernels of matrices take: beyond 131072 elements, and a column whose result has another pitch in its place."""
    check_ortho(g, [(1, 131073), (140000, 1)])
    buf = torch.zeros(3 * 500, device=DEV)
    a = buf.view(500, 3)[:, :1]
    a.copy_(torch.randn(500, 1, generator=gen(4), device=DEV))
    u = a.clone()
    out = buf[:1000].view(500, 2)[:, :1]
    run_ortho(g, [a], [out], "f32")
    exact = iterate(u.double(), 5, coefs(5), 1e-7, torch.float64)
    assert bool(((out.double() - exact).abs() <= ortho_tolerance(u, 5, coefs(5), 1e-7, exact)).all())


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("nesterov", [False, True])
def test_muon_step(g, t, nesterov):
    shapes = [(300, 200), (40, 90), (1, 33), (128, 512)]
    mu, decay = 0.9, 0.05
    grads = [gradient(m, n, 10 + i).to(TYPES[t]) for i, (m, n) in enumerate(shapes)]
    moms = [4 * gradient(m, n, 20 + i) for i, (m, n) in enumerate(shapes)]
    ws = [0.1 * torch.randn(m, n, generator=gen(30 + i), device=DEV) for i, (m, n) in enumerate(shapes)]
    lrs = [0.02 * (i + 1) for i in range(len(shapes))]

    def step(mom_out, w_out):
        items = g.muon_items([dict(rows=a.shape[0], cols=a.shape[1], lr=lr, d_grad=a.data_ptr(), ld_grad=a.shape[1], d_momentum=m.data_ptr(),
                                   d_momentum_out=m2.data_ptr(), ld_momentum=a.shape[1], d_weight=w.data_ptr(), d_weight_out=w2.data_ptr(),
                                   ld_weight=a.shape[1]) for a, m, m2, w, w2, lr in zip(grads, moms, mom_out, ws, w_out, lrs)])
        bytes_ = g.muon_workspace(items)
        work = torch.empty(bytes_, dtype=torch.uint8, device=DEV)
        g.muon_step(items, work.data_ptr(), bytes_, momentum=mu, nesterov=nesterov, weight_decay=decay, dtype=code(g, t), stream=stream())
        g.orthogonalize_status(work.data_ptr(), stream=stream())
    m2, w2 = [torch.empty_like(m) for m in moms], [torch.empty_like(w) for w in ws]
    step(m2, w2)
    for a, m, w, mo, wo, lr in zip(grads, moms, ws, m2, w2, lrs):
        em = mu * m.double() + a.double()
        # (mu itself is handed over in fp32: half a step of it)
        assert bool(((mo.double() - em).abs() <= 2 * U * (m.double().abs() + a.double().abs()) + TINY["f32"]).all())
        u = a.double() + mu * em if nesterov else em
        o = iterate(u, 5, coefs(5), 1e-7, torch.float64)
        tol = lr * (ortho_tolerance(u.float(), 5, coefs(5), 1e-7, o) + 2 * U * o.abs()) + 4 * U * (w.double().abs() + lr * o.abs())
        err = (wo.double() - ((1 - lr * decay) * w.double() - lr * o)).abs()
        assert bool((err <= tol).all()), float((err / tol).max())
    step(moms, ws)  # in place: the same bits
    for a, b in zip(m2 + w2, moms + ws):
        assert torch.equal(a, b)


# ---- streams, graphs, one behind the other ------------------------------------------------------------------
def test_operators_on_another_stream_and_in_a_graph(g):
    rows, n = 200, 320
    _, x, gain, shift, r = norm_inputs(rows, n, "f32", n, 0, 1, "plain")
    dy = torch.randn(rows, n, generator=r, device=DEV)
    w, mom = 0.1 * torch.randn(n, rows, generator=r, device=DEV), torch.zeros(n, rows, device=DEV)
    y, dx = torch.empty(rows, n, device=DEV), torch.empty(rows, n, device=DEV)
    mean, rstd = torch.empty(rows, device=DEV), torch.empty(rows, device=DEV)
    dg, ds = torch.empty(n, device=DEV), torch.empty(n, device=DEV)
    grad, w2, m2 = torch.empty(n, rows, device=DEV), torch.empty_like(w), torch.empty_like(mom)
    items = g.muon_items([dict(rows=n, cols=rows, lr=0.1, d_grad=grad.data_ptr(), ld_grad=rows, d_momentum=mom.data_ptr(),
                               d_momentum_out=m2.data_ptr(), ld_momentum=rows, d_weight=w.data_ptr(), d_weight_out=w2.data_ptr(),
                               ld_weight=rows)])
    nb, mb = g.layer_norm_backward_workspace(rows, n), g.muon_workspace(items)
    work = torch.empty(nb, dtype=torch.uint8, device=DEV), torch.empty(mb, dtype=torch.uint8, device=DEV)

    def whole():
        s = stream()
        g.layer_norm(x.data_ptr(), n, gain.data_ptr(), shift.data_ptr(), y.data_ptr(), n, mean.data_ptr(), rstd.data_ptr(), rows, n, stream=s)
        g.layer_norm_backward(dy.data_ptr(), n, x.data_ptr(), n, gain.data_ptr(), mean.data_ptr(), rstd.data_ptr(), dx.data_ptr(), n,
                              dg.data_ptr(), ds.data_ptr(), rows, n, work[0].data_ptr(), nb, stream=s)
        torch.mul(dx.t(), 1.0, out=grad)
        g.muon_step(items, work[1].data_ptr(), mb, stream=s)

    def results():
        torch.cuda.synchronize()
        return [t.clone() for t in (y, mean, rstd, dx, dg, ds, m2, w2)]
    whole()
    want = results()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        whole()
    for a, b in zip(want, results()):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        whole()
    x.mul_(-0.5)
    whole()
    want = results()
    for t in (y, mean, rstd, dx, dg, ds, m2, w2):
        t.zero_()
    for _ in range(3):
        graph.replay()
    for a, b in zip(want, results()):
        assert torch.equal(a, b)
    del graph


def test_two_orthogonalisations_at_once(g):
    """Two streams, a workspace each: the calls may run side by side or one behind the other."""
    ins = [gradient(600, 500, i) for i in range(2)]
    outs = [torch.empty_like(a) for a in ins]
    want = [torch.empty_like(a) for a in ins]
    items = [g.ortho_items([dict(rows=600, cols=500, d_in=a.data_ptr(), ld_in=500, d_out=b.data_ptr(), ld_out=500)]) for a, b in zip(ins, outs)]
    bytes_ = g.orthogonalize_workspace(items[0])
    work = [torch.empty(bytes_, dtype=torch.uint8, device=DEV) for _ in ins]
    for a, b in zip(ins, want):
        run_ortho(g, [a], [b], "f32")
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ins]
    for _ in range(5):
        for it, w, s in zip(items, work, streams):
            g.orthogonalize(it, w.data_ptr(), bytes_, stream=s.cuda_stream)
    for w, s in zip(work, streams):
        g.orthogonalize_status(w.data_ptr(), stream=s.cuda_stream)
    for a, b in zip(want, outs):
        assert torch.equal(a, b)
