"""What the operators' results are off by, and where they must be the same bits."""
import threading

import pytest

torch = pytest.importorskip("torch")

from test_gpu_operators import (DEV, HALF, TINY, TYPES, U, back_exact, chain, check_back, code, coefs, gen, gradient, iterate,  # noqa: E402
                                norm_exact, ortho_tolerance, run_ortho, stream)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("shapes", [[(256, 1000)], [(1000, 784), (500, 1000), (10, 500)], [(640, 2500)], [(300, 300), (1, 400)],
                                    [(64, 200), (5, 9), (1, 33)]])
def test_orthogonalised_16_bit_matrices_are_the_fp32_results_rounded(g, t, shapes):
    """The same products whatever the result's type: it is rounded once, at the end."""
    ins = [gradient(m, n, 40 + i, "noise").to(TYPES[t]) for i, (m, n) in enumerate(shapes)]
    outs, wide = [torch.empty_like(a) for a in ins], [torch.empty(a.shape, device=DEV) for a in ins]
    run_ortho(g, ins, outs, t)
    run_ortho(g, [a.float() for a in ins], wide, "f32")
    for a, b in zip(outs, wide):
        assert torch.equal(a, b.to(TYPES[t]))


def test_layer_norm_backward_from_several_threads_at_once(g):
    """Two shapes that need different amounts of shared memory, each from two host threads with a stream each: no call fails, and every
    one gives the bits that it gives alone."""
    calls, errors = [], []
    for i, (rows, n) in enumerate([(2000, 256), (8192, 256)] * 2):
        r = gen(i)
        x, dy = torch.randn(rows, n, generator=r, device=DEV), torch.randn(rows, n, generator=r, device=DEV)
        _, em, er = norm_exact(x, None, None, 1e-5)
        keep = (x, dy, em[:, 0].float(), er[:, 0].float(), torch.empty(rows, n, device=DEV), torch.empty(n, device=DEV), torch.empty(n, device=DEV),
                torch.empty(g.layer_norm_backward_workspace(rows, n), dtype=torch.uint8, device=DEV))

        def call(s, keep=keep, rows=rows, n=n):
            x, dy, mean, rstd, dx, dg, ds, work = keep
            g.layer_norm_backward(dy.data_ptr(), n, x.data_ptr(), n, None, mean.data_ptr(), rstd.data_ptr(), dx.data_ptr(), n, dg.data_ptr(),
                                  ds.data_ptr(), rows, n, work.data_ptr(), work.numel(), stream=s)
        call(stream())
        torch.cuda.synchronize()
        calls.append((call, keep[4:7], [a.clone() for a in keep[4:7]], torch.cuda.Stream()))
        for a in keep[4:7]:
            a.zero_()
    torch.cuda.synchronize()

    def work(call, s):
        try:
            for _ in range(20000):
                call(s.cuda_stream)
        except Exception as e:  # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=work, args=(c, s)) for c, _, _, s in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors
    for _, got, want, _ in calls:
        for a, b in zip(got, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("n", [15, 16, 17, 257, 512, 513, 1025, 1537, 2049, 4097, 8191, 8192])
def test_layer_norm_backward_of_full_blocks(g, t, n):
    """As many groups per block as there can be, and rows of one value more than their lanes hold: the most shared memory that the
    columns' sums take."""
    rows = 148 * 2 * max(1, 512 // max(1, n // 16)) + 3
    check_back(g, rows, n, t, n, n, n, 0, seed=n)
    check_back(g, rows, n, t, n, n, n, 1, seed=n, plain=True)


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("rows,n", [(70, 256), (70, 4096), (70, 1000), (33, 257), (41, 4097), (9, 8192), (9, 8193), (7, 20000)])
@pytest.mark.parametrize("size", [1e18, 1e-18])
def test_layer_norm_backward_of_very_large_and_very_small_activations(g, t, rows, n, size):
    """No factor on the way leaves fp32's range, whichever kernel a row's length leads to: the gradient is as exact as for activations of 1."""
    r = gen(n)
    x = (size * torch.randn(rows, n, generator=r, device=DEV)).to(TYPES[t])
    dy = (1e-4 * torch.randn(rows, n, generator=r, device=DEV)).to(TYPES[t])
    gain = 1.0 + 0.3 * torch.randn(n, generator=r, device=DEV)
    _, em, er = norm_exact(x, None, None, 0.0)
    mean, rstd = em[:, 0].float(), er[:, 0].float()
    dx, dgain, dshift = torch.empty(rows, n, device=DEV, dtype=TYPES[t]), torch.empty(n, device=DEV), torch.empty(n, device=DEV)
    bytes_ = g.layer_norm_backward_workspace(rows, n)
    work = torch.empty(bytes_, dtype=torch.uint8, device=DEV)
    g.layer_norm_backward(dy.data_ptr(), n, x.data_ptr(), n, gain.data_ptr(), mean.data_ptr(), rstd.data_ptr(), dx.data_ptr(), n,
                          dgain.data_ptr(), dshift.data_ptr(), rows, n, work.data_ptr(), bytes_, dtype=code(g, t), stream=stream())
    ex, eg, _ = back_exact(dy, x, gain, mean, rstd)
    # a sum of n terms: at most chain(n) additions; every other factor one rounding
    rd = rstd.double()[:, None]
    xh = ((x.double() - mean.double()[:, None]) * rd).abs()
    v = (dy.double() * gain.double()).abs()
    a, b = v.mean(1, keepdim=True), (v * xh).mean(1, keepdim=True)
    tol = 1.01 * rd * U * ((chain(n) + 4) * (a + xh * b) + 2 * xh * b + 6 * (v + a + xh * b))
    tol = tol + HALF[t] * (ex.abs() + tol) + TINY[t]
    assert bool(((dx.double() - ex).abs() <= tol).all()), float(((dx.double() - ex).abs() / tol).max())
    tol = 1.01 * U * ((rows + 23) * (dy.double().abs() * xh).sum(0)) + TINY["f32"]
    assert bool(((dgain.double() - eg).abs() <= tol).all())


@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_orthogonalize_matrices_whose_norm_is_beyond_fp32(g, t):
    """Finite elements of up to 3e38: the norm is taken and used in 64 bits."""
    for list_ in ([(1, 9), (600, 1)], [(2, 2), (16, 40), (100, 30), (1, 7)], [(200, 260), (1, 80), (90, 1)]):
        ins = [((2 * torch.rand(m, n, generator=gen(m + n), device=DEV) - 1) * 3e38).to(TYPES[t]) for m, n in list_]
        ins[0].fill_(3e38)
        ins[0][0, 0] = -2e38
        outs = [torch.empty_like(a) for a in ins]
        assert sum(float(a.double().norm()) > 3.5e38 for a in ins) >= 2  # (a short row's need not be)
        run_ortho(g, ins, outs, t)
        for a, b in zip(ins, outs):
            u = a.double() * 2.0 ** -100  # (the same matrix to the operator: eps is 1e-16 of its norm)
            exact = iterate(u, 5, coefs(5), 1e-7, torch.float64)
            tol = ortho_tolerance(u.float(), 5, coefs(5), 1e-7, exact)
            tol = tol + HALF[t] * (exact.abs() + tol)
            assert bool(((b.double() - exact).abs() <= tol).all()), tuple(a.shape)


@pytest.mark.parametrize("shapes", [[(1, 9), (70, 1)], [(16, 40), (100, 30), (1, 7)], [(200, 260), (1, 80)]])
def test_zero_matrices_give_zeros_without_eps_too(g, shapes):
    ins = [torch.zeros(m, n, device=DEV) for m, n in shapes]
    outs = [torch.full((m, n), 7.0, device=DEV) for m, n in shapes]
    run_ortho(g, ins, outs, "f32", eps=0.0)
    for a in outs:
        assert not a.any() and not torch.isnan(a).any()
    # and a gradient without eps is what it is with a negligible one
    ins = [gradient(m, n, 5) for m, n in shapes]
    run_ortho(g, ins, outs, "f32", eps=0.0)
    for a, b in zip(ins, outs):
        exact = iterate(a.double(), 5, coefs(5), 0.0, torch.float64)
        assert bool(((b.double() - exact).abs() <= ortho_tolerance(a, 5, coefs(5), 0.0, exact)).all())


@pytest.mark.parametrize("size", [1e-6, 1e-8, 1e-10, 1e-13, 1e-30])
@pytest.mark.parametrize("shapes", [[(1, 300), (200, 1)], [(40, 70), (90, 30)], [(300, 200), (260, 520)]])
def test_matrices_far_below_eps(g, shapes, size):
    """Where |U| lies below eps all of the result is small.  Parts of X_0 are exact to 2^-39 (half a step of the smallest fp16 number under
    the scale of 2^14), those of every later X too, and a step multiplies by 3.4445 at most: 2^-39 * 3.4445 * (1 + 3.4445 + ..) of an
    element, beside what is relative to the result.  Single rows and columns have no parts."""
    ins = [gradient(m, n, 17) for m, n in shapes]
    ins = [a * (size / a.double().norm().float()) for a in ins]
    outs = [torch.full((a.shape[0], a.shape[1]), 7.0, device=DEV) for a in ins]
    run_ortho(g, ins, outs, "f32")
    for a, b in zip(ins, outs):
        exact = iterate(a.double(), 5, fp32(coefs(5)), float(torch.tensor(1e-7, dtype=torch.float32)), torch.float64)
        plain = float((iterate(a, 5, fp32(coefs(5)), 1e-7, torch.float32).double() - exact).abs().max())
        tol = 2.5 * plain + 4 * U * 10.25 / 0.7 * float(exact.abs().max())
        if min(a.shape) > 1:
            tol += 2.0 ** -39 * sum(3.4445 ** k for k in range(1, 6))
        assert float(exact.abs().max()) > 0.0
        assert float((b.double() - exact).abs().max()) <= tol, tuple(a.shape)


def test_status_behind_a_call_without_matrices(g):
    items = g.ortho_items([])
    bytes_ = g.orthogonalize_workspace(items)
    work = torch.full((bytes_,), 0xFF, dtype=torch.uint8, device=DEV)
    g.orthogonalize(items, work.data_ptr(), bytes_, stream=stream())
    g.orthogonalize_status(work.data_ptr(), stream=stream())


# ---- the orthogonalisation's error beside that of fp32 products ---------------------------------------------------------
def fp32(coef):
    """Coefficients as the entry point holds them."""
    return [tuple(float(torch.tensor(v, dtype=torch.float32)) for v in c) for c in coef]


def structured(p, q, seed):
    """p x q matrices, p <= q, whose products differ in kind: sums of many terms of one sign or of both, of few terms, of one."""
    r = gen(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=r, device=DEV)
    eye = torch.zeros(p, q, device=DEV)
    eye[torch.arange(p), torch.arange(p)] = 1.0
    blocks = torch.zeros(p, q, device=DEV)
    for i in range(8):
        a, b = p * i // 8, p * (i + 1) // 8
        blocks[a:b, q * i // 8:q * (i + 1) // 8] = randn(b - a, q * (i + 1) // 8 - q * i // 8)
    signs = torch.ones(q, device=DEV)
    signs[1::2] = -1.0
    opposite = randn(p, q)
    opposite[1::2] = -opposite[0::2][:p // 2]
    u, v = torch.linalg.qr(randn(p, p).double())[0], torch.linalg.qr(randn(q, p).double())[0]
    return {
        "noise": randn(p, q),
        "near singular values": ((u * torch.linspace(0.5, 1, p, device=DEV, dtype=torch.float64)) @ v.t()).float(),
        "wide spectrum": ((u * torch.logspace(0, -4, p, device=DEV, dtype=torch.float64)) @ v.t()).float(),
        "orthogonal rows": v.t().float().contiguous(),
        "diagonal": eye * torch.exp(randn(p, 1)),
        "blocks": blocks,
        "blocks of different size": blocks * torch.logspace(0, -3, p, device=DEV)[:, None],
        "one strong direction": randn(p, 1) @ randn(1, q) + 1e-3 * randn(p, q),
        "positive": torch.rand(p, q, generator=r, device=DEV),
        "columns of alternating sign": randn(p, q).abs() * signs,
        "rows that cancel": opposite + 1e-3 * randn(p, q),
        "gradient": gradient(p, q, seed),
        # products that fp32 holds without a rounding
        "exact: identity": eye,
        "exact: permutation": eye[:, torch.randperm(q, generator=r, device=DEV)].contiguous(),
        "exact: ones": torch.ones(p, q, device=DEV),
        "exact: ones of alternating sign": torch.ones(p, 1, device=DEV) * signs,
    }


def check_structured(g, p, q, tall=False, steps=5, coefficients=None):
    """The result's error against 64 bits, root mean square over seeds, relative to the result: at most 2.5 times that of fp32
    products.  (An accumulator that cuts four additions off loses (1 + 2 + 3 + 4) / 4 half units in the last place of a sum of one sign on
    average, where a rounded sum is off by up to one.)  Matrices whose products fp32 holds without a rounding may be off by what
    the parts' roundings make of one step: the terms |a| + |b| + |c| = 10.25 of a result of 0.7 or more, each with four half units."""
    coef = fp32(coefficients or coefs(steps))
    error, plain = {}, {}
    seeds = 4
    for seed in range(seeds):
        for kind, u in structured(p, q, seed).items():
            if tall:
                u = u.t().contiguous()
            out = torch.empty_like(u)
            run_ortho(g, [u], [out], "f32", steps, coefficients)
            exact = iterate(u.double(), steps, coef, 1e-7, torch.float64)
            for sums, got in ((error, out), (plain, iterate(u, steps, coef, 1e-7, torch.float32))):
                sums[kind] = sums.get(kind, 0.0) + float((got.double() - exact).norm() / exact.norm()) ** 2 / seeds
    off = {}
    for kind in error:
        e, f = error[kind] ** 0.5, plain[kind] ** 0.5
        limit = 2.5 * f + (4 * U * 10.25 / 0.7 if kind.startswith("exact") else 0.0)
        if e > limit:
            off[kind] = (e, f)
    assert not off, off


@pytest.mark.parametrize("p,q", [(16, 64), (33, 90), (64, 128), (128, 128), (10, 500), (64, 512), (96, 200), (112, 300)])
def test_errors_of_small_matrices(g, p, q):
    check_structured(g, p, q)


@pytest.mark.parametrize("p,q", [(192, 192), (256, 256), (256, 1000), (500, 1000), (1000, 784), (1024, 1024), (20, 2048)])
def test_errors_of_matrices(g, p, q):
    check_structured(g, min(p, q), max(p, q), tall=p > q)


@pytest.mark.parametrize("p,q", [(512, 2048), (512, 4096), (300, 3000), (1024, 4096), (4096, 640)])
def test_errors_of_flat_matrices(g, p, q):
    check_structured(g, min(p, q), max(p, q), tall=p > q)


SCHEDULE = [(1.2, -0.9, 0.5), (2.6, -2.4, 0.8), (0.7, 0.3, -0.1), (2.2, -1.4, 0.3), (0.9, -0.2, 0.15), (1.6, -0.7, 0.2)]


@pytest.mark.parametrize("shapes", [[(1, 300), (500, 1), (1, 1)], [(20, 50), (1, 90), (64, 500), (30, 30)], [(300, 280), (40, 30), (1, 70)], [(400, 4096)],
                                    [(4096, 400), (5, 6)]])
def test_every_step_takes_its_own_coefficients(g, shapes):
    """Single rows and columns, small matrices, tiles, and flat ones: the error is that of fp32 products with the same list, and no
    other order of the list comes near."""
    coef = fp32(SCHEDULE)
    ins = [torch.randn(m, n, generator=gen(60 + i), device=DEV) for i, (m, n) in enumerate(shapes)]
    outs = [torch.empty_like(a) for a in ins]
    run_ortho(g, ins, outs, "f32", len(coef), SCHEDULE)
    for a, b in zip(ins, outs):
        exact = iterate(a.double(), len(coef), coef, 1e-7, torch.float64)
        plain = float((iterate(a, len(coef), coef, 1e-7, torch.float32).double() - exact).norm() / exact.norm())
        got = float((b.double() - exact).norm() / exact.norm())
        assert got <= 2.5 * plain + 4 * U * 10.25 / 0.7, (tuple(a.shape), got, plain)
        for k in range(len(coef) - 1):
            other = coef[:k] + [coef[k + 1], coef[k]] + coef[k + 2:]
            off = float((iterate(a.double(), len(coef), other, 1e-7, torch.float64) - exact).norm() / exact.norm())
            assert off > 100 * got, (tuple(a.shape), k, off, got)
