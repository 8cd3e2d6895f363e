"""Layer norm (forward and backward) and orthogonalised weight updates: cases, inputs, plain forms and exact results.

A case is a dict of plain values.  Layer sizes and windows come from the repository's benchmark configurations, or are
generic; data is synthetic, made from the seed.  `own` False: elementary torch operations in 32 bits; True: the package's
entry points (glades-ml_b200/capi.py, include/glades_b200.h) in torch's current stream.
"""
import importlib
import math

import torch

own = False

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
# the quintic whose five steps bring singular values from (0, 1] close to 1
QUINTIC = (3.4445, -4.7750, 2.0315)
NORM_EPS = 1e-5
ORTHO_EPS = 1e-7


# ---- cases ------------------------------------------------------------------------------------------------
def listed():
    return [
        # one request against a wide network: a single row of 4096 activations, where only latency counts
        dict(name="norm_single_row", kind="norm", type="f32", rows=1, n=4096),
        # the hidden activations of the wide network's training window
        dict(name="norm_wide_window", kind="norm", type="f32", rows=8192, n=4096),
        # half-width activations of an odd layer: rows that begin on no boundary, a row count that fills no grid
        dict(name="norm_odd_bf16", kind="norm", type="bf16", rows=10007, n=1025),
        # a minibatch of the window regressor, backward
        dict(name="norm_backward_minibatch", kind="norm_backward", type="f32", rows=1024, n=256),
        # the wide network's window, backward, activations and deltas kept in 16 bits
        dict(name="norm_backward_wide_bf16", kind="norm_backward", type="bf16", rows=8192, n=4096),
        # sizes that people choose by hand
        dict(name="norm_backward_hand_f16", kind="norm_backward", type="f16", rows=20300, n=1000),
        # the weight gradients of the window regressor: a thin, a square and a one-row matrix
        dict(name="ortho_regressor", kind="ortho", type="f32", shapes="256x32,256x256,1x256", steps=5),
        # the gradients of the digits classifier in 16 bits, no size a multiple of a tile
        dict(name="ortho_digits_bf16", kind="ortho", type="bf16", shapes="1000x784,500x1000,10x500", steps=5),
        # a layer that is eight times as wide as it is deep
        dict(name="ortho_flat_f16", kind="ortho", type="f16", shapes="1024x8192", steps=5),
        # the update step of the tiny tabular classifier: latency
        dict(name="step_tiny", kind="step", type="f32", shapes="16x4,3x16", steps=5, nesterov=True, decay=0.0),
        # the update step of the inference network's layers
        dict(name="step_middle", kind="step", type="f32", shapes="2048x784,2048x2048,10x2048", steps=5, nesterov=True, decay=0.01),
        # the update step of the wide teacher-student network: 25 million weights
        dict(name="step_wide", kind="step", type="f32", shapes="4096x1024,4096x4096,1024x4096", steps=5, nesterov=False, decay=0.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A layer's width: a multiple of 128, a multiple of 8, or any number."""
    n, how = _log(rng, lo, hi), rng.randrange(3)
    if how < 2:
        m = 128 if how == 0 and n >= 128 else 8
        n = max(m, int(round(n / m)) * m)
    return max(lo, min(hi, n))


_LARGEST_NORM = 8192 * 4096


def draw(rng):
    kind = rng.choice(["norm", "norm_backward", "ortho", "step"])
    type = rng.choice(["f32", "bf16", "f16"])
    if kind in ("norm", "norm_backward"):
        n = _width(rng, 1, 40000)
        return dict(kind=kind, type=type, rows=_log(rng, 1, max(1, min(32768, _LARGEST_NORM // n))), n=n)
    limit = 0.5 * max(_ortho_flops(c) for c in listed() if c["kind"] == kind)
    while True:
        top = _log(rng, 32, 4096)
        shapes = ",".join("%dx%d" % (_width(rng, 1, top), _width(rng, 1, top)) for _ in range(rng.randint(1, 3)))
        case = dict(kind=kind, type=type, shapes=shapes, steps=rng.choice([5, 5, 5, 3, 6]))
        if kind == "step":
            case.update(nesterov=rng.random() < 0.5, decay=rng.choice([0.0, 0.01]))
        if _ortho_flops(case) <= limit:
            return case


def _shapes(case):
    return [tuple(int(v) for v in s.split("x")) for s in case["shapes"].split(",")]


# ---- inputs -----------------------------------------------------------------------------------------------
class State:
    """What the program keeps between calls: its tensors, and the operators' workspace."""


def _package():
    return importlib.import_module("glades-ml_b200")


def _activations(gen, rows, n):
    """A hidden layer behind a ReLU: rows of different size, about half of the values zero, now and then a whole row."""
    x = torch.randn(rows, n, generator=gen, device=DEV)
    x = torch.relu(x + 0.1) * torch.exp(0.5 * torch.randn(rows, 1, generator=gen, device=DEV))
    return x * (torch.rand(rows, 1, generator=gen, device=DEV) > 0.002)


def _gradient(gen, m, n):
    """A weight gradient: a few strong directions over a floor of noise, nodes of different activity."""
    r = min(8, m, n)
    a = torch.randn(m, r, generator=gen, device=DEV) * torch.exp(torch.randn(1, r, generator=gen, device=DEV))
    g = a @ torch.randn(r, n, generator=gen, device=DEV) + 0.5 * torch.randn(m, n, generator=gen, device=DEV)
    return g * torch.exp(0.5 * torch.randn(m, 1, generator=gen, device=DEV)) * 1e-3


def _inputs(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    t = TYPES[case["type"]]
    s = State()
    s.case, s.type = case, t
    if case["kind"] in ("norm", "norm_backward"):
        rows, n = case["rows"], case["n"]
        s.x = _activations(gen, rows, n).to(t)
        s.gain = 1.0 + 0.2 * torch.randn(n, generator=gen, device=DEV)
        s.shift = 0.1 * torch.randn(n, generator=gen, device=DEV)
        if case["kind"] == "norm_backward":
            s.dy = (1e-2 * torch.randn(rows, n, generator=gen, device=DEV)).to(t)
        return s
    shapes = _shapes(case)
    s.grad = [_gradient(gen, m, n).to(t) for m, n in shapes]
    if case["kind"] == "step":
        s.momentum = [5.0 * _gradient(gen, m, n) for m, n in shapes]
        s.weight = [(torch.rand(m, n, generator=gen, device=DEV) * 2 - 1) * math.sqrt(1.5 / n) for m, n in shapes]
        # the length of a step goes with the layer's shape
        s.lr = [0.02 * math.sqrt(max(1.0, m / n)) for m, n in shapes]
    return s


MU = 0.95


def prepare(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "norm_backward":
        # the forward pass has left these
        x = s.x.double()
        mean = x.mean(1, keepdim=True)
        s.rstd = (1.0 / torch.sqrt(((x - mean) ** 2).mean(1) + NORM_EPS)).float()
        s.mean = mean[:, 0].float()
    if not own:
        return s
    g = _package()
    if case["kind"] == "norm":
        s.y = torch.empty_like(s.x)
        s.mean, s.rstd = (torch.empty(case["rows"], device=DEV) for _ in range(2))
    elif case["kind"] == "norm_backward":
        s.dx = torch.empty_like(s.x)
        s.dgain, s.dshift = (torch.empty(case["n"], device=DEV) for _ in range(2))
        s.work_bytes = g.layer_norm_backward_workspace(case["rows"], case["n"])
    elif case["kind"] == "ortho":
        s.out = [torch.empty_like(t) for t in s.grad]
        s.items = g.ortho_items([dict(rows=a.shape[0], cols=a.shape[1], d_in=a.data_ptr(), ld_in=a.shape[1], d_out=b.data_ptr(),
                                      ld_out=a.shape[1]) for a, b in zip(s.grad, s.out)])
        s.work_bytes = g.orthogonalize_workspace(s.items)
    else:
        s.new_momentum = [torch.empty_like(t) for t in s.momentum]
        s.new_weight = [torch.empty_like(t) for t in s.weight]
        s.items = g.muon_items([dict(rows=a.shape[0], cols=a.shape[1], lr=lr, d_grad=a.data_ptr(), ld_grad=a.shape[1],
                                     d_momentum=m.data_ptr(), d_momentum_out=m2.data_ptr(), ld_momentum=a.shape[1],
                                     d_weight=w.data_ptr(), d_weight_out=w2.data_ptr(), ld_weight=a.shape[1])
                                for a, m, m2, w, w2, lr in zip(s.grad, s.momentum, s.new_momentum, s.weight, s.new_weight, s.lr)])
        s.work_bytes = g.muon_workspace(s.items)
    if case["kind"] != "norm":
        s.work = torch.empty(max(1, s.work_bytes), dtype=torch.uint8, device=DEV)
    s.code = {"f32": g.F32, "bf16": g.BF16, "f16": g.F16}[case["type"]]
    return s


# ---- one pass ---------------------------------------------------------------------------------------------
def _plain_norm(s):
    x = s.x.float()
    n = x.shape[1]
    mean = x.sum(1, keepdim=True) / n
    c = x - mean
    rstd = 1.0 / torch.sqrt((c * c).sum(1, keepdim=True) / n + NORM_EPS)
    return (c * rstd * s.gain + s.shift).to(s.type), mean[:, 0], rstd[:, 0]


def _plain_norm_backward(s):
    x, dy = s.x.float(), s.dy.float()
    n = x.shape[1]
    xh = (x - s.mean[:, None]) * s.rstd[:, None]
    v = dy * s.gain
    dx = s.rstd[:, None] * (v - v.sum(1, keepdim=True) / n - xh * ((v * xh).sum(1, keepdim=True) / n))
    return dx.to(s.type), (dy * xh).sum(0), dy.sum(0)


def _plain_ortho(u, steps):
    a, b, c = QUINTIC
    x = u.float()
    x = x / (torch.sqrt((x.double() * x).sum()).float() + ORTHO_EPS)
    tall = x.shape[0] > x.shape[1]
    if tall:
        x = x.t()
    for _ in range(steps):
        gram = x @ x.t()
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.t() if tall else x


def _plain_step(s):
    case, out = s.case, []
    for g, m, w, lr in zip(s.grad, s.momentum, s.weight, s.lr):
        g = g.float()
        m = MU * m + g
        o = _plain_ortho(g + MU * m if case["nesterov"] else m, case["steps"])
        out += [m, (1.0 - lr * case["decay"]) * w - lr * o]
    return out


def run(s):
    case = s.case
    kind = case["kind"]
    if not own:
        if kind == "norm":
            return _plain_norm(s)
        if kind == "norm_backward":
            return _plain_norm_backward(s)
        if kind == "ortho":
            return [_plain_ortho(g, case["steps"]).to(s.type) for g in s.grad]
        return _plain_step(s)
    g = _package()
    stream = torch.cuda.current_stream().cuda_stream
    if kind == "norm":
        g.layer_norm(s.x.data_ptr(), case["n"], s.gain.data_ptr(), s.shift.data_ptr(), s.y.data_ptr(), case["n"], s.mean.data_ptr(),
                     s.rstd.data_ptr(), case["rows"], case["n"], eps=NORM_EPS, dtype=s.code, stream=stream)
        return s.y, s.mean, s.rstd
    if kind == "norm_backward":
        n = case["n"]
        g.layer_norm_backward(s.dy.data_ptr(), n, s.x.data_ptr(), n, s.gain.data_ptr(), s.mean.data_ptr(), s.rstd.data_ptr(),
                              s.dx.data_ptr(), n, s.dgain.data_ptr(), s.dshift.data_ptr(), case["rows"], n, s.work.data_ptr(),
                              s.work_bytes, dtype=s.code, stream=stream)
        return s.dx, s.dgain, s.dshift
    if kind == "ortho":
        g.orthogonalize(s.items, s.work.data_ptr(), s.work_bytes, steps=case["steps"], eps=ORTHO_EPS, dtype=s.code, stream=stream)
        return s.out
    g.muon_step(s.items, s.work.data_ptr(), s.work_bytes, momentum=MU, nesterov=case["nesterov"], weight_decay=case["decay"],
                steps=case["steps"], eps=ORTHO_EPS, dtype=s.code, stream=stream)
    return [t for pair in zip(s.new_momentum, s.new_weight) for t in pair]


# ---- what a pass cannot do without -------------------------------------------------------------------------
def _ortho_flops(case):
    """Of the two ways to the same polynomial the one with fewer operations: products of the short side's symmetric matrices
    (which commute, so that half of each is enough), and two that involve the long side."""
    total = 0
    for m, n in _shapes(case):
        p, q = min(m, n), max(m, n)
        total += 3 * p * p * q + max(1, 4 * case["steps"] - 3) * p ** 3
    return total


def work(case):
    size = 4 if case["type"] == "f32" else 2
    if case["kind"] == "norm":
        return {"bytes": 2 * case["rows"] * case["n"] * size + 8 * case["rows"] + 8 * case["n"], "flops": 8 * case["rows"] * case["n"]}
    if case["kind"] == "norm_backward":
        return {"bytes": 3 * case["rows"] * case["n"] * size + 8 * case["rows"] + 12 * case["n"], "flops": 16 * case["rows"] * case["n"]}
    weights = sum(m * n for m, n in _shapes(case))
    per = 2 * size if case["kind"] == "ortho" else size + 16
    return {"bytes": weights * per, "flops": _ortho_flops(case)}


# ---- the definition in 64 bits ------------------------------------------------------------------------------
def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"] in ("norm", "norm_backward"):
        x = s.x.to(torch.float64)
        var, mean = torch.var_mean(x, dim=1, unbiased=False)
        rstd = (var + NORM_EPS) ** -0.5
        h = (x - mean.unsqueeze(1)).mul_(rstd.unsqueeze(1))
        if case["kind"] == "norm":
            return torch.addcmul(s.shift.double(), h, s.gain.double()), mean, rstd
        dy = s.dy.to(torch.float64)
        k = dy * s.gain.double()
        # the projection of k off the constant vector and off h, row by row
        dx = (k - k.mean(1, keepdim=True) - h * torch.einsum("ij,ij->i", k, h).unsqueeze(1) / x.shape[1]) * rstd.unsqueeze(1)
        return dx, torch.einsum("ij,ij->j", dy, h), dy.sum(0)

    def polar(u):
        z = u / (torch.linalg.vector_norm(u) + ORTHO_EPS)
        if z.shape[0] > z.shape[1]:
            return polar_steps(z.mT).mT
        return polar_steps(z)

    def polar_steps(z):
        one = torch.eye(z.shape[0], dtype=torch.float64, device=DEV)
        for _ in range(case["steps"]):
            q = z @ z.mT
            z = torch.mm(QUINTIC[0] * one + q @ (QUINTIC[1] * one + QUINTIC[2] * q), z)
        return z

    if case["kind"] == "ortho":
        return [polar(g.double()) for g in s.grad]
    out = []
    for g, m, w, lr in zip(s.grad, s.momentum, s.weight, s.lr):
        g, v = g.double(), g.double() + MU * m.double()
        o = polar(v * MU + g if case["nesterov"] else v)
        out += [v, w.double() * (1.0 - lr * case["decay"]) - o * lr]
    return out
