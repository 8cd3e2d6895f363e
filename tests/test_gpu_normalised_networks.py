"""Networks with normalised layers and orthogonalised updates: training windows and inference against a plain 64-bit implementation
of the same step, on every engine that a layer's products can take; checkpoints; refusals."""
import numpy as np
import pytest

QUINTIC = (3.4445, -4.7750, 2.0315)


class Plain:
    """The network in 64 bits: tanh or ReLU hidden layers (the reference's ReLU: 0 up to 0.046), softmax head, one scalar bias per
    hidden layer."""

    def __init__(self, sizes, act, w, b, lr, norms=(), muons=None, eps=1e-5):
        self.sizes, self.act, self.lr, self.eps = sizes, act, lr, eps
        self.W, at = [], 0
        for i, o in zip(sizes, sizes[1:]):
            self.W.append(w[at:at + i * o].reshape(o, i).astype(np.float64))
            at += i * o
        self.b = b.astype(np.float64)
        self.gain = {l: np.ones(sizes[l]) for l in norms}
        self.shift = {l: np.zeros(sizes[l]) for l in norms}
        self.muons = muons or {}
        self.M = {l: np.zeros_like(self.W[l]) for l in self.muons}

    def forward(self, x):
        x = x.astype(np.float64)
        self.A, self.N, self.xh, self.r, self.margin = [x], [x], {}, {}, np.full(len(x), np.inf)
        h = x
        for l, w in enumerate(self.W):
            z = h @ w.T + (self.b[l - 1] if l >= 1 else 0.0)
            if l == len(self.W) - 1:
                e = np.exp(z - z.max(1, keepdims=True))
                return e / e.sum(1, keepdims=True)
            if self.act == "tanh":
                a = np.tanh(z)
            else:
                self.margin = np.minimum(self.margin, np.abs(z - 0.046).min(1))
                a = np.where(z > 0.046, z, 0.0)
            self.A.append(a)
            h = a
            if l + 1 in self.gain:
                m = a.mean(1, keepdims=True)
                r = 1.0 / np.sqrt(((a - m) ** 2).mean(1, keepdims=True) + self.eps)
                self.xh[l + 1], self.r[l + 1] = (a - m) * r, r
                h = self.xh[l + 1] * self.gain[l + 1] + self.shift[l + 1]
            self.N.append(h)

    def window(self, x, y):
        p = self.forward(x)
        rows = len(x)
        D = p - y
        W = [w.copy() for w in self.W]
        for l in range(len(W) - 1, -1, -1):
            G = D.T @ self.N[l] / rows
            if l in self.muons:
                mu, nesterov, decay, steps = self.muons[l]
                self.M[l] = mu * self.M[l] + G
                u = G + mu * self.M[l] if nesterov else self.M[l]
                o, i = G.shape
                lr = self.lr * np.sqrt(max(1.0, o / i))
                self.W[l] = (1 - lr * decay) * W[l] - lr * orthogonal(u, steps)
            else:
                self.W[l] = W[l] - self.lr * G
            if l == 0:
                break
            self.b[l - 1] -= self.lr * D.sum() / rows
            E = D @ W[l]
            if l in self.gain:
                xh, r = self.xh[l], self.r[l]
                dg, ds = (E * xh).sum(0), E.sum(0)
                v = E * self.gain[l]
                E = r * (v - v.mean(1, keepdims=True) - xh * (v * xh).mean(1, keepdims=True))
                self.gain[l] = self.gain[l] - self.lr * dg / rows
                self.shift[l] = self.shift[l] - self.lr * ds / rows
            a = self.A[l]
            D = E * (1 - a * a if self.act == "tanh" else (a > 0))

    def flat(self):
        return np.concatenate([w.ravel() for w in self.W])


def orthogonal(u, steps):
    x = u / (np.linalg.norm(u) + 1e-7)
    tall = x.shape[0] > x.shape[1]
    if tall:
        x = x.T
    a, b, c = QUINTIC
    for _ in range(steps):
        g = x @ x.T
        x = a * x + (b * g + c * g @ g) @ x
    return x.T if tall else x


def make(g, sizes, act, rows, seed, lr, gemm, norms, muons):
    rng = np.random.default_rng(seed)
    w = np.concatenate([rng.uniform(-1, 1, o * i) * np.sqrt(2.0 / i) for i, o in zip(sizes, sizes[1:])]).astype(np.float32)
    b = rng.uniform(-0.1, 0.1, len(sizes) - 2).astype(np.float32)
    d = g.make_desc(sizes, [act] * (len(sizes) - 2) + ["softmax"], "classification", batch=rows, lr=lr, mode=g.MODE_BATCHED, gemm=gemm)
    net = g.Net(d)
    net.set_weights(w, b)
    for l in norms:
        net.set_layer_norm(l)
    for l, (mu, nesterov, decay, steps) in muons.items():
        net.set_muon(l, mu, nesterov, decay, steps)
    return net, Plain(sizes, act, w, b, lr, norms, muons), rng


def data(rng, plain, rows, n_in, n_out):
    """Rows clear of the ReLU's jump, where two correct evaluations may differ by a whole activation."""
    keep = []
    while sum(len(k) for k in keep) < rows:
        x = rng.standard_normal((rows, n_in)).astype(np.float32)
        plain.forward(x)
        keep.append(x[plain.margin > 1e-4] if plain.act == "relu" else x)
    x = np.concatenate(keep)[:rows]
    y = np.zeros((rows, n_out), np.float32)
    y[np.arange(rows), rng.integers(0, n_out, rows)] = 1.0
    return x, y


def close(got, want, tol=1e-5):
    """The tolerance of re-ordered fp32 sums that this library holds its windows to: 1e-5 of the largest element."""
    err = np.max(np.abs(got - want)) / max(1e-30, np.max(np.abs(want)))
    assert err < tol, err


MUON = (0.9, True, 0.02, 5)
CASES = [
    # sizes, act, rows, engine, norms, muon layers, tensor cores
    ([13, 37, 29, 5], "tanh", 50, "AUTO", [1, 2], {}, False),
    ([13, 37, 29, 5], "tanh", 50, "FFMA", [], {0: MUON, 1: MUON, 2: MUON}, False),
    ([13, 37, 29, 5], "tanh", 50, "AUTO", [1], {1: (0.95, False, 0.0, 3)}, False),
    ([13, 37, 29, 5], "relu", 50, "FFMA", [2], {0: MUON, 2: (0.5, True, 0.0, 4)}, False),
    ([100, 300, 200, 10], "tanh", 333, "TCGEN05", [1, 2], {0: MUON, 1: MUON}, True),       # 3xFP16, ragged
    ([128, 256, 384, 128], "relu", 256, "TCGEN05", [1, 2], {1: MUON}, True),                # 3xTF32
    ([128, 256, 128, 16], "relu", 4096, "AUTO", [1], {0: MUON, 1: MUON}, True),              # 3xTF32 forward, 3xFP16 backward
    ([96, 200, 160, 7], "relu", 1, "AUTO", [1, 2], {}, False),                               # a window of one row
]


@pytest.mark.gpu
@pytest.mark.parametrize("sizes,act,rows,engine,norms,muons,tensor", CASES)
def test_window_against_64_bits(g, sizes, act, rows, engine, norms, muons, tensor):
    net, plain, rng = make(g, sizes, act, rows, 3, 0.05, getattr(g, "GEMM_" + engine), norms, muons)
    x, y = data(rng, plain, rows, sizes[0], sizes[-1])
    net.set_data(x, y)
    before = net.tensor_core_launches()
    out, am, _ = net.forward(0, rows)
    want = plain.forward(x)
    close(out, want)
    net.train_window(0, rows)
    plain.window(x, y)
    w, b = net.get_weights()
    at = 0
    for l, W in enumerate(plain.W):
        # an orthogonalised update has elements of lr / sqrt(n) whatever the gradient's size: the gradient's error relative to the
        # gradient (1e-6 of its largest element here) is passed on with the slope of the iteration at zero, at most 3.4445 ** 5 of it
        tol = 1e-5 if l not in muons else 1e-5 + 3.4445 ** 5 * 1e-6 * 0.05 * np.sqrt(max(1.0, W.shape[0] / W.shape[1])) / np.abs(W).max()
        close(w[at:at + W.size].reshape(W.shape), W, tol)
        at += W.size
    close(b, plain.b)
    for l in norms:
        gain, shift = net.get_norm_weights(l)
        close(gain, plain.gain[l])
        assert np.max(np.abs(shift - plain.shift[l])) < 1e-6
    assert (net.tensor_core_launches() > before) == tensor
    net.close()


@pytest.mark.gpu
def test_windows_one_behind_the_other_and_epochs(g):
    """The same windows through gl_train_window and gl_train_epochs give the same bits; a shorter last window."""
    sizes, rows, batch = [20, 64, 48, 6], 200, 64
    weights = []
    for way in range(2):
        net, plain, rng = make(g, sizes, "tanh", batch, 5, 0.05, g.GEMM_AUTO, [1, 2], {0: MUON, 2: MUON})
        x, y = data(rng, plain, rows, 20, 6)
        net.set_data(x, y)
        if way == 0:
            net.train_epochs(2)
        else:
            for _ in range(2):
                for r0 in range(0, rows, batch):
                    net.train_window(r0, min(batch, rows - r0))
        weights.append((net.get_weights(), [net.get_norm_weights(l) for l in (1, 2)]))
        net.close()
    (wa, na), (wb, nb) = weights
    assert np.array_equal(wa[0], wb[0]) and np.array_equal(wa[1], wb[1])
    for p, q in zip(na, nb):
        assert np.array_equal(p[0], q[0]) and np.array_equal(p[1], q[1])


@pytest.mark.gpu
def test_training_from_host_memory_and_serving_few_rows(g):
    sizes = [24, 96, 80, 9]
    net, plain, rng = make(g, sizes, "tanh", 128, 7, 0.05, g.GEMM_AUTO, [1, 2], {1: MUON})
    x, y = data(rng, plain, 128, 24, 9)
    net.train_window_host(x, y)
    plain.window(x, y)
    for rows in (1, 3, 17, 128):
        out, am, _ = net.forward_host(x[:rows])
        close(out, plain.forward(x[:rows]), 2e-5)  # (the window's tolerance and the pass's)
    net.set_data(x, y)
    a = net.activations(5)
    plain.forward(x)
    want = np.concatenate([plain.A[1][5], plain.A[2][5], plain.forward(x)[5]])
    close(a, want, 2e-5)
    net.close()


@pytest.mark.gpu
def test_checkpoint_goes_on_where_it_stood(g, tmp_path):
    sizes, rows = [16, 40, 32, 4], 60
    kw = dict(norms=[1], muons={0: MUON, 1: MUON})
    net, plain, rng = make(g, sizes, "tanh", rows, 9, 0.05, g.GEMM_AUTO, **kw)
    x, y = data(rng, plain, rows, 16, 4)
    net.set_data(x, y)
    for _ in range(3):
        net.train_window(0, rows)
    net.save_state(tmp_path / "s")
    other, _, _ = make(g, sizes, "tanh", rows, 10, 0.05, g.GEMM_AUTO, **kw)
    other.set_data(x, y)
    other.load_state(tmp_path / "s")
    for n in (net, other):
        for _ in range(2):
            n.train_window(0, rows)
    assert np.array_equal(net.get_weights()[0], other.get_weights()[0])
    assert np.array_equal(net.get_norm_weights(1)[0], other.get_norm_weights(1)[0])
    plainer, _, _ = make(g, sizes, "tanh", rows, 10, 0.05, g.GEMM_AUTO, norms=[], muons={})
    elsewhere, _, _ = make(g, sizes, "tanh", rows, 10, 0.05, g.GEMM_AUTO, norms=[2], muons={0: MUON, 1: MUON})
    for n in (plainer, elsewhere):
        with pytest.raises(g.GladesError):
            n.load_state(tmp_path / "s")
    plainer.save_state(tmp_path / "t")
    with pytest.raises(g.GladesError):
        other.load_state(tmp_path / "t")


@pytest.mark.gpu
def test_taking_it_out_again_and_non_finite_weights(g):
    """Without norms and orthogonalised updates the network trains as if they had never been there."""
    sizes, rows = [16, 40, 32, 4], 60
    w = []
    for special in (False, True):
        net, plain, rng = make(g, sizes, "tanh", rows, 11, 0.05, g.GEMM_AUTO, norms=[1] if special else [], muons={1: MUON} if special else {})
        x, y = data(rng, plain, rows, 16, 4)
        net.set_data(x, y)
        if special:
            net.train_window(0, rows)
            net.set_layer_norm(1, -1.0)
            net.set_muon(1, steps=0)
            net.set_weights(*start)
        else:
            start = net.get_weights()
        net.train_window(0, rows)
        w.append(net.get_weights()[0])
        net.close()
    assert np.array_equal(w[0], w[1])
    net, plain, rng = make(g, sizes, "tanh", rows, 11, 0.05, g.GEMM_AUTO, norms=[], muons={1: MUON})
    x, y = data(rng, plain, rows, 16, 4)
    bad = x.copy()
    bad[3, 2] = np.nan
    net.set_data(bad, y)
    assert net.train_window(0, rows).nonfinite == 1
    net.set_weights(*start)
    net.set_data(x, y)
    assert net.train_window(0, rows).nonfinite == 0  # weights and momentum are new
    net.close()


@pytest.mark.gpu
def test_refusals(g):
    net, _, _ = make(g, [8, 12, 10, 3], "tanh", 10, 1, 0.05, g.GEMM_AUTO, [], {})
    for call in (lambda: net.set_layer_norm(0), lambda: net.set_layer_norm(3), lambda: net.set_layer_norm(1, float("nan")),
                 lambda: net.set_layer_norm(1, float("inf")), lambda: net.set_muon(-1), lambda: net.set_muon(3), lambda: net.set_muon(0, steps=17),
                 lambda: net.set_muon(0, steps=-1), lambda: net.set_muon(0, momentum=float("nan")), lambda: net.get_norm_weights(1),
                 lambda: net.set_norm_weights(2, np.ones(10), np.ones(10))):
        with pytest.raises(g.GladesError):
            call()
    net.set_layer_norm(1)
    with pytest.raises(g.GladesError):
        net.snapshot_submit()
    d = g.make_desc([8, 12, 10, 3], ["tanh", "tanh", "softmax"], "classification", batch=4, lr=0.1, momentum=0.9, mode=g.MODE_BATCHED)
    with_momentum = g.Net(d)
    with pytest.raises(g.GladesError):
        with_momentum.set_muon(1)
    with_momentum.set_layer_norm(1)
    d = g.make_desc([8, 12, 10, 3], ["tanh", "tanh", "sigmoid"], "classification", batch=4, lr=0.1)
    reference = g.Net(d)
    for call in (lambda: reference.set_layer_norm(1), lambda: reference.set_muon(0)):
        with pytest.raises(g.GladesError):
            call()
