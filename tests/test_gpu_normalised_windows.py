"""Several windows of networks with normalised layers and orthogonalised updates on the tensor-core engines, against the plain 64-bit
implementation: what a window leaves behind for the next pass (parts of the new weights, scales, momenta)."""
import numpy as np
import pytest

from test_gpu_normalised_networks import MUON, Plain, close, data, make

pytestmark = pytest.mark.gpu

CASES = [
    # sizes, act, rows, engine, norms, muon layers
    ([100, 300, 200, 10], "tanh", 333, "TCGEN05", [1, 2], {0: MUON, 1: MUON}),     # 3xFP16, ragged
    ([128, 256, 384, 128], "relu", 256, "TCGEN05", [1, 2], {1: MUON}),             # 3xTF32
    ([128, 256, 384, 128], "relu", 256, "TCGEN05", [2], {0: MUON, 2: MUON}),
    ([128, 256, 128, 16], "relu", 4096, "AUTO", [1], {0: MUON, 1: MUON}),          # 3xTF32 forward, 3xFP16 backward
]


def network(g, sizes, act, rows, engine, norms, muons, seed=3, lr=0.05):
    """Weights and inputs whose hidden sums stay far above the reference's ReLU jump (0.046) in every window: positive ones of different
    size per node, normalised layers around 1."""
    rng = np.random.default_rng(seed)
    w = []
    for i, o in zip(sizes, sizes[1:-1]):
        w.append(rng.uniform(0.2, 1.0, (o, i)) * 1.7 / i * rng.uniform(0.5, 2.0, (o, 1)))
    w.append(rng.uniform(-1, 1, (sizes[-1], sizes[-2])) * np.sqrt(2.0 / sizes[-2]))
    w = np.concatenate([v.ravel() for v in w]).astype(np.float32)
    b = rng.uniform(0.0, 0.1, len(sizes) - 2).astype(np.float32)
    d = g.make_desc(sizes, [act] * (len(sizes) - 2) + ["softmax"], "classification", batch=rows, lr=lr, mode=g.MODE_BATCHED,
                    gemm=getattr(g, "GEMM_" + engine))
    net, plain = g.Net(d), Plain(sizes, act, w, b, lr, norms, dict(muons))
    net.set_weights(w, b)
    for l in norms:
        net.set_layer_norm(l)
        gain, shift = rng.uniform(0.1, 0.2, sizes[l]).astype(np.float32), rng.uniform(0.9, 1.1, sizes[l]).astype(np.float32)
        net.set_norm_weights(l, gain, shift)
        plain.gain[l], plain.shift[l] = gain.astype(np.float64), shift.astype(np.float64)
    for l, (mu, nesterov, decay, steps) in muons.items():
        net.set_muon(l, mu, nesterov, decay, steps)
    x = rng.uniform(0.5, 1.5, (rows, sizes[0])).astype(np.float32)
    y = np.zeros((rows, sizes[-1]), np.float32)
    y[np.arange(rows), rng.integers(0, sizes[-1], rows)] = 1.0
    net.set_data(x, y)
    return net, plain, x, y


def check(net, plain, muons, windows):
    """After `windows` windows: each adds what one window may be off by (test_gpu_normalised_networks.py), and passes on what the weights
    were off by through its gradient, by no more than that again."""
    w, b = net.get_weights()
    at = 0
    for l, W in enumerate(plain.W):
        tol = 1e-5 if l not in muons else 1e-5 + 3.4445 ** 5 * 1e-6 * 0.05 * np.sqrt(max(1.0, W.shape[0] / W.shape[1])) / np.abs(W).max()
        close(w[at:at + W.size].reshape(W.shape), W, 2 * windows * tol)
        at += W.size
    close(b, plain.b, 2 * windows * 1e-5)


@pytest.mark.parametrize("sizes,act,rows,engine,norms,muons", CASES)
def test_three_windows_and_inference(g, sizes, act, rows, engine, norms, muons):
    net, plain, x, y = network(g, sizes, act, rows, engine, norms, muons)
    for window in range(1, 4):
        before = net.tensor_core_launches()
        net.train_window(0, rows)
        assert net.tensor_core_launches() > before
        plain.window(x, y)
        assert act != "relu" or plain.margin.min() > 1e-2
        check(net, plain, muons, window)
        before = net.tensor_core_launches()
        out, _, _ = net.forward(0, rows)
        assert net.tensor_core_launches() > before
        close(out, plain.forward(x), 2 * (window + 1) * 1e-5)
    for l in norms:
        gain, shift = net.get_norm_weights(l)
        close(gain, plain.gain[l])
        close(shift, plain.shift[l])
    net.close()


@pytest.mark.parametrize("sizes,act,rows,engine,norms,muons", CASES)
def test_updates_and_norms_switched_between_windows(g, sizes, act, rows, engine, norms, muons):
    """An orthogonalised update goes back to SGD, a layer that had SGD gets one, a norm is taken out: the next window reads the weights that
    the last one left, whichever way they were written."""
    net, plain, x, y = network(g, sizes, act, rows, engine, norms, muons)

    def window(n):
        net.train_window(0, rows)
        plain.window(x, y)
        assert act != "relu" or plain.margin.min() > 1e-2
        check(net, plain, touched, n)
    touched = set(muons)
    window(1)
    out = sorted(muons)[0]
    net.set_muon(out, steps=0)
    del plain.muons[out], plain.M[out]
    window(2)
    new = next(l for l in range(len(sizes) - 1) if l not in muons)
    net.set_muon(new, *MUON)
    plain.muons[new], plain.M[new] = MUON, np.zeros_like(plain.W[new])
    touched.add(new)
    window(3)
    net.set_layer_norm(norms[0], -1.0)
    del plain.gain[norms[0]], plain.shift[norms[0]]
    window(4)
    close(net.forward(0, rows)[0], plain.forward(x), 1e-4)
    net.close()


@pytest.mark.parametrize("sizes,act,rows,norms,muons,tensor", [
    ([784, 2048, 2048, 10], "tanh", 512, [1, 2], {0: (0.95, True, 0.01, 5), 1: (0.95, True, 0.01, 5), 2: (0.95, True, 0.01, 5)}, True),
    ([784, 1000, 500, 10], "relu", 700, [1, 2], {0: MUON, 1: MUON}, False),  # fp32 tiles
    ([1024, 4096, 1024], "tanh", 128, [1], {1: MUON}, True),
])
def test_window_of_wide_layers(g, sizes, act, rows, norms, muons, tensor):
    """The benchmark networks' layers, one window and an inference pass."""
    net, plain, rng = make(g, sizes, act, rows, 3, 0.05, g.GEMM_AUTO, norms, muons)
    x, y = data(rng, plain, rows, sizes[0], sizes[-1])
    net.set_data(x, y)
    before = net.tensor_core_launches()
    close(net.forward(0, rows)[0], plain.forward(x))
    net.train_window(0, rows)
    assert (net.tensor_core_launches() > before) == tensor
    plain.window(x, y)
    check(net, plain, muons, 1)
    for l in norms:
        close(net.get_norm_weights(l)[0], plain.gain[l])
    net.close()
