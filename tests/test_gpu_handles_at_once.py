"""One host thread per handle: networks of different sizes that run on the same kernels at the same time."""
import threading

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

KINDS = {
    # two networks of one kernel each, whose shared memory differs
    "small networks": dict(epochs=1500, sizes=([16, 24, 4], [24, 30, 36, 9]), batch=16, rows=16, mode="BATCHED", gemm="AUTO", out="softmax"),
    "whole windows": dict(epochs=2000, sizes=([256, 256, 64, 8], [128, 320, 320, 8]), batch=64, rows=64, mode="BATCHED", gemm="GRID_FUSED", out="softmax"),
    "reference order, small": dict(epochs=1500, sizes=([8, 12, 1], [16, 20, 1]), batch=1, rows=4, mode="REFERENCE", gemm="AUTO", out="sigmoid"),
    "reference order": dict(epochs=600, sizes=([30, 60, 50, 20, 1], [30, 90, 70, 40, 1]), batch=4, rows=4, mode="REFERENCE", gemm="AUTO", out="sigmoid"),
    "layers": dict(epochs=1000, sizes=([300, 500, 7], [900, 500, 7]), batch=40, rows=40, mode="BATCHED", gemm="FFMA", out="softmax"),
}


def make(g, sizes, batch, rows, mode, gemm, out, seed):
    rng = np.random.default_rng(seed)
    w = np.concatenate([rng.uniform(-1, 1, o * i) / np.sqrt(i) for i, o in zip(sizes, sizes[1:])]).astype(np.float32)
    d = g.make_desc(list(sizes), ["tanh"] * (len(sizes) - 2) + [out], "classification" if sizes[-1] > 1 else "regression", batch=batch, lr=0.01,
                    mode=getattr(g, "MODE_" + mode), gemm=getattr(g, "GEMM_" + gemm))
    net = g.Net(d)
    net.set_weights(w, np.zeros(len(sizes) - 2, np.float32))
    x = rng.standard_normal((rows, sizes[0])).astype(np.float32)
    y = rng.uniform(0, 1, (rows, sizes[-1])).astype(np.float32)
    net.set_data(x, y)
    return net


@pytest.mark.parametrize("kind", list(KINDS))
def test_networks_of_different_sizes_in_threads_of_their_own(g, kind):
    """No call fails, and the weights are those of a network that trains alone."""
    k = dict(KINDS[kind])
    shapes, epochs = k.pop("sizes"), k.pop("epochs")

    def train(net):
        for _ in range(epochs):
            net.train_epochs(1)
    want = []
    for i, sizes in enumerate(shapes):
        net = make(g, sizes, seed=i, **k)
        train(net)
        want.append(net.get_weights())
        net.close()
    nets, errors = [make(g, shapes[i % 2], seed=i % 2, **k) for i in range(8)], []

    def work(net):
        try:
            train(net)
        except Exception as e:  # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=work, args=(n,)) for n in nets]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for i, net in enumerate(nets):
        w, b = net.get_weights()
        assert np.array_equal(w, want[i % 2][0]) and np.array_equal(b, want[i % 2][1])
        net.close()
