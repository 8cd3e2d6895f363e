"""What the operators' results are off by, and where they must be the same bits."""
import pytest

torch = pytest.importorskip("torch")

from test_gpu_operators import DEV, TYPES, gradient, run_ortho  # noqa: E402

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
