"""Operators on device buffers: what their entry points refuse, and the sizes of their workspaces.  Needs no GPU: every refusal
comes before the device is asked for."""
import ctypes

import numpy as np
import pytest

INVALID, NO_DEVICE, TOO_LARGE = -1, -3, -8
P = 1 << 20  # an aligned address that nothing reads


def status(g, call):
    try:
        call()
    except g.GladesError as e:
        assert str(e)
        return e.status
    return 0


def last(g, call):
    with pytest.raises(g.GladesError) as e:
        call()
    return str(e.value)


def norm(g, **over):
    a = dict(d_x=P, ldx=8, d_gain=P, d_shift=P, d_y=P + 4096, ldy=8, d_mean=P, d_rstd=P, rows=4, n=8)
    a.update(over)
    return status(g, lambda: g.layer_norm(**a))


def back(g, **over):
    a = dict(d_dy=P, lddy=8, d_x=P + 4096, ldx=8, d_gain=P, d_mean=P, d_rstd=P, d_dx=P + 8192, lddx=8, d_dgain=P, d_dshift=P, rows=4,
             n=8, d_work=P, work_bytes=1 << 30)
    a.update(over)
    return status(g, lambda: g.layer_norm_backward(**a))


@pytest.mark.parametrize("over", [
    dict(dtype=3), dict(dtype=-1), dict(rows=-1), dict(n=0), dict(n=-5), dict(eps=-1e-3), dict(eps=float("nan")), dict(eps=float("inf")),
    dict(d_x=None), dict(d_y=None), dict(ldx=7), dict(ldy=7), dict(ldx=-8), dict(d_x=P + 2), dict(d_y=P + 1, dtype=1), dict(d_gain=P + 2),
    dict(d_shift=P + 1), dict(d_mean=P + 2), dict(d_rstd=P + 3), dict(d_y=P, ldy=16), dict(device=-1), dict(device=64)])
def test_layer_norm_refuses(g, over):
    assert norm(g, **over) == INVALID


@pytest.mark.parametrize("over", [
    dict(dtype=3), dict(rows=-1), dict(n=0), dict(d_dy=None), dict(d_x=None), dict(lddy=7), dict(ldx=7), dict(lddx=7), dict(d_mean=None),
    dict(d_rstd=None), dict(d_dx=P + 2), dict(d_dgain=P + 2), dict(d_work=None), dict(work_bytes=8), dict(d_dx=P, lddx=16),
    dict(d_dx=P + 4096, lddx=9), dict(device=99)])
def test_layer_norm_backward_refuses(g, over):
    assert back(g, **over) == INVALID


def ortho_item(**over):
    a = dict(rows=4, cols=8, d_in=P, ld_in=8, d_out=P + 4096, ld_out=8)
    a.update(over)
    return a


def muon_item(**over):
    a = dict(rows=4, cols=8, lr=0.1, d_grad=P, ld_grad=8, d_momentum=P + 4096, d_momentum_out=P + 4096, ld_momentum=8, d_weight=P + 8192,
             d_weight_out=P + 8192, ld_weight=8)
    a.update(over)
    return a


@pytest.mark.parametrize("over", [
    dict(rows=0), dict(cols=0), dict(rows=-3), dict(d_in=None), dict(d_out=None), dict(ld_in=7), dict(ld_out=7), dict(d_in=P + 2),
    dict(rows=1 << 30, cols=(1 << 30) + 1)])
def test_orthogonalize_refuses_matrices(g, over):
    items = g.ortho_items([ortho_item(d_out=P + 12288), ortho_item(**over)])
    assert status(g, lambda: g.orthogonalize(items, P, 1 << 40)) == INVALID


@pytest.mark.parametrize("over", [
    dict(rows=0), dict(cols=-1), dict(d_grad=None), dict(d_momentum=None), dict(d_momentum_out=None), dict(d_weight=None),
    dict(d_weight_out=None), dict(ld_grad=7), dict(ld_momentum=7), dict(ld_weight=7), dict(d_weight=P + 2), dict(lr=float("nan"))])
def test_muon_refuses_matrices(g, over):
    items = g.muon_items([muon_item(**over)])
    assert status(g, lambda: g.muon_step(items, P, 1 << 40)) == INVALID


def test_orthogonalize_refuses_an_output_twice(g):
    one = ortho_item()
    free = dict(d_work=P, work_bytes=1 << 30)
    for other in (ortho_item(), ortho_item(d_in=P + 12288), ortho_item(d_in=P + 4096, d_out=P + 8192), ortho_item(d_in=P + 12288, d_out=P)):
        for items in ((one, other), (other, one)):
            assert status(g, lambda: g.orthogonalize(g.ortho_items(items), **free)) == INVALID
    # one input for two outputs, and every output in its input's place, are taken: only the device is missing, if that
    for items in ((one, ortho_item(d_out=P + 8192)), (ortho_item(d_out=P), ortho_item(d_in=P + 4096))):
        assert status(g, lambda: g.orthogonalize(g.ortho_items(items), P, 100)) == INVALID
        assert "workspace" in last(g, lambda: g.orthogonalize(g.ortho_items(items), P, 100))


@pytest.mark.parametrize("over", [
    dict(d_weight_out=P + 4096), dict(d_momentum_out=P), dict(d_weight_out=P), dict(d_momentum_out=P + 8192), dict(d_momentum=P + 8192)])
def test_muon_refuses_an_output_that_is_another_argument(g, over):
    free = dict(d_work=P, work_bytes=1 << 30)
    assert status(g, lambda: g.muon_step(g.muon_items([muon_item(**over)]), **free)) == INVALID
    assert "output" in last(g, lambda: g.muon_step(g.muon_items([muon_item(**over)]), P, 100))


def test_muon_refuses_a_matrix_twice(g):
    assert "output" in last(g, lambda: g.muon_step(g.muon_items([muon_item(), muon_item()]), P, 100))
    other = muon_item(d_momentum=P + 16384, d_momentum_out=P + 20480, d_weight=P + 24576, d_weight_out=P + 28672)
    assert "workspace" in last(g, lambda: g.muon_step(g.muon_items([muon_item(), other]), P, 100))


@pytest.mark.parametrize("over", [
    dict(steps=0), dict(steps=17), dict(eps=-1.0), dict(eps=float("nan")), dict(dtype=7), dict(work_bytes=100), dict(d_work=None),
    dict(coefficients=[(100.0, 0.0, 0.0)] * 5), dict(coefficients=[(float("nan"), 0.0, 0.0)] * 5),
    dict(coefficients=[(8.0, -1.0, 0.0)] * 5), dict(device=-1)])
def test_orthogonalisation_refuses_arguments(g, over):
    a = dict(d_work=P, work_bytes=1 << 30)
    a.update(over)
    items, muon = g.ortho_items([ortho_item()]), g.muon_items([muon_item()])
    assert status(g, lambda: g.orthogonalize(items, **a)) == INVALID
    assert status(g, lambda: g.muon_step(muon, **a)) == INVALID


def test_muon_refuses_factors_that_are_no_numbers(g):
    items = g.muon_items([muon_item()])
    assert status(g, lambda: g.muon_step(items, P, 1 << 30, momentum=float("nan"))) == INVALID
    assert status(g, lambda: g.muon_step(items, P, 1 << 30, weight_decay=float("inf"))) == INVALID


def test_coefficients_of_another_number_of_steps(g):
    items = g.ortho_items([ortho_item()])
    with pytest.raises(ValueError):
        g.orthogonalize(items, P, 1 << 30, coefficients=[(2.0, -1.5, 0.5)] * 4, steps=5)


def test_usual_coefficients_are_taken(g):
    """Without a GPU a call that is in order gets as far as the device."""
    if g.device_count() > 0:
        pytest.skip("there is a device: these addresses must not be used")
    items = g.ortho_items([ortho_item()])
    for c in (None, [(2.0, -1.5, 0.5)] * 5, [(1.5, -0.5, 0.0)] * 5, [(1.0, 0.0, 0.0)] * 5, [(0.0, 0.0, 0.0)] * 5,
              [(8.28721, -23.59589, 17.30039), (4.10706, -2.94785, 0.54484), (3.94869, -2.90890, 0.55182), (3.31842, -2.48849, 0.51005),
               (2.30065, -1.66890, 0.41881)]):
        assert status(g, lambda: g.orthogonalize(items, P, 1 << 30, coefficients=c)) == NO_DEVICE
    assert status(g, lambda: g.muon_step(g.muon_items([muon_item()]), P, 1 << 30)) == NO_DEVICE
    assert norm(g) == NO_DEVICE
    assert norm(g, d_gain=None, d_shift=None, d_mean=None, d_rstd=None) == NO_DEVICE
    assert back(g) == NO_DEVICE


def test_nothing_to_do(g):
    assert norm(g, rows=0, d_x=None, d_y=None) == 0
    assert status(g, lambda: g.orthogonalize(g.ortho_items([]), None, 0)) == 0
    assert g.orthogonalize_workspace(g.ortho_items([])) >= 0


def test_workspaces(g):
    assert g.layer_norm_backward_workspace(0, 4096) >= 0
    for rows, n in ((1, 1), (8192, 4096), (3, 40000), (1 << 40, 7), (5, 1 << 30)):
        assert g.layer_norm_backward_workspace(rows, n) >= 8 * n
    for rows, n in ((-1, 4), (4, 0), (4, -1)):
        assert status(g, lambda: g.layer_norm_backward_workspace(rows, n)) == INVALID
    small, large = g.ortho_items([ortho_item()]), g.ortho_items([ortho_item(rows=4096, cols=4096, ld_in=4096, ld_out=4096)] * 16)
    assert 0 < g.orthogonalize_workspace(small) < g.orthogonalize_workspace(large)
    # more matrices than one launch takes share its space
    twice = g.ortho_items([ortho_item(rows=4096, cols=4096, ld_in=4096, ld_out=4096)] * 32)
    assert g.orthogonalize_workspace(twice) == g.orthogonalize_workspace(large)
    assert status(g, lambda: g.orthogonalize_workspace(g.ortho_items([ortho_item(rows=0)]))) == INVALID
    vast = g.ortho_items([ortho_item(rows=1 << 30, cols=1 << 30)])
    assert status(g, lambda: g.orthogonalize_workspace(vast)) == TOO_LARGE
    assert g.muon_workspace(g.muon_items([muon_item()])) == g.orthogonalize_workspace(small)
