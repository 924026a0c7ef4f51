"""Tensors whose memory does not hold their values as they are (negative views, as conj().imag gives), and forward-mode derivatives, in
dpc_amd.dense: taken for what they stand for, or refused; through both bindings."""
import pytest
import torch

import dense_reference as ref
from test_dense import IDS, TYPES, bind, device, draw, emulated, dense_emulation  # noqa: F401  (fixtures)


def negative(t):
    """-t, as a view that is to be read with its sign turned"""
    v = torch._neg_view(t.clone())
    assert v.is_neg() and v.is_contiguous()
    return v


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_negative_views_are_read_with_their_sign(device, dtype):
    import dpc_amd
    d = dpc_amd.dense
    x, w, bias, dy = (draw(s, i, dtype, device) for i, s in enumerate(((5, 40), (9, 40), (9,), (5, 9))))
    nx, nw, nb, ndy = (negative(t) for t in (x, w, bias, dy))
    assert torch.equal(d.linear_fp8(nx, nw, nb), d.linear_fp8(-x, -w, -bias))
    want, got = d.pack_weight_fp8(-w), d.pack_weight_fp8(nw)
    assert torch.equal(got.values.view(torch.uint8), want.values.view(torch.uint8)) and torch.equal(got.scales, want.scales)
    assert torch.equal(d.linear_fp8(nx, want, nb), d.linear_fp8(-x, want, -bias))
    for rows in (1, 20):                                       # the form for few rows, and the tiles
        one = x[:1].repeat(rows, 1)
        assert torch.equal(d.linear_fp8(negative(one), want), d.linear_fp8(-one, want))
    assert torch.equal(d.newton_schulz(nx), d.newton_schulz(-x))
    assert torch.equal(d.newton_schulz([nx, nw])[1], d.newton_schulz([-x, -w])[1])
    leaves = [t.clone().requires_grad_() for t in (x, w, bias)]
    got, want = (torch.autograd.grad(d.linear_fp8(*leaves), leaves, t) for t in (ndy, -dy))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # through views of the leaves: y = (-x)(-w)^T - bias, whose gradients come back through the views
    got = torch.autograd.grad(d.linear_fp8(*[torch._neg_view(t) for t in leaves]), leaves, dy)
    want = torch.autograd.grad(d.linear_fp8(*[-t for t in leaves]), leaves, dy)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_the_imaginary_part_of_a_conjugate(device):
    import dpc_amd
    z = torch.complex(torch.ones(1, 12), torch.ones(1, 12)).to(device)
    x = z.conj().imag[:, :1].expand(1, 1)
    assert x.is_neg()
    assert float(dpc_amd.dense.linear_fp8(x, torch.ones(1, 1, device=device))) == -1.0


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_negative_views_in_the_update(device, dtype):
    import dpc_amd
    up = dpc_amd.dense.muon_update
    w, g = draw((8, 12), 1, dtype, device), draw((8, 12), 2, dtype, device)
    a, b = w.clone(), w.clone()
    ma, mb = torch.zeros(8, 12, device=device), torch.zeros(8, 12, device=device)
    up([a], [negative(g)], [ma], lr=0.1)
    up([b], [-g], [mb], lr=0.1)
    assert torch.equal(a, b) and torch.equal(ma, mb) and not torch.equal(a, w)
    keep = [a.clone(), ma.clone()]
    for bad in (([negative(w)], [g], [ma], 0.1), ([a], [g], [negative(ma)], 0.1), ([a], [g], [ma], negative(torch.full((1,), 0.1, device=device)))):
        with pytest.raises(ValueError):
            up(bad[0], bad[1], bad[2], lr=bad[3])
    assert torch.equal(a, keep[0]) and torch.equal(ma, keep[1])


def test_packed_weights_that_are_negative_views_are_refused(emulated):
    d = emulated.dense
    p = d.pack_weight_fp8(torch.ones(3, 8))
    try:
        values = torch._neg_view(p.values)
    except RuntimeError:
        pytest.skip("this torch makes no negative views of 8-bit types")
    with pytest.raises(ValueError):
        d.linear_fp8(torch.ones(2, 8), p._replace(values=values))


def test_forward_mode_derivatives_are_refused(device):
    """the tangent of a dual tensor is not dropped in silence, with gradients enabled or not"""
    import dpc_amd
    import torch.autograd.forward_ad as fw
    d = dpc_amd.dense
    x, w, bias = torch.ones(2, 8, device=device), torch.ones(3, 8, device=device), torch.ones(3, device=device)
    p, m = d.pack_weight_fp8(w), torch.zeros(3, 8, device=device)
    with fw.dual_level():
        dual = lambda t: fw.make_dual(t.clone(), torch.ones_like(t))
        calls = [lambda: d.linear_fp8(dual(x), w), lambda: d.linear_fp8(x, dual(w)), lambda: d.linear_fp8(x, w, dual(bias)),
                 lambda: d.linear_fp8(dual(x), p), lambda: d.linear_fp8(x, p, dual(bias)), lambda: d.pack_weight_fp8(dual(w)),
                 lambda: d.newton_schulz(dual(x)), lambda: d.newton_schulz([x, dual(x)]), lambda: d.muon_update([dual(w)], [w], [m], lr=0.1),
                 lambda: d.muon_update([w], [dual(w)], [m], lr=0.1), lambda: d.muon_update([w], [w.clone()], [dual(m)], lr=0.1),
                 lambda: d.muon_update([w], [w.clone()], [m], lr=dual(torch.ones(1, device=device)))]
        for call in calls:
            with pytest.raises(RuntimeError):                  # (NotImplementedError is one)
                call()
            with torch.no_grad(), pytest.raises(RuntimeError):
                call()
        want = d.linear_fp8(x, p)                              # what has no tangent runs as ever
    assert torch.equal(want, d.linear_fp8(x, p)) and not m.any() and torch.equal(w, torch.ones_like(w))
