"""Every tile that the dense products are made of (256, 128 and 64 squares, and the 64 square with two groups of wavefronts), with and without
cut sums: on the CPU at ragged sizes with the tile chosen by the test, on the GPU at sizes whose launches choose it."""
import pytest
import torch

import dense_reference as ref
from test_dense import IDS, TYPES, bind, check_product, draw, gpu, gradients  # noqa: F401  (a fixture)
from test_dense import dense_emulation  # noqa: F401  (a fixture)

TILES = {"256": 0, "128": 1, "64": 2, "64-two-groups": 3}


@pytest.fixture(params=sorted(TILES))
def tile(request, dense_emulation, monkeypatch):  # noqa: F811
    import dpc_amd
    bind(monkeypatch, "ctypes")                                # (which asks for sizes anew when the plan changes)
    monkeypatch.setattr(dpc_amd.dense, "_SIZES", {})
    monkeypatch.setenv("DPC_EMU_TILE", str(TILES[request.param]))
    prev = dpc_amd._dense_capi.set_library(dense_emulation)
    yield request.param
    dpc_amd._dense_capi.set_library(prev)


@pytest.fixture(params=["whole", "cut"])
def cut(request, monkeypatch):
    if request.param == "cut":
        monkeypatch.setenv("DPC_EMU_DEAR", "1")
    return request.param == "cut"


def tolerance(a, b, want, dtype):
    """ref.product_tolerance, whose half step is relative; a half below 2^-14 has steps of 2^-24 whatever its size, and is off by half of one"""
    return ref.product_tolerance(a, b, want, dtype) + (2.0 ** -25 if dtype == torch.float16 else 0.0)


def check_gradients(x, w, bias, dy, got):
    """all of y, dx, dw, db against the held values' products"""
    y, dx, dw, db = got
    h = lambda t: ref.held(t.cpu())
    check_product(x, w, bias, y)
    for g, a, b, dtype in ((dx, h(dy), h(w.t()), x.dtype), (dw, h(dy.t()), h(x.t()), w.dtype)):
        want = a @ b.t()
        assert bool(((g.cpu().double() - want).abs() <= tolerance(a, b, want, dtype)).all())
    want = dy.cpu().double().sum(0)
    tol = ref.HALF_STEP[bias.dtype] * want.abs() + (x.shape[0] + 8) * 2.0 ** -24 * dy.cpu().double().abs().sum(0)
    assert bool(((db.cpu().double() - want).abs() <= tol).all())


@pytest.mark.parametrize("dtype", TYPES[:2], ids=IDS[:2])
def test_products_in_every_tile(tile, cut, dtype):
    """several tiles of each kind, odd ends; 9 lines are cut in two where the tile is, 6 are not; gradients with 3 and 2 lines"""
    import dpc_amd
    if dtype == torch.float32 and tile == "256":
        pytest.skip("sums through halves take tiles of at most 128")
    k = 1100 if cut else 700
    m, n = (261, 300) if tile in ("256", "128") else (70, 133)
    lib = dpc_amd._dense_capi.get_library()
    need = lib.dpc_dense_product_workspace(m, n, -(-k // 128), 0 if dtype == torch.float32 else 1)
    assert need == (2 * m * n * 4 if cut and tile != "64-two-groups" else 0)
    x, w, bias, dy = draw((m, k), 1, dtype, "cpu"), draw((n, k), 2, dtype, "cpu"), draw((n,), 3, dtype, "cpu"), draw((m, n), 4, dtype, "cpu", 1e-3)
    check_gradients(x, w, bias, dy, gradients(dpc_amd, x, w, bias, dy))


@pytest.mark.parametrize("dtype", TYPES[:2], ids=IDS[:2])
def test_orthogonalisation_in_every_tile(tile, cut, dtype):
    """two ragged matrices, one of them tall, in the same launches; two steps in one pass over X and one by itself where lines are dear"""
    import dpc_amd
    shapes = [(140, 600), (300, 131)] if tile in ("256", "128") else [(70, 600), (140, 131)]
    mats = [ref.gradient(s, i, dtype, 0.1) for i, s in enumerate(shapes)]
    steps = 3 if cut else 2
    for g, o in zip(mats, dpc_amd.dense.newton_schulz(mats, steps=steps)):
        assert ref.off(o, ref.newton_schulz(g, steps)) <= ref.orthogonal_tolerance(torch.float32, steps) + ref.HALF_STEP[dtype], tuple(g.shape)
    w = [draw(s, 9, dtype, "cpu") for s in shapes]
    was, mom = [t.double() for t in w], [torch.zeros(s) for s in shapes]
    dpc_amd.dense.muon_update(w, mats, mom, lr=0.5, adjust="none", momentum=0.0, steps=1)
    for g, now, before in zip(mats, w, was):
        o = ref.newton_schulz(g, 1)
        want = before - 0.5 * o
        tol = (ref.HALF_STEP[dtype] + 2.0 ** -23) * want.norm() + 0.5 * o.norm() * (ref.orthogonal_tolerance(torch.float32, 1) + 2.0 ** -23)
        assert (now.double() - want).norm() <= tol


# ---- on the GPU, at sizes that take them ------------------------------------------------------------------------------------------------
def sampled(got, a, b, bias, rows, dtype):
    """rows of got against a b^T (+ bias), a and b held values"""
    want = a[rows] @ b.t() + (0 if bias is None else bias.double())
    assert bool(((got[rows].double() - want).abs() <= tolerance(a[rows], b, want, dtype)).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("m,k,n", [(8192, 4096, 4096), (8191, 4100, 4095), (2050, 4096, 4090)])
def test_large_products(gpu, m, k, n, dtype):  # noqa: F811
    """tiles of 256 (16-bit results) and 128; rows from both ends and the middle, every column"""
    import dpc_amd
    x, w, bias = draw((m, k), 1, dtype, gpu), draw((n, k), 2, dtype, gpu, k ** -0.5), draw((n,), 3, torch.float32, gpu)
    dy = draw((m, n), 4, dtype, gpu, 1e-3)
    y, dx, dw, db = gradients(dpc_amd, x, w, bias, dy)
    pick = lambda size: torch.tensor(sorted({0, 1, 127, 128, 255, 256, size // 2, size // 2 + 37, size - 130, size - 2, size - 1}), device=gpu)
    sampled(y, ref.held(x), ref.held(w), bias, pick(m), dtype)
    sampled(dx, ref.held(dy), ref.held(w.t()), None, pick(m), dtype)
    sampled(dw, ref.held(dy.t()), ref.held(x.t()), None, pick(n), dtype)
    want = dy.double().sum(0)
    assert bool(((db.double() - want).abs() <= (ref.HALF_STEP[torch.float32] * want.abs() + (m + 8) * 2.0 ** -24 * dy.double().abs().sum(0))).all())
    packed = dpc_amd.dense.pack_weight_fp8(w)
    assert torch.equal(dpc_amd.dense.linear_fp8(x, packed, bias), y)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("m,k,n", [(1, 1024, 24000), (3, 700, 9000), (17, 500, 24000)])
def test_gradients_whose_sums_are_cut(gpu, m, k, n, dtype):  # noqa: F811
    """dx adds up 24000 values in up to 32 parts"""
    import dpc_amd
    x, w, bias, dy = draw((m, k), 1, dtype, gpu), draw((n, k), 2, dtype, gpu, k ** -0.5), draw((n,), 3, dtype, gpu), draw((m, n), 4, dtype, gpu, 1e-3)
    check_gradients(x, w, bias, dy, gradients(dpc_amd, x, w, bias, dy))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("shape", [(24000, 1024), (4096, 4096), (3001, 3000), (1500, 8001)], ids=lambda s: "%dx%d" % s)
def test_large_orthogonalisations(gpu, shape, dtype):  # noqa: F811
    """tiles of 128 and 256 in X X^T (cut in 14 and 3 parts) and in P X, of 128 between"""
    import dpc_amd
    g = ref.gradient(shape, 1, dtype, 0.1).to(gpu)
    want = ref.newton_schulz(g)
    assert ref.off(dpc_amd.dense.newton_schulz(g), want) <= ref.orthogonal_tolerance(torch.float32) + ref.HALF_STEP[dtype]
    w, mom = draw(shape, 2, dtype, gpu), torch.zeros(shape, device=gpu)
    was = w.double()
    dpc_amd.dense.muon_update([w], [g], [mom], lr=0.5, adjust="none", momentum=0.0)
    to = was - 0.5 * want
    tol = (ref.HALF_STEP[dtype] + 2.0 ** -23) * to.norm() + 0.5 * want.norm() * (ref.orthogonal_tolerance(torch.float32) + 2.0 ** -23)
    assert (w.double() - to).norm() <= tol
