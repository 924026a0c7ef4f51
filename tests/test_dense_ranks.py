"""Orthogonalisation and the update (dpc_amd.dense) where the matrix has fewer ranks than rows, as a small batch's gradient has, and over many
steps; on the CPU through the emulation of the kernels and on the GPU (-m gpu)."""
import pytest
import torch

import dense_reference as ref
from test_dense import IDS, TYPES, bind, dense_emulation  # noqa: F401  (a fixture)

DEFAULT = ref.COEFFICIENTS


@pytest.fixture(params=["emulation", pytest.param("gpu", marks=pytest.mark.gpu)])
def device(request, monkeypatch):
    """where the operators run, through the compiled binding (the other one calls the same library)"""
    import dpc_amd
    bind(monkeypatch, "compiled")
    lib = request.getfixturevalue("dense_emulation") if request.param == "emulation" else None
    prev = dpc_amd._dense_capi.set_library(lib)
    yield torch.device("cpu" if lib is not None else "cuda")
    dpc_amd._dense_capi.set_library(prev)


def of_rank(shape, rank, seed, dtype=torch.float32):
    """a product of two random factors; rank 0: of full rank"""
    g = torch.Generator().manual_seed(seed)
    r, c = shape
    x = torch.randn(r, rank, generator=g) @ torch.randn(rank, c, generator=g) if rank else torch.randn(r, c, generator=g)
    return (1e-3 * x).to(dtype)


def scalar_bound(steps, coefficients):
    """the largest value that x <- a x + b x^3 + c x^5 reaches from [0, 1]: what no singular value passes but for rounding"""
    top, reached = 1.0, 0.0
    for a, b, c in coefficients if isinstance(coefficients[0], tuple) else [coefficients] * steps:
        x = torch.linspace(0, top, 20001, dtype=torch.float64)
        top = float((a * x + b * x ** 3 + c * x ** 5).abs().max())
        reached = max(reached, top)
    return reached


NARROW = [(16, 40), (32, 64), (48, 64), (70, 64), (100, 31)]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("steps,coefficients", [(12, DEFAULT), (16, DEFAULT), (20, DEFAULT), (64, DEFAULT), (40, (2.0, -1.5, 0.5)), (64, (1.5, -0.5, 0.0))],
                         ids=lambda v: str(v) if isinstance(v, int) else "%g" % v[0])
def test_many_steps_of_matrices_of_few_ranks(device, steps, coefficients, dtype):
    """singular values stay within what the scalar iteration reaches: 1 + 2^-5 of it (a map of slope at most 3.5 there, and what 32 bits or the
    result's 8 move a value by in the last steps, is well below)"""
    import dpc_amd
    if device.type == "cpu" and (steps, dtype) not in ((20, torch.float32), (64, torch.bfloat16)):
        pytest.skip("an emulated work-group of a thousand threads takes seconds a step")
    mats = [of_rank(s, rank, i, dtype).to(device) for i, s in enumerate(NARROW[:1] + NARROW[3:4] if device.type == "cpu" else NARROW)
            for rank in ((3,) if device.type == "cpu" else (1, 3, 5, 0))]
    bound = scalar_bound(steps, coefficients)
    for g, o in zip(mats, dpc_amd.dense.newton_schulz(mats, steps=steps, coefficients=coefficients)):
        assert bool(torch.isfinite(o).all()), tuple(g.shape)
        assert float(torch.linalg.matrix_norm(o.cpu().double(), 2)) <= bound * (1 + 2.0 ** -5), tuple(g.shape)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_many_steps_converge_to_the_polar_factor(device, dtype):
    """coefficients whose iteration ends at 1: every later rounding is taken back, so that the result is the polar factor of a matrix of full
    rank as exactly as one step computes it"""
    import dpc_amd
    for shape in NARROW[:1] if device.type == "cpu" else NARROW:
        g = of_rank(shape, 0, 7, dtype)
        u, _, v = torch.linalg.svd(g.double(), full_matrices=False)
        for steps in (20, 40, 64):
            o = dpc_amd.dense.newton_schulz(g.to(device), steps=steps, coefficients=(2.0, -1.5, 0.5))
            # P X adds up 64 products of 2^-24 each, of factors that are at most twice the result
            assert ref.off(o.cpu(), u @ v) <= ref.HALF_STEP[dtype] + 2 * 64 * 2.0 ** -24, (shape, steps)


def test_narrow_matrices_of_few_ranks(device):
    """up to nine steps are one polynomial P of A.  On what U has (almost) nothing of, P is a^steps, and P X takes that back where U has
    something: P's own rounding, and that of the products' sums, leave 2^-24 a^steps each, against singular values that end above 0.68"""
    import dpc_amd
    for steps in (5, 8):
        for i, shape in enumerate(NARROW[:3] if device.type == "cpu" else NARROW):
            for rank in (1, 5):
                g = of_rank(shape, rank, 10 * i + rank)
                o = dpc_amd.dense.newton_schulz(g.to(device), steps=steps)
                assert ref.off(o.cpu(), ref.newton_schulz(g, steps)) <= 2 * 2.0 ** -24 * DEFAULT[0] ** steps / 0.68, (shape, rank, steps)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_muon_update_of_many_steps(device, dtype):
    import dpc_amd
    shapes = [(100, 16), (32, 100), (64, 70)][:1 if device.type == "cpu" else 3]
    w = [of_rank(s, 0, i, dtype).to(device) for i, s in enumerate(shapes)]
    m = [torch.zeros(s, device=device) for s in shapes]
    before, bound = [t.cpu().double() for t in w], scalar_bound(20, DEFAULT)
    g = [of_rank(s, 2, 9 + i, dtype).to(device) for i, s in enumerate(shapes)]
    dpc_amd.dense.muon_update(w, g, m, lr=0.02, steps=20, weight_decay=0.1, momentum=0.9, nesterov=False)
    for s, now, was, mom, grad in zip(shapes, w, before, m, g):
        assert bool(torch.isfinite(now).all())
        assert torch.allclose(mom.cpu(), 0.1 * grad.cpu().float(), rtol=2.0 ** -20, atol=0)      # moved once, not once a round
        step = now.cpu().double() - (1 - 0.02 * 0.1) * was
        most = 0.02 * 0.2 * max(s) ** 0.5 * bound * (1 + 2.0 ** -5) + 2 * ref.HALF_STEP[dtype] * now.cpu().double().norm()
        assert float(torch.linalg.matrix_norm(step, 2)) <= most
        assert float(step.abs().max()) > 0
