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
    bound = scalar_bound(steps, coefficients)
    # (beside larger matrices sides of 33 .. 64 are tiled: the last list is a call of its own)
    for shapes in [NARROW[:1] + NARROW[3:4]] if device.type == "cpu" else [NARROW, [(80, 90), (130, 300)]]:
        mats = [of_rank(s, rank, i, dtype).to(device) for i, s in enumerate(shapes) for rank in ((3,) if device.type == "cpu" else (1, 3, 5, 0))]
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


def few_ranks_tolerance(dtype, steps):
    """A step is off by at most 12.3 * 2^-22 of what it computes with (X and the polynomial's matrices, held in 22 bits), and the steps behind
    enlarge that by a each, at most, where the matrix has nothing itself; singular values pass 1.21 at no step and end above 0.68.  Then the
    result's rounding.  (That is half of bf16's for five steps, so what is held in fewer bits than 22 shows.)"""
    a = DEFAULT[0]
    return ref.HALF_STEP[dtype] + 12.3 * 2.0 ** -22 * (a ** steps - 1) / (a - 1) * 1.21 / 0.68


FEW_RANKS = [((70, 200), 1, 5), ((80, 90), 5, 5), ((80, 90), 5, 6), ((80, 90), 5, 8), ((130, 300), 4, 5)]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("shape,rank,steps", FEW_RANKS + [pytest.param(s, r, n, marks=pytest.mark.gpu) for s, r, n in (
    ((300, 320), 8, 5), ((300, 320), 32, 5), ((320, 300), 1, 3), ((512, 640), 16, 5), ((700, 701), 16, 6), ((128, 8000), 4, 5), ((24000, 256), 16, 5))],
    ids=lambda v: "x".join(map(str, v)) if isinstance(v, tuple) else str(v))
def test_matrices_of_few_ranks(device, shape, rank, steps, dtype):
    """a small batch's gradient: as exact as its type's rounding in every type, whatever the rank"""
    if device.type == "cpu" and (shape, rank, steps) not in FEW_RANKS:
        pytest.skip("sizes for the GPU")
    import dpc_amd
    g = of_rank(shape, rank, 5, dtype)
    o = dpc_amd.dense.newton_schulz(g.to(device), steps=steps)
    assert ref.off(o.cpu(), ref.newton_schulz(g.to(device), steps).cpu()) <= few_ranks_tolerance(dtype, steps)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_strong_directions(device, dtype):
    """a few directions 64 and 256 times as strong as the rest"""
    import dpc_amd
    for shape, n, size in (((70, 130), 4, 64.0),) if device.type == "cpu" else (((128, 400), 4, 64.0), ((300, 320), 16, 256.0)):
        g = torch.Generator().manual_seed(3)
        x = torch.randn(shape, generator=g) + size / n ** 0.5 * torch.randn(shape[0], n, generator=g) @ torch.randn(n, shape[1], generator=g)
        x = x.mul(1e-4).to(dtype)
        assert ref.off(dpc_amd.dense.newton_schulz(x.to(device)).cpu(), ref.newton_schulz(x)) <= few_ranks_tolerance(dtype, 5)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=IDS[:2])
def test_update_with_a_small_batchs_gradient(device, dtype):
    """linear_fp8's gradient of 16 rows into muon_update: the weights move by the formula's step"""
    import dpc_amd
    n, k = (150, 70) if device.type == "cpu" else (600, 256)
    g = torch.Generator().manual_seed(1)
    x, dy = (torch.randn(16, s, generator=g).to(dtype).to(device) for s in (k, n))
    w = (torch.randn(n, k, generator=g) / 16).to(dtype).to(device).requires_grad_()
    dw, = torch.autograd.grad(dpc_amd.dense.linear_fp8(x, w), w, 1e-3 * dy)
    was, m = w.detach().cpu().double(), torch.zeros(n, k, device=device)
    dpc_amd.dense.muon_update([w], [dw], [m], lr=0.5, adjust="none", momentum=0.5, nesterov=False)
    u = 0.5 * dw.cpu().double()
    o = ref.newton_schulz(u)
    want = was - 0.5 * o
    tol = (ref.HALF_STEP[dtype] + 2.0 ** -23) * want.norm() + 0.5 * o.norm() * (few_ranks_tolerance(dtype, 5) - ref.HALF_STEP[dtype] + 2.0 ** -23)
    assert (w.detach().cpu().double() - want).norm() <= tol


@pytest.mark.gpu
def test_recorded_many_steps(monkeypatch):
    """several rounds on narrow matrices in a graph, replayed between eager work"""
    import dpc_amd
    bind(monkeypatch, "compiled")
    prev = dpc_amd._dense_capi.set_library(None)
    try:
        gpu = torch.device("cuda")
        g = [of_rank(s, 3, i).to(gpu) for i, s in enumerate(NARROW)]
        w, m = [torch.zeros_like(t) for t in g], [torch.zeros_like(t) for t in g]
        moved, mom = [t.clone() for t in w], [t.clone() for t in m]
        run = lambda w, m: (dpc_amd.dense.newton_schulz(g, steps=20), dpc_amd.dense.muon_update(w, g, m, lr=0.1, steps=20))[0]
        want = run([t.clone() for t in w], [t.clone() for t in m])
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = run(w, m)
        for _ in range(3):
            graph.replay()
            dpc_amd.dense.newton_schulz(of_rank((60, 64), 0, 3).to(gpu), steps=12)
            torch.cuda.synchronize()
            run(moved, mom)
            assert all(torch.equal(a, b) for a, b in zip(got + w + m, want + moved + mom))
    finally:
        dpc_amd._dense_capi.set_library(prev)


@pytest.mark.gpu
@pytest.mark.parametrize("shape,steps", [((1 << 20, 1024), 5), ((64, 1 << 20), 12), ((1 << 20, 3), 5)], ids=["2^20x1024", "64x2^20", "2^20x3"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=IDS[:2])
def test_the_longest_sides(monkeypatch, shape, steps, dtype):
    """2^20, the longest side taken: lines of more than 2^32 bytes, sums of 2^20 terms"""
    import dpc_amd
    bind(monkeypatch, "compiled")
    prev = dpc_amd._dense_capi.set_library(None)
    try:
        g = torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").mul_(1e-3).to(dtype)
        coefficients = DEFAULT if steps == 5 else (2.0, -1.5, 0.5)
        o = dpc_amd.dense.newton_schulz(g, steps=steps, coefficients=coefficients)
        want = ref.newton_schulz(g, steps, coefficients)
        assert ref.off(o, want) <= ref.orthogonal_tolerance(torch.float32, steps) + ref.HALF_STEP[dtype]
    finally:
        dpc_amd._dense_capi.set_library(prev)
        torch.cuda.empty_cache()
