"""The dense layers' operators (dpc_amd.dense, dpc_amd.optim) against their definitions in 64 bits: on the CPU through the emulation of
the kernels (small sizes, every refusal), and on the GPU (-m gpu)."""
import os

import pytest
import torch

import dense_reference as ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["fp32", "bf16", "fp16"]


@pytest.fixture(scope="session")
def dense_emulation():
    import subprocess
    emu_dir = os.path.join(ROOT, "tests", "hipemu")
    subprocess.check_call(["make", "-s", "-C", emu_dir, "-f", "Makefile.dense"])
    import dpc_amd
    return dpc_amd._dense_capi.DenseLibrary(os.path.join(emu_dir, "libdpc_dense_emu.so"), host_memory=True)


def bind(monkeypatch, binding):
    """through the compiled binding (which has to be there: the build makes it) or through ctypes"""
    from importlib import import_module
    ext = import_module("differentiable-point-clouds_amd._dense_ext")
    if binding == "ctypes":
        monkeypatch.setattr(ext, "module", lambda: None)
    else:
        assert ext.module() is not None, "the compiled binding is not built: python __graft_entry__.py"


@pytest.fixture(params=["emulation-compiled", "emulation-ctypes", pytest.param("gpu-compiled", marks=pytest.mark.gpu),
                        pytest.param("gpu-ctypes", marks=pytest.mark.gpu)])
def device(request, monkeypatch):
    """where the operators run: "cpu" through the emulated kernels, or the GPU; through either binding"""
    import dpc_amd
    where, binding = request.param.split("-")
    bind(monkeypatch, binding)
    lib = request.getfixturevalue("dense_emulation") if where == "emulation" else None
    prev = dpc_amd._dense_capi.set_library(lib)
    yield torch.device("cpu" if lib is not None else "cuda")
    dpc_amd._dense_capi.set_library(prev)


@pytest.fixture()
def gpu():
    import dpc_amd
    prev = dpc_amd._dense_capi.set_library(None)
    yield torch.device("cuda")
    dpc_amd._dense_capi.set_library(prev)


@pytest.fixture(params=["compiled", "ctypes"])
def emulated(dense_emulation, request, monkeypatch):
    import dpc_amd
    bind(monkeypatch, request.param)
    prev = dpc_amd._dense_capi.set_library(dense_emulation)
    yield dpc_amd
    dpc_amd._dense_capi.set_library(prev)


def draw(shape, seed, dtype, device, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (scale * torch.randn(shape, generator=g)).to(dtype).to(device)


def check_product(x, w, bias, y):
    """y against Q(x) Q(w)^T + bias, every entry"""
    a, b = ref.held(x.cpu()), ref.held(w.cpu())
    want = a @ b.t() + (0 if bias is None else bias.detach().cpu().double())
    assert y.dtype == x.dtype and tuple(y.shape) == (x.shape[0], w.shape[0])
    worst = ((y.detach().cpu().double() - want).abs() / ref.product_tolerance(a, b, want, x.dtype)).max()
    assert worst <= 1, float(worst)


# ---- the product -----------------------------------------------------------------------------------------------------------
SIZES = [(1, 1, 1), (1, 128, 5), (3, 129, 17), (16, 256, 64), (17, 100, 130), (65, 640, 33), (129, 300, 131)]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("m,k,n", SIZES)
def test_product_forward(device, m, k, n, dtype):
    import dpc_amd
    x, w = draw((m, k), 1, dtype, device), draw((n, k), 2, dtype, device)
    bias = draw((n,), 3, dtype, device) if n % 2 else None
    check_product(x, w, bias, dpc_amd.dense.linear_fp8(x, w, bias))
    packed = dpc_amd.dense.pack_weight_fp8(w)
    check_product(x, w, bias, dpc_amd.dense.linear_fp8(x, packed, bias))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("m,k,n", [(1, 1024, 24000), (5, 8200, 70), (16, 4096, 1024), (64, 1000, 999), (80, 4096, 1024), (333, 1000, 777),
                                   (2000, 129, 1025), (513, 2048, 4096), (1, 20000, 3), (4100, 300, 8)])
def test_product_forward_larger(gpu, m, k, n, dtype):
    import dpc_amd
    x, w = draw((m, k), 1, dtype, gpu), draw((n, k), 2, dtype, gpu, k ** -0.5)
    bias = draw((n,), 3, torch.float32, gpu)
    check_product(x, w, bias, dpc_amd.dense.linear_fp8(x, dpc_amd.dense.pack_weight_fp8(w), bias))


def gradients(dpc_amd, x, w, bias, dy):
    leaves = [t.detach().requires_grad_() for t in (x, w)] + ([] if bias is None else [bias.detach().requires_grad_()])
    y = dpc_amd.dense.linear_fp8(leaves[0], leaves[1], leaves[2] if bias is not None else None)
    return [y.detach()] + list(torch.autograd.grad(y, leaves, dy))


@pytest.mark.parametrize("x_type,w_type", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32),
                                           (torch.float16, torch.float32)], ids=["fp32", "bf16", "bf16-fp32", "fp16-fp32"])
@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (2, 130, 3), (130, 70, 129), pytest.param(333, 1000, 777, marks=pytest.mark.gpu),
                                   pytest.param(80, 4096, 1024, marks=pytest.mark.gpu)])
def test_product_gradients_are_the_formulas(device, m, k, n, x_type, w_type):
    if device.type != "cuda" and m * k * n > 1 << 22:
        pytest.skip("sizes for the GPU")
    import dpc_amd
    x, w, bias = draw((m, k), 1, x_type, device), draw((n, k), 2, w_type, device), draw((n,), 3, w_type, device)
    dy = draw((m, n), 4, x_type, device, 1e-3)
    y, dx, dw, db = gradients(dpc_amd, x, w, bias, dy)
    h = lambda t: ref.held(t.cpu())
    check_product(x, w, bias, y)
    for got, a, b, dtype in ((dx, h(dy), h(w.t()), x_type), (dw, h(dy.t()), h(x.t()), w_type)):
        want = a @ b.t()
        assert got.dtype == dtype
        assert bool(((got.cpu().double() - want).abs() <= ref.product_tolerance(a, b, want, dtype)).all())
    want = dy.cpu().double().sum(0)
    tol = ref.HALF_STEP[w_type] * want.abs() + (m + 8) * 2.0 ** -24 * dy.cpu().double().abs().sum(0)
    assert db.dtype == w_type and bool(((db.cpu().double() - want).abs() <= tol).all())


def test_product_gradients_against_differences(device):
    """small whole numbers are held exactly, so y is linear in them and differences over whole steps are the derivatives"""
    import dpc_amd
    g = torch.Generator().manual_seed(0)
    whole = lambda *s: torch.randint(-7, 8, s, generator=g).float()
    x, w, bias, dy = whole(5, 140), whole(6, 140), whole(6), whole(5, 6)
    _, dx, dw, db = gradients(dpc_amd, x.to(device), w.to(device), bias.to(device), dy.to(device))
    f = lambda x, w, bias: float((dpc_amd.dense.linear_fp8(x.to(device), w.to(device), bias.to(device)).cpu().double() * dy).sum())
    for t, d, at in ((x, dx, (0, 0)), (x, dx, (4, 139)), (x, dx, (2, 127)), (w, dw, (5, 128)), (w, dw, (0, 1)), (bias, db, (3,))):
        up, down = t.clone(), t.clone()
        up[at] += 1
        down[at] -= 1
        args = [up if s is t else s for s in (x, w, bias)], [down if s is t else s for s in (x, w, bias)]
        assert (f(*args[0]) - f(*args[1])) / 2 == float(d[at])


def test_product_only_asks_for_the_gradients_needed(device):
    import dpc_amd
    x, w, bias = draw((4, 30), 1, torch.float32, device), draw((7, 30), 2, torch.float32, device), draw((7,), 3, torch.float32, device)
    full = gradients(dpc_amd, x, w, bias, torch.ones(4, 7, device=device))[1:]
    for need in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 1, 1), (1, 0, 1)):
        leaves = [t.detach().requires_grad_(bool(n)) for t, n in zip((x, w, bias), need)]
        dpc_amd.dense.linear_fp8(*leaves).sum().backward()               # an expanded gradient of ones
        for t, n, want in zip(leaves, need, full):
            assert (t.grad is not None) == bool(n) and (not n or torch.equal(t.grad, want))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_product_strides_and_leading_axes(device, dtype):
    import dpc_amd
    x, w = draw((6, 5, 40), 1, dtype, device), draw((9, 40), 2, dtype, device)
    y = dpc_amd.dense.linear_fp8(x, w)
    assert tuple(y.shape) == (6, 5, 9)
    flat = dpc_amd.dense.linear_fp8(x.reshape(30, 40).contiguous(), w)
    assert torch.equal(y.reshape(30, 9), flat)
    wide = draw((30, 83), 3, dtype, device)                               # rows of a wider matrix, from an odd column on
    assert torch.equal(dpc_amd.dense.linear_fp8(wide[:, 3:43], w), dpc_amd.dense.linear_fp8(wide[:, 3:43].contiguous(), w))
    turned = draw((40, 30), 4, dtype, device).t()
    wt = draw((40, 9), 5, dtype, device).t()
    assert torch.equal(dpc_amd.dense.linear_fp8(turned, wt), dpc_amd.dense.linear_fp8(turned.contiguous(), wt.contiguous()))
    one = draw((1, 40), 6, dtype, device).expand(30, 40)
    assert torch.equal(dpc_amd.dense.linear_fp8(one, w), dpc_amd.dense.linear_fp8(one.contiguous(), w))


def test_product_of_empty_sizes(device):
    import dpc_amd
    for m, k, n in ((0, 5, 3), (2, 0, 3), (2, 5, 0), (0, 0, 0)):
        x, w, b = torch.ones(m, k, device=device), torch.ones(n, k, device=device), torch.arange(n, device=device).float()
        for t in (x, w, b):
            t.requires_grad_()
        y = dpc_amd.dense.linear_fp8(x, w, b)
        assert torch.equal(y.detach(), (x @ w.t() + b).detach())
        got = torch.autograd.grad(y, (x, w, b), torch.ones_like(y))
        assert [tuple(t.shape) for t in got] == [(m, k), (n, k), (n,)]
        assert torch.equal(got[2], torch.full((n,), float(m), device=device))
        assert not got[0].any() and not got[1].any()
        with torch.no_grad():
            assert torch.equal(dpc_amd.dense.linear_fp8(x, dpc_amd.dense.pack_weight_fp8(w), b), y)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_product_of_values_at_the_ends(device, dtype):
    """zero blocks, the largest e4m3 number and what rounds to it, subnormal quotients, far magnitudes, and what is not finite"""
    import dpc_amd
    x = torch.zeros(7, 260)
    x[1, :] = 448.0
    x[2, 0], x[2, 1] = 448.0, 449.0                       # the second needs the next scale
    x[3, :128], x[3, 128:] = 1e-3, 1e3
    x[4, ::2] = 2.0 ** -13                                 # beside 1.0: far below e4m3's normal numbers
    x[4, 1] = 1.0
    x[5, 7], x[6, 200] = float("nan"), float("-inf")
    x[5, 8] = x[6, 0] = 1.0
    big = 2.0 ** 90 if dtype != torch.float16 else 1024.0
    x, w = x.to(dtype).to(device), torch.eye(260).to(dtype).to(device)
    w[3] = w[3] * big
    w[4] = w[4] / big
    y = dpc_amd.dense.linear_fp8(x, w)
    a, b = ref.held(x.cpu()), ref.held(w.cpu())
    want = a @ b.t()                                       # a NaN in a row of x spoils that row
    y = y.cpu().double()
    assert bool(torch.isnan(y[5:]).all()) and not bool(torch.isnan(y[:5]).any())
    over = want.abs() > torch.finfo(dtype).max             # 448 * 1024 is past fp16's 65504: infinite in that type
    assert torch.equal(torch.isinf(y[:5]), over[:5])
    want[over], y[over] = 0.0, 0.0
    assert bool(((y[:5] - want[:5]).abs() <= ref.product_tolerance(a[:5], b, want[:5], dtype)).all())
    assert bool((y[0] == 0).all()) and y[1, 0] == 448.0


def test_packed_weight_is_the_documented_layout(device):
    import dpc_amd
    w = draw((5, 200), 1, torch.float32, device)
    p = dpc_amd.dense.pack_weight_fp8(w)
    assert p.values.dtype == torch.float8_e4m3fn and tuple(p.values.shape) == (5, 256) and tuple(p.scales.shape) == (2, 5)
    assert p.out_features == 5 and p.in_features == 200
    e = torch.repeat_interleave(p.scales.cpu().t().double() - 127, 128, dim=1)
    assert torch.equal((p.values.cpu().double() * torch.exp2(e))[:, :200], ref.held(w.cpu()))
    assert not p.values.cpu().float()[:, 200:].any()


def test_fp8_linear_module(device):
    import dpc_amd
    torch.manual_seed(0)
    layer = dpc_amd.dense.Fp8Linear(40, 9).to(device)
    x = draw((6, 40), 1, torch.float32, device)
    y = layer(x)
    assert torch.equal(y, dpc_amd.dense.linear_fp8(x, layer.weight, layer.bias))
    y.sum().backward()
    assert layer.weight.grad.shape == layer.weight.shape and layer.bias.grad.shape == layer.bias.shape
    assert sorted(layer.state_dict()) == ["bias", "weight"]


@pytest.mark.gpu
def test_product_of_more_than_32_bits_of_results(gpu):
    import dpc_amd
    x, w = draw((70000, 200), 1, torch.bfloat16, gpu), draw((70000, 200), 2, torch.bfloat16, gpu)
    y = dpc_amd.dense.linear_fp8(x, w)
    assert y.numel() > 2 ** 32
    for rows in (slice(0, 2), slice(61355, 61358), slice(69998, 70000)):
        check_product(x[rows], w, None, y[rows])


@pytest.mark.parametrize("offset", [0, 16, 144])
def test_product_kept_forms_may_be_moved(device, offset):
    """hooks on saved tensors (offloading) bring back what the forward pass kept at another address"""
    import dpc_amd
    x, w, dy = draw((130, 200), 1, torch.float32, device), draw((70, 200), 2, torch.float32, device), draw((130, 70), 3, torch.float32, device)
    want = gradients(dpc_amd, x, w, None, dy)

    def move(t):
        there = torch.empty(t.numel() + 256, dtype=t.dtype, device=t.device)[offset:offset + t.numel()]
        return there.copy_(t)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: move(t.to(device))):
        got = gradients(dpc_amd, x, w, None, dy)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_product_refusals(emulated):
    d = emulated.dense
    x, w = torch.ones(2, 8), torch.ones(3, 8)
    p = d.pack_weight_fp8(w)
    for bad in (lambda: d.linear_fp8(x, w.double()), lambda: d.linear_fp8(x.int(), w), lambda: d.linear_fp8([1.0], w),
                lambda: d.linear_fp8(x, w, torch.ones(3).double()), lambda: d.linear_fp8(x.to_sparse(), w)):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: d.linear_fp8(x, torch.ones(3, 9)), lambda: d.linear_fp8(x, torch.ones(8)), lambda: d.linear_fp8(torch.tensor(1.0), w),
                lambda: d.linear_fp8(x, w, torch.ones(2)), lambda: d.pack_weight_fp8(torch.ones(3)),
                lambda: d.linear_fp8(x, p._replace(in_features=200)), lambda: d.linear_fp8(x, p._replace(scales=p.scales.t())),
                lambda: d.linear_fp8(x, p._replace(values=p.values.float())), lambda: d.linear_fp8(x, p._replace(in_features=-1)),
                lambda: d.linear_fp8(x.clone().requires_grad_(), p), lambda: d.linear_fp8(x, p, torch.ones(3, requires_grad=True))):
        with pytest.raises(ValueError):
            bad()
    with torch.no_grad():
        d.linear_fp8(x.clone().requires_grad_(), p)
    leaf = x.clone().requires_grad_()
    dx, = torch.autograd.grad(d.linear_fp8(leaf, w.clone().requires_grad_()).square().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()                                # once differentiable


# ---- orthogonalisation --------------------------------------------------------------------------------------------------------
SHAPES = [(1, 1), (1, 7), (9, 1), (4, 32), (33, 31), (75, 16), (20, 200), (66, 130), (140, 131)]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_newton_schulz(device, dtype):
    import dpc_amd
    mats = [ref.gradient(s, i, dtype, 0.1).to(device) for i, s in enumerate(SHAPES)]
    for g, o in zip(mats, dpc_amd.dense.newton_schulz(mats)):
        assert o.dtype == dtype and o.shape == g.shape
        assert ref.off(o.cpu(), ref.newton_schulz(g.cpu())) <= ref.orthogonal_tolerance(dtype), tuple(g.shape)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("shapes", [[(1024, 1024)], [(24000, 64), (3, 9000)], [(700, 701), (288, 65), (1, 513)], [(128, 5000), (130, 129), (4, 4)],
                                    [(2050, 515)], [(i + 1, 3 * i + 2) for i in range(95)]])
def test_newton_schulz_larger(gpu, shapes, dtype):
    import dpc_amd
    mats = [ref.gradient(s, i, dtype, 0.1).to(gpu) for i, s in enumerate(shapes)]
    for g, o in zip(mats, dpc_amd.dense.newton_schulz(mats)):
        assert ref.off(o.cpu(), ref.newton_schulz(g).cpu()) <= ref.orthogonal_tolerance(dtype), tuple(g.shape)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_small_matrices_beside_larger_ones(device, dtype):
    """a few strong directions leave little of the other singular values: sides of at most 32 are as exact beside a larger matrix as alone,
    that is 64-bit steps, 32-bit sums over at most 32 products and the result's rounding (half a step of every value)"""
    import dpc_amd
    gen = torch.Generator().manual_seed(7)
    mats = []
    for r, c in ((8, 2500), (400, 3), (24, 96), (66, 70)):
        x = torch.randn(r, c, generator=gen) * torch.exp(0.5 * torch.randn(1, c, generator=gen))
        mats.append((1e-3 * (x + torch.randn(r, 4, generator=gen) @ torch.randn(4, c, generator=gen))).to(dtype).to(device))
    for g, o in list(zip(mats, dpc_amd.dense.newton_schulz(mats)))[:3]:
        # a product's terms are at most 32 times the result's size (P to 3.5^5 / |U| against singular values of X that they raise): 2^-24 each
        assert ref.off(o.cpu(), ref.newton_schulz(g.cpu())) <= ref.HALF_STEP[dtype] + 32 * 32 * 2.0 ** -24, tuple(g.shape)


@pytest.mark.parametrize("steps", [1, 2, 3, 4, 6])
def test_newton_schulz_steps_and_coefficients(device, steps):
    import dpc_amd
    mats = [ref.gradient(s, 3, torch.float32).to(device) for s in ((40, 70), (70, 66))]
    triples = [(3.4445, -4.7750, 2.0315), (2.0, -1.5, 0.5), (1.5, -0.5, 0.0), (1.875, -1.25, 0.375), (2.0, -1.5, 0.5), (1.0, 0.0, 0.0)][:steps]
    for g, o, p in zip(mats, dpc_amd.dense.newton_schulz(mats, steps=steps), dpc_amd.dense.newton_schulz(mats, steps=steps, coefficients=triples)):
        assert ref.off(o.cpu(), ref.newton_schulz(g.cpu(), steps)) <= ref.orthogonal_tolerance(torch.float32, steps)
        assert ref.off(p.cpu(), ref.newton_schulz(g.cpu(), steps, triples)) <= ref.orthogonal_tolerance(torch.float32, steps)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_newton_schulz_batches_strides_and_ends(device, dtype):
    import dpc_amd
    ns = dpc_amd.dense.newton_schulz
    batch = torch.stack([ref.gradient((20, 33), i, dtype, 0.1) for i in range(3)]).to(device)
    out = ns(batch)
    assert out.shape == batch.shape
    for i in range(3):
        assert torch.equal(out[i], ns(batch[i]))
    turned = batch[0].t()
    assert torch.equal(ns(turned), ns(turned.contiguous()))
    assert torch.equal(ns(batch[:, 3:19, 5:]), ns(batch[:, 3:19, 5:].contiguous()))
    assert ns(batch[:0]).shape == (0, 20, 33) and ns([]) == [] and ns(batch[:, :0]).shape == (3, 0, 33)
    zero = torch.zeros(70, 80, dtype=dtype, device=device)
    small = torch.zeros(3, 5, dtype=dtype, device=device)
    for z in (zero, small):
        assert torch.equal(ns(z), z)                        # |G| = 0: 0 / eps
        for v in (float("nan"), float("inf")):
            bad = torch.ones_like(z)
            bad[2, 3] = v
            good = ref.gradient((20, 20), 0, dtype).to(device)
            a, b = ns([bad, good])
            assert bool(torch.isnan(a).all()) and torch.equal(b, ns(good))     # its neighbours in the list are not touched
    same = ns([batch[0], batch[0]])
    assert torch.equal(same[0], same[1])
    keep = batch.clone()
    ns(batch)
    assert torch.equal(batch, keep)


@pytest.mark.parametrize("size", [1e-18, 1e-30, 1e25])
def test_newton_schulz_of_far_magnitudes(device, size):
    """the norm's squares neither vanish nor overflow"""
    import dpc_amd
    for shape in ((40, 70), (70, 90)):
        g = ref.gradient(shape, 1, torch.float32, 1.0).to(device) * size
        got = dpc_amd.dense.newton_schulz(g, eps=1e-38)
        assert ref.off(got.cpu(), ref.newton_schulz(g.cpu(), eps=1e-38)) <= ref.orthogonal_tolerance(torch.float32)


def test_newton_schulz_refusals(emulated):
    ns = emulated.dense.newton_schulz
    g = torch.ones(3, 4)
    for bad in (lambda: ns(g.double()), lambda: ns([g, 1.0]), lambda: ns(g.to_sparse())):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: ns(torch.ones(3)), lambda: ns([torch.ones(2, 3, 4)]), lambda: ns(g, steps=0), lambda: ns(g, steps=65), lambda: ns(g, steps=2.5),
                lambda: ns(g, steps=True), lambda: ns(g, eps=0.0), lambda: ns(g, eps=-1.0), lambda: ns(g, eps=float("nan")),
                lambda: ns(g, coefficients=(1.0, 2.0)), lambda: ns(g, coefficients=[(1.0, 0.0, 0.0)] * 4),
                lambda: ns(g, coefficients=(4.0, 0.0, 0.0)), lambda: ns(g, coefficients=(float("nan"), 0.0, 0.0)),
                lambda: ns([], coefficients=(4.0, 0.0, 0.0)), lambda: ns(g, coefficients=(3.0, -3.2, 30.0))):
        with pytest.raises(ValueError):
            bad()


# ---- the update -----------------------------------------------------------------------------------------------------------------
def run_update(dpc_amd, shapes, dtype, device, calls=1, **kw):
    """(weights, momenta) after `calls` updates, with what they should be and may be off by, checked"""
    w = [draw(s, i, dtype, device, 0.05) for i, s in enumerate(shapes)]
    m = [0.1 * ref.gradient(s, 50 + i).to(device) for i, s in enumerate(shapes)]
    lr, mu, wd = kw.get("lr", 0.02), kw.get("momentum", 0.95), kw.get("weight_decay", 0.0)
    lr = float(lr)
    for call in range(calls):
        g = [ref.gradient(s, 100 + i + call, dtype).to(device) for i, s in enumerate(shapes)]
        before = [(a.cpu().double(), b.cpu().double()) for a, b in zip(w, m)]
        dpc_amd.dense.muon_update(w, g, m, **kw)
        for i, s in enumerate(shapes):
            w0, m0 = before[i]
            gi = g[i].cpu().double()
            m1 = mu * m0 + (1 - mu) * gi
            assert bool(((m[i].cpu().double() - m1).abs() <= 5 * 2.0 ** -24 * ((mu * m0).abs() + ((1 - mu) * gi).abs()) + 1e-44).all())
            u = (1 - mu) * gi + mu * m1 if kw.get("nesterov", True) else m1
            size = {"rms": 0.2 * max(s) ** 0.5, "spectral": max(1.0, s[0] / s[1]) ** 0.5, "none": 1.0}[kw.get("adjust", "rms")]
            o = ref.newton_schulz(u)
            want = (1 - lr * wd) * w0 - lr * size * o
            err = (w[i].cpu().double() - want).norm()
            tol = (ref.HALF_STEP[dtype] + 2 * 2.0 ** -24) * want.norm() + lr * size * o.norm() * (ref.orthogonal_tolerance(dtype) - ref.HALF_STEP[dtype] + 2.0 ** -23)
            assert err <= tol, (s, float(err), float(tol))
    return w, m


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("kw", [dict(), dict(nesterov=False, weight_decay=0.1), dict(momentum=0.0, adjust="spectral"), dict(adjust="none", lr=0.5)],
                         ids=["plain", "decayed", "no-momentum", "unscaled"])
def test_muon_update(device, dtype, kw):
    import dpc_amd
    run_update(dpc_amd, [(20, 33), (70, 66), (1, 5), (40, 3)], dtype, device, calls=2, **{"lr": 0.02, **kw})


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_muon_update_larger(gpu, dtype):
    import dpc_amd
    run_update(dpc_amd, [(333, 1000), (65, 130), (7, 2049), (1024, 1024), (2400, 256), (256, 1152)], dtype, gpu, calls=2, lr=0.02, weight_decay=0.1)


def test_muon_update_reads_the_rate_from_the_device(device):
    import dpc_amd
    lr = torch.tensor([0.03], device=device)
    a = run_update(dpc_amd, [(20, 33), (70, 66)], torch.float32, device, lr=lr, weight_decay=0.01)
    b = run_update(dpc_amd, [(20, 33), (70, 66)], torch.float32, device, lr=0.03, weight_decay=0.01)
    for x, y in zip(a[0] + a[1], b[0] + b[1]):
        assert torch.allclose(x, y, rtol=2.0 ** -22, atol=0)


def test_muon_update_of_filters_in_both_layouts(device):
    """a channels_last filter is the same matrix with its columns in another order"""
    import dpc_amd
    w = draw((8, 5, 3, 3), 1, torch.float32, device)
    g, m = draw((8, 5, 3, 3), 2, torch.float32, device), torch.zeros(8, 5, 3, 3, device=device)
    flat = [t.reshape(8, 45).clone() for t in (w, g, m)]
    dpc_amd.dense.muon_update([flat[0]], [flat[1]], [flat[2]], lr=0.1)
    last = [t.clone(memory_format=torch.channels_last) for t in (w, g, m)]
    dpc_amd.dense.muon_update([last[0]], [g], [last[2]], lr=0.1)          # the gradient in the other layout
    dpc_amd.dense.muon_update([w], [last[1]], [m], lr=0.1)
    assert last[0].is_contiguous(memory_format=torch.channels_last)
    for got in (w.reshape(8, 45), last[0].contiguous().reshape(8, 45)):
        assert ref.off(got, flat[0]) <= 2 * ref.orthogonal_tolerance(torch.float32)


def test_muon_update_is_seen_by_autograd(device):
    """a graph that holds the weights as they were refuses its backward pass after the update, as after any change in place"""
    import dpc_amd
    w = draw((8, 12), 1, torch.float32, device).requires_grad_()
    x = draw((3, 12), 2, torch.float32, device).requires_grad_()
    y = x @ w.t()
    dpc_amd.dense.muon_update([w], [torch.ones_like(w)], [torch.zeros(8, 12, device=device)], lr=0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    (x @ w.t()).sum().backward()


def test_muon_update_refusals(emulated):
    up = emulated.dense.muon_update
    w, g, m = torch.ones(3, 4), torch.ones(3, 4), torch.zeros(3, 4)
    buf = torch.zeros(24)
    bad_type = [([w.double()], [g.double()], [m], {}), ([w], [g], [m.tolist()], {})]
    for a, b, c, kw in bad_type:
        with pytest.raises(TypeError):
            up(a, b, c, lr=0.1, **kw)
    bad = [([w], [g, g], [m], {}), ([w], [g.bfloat16()], [m], {}), ([w], [g[:2]], [m], {}), ([w], [g], [m.bfloat16()], {}), ([w], [g], [m[:2]], {}),
           ([torch.ones(4)], [torch.ones(4)], [torch.zeros(4)], {}), ([w.t()], [g.t()], [m.t()], {}), ([w], [g], [torch.zeros(4, 3).t()], {}),
           ([w, w], [g, g], [m, m.clone()], {}), ([w, w.clone()], [g, g], [m, m], {}), ([w], [w], [m], {}), ([w], [m], [m], {}),
           ([buf[:12].view(3, 4)], [g], [buf[6:18].view(3, 4)], {}), ([buf[:12].view(3, 4)], [buf[11:23].view(3, 4)], [m], {}),
           ([w], [g], [m], dict(momentum=1.0)), ([w], [g], [m], dict(momentum=-0.1)), ([w], [g], [m], dict(weight_decay=-1.0)),
           ([w], [g], [m], dict(adjust="other")), ([w], [g], [m], dict(steps=0)), ([w], [g], [m], dict(coefficients=(5.0, 0.0, 0.0)))]
    for a, b, c, kw in bad:
        with pytest.raises(ValueError):
            up(a, b, c, lr=0.1, **kw)
    for lr in (-1.0, float("nan"), torch.zeros(2), torch.zeros(1, dtype=torch.float64)):
        with pytest.raises(ValueError):
            up([w], [g], [m], lr=lr)
    assert torch.equal(w, torch.ones(3, 4)) and torch.equal(m, torch.zeros(3, 4))
    up([], [], [], lr=0.1)
    up([torch.ones(0, 4)], [torch.ones(0, 4)], [torch.ones(0, 4)], lr=0.1)
    up([w, w.clone()], [g, g], [m, m.clone()], lr=0.1)                     # one gradient for two weights is only read
    assert torch.equal(w, w.clone())


def test_refusals_by_the_library_itself(dense_emulation):
    """what the C entry points refuse before anything is launched"""
    import ctypes
    from importlib import import_module
    capi = import_module("differentiable-point-clouds_amd._dense_capi")
    lib = dense_emulation
    buf = (ctypes.c_char * 65536)()
    a = (ctypes.addressof(buf) + 255) & ~255
    assert lib.dpc_dense_quantize(None, 1, 4, 9, a, 4, a, a, None, None, None) == -3
    assert lib.dpc_dense_quantize(None, -1, 4, 0, a, 4, a, a, None, None, None) == -2
    assert lib.dpc_dense_quantize(None, 2, 4, 0, a, 3, a, a, None, None, None) == -2
    assert lib.dpc_dense_quantize(None, 1, 4, 0, a, 4, a, None, None, None, None) == -1
    assert lib.dpc_dense_quantize(None, 1, 4, 0, a, 4, None, None, None, None, None) == -1
    assert lib.dpc_dense_quantize(None, 1, 4, 0, a, 4, a, a, None, None, a) == -1
    assert lib.dpc_dense_quantize(None, 1, 4, 0, a, 4, a + 1, a, None, None, None) == -4
    for far in (0x7fffffff, 0x7fffffff - 128):
        assert lib.dpc_dense_quantize(None, 1, far, 0, a, far, a, a, None, None, None) == -2
        assert lib.dpc_dense_quantize(None, far, 1, 0, a, 1, None, None, a, a, None) == -2
        assert lib.dpc_dense_colsum(None, 1, far, a, 0, a) == -2
        assert lib.dpc_dense_product(None, far, 1, 1, a, a, a, a, None, 0, a, 0, None, 0) == -2
        assert lib.dpc_dense_product(None, 1, far, 1, a, a, a, a, None, 0, a, 0, None, 0) == -2
    assert lib.dpc_dense_product(None, 1, 1, 65536, a, a, a, a, None, 0, a, 0, None, 0) == -2
    assert lib.dpc_dense_linear_serve(None, 1, 128 * 65535 + 1, 1, a, 1 << 30, 0, a, a, None, 0, a, None, 0) == -2
    assert lib.dpc_dense_colsum(None, 1, 4, None, 0, a) == -1
    assert lib.dpc_dense_product(None, 1, 1, 1, a, a, a, a, None, 0, None, 0, None, 0) == -1
    assert lib.dpc_dense_product(None, 1, 1, 1, a, a, a, a, a, 7, a, 0, None, 0) == -3
    assert lib.dpc_dense_product(None, 1, -1, 1, a, a, a, a, None, 0, a, 0, None, 0) == -2
    assert lib.dpc_dense_product(None, 1, 1, 1, a + 1, a, a, a, None, 0, a, 0, None, 0) == -4
    need = lib.dpc_dense_product_workspace(64, 64, 64, 0)
    assert need > 0
    assert lib.dpc_dense_product(None, 64, 64, 64, a, a, a, a, None, 0, a, 0, a, need - 1) == -4
    s = capi.DpcDenseSteps()
    s.steps, s.eps = 1, 1e-7
    s.coefficients[0][0] = 1.0
    m = (capi.DpcDenseMatrix * 1)()
    m[0].grad, m[0].out, m[0].rows, m[0].cols = a, a, 2, 2
    need = lib.dpc_dense_orthogonal_workspace(1, m, 0)
    assert need > 0
    go = lambda count=1, dtype=0, ws=a, size=need: lib.dpc_dense_orthogonal(None, count, m, dtype, ctypes.byref(s), ws, size)
    assert go(ws=None) == -4 and go(size=need - 1) == -4 and go(ws=a + 1) == -4 and go(dtype=5) == -3 and go(count=-1) == -2
    assert go(count=capi.MAX_MATRICES + 1) == -2
    m[0].rows = 0
    assert go() == -2
    m[0].rows, m[0].cols = 20000, 20000
    assert go() == -2
    m[0].rows, m[0].cols, m[0].grad = 2, 2, None
    assert go() == -1
    m[0].grad, s.eps = a, 0.0
    assert go() == -5


# ---- the optimiser, and a run of the operators together ------------------------------------------------------------------------------
def toy(dpc_amd, device, dtype=torch.float32):
    torch.manual_seed(0)
    return torch.nn.Sequential(dpc_amd.dense.Fp8Linear(24, 70), torch.nn.LeakyReLU(0.2), dpc_amd.dense.Fp8Linear(70, 10)).to(device, dtype)


@pytest.mark.parametrize("dtype", TYPES[:2], ids=IDS[:2])
def test_muon_steps_a_network_of_8_bit_layers(device, dtype):
    """forward, backward and step together equal the operators called one by one"""
    import dpc_amd
    net, twin = toy(dpc_amd, device, dtype), toy(dpc_amd, device, dtype)
    opt = dpc_amd.optim.muon_with_adam(net, lr=0.02, adam_lr=1e-3, weight_decay=0.01)
    adam = torch.optim.Adam([p for p in twin.parameters() if p.dim() < 2], lr=1e-3)
    mats = [p for p in twin.parameters() if p.dim() >= 2]
    mom = [torch.zeros_like(p, dtype=torch.float32) for p in mats]
    for i in range(3):
        x = draw((5, 24), i, dtype, device)
        opt.zero_grad()
        net(x).float().square().sum().backward()
        opt.step()
        twin.zero_grad()
        twin(x).float().square().sum().backward()
        dpc_amd.dense.muon_update(mats, [p.grad for p in mats], mom, lr=0.02, weight_decay=0.01)
        adam.step()
    for p, q in zip(net.parameters(), twin.parameters()):
        assert torch.equal(p, q)
    assert opt.optimizers[0].state[net[0].weight]["momentum_buffer"].dtype == torch.float32


def test_muon_state_and_groups(device):
    import copy
    import dpc_amd
    net = toy(dpc_amd, device, torch.bfloat16)
    opt = dpc_amd.optim.muon_with_adam(net)
    assert len(opt.param_groups) == 2 and opt.param_groups[0]["lr"] == 0.02
    net(draw((5, 24), 0, torch.bfloat16, device)).float().square().sum().backward()
    opt.step()
    saved = copy.deepcopy(opt.state_dict())
    other = dpc_amd.optim.muon_with_adam(net)
    other.load_state_dict(saved)
    for p in net.parameters():
        if p.dim() >= 2:
            a, b = (o.optimizers[0].state[p]["momentum_buffer"] for o in (opt, other))
            assert b.dtype == torch.float32 and torch.equal(a, b)          # all bits of the momenta
    with pytest.raises(ValueError):
        dpc_amd.optim.Together(*opt.optimizers, *opt.optimizers).load_state_dict(saved)
    with pytest.raises(ValueError):
        dpc_amd.optim.Muon(net.parameters())                               # biases are no matrices
    muon = dpc_amd.optim.Muon([net[0].weight])
    net[0].weight.grad = None
    before = net[0].weight.detach().clone()
    muon.step()                                                            # no gradient: nothing to do
    assert torch.equal(before, net[0].weight) and not muon.state
    assert float(muon.step(lambda: torch.ones(()))) == 1.0


def test_muon_beside_gradient_buckets(device):
    """the buckets' views are gradients at odd addresses"""
    import dpc_amd
    finals = []
    for gather in (None, "accumulate", "copy"):
        net = toy(dpc_amd, device)
        opt = dpc_amd.optim.muon_with_adam(net)
        red = dpc_amd.distributed.GradBuckets(net.parameters(), bucket_mb=0.001, gather=gather) if gather else None
        for i in range(2):
            if red is None:
                opt.zero_grad()
            net(draw((5, 24), i, torch.float32, device)).square().sum().backward()
            if red is not None:
                red.finish()
            opt.step()
            if red is not None:
                red.zero_()
        finals.append([p.detach().clone() for p in net.parameters()])
    for a in finals[1:]:
        for p, q in zip(finals[0], a):
            assert torch.equal(p, q)


@pytest.mark.gpu
def test_recorded_steps_equal_eager_ones(gpu):
    """the whole step in a graph (forward and backward in 8 bits, Muon with its rate on the gpu), replayed between eager work, twice:
    two recordings live at once"""
    import dpc_amd
    runs = []
    for recorded in (False, True):
        nets = [toy(dpc_amd, gpu) for _ in range(2)]
        lrs = [torch.full((1,), 0.02, device=gpu) for _ in nets]
        x = draw((5, 24), 1, torch.float32, gpu)
        steps = []
        for net, lr in zip(nets, lrs):
            opt = dpc_amd.optim.Muon([net[0].weight, net[2].weight], lr=lr)

            def step(net=net, opt=opt):
                opt.zero_grad()
                loss = net(x).square().sum()
                loss.backward()
                opt.step()
                return loss.detach()
            if recorded:
                steps.append(dpc_amd.graphs.RecordedStep(step, device=gpu, warmup=3))
            else:
                for _ in range(3):
                    step()
                steps.append(step)
        losses = []
        for i in range(4):
            for j, s in enumerate(steps):
                lrs[j].fill_(0.02 / (1 + i + j))
                losses.append(s().clone())
                dpc_amd.dense.newton_schulz(draw((40, 70), i, torch.float32, gpu))     # eager work between replays
                torch.cuda.synchronize()
        runs.append((losses, [p.detach().clone() for net in nets for p in net.parameters()]))
    for a, b in zip(runs[0][0] + runs[0][1], runs[1][0] + runs[1][1]):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_recording_beside_a_living_eager_graph_is_refused(gpu):
    """the recorded backward pass would wait for the eager graph's stream; refused before anything is enqueued, and fine once it is gone"""
    import dpc_amd
    x, w, dy = (draw(s, i, torch.float32, gpu) for i, s in enumerate(((5, 24), (70, 24), (5, 70))))
    w.requires_grad_()
    eager = dpc_amd.dense.linear_fp8(x, w)
    want, = torch.autograd.grad(eager, w, dy, retain_graph=True)
    torch.cuda.synchronize()
    refused = torch.cuda.CUDAGraph()
    with torch.cuda.graph(refused):
        with pytest.raises(RuntimeError, match="earlier eager call of the same leaf"):
            dpc_amd.dense.linear_fp8(x, w)
        with torch.no_grad():
            z = dpc_amd.dense.linear_fp8(x, w)               # nothing to differentiate, nothing to refuse
    refused.replay()
    assert torch.equal(z, eager)
    del eager
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = dpc_amd.dense.linear_fp8(x, w)
        y2 = dpc_amd.dense.linear_fp8(x, w)                  # the leaf's graph now lives, but it is the recorded one
        got, = torch.autograd.grad(y + 0 * y2, w, dy)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


@pytest.mark.gpu
def test_other_streams_and_two_calls_at_once(gpu):
    import dpc_amd
    g = [ref.gradient((300, 500), i).to(gpu) for i in range(2)]
    x, w = draw((70, 500), 1, torch.bfloat16, gpu), draw((900, 500), 2, torch.bfloat16, gpu)
    want = [dpc_amd.dense.newton_schulz(t) for t in g], dpc_amd.dense.linear_fp8(x, w)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(5):
        got = []
        for s, t in zip(streams, g):
            with torch.cuda.stream(s):
                got.append(dpc_amd.dense.newton_schulz(t))
        with torch.cuda.stream(streams[2]):
            y = dpc_amd.dense.linear_fp8(x, w)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want[0])) and torch.equal(y, want[1])
    # a backward pass runs on its forward pass' stream, behind what that stream still has to do
    xf, wf, dy = draw((300, 2000), 3, torch.float32, gpu), draw((700, 2000), 4, torch.float32, gpu), draw((300, 700), 5, torch.float32, gpu)
    want = gradients(dpc_amd, xf, wf, None, dy)
    late, big = torch.zeros_like(xf), torch.randn(4096, 4096, device=gpu)
    torch.cuda.synchronize()
    with torch.cuda.stream(streams[0]):
        for _ in range(20):
            big = big @ big * 1e-3
        late.copy_(xf)
        got = gradients(dpc_amd, late, wf, None, dy)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_same_results_every_time(gpu):
    import dpc_amd
    x, w, b, dy = (draw(s, i, torch.float32, gpu) for i, s in enumerate(((80, 4096), (1024, 4096), (1024,), (80, 1024))))
    g = ref.gradient((2000, 300), 1).to(gpu)
    first = gradients(dpc_amd, x, w, b, dy) + [dpc_amd.dense.newton_schulz(g)]
    for _ in range(3):
        assert all(torch.equal(p, q) for p, q in zip(first, gradients(dpc_amd, x, w, b, dy) + [dpc_amd.dense.newton_schulz(g)]))


# ---- the training example with both --------------------------------------------------------------------------------------------------
def example():
    import sys
    here = os.path.join(ROOT, "examples", "chair_unsupervised")
    if here not in sys.path:
        sys.path.insert(0, here)
    import nets
    import train_step
    return nets, train_step


def check_points_layer(dpc_amd, nets, ts, device, cfg, image_size, net_kw, graph=False):
    """steps of the example with 8-bit layers and Muon: everything stays finite and moves, and the points layer's gradient is its
    formula's"""
    torch.manual_seed(0)
    net = nets.Im2PointCloud(cfg, image_size=image_size, dense="fp8", **net_kw).to(device)
    torch.manual_seed(0)
    stock = nets.Im2PointCloud(cfg, image_size=image_size, **net_kw)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(net.state_dict().values(), stock.state_dict().values()))
    seen = {}

    def watch(module, args, y):
        seen["x"] = args[0].detach()
        y.register_hook(lambda g: seen.update(dy=g.detach()))

    net.decoder.pts.register_forward_hook(watch)
    proj = dpc_amd.model_pc.ModelPointCloud(cfg, global_step=0, device=device)
    opt = ts.make_optimizer(net, "muon", recorded=graph, fused=device.type == "cuda")
    g = torch.Generator().manual_seed(5)
    n = cfg.batch_size * cfg.step_size
    inputs = {"images": torch.rand(n, image_size, image_size, 3, generator=g).to(device),
              "masks": (torch.rand(n, image_size, image_size, 1, generator=g) > 0.5).float().to(device)}
    before = {k: v.detach().clone() for k, v in net.named_parameters()}
    for _ in range(2):
        loss = ts.train_step(net, proj, inputs, opt, is_training=False)
        assert bool(torch.isfinite(loss))
    a, b = ref.held(seen["dy"].cpu().t()), ref.held(seen["x"].cpu().t())
    want = a @ b.t()
    got = net.decoder.pts.weight.grad.cpu().double()
    assert bool(((got - want).abs() <= ref.product_tolerance(a, b, want, torch.float32)).all()) and float(want.abs().max()) > 0
    for k, v in net.named_parameters():
        assert bool(torch.isfinite(v).all()), k
        if k.startswith(("decoder.pts", "encoder.fc")):
            assert not torch.equal(v, before[k]), k


def test_training_example_in_8_bits_with_muon(emu, emulated):
    nets, ts = example()
    cfg = ts.make_cfg(vox_size=16, pc_gauss_kernel_size=5, pc_num_points=64, pose_predict_num_candidates=2, step_size=2, batch_size=2,
                      pc_point_dropout=1.0)
    check_points_layer(emulated, nets, ts, torch.device("cpu"), cfg, 32, dict(f_dim=4, fc_dim=32, z_dim=32))
    with pytest.raises(ValueError):
        nets.Im2PointCloud(cfg, 32, f_dim=4, fc_dim=32, z_dim=32, dense="int4")
    with pytest.raises(ValueError):
        ts.make_optimizer(torch.nn.Linear(2, 2), "sgd")


@pytest.mark.gpu
def test_training_example_in_8_bits_with_muon_on_the_gpu(gpu):
    import dpc_amd
    nets, ts = example()
    cfg = ts.make_cfg(batch_size=2, pc_point_dropout=1.0, pc_num_points=2000)
    check_points_layer(dpc_amd, nets, ts, gpu, cfg, 64, {})


@pytest.mark.gpu
def test_recorded_training_example_with_muon(gpu):
    """the example's step in one graph: every replay moves the weights, and they stay finite"""
    import dpc_amd
    nets, ts = example()
    cfg = ts.make_cfg(batch_size=1, step_size=2, pc_point_dropout=1.0, pc_num_points=500, vox_size=32, pc_gauss_kernel_size=11)
    torch.manual_seed(0)
    net = nets.Im2PointCloud(cfg, image_size=32, f_dim=4, fc_dim=64, z_dim=64, dense="fp8").to(gpu)
    proj = dpc_amd.model_pc.ModelPointCloud(cfg, global_step=0, device=gpu)
    opt = ts.make_optimizer(net, "muon", recorded=True)
    inputs = ts.synthetic_batch(cfg, gpu, 32, seed=1)
    proj.enable_graph_replay()
    step = dpc_amd.graphs.RecordedStep(lambda: ts.train_step(net, proj, inputs, opt), device=gpu, warmup=3)
    last = net.decoder.pts.weight.detach().clone()
    for _ in range(3):
        assert bool(torch.isfinite(step()))
        torch.cuda.synchronize()
        now = net.decoder.pts.weight.detach().clone()
        assert bool(torch.isfinite(now).all()) and not torch.equal(now, last)
        last = now
