"""The operators of the networks' dense layers, as cases that can be timed and compared.

Three operators, each in a plain form (elementary torch operations in 32 bits) and as the framework offers it:

* ``product``: y = x w^T (+ bias) with both sides held in 8 bits (e4m3) and one power-of-two scale for each block of 128
  along the summed axis; a serving call with weights laid out before, or a training call with its three gradients;
* ``orthogonalise``: Newton-Schulz products, X <- (a I + b X X^T + c (X X^T)^2) X from X = G / (|G| + eps);
* ``update``: one step of the optimiser built on it: momentum, orthogonalisation, decayed weights.
"""
import math

import torch

own = False

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
STEPS = 5
EPS = 1e-7
BLOCK = 128
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}

# the weights of the training example's networks at 128 x 128 images: convolution filters as [out, in * height * width], the
# encoder's dense layers, four pose branches and the student's, the layer that makes 8000 points
POSE = "32x1024,32x32,4x32," * 5
NETWORKS = ("16x75,32x144,32x288,64x288,64x576,128x576,128x1152,256x1152,256x2304,1024x4096,1024x1024,1024x1024,1024x1024,"
            + POSE + "24000x1024")


def listed():
    return [
        # one image's latent vector to 8000 points, weights packed when the program started: latency and one read of the weights
        {"name": "product: one view", "op": "product", "way": "serve", "m": 1, "k": 1024, "n": 24000, "type": "bf16", "bias": False},
        # the encoder's first dense layer in a training step of 16 models x 5 views, in single precision
        {"name": "product: views of a step", "op": "product", "way": "train", "m": 80, "k": 4096, "n": 1024, "type": "fp32", "bias": True},
        # nothing a multiple of a block or of a tile: a last batch, a layer of no round size
        {"name": "product: odd sizes", "op": "product", "way": "train", "m": 333, "k": 1000, "n": 777, "type": "bf16", "bias": True},
        # a training step with many views at once: bound by the matrix instructions
        {"name": "product: many views", "op": "product", "way": "train", "m": 8192, "k": 4096, "n": 4096, "type": "bf16", "bias": False},
        # one layer of a pose branch: the smallest call
        {"name": "orthogonalise: pose layer", "op": "orthogonalise", "shapes": "32x1024", "type": "fp32"},
        # the three square layers of the encoder, in 16 bits
        {"name": "orthogonalise: square", "op": "orthogonalise", "shapes": "1024x1024,1024x1024,1024x1024", "type": "bf16"},
        # a row, a tall one, near-square and ragged ones together
        {"name": "orthogonalise: odd sizes", "op": "orthogonalise", "shapes": "75x16,288x65,1x513,700x701", "type": "fp32"},
        # the layer that makes the points: tall and by far the largest
        {"name": "orthogonalise: points layer", "op": "orthogonalise", "shapes": "24000x1024", "type": "fp32"},
        # the optimiser's step over the pose network alone: fifteen small matrices, latency
        {"name": "update: pose network", "op": "update", "shapes": POSE.rstrip(","), "type": "fp32", "decay": 0.0, "nesterov": True},
        # ... over every matrix of the networks: what a training step waits for
        {"name": "update: all networks", "op": "update", "shapes": NETWORKS, "type": "fp32", "decay": 0.0, "nesterov": True},
        # ragged sizes, weights in 16 bits, decayed
        {"name": "update: odd sizes", "op": "update", "shapes": "333x1000,65x130,7x2049", "type": "bf16", "decay": 0.1, "nesterov": False},
        # two wide square layers in 16 bits: bound by the matrix instructions
        {"name": "update: wide layers", "op": "update", "shapes": "4096x4096,4096x4096", "type": "bf16", "decay": 0.01, "nesterov": True},
    ]


def _size(rng, low, high):
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if v > 64 and rng.random() < 0.5:
        v = max(low, v // 64 * 64)
    return min(high, max(low, v))


def draw(rng):
    kind = rng.choice(["product", "product", "orthogonalise", "update"])
    if kind == "product":
        while True:
            m, k, n = _size(rng, 1, 8192), _size(rng, 1, 8192), _size(rng, 1, 24000)
            if m * k * n <= 1 << 36 and k * n <= 1 << 26 and m * n <= 1 << 27:
                break
        way = "serve" if m <= 16 or rng.random() < 0.3 else "train"
        return {"op": kind, "way": way, "m": m, "k": k, "n": n, "type": rng.choice(["fp32", "bf16"]), "bias": rng.random() < 0.5}
    shapes, work = [], 0
    for _ in range(rng.choice([1, 1, 2, 4, 9])):
        while True:
            r, c = _size(rng, 1, 4096), _size(rng, 1, 24000)
            cost = min(r, c) ** 2 * max(r, c)
            if cost + work <= 1 << 34:
                break
        work += cost
        shapes.append("%dx%d" % ((r, c) if rng.random() < 0.5 else (c, r)))
    case = {"op": kind, "shapes": ",".join(shapes), "type": rng.choice(["fp32", "bf16"])}
    if kind == "update":
        case.update(decay=rng.choice([0.0, 0.01, 0.1]), nesterov=rng.random() < 0.7)
    return case


def _shapes(case):
    return [tuple(int(v) for v in s.split("x")) for s in case["shapes"].split(",")]


# ---- inputs ------------------------------------------------------------------------------------------------------------
def _blocks_of(x):
    """the last axis in blocks of 128 (zeros behind its end): [rows, blocks, 128]"""
    x = torch.nn.functional.pad(x.float(), (0, -x.shape[-1] % BLOCK))
    return x.reshape(x.shape[0], -1, BLOCK)


def _held(x):
    """rows of x in 8 bits: (e4m3 values [rows, blocks, 128], exponents [rows, blocks]), x ~ value * 2^exponent.  The
    exponent is the smallest for which a block's largest magnitude stays within e4m3's 448 = 0.875 * 2^9."""
    b = _blocks_of(x)
    top = b.abs().amax(dim=-1)
    mantissa, exponent = torch.frexp(top)
    exponent = torch.where(mantissa > 0.875, exponent - 8, exponent - 9).clamp(-126, 127)
    exponent = torch.where(top == 0, torch.full_like(exponent, -126), exponent)
    return (b / _power(exponent)[..., None]).to(torch.float8_e4m3fn), exponent


def _power(exponent):
    """2^exponent, exactly, in single precision (exponents of normal numbers)"""
    return ((exponent.int() + 127) << 23).view(torch.float32)


def _gradient(shape, g, device):
    """what a layer's gradient looks like: columns of unequal size and a few strong common directions"""
    r, c = shape
    x = torch.randn(r, c, generator=g, device=device) * torch.exp(0.5 * torch.randn(1, c, generator=g, device=device))
    common = torch.randn(r, 4, generator=g, device=device) @ torch.randn(4, c, generator=g, device=device)
    return 1e-3 * (x + common)


def prepare(case, seed):
    device = torch.device("cuda", 0)
    g = torch.Generator(device=device).manual_seed(seed)
    dtype = TYPES[case["type"]]
    if case["op"] == "product":
        m, k, n = case["m"], case["k"], case["n"]
        x = torch.nn.functional.leaky_relu(torch.randn(m, k, generator=g, device=device), 0.2).to(dtype)
        w = (torch.randn(n, k, generator=g, device=device) / math.sqrt(k)).to(dtype)
        bias = (0.1 * torch.randn(n, generator=g, device=device)).to(dtype) if case["bias"] else None
        if case["way"] == "serve":
            q, e = _held(w)                              # the layout that a serving program keeps: rows of values, padded to
            return dict(case=case, x=x, bias=bias, values=q.reshape(n, -1),          # whole blocks, and [blocks, rows] exponents
                        scales=(e + 127).to(torch.uint8).t().contiguous())
        dy = 1e-3 * torch.randn(m, n, generator=g, device=device) * torch.exp(torch.randn(m, 1, generator=g, device=device))
        return dict(case=case, x=x.requires_grad_(), w=w.requires_grad_(),
                    bias=None if bias is None else bias.requires_grad_(), dy=dy.to(dtype))
    grads = [_gradient(s, g, device).to(dtype) for s in _shapes(case)]
    if case["op"] == "orthogonalise":
        return dict(case=case, grads=grads)
    weights = [(torch.randn(s, generator=g, device=device) / math.sqrt(s[1])).to(dtype) for s in _shapes(case)]
    return dict(case=case, grads=grads, weights=weights, momenta=[_gradient(s, g, device) for s in _shapes(case)])


# ---- plain forms -------------------------------------------------------------------------------------------------------
def _values(x):
    """what the 8-bit form of x's rows stands for, in single precision, cut back to x's own length"""
    q, e = _held(x)
    return (q.float() * _power(e)[..., None]).reshape(x.shape[0], -1)[:, :x.shape[1]]


def _serve(state):
    x, k = state["x"], state["case"]["k"]
    w = state["values"].float().reshape(state["values"].shape[0], -1, BLOCK)
    w = (w * _power(state["scales"].t().int() - 127)[..., None]).flatten(1)[:, :k]
    y = _values(x) @ w.t()
    return (y if state["bias"] is None else y + state["bias"].float()).to(x.dtype)


def _train(state):
    x, w, bias, dy = (None if v is None else v.detach() for v in (state["x"], state["w"], state["bias"], state["dy"]))
    y = _values(x) @ _values(w).t()
    y = y if bias is None else y + bias.float()
    dx = _values(dy) @ _values(w.t()).t()
    dw = _values(dy.t()) @ _values(x.t()).t()
    db = None if bias is None else dy.float().sum(0).to(bias.dtype)
    return [v for v in (y.to(x.dtype), dx.to(x.dtype), dw.to(w.dtype), db) if v is not None]


def _orthogonal(u):
    x = u.float()
    x = x.t() if x.shape[0] > x.shape[1] else x
    x = x / (x.norm() + EPS)
    a, b, c = COEFFICIENTS
    for _ in range(STEPS):
        s = x @ x.t()
        x = a * x + (b * s + c * (s @ s)) @ x
    return x.t() if u.shape[0] > u.shape[1] else x


LR, MOMENTUM = 0.02, 0.95


def _update(case, w, g, m):
    g = g.float()
    m.mul_(MOMENTUM).add_((1 - MOMENTUM) * g)
    u = (1 - MOMENTUM) * g + MOMENTUM * m if case["nesterov"] else m
    size = 0.2 * math.sqrt(max(w.shape))
    w.copy_((1 - LR * case["decay"]) * w.float() - LR * size * _orthogonal(u))


def run(state):
    case = state["case"]
    if own:
        import dpc_amd
        if case["op"] == "product" and case["way"] == "serve":
            packed = dpc_amd.dense.Fp8Weight(state["values"], state["scales"], case["k"])
            return dpc_amd.dense.linear_fp8(state["x"], packed, state["bias"])
        if case["op"] == "product":
            y = dpc_amd.dense.linear_fp8(state["x"], state["w"], state["bias"])
            leaves = [state[v] for v in ("x", "w", "bias") if state[v] is not None]
            return [y.detach()] + list(torch.autograd.grad(y, leaves, state["dy"]))
        if case["op"] == "orthogonalise":
            return dpc_amd.dense.newton_schulz(state["grads"], steps=STEPS, coefficients=COEFFICIENTS, eps=EPS)
        dpc_amd.dense.muon_update(state["weights"], state["grads"], state["momenta"], lr=LR, momentum=MOMENTUM,
                                  nesterov=case["nesterov"], weight_decay=case["decay"], steps=STEPS,
                                  coefficients=COEFFICIENTS, eps=EPS)
    elif case["op"] == "product":
        return _serve(state) if case["way"] == "serve" else _train(state)
    elif case["op"] == "orthogonalise":
        return [_orthogonal(u).to(u.dtype) for u in state["grads"]]
    else:
        for w, g, m in zip(state["weights"], state["grads"], state["momenta"]):
            _update(case, w, g, m)
    return {"weights": state["weights"], "momenta": state["momenta"]}


# ---- what one pass cannot do without -----------------------------------------------------------------------------------
def work(case):
    e = 4 if case["type"] == "fp32" else 2
    if case["op"] == "product":
        m, k, n = case["m"], case["k"], case["n"]
        bias = n * e if case["bias"] else 0
        if case["way"] == "serve":
            return {"bytes": m * k * e + n * k * (1 + 1 / BLOCK) + bias + m * n * e, "flops": 2 * m * k * n}
        return {"bytes": 2 * (m * k + n * k + m * n) * e + 2 * bias, "flops": 6 * m * k * n}
    flops = nbytes = 0
    for shape in _shapes(case):
        r, c = min(shape), max(shape)
        # X X^T and its square are symmetric: half of each is enough
        flops += STEPS * (r * r * c + r ** 3 + 2 * r * r * c)
        nbytes += r * c * (2 * e if case["op"] == "orthogonalise" else 3 * e + 8)
    return {"bytes": nbytes, "flops": flops}


# ---- the definition in 64 bits, written apart from the plain form ------------------------------------------------------
def _exact_power(v):
    """2^floor(log2 v) of positive normal numbers in 64 bits: the number without its fraction's bits"""
    return ((v.contiguous().view(torch.int64) >> 52) << 52).view(torch.float64)


def _exact_held(x):
    x = x.detach().double()
    out = torch.empty_like(x)
    for at in range(0, x.shape[1], BLOCK):
        part = x[:, at:at + BLOCK]
        top = part.abs().max(dim=1, keepdim=True).values / 448.0
        scale = _exact_power(top.clamp(min=2.0 ** -126))
        scale = torch.where(scale < top, 2 * scale, scale)
        v = part / scale
        grid = _exact_power(v.abs().clamp(min=2.0 ** -6)) / 8                             # e4m3: three bits behind the point
        out[:, at:at + BLOCK] = torch.round(v / grid) * grid * scale
    return out


def _exact_orthogonal(u):
    u = u.double()
    tall = u.shape[0] > u.shape[1]
    x = u / (torch.sqrt((u * u).sum()) + EPS)
    a, b, c = COEFFICIENTS
    for _ in range(STEPS):
        s = x.t() @ x if tall else x @ x.t()
        p = a * torch.eye(s.shape[0], dtype=s.dtype, device=s.device) + b * s + c * torch.matmul(s, s)
        x = x @ p if tall else p @ x
    return x


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "product":
        bias = 0.0 if s["bias"] is None else s["bias"].detach().double()
        x = _exact_held(s["x"])
        if case["way"] == "serve":
            e = torch.repeat_interleave(s["scales"].double() - 127, BLOCK, dim=0).t()
            return x @ (s["values"].double() * torch.exp2(e))[:, :case["k"]].t() + bias
        dy = s["dy"].double()
        out = [x @ _exact_held(s["w"]).t() + bias, _exact_held(dy) @ _exact_held(s["w"].detach().t()).t(),
               _exact_held(dy.t()) @ _exact_held(s["x"].detach().t()).t()]
        return out + ([] if s["bias"] is None else [dy.sum(0)])
    if case["op"] == "orthogonalise":
        return [_exact_orthogonal(u) for u in s["grads"]]
    weights, momenta = [], []
    for w, g, m in zip(s["weights"], s["grads"], s["momenta"]):
        w, g, m = w.double(), g.double(), m.double()
        m = MOMENTUM * m + (1 - MOMENTUM) * g
        u = MOMENTUM * m + (1 - MOMENTUM) * g if case["nesterov"] else m
        weights.append(w - LR * (case["decay"] * w + 0.2 * max(w.shape) ** 0.5 * _exact_orthogonal(u)))
        momenta.append(m)
    return {"weights": weights, "momenta": momenta}
