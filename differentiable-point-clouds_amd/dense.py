"""The dense layers around the projector: their product in 8 bits, and the orthogonalised update of their weights.

    y = linear_fp8(x, weight, bias)              # differentiable; weight a tensor, or packed once with pack_weight_fp8
    layer = Fp8Linear(1024, 24000)               # torch.nn.Linear whose products run in 8 bits
    o = newton_schulz(g)                         # a matrix, a batch of them or a list: (nearly) orthogonal factors
    muon_update(weights, grads, momenta, lr=...) # one optimiser step in place (optim.Muon calls it)

The reference leaves both to stock TensorFlow: fully connected layers (dpc/nets/img_encoder.py:11-50, pc_decoder.py:5-42) and
its optimiser (dpc/run/train.py:86-92).  Kernels: csrc/dense, C ABI: include/dpc_dense.h.  Calls only enqueue work on the current
stream of the tensors' device, allocate through torch, and can be recorded into a HIP graph."""
import collections
import contextlib
import ctypes
import math

import torch

from . import _dense_capi, _dense_ext, ops
from ._dense_capi import BLOCK, DpcDenseMatrix, DpcDenseSteps

_CODES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
COEFFICIENTS = (3.4445, -4.7750, 2.0315)


# ---------------------------------------------------------------------------
# helpers
# ---------------------------------------------------------------------------
def _library(*tensors):
    """the active library, after checking that every tensor (None aside) lies where it computes, on one device"""
    lib, device = _dense_capi.get_library(), None
    for t in tensors:
        if t is None:
            continue
        if not isinstance(t, torch.Tensor):
            raise TypeError("expected a torch.Tensor, got %r" % type(t))
        if t.layout != torch.strided:
            raise TypeError("expected a dense tensor, got layout %s" % t.layout)
        if lib.host_memory:
            if t.is_cuda:
                raise ValueError("emulation library needs host tensors")
        elif not t.is_cuda:
            raise ValueError("the dense operators need tensors on a ROCm device (no CPU fallback)")
        if device is not None and t.device != device:
            raise ValueError("tensors on different devices: %s and %s" % (device, t.device))
        device = t.device
    return lib


def _compiled():
    """(compiled binding, id of the active library in it), or (None, None): ctypes then drives the same library"""
    ext = _dense_ext.module()
    if ext is None:
        return None, None
    lib = _dense_capi.get_library()
    lib_id = lib.__dict__.get("_ext_id")
    if lib_id is None:
        lib_id = lib.__dict__["_ext_id"] = ext.open_library(lib.path, lib.host_memory)
    return ext, lib_id


def _raise_rc(e):
    """a status of the library that the compiled binding passed on: raise what the ctypes binding raises"""
    msg = str(e)
    if msg.startswith("DPC_RC:"):
        _, rc, what = msg.split("\n", 1)[0].split(":", 2)
        _dense_capi.DenseLibrary.check(int(rc), what.strip())


def _check_tensors(*ts):
    for t in ts:
        if not isinstance(t, torch.Tensor):
            raise TypeError("expected a torch.Tensor, got %r" % type(t))


def _check_no_tangent(*ts):
    """forward-mode derivatives are not computed here, and not dropped either"""
    for t in ts:
        if t is not None and torch.autograd.forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError("the dense operators carry no forward-mode derivatives: pass the primal, or detach")


def _code(t, what):
    if t.dtype not in _CODES:
        raise TypeError("%s must be float32, bfloat16 or float16, got %s" % (what, t.dtype))
    return _CODES[t.dtype]


_HERE = contextlib.nullcontext()


def _on(lib, device):
    """(context that makes `device` current, its current stream)"""
    if lib.host_memory:
        return _HERE, None
    guard = _HERE if device.index == torch.cuda.current_device() else torch.cuda.device(device)
    return guard, torch._C._cuda_getCurrentRawStream(device.index)


def _bytes(n, device):
    """n bytes, 256-byte aligned: (tensor that owns them, address)"""
    t = torch.empty(n + 256, dtype=torch.uint8, device=device)
    if ops._POISON:
        t.fill_(255)
    return t, (t.data_ptr() + 255) & ~255


def _buffer(shape, dtype, device):
    t = torch.empty(shape, dtype=dtype, device=device)
    if ops._POISON:
        t.view(torch.uint8).fill_(255)
    return t


def _rows(t):
    """t [rows, cols] with neighbouring columns and rows that do not overlap, its values as they lie in memory"""
    t = t.resolve_neg()
    if t.shape[1] > 1 and t.stride(1) != 1 or t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        return t.contiguous()
    return t


# ---------------------------------------------------------------------------
# the product
# ---------------------------------------------------------------------------
class Fp8Weight(collections.namedtuple("Fp8Weight", ["values", "scales", "in_features"])):
    """A weight [out_features, in_features] in 8 bits, laid out once for serving.

    values  float8_e4m3fn [out_features, 128 * blocks], blocks = ceil(in_features / 128); zeros behind in_features
    scales  uint8 [blocks, out_features]: the 128 values of a block stand for value * 2^(scale - 127)"""
    __slots__ = ()

    @property
    def out_features(self):
        return self.values.shape[0]


def _check_packed(w):
    blocks = -(-int(w.in_features) // BLOCK)
    if w.in_features < 0 or w.values.dim() != 2 or w.values.dtype != torch.float8_e4m3fn or w.values.shape[1] != blocks * BLOCK:
        raise ValueError("values must be float8_e4m3fn [out_features, %d], got %s %s" % (blocks * BLOCK, w.values.dtype, tuple(w.values.shape)))
    if w.scales.dtype != torch.uint8 or tuple(w.scales.shape) != (blocks, w.values.shape[0]):
        raise ValueError("scales must be uint8 [%d, %d], got %s %s" % (blocks, w.values.shape[0], w.scales.dtype, tuple(w.scales.shape)))
    if not (w.values.is_contiguous() and w.scales.is_contiguous()) or w.values.data_ptr() % 16 or w.values.is_neg() or w.scales.is_neg():
        raise ValueError("values and scales must be contiguous, values 16-byte aligned and no negative views")


_SIZES = {}


def _sizes(lib, m, k, n, x_type, w_type, needs):
    """bytes that a layer's passes need: (kept for the backward pass, forward workspace, backward workspace); by sizes alone"""
    key = (id(lib), m, k, n, x_type, w_type, needs)
    got = _SIZES.get(key)
    if got is None:
        out = (ctypes.c_size_t * 3)()
        lib.check(lib.dpc_dense_linear_sizes(m, k, n, x_type, w_type, needs, out), "dpc_dense_linear_sizes")
        if len(_SIZES) > 1024:
            _SIZES.clear()
        got = _SIZES[key] = tuple(out)
    return got


def _dims(*sizes):
    """sizes as the library's 32-bit numbers"""
    for n in sizes:
        if n > 0x7fffffff:
            raise ValueError("an axis of %d is too long" % n)
    return sizes


def _recording_stream(lib, device):
    """the current stream of the device if it records a graph, else None"""
    if lib.host_memory:
        return None
    with torch.cuda.device(device):
        return torch.cuda.current_stream().cuda_stream if torch.cuda.is_current_stream_capturing() else None


_MADE_ON, _ASKED = "dpc_amd.dense: recorded on", "dpc_amd.dense: asked for"


def _check_recording(lib, *tensors):
    """While a stream records a graph: a leaf whose earlier, eager autograd graph still lives would make the recorded backward pass wait for that
    graph's stream, which ends the process.  Refused here, where it can still be said.  That graph holds the leaf's accumulator: what is
    written into the accumulator's metadata is still there when it is asked for again.  One that lives is let pass if a call of this recording
    made it; returns the accumulators, which have to live until the leaves are used."""
    leaves = [t for t in tensors if t is not None and t.requires_grad and t.grad_fn is None]
    stream = _recording_stream(lib, leaves[0].device) if leaves and torch.is_grad_enabled() else None
    held = []
    for t in leaves if stream is not None else ():
        accumulator = lambda: torch.autograd.graph.get_gradient_edge(t).node
        if accumulator().metadata.get(_MADE_ON) != stream:
            accumulator().metadata[_ASKED] = True
            if _ASKED in accumulator().metadata:
                raise RuntimeError("linear_fp8 is being recorded into a graph while the autograd graph of an earlier eager call of the same leaf "
                                   "lives: drop what keeps it (an output, a loss) before the recording")
        held.append(accumulator())
        held[-1].metadata[_MADE_ON] = stream
    return held


def _ld(t):
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


class _LinearFp8(torch.autograd.Function):
    """y = Q(x) Q(w)^T + bias.  The gradients are those of the product of the held values, with dy held in 8 bits too, each in
    blocks along the axis that its product sums over: dx = Q(dy) Q(w^T)^T, dw = Q(dy^T) Q(x^T)^T, dbias = sum of dy's rows."""

    @staticmethod
    def forward(ctx, x, w, bias, lib):
        need = ctx.needs_input_grad
        needs = (1 if need[0] else 0) | (2 if need[1] else 0) | (4 if need[2] else 0)
        x, w = _rows(x), _rows(w)
        m, k, n = _dims(x.shape[0], x.shape[1], w.shape[0])
        x_type, w_type = _CODES[x.dtype], _CODES[w.dtype]
        saved_bytes, forward_bytes, _ = _sizes(lib, m, k, n, x_type, w_type, needs)
        out = _buffer((m, n), x.dtype, x.device)
        saved, saved_at = _bytes(saved_bytes, x.device)
        hold, ws = _bytes(forward_bytes, x.device)
        guard, stream = _on(lib, x.device)
        with guard:
            rc = lib.dpc_dense_linear_forward(stream, m, k, n, x.data_ptr(), _ld(x), x_type, w.data_ptr(), _ld(w), w_type, ops._ptr(bias),
                                              0 if bias is None else _CODES[bias.dtype], out.data_ptr(), needs, saved_at, saved_bytes, ws,
                                              forward_bytes)
        lib.check(rc, "dpc_dense_linear_forward")
        ctx.save_for_backward(saved)
        ctx.plan = (lib, m, k, n, x.dtype, w.dtype, None if bias is None else bias.dtype, needs, saved_at - saved.data_ptr())
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        lib, m, k, n, x_dtype, w_dtype, b_dtype, needs, offset = ctx.plan
        saved, = ctx.saved_tensors
        dy = _rows(dy)
        dev = dy.device
        x_type, w_type = _CODES[x_dtype], _CODES[w_dtype]
        saved_bytes, _, need = _sizes(lib, m, k, n, x_type, w_type, needs)
        dx = _buffer((m, k), x_dtype, dev) if needs & 1 else None
        dw = _buffer((n, k), w_dtype, dev) if needs & 2 else None
        db = _buffer((n,), b_dtype, dev) if needs & 4 else None
        saved_at = saved.data_ptr() + offset
        if saved_at % 256:                       # hooks on saved tensors may have brought it back at another address
            moved, saved_at = _bytes(saved_bytes, dev)
            moved[saved_at - moved.data_ptr():][:saved_bytes].copy_(saved[offset:offset + saved_bytes])
        hold, ws = _bytes(need, dev)
        guard, stream = _on(lib, dev)
        p = ops._ptr
        with guard:
            rc = lib.dpc_dense_linear_backward(stream, m, k, n, dy.data_ptr(), _ld(dy), x_type, w_type, _CODES[b_dtype] if needs & 4 else 0,
                                               saved_at, saved_bytes, p(dx), p(dw), p(db), ws, need)
        lib.check(rc, "dpc_dense_linear_backward")
        return dx, dw, db, None


def pack_weight_fp8(weight):
    """The 8-bit form of ``weight`` [out_features, in_features], to be kept for calls of ``linear_fp8``."""
    lib = _library(weight)
    _check_no_tangent(weight)
    _code(weight, "weight")
    if weight.dim() != 2:
        raise ValueError("weight must be [out_features, in_features], got %s" % (tuple(weight.shape),))
    w = _rows(weight.detach())
    n, k = _dims(*w.shape)
    blocks = -(-k // BLOCK)
    q, s = _buffer((n, blocks * BLOCK), torch.float8_e4m3fn, w.device), _buffer((blocks, n), torch.uint8, w.device)
    guard, stream = _on(lib, w.device)
    with guard:
        rc = lib.dpc_dense_quantize(stream, n, k, _CODES[w.dtype], w.data_ptr(), _ld(w), q.data_ptr(), s.data_ptr(), None, None, None)
    lib.check(rc, "dpc_dense_quantize")
    return Fp8Weight(q, s, k)


def linear_fp8(x, weight, bias=None):
    """x [..., in_features] times weight^T, both held in 8 bits (e4m3) with one power-of-two scale for each 128 neighbours along
    the summed axis; the result has x's type.  Sums are held in 32 bits; results of 16 bits take the 8-bit matrix instruction
    (whose sums are off by 1.4e-5 of the result), float32 results the half-precision one (1e-7).

    ``weight`` [out_features, in_features], float32, bfloat16 or float16 (not necessarily x's type): differentiable in x, weight
    and bias, once; the gradients' products run in 8 bits as well (forward-mode derivatives are refused, here and below).  ``weight`` an
    ``Fp8Weight``: serving; x must not require a gradient.  A value that is not finite makes NaN of every result that it enters.  float32 magnitudes are meant to lie within
    2^-100 .. 2^100.  No axis longer than 128 * 65535."""
    packed = isinstance(weight, Fp8Weight)
    ext, lib_id = _compiled()
    if ext is not None:
        _check_tensors(x, *((weight.values, weight.scales) if packed else (weight,)), *(() if bias is None else (bias,)))
        try:
            if packed:
                return ext.serve(x, weight.values, weight.scales, int(weight.in_features), bias, lib_id, bool(ops._POISON))
            return ext.linear(x, weight, bias, lib_id, bool(ops._POISON))
        except RuntimeError as e:
            _raise_rc(e)
            raise
    lib = _library(x, weight.values if packed else weight, weight.scales if packed else None, bias)
    _code(x, "x")
    if packed:
        _check_packed(weight)
        n, k = weight.out_features, int(weight.in_features)
    else:
        _code(weight, "weight")
        if weight.dim() != 2:
            raise ValueError("weight must be [out_features, in_features], got %s" % (tuple(weight.shape),))
        n, k = weight.shape
    if x.dim() < 1 or x.shape[-1] != k:
        raise ValueError("x must be [..., %d], got %s" % (k, tuple(x.shape)))
    if bias is not None:
        _code(bias, "bias")
        if tuple(bias.shape) != (n,):
            raise ValueError("bias must be [%d], got %s" % (n, tuple(bias.shape)))
    held = None if packed else _check_recording(lib, x, weight, bias)      # noqa: F841 (lives until the leaves are used)
    if bias is not None:
        bias = bias.resolve_neg().contiguous()
    lead = x.shape[:-1]
    rows = math.prod(lead)
    x2 = x if len(lead) == 1 else x.reshape(rows, k)
    if not packed:
        y = _LinearFp8.apply(x2, weight, bias, lib)
        return y if len(lead) == 1 else y.reshape(*lead, n)
    if torch.is_grad_enabled() and (x.requires_grad or bias is not None and bias.requires_grad):
        raise ValueError("a packed weight serves only: call under torch.no_grad(), or pass the weight itself")
    _check_no_tangent(x, bias)
    x2 = _rows(x2)
    _dims(rows, n, k)
    out = _buffer((rows, n), x.dtype, x.device)
    code = _CODES[x.dtype]
    need = lib.dpc_dense_linear_serve_workspace(rows, k, n, code)
    hold, ws = _bytes(need, x.device) if need else (None, None)
    guard, stream = _on(lib, x.device)
    with guard:
        rc = lib.dpc_dense_linear_serve(stream, rows, k, n, x2.data_ptr(), _ld(x2), code, weight.values.data_ptr(), weight.scales.data_ptr(),
                                        ops._ptr(bias), 0 if bias is None else _CODES[bias.dtype], out.data_ptr(), ws, need)
    lib.check(rc, "dpc_dense_linear_serve")
    return out if len(lead) == 1 else out.reshape(*lead, n)


class Fp8Linear(torch.nn.Linear):
    """torch.nn.Linear whose product and gradients run in 8 bits (``linear_fp8``); weights and optimiser state keep their type."""

    def forward(self, x):
        return linear_fp8(x, self.weight, self.bias)


# ---------------------------------------------------------------------------
# orthogonalisation and the update
# ---------------------------------------------------------------------------
def _coefficients_of(steps, coefficients, eps):
    """a, b, c of every step in one list, after the checks"""
    if isinstance(steps, bool) or not isinstance(steps, int) or not 1 <= steps <= _dense_capi.MAX_STEPS:
        raise ValueError("steps must be a whole number in 1 .. %d, got %r" % (_dense_capi.MAX_STEPS, steps))
    if not (eps > 0 and math.isfinite(eps)):
        raise ValueError("eps must be positive, got %r" % (eps,))
    coefficients = tuple(coefficients)
    if len(coefficients) == 3 and not any(hasattr(c, "__len__") for c in coefficients):
        coefficients = (coefficients,) * steps
    if len(coefficients) != steps or any(len(c) != 3 for c in coefficients):
        raise ValueError("coefficients must be (a, b, c), or one such triple for each of the %d steps" % steps)
    return [float(v) for abc in coefficients for v in abc]


def _steps_of(steps, coefficients, eps):
    flat = _coefficients_of(steps, coefficients, eps)
    s = DpcDenseSteps()
    s.steps, s.eps = steps, float(eps)
    for i, v in enumerate(flat):
        s.coefficients[i // 3][i % 3] = v
    return s


def _plan_orthogonal(lib, by_type, steps):
    """the library's calls for by_type: {dtype: [(grad, momentum | None, out, rows, cols, scale)]}, contiguous storage; everything that can be
    refused is refused here, before the first of them runs"""
    lib.check(lib.dpc_dense_orthogonal(None, 0, None, 0, ctypes.byref(steps), None, 0), "dpc_dense_orthogonal")      # (coefficients)
    calls = []
    for dtype, entries in by_type.items():
        for at in range(0, len(entries), _dense_capi.MAX_MATRICES):
            part = entries[at:at + _dense_capi.MAX_MATRICES]
            ms = (DpcDenseMatrix * len(part))()
            for m, (g, mom, out, rows, cols, scale) in zip(ms, part):
                m.grad, m.momentum, m.out, m.rows, m.cols, m.scale = g.data_ptr(), ops._ptr(mom), out.data_ptr(), rows, cols, scale
            need = lib.dpc_dense_orthogonal_workspace(len(part), ms, _CODES[dtype])
            lib.check(0 if need else -2, "dpc_dense_orthogonal")                    # (sides)
            calls.append((len(part), ms, _CODES[dtype], need))
    return calls


def _run_orthogonal(lib, device, calls, steps):
    """one workspace for all calls, which follow each other on the stream"""
    most = max(need for _, _, _, need in calls)
    hold, ws = _bytes(most, device)
    guard, stream = _on(lib, device)
    with guard:
        for count, ms, code, _ in calls:
            lib.check(lib.dpc_dense_orthogonal(stream, count, ms, code, ctypes.byref(steps), ws, most), "dpc_dense_orthogonal")


def newton_schulz(grads, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    """X0 = G / (|G| + eps) (Frobenius norm), then ``steps`` times X <- (a I + b A + c A^2) X with A = X X^T (X turned so that it
    is at least as wide as tall): with the default coefficients the singular values move to about 1.

    ``grads``: a tensor [..., rows, cols], or a list of matrices of any sizes; all of a list run in the same launches.  The result
    has the same form and type; no gradient flows.  The steps compute to single precision's accuracy whatever
    the type.  Sides up to 2^20, the shorter one up to 16384.  ``coefficients``: (a, b, c), or a triple for each step; refused where
    the scalar iteration leaves (-3.5, 3.5)."""
    single = isinstance(grads, torch.Tensor)
    mats = [grads] if single else list(grads)
    ext, lib_id = _compiled()
    if ext is not None:
        _check_tensors(*mats)
        flat = _coefficients_of(steps, coefficients, eps)
        try:
            outs = ext.newton_schulz(mats, steps, flat, eps, single, lib_id, bool(ops._POISON))
        except RuntimeError as e:
            _raise_rc(e)
            raise
        return outs[0] if single else outs
    lib = _library(*mats)
    _check_no_tangent(*mats)
    s = _steps_of(steps, coefficients, eps)
    for g in mats:
        _code(g, "a matrix")
        if g.dim() < 2 or not single and g.dim() != 2:
            raise ValueError("expected %s, got %s" % ("[..., rows, cols]" if single else "matrices", tuple(g.shape)))
    with torch.no_grad():
        sources = [g.detach().resolve_neg().contiguous() for g in mats]
        outs = [_buffer(g.shape, g.dtype, g.device) for g in sources]
        by_type = {}
        for g, o in zip(sources, outs):
            if not g.numel():
                continue
            rows, cols = _dims(*g.shape[-2:])
            for a, b in zip(g.reshape(-1, rows, cols).unbind(0), o.view(-1, rows, cols).unbind(0)):
                by_type.setdefault(g.dtype, []).append((a, None, b, rows, cols, 1.0))
        calls = _plan_orthogonal(lib, by_type, s)
        if calls:
            _run_orthogonal(lib, sources[0].device, calls, s)
    return outs[0] if single else outs


_ADJUST = {
    "rms": lambda r, c: 0.2 * math.sqrt(max(r, c)),
    "spectral": lambda r, c: math.sqrt(max(1.0, r / c)),
    "none": lambda r, c: 1.0,
}


_ADJUST_CODES = {"rms": 0, "spectral": 1, "none": 2}


def _span(t):
    return t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()


def _check_apart(written, read):
    """no two written tensors share memory, and no read one lies in a written one"""
    spans = sorted([_span(t) + (True,) for t in written if t.numel()] + [_span(t) + (False,) for t in read if t.numel()])
    end, end_written = 0, 0                   # how far the spans so far reach, and the written ones among them
    for lo, hi, w in spans:
        if lo < (end if w else end_written):
            raise ValueError("weights and momenta must not share memory with each other or with the gradients")
        end = max(end, hi)
        if w:
            end_written = max(end_written, hi)


def _matrix_format(t):
    """how a weight's storage is a matrix [shape[0], the rest]: torch.contiguous_format, torch.channels_last or None.  The order
    of the columns does not matter to the update, only that it is the same in weight, gradient and momentum."""
    if t.is_contiguous():
        return torch.contiguous_format
    if t.dim() == 4 and t.is_contiguous(memory_format=torch.channels_last):
        return torch.channels_last
    return None


def muon_update(weights, grads, momenta, *, lr, momentum=0.95, nesterov=True, weight_decay=0.0, steps=5, coefficients=COEFFICIENTS,
                eps=1e-7, adjust="rms"):
    """One optimiser step on lists of weights, in place, all matrices in the same launches:

        m <- momentum m + (1 - momentum) g;   u = (1 - momentum) g + momentum m  (nesterov), else m
        w <- (1 - lr weight_decay) w - lr s newton_schulz(u)

    with s = 0.2 sqrt(max(rows, cols)) (``adjust="rms"``: updates of the size that Adam's have), sqrt(max(1, rows / cols))
    ("spectral") or 1 ("none").  A weight of more than two dimensions counts as [shape[0], the rest].  float32, bfloat16 or float16,
    contiguous or channels_last; gradients of the weight's type and shape; momenta float32, laid out like their weights.  ``lr`` a
    number, or a one-element float32 tensor on the device that is read when the work runs (a recorded step follows it)."""
    weights, grads, momenta = list(weights), list(grads), list(momenta)
    if not len(weights) == len(grads) == len(momenta):
        raise ValueError("%d weights, %d gradients, %d momenta" % (len(weights), len(grads), len(momenta)))
    if adjust not in _ADJUST:
        raise ValueError("adjust must be one of %s, got %r" % (sorted(_ADJUST), adjust))
    lr_tensor = lr if isinstance(lr, torch.Tensor) else None
    momentum, weight_decay, eps = float(momentum), float(weight_decay), float(eps)
    if not 0.0 <= momentum < 1.0:
        raise ValueError("momentum must be in [0, 1), got %r" % (momentum,))
    if not (weight_decay >= 0.0 and math.isfinite(weight_decay)):
        raise ValueError("weight_decay must not be negative, got %r" % (weight_decay,))
    if lr_tensor is not None:
        if lr_tensor.numel() != 1 or lr_tensor.dtype != torch.float32:
            raise ValueError("lr must be a number or a one-element float32 tensor, got %s %s" % (lr.dtype, tuple(lr.shape)))
        if lr_tensor.is_neg():
            raise ValueError("lr is a negative view: what lies in its memory is read when the work runs")
        lr = 0.0
    lr = float(lr)
    if not (lr >= 0.0 and math.isfinite(lr)):
        raise ValueError("lr must not be negative, got %r" % (lr,))
    ext, lib_id = _compiled()
    if ext is not None:
        _check_tensors(*weights, *grads, *momenta)
        flat = _coefficients_of(steps, coefficients, eps)
        try:
            ext.muon_update(weights, grads, momenta, lr, lr_tensor, momentum, bool(nesterov), weight_decay, steps, flat, eps,
                            _ADJUST_CODES[adjust], lib_id, bool(ops._POISON))
        except RuntimeError as e:
            _raise_rc(e)
            raise
        return
    lib = _library(*weights, *grads, *momenta, lr_tensor)
    _check_no_tangent(*weights, *grads, *momenta, lr_tensor)
    s = _steps_of(steps, coefficients, eps)
    s.nesterov, s.momentum, s.weight_decay, s.lr = 1 if nesterov else 0, momentum, weight_decay, lr
    if lr_tensor is not None:
        s.lr_device = lr_tensor.data_ptr()
    by_type = {}
    with torch.no_grad():
        for i, (w, g, m) in enumerate(zip(weights, grads, momenta)):
            _code(w, "a weight")
            if w.dim() < 2:
                raise ValueError("weight %d has shape %s: only matrices can be orthogonalised" % (i, tuple(w.shape)))
            if g.dtype != w.dtype or g.shape != w.shape:
                raise ValueError("gradient %d is %s %s, its weight %s %s" % (i, g.dtype, tuple(g.shape), w.dtype, tuple(w.shape)))
            if m.dtype != torch.float32 or m.shape != w.shape:
                raise ValueError("momentum %d must be float32 %s, got %s %s" % (i, tuple(w.shape), m.dtype, tuple(m.shape)))
            form = _matrix_format(w)
            if form is None or not m.is_contiguous(memory_format=form):
                raise ValueError("weight %d and its momentum must be contiguous, or both channels_last" % i)
            if w.is_neg() or m.is_neg():
                raise ValueError("weight %d or its momentum is a negative view: nothing can be written through it" % i)
            if not w.numel():
                continue
            g = g.detach().resolve_neg()
            if not g.is_contiguous(memory_format=form):
                g = g.contiguous(memory_format=form)
            rows = w.shape[0]
            cols = w.numel() // rows
            _dims(rows, cols)
            by_type.setdefault(w.dtype, []).append((g, m, w, rows, cols, _ADJUST[adjust](rows, cols)))
        entries = [e for es in by_type.values() for e in es]
        _check_apart([e[2] for e in entries] + [e[1] for e in entries], [e[0] for e in entries] + ([lr_tensor] if lr_tensor is not None else []))
        calls = _plan_orthogonal(lib, by_type, s)
        if not calls:
            return
        torch.autograd.graph.increment_version([e[i] for e in entries for i in (1, 2)])   # autograd graphs that hold the old weights are told
        _run_orthogonal(lib, weights[0].device, calls, s)
