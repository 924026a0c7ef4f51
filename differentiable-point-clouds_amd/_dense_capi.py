"""ctypes binding of the C ABI in include/dpc_dense.h (the dense layers' operators).

Like ``_capi``: the product path loads exactly one library, ``csrc/dense/libdpc_dense.so`` (hipcc, gfx950), and fails loudly
if it is missing; there is no CPU fallback.  The test-suite can install the CPU emulation build of the same kernel source."""
import ctypes
import os

from ._capi import DpcError

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "csrc", "dense", "libdpc_dense.so")

BLOCK = 128
MAX_MATRICES = 40
MAX_STEPS = 64

_ERRORS = {
    -1: "DPC_DENSE_E_NULL (required pointer is null)",
    -2: "DPC_DENSE_E_SHAPE (negative or unsupported sizes)",
    -3: "DPC_DENSE_E_TYPE (unknown element type)",
    -4: "DPC_DENSE_E_WORKSPACE (workspace too small or misaligned)",
    -5: "DPC_DENSE_E_VALUE (coefficients or steps outside what can be held)",
}


class DpcDenseMatrix(ctypes.Structure):
    _fields_ = [("grad", ctypes.c_void_p), ("momentum", ctypes.c_void_p), ("out", ctypes.c_void_p), ("rows", ctypes.c_int32),
                ("cols", ctypes.c_int32), ("scale", ctypes.c_float), ("reserved", ctypes.c_int32)]


class DpcDenseSteps(ctypes.Structure):
    _fields_ = [("steps", ctypes.c_int32), ("nesterov", ctypes.c_int32), ("momentum", ctypes.c_double), ("lr", ctypes.c_double),
                ("weight_decay", ctypes.c_double), ("eps", ctypes.c_double), ("lr_device", ctypes.c_void_p),
                ("coefficients", (ctypes.c_float * 3) * MAX_STEPS)]


_P, _I, _Z = ctypes.c_void_p, ctypes.c_int, ctypes.c_size_t
_MP, _TP = ctypes.POINTER(DpcDenseMatrix), ctypes.POINTER(DpcDenseSteps)

# name -> (restype, argtypes); mirrors include/dpc_dense.h one to one
SIGNATURES = {
    "dpc_dense_version": (ctypes.c_char_p, []),
    "dpc_dense_abi_struct_bytes": (_Z, [_I]),
    "dpc_dense_quantize": (_I, [_P, _I, _I, _I, _P, _Z, _P, _P, _P, _P, _P]),
    "dpc_dense_colsum": (_I, [_P, _I, _I, _P, _I, _P]),
    "dpc_dense_product_workspace": (_Z, [_I, _I, _I, _I]),
    "dpc_dense_product": (_I, [_P, _I, _I, _I, _P, _P, _P, _P, _P, _I, _P, _I, _P, _Z]),
    "dpc_dense_linear_sizes": (_I, [_I, _I, _I, _I, _I, _I, ctypes.POINTER(_Z)]),
    "dpc_dense_linear_forward": (_I, [_P, _I, _I, _I, _P, _Z, _I, _P, _Z, _I, _P, _I, _P, _I, _P, _Z, _P, _Z]),
    "dpc_dense_linear_backward": (_I, [_P, _I, _I, _I, _P, _Z, _I, _I, _I, _P, _Z, _P, _P, _P, _P, _Z]),
    "dpc_dense_linear_serve_workspace": (_Z, [_I, _I, _I, _I]),
    "dpc_dense_linear_serve": (_I, [_P, _I, _I, _I, _P, _Z, _I, _P, _P, _P, _I, _P, _P, _Z]),
    "dpc_dense_orthogonal_workspace": (_Z, [_I, _MP, _I]),
    "dpc_dense_orthogonal": (_I, [_P, _I, _MP, _I, _TP, _P, _Z]),
}


class DenseLibrary(object):
    """A loaded library.  ``host_memory`` marks the CPU emulation build (host pointers, no stream); only tests create those."""

    def __init__(self, path, host_memory=False):
        if not os.path.exists(path):
            raise DpcError("%s not found" % path)
        self.path = path
        self.host_memory = bool(host_memory)
        self._dll = ctypes.CDLL(path)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(self._dll, name)
            fn.restype = res
            fn.argtypes = args
            setattr(self, name, fn)
        for which, mirror in ((0, DpcDenseMatrix), (1, DpcDenseSteps)):
            if self.dpc_dense_abi_struct_bytes(which) != ctypes.sizeof(mirror):
                raise DpcError("%s: sizeof(%s) is %d in the library, %d in this binding (rebuild the library)"
                               % (path, mirror.__name__, self.dpc_dense_abi_struct_bytes(which), ctypes.sizeof(mirror)))

    def version(self):
        return self.dpc_dense_version().decode()

    @staticmethod
    def check(rc, what):
        if rc == 0:
            return
        if rc == -5:
            raise ValueError("%s: %s" % (what, _ERRORS[rc]))
        if rc < 0:
            raise DpcError("%s: %s" % (what, _ERRORS.get(rc, "error %d" % rc)))
        raise DpcError("%s: hipError_t %d" % (what, rc))


_ACTIVE = None


def get_library():
    """The product loader: libdpc_dense.so or an exception.  Never falls back."""
    global _ACTIVE
    if _ACTIVE is None:
        if not os.path.exists(LIB_PATH):
            raise DpcError("HIP extension %s is not built. Build it with `python __graft_entry__.py` (or `make -C "
                           "differentiable-point-clouds_amd/csrc/dense`). There is no CPU fallback." % LIB_PATH)
        _ACTIVE = DenseLibrary(LIB_PATH)
    return _ACTIVE


def set_library(lib):
    """Install a specific DenseLibrary; returns the previously active one (possibly None).  As with ``_capi.set_library`` an
    emulation library is refused unless DPC_TEST_HOOKS=1 is set."""
    global _ACTIVE
    if lib is not None and getattr(lib, "host_memory", False) and os.environ.get("DPC_TEST_HOOKS") != "1":
        raise DpcError("a host-memory (emulation) library can only be installed with DPC_TEST_HOOKS=1 (tests)")
    prev, _ACTIVE = _ACTIVE, lib
    return prev
