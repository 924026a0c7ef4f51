// dense.hip -- the dense-layer operators' library: kernels (k_*.inc) and the C ABI of include/dpc_dense.h.
#include "k_device.inc"
#include "k_quantize.inc"
#include "k_tile.inc"
#include "k_product.inc"
#include "k_orthogonal.inc"
#include "k_narrow.inc"

#include "host.inc"
