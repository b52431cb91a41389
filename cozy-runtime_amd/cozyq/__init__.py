"""cozyq: cozy-runtime's quantized-linear hot path, MI355X-native.

Hand-written HIP kernels for gfx950 (`csrc/`, built into `libcozyq.so` behind the C ABI of
`include/cozyq.h`) with a Python host layer that mirrors the reference's op surface:
`prebuilt.Prebuilt` (the op library), the per-format dispatchers `int8_linear`, `fp8_linear`,
`mx_linear` and `svdq_linear`, the operand-sharing API in `kernels`, and the encoded leaves and
their providers in `leaves` / `selection`. `heads`, `kv_cache`, `attention` and `norms` are a language model's step
between its linears: head norms with the rotation, the paged 8-bit cache and attention over it, attention to an
encoder's states, and the residual stream's norms in 8 bits.
"""

from cozyq._lib import KernelsAbsent  # noqa: F401
