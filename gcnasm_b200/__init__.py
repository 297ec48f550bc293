"""gcnasm_b200 -- B200-native (sm_100a) block-scaled FP8 GEMM.

The product is the C ABI in ``include/b2g/gemm.h`` implemented by
``gcnasm_b200/_lib/libb2g.so`` (hand-written tcgen05 / TMA kernels).  This
package binds it (``capi``), mirrors the reference's f4gemm host helpers
(``f4gemm``) and offers torch-tensor wrappers (``ops``).  Beside the GEMMs stand
the 4-bit key/value cache and its attention (``include/b2g/kv4.h``, ``kv4``).
"""
from . import capi  # noqa: F401

__all__ = ["capi", "f4gemm", "kv4", "ops", "build"]
