"""lockstep_amd -- MI355X (gfx950) MXFP4 hot path of lockstep.

Modules mirror the reference's Python API:
    lockstep_amd.fp4          <- fp4.py
    lockstep_amd.mxfp4_gemm   <- mxfp4_gemm.py
    lockstep_amd.dual_gemm    <- dual_gemm.py
    lockstep_amd.fp4_linear   <- fp4_linear.py
    lockstep_amd.device       <- h100.py (device guard)
and next to them, without a counterpart there:
    lockstep_amd.attention      sliding-window attention with sinks, forward and backward
    lockstep_amd.kv_cache       a paged MXFP4 key-value cache: append, attend, evict
    lockstep_amd.fp4_attention  a self-attention layer of all of them, trained and served
The kernels live in liblsmx.so (C ABI: include/lsmx.h), built by
lockstep_amd.build.
"""

__version__ = "0.1.0"
