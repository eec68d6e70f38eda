"""``my_int4._C``: the 16 reference ops (reference ``csrc/bindings.cpp:28-68``),
implemented by ``wush_int4_kernel_amd._C`` on gfx950 HIP kernels, and the
8-bit operators around them (``quant_int8_token``, ``w8a8_*``, ``kv8_*``), which
the reference does not have."""
from wush_int4_kernel_amd._C import (  # noqa: F401
    abi_version,
    fused_transform_quant_int4,
    fused_transform_quant_int4_smallm,
    fused_transform_quant_int4_v3,
    fused_transform_quant_int4_wmma,
    kv8_append,
    kv8_attention,
    kv8_read,
    quant_int4,
    quant_int4_tensor_scale,
    quant_int4_tensor_scale_dev,
    quant_int8_token,
    s4_atom_selftest,
    w4a4_gemm,
    w4a4_gemm_cutlass,
    w4a4_gemm_cutlass_dev,
    w4a4_gemm_s4,
    w4a4_gemm_v1,
    w4a4_gemm_v2,
    w4a4_gemv,
    w4a4_gemv_multi,
    w8a8_gemm,
    w8a8_linear,
)
