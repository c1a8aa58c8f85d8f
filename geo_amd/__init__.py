"""MI355X-native stochastic-computing convolution path (LFSR streams, AND/OR/popcount
convolution with partial binary accumulation, surrogate backward).

``geo_amd.capi``              - Python callers of the C ABI (include/geo_sc.h)
``geo_amd.utils_functional``  - conv2d_generic / quantize with the reference's signatures
``geo_amd.utils_class``       - Conv2d_Add_Partial and the fixed-point batch norms
``geo_amd.main_distill``      - an SC network trained from a teacher of dense 8-bit layers (``utils_functional.linear_q8`` and
                                its relatives, ``distill_topk``)
"""
__all__ = ["capi", "utils_functional", "utils_class", "workloads"]
