"""Operator surface of the reference's four extension modules
(actnn/setup.py:6-21: actnn.cpp_extension.{calc_precision,minimax,backward_func,quantization}),
implemented over the C ABI in include/actnn_hip.h, and the 8-bit tokens (`tokens`), which the reference does not have."""
from . import minimax, quantization, calc_precision, backward_func, tokens  # noqa: F401
