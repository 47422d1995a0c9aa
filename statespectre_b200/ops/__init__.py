"""Operators on torch tensors, and the kernel profiling command (``profile_case``)."""

from .block128 import (dequantize, linear, linear_input_grad, linear_weight_grad, product_error, quantize, swiglu,
                       swiglu_backward, swiglu_forward)

__all__ = ["quantize", "dequantize", "linear", "linear_input_grad", "linear_weight_grad", "swiglu", "swiglu_forward",
           "swiglu_backward", "product_error"]
