"""8-bit tokens: rows of features kept as int8 codes with one fp32 scale a row (no reference counterpart).

A token is the last dimension of a tensor [..., K]: a word's hidden state, a row of a linear layer's input, or the channels of
one pixel of a channels-last image.  Its codes are 127 x / max|x|, rounded to the nearest whole number (halves away from
zero), its scale is max|x| / 127.  Unlike the streams of `quantization` they are symmetric about zero and rounded the
same way each time, so that a product in 8-bit integers can read them as they are; the same codes are the checkpoint that the
weight gradient reads in the backward pass.

A row without a magnitude of 2^-100 or more (a padded token) has scale 0 and codes 0.  A row that holds a NaN or an
infinity has scale NaN: everything made from it is NaN.

Codes come in rows that begin at multiples of 16 bytes (their stride is K rounded up to 16), the layout the kernels read;
codes laid out otherwise are taken too, and copied first.  Everything runs on the current stream of the tensors' device.
torch.jit.trace does not see these calls, which refuse to be recorded; the layers over them can be traced.
"""
import torch

from . import _glue as g


def _dtype_code(dtype, what):
    if dtype not in g.DTYPE_CODE:
        raise RuntimeError(f"{what}: float32, float16 or bfloat16 expected, got {dtype}")
    return g.DTYPE_CODE[dtype]


def quantize_tokens(data):
    """-> (codes, scale): int8 [..., K] and fp32 [...] of a float32, float16 or bfloat16 tensor [..., K]."""
    return g.untraced("quantize_tokens").quantize_tokens(data)


def dequantize_tokens(codes, scale, dtype=torch.float32):
    """codes * scale, rounded to `dtype`: once, for bfloat16 by way of 32 bits.  In 16 bits these are the values that
    linear_tokens_grad_weight multiplies, bit for bit."""
    return g.untraced("dequantize_tokens").dequantize_tokens(codes, scale, _dtype_code(dtype, "dequantize_tokens"))


def matmul_tokens(codes, scale, weight_codes, weight_scale, bias=None, dtype=torch.float32):
    """scale[m] * weight_scale[o] * sum_k codes[m, k] * weight_codes[o, k] + bias[o] -> [..., O] in `dtype`.

    The weight is kept as tokens itself (`quantize_tokens` of a linear layer's [O, K] weight: one scale for each output
    channel).  The sums are 32-bit integers and exact, for up to 131071 features."""
    dtype = _dtype_code(dtype, "matmul_tokens")
    return g.untraced("matmul_tokens").matmul_tokens(codes, scale, weight_codes, weight_scale, bias, dtype)


def linear_tokens(data, weight_codes, weight_scale, bias=None, keep=False):
    """matmul_tokens(*quantize_tokens(data), ...) in the type of `data`.  With `keep` also the tokens as they were
    multiplied, which are the checkpoint that linear_tokens_grad_weight reads: (output, codes, scale)."""
    out, codes, scale = g.untraced("linear_tokens").linear_tokens(data, weight_codes, weight_scale, bias, bool(keep))
    return (out, codes, scale) if keep else out


def linear_tokens_grad_weight(grad_output, codes, scale, dtype=None):
    """grad_output[..., O]^T @ (codes * scale)[..., K] -> [O, K], summed over all tokens in fp32: the weight gradient of
    a linear layer from the tokens it kept.  grad_output is float16 or bfloat16 (the values of the codes are rounded to its type
    on their way into the product); the result comes in its type, or with `dtype` in float32."""
    dtype = None if dtype is None else _dtype_code(dtype, "linear_tokens_grad_weight")
    return g.untraced("linear_tokens_grad_weight").linear_tokens_grad_weight(grad_output, codes, scale, dtype)
