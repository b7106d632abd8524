"""8-bit values with a scale for each block of 128, and their products.

The format (include/mamba_lm_ops.h): codes e4m3 in rows, each block of 128
along a row with a power-of-two scale, the least one under which the block's
largest magnitude fits 448. ``fp8_matmul`` hands both to the tensor cores,
which apply the scales; ``fp8_linear`` is a linear layer whose three products
(output, input gradient, weight gradient) all run in 8 bits. There is no
fallback: without the built library the calls raise.
"""
from __future__ import annotations

import torch

from ._ops import ops


def quantize_fp8(x, channel_major=False):
    """Codes (rows, K) float8_e4m3fn and scales (rows, ceil(K / 128))
    float8_e8m0fnu of x.

    x (..., K), float32 or bfloat16: its rows. With channel_major x is
    (B, K, L), the layout of the scan's activations, and row b * L + l holds
    x[b, :, l]; so x.t() of a matrix is quantised along its rows' axis by
    ``quantize_fp8(x[None], channel_major=True)``. NaN and infinities become
    NaN codes and do not enter the scale. Codes and scales carry no gradient:
    ``fp8_linear`` is the differentiable form.
    """
    return ops().quantize_fp8(x, channel_major)


def quantize_fp8_both(x):
    """(codes, scales) of x (M, K), and of x.t(), from one pass over x: what the
    products need that sum over K, and those that sum over the rows. M up to 2^22."""
    return ops().quantize_fp8_both(x)


def dequantize_fp8(codes, scales, dtype=torch.float32):
    """The values (rows, K) that codes and scales stand for, rounded to float32
    (exact between its smallest normal and largest number) or bfloat16."""
    return ops().dequantize_fp8(codes, scales, dtype)


def fp8_matmul(a, a_scale, b, b_scale, out_dtype=torch.bfloat16, channel_major_batch=None):
    """a @ b.T for 8-bit operands a (M, K) and b (N, K), fp32 sums, rounded once.

    out_dtype float32 or bfloat16. The result is (M, N); with
    channel_major_batch = B (M = B * L) it is (B, N, L), the scan's layout.
    For inference and as the building block of ``fp8_linear``: 8-bit operands
    carry no gradient. A product that gives up a wait leaves its output incomplete
    and sets bit 0 of the library's device error word (mamba_ss_take_device_error).
    """
    return ops().fp8_matmul(a, a_scale, b, b_scale, out_dtype, channel_major_batch)


def fp8_linear(x, w):
    """y = x @ w.T with every product in 8 bits, differentiable in x and w.

    x (..., K), up to 2^22 rows, and w (N, K) float32 or bfloat16; y (..., N) has x's type. The
    operands of each product (y, the gradients of x and of w) are quantised in
    blocks of 128 along the axis that it sums over; sums are fp32.
    """
    return ops().fp8_linear(x, w)
