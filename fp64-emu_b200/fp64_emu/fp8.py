"""Products of 8-bit floating-point codes with a power-of-two scale per 128 values.

A block of up to 128 values with largest finite magnitude amax is held as codes
(float8_e4m3fn, or float8_e5m2 for values of wider range) and one scale 2^e
(float8_e8m0fnu), e the smallest integer >= -127 with amax <= FMAX * 2^e; a code
is the round-to-nearest-even 8-bit float of x * 2^-e.  NaN stays NaN,
infinity becomes NaN, and neither counts towards amax.

Which values of a matrix [R, C] share a scale:
  "row"   128 neighbours of a row       scales [R, ceil(C / 128)]
  "col"   128 neighbours of a column    scales [ceil(R / 128), C]
  "tile"  a 128 x 128 square            scales [ceil(R / 128), ceil(C / 128)]
A product contracts along blocks, so an operand carries "row" scales where its
rows are contracted, "col" where its columns are, and "tile" fits both.

Codes and scales carry no gradient: what quantize_fp8, quantize_fp8_both,
dequantize_fp8 and the mm_*_fp8 products return is a constant to autograd, in
reverse and in forward mode, whatever their inputs require, as if detached.  A
round trip inside a model therefore cuts the gradient there; linear_fp8 is the
operator that has one.

No counterpart in the reference, whose products take float64 operands.
"""
import torch

from ._ops import ops

_BLOCKS = {"row": 0, "col": 1, "tile": 2}

_quantize = ops.fp8_quantize.default
_quantize_both = ops.fp8_quantize_both.default
_dequantize = ops.fp8_dequantize.default
_mm = ops.fp8_mm.default
_linear = ops.fp8_linear.default


def quantize_fp8(x: torch.Tensor, blocks: str = "row", code: torch.dtype = torch.float8_e4m3fn) -> tuple:
    """(codes, scales) of a float32 / float16 / bfloat16 CUDA matrix.  The
    codes' rows start on 16-byte boundaries, as the products read them.  The
    result is detached from x."""
    assert blocks in _BLOCKS, "blocks must be 'row', 'col' or 'tile'"
    return _quantize(x, _BLOCKS[blocks], code)


def quantize_fp8_both(x: torch.Tensor, code: torch.dtype = torch.float8_e4m3fn, transposed: bool = False) -> tuple:
    """(row codes, row scales, col codes, col scales) in one pass over x: what
    a layer's forward product and its weight gradient contract.  transposed:
    the col codes, of the same shape, are stored with columns contiguous; a
    product that contracts columns needs one of its operands so, and makes
    that copy itself otherwise.  The result is detached from x."""
    return _quantize_both(x, code, transposed)


def dequantize_fp8(codes: torch.Tensor, scales: torch.Tensor, blocks: str = "row",
                   dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values codes and scales stand for, rounded once to dtype, without a
    gradient.  In float16 a value that rounded up past 65504 when it was coded
    becomes infinity: 63488 and more in e4m3 (the next code is 65536), 61440 and
    more in e5m2."""
    assert blocks in _BLOCKS, "blocks must be 'row', 'col' or 'tile'"
    return _dequantize(codes, scales, _BLOCKS[blocks], dtype)


def mm_fp8(A: torch.Tensor, B: torch.Tensor, a_scale: torch.Tensor, b_scale: torch.Tensor,
           dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """C = A @ B^T with A [M, K] and B [N, K] codes, both with "row" or "tile"
    scales.  Sums are held in 32 bits and rounded once to dtype (bfloat16,
    float16 or float32).  The tensor cores cut off what an addition into such a
    sum shifts out, so float32 results are 1e-7 of their norm off (4e-7 at K = 2^20;
    torch's own product 6e-8 at K = 2048 and 2e-7 at 16384), and the sums behind
    16-bit results up to 2e-5, below their rounding."""
    return _mm(A, B, a_scale, b_scale, 0, dtype)


def mm_nt_fp8(A: torch.Tensor, Bt: torch.Tensor, a_scale: torch.Tensor, bt_scale: torch.Tensor,
              dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """C = A @ Bt with Bt [K, N] consumed in place; A with "row" or "tile"
    scales, Bt with "col" or "tile" scales."""
    return _mm(A, Bt, a_scale, bt_scale, 1, dtype)


def mm_tn_fp8(At: torch.Tensor, Bt: torch.Tensor, at_scale: torch.Tensor, bt_scale: torch.Tensor,
              dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """C = At^T @ Bt with At [K, M] and Bt [K, N] consumed in place, both with
    "col" or "tile" scales."""
    return _mm(At, Bt, at_scale, bt_scale, 2, dtype)


def linear_fp8(x: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor = None) -> torch.Tensor:
    """y = x @ w^T in 8 bits, y in x's type; x [..., K] float32, float16 or bfloat16.

    w: weights [N, K] in one of these types, quantised in squares on every
    call, or (with w_scale) kept e4m3 / e5m2 codes with "tile" scales, as a
    server holds them.  x is quantised in row blocks.

    Differentiable in x, and in w where w is not kept codes.  For the weight
    gradient x is kept in 8 bits, with blocks along its rows (the tokens):
    one byte a value instead of x itself.  With gradients dy quantised in row
    blocks and in column blocks (e4m3),
        dx = q_row(dy) @ q_tile(w),    dw = q_col(dy)^T @ q_col(x).
    There is no second derivative and no forward mode: both are refused."""
    return _linear(x, w, w_scale)


def fp8_status(device: torch.device = None) -> int:
    """0, or the site code of the first bounded device wait of an 8-bit product
    that ran out on the device (default: the current one) since the last call;
    the outputs of that product are not valid then.  Waits for the current
    stream."""
    index = torch.cuda.current_device() if device is None else torch.device(device).index
    return ops.fp8_status(torch.cuda.current_device() if index is None else index)
