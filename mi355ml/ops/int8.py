"""Products of 8-bit matrices with a scale for each row.

A float matrix is held as 8-bit integers and one float32 scale for each row,
a quarter of its float32 bytes; the product of two such matrices runs on the
int8 matrix cores, at twice the rate of 16-bit floats. For activations the
rows are tokens (samples), for weights of layout [n, k] (``components_``,
``coef_``) they are output channels, so the product has one scale for each of
its rows and one for each of its columns:

    y[i, j] = (sum_k xq[i, k] wq[j, k]) * x_scale[i] * w_scale[j] + bias[j]

The sum is exact: it is taken in 32-bit integers, which k < 131072 values
cannot overflow. None of this is differentiable: results carry no gradient.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from ._ext import hip_ext, use_hip

_FLOATS = (torch.float32, torch.float16, torch.bfloat16)
#: the longest sum of products of 8-bit values that 32 bits always hold
MAX_K = 131071
#: most rows of either operand of a product
MAX_ROWS = 2 ** 27 - 1


def _check_floats(x: torch.Tensor, name: str) -> None:
    if x.dim() != 2:
        raise ValueError(f"{name} must be 2-D, got {x.dim()}-D")
    if x.dtype not in _FLOATS:
        raise TypeError(f"{name} must be float32, float16 or bfloat16, "
                        f"got {x.dtype}")


def quantize_rows(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """8-bit rows of a float matrix: (q int8 [m, k], scale float32 [m]).

    scale[i] = float32(max_k |x[i, k]| / 127) and q = x / scale, rounded to
    the nearest integer (halves to the even one) from the exact quotient;
    x is q * scale within half a scale. A row of zeros has scale 0. A row
    that holds an infinity or NaN has scale NaN and zeros for q, so that it
    gives NaN wherever it is used.

    The rows of q begin at multiples of 16 bytes (of 128 from k = 1024 on),
    as the product wants them: q is a view of a wider matrix where k is no
    such multiple.
    """
    _check_floats(x, "x")
    if use_hip(x):
        return hip_ext().quantize_rows(x)
    x = x.detach()
    if x.shape[1] == 0:
        return (torch.empty(x.shape, dtype=torch.int8, device=x.device),
                torch.zeros(x.shape[0], device=x.device))
    xd = x.double()
    big = xd.abs().amax(dim=1)
    scale = (big / 127.0).float()
    fine = torch.isfinite(big)
    some = fine & (scale > 0)
    q = torch.round(xd / torch.where(some, scale.double(), 1.0)[:, None])
    # a scale among the subnormal numbers is rounded too coarsely to keep
    # the quotient below 127.5
    q = torch.where(some[:, None], q.clamp(-127, 127), 0.0)
    scale = torch.where(fine, scale, float("nan"))
    return q.to(torch.int8), scale


def _check_int8(q: torch.Tensor, name: str) -> None:
    if q.dim() != 2:
        raise ValueError(f"{name} must be 2-D, got {q.dim()}-D")
    if q.dtype != torch.int8:
        raise TypeError(f"{name} must be int8, got {q.dtype}")


def _check_vector(s: torch.Tensor, size: int, device, name: str) -> None:
    if s.dim() != 1 or s.shape[0] != size:
        raise ValueError(f"{name} must have shape ({size},), got "
                         f"{tuple(s.shape)}")
    if s.dtype != torch.float32:
        raise TypeError(f"{name} must be float32, got {s.dtype}")
    if s.device != device:
        raise ValueError(f"{name} is on {s.device}, the rows are on {device}")


def _check_weights(x, x_name, wq, w_scale, bias, out_dtype) -> None:
    _check_int8(wq, "wq")
    if x.shape[1] != wq.shape[1]:
        raise ValueError(f"{x_name} has rows of {x.shape[1]} values and wq "
                         f"of {wq.shape[1]}")
    if x.shape[1] > MAX_K:
        raise ValueError(f"rows of more than {MAX_K} values could overflow "
                         f"the 32-bit sums, got {x.shape[1]}")
    for name, rows in ((x_name, x.shape[0]), ("wq", wq.shape[0])):
        if rows > MAX_ROWS:
            raise ValueError(f"{name} may have at most {MAX_ROWS} rows, got "
                             f"{rows}")
    if wq.device != x.device:
        raise ValueError(f"wq is on {wq.device}, the rows are on {x.device}")
    _check_vector(w_scale, wq.shape[0], x.device, "w_scale")
    if bias is not None:
        _check_vector(bias, wq.shape[0], x.device, "bias")
    if out_dtype not in _FLOATS:
        raise TypeError(f"out_dtype must be float32, float16 or bfloat16, "
                        f"got {out_dtype}")


def int8_matmul(xq: torch.Tensor, x_scale: torch.Tensor, wq: torch.Tensor,
                w_scale: torch.Tensor, bias: Optional[torch.Tensor] = None,
                out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """y[i, j] = (sum_k xq[i, k] wq[j, k]) x_scale[i] w_scale[j] + bias[j].

    xq: int8 [m, k]; wq: int8 [n, k]; scales and bias float32. Returns
    [m, n] in out_dtype, computed in float32 from the exact sum and rounded
    once. Rows that do not begin at multiples of 16 bytes (``quantize_rows``
    lays them out so) are copied first.
    """
    _check_int8(xq, "xq")
    _check_weights(xq, "xq", wq, w_scale, bias, out_dtype)
    _check_vector(x_scale, xq.shape[0], xq.device, "x_scale")
    if use_hip(xq):
        return hip_ext().int8_product(xq, x_scale, wq, w_scale, bias,
                                      out_dtype)
    # float64 holds every one of the integer sums
    y = (xq.double() @ wq.double().t()).float()
    y = y * x_scale.detach()[:, None] * w_scale.detach()[None, :]
    if bias is not None:
        y = y + bias.detach()
    return y.to(out_dtype)


def int8_linear(x: torch.Tensor, wq: torch.Tensor, w_scale: torch.Tensor,
                bias: Optional[torch.Tensor] = None,
                out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``int8_matmul`` of float rows with weights that were quantised once.

    x: [m, k] float32, float16 or bfloat16, quantised row by row on the way;
    returns [m, n] in out_dtype (default: x's type).
    """
    _check_floats(x, "x")
    out_dtype = x.dtype if out_dtype is None else out_dtype
    _check_weights(x, "x", wq, w_scale, bias, out_dtype)
    if use_hip(x):
        return hip_ext().int8_linear(x, wq, w_scale, bias, out_dtype)
    xq, x_scale = quantize_rows(x)
    return int8_matmul(xq, x_scale, wq, w_scale, bias, out_dtype)
