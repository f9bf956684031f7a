"""Products in 8-bit floating point with a scale for each block of 128, for serving (csrc/device/gemm/fp8_core.cuh,
csrc/ops/fp8_quantize.cu): e4m3 values, power-of-two scales (e8m0) that the tensor core applies itself, fp32 sums.

    w8 = fp8_quantize(linear.weight, rows=128)                # once; [N, K], or [E, N, K] for experts
    y = fp8_gemm(x, w8)                                       # x [M, K] in bf16: quantised by blocks of 128 of a row within the call
    y = fp8_gemm(x, experts8, ends)                           # ragged groups of rows, as in ops.gemm.grouped_gemm
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Union

import torch

from .. import _ext
from .gemm import check_groups, launches  # noqa: F401  (these kernels are counted with the other products)

BLOCK = 128


class BlockScaled(NamedTuple):
    """`data` (float8_e4m3fn, [..., M, K]) and the scale of each block (float8_e8m0fnu, [..., M / rows, K / 128] rounded up), rows being
    1 or 128.  `fp8_quantize` keeps the rows of the scales a multiple of four bytes apart, as the kernels read them, and the rows of weights a
    multiple of 128; scales of another pitch, and values whose elements are not adjacent or whose rows are not a multiple of 16 bytes apart,
    are copied in every call."""
    data: torch.Tensor
    scale: torch.Tensor

    def dequantize(self) -> torch.Tensor:
        """The values in fp32."""
        (m, k), s = self.data.shape[-2:], self.scale.float()
        if s.shape[-2] != m:
            s = s.repeat_interleave(BLOCK, -2)[..., :m, :]
        return self.data.float() * s.repeat_interleave(BLOCK, -1)[..., :k]


def fp8_quantize(x: torch.Tensor, rows: int = 1) -> BlockScaled:
    """bf16 `x` in 8 bits: a scale for each 1 x 128 values of [M, K] (`rows=1`, activations) or for 128 x 128 of [N, K] or [E, N, K]
    (`rows=128`, weights).  The scale is the smallest power of two that brings the block's largest magnitude to 448 or less (1 for a block of
    zeros, never below 2^-127), the values the nearest e4m3 numbers of x / scale.  Inf and NaN take no part in the scale and become
    NaN.  K is a multiple of 16; the last block of a row may be shorter than 128.  The result is a constant for autograd."""
    if rows not in (1, BLOCK):
        raise ValueError(f"fp8_quantize: blocks of 1 or {BLOCK} rows (got {rows})")
    if x.dtype != torch.bfloat16 or x.dim() not in ((2,) if rows == 1 else (2, 3)):
        raise ValueError(f"fp8_quantize: a bf16 matrix, or [E, N, K] for blocks of {BLOCK} rows (got {x.dtype} {list(x.shape)})")
    if x.shape[-1] == 0 or x.shape[-1] % 16 or (rows == BLOCK and 0 in x.shape) or max(x.shape) >= 2 ** 31 - 256:
        raise ValueError(f"fp8_quantize: K is a multiple of 16 (got {list(x.shape)})")
    if not x.is_cuda:
        raise RuntimeError("fp8_quantize runs on CUDA (sm_100a) only")
    return BlockScaled(*_ext.load().fp8_quantize(x.detach(), rows == BLOCK))


def _blocks(n: int) -> int:
    return (n + BLOCK - 1) // BLOCK


def fp8_gemm(x: Union[torch.Tensor, BlockScaled], w: BlockScaled, ends: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y [M, N] (bf16) = x @ w.T in 8 bits with fp32 sums.  `x`: bf16 [M, K], quantised by blocks of 128 of a row within the call, or
    BlockScaled with a scale for each 1 x 128; `w`: BlockScaled [N, K] with a scale for each 128 x 128.  With `ends` the rows
    [ends[e - 1], ends[e]) go through w[e] of [E, N, K], as in `grouped_gemm`: ends on the device, rows behind the last one zero.
    N is a multiple of 8, K of 16.  There is no gradient: an x that asks for one is refused (use torch.no_grad)."""
    data, scale = (x.data, x.scale) if isinstance(x, BlockScaled) else (x, None)
    wd, ws = w
    y = _ext.load().fp8_gemm(data, scale, wd, ws, ends) if data.is_cuda else None
    if y is not None:
        return y
    # Not taken by the kernels: say why.
    if ends is not None:
        check_groups("fp8_gemm", data, wd, ends)
    elif data.dim() != 2 or wd.dim() != 2 or data.shape[1] != wd.shape[1] or max(*data.shape, *wd.shape) >= 2 ** 31 - 256:
        raise ValueError(f"fp8_gemm: rows [M, K] and weights [N, K], or [E, N, K] with ends (got {list(data.shape)} and {list(wd.shape)})")
    n, k = wd.shape[-2:]
    if n % 8 or k % 16 or n == 0 or k == 0:
        raise ValueError(f"fp8_gemm: N is a multiple of 8 and K of 16 (got {n} and {k})")
    if wd.dtype != torch.float8_e4m3fn or ws.dtype != torch.float8_e8m0fnu or tuple(ws.shape) != (*wd.shape[:-2], _blocks(n), _blocks(k)):
        raise ValueError(f"fp8_gemm: weights are float8_e4m3fn with float8_e8m0fnu scales {[*wd.shape[:-2], _blocks(n), _blocks(k)]} "
                         f"(got {wd.dtype}, {ws.dtype} {list(ws.shape)})")
    if scale is None:
        if data.dtype != torch.bfloat16:
            raise ValueError(f"fp8_gemm: rows are bf16 or BlockScaled (got {data.dtype})")
    elif data.dtype != torch.float8_e4m3fn or scale.dtype != torch.float8_e8m0fnu or scale.shape != (data.shape[0], _blocks(k)):
        raise ValueError(f"fp8_gemm: quantised rows are float8_e4m3fn with float8_e8m0fnu scales {[data.shape[0], _blocks(k)]} "
                         f"(got {data.dtype}, {scale.dtype} {list(scale.shape)})")
    if any(t is not None and t.device != data.device for t in (scale, wd, ws)):
        raise ValueError("fp8_gemm: rows, weights and scales are on one device")
    if torch.is_grad_enabled() and data.requires_grad:
        raise RuntimeError("fp8_gemm has no gradient: detach its rows or call it under torch.no_grad()")
    if not data.is_cuda:
        raise RuntimeError("fp8_gemm runs on CUDA (sm_100a) only")
    raise RuntimeError("fp8_gemm does not run under tracing, a dispatch mode or torch.func")
