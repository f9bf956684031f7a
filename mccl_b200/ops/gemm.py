"""bf16 GEMM on the 5th-generation tensor cores (tcgen05 + TMEM + TMA, csrc/device/gemm) and its fused
tensor-parallel forms.  `y = act(x @ w.T)` with x [M, K], w [N, K] (the nn.Linear weight layout), and the product of ragged
groups of rows, each with its expert's weights."""
from __future__ import annotations

import ctypes as C

import torch

from .. import _ext
from .. import _lib as L

_counter = {"launches": 0}
EPI = {"none": 0, "silu": 1}


def launches() -> int:
    return _counter["launches"] + _ext.load().launches("gemm")


def _lib():
    lib = L.load()
    if not getattr(lib, "_gemm_declared", False):
        vp, i = C.c_void_p, C.c_int
        lib.mcclTpGemm.restype = i
        lib.mcclTpGemm.argtypes = [vp, vp, vp, i, i, i, i, i, vp]
        lib.mcclTpGemm2.restype = i
        lib.mcclTpGemm2.argtypes = [vp, vp, vp, i, i, i, i, i, vp]
        lib.mcclTpAllGatherGemm.restype = i
        lib.mcclTpAllGatherGemm.argtypes = [vp, vp, vp, vp, vp, vp, i, i, i, i, vp]
        lib.mcclTpGemmReduceScatter.restype = i
        lib.mcclTpGemmReduceScatter.argtypes = [vp, vp, vp, vp, vp, vp, vp, i, i, i, C.c_uint64, vp]
        lib.mcclTpGemmLastError.restype = i
        lib.mcclTpGemmLastError.argtypes = []
        lib._gemm_declared = True
    return lib


def _stream(t, stream):
    return C.c_void_p(stream.cuda_stream if stream is not None else torch.cuda.current_stream(t.device).cuda_stream)


def supported(M: int, N: int, K: int, ranks: int = 1) -> bool:
    return M % (128 * ranks) == 0 and N % 64 == 0 and K % 64 == 0 and min(M, N, K) > 0


def gemm(x: torch.Tensor, w: torch.Tensor, out: torch.Tensor | None = None, epilogue: str = "none", max_ctas: int = 0,
         stream=None, two_sm: bool | None = None) -> torch.Tensor:
    """out[M, N] = act(x[M, K] @ w[N, K].T) in bf16 with fp32 accumulation, by the library's own tcgen05 kernel.
    `two_sm` selects the form in which pairs of SMs share a 256-row tile (needs M % 256 == 0); by default it is
    used whenever the shape allows it."""
    if x.is_cuda:
        y = _ext.load().gemm(x, w, out, EPI[epilogue], max_ctas, stream.cuda_stream if stream is not None else None, two_sm)
        if isinstance(y, torch.Tensor):
            return y
    else:
        raise RuntimeError("mccl gemm runs on CUDA (sm_100a) only")
    # Not taken by the kernels: say why.
    assert x.dtype == w.dtype == torch.bfloat16 and x.is_contiguous() and w.is_contiguous()
    M, K = x.shape
    N = w.shape[0]
    assert w.shape[1] == K
    if not supported(M, N, K):
        raise ValueError(f"unsupported GEMM shape {M}x{N}x{K}: M % 128, N % 64 and K % 64 must be 0")
    if two_sm and M % 256:
        raise ValueError(f"the two-SM GEMM needs M % 256 == 0 (got {M})")
    L.check(L.INVALID_ARGUMENT if y is None else y, "mcclTpGemm2" if (M % 256 == 0 if two_sm is None else two_sm) else "mcclTpGemm")


MAX_GROUPS = 1024


def check_groups(name: str, x: torch.Tensor, w: torch.Tensor, ends: torch.Tensor) -> None:
    """Shapes, types and devices of rows x [T, K], weights w [E, N, K] and ends [E]."""
    if x.dim() != 2 or w.dim() != 3 or w.shape[2] != x.shape[1]:
        raise ValueError(f"{name}: rows [T, K] and weights [E, N, K] (got {list(x.shape)} and {list(w.shape)})")
    if not 0 < w.shape[0] <= MAX_GROUPS:
        raise ValueError(f"{name}: 1 to {MAX_GROUPS} experts (got {w.shape[0]})")
    if ends.dtype not in (torch.int32, torch.int64) or ends.shape != (w.shape[0],) or not ends.is_contiguous():
        raise ValueError(f"{name}: ends are contiguous int32 or int64 [{w.shape[0]}] (got {ends.dtype} {list(ends.shape)})")
    if not (x.device == w.device == ends.device):
        raise ValueError(f"{name}: rows, weights and ends are on one device (got {x.device}, {w.device}, {ends.device})")
    if x.shape[0] >= 2 ** 31 - 256 or max(w.shape[1:]) >= 2 ** 31 - 256:
        raise ValueError(f"{name}: sizes below 2^31 - 256 (got {list(x.shape)} and {list(w.shape)})")


def grouped_gemm(x: torch.Tensor, w: torch.Tensor, ends: torch.Tensor) -> torch.Tensor:
    """y[t] = x[t] @ w[e].T for the rows t of expert e, which are [ends[e - 1], ends[e]) (from 0 for the first): products of ragged
    groups by the library's tcgen05 kernels (csrc/device/gemm/grouped_core.cuh), fp32 accumulation, differentiable in x and w, once.

    bf16 x [T, K] and w [E, N, K] (an nn.Linear weight for each expert), K and N multiples of 8; `ends` [E] int32 or int64 on the
    device, e.g. the cumulative sum of the tokens per expert: the host never waits for it.  An end below an earlier one is read as
    that one, one outside [0, T] as the nearest.  Rows from ends[-1] on belong to no expert: they are zero in y and in x's gradient
    and no part of w's; the gradient of an expert without rows is zero.  Weights that are a view with gaps or in another order (half of a
    joined matrix, a transposed one) are copied in every call, and so are rows whose elements are not adjacent or that are not a multiple of 16
    bytes apart."""
    y = _ext.load().grouped_gemm(x, w, ends) if x.is_cuda else None
    if y is not None:
        return y
    # Not taken by the kernels: say why.
    check_groups("grouped_gemm", x, w, ends)
    if x.dtype != torch.bfloat16 or w.dtype != torch.bfloat16:
        raise ValueError(f"grouped_gemm: bf16 rows and weights (got {x.dtype} and {w.dtype})")
    if w.shape[1] % 8 or w.shape[2] % 8 or 0 in w.shape:
        raise ValueError(f"grouped_gemm: N and K are multiples of 8, a row is a multiple of 16 bytes (got {w.shape[1]} and {w.shape[2]})")
    if not x.is_cuda:
        raise RuntimeError("grouped_gemm runs on CUDA (sm_100a) only")
    raise RuntimeError("grouped_gemm does not run under tracing, a dispatch mode or torch.func")


def last_error() -> int:
    """Error code a GEMM kernel recorded on the current device since the last call (0 = none): one that waited in vain gives up and leaves its
    results incomplete.  `grouped_gemm` and `fp8_gemm` raise from then on until this has been called; what a recorded graph replays
    does not ask."""
    return _lib().mcclTpGemmLastError()
