"""Decode projections by 4-bit weights on gfx950 (``csrc/tf_linear_mxfp4.hip``):
e2m1 codes with a power-of-two scale for each 32 columns of K.  A projection
of a decode step reads its weight once, so it reads 4.25 bits a weight in
place of 16.  The reference keeps its nn.Linear weights in the model's dtype
(``tensorforge/model/layers.py:88-95, 144-146``).
"""

from __future__ import annotations

import torch
from torch import Tensor

from tensorforge_amd import _native

MAX_ROWS = 64
GROUP = 32
# The halves between neighbouring e2m1 values 0, 0.5, 1, 1.5, 2, 3, 4, 6, and
# which of the two a tie goes to (the one with an even code).
_BORDERS = ((0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False))


def quantize_mxfp4(weight: Tensor) -> tuple[Tensor, Tensor]:
    """``(codes, scales)`` of a ``[n, k]`` weight for :func:`linear_mxfp4`: each
    group of 32 columns gets the power of two that puts its largest value
    between 4 and 8 (``2^(floor(log2(max)) - 2)``, at least ``2^-126``; finite
    weights only), and each weight the nearest e2m1 value (ties to the even
    code, magnitudes above 6 to 6).  ``codes [n, k / 2]`` (uint8) hold the even
    column in the low half, ``scales [n, k / 32]`` are float8_e8m0fnu.  A zero
    group has scale ``2^-126``."""

    if weight.ndim != 2 or weight.shape[1] % GROUP or weight.shape[1] == 0:
        raise ValueError("weight must be [n, k] with k a multiple of 32")
    if not weight.is_floating_point():
        raise TypeError(f"unsupported dtype: {weight.dtype}")
    n, k = weight.shape
    values = weight.detach().float().view(n, k // GROUP, GROUP) if weight.is_contiguous() else (
        weight.detach().float().contiguous().view(n, k // GROUP, GROUP))
    largest = values.abs().amax(-1)
    if not bool(torch.isfinite(largest).all()):
        raise ValueError("weights must be finite")
    exponents = (torch.frexp(largest)[1] - 3).clamp(min=-126)
    exponents = torch.where(largest > 0, exponents, -126)
    size = torch.ldexp(values.abs(), -exponents[..., None])
    codes = torch.zeros_like(size, dtype=torch.uint8)
    for border, tie_up in _BORDERS:
        codes += size >= border if tie_up else size > border
    codes += 8 * (values < 0).to(torch.uint8)
    codes = codes.view(n, k // 2, 2)
    return (codes[..., 0] | (codes[..., 1] << 4)).contiguous(), (exponents + 127).to(torch.uint8).view(
        torch.float8_e8m0fnu)


def linear_mxfp4(x: Tensor, weight: Tensor, scales: Tensor, *, output: Tensor | None = None,
                 residual: Tensor | None = None) -> Tensor:
    """``x [m, k] @ W[n, k].T`` for m <= 64 rows of fp16 or bf16, W given by
    e2m1 ``weight [n, k / 2]`` (uint8, the even column in the low half) and
    ``scales [n, k / 32]`` (float8_e8m0fnu) as :func:`quantize_mxfp4` makes
    them; summed in fp32 and rounded once.  ``residual [m, n]``:
    ``round(round(x . W) + residual)``, as in :func:`linear_kstream`; ``output``
    may be the residual itself."""

    if not _native.is_available():
        raise RuntimeError(
            "the gfx950 kernel library is unavailable; build it with "
            "`python -m tensorforge_amd.build`"
        )
    if not x.is_cuda:
        raise ValueError("linear_mxfp4 requires CUDA tensors")
    device = x.device
    if device.index != _native.current_device():
        with torch.cuda.device(device):
            return linear_mxfp4(x, weight, scales, output=output, residual=residual)
    if x.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"unsupported dtype: {x.dtype}")
    if x.ndim != 2 or x.shape[0] > MAX_ROWS or x.stride(1) != 1 or x.stride(0) % 8 or x.data_ptr() % 16:
        raise ValueError("linear_mxfp4 needs x [m <= 64, k] with 16-byte aligned contiguous rows")
    m, k = x.shape
    if k == 0 or k % GROUP:
        raise ValueError("linear_mxfp4 needs a K that is a multiple of 32")
    if weight.dtype != torch.uint8 or weight.ndim != 2 or weight.shape[1] != k // 2:
        raise ValueError("weight must be uint8 [n, k / 2]")
    n = weight.shape[0]
    if scales.dtype != torch.float8_e8m0fnu or scales.shape != (n, k // GROUP):
        raise ValueError("scales must be float8_e8m0fnu [n, k / 32]")
    if weight.device != device or scales.device != device:
        raise ValueError("x, weight and scales must share one device")
    if weight.stride(1) != 1 or weight.stride(0) % 16 or weight.data_ptr() % 16 or not scales.is_contiguous():
        raise ValueError("weight rows must be contiguous and 16-byte aligned, scales contiguous")
    if x.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("TensorForge HIP kernels are inference-only")
    if output is None:
        output = torch.empty((m, n), dtype=x.dtype, device=device)
    elif output.shape != (m, n) or output.dtype != x.dtype or output.device != device or output.stride(1) != 1:
        raise ValueError("output must be [m, n] with contiguous rows, x's dtype and device")
    residual_ptr, residual_stride = None, 0
    if residual is not None:
        if (residual.shape != (m, n) or residual.dtype != x.dtype or residual.device != device
                or residual.stride(1) != 1):
            raise ValueError("residual must be [m, n] with contiguous rows, x's dtype and device")
        residual_ptr, residual_stride = residual.data_ptr(), residual.stride(0)
    _native.check(
        _native.launch().tf_linear_mxfp4(
            x.data_ptr(), x.stride(0), weight.data_ptr(), weight.stride(0), scales.data_ptr(), k // GROUP,
            residual_ptr, residual_stride, output.data_ptr(), output.stride(0), m, n, k,
            _native.dtype_code(x.dtype), _native.current_stream(device),
        ),
        "linear_mxfp4",
    )
    return output
