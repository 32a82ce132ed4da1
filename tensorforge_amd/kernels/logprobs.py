"""Log probabilities of given tokens, with entropy and the most likely
alternatives, in one pass over the logits (``csrc/tf_logprobs.hip``): what a
serving API reports beside the sampled token, and a prompt's score.  The
reference samples greedily and reports no probabilities
(``tensorforge/scheduler/continuous.py:265-275``).
"""

from __future__ import annotations

from dataclasses import dataclass

import torch
from torch import Tensor

from tensorforge_amd import _native

MAX_TOP_K = 32


@dataclass(frozen=True, slots=True)
class TokenLogprobs:
    """fp32 ``logprobs [rows]`` and ``entropy [rows]``, the ``top_logprobs
    [rows, top_k]`` and their int64 ``top_tokens [rows, top_k]``."""

    logprobs: Tensor
    entropy: Tensor
    top_logprobs: Tensor
    top_tokens: Tensor

    @classmethod
    def allocate(cls, *, rows: int, top_k: int, device: torch.device) -> TokenLogprobs:
        return cls(
            logprobs=torch.empty(rows, dtype=torch.float32, device=device),
            entropy=torch.empty(rows, dtype=torch.float32, device=device),
            top_logprobs=torch.empty((rows, top_k), dtype=torch.float32, device=device),
            top_tokens=torch.empty((rows, top_k), dtype=torch.int64, device=device),
        )


def token_logprobs(logits: Tensor, tokens: Tensor, *, top_k: int = 0,
                   output: TokenLogprobs | None = None) -> TokenLogprobs:
    """``log_softmax(logits, -1)`` of a ``[rows, columns]`` matrix (fp32, fp16
    or bf16, contiguous rows that may be strided) at int64 ``tokens [rows]``,
    the entropy of each row (natural logarithm, fp32) and its ``top_k`` (at most
    32) largest logits in descending order, equal ones by index, a NaN above
    every number.  A token outside the row gives NaN (a padded row's, say); a
    row that holds a NaN or +inf, or nothing above -inf, has NaN log
    probabilities and entropy, as log_softmax has."""

    if not _native.is_available():
        raise RuntimeError(
            "the gfx950 kernel library is unavailable; build it with "
            "`python -m tensorforge_amd.build`"
        )
    if not logits.is_cuda:
        raise ValueError("token_logprobs requires CUDA tensors")
    device = logits.device
    if device.index != _native.current_device():
        with torch.cuda.device(device):
            return token_logprobs(logits, tokens, top_k=top_k, output=output)
    if logits.ndim != 2 or logits.stride(1) != 1:
        raise ValueError("logits must be [rows, columns] with contiguous rows")
    if logits.dtype not in _native.DTYPE_CODES:
        raise TypeError(f"unsupported dtype: {logits.dtype}")
    rows, columns = logits.shape
    if columns < 1:
        raise ValueError("log probabilities of an empty row")
    if not 0 <= top_k <= min(MAX_TOP_K, columns):
        raise ValueError("top_k must lie between 0 and 32 and not exceed the columns")
    if tokens.shape != (rows,) or tokens.dtype != torch.int64 or tokens.device != device or not tokens.is_contiguous():
        raise ValueError("tokens must be a contiguous int64 [rows] tensor on the logits' device")
    if logits.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("TensorForge HIP kernels are inference-only")
    if output is None:
        output = TokenLogprobs.allocate(rows=rows, top_k=top_k, device=device)
    else:
        for tensor, shape, dtype in ((output.logprobs, (rows,), torch.float32),
                                     (output.entropy, (rows,), torch.float32),
                                     (output.top_logprobs, (rows, top_k), torch.float32),
                                     (output.top_tokens, (rows, top_k), torch.int64)):
            if tensor.shape != shape or tensor.dtype != dtype or tensor.device != device or not tensor.is_contiguous():
                raise ValueError("output must hold contiguous fp32 [rows] and [rows, top_k] and int64 [rows, top_k] "
                                 "tensors on the logits' device")
    _native.check(
        _native.launch().tf_token_logprobs(
            logits.data_ptr(), logits.stride(0) if rows > 1 else columns, rows, columns, tokens.data_ptr(),
            output.logprobs.data_ptr(), output.entropy.data_ptr(), output.top_logprobs.data_ptr(),
            output.top_tokens.data_ptr(), top_k, _native.dtype_code(logits.dtype), _native.current_stream(device),
        ),
        "token_logprobs",
    )
    return output
