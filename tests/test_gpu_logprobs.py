"""Token log probabilities, entropies and top tokens against log_softmax in 64
bits: types, widths, strides, ties, infinities, NaN and empty rows."""

from __future__ import annotations

import pytest
import torch

from tensorforge_amd.kernels import TokenLogprobs, token_logprobs
from tests.q8_reference import logprobs

pytestmark = pytest.mark.gpu


def _close(got, want, bound):
    got, want = got.double().cpu(), want.double()
    same = (got == want) | (got.isnan() & want.isnan())
    return bool((same | ((got - want).abs() <= bound)).all())


def _check(result, values, tokens, top_k, what=""):
    given, entropy, top, top_tokens, bound, entropy_bound = logprobs(values, tokens, top_k)
    assert torch.equal(result.top_tokens.cpu(), top_tokens), what
    assert _close(result.logprobs, given, bound), what
    assert _close(result.entropy, entropy, entropy_bound), what
    assert _close(result.top_logprobs, top, bound[:, None]), what


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize(("rows", "columns", "top_k"), [
    (64, 32000, 5), (1, 32000, 32), (3, 1, 1), (2, 7, 7), (5, 1031, 20), (300, 257, 3), (2, 65536, 8), (1, 131072, 20),
    (2, 140001, 32), (4, 33000, 0), (3, 32, 32), (2, 8192, 1), (2, 16385, 4)])
def test_shapes(device, dtype, rows, columns, top_k):
    generator = torch.Generator().manual_seed(rows + columns)
    values = (2.5 * torch.randn(rows, columns, generator=generator)).to(dtype)
    tokens = torch.randint(columns, (rows,), generator=generator)
    result = token_logprobs(values.to(device), tokens.to(device), top_k=top_k)
    assert result.top_tokens.dtype == torch.int64 and result.top_logprobs.shape == (rows, top_k)
    _check(result, values, tokens, top_k)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("columns", [900, 32000, 70000, 140001])
def test_ties(device, dtype, columns):
    """Equal values by index: a constant row, rows of two and of 32 values, more
    ties than any list of candidates holds, and zeros of both signs."""

    generator = torch.Generator().manual_seed(columns)
    values = torch.zeros(6, columns)
    values[1] = torch.randint(2, (columns,), generator=generator).float()
    values[2] = torch.randint(32, (columns,), generator=generator).float()
    values[3, 5::9] = -0.0
    values[4] = torch.arange(columns).float().neg() / 64   # descending, ties by rounding
    values[5] = torch.arange(columns).float() / 64
    values = values.to(dtype)
    tokens = torch.arange(6)
    _check(token_logprobs(values.to(device), tokens.to(device), top_k=32), values, tokens, 32)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("columns", [64, 32000, 140001])
def test_masked_and_non_finite_rows(device, dtype, columns):
    generator = torch.Generator().manual_seed(2)
    values = torch.randn(9, columns, generator=generator)
    lowest, largest = torch.finfo(dtype).min, torch.finfo(dtype).max
    values[0, 10:] = float("-inf")                  # a mask that leaves ten tokens
    values[1] = float("-inf")
    values[1, 40] = 1.5                             # one token
    values[2] = float("-inf")                       # nothing
    values[3, 7:] = lowest                          # a mask of the type's lowest value
    values[4, 3] = float("inf")
    values[5, 20] = float("nan")
    values[5, 50] = float("nan")
    values[6] = lowest                              # equal: uniform
    values[7, 12] = largest
    values[8] *= 30                                 # sharp
    values = values.to(dtype)
    tokens = torch.tensor([3, 40, 0, 6, 3, 1, 5, 12, 9])
    _check(token_logprobs(values.to(device), tokens.to(device), top_k=12), values, tokens, 12)


def test_tokens_outside_the_row(device):
    values = torch.randn(5, 100, generator=torch.Generator().manual_seed(3))
    tokens = torch.tensor([-1, 100, 99, -100, 1 << 40])
    result = token_logprobs(values.to(device), tokens.to(device), top_k=2)
    assert result.logprobs.isnan().tolist() == [True, True, False, True, True]
    _check(result, values, tokens, 2)


def test_the_sampled_token_is_the_first_alternative(device):
    from tensorforge_amd.kernels import argmax_rows

    values = torch.randn(40, 32000, generator=torch.Generator().manual_seed(4)).bfloat16().to(device)
    tokens = argmax_rows(values)
    result = token_logprobs(values, tokens, top_k=3)
    assert torch.equal(result.top_tokens[:, 0], tokens)
    assert torch.equal(result.top_logprobs[:, 0], result.logprobs)


@pytest.mark.parametrize("first", [0, 1, 3, 8])
def test_strided_rows_and_given_outputs(device, first):
    wide = torch.randn(9, 1003, generator=torch.Generator().manual_seed(5)).bfloat16()
    values = wide[:, first:first + 990]
    tokens = torch.arange(9) * 100
    output = TokenLogprobs.allocate(rows=9, top_k=4, device=device)
    result = token_logprobs(wide.to(device)[:, first:first + 990], tokens.to(device), top_k=4, output=output)
    assert result is output
    _check(result, values, tokens, 4)


def test_replays(device):
    values = torch.zeros(6, 32000, dtype=torch.bfloat16, device=device)
    tokens = torch.zeros(6, dtype=torch.int64, device=device)
    output = TokenLogprobs.allocate(rows=6, top_k=5, device=device)
    token_logprobs(values, tokens, top_k=5, output=output)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream(device)):
        token_logprobs(values, tokens, top_k=5, output=output)
    for step in range(3):
        generator = torch.Generator().manual_seed(step)
        values.copy_(2 * torch.randn(6, 32000, generator=generator))
        tokens.copy_(torch.randint(32000, (6,), generator=generator))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        eager = token_logprobs(values, tokens, top_k=5)
        for name in ("logprobs", "entropy", "top_logprobs", "top_tokens"):
            assert torch.equal(getattr(output, name), getattr(eager, name)), (step, name)


def test_refusals(device):
    values = torch.zeros(3, 50, device=device)
    tokens = torch.zeros(3, dtype=torch.int64, device=device)
    for top_k in (-1, 33, 51):
        with pytest.raises(ValueError, match="top_k"):
            token_logprobs(values, tokens, top_k=top_k)
    with pytest.raises(ValueError, match="top_k"):
        token_logprobs(values[:, :4], tokens, top_k=5)
    with pytest.raises(ValueError, match="empty row"):
        token_logprobs(values[:, :0], tokens)
    with pytest.raises(ValueError, match="contiguous rows"):
        token_logprobs(values.t(), tokens)
    with pytest.raises(TypeError, match="dtype"):
        token_logprobs(values.double(), tokens)
    with pytest.raises(ValueError, match="int64"):
        token_logprobs(values, tokens.int())
    with pytest.raises(ValueError, match="int64"):
        token_logprobs(values, tokens[:2])
    with pytest.raises(ValueError, match="output must hold"):
        token_logprobs(values, tokens, top_k=3, output=TokenLogprobs.allocate(rows=3, top_k=2, device=device))
    with pytest.raises(RuntimeError, match="inference-only"):
        token_logprobs(values.clone().requires_grad_(), tokens)
    assert token_logprobs(values[:0], tokens[:0], top_k=2).top_tokens.shape == (0, 2)
