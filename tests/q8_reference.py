"""The 8-bit cache, attention over it, 4-bit projections and log probabilities
from their definitions in 64 bits (numpy and torch on the CPU), and the error
bounds the tests hold the kernels to."""

from __future__ import annotations

import math

import numpy as np
import torch
from torch import Tensor

# Half a rounding step relative to the value.
HALF_STEP = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
# Below its smallest normal value 2^-14 fp16 keeps steps of 2^-24, so a
# rounding there is off by up to 2^-25 whatever the value (the other types'
# normal range goes down to 2^-126).
HALF_SUBNORMAL_STEP = {torch.float32: 0.0, torch.float16: 2.0**-25, torch.bfloat16: 0.0}
E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6])


def _e4m3(code: int) -> float:
    exponent, fraction = code >> 3 & 15, code & 7
    if code & 127 == 127:
        return math.nan
    size = math.ldexp(8 + fraction, exponent - 10) if exponent else math.ldexp(fraction, -9)
    return -size if code & 128 else size


E4M3 = np.array([_e4m3(code) for code in range(256)])


def encode_e4m3(x: np.ndarray) -> np.ndarray:
    """The code of the e4m3 value nearest to x (|x| <= 448, or NaN), ties to the even code."""

    positive = E4M3[:127]
    size = np.abs(x)
    above = np.minimum(np.searchsorted(positive, np.where(np.isnan(size), 0, size)), 126)
    below = np.maximum(above - 1, 0)
    up, down = positive[above] - size, size - positive[below]
    code = np.where((up < down) | ((up == down) & (above % 2 == 0)), above, below)
    code = np.where(np.isnan(x), 127, code)
    return (code | np.where(np.signbit(x), 128, 0)).astype(np.uint8)


def smallest_exponent(largest: float) -> int:
    t = -126
    if largest > 0:
        t = max(t, math.ceil(math.log2(largest / 448)) - 2)
        while largest > math.ldexp(448, t):
            t += 1
    return t


class CacheReference:
    """Token-major codes ``[blocks, heads, block_size, head_dim]`` of keys and
    values and their exponents ``[blocks, heads]``."""

    def __init__(self, blocks: int, heads: int, block_size: int, head_dim: int, seed: int | None = None) -> None:
        rng = np.random.default_rng(seed)
        shape = (2, blocks, heads, block_size, head_dim)
        self.codes = (rng.integers(0, 256, shape) if seed is not None else np.zeros(shape)).astype(np.uint8)
        self.exponents = (rng.integers(-9, 3, shape[:3]) if seed is not None else np.full(shape[:3], -126))

    def tensors(self, device) -> tuple[Tensor, Tensor, Tensor, Tensor]:
        codes = [torch.from_numpy(self.codes[0].copy()),
                 torch.from_numpy(np.ascontiguousarray(self.codes[1].swapaxes(2, 3)))]
        scales = [torch.from_numpy((e + 127).astype(np.uint8)) for e in self.exponents]
        return (*(c.to(device).view(torch.float8_e4m3fn) for c in codes),
                *(s.to(device).view(torch.float8_e8m0fnu) for s in scales))

    def values(self) -> np.ndarray:
        return E4M3[self.codes] * np.exp2(self.exponents.astype(np.float64))[..., None, None]

    def write(self, keys: Tensor, values: Tensor, blocks, offsets, active) -> None:
        """Runs of neighbouring rows at ascending offsets of a page."""

        count, _, size, _ = self.codes.shape[1:]
        rows = [r for r in range(len(blocks)) if active[r] and 0 <= blocks[r] < count and 0 <= offsets[r] < size]
        runs: list[list[int]] = []
        for r in rows:
            if runs and runs[-1][-1] == r - 1 and blocks[r] == blocks[r - 1] and offsets[r] == offsets[r - 1] + 1:
                runs[-1].append(r)
            else:
                runs.append([r])
        for side, new in enumerate((keys.double().numpy(), values.double().numpy())):
            for run in runs:
                block, first = blocks[run[0]], offsets[run[0]]
                for head in range(new.shape[1]):
                    x = new[run, head]
                    finite = np.where(np.isfinite(x), np.abs(x), 0)
                    t = smallest_exponent(float(finite.max()))
                    page = self.codes[side, block, head]
                    if first > 0:
                        old = int(self.exponents[side, block, head])
                        t = max(t, old)
                        if t > old:
                            page[:] = encode_e4m3(E4M3[page] * 2.0 ** (old - t))
                    self.exponents[side, block, head] = t
                    scaled = np.where(np.isfinite(x), x, np.nan) * 2.0 ** -t
                    page[first:first + len(run)] = encode_e4m3(scaled)


def same_codes(got: Tensor, want: np.ndarray) -> bool:
    """Equal codes; any NaN code stands for any other, -0 for 0 never."""

    got = got.view(torch.uint8).cpu().numpy()
    return bool(((got == want) | ((got & 127 == 127) & (want & 127 == 127))).all())


def attention(query: Tensor, reference: CacheReference, tables, lengths, scale: float) -> tuple[Tensor, Tensor]:
    """(outputs, error bounds) in 64 bits.

    The bound: the weights p are rounded to the products' operands (bf16 once
    for bf16 queries, in two or three bf16 parts for fp16 and fp32), a score in
    fp32 is off by at most (D + 4) 2^-24 of its terms' size and shifts p by as
    much (times two with the maximum's), the exponential and its argument
    (|s| 2^-23), the sums add at most one rounding a token, the output one."""

    q = query.double().cpu().numpy()
    rows, heads, dim = q.shape
    blocks, kv_heads, size, _ = reference.codes.shape[1:]
    values = reference.values()
    out, bound = np.zeros_like(q), np.zeros_like(q)
    weight_step = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-16, torch.float32: 2.0**-22}[query.dtype]
    for r in range(rows):
        pages = [(int(tables[r][j]), min(size, lengths[r] - j * size)) for j in range(-(-max(lengths[r], 0) // size))]
        pages = [(page, n) for page, n in pages if 0 <= page < blocks]
        if not pages:
            continue
        for h in range(heads):
            kv = h * kv_heads // heads
            k, v = (np.concatenate([values[side, page, kv, :n] for page, n in pages]) for side in (0, 1))
            s = k @ q[r, h] * scale
            p = np.exp(s - s.max())
            p /= p.sum()
            out[r, h] = p @ v
            size_s = (np.abs(k) @ np.abs(q[r, h])).max() * abs(scale)
            relative = weight_step + 2 * (dim + 4) * 2.0**-24 * size_s + 2.0**-21 * (1 + np.abs(s).max()) + (
                len(p) + 64) * 2.0**-24
            bound[r, h] = relative * (p @ np.abs(v)) * 2
    out_t = torch.from_numpy(out)
    return out_t, torch.from_numpy(bound) + HALF_STEP[query.dtype] * out_t.abs() + (
        HALF_SUBNORMAL_STEP[query.dtype] + 1e-30)


def mxfp4_weight(codes: Tensor, scales: Tensor) -> np.ndarray:
    packed = codes.cpu().numpy()
    n, half = packed.shape
    weight = np.stack((E2M1[packed & 15], E2M1[packed >> 4]), -1).reshape(n, 2 * half)
    return weight * np.repeat(np.exp2(scales.view(torch.uint8).cpu().numpy().astype(np.float64) - 127), 32, 1)


def linear(x: Tensor, codes: Tensor, scales: Tensor, residual: Tensor | None) -> tuple[Tensor, Tensor]:
    """(outputs, error bounds): exact products, at most one rounding a term in the fp32 sums, one of the result and
    one of the residual sum."""

    weight = mxfp4_weight(codes, scales)
    x64 = x.double().cpu().numpy()
    y = torch.from_numpy(x64 @ weight.T)
    half = HALF_STEP[x.dtype]
    bound = half * y.abs() + 2.0**-24 * x.shape[1] * torch.from_numpy(np.abs(x64) @ np.abs(weight).T) * (1 + half)
    bound = bound + HALF_SUBNORMAL_STEP[x.dtype]
    if residual is not None:
        y = y + residual.double().cpu()
        bound = bound + half * (y.abs() + bound)
    return y, bound


def logprobs(logits: Tensor, tokens: Tensor, top_k: int):
    """(logprobs, entropy, top logprobs, top tokens, bound of a log probability, bound of the entropy).

    In fp32: x - m and log S round once each, exp is good to 2^-22 with its
    argument's rounding |d| 2^-24 in each term, and a sum of n terms over at
    least 256 lanes adds n / 256 + 16 roundings to S and to the entropy's sum."""

    x = logits.double().cpu()
    columns = x.shape[1]
    lp = torch.log_softmax(x, -1)
    p = lp.exp()
    entropy = -torch.where(p == 0, 0, p * lp).sum(-1)  # NaN stays NaN
    order = torch.sort(torch.where(x.isnan(), torch.inf, x) , dim=-1, descending=True, stable=True).indices
    if bool(x.isnan().any()):
        keys = [sorted(range(columns), key=lambda c: (not math.isnan(row[c]), -row[c] if not math.isnan(row[c]) else 0, c))
                for row in x.tolist()]
        order = torch.tensor(keys)
    top = order[:, :top_k]
    tokens = tokens.cpu()
    inside = (tokens >= 0) & (tokens < columns)
    given = torch.where(inside, lp.gather(1, tokens.clamp(0, columns - 1)[:, None])[:, 0], torch.nan)
    shifted = x - x.amax(-1, keepdim=True)
    mean = -(torch.where(p == 0, 0, shifted * p).sum(-1))
    sums = 2.0**-21 * (1 + mean) + (columns / 256 + 16) * 2.0**-24
    spread = shifted.abs().where(torch.isfinite(shifted), torch.zeros(())).amax(-1)
    log_sum = torch.logsumexp(shifted, -1)
    lp_bound = 2.0**-22 * (spread + log_sum) + 2 * sums
    entropy_bound = 2.0**-22 * (log_sum + mean) + 2 * sums * (1 + mean + 2)
    return given, entropy, lp.gather(1, top), top, lp_bound, entropy_bound
