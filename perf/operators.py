"""Performance cases of the operators on 8-bit and 4-bit state, and of token log probabilities: inputs, one pass in its
plain form or through the framework, the work a pass cannot do without and the same outputs in 64 bits.

A case's ``kind`` names the operator:

  cache      new tokens appended to an 8-bit paged cache, then token rows read back as values
  attention  paged GQA decode attention over an 8-bit cache
  linear     a projection of a decode step by 4-bit weights
  logprobs   log probabilities of given tokens, with entropy and the top alternatives

Formats.  Cache: e4m3 codes, keys ``[pages, kv_heads, page, head_dim]`` and values ``[pages, kv_heads, head_dim, page]``,
with a power-of-two scale (e8m0) for each page and head; a page's scale is the smallest that holds its finite values, it
begins anew with the token at offset 0, and where a later token raises it the page's codes are rounded to the new one.
Weights: e2m1 codes ``[n, k / 2]`` (the even column in the low half) with an e8m0 scale for each 32 columns.

New tokens of a cache case are written out per sequence (64 lanes of one: "1*64"); context lengths of decode rows are
drawn from the seed.
"""

from __future__ import annotations

import math
import random

import torch
from torch import Tensor

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
DEVICE = "cuda"
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
LOWEST_EXPONENT = -126
# 19 prompts of one admission of the serving workload (lognormal, median 256, clipped to [16, 2048]).
ADMISSION = "262,218,421,279,98,331,733,553,145,93,158,263,39,215,95,142,1661,304,2048"


def listed() -> list[dict]:
    return [
        # A full batch's append in one layer of a decode step, eight padded lanes; the pages written are read back.
        {"name": "append_b64", "kind": "cache", "new": "1*64", "prefix": 700, "padded": 8, "read": "page",
         "kv_heads": 4, "head_dim": 64, "page": 16, "dtype": "bf16"},
        # Chunks of three prompts that continue inside a page, and all their tokens read for the chunks' attention.
        {"name": "append_chunks", "kind": "cache", "new": "509,261,130", "prefix": 700, "padded": 0, "read": "all",
         "kv_heads": 8, "head_dim": 128, "page": 16, "dtype": "fp16"},
        # A whole admission's tokens in one layer.
        {"name": "append_admission", "kind": "cache", "new": ADMISSION, "prefix": 0, "padded": 0, "read": "all",
         "kv_heads": 4, "head_dim": 64, "page": 16, "dtype": "bf16"},
        # One request alone: latency.
        {"name": "attention_b1", "kind": "attention", "rows": 1, "padded": 0, "low": 300, "high": 300,
         "query_heads": 32, "kv_heads": 4, "head_dim": 64, "page": 16, "dtype": "bf16"},
        # The headline batch: 64 ragged rows and 8 padded ones.
        {"name": "attention_b64", "kind": "attention", "rows": 64, "padded": 8, "low": 128, "high": 2048,
         "query_heads": 32, "kv_heads": 4, "head_dim": 64, "page": 16, "dtype": "bf16"},
        # Long contexts, few rows.
        {"name": "attention_long", "kind": "attention", "rows": 4, "padded": 0, "low": 8192, "high": 32768,
         "query_heads": 32, "kv_heads": 8, "head_dim": 128, "page": 16, "dtype": "fp16"},
        # Full precision queries over the 8-bit cache.
        {"name": "attention_fp32", "kind": "attention", "rows": 32, "padded": 0, "low": 64, "high": 2048,
         "query_heads": 32, "kv_heads": 4, "head_dim": 64, "page": 16, "dtype": "fp32"},
        # The down projection of one request, added to its residual.
        {"name": "linear_b1", "kind": "linear", "rows": 1, "n": 2048, "k": 5632, "residual": True, "dtype": "bf16"},
        # A wide gate|up projection for a few requests.
        {"name": "linear_b8", "kind": "linear", "rows": 8, "n": 28672, "k": 4096, "residual": False, "dtype": "fp16"},
        # The gate|up projection of a full batch.
        {"name": "linear_b64", "kind": "linear", "rows": 64, "n": 11264, "k": 2048, "residual": False, "dtype": "bf16"},
        # The sampled tokens of a decode step, with five alternatives each.
        {"name": "logprobs_b64", "kind": "logprobs", "rows": 64, "columns": 32000, "top_k": 5, "dtype": "bf16"},
        # A prompt's tokens scored.
        {"name": "logprobs_prompt", "kind": "logprobs", "rows": 2048, "columns": 32000, "top_k": 20, "dtype": "bf16"},
    ]


def _log_uniform(rng: random.Random, low: int, high: int) -> int:
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(["cache", "attention", "attention", "linear", "linear", "logprobs"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    query_heads, kv_heads, head_dim = rng.choice([(32, 4, 64), (32, 8, 128), (8, 2, 32), (12, 3, 96), (16, 16, 64)])
    if kind == "cache":
        page = rng.choice([16, 16, 32])
        if rng.random() < 0.4:
            return {"kind": kind, "new": f"1*{_log_uniform(rng, 1, 256)}", "prefix": rng.randint(0, 2000),
                    "padded": rng.choice([0, 3]), "read": "page", "kv_heads": kv_heads, "head_dim": head_dim,
                    "page": page, "dtype": dtype}
        most = 2_000_000 // (kv_heads * head_dim)
        total = _log_uniform(rng, 16, most)
        count = rng.randint(1, min(16, total))
        cuts = sorted(rng.sample(range(1, total), count - 1)) if count > 1 else []
        lengths = [b - a for a, b in zip([0, *cuts], [*cuts, total])]
        return {"kind": kind, "new": ",".join(map(str, lengths)), "prefix": rng.choice([0, 0, rng.randint(1, 60)]),
                "padded": 0, "read": "all", "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "dtype": dtype}
    if kind == "attention":
        rows = _log_uniform(rng, 1, 64)
        most = (160 << 20) // (rows * kv_heads * head_dim * 2)
        high = _log_uniform(rng, 1, max(2, min(32768, most)))
        return {"kind": kind, "rows": rows, "padded": rng.choice([0, 0, 3]), "low": max(1, high // 16), "high": high,
                "query_heads": query_heads, "kv_heads": kv_heads, "head_dim": head_dim, "page": rng.choice([16, 16, 32]),
                "dtype": dtype}
    if kind == "linear":
        n, k = rng.choice([(2560, 2048), (2048, 2048), (11264, 2048), (2048, 5632), (32000, 2048), (6144, 4096),
                           (4096, 4096), (28672, 4096), (4096, 14336),
                           (_log_uniform(rng, 16, 16384), 32 * _log_uniform(rng, 1, 256))])
        most = max(1, min(64, 4_600_000_000 // (n * k)))
        return {"kind": kind, "rows": _log_uniform(rng, 1, most), "n": n, "k": k, "residual": rng.random() < 0.3,
                "dtype": rng.choice(["bf16", "fp16"])}
    columns = rng.choice([32000, _log_uniform(rng, 64, 131072)])
    size = 4 if dtype == "fp32" else 2
    return {"kind": kind, "rows": _log_uniform(rng, 1, max(2, min(2048, (130 << 20) // (columns * size)))),
            "columns": columns, "top_k": rng.choice([0, 1, 5, 20, 32]), "dtype": dtype}


# -- inputs -------------------------------------------------------------------------------------------------------------


def _generator(seed: int) -> torch.Generator:
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _new_lengths(case: dict) -> list[int]:
    parts = (part.partition("*") for part in case["new"].split(","))
    return [int(length) for length, _, times in parts for _ in range(int(times or 1))]


def _starts(case: dict) -> tuple[list[int], list[int]]:
    """Each sequence's tokens before the append, and the first one that is read: the same for every seed."""

    rng = random.Random(case["prefix"])
    starts = [rng.randint(0, case["prefix"]) for _ in _new_lengths(case)]
    return starts, [start // case["page"] * case["page"] if case["read"] == "page" else 0 for start in starts]


def _row_lengths(case: dict, seed: int) -> list[int]:
    """Context lengths of a decode call's rows: uniform, the longest one present."""

    rng = random.Random(seed)
    lengths = [rng.randint(case["low"], case["high"]) for _ in range(case["rows"])]
    lengths[rng.randrange(case["rows"])] = case["high"]
    return lengths


def _tables(lengths: list[int], page: int, width: int, rng: random.Random) -> tuple[Tensor, int]:
    """Block tables over a permuted pool of exactly the pages the rows need."""

    counts = [-(-n // page) for n in lengths]
    pool = max(sum(counts), 1)
    order = list(range(pool))
    rng.shuffle(order)
    tables = torch.full((len(lengths), width), -1, dtype=torch.int32)
    at = 0
    for row, count in enumerate(counts):
        tables[row, :count] = torch.tensor(order[at:at + count], dtype=torch.int32)
        at += count
    return tables, pool


def _smallest_exponent(largest: Tensor) -> Tensor:
    """The smallest t >= -126 with largest <= 448 * 2^t (448 = 0.875 * 2^9)."""

    mantissa, exponent = torch.frexp(largest)
    t = exponent - 9 + (mantissa > 0.875)
    return torch.where(largest > 0, t, LOWEST_EXPONENT).clamp(min=LOWEST_EXPONENT)


def _page_codes(generator: torch.Generator, pool: int, heads: int, page: int, dim: int) -> tuple[Tensor, Tensor]:
    """e4m3 codes ``[pool, heads, page, dim]`` of normal values whose channels differ in size, and their scales."""

    channels = torch.exp(0.5 * torch.randn(heads, 1, dim, generator=generator, device=DEVICE))
    values = torch.randn(pool, heads, page, dim, generator=generator, device=DEVICE) * channels
    exponents = _smallest_exponent(values.abs().amax((-2, -1)))
    codes = torch.ldexp(values, -exponents[..., None, None]).to(torch.float8_e4m3fn)
    return codes, (exponents + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _cache(generator: torch.Generator, pool: int, heads: int, page: int, dim: int) -> dict:
    key, key_scales = _page_codes(generator, pool, heads, page, dim)
    value, value_scales = _page_codes(generator, pool, heads, page, dim)
    return {"key": key, "value": value.transpose(2, 3).contiguous(), "key_scales": key_scales,
            "value_scales": value_scales}


def prepare(case: dict, seed: int) -> dict:
    return {"kind": case["kind"], **globals()["_prepare_" + case["kind"]](case, seed)}


def _prepare_cache(case: dict, seed: int) -> dict:
    dtype, page = DTYPES[case["dtype"]], case["page"]
    new, (starts, first_read) = _new_lengths(case), _starts(case)
    lengths = [start + n for start, n in zip(starts, new)]
    tables, pool = _tables(lengths, page, -(-max(lengths) // page), random.Random(seed))
    generator = _generator(seed + 1)
    total, padded = sum(new), case["padded"]

    def slots(first: list[int]) -> tuple[Tensor, Tensor]:
        positions = torch.cat([torch.arange(a, b) for a, b in zip(first, lengths)])
        rows = torch.cat([torch.full((b - a,), row) for row, (a, b) in enumerate(zip(first, lengths))])
        return tables[rows, positions // page].to(torch.int32), (positions % page).to(torch.int32)

    blocks, offsets = slots(starts)
    read = slots(first_read)
    lanes = torch.zeros(padded, dtype=torch.int32)
    shape = (total + padded, case["kv_heads"], case["head_dim"])
    return {
        **_cache(generator, pool, case["kv_heads"], page, case["head_dim"]),
        "keys": torch.randn(shape, generator=generator, device=DEVICE).to(dtype),
        "values": torch.randn(shape, generator=generator, device=DEVICE).to(dtype),
        "blocks": torch.cat((blocks, lanes)).to(DEVICE), "offsets": torch.cat((offsets, lanes)).to(DEVICE),
        "active": torch.cat((torch.ones(total, dtype=torch.int32), lanes)).to(DEVICE),
        "read_blocks": read[0].to(DEVICE), "read_offsets": read[1].to(DEVICE),
        "key_output": torch.empty((read[0].numel(), *shape[1:]), dtype=dtype, device=DEVICE),
        "value_output": torch.empty((read[0].numel(), *shape[1:]), dtype=dtype, device=DEVICE),
    }


def _prepare_attention(case: dict, seed: int) -> dict:
    dtype, page, heads, dim = DTYPES[case["dtype"]], case["page"], case["query_heads"], case["head_dim"]
    lengths = _row_lengths(case, seed) + [0] * case["padded"]
    width = -(-case["high"] // page)
    tables, pool = _tables(lengths, page, width, random.Random(seed))
    generator = _generator(seed + 1)
    query = torch.randn(len(lengths), heads, dim, generator=generator, device=DEVICE).to(dtype)
    splits = max(-(-width * page // 64), 1)  # partial sums for as many partitions as a narrow call may take
    rows = len(lengths) * heads * min(splits, max(1, 4096 // len(lengths)))
    return {
        **_cache(generator, pool, case["kv_heads"], page, dim), "query": query, "tables": tables.to(DEVICE),
        "contexts": torch.tensor(lengths, dtype=torch.int32, device=DEVICE), "capacity": width * page,
        "output": torch.empty_like(query),
        "partial_max": torch.empty(rows, device=DEVICE), "partial_sum": torch.empty(rows, device=DEVICE),
        "partial_accumulator": torch.empty(rows, 1 << (dim - 1).bit_length(), device=DEVICE),
    }


def _prepare_linear(case: dict, seed: int) -> dict:
    """Normal weights rounded to e2m1 under the exponent of each group's largest less two."""

    dtype, generator = DTYPES[case["dtype"]], _generator(seed)
    rows, n, k = case["rows"], case["n"], case["k"]
    weight = 0.02 * torch.randn(n, k // 32, 32, generator=generator, device=DEVICE)
    exponents = torch.frexp(weight.abs().amax(-1))[1] - 3
    size = torch.ldexp(weight.abs(), -exponents[..., None])
    codes = sum((size > (low + high) / 2).to(torch.uint8) for low, high in zip(E2M1, E2M1[1:]))
    codes = (codes + 8 * (weight < 0).to(torch.uint8)).view(n, k // 2, 2)
    return {
        "x": torch.randn(rows, k, generator=generator, device=DEVICE).to(dtype),
        "weight": codes[..., 0] | (codes[..., 1] << 4),
        "scales": (exponents + 127).to(torch.uint8).view(torch.float8_e8m0fnu),
        "residual": torch.randn(rows, n, generator=generator, device=DEVICE).to(dtype) if case["residual"] else None,
        "table": torch.tensor([*E2M1, *(-v for v in E2M1)], device=DEVICE),
        "output": torch.empty(rows, n, dtype=dtype, device=DEVICE),
    }


def _prepare_logprobs(case: dict, seed: int) -> dict:
    generator = _generator(seed)
    rows, columns, top_k = case["rows"], case["columns"], case["top_k"]
    return {
        "logits": (2.5 * torch.randn(rows, columns, generator=generator, device=DEVICE)).to(DTYPES[case["dtype"]]),
        "tokens": torch.randint(columns, (rows,), generator=generator, device=DEVICE),
        "top_k": top_k,
    }


# -- one pass -----------------------------------------------------------------------------------------------------------


def run(state: dict):
    if own:
        return globals()["_run_" + state["kind"]](state)
    return globals()["_plain_" + state["kind"]](state)


def _handle(state: dict):
    from tensorforge_amd.kernels import PagedKVCacheQ8

    return PagedKVCacheQ8(state["key"], state["value"], state["key_scales"], state["value_scales"])


def _run_cache(state: dict) -> dict:
    from tensorforge_amd.kernels import paged_kv_read_token_q8, paged_kv_write_token_q8

    cache = _handle(state)
    paged_kv_write_token_q8(state["keys"], state["values"], cache, state["blocks"], state["offsets"], state["active"])
    keys, values = paged_kv_read_token_q8(cache, state["read_blocks"], state["read_offsets"],
                                          key_output=state["key_output"], value_output=state["value_output"])
    return {"keys": keys, "values": values}


def _run_attention(state: dict) -> Tensor:
    from tensorforge_amd.kernels import PagedAttentionWorkspace, paged_gqa_decode_attention_q8

    workspace = PagedAttentionWorkspace(state["partial_max"], state["partial_sum"], state["partial_accumulator"])
    return paged_gqa_decode_attention_q8(state["query"], _handle(state), state["tables"], state["contexts"],
                                         max_context_length=state["capacity"], output=state["output"],
                                         workspace=workspace)


def _run_linear(state: dict) -> Tensor:
    from tensorforge_amd.kernels import linear_mxfp4

    return linear_mxfp4(state["x"], state["weight"], state["scales"], residual=state["residual"], output=state["output"])


def _run_logprobs(state: dict) -> dict:
    from tensorforge_amd.kernels import token_logprobs

    result = token_logprobs(state["logits"], state["tokens"], top_k=state["top_k"])
    return {"logprobs": result.logprobs, "entropy": result.entropy, "top_logprobs": result.top_logprobs,
            "top_tokens": result.top_tokens}


def _exponents(scales: Tensor) -> Tensor:
    return scales.view(torch.uint8).to(torch.int32) - 127


def _values(codes: Tensor) -> Tensor:
    return codes.view(torch.float8_e4m3fn).float()


def _plain_append(codes: Tensor, scales: Tensor, rows: Tensor, blocks: Tensor, offsets: Tensor) -> Tensor:
    """The values ``[pages + 1, page, heads, dim]`` of a cache (its codes token-major) after the append of ``rows``;
    inactive rows are sent to a page behind the last."""

    pool, heads = scales.shape
    x = rows.float()
    finite = torch.isfinite(x)
    needed = _smallest_exponent(torch.where(finite, x.abs(), 0).amax(-1)).to(torch.int32)
    old = torch.cat((_exponents(scales), torch.zeros(1, heads, dtype=torch.int32, device=x.device)))
    at = blocks.to(torch.int64)
    index = at[:, None].expand(-1, heads)
    most = torch.full_like(old, LOWEST_EXPONENT).scatter_reduce(0, index, needed, "amax")
    touched = torch.zeros(pool + 1, dtype=torch.int32, device=x.device).index_fill(0, at, 1)[:, None] > 0
    begun = torch.zeros(pool + 1, dtype=torch.int32, device=x.device).scatter_reduce(
        0, at, (offsets == 0).to(torch.int32), "amax")[:, None] > 0
    new = torch.where(touched, torch.where(begun, most, torch.maximum(old, most)), old)
    kept = torch.cat((codes.float(), torch.zeros_like(codes[:1], dtype=torch.float32)))
    lower = torch.where(begun, 0, old - new)[:, None, :, None]
    kept = torch.ldexp(kept, lower).to(torch.float8_e4m3fn).float()
    added = torch.where(finite, torch.ldexp(x, -new[at][..., None]), torch.nan).to(torch.float8_e4m3fn).float()
    kept[at, offsets.to(torch.int64)] = added
    return torch.ldexp(kept, new[:, None, :, None])


def _plain_cache(state: dict) -> dict:
    pool = state["key"].shape[0]
    blocks = torch.where(state["active"] != 0, state["blocks"], pool)
    key = _plain_append(state["key"].transpose(1, 2), state["key_scales"], state["keys"], blocks, state["offsets"])
    value = _plain_append(state["value"].permute(0, 3, 1, 2), state["value_scales"], state["values"], blocks,
                          state["offsets"])
    at = state["read_blocks"].to(torch.int64), state["read_offsets"].to(torch.int64)
    return {"keys": key[at].to(state["keys"].dtype), "values": value[at].to(state["values"].dtype)}


def _plain_attention(state: dict) -> Tensor:
    query, key, value = state["query"], state["key"], state["value"]
    rows, heads, dim = query.shape
    pool, kv_heads, page, _ = key.shape
    valid = (state["tables"] >= 0) & (state["tables"] < pool)
    at = state["tables"].clamp(0, pool - 1).to(torch.int64)
    k = torch.ldexp(_values(key.view(torch.uint8)[at]), _exponents(state["key_scales"])[at][..., None, None])
    v = torch.ldexp(_values(value.view(torch.uint8)[at]), _exponents(state["value_scales"])[at][..., None, None])
    k = k.permute(0, 2, 4, 1, 3).reshape(rows, kv_heads, dim, -1)
    v = v.permute(0, 2, 1, 4, 3).reshape(rows, kv_heads, -1, dim)
    scores = torch.matmul(query.float().view(rows, kv_heads, heads // kv_heads, dim), k) * dim**-0.5
    tokens = torch.arange(scores.shape[-1], device=query.device)
    seen = valid.repeat_interleave(page, 1) & (tokens < state["contexts"][:, None])
    seen = seen[:, None, None, :]
    scores = torch.where(seen, scores, -torch.inf)
    largest = scores.amax(-1, keepdim=True)
    p = torch.where(seen, torch.exp(scores - torch.where(torch.isinf(largest), 0, largest)), 0)
    total = p.sum(-1, keepdim=True)
    v = torch.where(seen[:, :, 0, :, None], v, 0)
    out = torch.matmul(p, v) / torch.where(total == 0, 1, total)
    return out.reshape(rows, heads, dim).to(query.dtype)


def _plain_linear(state: dict) -> Tensor:
    x, packed = state["x"], state["weight"]
    n, k = packed.shape[0], x.shape[1]
    codes = torch.stack((packed & 15, packed >> 4), -1).view(n, k // 32, 32)
    weight = torch.ldexp(state["table"][codes.to(torch.int32)], _exponents(state["scales"])[..., None]).view(n, k)
    y = torch.matmul(x.float(), weight.t()).to(x.dtype)
    if state["residual"] is None:
        return y
    return (y.float() + state["residual"].float()).to(x.dtype)


def _plain_logprobs(state: dict) -> dict:
    x = state["logits"].float()
    shifted = x - x.amax(-1, keepdim=True)
    weights = torch.exp(shifted)
    total = weights.sum(-1, keepdim=True)
    logprobs = shifted - torch.log(total)
    entropy = torch.log(total[:, 0]) - torch.where(weights > 0, shifted * weights, 0).sum(-1) / total[:, 0]
    top = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :state["top_k"]]
    return {"logprobs": logprobs.gather(1, state["tokens"][:, None])[:, 0], "entropy": entropy,
            "top_logprobs": logprobs.gather(1, top), "top_tokens": top}


# -- the work of a pass -------------------------------------------------------------------------------------------------


def work(case: dict) -> dict:
    size = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "linear":
        m, n, k = case["rows"], case["n"], case["k"]
        nbytes = n * k / 2 + n * k / 32 + size * (m * k + m * n * (2 if case["residual"] else 1))
        return {"bytes": nbytes, "flops": 2 * m * n * k}
    if case["kind"] == "logprobs":
        rows = case["rows"]
        return {"bytes": rows * (case["columns"] * size + 8 + 8 + 12 * case["top_k"]), "flops": 6 * rows * case["columns"]}
    width = case["kv_heads"] * case["head_dim"]
    if case["kind"] == "cache":
        # The new rows read and written as codes, the rows read back; the control vectors.
        new, (starts, first_read) = _new_lengths(case), _starts(case)
        read = sum(new) + sum(starts) - sum(first_read)
        return {"bytes": 2 * width * (size + 1) * (sum(new) + read) + 12 * sum(new) + 8 * read,
                "flops": 2 * width * (sum(new) + read)}
    tokens = case["high"] + (case["rows"] - 1) * (case["low"] + case["high"]) / 2
    queries = (case["rows"] + case["padded"]) * case["query_heads"] * case["head_dim"]
    pages = tokens / case["page"]
    return {"bytes": 2 * tokens * width + pages * (4 + 2 * case["kv_heads"]) + 2 * queries * size,
            "flops": 4 * tokens * case["query_heads"] * case["head_dim"]}


# -- the outputs in 64 bits ---------------------------------------------------------------------------------------------


def exact(case: dict, seed: int):
    state = prepare(case, seed)
    return globals()["_exact_" + case["kind"]](case, state)


def _code_values() -> Tensor:
    """The 256 values of e4m3: sign, four exponent bits of bias 7, three bits of fraction, 0x7f a NaN."""

    def value(code: int) -> float:
        exponent, fraction = code >> 3 & 15, code & 7
        size = math.nan if code & 127 == 127 else (
            math.ldexp(8 + fraction, exponent - 10) if exponent else math.ldexp(fraction, -9))
        return -size if code & 128 else size

    return torch.tensor([value(code) for code in range(256)], dtype=torch.float64, device=DEVICE)


def _decoded(codes: Tensor, scales: Tensor) -> Tensor:
    values = _code_values()[codes.view(torch.uint8).to(torch.int64)]
    return values * torch.exp2(scales.view(torch.uint8).double() - 127)[..., None, None]


def _nearest_code(x: Tensor) -> Tensor:
    """The e4m3 value nearest to x (|x| <= 448), ties to the even code."""

    positive = _code_values()[:127]
    size = x.abs()
    above = torch.searchsorted(positive, size.contiguous()).clamp(max=126)
    below = (above - 1).clamp(min=0)
    up, down = positive[above] - size, size - positive[below]
    pick = torch.where((up < down) | ((up == down) & (above % 2 == 0)), above, below)
    return torch.copysign(positive[pick], x)


def _exact_cache(case: dict, state: dict) -> dict:
    blocks, offsets, active = (state[name].tolist() for name in ("blocks", "offsets", "active"))
    pages: dict[int, list[int]] = {}
    for row, (block, on) in enumerate(zip(blocks, active)):
        if on:
            pages.setdefault(block, []).append(row)
    if len(pages) > 4000:
        return None
    outputs = {}
    for name, rows in (("keys", "keys"), ("values", "values")):
        codes = state["key"] if name == "keys" else state["value"].transpose(2, 3)
        scales = state["key_scales" if name == "keys" else "value_scales"]
        content = _decoded(codes.contiguous(), scales).transpose(1, 2).contiguous()  # [pages, page, heads, dim]
        bytes_ = scales.view(torch.uint8).cpu()
        new = state[rows].double()
        largest = new.abs().amax(-1).cpu()
        for block, members in pages.items():
            begins = any(offsets[row] == 0 for row in members)
            step = []
            for head in range(new.shape[1]):
                most = max(float(largest[row, head]) for row in members)
                t = LOWEST_EXPONENT
                if most > 0:
                    t = max(t, math.ceil(math.log2(most / 448)) - 2)
                    while most > math.ldexp(448, t):
                        t += 1
                step.append(t if begins else max(t, int(bytes_[block, head]) - 127))
            unit = torch.tensor([math.ldexp(1.0, t) for t in step], dtype=torch.float64, device=DEVICE)[:, None]
            if not begins:
                content[block] = _nearest_code(content[block] / unit) * unit
            at = torch.tensor([offsets[row] for row in members], device=DEVICE)
            content[block, at] = _nearest_code(new[torch.tensor(members, device=DEVICE)] / unit) * unit
        outputs[name] = content[state["read_blocks"].long(), state["read_offsets"].long()]
    return outputs


def _exact_attention(case: dict, state: dict) -> Tensor:
    query = state["query"].double()
    rows, heads, dim = query.shape
    kv_heads, page = case["kv_heads"], case["page"]
    out = torch.zeros_like(query)
    for row, length in enumerate(state["contexts"].tolist()):
        if not length:
            continue
        at = state["tables"][row, :-(-length // page)].long()
        for head in range(kv_heads):
            group = slice(head * heads // kv_heads, (head + 1) * heads // kv_heads)
            key, value, key_scales, value_scales = (
                state[name].view(torch.uint8)[at, head] for name in ("key", "value", "key_scales", "value_scales"))
            k = _decoded(key, key_scales).reshape(-1, dim)[:length]
            v = _decoded(value, value_scales)
            v = v.transpose(1, 2).reshape(-1, dim)[:length]
            p = torch.softmax(query[row, group] @ k.t().contiguous() / math.sqrt(dim), -1)
            out[row, group] = p @ v
    return out


def _exact_linear(case: dict, state: dict) -> Tensor:
    x, packed = state["x"].double(), state["weight"].to(torch.int64)
    n, k = packed.shape[0], x.shape[1]
    weight = torch.empty(n, k, dtype=torch.float64, device=DEVICE)
    for half in range(2):
        code = packed >> (4 * half) & 15
        exponent, fraction = (code >> 1 & 3).double(), (code & 1).double()
        size = torch.where(exponent > 0, torch.exp2(exponent - 1) * (1 + fraction / 2), fraction / 2)
        weight[:, half::2] = torch.where(code > 7, -size, size)
    weight *= torch.exp2(state["scales"].view(torch.uint8).double() - 127).repeat_interleave(32, 1)
    y = x @ weight.t().contiguous()
    return y if state["residual"] is None else y + state["residual"].double()


def _exact_logprobs(case: dict, state: dict) -> dict:
    x = state["logits"].double()
    logprobs = torch.log_softmax(x, -1)
    entropy = -(logprobs.exp() * logprobs).sum(-1)
    top = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :state["top_k"]]
    return {"logprobs": logprobs.gather(1, state["tokens"][:, None])[:, 0], "entropy": entropy,
            "top_logprobs": logprobs.gather(1, top), "top_tokens": top}
