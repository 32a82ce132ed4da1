"""The 8-bit cache, the 4-bit projections and the log probabilities without a
GPU: refusals of the Python entry points and of the C ABI (no call here
reaches a launch), and the weight quantisation."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tensorforge_amd import _native
from tensorforge_amd.kernels import (
    PagedKVCacheQ8,
    TokenLogprobs,
    linear_mxfp4,
    paged_gqa_decode_attention_q8,
    paged_kv_read_token_q8,
    paged_kv_write_token_q8,
    quantize_mxfp4,
    token_logprobs,
)
from tests.q8_reference import mxfp4_weight

FAKE = 0x1000  # never dereferenced


def _cache(blocks=3, block_size=16, kv_heads=2, head_dim=32):
    return PagedKVCacheQ8.allocate(num_blocks=blocks, block_size=block_size, kv_heads=kv_heads, head_dim=head_dim,
                                   device=torch.device("cpu"))


def test_cache_allocation_and_sizes():
    cache = _cache()
    assert (cache.num_blocks, cache.kv_heads, cache.block_size, cache.head_dim) == (3, 2, 16, 32)
    assert cache.value.shape == (3, 2, 32, 16)
    assert not cache.key.float().any() and torch.equal(cache.key_scales.float(), torch.full((3, 2), 2.0**-126))


@pytest.mark.parametrize(("sizes", "message"), [
    ({"head_dim": 24}, "multiples of 16"), ({"head_dim": 272}, "multiples of 16"), ({"head_dim": 0}, "multiples of 16"),
    ({"block_size": 8}, "multiple of 16 tokens"), ({"block_size": 1040}, "multiple of 16 tokens"),
    ({"blocks": 0}, "positive"),
])
def test_cache_refuses_sizes(sizes, message):
    with pytest.raises(ValueError, match=message):
        _cache(**sizes)


def test_cache_refuses_tensors():
    cache = _cache()
    key, value, ks, vs = cache.key, cache.value, cache.key_scales, cache.value_scales
    with pytest.raises(ValueError, match="value codes"):
        PagedKVCacheQ8(key, key, ks, vs)
    with pytest.raises(TypeError, match="e4m3fn"):
        PagedKVCacheQ8(key.view(torch.uint8), value, ks, vs)
    with pytest.raises(ValueError, match="scales"):
        PagedKVCacheQ8(key, value, ks[:, :1], vs)
    with pytest.raises(TypeError, match="e8m0fnu"):
        PagedKVCacheQ8(key, value, ks.view(torch.uint8), vs)
    with pytest.raises(ValueError, match="contiguous"):
        PagedKVCacheQ8(key, value.view(torch.uint8).transpose(2, 3).contiguous().transpose(2, 3)
                       .view(torch.float8_e4m3fn), ks, vs)
    flat = torch.zeros(3 * 2 * 16 * 32 + 1, dtype=torch.uint8)
    with pytest.raises(ValueError, match="16-byte"):
        PagedKVCacheQ8(flat[1:].view(3, 2, 16, 32).view(torch.float8_e4m3fn), value, ks, vs)


def test_entry_points_refuse_cpu_tensors():
    cache = _cache()
    rows = torch.zeros(2, 2, 32)
    control = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        paged_kv_write_token_q8(rows, rows, cache, control, control, control)
    with pytest.raises(ValueError, match="CUDA"):
        paged_kv_read_token_q8(cache, control, control)
    with pytest.raises(ValueError, match="CUDA"):
        paged_gqa_decode_attention_q8(torch.zeros(2, 4, 32), cache, control[:, None], control, max_context_length=16)
    with pytest.raises(ValueError, match="CUDA"):
        linear_mxfp4(torch.zeros(1, 32, dtype=torch.bfloat16), *quantize_mxfp4(torch.ones(4, 32)))
    with pytest.raises(ValueError, match="CUDA"):
        token_logprobs(torch.zeros(2, 4), torch.zeros(2, dtype=torch.int64))


def _write(library, **changed):
    names = ("keys", "values", "key_cache", "value_cache", "key_scales", "value_scales", "blocks", "offsets", "active")
    args = {name: FAKE for name in names} | {"rows": 2, "kv_heads": 2, "head_dim": 32, "num_blocks": 3,
                                             "block_size": 16, "dtype": 2, "stream": None} | changed
    return library.tf_paged_kv_write_token_q8(*args.values())


def _read(library, **changed):
    names = ("key_cache", "value_cache", "key_scales", "value_scales", "blocks", "offsets", "keys", "values")
    args = {name: FAKE for name in names} | {"rows": 2, "kv_heads": 2, "head_dim": 32, "num_blocks": 3,
                                             "block_size": 16, "dtype": 2, "stream": None} | changed
    return library.tf_paged_kv_read_token_q8(*args.values())


def _attend(library, **changed):
    names = ("query", "key_cache", "value_cache", "key_scales", "value_scales", "tables", "lengths", "output",
             "partial_max", "partial_sum", "partial_acc")
    args = {name: FAKE for name in names} | {
        "capacity": 1024, "stride": 64, "batch": 2, "query_heads": 4, "kv_heads": 2, "head_dim": 32, "num_blocks": 3,
        "block_size": 16, "table_width": 8, "split_size": 64, "num_splits": 2, "scale": 0.5, "dtype": 2,
        "stream": None} | changed
    return library.tf_paged_gqa_decode_q8(*args.values())


def _project(library, **changed):
    args = {"x": FAKE, "x_stride": 64, "weight": FAKE, "weight_stride": 32, "scales": FAKE, "scale_stride": 2,
            "residual": None, "residual_stride": 0, "y": FAKE, "y_stride": 8, "m": 4, "n": 8, "k": 64, "dtype": 2,
            "stream": None} | changed
    return library.tf_linear_mxfp4(*args.values())


def _score(library, **changed):
    args = {"logits": FAKE, "stride": 100, "rows": 2, "columns": 100, "tokens": FAKE, "logprobs": FAKE,
            "entropy": FAKE, "top": FAKE, "top_tokens": FAKE, "top_k": 5, "dtype": 2, "stream": None} | changed
    return library.tf_token_logprobs(*args.values())


@pytest.mark.parametrize(("call", "changed", "status", "message"), [
    (_write, {"dtype": 3}, 1, "dtype"), (_write, {"head_dim": 40}, 2, "head dimensions"),
    (_write, {"head_dim": 288}, 2, "head dimensions"), (_write, {"block_size": 24}, 2, "pages"),
    (_write, {"kv_heads": 0}, 1, "positive"), (_write, {"rows": -1}, 1, "non-negative"),
    (_write, {"keys": None}, 1, "null"), (_write, {"key_scales": None}, 1, "null"),
    (_write, {"active": None}, 1, "null"), (_write, {"blocks": None}, 1, "null"),
    (_write, {"value_cache": FAKE + 8}, 1, "16-byte"), (_write, {"kv_heads": 70000}, 2, "grid"),
    (_read, {"dtype": 3}, 1, "dtype"), (_read, {"values": None}, 1, "null"), (_read, {"offsets": None}, 1, "null"),
    (_read, {"key_cache": FAKE + 4}, 1, "16-byte"),
    (_attend, {"dtype": 3}, 1, "dtype"), (_attend, {"head_dim": 20}, 2, "head dimensions"),
    (_attend, {"query_heads": 3}, 1, "multiple of kv heads"), (_attend, {"query_heads": 0}, 1, "positive"),
    (_attend, {"split_size": 32}, 1, "partitions"), (_attend, {"num_splits": 0}, 1, "partitions"),
    (_attend, {"table_width": 1 << 30}, 2, "tokens"), (_attend, {"batch": 70000}, 2, "grid"),
    (_attend, {"partial_acc": None}, 1, "partial buffers"), (_attend, {"capacity": 15}, 1, "too small"),
    (_attend, {"stride": 16}, 1, "too small"), (_attend, {"lengths": None}, 1, "null"),
    (_attend, {"value_cache": FAKE + 8}, 1, "16-byte"),
    (_project, {"dtype": 0}, 2, "fp16 or bf16"), (_project, {"m": 65}, 1, "64 rows"), (_project, {"k": 48}, 1, "multiple of 32"),
    (_project, {"k": 0}, 1, "multiple of 32"), (_project, {"scales": None}, 1, "null"),
    (_project, {"x_stride": 32}, 1, "shorter"), (_project, {"weight_stride": 16}, 1, "shorter"),
    (_project, {"scale_stride": 1}, 1, "shorter"), (_project, {"y_stride": 7}, 1, "shorter"),
    (_project, {"residual": FAKE, "residual_stride": 7}, 1, "shorter"), (_project, {"x": FAKE + 2}, 1, "16-byte"),
    (_project, {"weight_stride": 40}, 1, "16-byte"),
    (_score, {"dtype": 4}, 1, "dtype"), (_score, {"rows": -1}, 1, "non-negative"), (_score, {"columns": 0}, 1, "column"),
    (_score, {"stride": 99}, 1, "shorter"), (_score, {"top_k": 33}, 1, "top_k"), (_score, {"top_k": -1}, 1, "top_k"),
    (_score, {"columns": 4, "top_k": 5}, 1, "top_k"), (_score, {"tokens": None}, 1, "null"),
    (_score, {"top_tokens": None}, 1, "null"),
])
def test_c_abi_refusals(call, changed, status, message):
    library = _native.library()
    assert call(library, **changed) == status
    assert message in library.tf_last_error().decode()


@pytest.mark.parametrize("changed", [
    {"n": (1 << 28) + 1, "y_stride": 1 << 29},
    {"k": (1 << 28) + 32, "x_stride": 1 << 29, "weight_stride": 1 << 28, "scale_stride": 1 << 24}])
def test_projections_past_32_bit_indexes_are_refused(changed):
    library = _native.library()
    assert _project(library, **changed) == 2
    assert "2^28" in library.tf_last_error().decode()


def test_c_abi_calls_without_rows_do_nothing():
    library = _native.library()
    assert _write(library, rows=0, keys=None, values=None, blocks=None, offsets=None, active=None) == 0
    assert _read(library, rows=0, keys=None, values=None) == 0
    assert _attend(library, batch=0, query=None) == 0
    assert _project(library, m=0, x=None) == 0 and _project(library, n=0) == 0
    assert _score(library, rows=0, logits=None) == 0


def test_attention_plan():
    """Partitions cover the context in multiples of 64 tokens, as many as the
    workspace holds; one pass for short contexts and full grids."""

    from tensorforge_amd.kernels.cache_q8 import attention_q8_plan

    for context in (1, 63, 64, 300, 1024, 1025, 2048, 5000, 32768, 1 << 20):
        for batch in (0, 1, 3, 64, 500):
            for slots in (0, 1, 2, 7, 64, 1 << 20):
                size, splits = attention_q8_plan(context, batch, 4, slots)
                assert size % 64 == 0 and splits * size >= context > (splits - 1) * size
                assert splits <= max(slots, 1)
    assert attention_q8_plan(1024, 1, 4, 100)[1] == 1
    assert attention_q8_plan(2048, 64, 4, 100)[1] == 1
    assert attention_q8_plan(32768, 4, 8, 100) == (4096, 8)
    assert attention_q8_plan(2048, 1, 4, 100) == (128, 16)


def test_quantize_mxfp4_rounds_to_the_nearest_value():
    generator = torch.Generator().manual_seed(3)
    weight = torch.randn(7, 96, generator=generator) * torch.exp(2 * torch.randn(7, 1, generator=generator))
    weight[2, 32:64] = 0
    weight[3, :32] = torch.tensor([4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, -0.25, -0.75, -5.0, -2.5] + [0.0] * 21)
    codes, scales = quantize_mxfp4(weight)
    assert codes.shape == (7, 48) and codes.dtype == torch.uint8
    assert scales.shape == (7, 3) and scales.dtype == torch.float8_e8m0fnu
    got = mxfp4_weight(codes, scales)
    unit = np.repeat(np.exp2(scales.view(torch.uint8).numpy().astype(np.float64) - 127), 32, 1)
    grid = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
    grid = np.concatenate((-grid[::-1], grid))
    exact = weight.double().numpy() / unit
    assert np.abs(exact).max() < 8
    nearest = np.abs(exact[..., None] - grid).min(-1)
    assert np.array_equal(np.abs(got / unit - exact), nearest)
    # Ties go to the even code: 0.25 -> 0, 0.75 -> 1, 1.25 -> 1, 1.75 -> 2, 2.5 -> 2, 3.5 -> 4, 5 -> 4.
    assert (got[3, :11] / unit[3, 0]).tolist() == [4, 0, 1, 1, 2, 2, 4, 0, -1, -4, -2]
    assert not got[2, 32:64].any() and int(scales.view(torch.uint8)[2, 1]) == 1
    strided = torch.empty(96, 7).t().copy_(weight)
    assert torch.equal(quantize_mxfp4(strided)[0], codes)
    assert torch.equal(quantize_mxfp4(weight.bfloat16())[0], quantize_mxfp4(weight.bfloat16().float())[0])


def test_quantize_mxfp4_refusals():
    with pytest.raises(ValueError, match="multiple of 32"):
        quantize_mxfp4(torch.ones(4, 48))
    with pytest.raises(ValueError, match="multiple of 32"):
        quantize_mxfp4(torch.ones(4, 0))
    with pytest.raises(TypeError, match="dtype"):
        quantize_mxfp4(torch.ones(4, 32, dtype=torch.int32))
    for bad in (float("inf"), float("nan")):
        weight = torch.ones(4, 32)
        weight[1, 2] = bad
        with pytest.raises(ValueError, match="finite"):
            quantize_mxfp4(weight)


def test_logprobs_output_sizes():
    result = TokenLogprobs.allocate(rows=3, top_k=0, device=torch.device("cpu"))
    assert result.logprobs.shape == (3,) and result.top_tokens.shape == (3, 0)
