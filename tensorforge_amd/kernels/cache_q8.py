"""The 8-bit paged KV cache on gfx950 HIP kernels: its storage, the append,
the read-back and decode attention over it (``csrc/tf_cache_q8.hip``,
``csrc/tf_paged_attention_q8.hip``).  It holds half the bytes of a bf16 cache
and a decode step reads half as many; the reference has no counterpart, its
cache keeps the model's dtype (``tensorforge/cache/paged.py:27-60``).

Each page of a kv head holds e4m3 codes with one power-of-two scale, so a
code stands for ``code * scale`` exactly in bf16 and a page is requantised
without rounding (but for codes that become subnormal) when a later token
raises its scale.  Keys are token-major and values dimension-major within a
page: the order in which the attention kernel's matrix operands read them.
"""

from __future__ import annotations

import functools
from dataclasses import dataclass

import torch
from torch import Tensor

from tensorforge_amd import _native
from tensorforge_amd.kernels.attention import PagedAttentionWorkspace, _next_power_of_2

MAX_HEAD_DIM = 256
MAX_BLOCK_SIZE = 1024


@dataclass(frozen=True, slots=True)
class PagedKVCacheQ8:
    """One layer's 8-bit pages: ``key [blocks, kv_heads, block_size,
    head_dim]`` and ``value [blocks, kv_heads, head_dim, block_size]``
    (float8_e4m3fn), ``key_scales`` and ``value_scales [blocks, kv_heads]``
    (float8_e8m0fnu).  The tensors may be slices of larger ones (a layer of a
    whole model's cache), each contiguous.  A page needs no clearing: its scale
    is set by the token written at its offset 0."""

    key: Tensor
    value: Tensor
    key_scales: Tensor
    value_scales: Tensor

    def __post_init__(self) -> None:
        key, value, key_scales, value_scales = self.key, self.value, self.key_scales, self.value_scales
        if key.ndim != 4 or value.ndim != 4:
            raise ValueError("cache codes must be [blocks, kv_heads, block_size, head_dim] keys and "
                             "[blocks, kv_heads, head_dim, block_size] values")
        blocks, kv_heads, block_size, head_dim = key.shape
        if value.shape != (blocks, kv_heads, head_dim, block_size):
            raise ValueError("value codes must be [blocks, kv_heads, head_dim, block_size] of the keys' sizes")
        if key.dtype != torch.float8_e4m3fn or value.dtype != torch.float8_e4m3fn:
            raise TypeError("cache codes must use torch.float8_e4m3fn")
        if blocks < 1 or kv_heads < 1:
            raise ValueError("cache dimensions must be positive")
        if head_dim % 16 or not 0 < head_dim <= MAX_HEAD_DIM:
            raise ValueError("the 8-bit cache takes head dimensions that are multiples of 16 up to 256")
        if block_size % 16 or not 0 < block_size <= MAX_BLOCK_SIZE:
            raise ValueError("the 8-bit cache takes pages of a multiple of 16 tokens up to 1024")
        if key_scales.shape != (blocks, kv_heads) or value_scales.shape != (blocks, kv_heads):
            raise ValueError("scales must be [blocks, kv_heads]")
        if key_scales.dtype != torch.float8_e8m0fnu or value_scales.dtype != torch.float8_e8m0fnu:
            raise TypeError("scales must use torch.float8_e8m0fnu")
        device = key.device
        if value.device != device or key_scales.device != device or value_scales.device != device:
            raise ValueError("cache tensors must share one device")
        if not (key.is_contiguous() and value.is_contiguous() and key_scales.is_contiguous()
                and value_scales.is_contiguous()):
            raise ValueError("cache tensors must be contiguous")
        if key.data_ptr() % 16 or value.data_ptr() % 16:
            raise ValueError("cache codes must be 16-byte aligned")

    @classmethod
    def allocate(cls, *, num_blocks: int, block_size: int, kv_heads: int, head_dim: int,
                 device: torch.device) -> PagedKVCacheQ8:
        """A cache of zeros."""

        codes = (num_blocks, kv_heads)
        return cls(
            key=torch.zeros(*codes, block_size, head_dim, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn),
            value=torch.zeros(*codes, head_dim, block_size, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn),
            key_scales=torch.ones(codes, dtype=torch.uint8, device=device).view(torch.float8_e8m0fnu),
            value_scales=torch.ones(codes, dtype=torch.uint8, device=device).view(torch.float8_e8m0fnu),
        )

    @property
    def num_blocks(self) -> int:
        return self.key.shape[0]

    @property
    def kv_heads(self) -> int:
        return self.key.shape[1]

    @property
    def block_size(self) -> int:
        return self.key.shape[2]

    @property
    def head_dim(self) -> int:
        return self.key.shape[3]


def _require_library() -> None:
    if not _native.is_available():
        raise RuntimeError(
            "the gfx950 kernel library is unavailable; build it with "
            "`python -m tensorforge_amd.build`"
        )


def _check_slots(name: str, tensor: Tensor, rows: int, device: torch.device) -> None:
    if tensor.dtype != torch.int32 or tensor.shape != (rows,):
        raise ValueError(f"{name} must be int32 with one value per row")
    if tensor.device != device or not tensor.is_contiguous():
        raise ValueError(f"{name} must be contiguous on the cache's device")


def _check_rows(name: str, tensor: Tensor, shape: tuple[int, int, int], dtype: torch.dtype,
                device: torch.device) -> None:
    if tensor.shape != shape:
        raise ValueError(f"{name} must be [rows, kv_heads, head_dim] of the cache's heads")
    if tensor.dtype != dtype:
        raise ValueError("keys and values must share dtype")
    if tensor.device != device or not tensor.is_contiguous():
        raise ValueError(f"{name} must be contiguous on the cache's device")


def paged_kv_write_token_q8(
    keys: Tensor,
    values: Tensor,
    cache: PagedKVCacheQ8,
    physical_blocks: Tensor,
    block_offsets: Tensor,
    active_mask: Tensor,
) -> None:
    """Append token rows to the 8-bit cache: row ``r`` of ``keys``/``values
    [rows, kv_heads, head_dim]`` (fp32, fp16 or bf16) with ``active_mask[r] !=
    0`` goes to slot (``physical_blocks[r]``, ``block_offsets[r]``); other rows
    and slots outside the cache store nothing -- the arguments of
    :func:`paged_kv_write_token`, for the lanes of a decode step or the packed
    tokens of prompts.

    Neighbouring rows at ascending offsets of one page are written together; a
    page takes one such run per call (a second one elsewhere in the call would
    race for the page's scale).  A run from offset 0 begins its page: the page's
    scale is set by it and what the page held is void.  A run behind earlier
    tokens raises the scale where it needs to, and the page's codes are rounded
    to it.  Infinities and NaN are stored as NaN."""

    _require_library()
    device = cache.key.device
    if not cache.key.is_cuda:
        raise ValueError("paged KV writes require CUDA tensors")
    if device.index != _native.current_device():
        with torch.cuda.device(device):
            return paged_kv_write_token_q8(keys, values, cache, physical_blocks, block_offsets, active_mask)
    dtype = keys.dtype
    if dtype not in _native.DTYPE_CODES:
        raise TypeError(f"unsupported dtype: {dtype}")
    rows = keys.shape[0] if keys.ndim else 0
    num_blocks, kv_heads, block_size, head_dim = cache.key.shape
    shape = (rows, kv_heads, head_dim)
    _check_rows("keys", keys, shape, dtype, device)
    _check_rows("values", values, shape, dtype, device)
    _check_slots("physical_blocks", physical_blocks, rows, device)
    _check_slots("block_offsets", block_offsets, rows, device)
    _check_slots("active_mask", active_mask, rows, device)
    _native.check(
        _native.launch().tf_paged_kv_write_token_q8(
            keys.data_ptr(), values.data_ptr(), cache.key.data_ptr(), cache.value.data_ptr(),
            cache.key_scales.data_ptr(), cache.value_scales.data_ptr(), physical_blocks.data_ptr(),
            block_offsets.data_ptr(), active_mask.data_ptr(), rows, kv_heads, head_dim, num_blocks, block_size,
            _native.dtype_code(dtype), _native.current_stream(device),
        ),
        "paged_kv_write_token_q8",
    )


def paged_kv_read_token_q8(
    cache: PagedKVCacheQ8,
    physical_blocks: Tensor,
    block_offsets: Tensor,
    *,
    dtype: torch.dtype = torch.bfloat16,
    key_output: Tensor | None = None,
    value_output: Tensor | None = None,
) -> tuple[Tensor, Tensor]:
    """Token rows of the 8-bit cache as values: ``(keys, values)``, each
    ``[rows, kv_heads, head_dim]``, of the slots (``physical_blocks[r]``,
    ``block_offsets[r]``) -- what a prompt's next chunk attends to.  Exact in
    bf16 and fp32, rounded once (to infinity where too large) in fp16; zeros
    for slots outside the cache.  ``dtype`` is the outputs' where none is
    given."""

    _require_library()
    device = cache.key.device
    if not cache.key.is_cuda:
        raise ValueError("paged KV reads require CUDA tensors")
    if device.index != _native.current_device():
        with torch.cuda.device(device):
            return paged_kv_read_token_q8(cache, physical_blocks, block_offsets, dtype=dtype, key_output=key_output,
                                          value_output=value_output)
    given = key_output if key_output is not None else value_output
    if given is not None:
        dtype = given.dtype
    if dtype not in _native.DTYPE_CODES:
        raise TypeError(f"unsupported dtype: {dtype}")
    if physical_blocks.ndim != 1:
        raise ValueError("physical_blocks must be int32 with one value per row")
    rows = physical_blocks.shape[0]
    num_blocks, kv_heads, block_size, head_dim = cache.key.shape
    shape = (rows, kv_heads, head_dim)
    _check_slots("physical_blocks", physical_blocks, rows, device)
    _check_slots("block_offsets", block_offsets, rows, device)
    if key_output is None:
        key_output = torch.empty(shape, dtype=dtype, device=device)
    else:
        _check_rows("key_output", key_output, shape, dtype, device)
    if value_output is None:
        value_output = torch.empty(shape, dtype=dtype, device=device)
    else:
        _check_rows("value_output", value_output, shape, dtype, device)
    _native.check(
        _native.launch().tf_paged_kv_read_token_q8(
            cache.key.data_ptr(), cache.value.data_ptr(), cache.key_scales.data_ptr(),
            cache.value_scales.data_ptr(), physical_blocks.data_ptr(), block_offsets.data_ptr(),
            key_output.data_ptr(), value_output.data_ptr(), rows, kv_heads, head_dim, num_blocks, block_size,
            _native.dtype_code(dtype), _native.current_stream(device),
        ),
        "paged_kv_read_token_q8",
    )
    return key_output, value_output


# Contexts up to which a row is one partition whatever the batch, tokens of the
# smallest partition, and tokens from which one is cut to spread ragged rows.
# On MI355X, graph-timed, the merge launch (2.2 us) included: 8 rows of 1000
# tokens at 4 kv heads of 64 7.6 us in one pass, 7.1-7.5 in partitions; 1 of
# 2048 9.6 and 6.9 (16 partitions); 32 of up to 2048 fp32 13.3 and 12.4 (2);
# 16 of up to 4096 at 8 heads of 128 27.2 and 21.9 (2); 4 of 8k-32k 167 and 35.5
# (8); 1 of 32k 158 and 18.3 (32).
ONE_PASS_CONTEXT = 1024
SMALLEST_PARTITION = 128
LARGEST_PARTITION = 4096
COMPUTE_UNITS = 256


@functools.lru_cache(maxsize=4096, typed=True)
def attention_q8_plan(launch_context: int, batch: int, kv_heads: int, slot_limit: int) -> tuple[int, int]:
    """(tokens per partition, partitions per row) of a call, from host-known
    sizes only: about one workgroup per compute unit, more where the partitions
    would pass LARGEST_PARTITION, as many as the workspace holds per (row, query
    head); one pass for contexts up to ONE_PASS_CONTEXT."""

    want = 1
    if launch_context > ONE_PASS_CONTEXT:
        want = max(COMPUTE_UNITS // max(batch * kv_heads, 1), launch_context // LARGEST_PARTITION)
    want = max(1, min(want, slot_limit))
    size = max((-(-launch_context // want) + 63) // 64 * 64, SMALLEST_PARTITION)
    return size, -(-launch_context // size)


def paged_gqa_decode_attention_q8(
    query: Tensor,
    cache: PagedKVCacheQ8,
    block_tables: Tensor,
    context_lengths: Tensor,
    *,
    scale: float | None = None,
    max_context_length: int | None = None,
    output: Tensor | None = None,
    workspace: PagedAttentionWorkspace | None = None,
) -> Tensor:
    """Attend one query token per sequence over the pages of an 8-bit cache:
    :func:`paged_gqa_decode_attention` with ``cache`` in place of the key and
    value caches (fp32, fp16 or bf16 ``query [batch, query_heads, head_dim]``,
    int32 ``block_tables`` and ``context_lengths``).  Rows with
    ``context_lengths <= 0`` are zeros, tokens whose page lies outside the cache
    are skipped.  Give ``max_context_length`` to keep the call free of host
    synchronisation, and ``output`` and ``workspace`` to keep it free of
    allocation.  Calls that share a workspace must not overlap in time."""

    _require_library()
    if not query.is_cuda or not cache.key.is_cuda:
        raise ValueError("paged GQA attention requires CUDA tensors")
    device = query.device
    if device.index != _native.current_device():
        with torch.cuda.device(device):
            return paged_gqa_decode_attention_q8(
                query, cache, block_tables, context_lengths, scale=scale, max_context_length=max_context_length,
                output=output, workspace=workspace)
    if query.ndim != 3:
        raise ValueError("query must have shape [batch, query_heads, head_dim]")
    if query.dtype not in _native.DTYPE_CODES:
        raise TypeError(f"unsupported query dtype: {query.dtype}")
    if block_tables.dtype != torch.int32 or context_lengths.dtype != torch.int32:
        raise TypeError("block tables and context lengths must use torch.int32")
    batch, query_heads, head_dim = query.shape
    num_blocks, kv_heads, block_size, cache_head_dim = cache.key.shape
    if head_dim != cache_head_dim or query_heads < 1 or query_heads % kv_heads != 0:
        raise ValueError("query/cache head dimensions do not form valid GQA groups")
    if block_tables.ndim != 2 or block_tables.shape[0] != batch:
        raise ValueError("block_tables must have one row per query")
    if context_lengths.shape != (batch,):
        raise ValueError("context_lengths must have one value per query")
    for tensor in (query, block_tables, context_lengths):
        if tensor.device != device or not tensor.is_contiguous():
            raise ValueError("paged GQA attention requires contiguous tensors on one device")
    if cache.key.device != device:
        raise ValueError("query and cache must share one device")
    if query.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("TensorForge HIP kernels are inference-only")
    table_width = block_tables.shape[1]
    capacity = table_width * block_size
    if max_context_length is None:
        launch_context = int(context_lengths.max().item()) if batch > 0 else 0
        if launch_context <= 0:
            raise ValueError("context lengths must be positive")
    else:
        launch_context = max_context_length
    if launch_context <= 0 or launch_context > capacity:
        raise ValueError("max_context_length must be positive and within table capacity")
    if output is None:
        output = torch.empty_like(query)
    elif (output.shape != query.shape or output.dtype != query.dtype or output.device != device
          or not output.is_contiguous()):
        raise ValueError("output must be contiguous and share query shape, dtype, and device")
    programs = max(batch * query_heads, 1)
    if workspace is None:
        held = 1 << 30
    else:
        partials = (workspace.partial_max, workspace.partial_sum, workspace.partial_accumulator)
        for partial in partials:
            if partial.device != device or partial.dtype != torch.float32 or not partial.is_contiguous():
                raise ValueError("split-KV workspace has insufficient or incompatible capacity")
        if partials[2].ndim != 2 or partials[2].shape[1] < head_dim:
            raise ValueError("split-KV workspace has insufficient or incompatible capacity")
        held = min(partials[0].numel(), partials[1].numel(), partials[2].shape[0])
    split_size, num_splits = attention_q8_plan(launch_context, batch, kv_heads, held // programs)
    maximum = total = accumulator = None
    stride = 0
    if num_splits > 1:
        if workspace is None:
            held, stride = programs * num_splits, _next_power_of_2(head_dim)
            buffers = torch.empty(held * (stride + 2), dtype=torch.float32, device=device)
            accumulator = buffers.data_ptr()
            maximum = accumulator + 4 * held * stride
            total = maximum + 4 * held
        else:
            stride = partials[2].shape[1]
            maximum, total, accumulator = (t.data_ptr() for t in partials)
    _native.check(
        _native.launch().tf_paged_gqa_decode_q8(
            query.data_ptr(), cache.key.data_ptr(), cache.value.data_ptr(), cache.key_scales.data_ptr(),
            cache.value_scales.data_ptr(), block_tables.data_ptr(), context_lengths.data_ptr(), output.data_ptr(),
            maximum, total, accumulator, held, stride, batch, query_heads, kv_heads, head_dim, num_blocks,
            block_size, table_width, split_size, num_splits, head_dim**-0.5 if scale is None else scale,
            _native.dtype_code(query.dtype), _native.current_stream(device),
        ),
        "paged_gqa_decode_attention_q8",
    )
    return output
