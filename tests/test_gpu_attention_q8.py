"""Decode attention over the 8-bit cache against its definition in 64 bits,
element by element within the bound of its roundings: head layouts, types,
pages, lengths of 0, 1 and across every border, pages outside the cache, stale
NaN codes behind a row's end, splits, graphs and streams."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tensorforge_amd.kernels import PagedAttentionWorkspace, PagedKVCacheQ8, paged_gqa_decode_attention_q8
from tests.q8_reference import CacheReference, attention

pytestmark = pytest.mark.gpu


def _reference(blocks, heads, page, dim, seed, finite=True):
    reference = CacheReference(blocks, heads, page, dim, seed=seed)
    if finite:
        reference.codes[reference.codes & 127 == 127] = 0x40
    # Codes near one another in size, as values of one distribution are.
    reference.codes[...] = np.where(np.random.default_rng(seed).random(reference.codes.shape) < 0.9,
                                    reference.codes & 0x87 | 0x38, reference.codes)
    return reference


def _tables(lengths, page, blocks, seed, extra=1):
    rng = np.random.default_rng(seed)
    width = max(1, -(-max(max(lengths), 1) // page)) + extra
    tables = np.full((len(lengths), width), -1)
    order = rng.permutation(blocks).tolist()
    for row, length in enumerate(lengths):
        for j in range(-(-max(length, 0) // page)):
            tables[row, j] = order.pop()
    return tables


def _run(device, reference, query, tables, lengths, scale=None, **options):
    cache = PagedKVCacheQ8(*reference.tensors(device))
    return paged_gqa_decode_attention_q8(
        query.to(device), cache, torch.tensor(tables, dtype=torch.int32, device=device),
        torch.tensor(lengths, dtype=torch.int32, device=device), scale=scale,
        max_context_length=max(1, max(lengths)), **options)


def _check(got, reference, query, tables, lengths, scale=None, what=""):
    want, bound = attention(query, reference, tables, lengths, query.shape[-1] ** -0.5 if scale is None else scale)
    got = got.double().cpu()
    assert torch.isfinite(got).all(), what
    worst = ((got - want).abs() / bound).max()
    assert worst <= 1, (what, float(worst))


def _query(rows, heads, dim, dtype, seed):
    return torch.randn(rows, heads, dim, generator=torch.Generator().manual_seed(seed)).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize(("heads", "kv_heads", "dim", "page"), [
    (32, 4, 64, 16), (8, 2, 32, 16), (8, 2, 128, 32), (12, 3, 96, 16), (5, 5, 16, 16), (20, 1, 80, 48),
    (48, 1, 64, 16), (64, 1, 64, 16), (6, 2, 256, 64), (4, 2, 192, 16), (3, 1, 112, 16)])
def test_layouts(device, dtype, heads, kv_heads, dim, page):
    lengths = [1, 0, page - 1, page, page + 1, 63, 64, 65, 200, -3]
    blocks = sum(-(-max(n, 0) // page) for n in lengths) + 2
    reference = _reference(blocks, kv_heads, page, dim, seed=dim + heads)
    tables = _tables(lengths, page, blocks, seed=1)
    query = _query(len(lengths), heads, dim, dtype, seed=2)
    got = _run(device, reference, query, tables, lengths)
    assert got.dtype == dtype
    _check(got, reference, query, tables, lengths)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize(("rows", "longest"), [(1, 5000), (3, 2500), (1, 1), (2, 257), (40, 700), (130, 90)])
def test_lengths_and_batches(device, dtype, rows, longest):
    """Calls of one partition and of many, rows far shorter than the longest."""

    rng = np.random.default_rng(rows)
    lengths = rng.integers(0, longest + 1, rows).tolist()
    lengths[rows // 2] = longest
    blocks = sum(-(-n // 16) for n in lengths) + 1
    reference = _reference(blocks, 2, 16, 64, seed=rows)
    tables = _tables(lengths, 16, blocks, seed=rows)
    query = _query(rows, 8, 64, dtype, seed=3)
    _check(_run(device, reference, query, tables, lengths), reference, query, tables, lengths)


@pytest.mark.parametrize("rows", [1, 60])
def test_pages_outside_the_cache_are_skipped(device, rows):
    lengths = [300 + r for r in range(rows)]
    lengths[0] = 1000
    blocks = sum(-(-n // 16) for n in lengths)
    reference = _reference(blocks, 2, 16, 64, seed=9)
    tables = _tables(lengths, 16, blocks, seed=9)
    tables[0, :3] = -1
    tables[0, 20:40] = blocks
    tables[0, 62] = 1 << 30
    tables[-1, 5] = -(1 << 31)
    if rows > 1:
        tables[1, :] = -7  # a row with no page at all
    query = _query(rows, 8, 64, torch.bfloat16, seed=1)
    got = _run(device, reference, query, tables, lengths)
    _check(got, reference, query, tables, lengths)
    if rows > 1:
        assert not got[1].any()


def test_stale_codes_behind_a_row_are_not_read_into_it(device):
    """Every code and scale behind a row's last token is NaN or huge."""

    lengths = [1, 17, 64, 100, 511, 33]
    blocks = sum(-(-n // 16) for n in lengths) + 3
    reference = _reference(blocks, 2, 16, 64, seed=4)
    tables = _tables(lengths, 16, blocks, seed=4)
    used = set()
    for row, length in enumerate(lengths):
        for j in range(-(-length // 16)):
            used.add(int(tables[row, j]))
            reference.codes[:, tables[row, j], :, max(0, min(16, length - 16 * j)):] = 0x7f
    for block in set(range(blocks)) - used:
        reference.codes[:, block] = 0x7f
        reference.exponents[:, block] = 120
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        query = _query(len(lengths), 8, 64, dtype, seed=5)
        _check(_run(device, reference, query, tables, lengths), reference, query, tables, lengths, what=dtype)


def test_table_entries_behind_a_row_are_not_followed(device):
    lengths = [40, 700]
    reference = _reference(60, 2, 16, 64, seed=14)
    tables = _tables(lengths, 16, 60, seed=14)
    query = _query(2, 8, 64, torch.bfloat16, seed=15)
    clean = _run(device, reference, query, tables, lengths)
    tables[0, 3:] = 1 << 30
    assert torch.equal(_run(device, reference, query, tables, lengths), clean)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_scales_far_apart(device, dtype):
    """Pages whose scales differ by 2^40, for keys (scores from flat to sharp)
    and for values."""

    lengths = [500, 77]
    blocks = 40
    reference = _reference(blocks, 2, 16, 64, seed=6)
    rng = np.random.default_rng(6)
    reference.exponents[0] = rng.integers(-30, -1, reference.exponents[0].shape)
    reference.exponents[1] = rng.integers(-40, 1, reference.exponents[1].shape)
    tables = _tables(lengths, 16, blocks, seed=6)
    query = _query(2, 8, 64, dtype, seed=7)
    _check(_run(device, reference, query, tables, lengths), reference, query, tables, lengths)


def test_sharp_scores_and_negative_scale(device):
    lengths = [300, 129, 2]
    reference = _reference(40, 2, 16, 64, seed=16)
    tables = _tables(lengths, 16, 40, seed=16)
    for scale in (3.0, -0.25, 1e-4, 0.0):
        query = _query(3, 8, 64, torch.float32, seed=17)
        _check(_run(device, reference, query, tables, lengths, scale=scale), reference, query, tables, lengths, scale,
               what=scale)


def test_nan_query_and_nan_codes_stay_in_their_rows(device):
    lengths = [100, 100, 100]
    reference = _reference(30, 2, 16, 64, seed=18)
    tables = _tables(lengths, 16, 30, seed=18)
    query = _query(3, 8, 64, torch.bfloat16, seed=19)
    clean = _run(device, reference, query, tables, lengths)
    broken = query.clone()
    broken[1, 3, 7] = float("nan")
    got = _run(device, reference, broken, tables, lengths)
    assert got[1, 3].isnan().all()
    keep = torch.ones(3, 8, dtype=torch.bool)
    keep[1, 3] = False
    assert torch.equal(got[keep.to(device)], clean[keep.to(device)])
    reference.codes[1, tables[2, 1], 0, 5, 9] = 0x7f   # one value of row 2, kv head 0
    got = _run(device, reference, query, tables, lengths)
    assert got[2, :4, 9].isnan().all() and int(got.isnan().sum()) == 4


def test_nan_query_over_many_partitions(device):
    """Every score of one head NaN in every partition."""

    lengths = [3000]
    reference = _reference(190, 2, 16, 64, seed=28)
    tables = _tables(lengths, 16, 190, seed=28)
    query = _query(1, 8, 64, torch.bfloat16, seed=29)
    query[0, 5] = float("nan")
    got = _run(device, reference, query, tables, lengths)
    assert got[0, 5].isnan().all() and int(got.isnan().sum()) == 64


@pytest.mark.parametrize("held", [1, 2, 5, 64])
def test_workspace_and_output_are_used(device, held):
    """Fewer partitions where the workspace holds fewer; the same result within
    the bound, the caller's output returned."""

    lengths = [1900, 1000]
    blocks = 190
    reference = _reference(blocks, 2, 16, 64, seed=20)
    tables = _tables(lengths, 16, blocks, seed=20)
    query = _query(2, 8, 64, torch.bfloat16, seed=21)
    workspace = PagedAttentionWorkspace(torch.full((16 * held,), float("nan"), device=device),
                                        torch.full((16 * held,), float("nan"), device=device),
                                        torch.full((16 * held, 64), float("nan"), device=device))
    output = torch.full((2, 8, 64), float("nan"), dtype=torch.bfloat16, device=device)
    got = _run(device, reference, query, tables, lengths, output=output, workspace=workspace)
    assert got is output
    _check(got, reference, query, tables, lengths)


def test_replays_and_streams(device):
    """Captured with its own workspace, replayed with changed inputs between
    eager calls on another stream; every replay equals the eager result."""

    lengths = [900, 30, 0, 333]
    blocks = 100
    reference = _reference(blocks, 2, 16, 64, seed=22)
    tables = _tables(lengths, 16, blocks, seed=22)
    cache = PagedKVCacheQ8(*reference.tensors(device))
    block_tables = torch.tensor(tables, dtype=torch.int32, device=device)
    contexts = torch.tensor(lengths, dtype=torch.int32, device=device)
    query = torch.zeros(4, 8, 64, dtype=torch.bfloat16, device=device)
    output = torch.empty_like(query)
    workspace = PagedAttentionWorkspace.allocate(batch_capacity=4, query_heads=8, head_dim=64,
                                                 max_context_length=1024, device=device)

    def call(**options):
        return paged_gqa_decode_attention_q8(query, cache, block_tables, contexts, max_context_length=900, **options)

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream(device)):
        call(output=output, workspace=workspace)
    side = torch.cuda.Stream(device)
    for step in range(4):
        query.copy_(_query(4, 8, 64, torch.bfloat16, seed=30 + step))
        contexts.copy_(torch.tensor([900 - 100 * step, 30 + step, step, 333], dtype=torch.int32))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            eager = call(workspace=PagedAttentionWorkspace.allocate(
                batch_capacity=4, query_heads=8, head_dim=64, max_context_length=1024, device=device))
        side.synchronize()
        assert torch.equal(output, eager), step


def test_offsets_past_32_bits(device):
    """A cache of more than 2^32 bytes of keys: pages at both ends."""

    blocks, heads, page, dim = 131072 + 64, 8, 32, 128  # 32 KiB of keys a page
    codes = torch.full((blocks, heads, page, dim), 0x38, dtype=torch.uint8, device=device)
    scales = torch.full((blocks, heads), 127, dtype=torch.uint8, device=device).view(torch.float8_e8m0fnu)
    value = codes.view(blocks, heads, dim, page)
    value[blocks - 1] = 0x40   # 2.0 at the far end, 1.0 elsewhere
    cache = PagedKVCacheQ8(codes.view(torch.float8_e4m3fn), value.view(torch.float8_e4m3fn), scales, scales)
    tables = torch.tensor([[0, blocks - 1], [blocks - 1, 1]], dtype=torch.int32, device=device)
    lengths = torch.tensor([48, 16], dtype=torch.int32, device=device)
    query = torch.zeros(2, 32, dim, dtype=torch.bfloat16, device=device)
    out = paged_gqa_decode_attention_q8(query, cache, tables, lengths, max_context_length=64)
    assert torch.allclose(out[0].float(), torch.tensor(4.0 / 3, device=device), rtol=2.0**-7)
    assert torch.equal(out[1].float(), torch.full((32, dim), 2.0, device=device))


def test_refusals(device):
    cache = PagedKVCacheQ8.allocate(num_blocks=3, block_size=16, kv_heads=2, head_dim=32, device=device)
    query = torch.zeros(2, 4, 32, dtype=torch.bfloat16, device=device)
    tables = torch.zeros(2, 3, dtype=torch.int32, device=device)
    lengths = torch.ones(2, dtype=torch.int32, device=device)

    def call(query=query, tables=tables, lengths=lengths, **options):
        return paged_gqa_decode_attention_q8(query, cache, tables, lengths, **{"max_context_length": 48} | options)

    with pytest.raises(ValueError, match="GQA groups"):
        call(query=query[:, :3].contiguous())
    with pytest.raises(ValueError, match="GQA groups"):
        call(query=query[..., :16].contiguous())
    with pytest.raises(ValueError, match="must have shape"):
        call(query=query[0])
    with pytest.raises(TypeError, match="query dtype"):
        call(query=query.double())
    with pytest.raises(TypeError, match="int32"):
        call(lengths=lengths.long())
    with pytest.raises(ValueError, match="one row per query"):
        call(tables=tables[:1])
    with pytest.raises(ValueError, match="one value per query"):
        call(lengths=lengths[:1])
    with pytest.raises(ValueError, match="contiguous"):
        call(query=query.transpose(0, 1).contiguous().transpose(0, 1))
    with pytest.raises(ValueError, match="table capacity"):
        call(max_context_length=49)
    with pytest.raises(ValueError, match="table capacity"):
        call(max_context_length=0)
    with pytest.raises(ValueError, match="must be positive"):
        call(lengths=lengths * 0, max_context_length=None)
    with pytest.raises(ValueError, match="output"):
        call(output=query.float())
    with pytest.raises(ValueError, match="workspace"):
        call(workspace=PagedAttentionWorkspace(*(torch.empty(8, 8, device=device, dtype=torch.float64),) * 3))
    with pytest.raises(RuntimeError, match="inference-only"):
        call(query=query.clone().requires_grad_())
    assert call(query=query[:0], tables=tables[:0], lengths=lengths[:0]).shape == (0, 4, 32)
    assert torch.equal(call(max_context_length=None), call())
