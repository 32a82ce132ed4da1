"""The 8-bit cache's append and read-back against their definition in 64 bits:
codes and scales exactly, over head sizes, pages, types, runs that begin,
continue and end inside pages, padded lanes, slots outside the cache, and
values that are zero, subnormal, huge or not finite."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tensorforge_amd.kernels import PagedKVCacheQ8, paged_kv_read_token_q8, paged_kv_write_token_q8
from tests.q8_reference import CacheReference, same_codes

pytestmark = pytest.mark.gpu


def _int32(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def _check(cache: PagedKVCacheQ8, reference: CacheReference, what="") -> None:
    for got, want in ((cache.key, reference.codes[0]), (cache.value, reference.codes[1].swapaxes(2, 3))):
        assert same_codes(got, want), what
    for got, want in zip((cache.key_scales, cache.value_scales), reference.exponents):
        assert np.array_equal(got.view(torch.uint8).cpu().numpy().astype(int) - 127, want), what


def _rows(count, heads, dim, dtype, seed):
    generator = torch.Generator().manual_seed(seed)
    spread = torch.exp2(torch.randint(-6, 7, (count, heads, 1), generator=generator).float())
    return tuple((torch.randn(count, heads, dim, generator=generator) * spread).to(dtype) for _ in range(2))


def _write_both(cache, reference, keys, values, blocks, offsets, active, device):
    paged_kv_write_token_q8(keys.to(device), values.to(device), cache, _int32(blocks, device),
                            _int32(offsets, device), _int32(active, device))
    reference.write(keys, values, blocks, offsets, active)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize(("heads", "dim", "page"), [(4, 64, 16), (8, 128, 16), (1, 16, 32), (3, 80, 48), (2, 256, 64),
                                                    (2, 32, 128)])
def test_prompt_then_tokens(device, dtype, heads, dim, page):
    """A prompt that ends inside a page, a chunk that continues it past the
    page's end, then single tokens."""

    reference = CacheReference(9, heads, page, dim, seed=5)
    cache = PagedKVCacheQ8(*reference.tensors(device))
    table = [7, 2, 5, 0]
    start = 0
    for step, count in enumerate([page + 5, page // 2 + page, 1, 1, 1]):
        keys, values = _rows(count, heads, dim, dtype, 10 * step + dim)
        blocks = [table[p // page] for p in range(start, start + count)]
        offsets = [p % page for p in range(start, start + count)]
        _write_both(cache, reference, keys, values, blocks, offsets, [1] * count, device)
        _check(cache, reference, (step, count))
        start += count


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows", [1, 2, 37, 300])
def test_decode_lanes(device, dtype, rows):
    """One token per lane into pages at any offset, padded lanes and slots
    outside the cache between them; the untouched pages stay as they were."""

    heads, dim, page = 4, 64, 16
    reference = CacheReference(rows + 5, heads, page, dim, seed=rows)
    cache = PagedKVCacheQ8(*reference.tensors(device))
    rng = np.random.default_rng(rows)
    blocks = rng.permutation(rows + 5)[:rows].tolist()
    offsets = rng.integers(0, page, rows).tolist()
    active = [1] * rows
    for r in range(0, rows, 7):
        kind = r // 7 % 6
        if rows > 2 and kind < 5:
            active[r] = 0 if kind == 0 else -1
            blocks[r] = (blocks[r], -1, rows + 5, blocks[r], blocks[r])[kind]
            offsets[r] = (offsets[r], 3, 3, -1, page)[kind]
    keys, values = _rows(rows, heads, dim, dtype, rows)
    _write_both(cache, reference, keys, values, blocks, offsets, active, device)
    _check(cache, reference)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_values_at_the_borders(device, dtype):
    """Zero tokens, the largest code and one step above it, subnormals, the
    type's largest values, infinities and NaN; a small page raised by a huge
    token and a huge page given a small one."""

    page, dim = 16, 16
    reference = CacheReference(8, 1, page, dim, seed=1)
    cache = PagedKVCacheQ8(*reference.tensors(device))
    largest = torch.finfo(dtype).max
    tiny = torch.finfo(dtype).smallest_normal / 4
    special = torch.zeros(8, 1, dim)
    special[1, 0, :4] = torch.tensor([448.0, -448.0, 1.0, 2.0**-10])
    special[2, 0, :4] = torch.tensor([450.0, -1.0, 17.0, 0.3])
    special[3, 0, :3] = torch.tensor([tiny, -tiny, 3 * tiny])
    special[4, 0, :4] = torch.tensor([largest / 2, -largest / 3, 1.0, 0.0])
    special[5, 0, :5] = torch.tensor([float("inf"), float("-inf"), float("nan"), 2.0, -7.0])
    special[6, 0] = float("nan")
    special[7, 0, :2] = torch.tensor([448 * 2.0**-130, -0.0])
    special = special.to(dtype)
    rows = list(range(8))
    _write_both(cache, reference, special, special.flip(0), rows, [0] * 8, [1] * 8, device)
    _check(cache, reference, "begun")
    later = torch.ones(8, 1, dim)
    later[0] *= 1e9
    later[1] *= 1e30
    later[2] = torch.linspace(440, 460, dim)
    later[4] *= 1e-30
    later = later.to(dtype)
    _write_both(cache, reference, later, later, rows, [3] * 8, [1] * 8, device)
    _check(cache, reference, "continued")


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize(("heads", "dim", "page"), [(4, 64, 16), (3, 80, 48), (2, 256, 32)])
def test_read(device, dtype, heads, dim, page):
    """Any slots in any order, twice the same, outside the cache (zeros), with
    and without outputs given."""

    reference = CacheReference(6, heads, page, dim, seed=3)
    cache = PagedKVCacheQ8(*reference.tensors(device))
    rng = np.random.default_rng(4)
    blocks = rng.integers(-1, 7, 203).tolist() + [2] * page + [3, 3]
    offsets = rng.integers(-1, page + 1, 203).tolist() + list(range(page)) + [4, 4]
    values = torch.from_numpy(reference.values())
    want = torch.zeros(2, len(blocks), heads, dim, dtype=torch.float64)
    for r, (block, offset) in enumerate(zip(blocks, offsets)):
        if 0 <= block < 6 and 0 <= offset < page:
            want[:, r] = values[:, block, :, offset]
    got = paged_kv_read_token_q8(cache, _int32(blocks, device), _int32(offsets, device), dtype=dtype)
    out = torch.full((2, len(blocks), heads, dim), 7.0, dtype=dtype, device=device)
    again = paged_kv_read_token_q8(cache, _int32(blocks, device), _int32(offsets, device), key_output=out[0],
                                   value_output=out[1])
    for side in (0, 1):
        assert got[side].dtype == dtype and again[side].data_ptr() == out[side].data_ptr()
        assert torch.equal(got[side].cpu().nan_to_num(nan=-77.0), want[side].to(dtype).nan_to_num(nan=-77.0))
        assert torch.equal(got[side].nan_to_num(nan=-77.0), again[side].nan_to_num(nan=-77.0))


def test_append_is_captured_and_replayed(device):
    """A decode step's append in a graph, its inputs changed between replays."""

    heads, dim, page, rows = 2, 32, 16, 5
    reference = CacheReference(rows, heads, page, dim, seed=8)
    cache = PagedKVCacheQ8(*reference.tensors(device))
    keys = torch.zeros(rows, heads, dim, dtype=torch.bfloat16, device=device)
    values = torch.zeros_like(keys)
    blocks, active = _int32(list(range(rows)), device), _int32([1] * rows, device)
    offsets = _int32([0] * rows, device)
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream(device)
    with torch.cuda.graph(graph, stream=side):
        paged_kv_write_token_q8(keys, values, cache, blocks, offsets, active)
    for step in range(4):
        new = _rows(rows, heads, dim, torch.bfloat16, step)
        keys.copy_(new[0])
        values.copy_(new[1])
        offsets.fill_(step)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        reference.write(*new, list(range(rows)), [step] * rows, [1] * rows)
        _check(cache, reference, step)


def test_refusals(device):
    cache = PagedKVCacheQ8.allocate(num_blocks=3, block_size=16, kv_heads=2, head_dim=32, device=device)
    rows = torch.zeros(4, 2, 32, device=device)
    control = torch.zeros(4, dtype=torch.int32, device=device)
    with pytest.raises(ValueError, match="cache's heads"):
        paged_kv_write_token_q8(rows[:, :1], rows, cache, control, control, control)
    with pytest.raises(ValueError, match="share dtype"):
        paged_kv_write_token_q8(rows, rows.half(), cache, control, control, control)
    with pytest.raises(TypeError, match="dtype"):
        paged_kv_write_token_q8(rows.double(), rows.double(), cache, control, control, control)
    with pytest.raises(ValueError, match="contiguous"):
        paged_kv_write_token_q8(rows.transpose(0, 1).contiguous().transpose(0, 1), rows, cache, control, control,
                                control)
    with pytest.raises(ValueError, match="block_offsets must be int32"):
        paged_kv_write_token_q8(rows, rows, cache, control, control.long(), control)
    with pytest.raises(ValueError, match="active_mask must be int32"):
        paged_kv_write_token_q8(rows, rows, cache, control, control, control[:3])
    with pytest.raises(ValueError, match="cache's heads"):
        paged_kv_read_token_q8(cache, control, control, key_output=rows[:3])
    with pytest.raises(ValueError, match="share dtype"):
        paged_kv_read_token_q8(cache, control, control, key_output=rows, value_output=rows.half())
    with pytest.raises(TypeError, match="dtype"):
        paged_kv_read_token_q8(cache, control, control, dtype=torch.float64)
    assert paged_kv_read_token_q8(cache, control[:0], control[:0])[0].shape == (0, 2, 32)
    paged_kv_write_token_q8(rows[:0], rows[:0], cache, control[:0], control[:0], control[:0])
