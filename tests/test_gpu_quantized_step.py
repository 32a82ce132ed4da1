"""The 8-bit cache, the attention over it, the 4-bit projections and the token
log probabilities as a decode step runs them: prompts admitted and read back,
then steps of norm, fused qkv projection, rotation, append, attention, output
projection on the residual, LM head and scores.  Each operator is held to its
definition in 64 bits on the very inputs it got, within the bound of its
roundings, and captured steps to the eager ones bit by bit."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from helpers import assert_bit_exact
from oracle.model import rope_tables
from tensorforge_amd.kernels import (
    PagedAttentionWorkspace,
    PagedKVCacheQ8,
    TokenLogprobs,
    linear_mxfp4,
    paged_gqa_decode_attention_q8,
    paged_kv_read_token_q8,
    paged_kv_write_token_q8,
    quantize_mxfp4,
    rms_norm,
    rope_paged_kv_append,
    token_logprobs,
)
from tests import q8_reference

pytestmark = pytest.mark.gpu

HEADS, KV_HEADS, PAGE, BLOCKS, VOCAB, TOP_K, STEPS = 8, 2, 16, 48, 1003, 5, 4
# The last lane is padding: no context, nothing stored, a token outside the row.
PROMPTS = [0, 15, 16, 31, 150, -1]


class _Step:
    """The buffers of a decode step of one layer, and the step."""

    def __init__(self, device, dtype, dim):
        generator = torch.Generator().manual_seed(dim)
        hidden = HEADS * dim
        lanes = len(PROMPTS)

        def weight(n, k):
            return torch.randn(n, k, generator=generator) / k**0.5

        self.device, self.dtype, self.dim = device, dtype, dim
        self.qkv_weight, self.qkv_scales = (t.to(device) for t in quantize_mxfp4(
            weight((HEADS + 2 * KV_HEADS) * dim, hidden)))
        self.o_weight, self.o_scales = (t.to(device) for t in quantize_mxfp4(weight(hidden, hidden)))
        self.head_weight, self.head_scales = (t.to(device) for t in quantize_mxfp4(weight(VOCAB, hidden)))
        self.gain = torch.ones(hidden, dtype=dtype, device=device)
        cos, sin = rope_tables(dim, 10000.0, torch.arange(256))
        self.cos, self.sin = cos.to(dtype).to(device), sin.to(dtype).to(device)
        self.cache = PagedKVCacheQ8.allocate(num_blocks=BLOCKS, block_size=PAGE, kv_heads=KV_HEADS, head_dim=dim,
                                             device=device)
        self.unused = torch.zeros(1, PAGE, KV_HEADS, dim, dtype=dtype, device=device)
        self.nothing = torch.zeros(lanes, dtype=torch.int32, device=device)
        self.workspace = PagedAttentionWorkspace.allocate(
            batch_capacity=lanes, query_heads=HEADS, head_dim=dim, max_context_length=256, device=device)
        self.tables = torch.full((lanes, 256 // PAGE), -1, dtype=torch.int32)
        order = torch.randperm(BLOCKS, generator=generator).tolist()
        for lane, length in enumerate(PROMPTS):
            for j in range(-(-(length + STEPS) // PAGE) if length >= 0 else 0):
                self.tables[lane, j] = order.pop()
        self.x = torch.empty(lanes, hidden, dtype=dtype, device=device)
        self.norm = torch.empty_like(self.x)
        self.qkv = torch.empty(lanes, (HEADS + 2 * KV_HEADS) * dim, dtype=dtype, device=device)
        self.query = torch.empty(lanes, HEADS, dim, dtype=dtype, device=device)
        self.keys = torch.empty(lanes, KV_HEADS, dim, dtype=dtype, device=device)
        self.values = torch.empty_like(self.keys)
        self.attended = torch.empty_like(self.query)
        self.out = torch.empty_like(self.x)
        self.logits = torch.empty(lanes, VOCAB, dtype=dtype, device=device)
        self.scores = TokenLogprobs.allocate(rows=lanes, top_k=TOP_K, device=device)
        self.tables_dev = self.tables.to(device)
        self.positions = torch.zeros(lanes, dtype=torch.int64, device=device)
        self.pages, self.offsets, self.active, self.lengths = (torch.zeros_like(self.nothing) for _ in range(4))
        self.tokens = torch.zeros(lanes, dtype=torch.int64, device=device)

    def set(self, step):
        """The inputs of a step, copied into its buffers."""

        generator = torch.Generator().manual_seed(100 + step)
        self.x.copy_(torch.randn(self.x.shape, generator=generator))
        lengths = [n + step if n >= 0 else 0 for n in PROMPTS]
        self.positions.copy_(torch.tensor(lengths))
        self.host_pages = [int(self.tables[lane, n // PAGE]) for lane, n in enumerate(lengths)]
        self.host_offsets = [n % PAGE for n in lengths]
        self.host_active = [int(n >= 0) for n in PROMPTS]
        self.host_lengths = [n + 1 if on else 0 for n, on in zip(lengths, self.host_active)]
        for name in ("pages", "offsets", "active", "lengths"):
            getattr(self, name).copy_(torch.tensor(getattr(self, f"host_{name}")))
        tokens = torch.randint(0, VOCAB, (len(PROMPTS),), generator=generator)
        tokens[-1] = -1
        self.tokens.copy_(tokens)

    def run(self):
        dim = self.dim
        rms_norm(self.x, self.gain, output=self.norm)
        linear_mxfp4(self.norm, self.qkv_weight, self.qkv_scales, output=self.qkv)
        rope_paged_kv_append(self.qkv, self.positions, self.cos, self.sin, self.unused, self.unused, self.pages,
                             self.offsets, self.nothing, query_heads=HEADS, query_output=self.query,
                             key_output=self.keys)
        self.values.copy_(self.qkv[:, (HEADS + KV_HEADS) * dim:].view(-1, KV_HEADS, dim))
        paged_kv_write_token_q8(self.keys, self.values, self.cache, self.pages, self.offsets, self.active)
        paged_gqa_decode_attention_q8(self.query, self.cache, self.tables_dev, self.lengths, max_context_length=256,
                                      output=self.attended, workspace=self.workspace)
        linear_mxfp4(self.attended.view(self.x.shape), self.o_weight, self.o_scales, output=self.out,
                     residual=self.x)
        linear_mxfp4(self.out, self.head_weight, self.head_scales, output=self.logits)
        token_logprobs(self.logits, self.tokens, top_k=TOP_K, output=self.scores)

    def cache_tensors(self):
        cache = self.cache
        return [t.view(torch.uint8) for t in (cache.key, cache.value, cache.key_scales, cache.value_scales)]

    def results(self):
        scores = self.scores
        return [t.clone() for t in (self.qkv, self.query, self.keys, self.attended, self.out, self.logits,
                                    scores.logprobs, scores.entropy, scores.top_logprobs, scores.top_tokens,
                                    *self.cache_tensors())]

    def admit(self, reference):
        """The prompts' tokens in one call, and their read-back."""

        generator = torch.Generator().manual_seed(7)
        slots = [(int(self.tables[lane, t // PAGE]), t % PAGE) for lane, n in enumerate(PROMPTS) for t in range(n)]
        rows = (2, len(slots), KV_HEADS, self.dim)
        keys, values = torch.randn(rows, generator=generator).to(self.dtype)
        pages, offsets = ([slot[i] for slot in slots] for i in (0, 1))
        vectors = [torch.tensor(v, dtype=torch.int32, device=self.device) for v in (pages, offsets, [1] * len(slots))]
        paged_kv_write_token_q8(keys.to(self.device), values.to(self.device), self.cache, *vectors)
        reference.write(keys, values, pages, offsets, [1] * len(slots))
        read = paged_kv_read_token_q8(self.cache, *vectors[:2], dtype=self.dtype)
        for got, want in zip(read, reference.values()):
            assert torch.equal(got.double().cpu(), torch.from_numpy(want[pages, :, offsets]))


def _within(got, want, bound, what):
    worst = ((got.double().cpu() - want).abs() / bound).max()
    assert worst <= 1, (what, float(worst))


def _check(step, reference):
    x = step.norm.cpu()
    for got, inputs, weight, scales, residual in (
            (step.qkv, x, step.qkv_weight, step.qkv_scales, None),
            (step.out, step.attended.view(x.shape).cpu(), step.o_weight, step.o_scales, step.x),
            (step.logits, step.out.cpu(), step.head_weight, step.head_scales, None)):
        _within(got, *q8_reference.linear(inputs, weight, scales, residual), "projection")
    reference.write(step.keys.cpu(), step.values.cpu(), step.host_pages, step.host_offsets, step.host_active)
    key, value, key_scales, value_scales = step.cache_tensors()
    used = [(lane, page) for lane, n in enumerate(step.host_lengths) for page in
            step.tables[lane, :-(-n // PAGE)].tolist()]
    for lane, page in used:  # what other pages hold is void
        held = min(PAGE, step.host_lengths[lane] - PAGE * step.tables[lane].tolist().index(page))
        assert q8_reference.same_codes(key[page, :, :held], reference.codes[0, page, :, :held])
        assert q8_reference.same_codes(value[page, :, :, :held], reference.codes[1, page, :, :held].swapaxes(1, 2))
        for side, scales in enumerate((key_scales, value_scales)):
            assert (scales[page].cpu().numpy().astype(np.int64) - 127 == reference.exponents[side, page]).all()
    _within(step.attended, *q8_reference.attention(step.query, reference, step.tables.numpy(), step.host_lengths,
                                                   step.dim**-0.5), "attention")
    assert not step.attended[-1].any()
    given, entropy, top, top_tokens, bound, entropy_bound = q8_reference.logprobs(step.logits, step.tokens, TOP_K)
    scores = step.scores
    assert torch.equal(scores.top_tokens.cpu(), top_tokens)
    assert torch.isnan(scores.logprobs[-1])
    rows = slice(0, len(PROMPTS) - 1)
    _within(scores.logprobs[rows], given[rows], bound[rows], "log probability")
    _within(scores.entropy, entropy, entropy_bound, "entropy")
    _within(scores.top_logprobs, top, bound[:, None], "alternatives")


@pytest.mark.parametrize(("dtype", "dim"), [(torch.bfloat16, 64), (torch.float16, 128), (torch.bfloat16, 48)])
def test_steps_and_their_captured_replays(device, dtype, dim):
    step = _Step(device, dtype, dim)
    reference = q8_reference.CacheReference(BLOCKS, KV_HEADS, PAGE, dim)
    step.admit(reference)
    admitted = [t.clone() for t in step.cache_tensors()]
    eager = []
    for i in range(STEPS):
        step.set(i)
        step.run()
        eager.append(step.results())
        _check(step, reference)

    # Captured on a stream of its own; the captured step does not run.
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream(device)):
        step.run()
    for _ in range(2):
        for tensor, held in zip(step.cache_tensors(), admitted):
            tensor.copy_(held)
        for i in range(STEPS):
            step.set(i)
            graph.replay()
            got = step.results()
            torch.cuda.synchronize()
            for name, (a, b) in enumerate(zip(got, eager[i])):
                assert_bit_exact(a, b, f"step {i}, result {name}")


def test_steps_on_two_streams(device):
    """Two models' steps at once, each on its own stream with its own buffers."""

    steps = [_Step(device, torch.bfloat16, 64) for _ in range(2)]
    alone = []
    for step in steps:
        step.admit(q8_reference.CacheReference(BLOCKS, KV_HEADS, PAGE, 64))
    start = [[t.clone() for t in step.cache_tensors()] for step in steps]
    for step, offset in zip(steps, (0, 1)):
        step.set(offset)
        step.run()
        alone.append(step.results())
        for tensor, held in zip(step.cache_tensors(), start[offset]):
            tensor.copy_(held)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(device) for _ in steps]
    for step, stream in zip(steps, streams):
        with torch.cuda.stream(stream):
            step.run()
    torch.cuda.synchronize()
    for step, want in zip(steps, alone):
        for got, expected in zip(step.results(), want):
            assert_bit_exact(got, expected)
