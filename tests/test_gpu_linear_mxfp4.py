"""The 4-bit projection against its definition in 64 bits, element by element
within the bound of its roundings."""

from __future__ import annotations

import pytest
import torch

from tensorforge_amd.kernels import linear_mxfp4, quantize_mxfp4
from tests.q8_reference import linear

pytestmark = pytest.mark.gpu


def _inputs(m, n, k, dtype, seed, spread=0.0):
    generator = torch.Generator().manual_seed(seed)
    x = torch.randn(m, k, generator=generator).to(dtype)
    weight = 0.02 * torch.randn(n, k // 32, 32, generator=generator)
    weight *= torch.exp2(spread * torch.randn(n, k // 32, 1, generator=generator))
    codes, scales = quantize_mxfp4(weight.view(n, k))
    residual = torch.randn(m, n, generator=generator).to(dtype)
    return x, codes, scales, residual


def _on(device, codes, scales):
    return codes.to(device), scales.view(torch.uint8).to(device).view(torch.float8_e8m0fnu)


def _check(got, want, bound, what=""):
    """Within the bound, and infinite where the value is past the type's range."""

    over = torch.isinf(want.to(got.dtype))
    got = got.double().cpu()
    assert torch.equal(got[over], want[over].sign() * torch.inf), what
    excess = (got - want).abs()[~over] - bound[~over]
    assert torch.isfinite(got[~over]).all() and (excess <= 0).all(), (what, float(excess.max()))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize(("m", "n", "k"), [
    (1, 2048, 5632), (1, 1, 32), (3, 17, 96), (16, 256, 768), (17, 100, 2048), (33, 2560, 2048), (48, 31, 160),
    (49, 257, 1024), (64, 513, 4096), (64, 16, 32), (2, 4099, 224), (8, 96, 14336)])
def test_shapes(device, dtype, m, n, k):
    x, codes, scales, residual = _inputs(m, n, k, dtype, seed=m + n + k)
    weight = _on(device, codes, scales)
    got = linear_mxfp4(x.to(device), *weight)
    assert got.shape == (m, n) and got.dtype == dtype
    _check(got, *linear(x, codes, scales, None))
    added = linear_mxfp4(x.to(device), *weight, residual=residual.to(device))
    _check(added, *linear(x, codes, scales, residual), what="residual")
    # The residual is added to the rounded product.
    assert torch.equal(added, (got.float() + residual.to(device).float()).to(dtype))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize(("m", "n", "k"), [
    (17, 8193, 32), (32, 12300, 288), (33, 16385, 96), (48, 20481, 544), (49, 24577, 256), (64, 28673, 160),
    (64, 40001, 800), (40, 8200, 8224)])
def test_many_columns(device, dtype, m, n, k):
    """All rows in one workgroup: every width of its tiles, K behind a chunk, a ring and a panel of scales."""

    generator = torch.Generator().manual_seed(m + n + k)
    x = torch.randn(m, k + 8, generator=generator).to(dtype)[:, :k]
    codes = torch.randint(0, 256, (n, k // 2), generator=generator, dtype=torch.uint8)
    scales = torch.randint(118, 124, (n, k // 32), generator=generator, dtype=torch.uint8)
    if dtype == torch.float16:
        scales[::37, 0] = 100  # weights that fp16 cannot hold
    scales = scales.view(torch.float8_e8m0fnu)
    residual = torch.randn(m, n, generator=generator).to(dtype)
    buffer = torch.full((m + 2, n + 3), 7, dtype=dtype, device=device)
    rows = torch.empty(m, k + 8, dtype=dtype, device=device)[:, :k].copy_(x)
    got = linear_mxfp4(rows, *_on(device, codes, scales), residual=residual.to(device), output=buffer[1:-1, :n])
    _check(got, *linear(x, codes, scales, residual))
    assert (buffer[0] == 7).all() and (buffer[-1] == 7).all() and (buffer[:, n:] == 7).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_many_columns_keep_values_that_are_not_finite_in_their_rows(device, dtype):
    m, n, k = 50, 8400, 320
    x, codes, scales, _ = _inputs(m, n, k, dtype, seed=3)
    clean = linear_mxfp4(x.to(device), *_on(device, codes, scales))
    bad = x.clone()
    bad[7, 300] = torch.nan
    bad[49, 0] = torch.inf
    got = linear_mxfp4(bad.to(device), *_on(device, codes, scales))
    assert torch.isnan(got[7]).all() and not torch.isfinite(got[49]).any()
    keep = [r for r in range(m) if r not in (7, 49)]
    assert torch.equal(got[keep], clean[keep])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_every_code_in_every_place(device, dtype):
    """One-hot rows read single weights back exactly, for all 16 codes in every
    column of a group and scales far apart."""

    k, n = 128, 48
    generator = torch.Generator().manual_seed(1)
    codes = torch.randint(0, 256, (n, k // 2), generator=generator, dtype=torch.uint8)
    scales = torch.randint(110, 139, (n, k // 32), generator=generator, dtype=torch.uint8)
    scales = scales.view(torch.float8_e8m0fnu)
    weight = _on(device, codes, scales)
    for first in range(0, k, 64):
        x = torch.zeros(64, k, dtype=dtype)
        x[torch.arange(64), first + torch.arange(64)] = 1
        want, _ = linear(x, codes, scales, None)
        assert torch.equal(linear_mxfp4(x.to(device), *weight).double().cpu(), want.to(dtype).double())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_scales_far_apart_and_extreme_rows(device, dtype):
    x, codes, scales, residual = _inputs(5, 70, 512, dtype, seed=2, spread=8.0)
    x[1] *= 1000
    x[2] *= 2.0**-14
    x[3] = 0
    _check(linear_mxfp4(x.to(device), *_on(device, codes, scales)), *linear(x, codes, scales, None))


def test_bf16_scales_at_the_ends(device):
    """Scale bytes 1 and 254: 2^-126 and 2^127."""

    codes = torch.full((16, 32), 0x22, dtype=torch.uint8)  # 1.0
    scales = torch.tensor([[1, 1]] * 8 + [[254, 254]] * 8, dtype=torch.uint8).view(torch.float8_e8m0fnu)
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    x[0, 3], x[1, 40] = 2.0**100, 2.0**-120
    got = linear_mxfp4(x.to(device), *_on(device, codes, scales)).double().cpu()
    assert torch.equal(got, linear(x, codes, scales, None)[0].to(torch.bfloat16).double())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_values_that_are_not_finite_stay_in_their_rows(device, dtype):
    x, codes, scales, _ = _inputs(20, 40, 256, dtype, seed=3)
    weight = _on(device, codes, scales)
    clean = linear_mxfp4(x.to(device), *weight)
    x[4, 100] = float("nan")
    x[17, 3] = float("inf")
    got = linear_mxfp4(x.to(device), *weight)
    keep = [r for r in range(20) if r not in (4, 17)]
    assert torch.equal(got[keep], clean[keep])
    assert got[4].isnan().all() and not torch.isfinite(got[17]).any()


@pytest.mark.parametrize("m", [1, 30, 64])
def test_strides_output_and_aliased_residual(device, m):
    n, k = 100, 320
    x, codes, scales, residual = _inputs(m, n, k, torch.bfloat16, seed=4)
    wide = torch.full((m, k + 24), float("nan"), dtype=torch.bfloat16, device=device)
    wide[:, 8:8 + k] = x.to(device)
    packed = torch.full((n, k // 2 + 32), 0xff, dtype=torch.uint8, device=device)
    packed[:, 16:16 + k // 2] = codes.to(device)
    _, scale = _on(device, codes, scales)
    out = torch.full((m + 1, n + 7), 5.0, dtype=torch.bfloat16, device=device)
    view = out[:m, 3:3 + n]
    got = linear_mxfp4(wide[:, 8:8 + k], packed[:, 16:16 + k // 2], scale, output=view)
    assert got.data_ptr() == view.data_ptr()
    plain = linear_mxfp4(x.to(device), codes.to(device), scale)
    assert torch.equal(got, plain)
    assert (out[m] == 5).all() and (out[:, :3] == 5).all() and (out[:, 3 + n:] == 5).all()
    stream = residual.to(device)
    want = linear_mxfp4(x.to(device), codes.to(device), scale, residual=stream)
    assert torch.equal(linear_mxfp4(x.to(device), codes.to(device), scale, residual=stream, output=stream), want)


def test_results_do_not_depend_on_the_other_rows(device):
    x, codes, scales, _ = _inputs(64, 64, 1024, torch.bfloat16, seed=5)
    weight = _on(device, codes, scales)
    whole = linear_mxfp4(x.to(device), *weight)
    again = linear_mxfp4(x.to(device), *weight)
    assert torch.equal(whole, again)


def test_replays(device):
    x, codes, scales, residual = _inputs(7, 300, 1024, torch.bfloat16, seed=6)
    weight = _on(device, codes, scales)
    held, output = x.to(device), torch.empty(7, 300, dtype=torch.bfloat16, device=device)
    linear_mxfp4(held, *weight, output=output)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream(device)):
        linear_mxfp4(held, *weight, output=output)
    for step in range(3):
        held.copy_(_inputs(7, 300, 1024, torch.bfloat16, seed=60 + step)[0])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(output, linear_mxfp4(held, *weight))


def test_refusals(device):
    x, codes, scales, residual = _inputs(4, 24, 64, torch.bfloat16, seed=7)
    x, residual = x.to(device), residual.to(device)
    codes, scales = _on(device, codes, scales)
    with pytest.raises(TypeError, match="dtype"):
        linear_mxfp4(x.float(), codes, scales)
    with pytest.raises(ValueError, match="64"):
        linear_mxfp4(x.repeat(17, 1), codes, scales)
    with pytest.raises(ValueError, match="16-byte"):
        linear_mxfp4(torch.zeros(4, 65, dtype=torch.bfloat16, device=device)[:, 1:], codes, scales)
    with pytest.raises(ValueError, match="multiple of 32"):
        linear_mxfp4(x[:, :48], codes[:, :24], scales)
    with pytest.raises(ValueError, match="uint8"):
        linear_mxfp4(x, codes[:, :16], scales)
    with pytest.raises(ValueError, match="scales"):
        linear_mxfp4(x, codes, scales[:, :1])
    with pytest.raises(ValueError, match="scales"):
        linear_mxfp4(x, codes, scales.view(torch.uint8))
    with pytest.raises(ValueError, match="output"):
        linear_mxfp4(x, codes, scales, output=residual.float())
    with pytest.raises(ValueError, match="residual"):
        linear_mxfp4(x, codes, scales, residual=residual[:, :8])
    with pytest.raises(ValueError, match="device"):
        linear_mxfp4(x, codes.cpu(), scales)
    with pytest.raises(RuntimeError, match="inference-only"):
        linear_mxfp4(x.clone().requires_grad_(), codes, scales)
    assert linear_mxfp4(x[:0], codes, scales).shape == (0, 24)
    assert linear_mxfp4(x, codes[:0], scales[:0]).shape == (4, 0)
