"""8-bit products whose CTAs take several tiles each (the accumulator, the scale tiles, the output boxes and the residual's
barrier pass from one tile to the next), and the quantiser's forms for many rows and for infinities and NaN in bf16."""
import pytest
import torch

from sana_b200 import ops
from test_gpu_fp8 import check, operands, reference_quantise


@pytest.mark.gpu
@pytest.mark.parametrize("K", [16, 272, 656, 1152, 2192])  # 1, 1, 2, 3 and 5 groups of four scale blocks to a tile
@pytest.mark.parametrize("M,N", [(1031, 6728), (4100, 5000)])  # 477 tiles of one CTA, 340 of a pair: three or more each
def test_several_tiles_to_a_cta(M, N, K):
    a, w, g = operands(M, N, K)
    plain = ops.gemm_fp8(a, w)
    check(plain, a, w)
    bias = torch.randn(N, generator=g).bfloat16().cuda()
    gate = (torch.randn(6, N, generator=g).bfloat16().cuda(), torch.randn(3, 6 * N, generator=g).bfloat16().cuda(), 4, (M + 2) // 3)
    residual = torch.randn(M, N, generator=g).bfloat16().cuda()
    full = dict(bias=bias, act=ops.ACT_SILU, gate=gate, residual=residual)
    out = ops.gemm_fp8(a, w, **full)
    check(out, a, w, **full)
    for _ in range(4):
        assert torch.equal(ops.gemm_fp8(a, w), plain) and torch.equal(ops.gemm_fp8(a, w, **full), out)
    in_place = residual.clone()
    ops.gemm_fp8(a, w, bias=bias, act=ops.ACT_SILU, gate=gate, residual=in_place, out=in_place)
    assert torch.equal(in_place, out)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,K", [(9001, 1152), (1, 144), (131, 400)])  # 9001 rows of nine blocks: two rows to a thread
@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantiser_with_infinities_and_nan(dtype, rows, K, block_rows):
    g = torch.Generator().manual_seed(rows + K)
    x = torch.randn(rows, K, generator=g) * torch.exp2(torch.randint(-20, 20, (rows, 1), generator=g).float())
    for i, bad in enumerate((float("inf"), float("-inf"), float("nan"))):
        x[rows // 2, 5 + 17 * i] = bad  # beside finite values of its block
        x[rows - 1, K - 1 - 33 * i] = bad
    x = x.to(dtype)
    t = ops.fp8_quantize(x.cuda(), block_rows)
    ref, exp = reference_quantise(x, block_rows)
    assert torch.equal(t.scales.cpu().int() - 127, exp.int())
    got = t.dequantize().double().cpu()
    assert torch.equal(got.isnan(), ref.isnan()) and torch.equal(got.isnan(), ~torch.isfinite(x))
    assert torch.equal(got.nan_to_num(0.0), ref.nan_to_num(0.0))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantiser_many_rows(dtype):
    x = torch.randn(16385, 1152, generator=torch.Generator().manual_seed(0)).to(dtype)
    t = ops.fp8_quantize(x.cuda())
    ref, exp = reference_quantise(x, 1)
    assert torch.equal(t.scales.cpu().int() - 127, exp.int()) and torch.equal(t.dequantize().double().cpu(), ref)
