"""8-bit projections with a power-of-two scale for each block of 128: the quantiser against its definition (bit for
bit), the product against 64-bit arithmetic on the dequantised operands."""
import pytest
import torch

from sana_b200 import ops
from sana_b200._lib import SanaLibraryError

BF16_HALF_STEP = torch.finfo(torch.bfloat16).eps / 2


def reference_quantise(x, block_rows):
    """(values in fp64, exponents) from the definition, on the CPU."""
    x = x.detach().double().cpu()
    R, K = x.shape
    fin = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x))
    a = torch.nn.functional.pad(fin, (0, -K % 128, 0, -R % block_rows))
    amax = a.reshape(a.shape[0] // block_rows, block_rows, -1, 128).amax(dim=(1, 3))
    m, e = torch.frexp(amax)  # amax = m 2^e, m in [0.5, 1);  448 = 0.875 * 2^9
    exp = (e - 9 + (m > 0.875)).clamp(min=-126)
    exp = torch.where(amax > 0, exp, torch.full_like(exp, -126))
    wide = exp.repeat_interleave(block_rows, 0)[:R].repeat_interleave(128, 1)[:, :K]
    y = torch.where(torch.isfinite(x), torch.ldexp(x, -wide), torch.full_like(x, float("nan")))
    return torch.ldexp(y.float().to(torch.float8_e4m3fn).double(), wide), exp


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("rows,K", [(1, 16), (1, 128), (3, 144), (128, 256), (129, 2240), (300, 5600), (77, 1152)])
def test_quantiser_is_exact(dtype, block_rows, rows, K):
    g = torch.Generator().manual_seed(rows * 7 + K)
    x = torch.randn(rows, K, generator=g) * torch.exp2(torch.randint(-20, 20, (rows, 1), generator=g).float())
    x[0, :16] = 0
    if K >= 128:
        x[rows // 2, :128] = 0  # a block of zeros
    x = x.to(dtype).cuda()
    t = ops.fp8_quantize(x, block_rows)
    ref, exp = reference_quantise(x, block_rows)
    assert torch.equal(t.scales.cpu().int() - 127, exp.int())
    assert torch.equal(t.dequantize().double().cpu(), ref)


@pytest.mark.gpu
def test_quantiser_borders_and_non_finite_values():
    inf, nan, big = float("inf"), float("nan"), torch.finfo(torch.float32).max
    rows = [[448.0, 1.0], [448.0000305, 1.0], [447.99, -3.0], [2.0 ** -149, 0.0], [2.0 ** -118, 2.0 ** -126], [big, -big],
            [inf, 5.0], [nan, -2.0], [-inf, nan], [0.0, -0.0], [1e-30, inf], [896.0, 896.1]]
    x = torch.zeros(len(rows), 32)
    for i, r in enumerate(rows):
        x[i, 3], x[i, 17] = r
    t = ops.fp8_quantize(x.cuda())
    ref, exp = reference_quantise(x, 1)
    assert torch.equal(t.scales.cpu().int() - 127, exp.int())
    got = t.dequantize().double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(ref)) and torch.equal(torch.isnan(got), ~torch.isfinite(x))
    # dequantize() gives fp32: the largest fp32 value rounds up to 2^128, an infinity there
    same = (got == ref.float().double()) | torch.isnan(ref)
    assert same.all(), x[~same].tolist()


@pytest.mark.gpu
def test_quantiser_strided_rows():
    x = torch.randn(65, 640, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    for br in (1, 128):
        a, b = ops.fp8_quantize(x[:, 128:400], br), ops.fp8_quantize(x[:, 128:400].contiguous(), br)
        assert torch.equal(a.q.view(torch.uint8), b.q.view(torch.uint8)) and torch.equal(a.scales, b.scales)


def product_bound(a, w, acc_terms):
    """|error| of the fp32 sum of products before the epilogue, per element: each of the K products and additions is off
    by at most one fp32 step relative to the sum of magnitudes (the tensor core may truncate: a whole step, not half)."""
    return (a.abs() @ w.abs().T) * acc_terms * torch.finfo(torch.float32).eps


def check(out, a, w, bias=None, act=0, gate=None, residual=None):
    ad, wd = a.dequantize().double(), w.dequantize().double()
    z = ad @ wd.T
    slack = product_bound(ad, wd, a.K)
    if bias is not None:
        z = z + bias.double()
    slack = slack + z.abs() * 4 * torch.finfo(torch.float32).eps
    if act == ops.ACT_SILU:
        z = z * torch.sigmoid(z)
        slack = 1.1 * slack + z.abs() * 2.0 ** -18  # |silu'| < 1.1; the fast exponential and reciprocal: 2^-20 each
    elif act == ops.ACT_GELU_TANH:
        z = torch.nn.functional.gelu(z, approximate="tanh")
        slack = 1.13 * slack + 2.0 ** -20 * (1 + z.abs())  # |gelu'| < 1.13
    if gate is not None:
        table, t, row, rows = gate
        N = wd.shape[0]
        img = torch.arange(z.shape[0], device=z.device) // rows
        gv = table[row].double() + t.double().reshape(-1, 6, N)[img, row]
        z, slack = z * gv, slack * gv.abs()
    if residual is not None:
        z = z + residual.double()
    slack = slack + z.abs() * 4 * torch.finfo(torch.float32).eps
    bad = (out.double() - z).abs() > z.abs() * BF16_HALF_STEP * (1 + 1e-3) + slack + 2.0 ** -130
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} elements off, e.g. {(out.double() - z)[bad][:4].tolist()} of {z[bad][:4].tolist()}"
    assert ops.take_gemm_fp8_device_status() == 0


def operands(M, N, K, seed=0, block=128, spread=True):
    g = torch.Generator().manual_seed(seed + 31 * M + 7 * N + K)
    x = torch.randn(M, K, generator=g)
    w = torch.randn(N, K, generator=g) / K ** 0.5
    if spread:  # scales that differ from row to row and from block to block
        x = x * torch.exp2(torch.randint(-6, 7, (M, (K + 127) // 128), generator=g).float()).repeat_interleave(128, 1)[:, :K]
        w = w * torch.exp2(torch.randint(-6, 7, (N, (K + 127) // 128), generator=g).float()).repeat_interleave(128, 1)[:, :K]
    return ops.fp8_quantize(x.bfloat16().cuda()), ops.fp8_quantize(w.bfloat16().cuda(), block), g


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 2, 7, 8, 9, 16, 17, 31, 33, 64, 65, 127, 128, 129, 300, 2048, 2305])
@pytest.mark.parametrize("N,K", [(8, 16), (136, 144), (256, 128), (264, 512), (520, 656), (384, 2240)])
def test_product_matches_64_bits(M, N, K):
    a, w, _ = operands(M, N, K)
    check(ops.gemm_fp8(a, w), a, w)


@pytest.mark.gpu
@pytest.mark.parametrize("block_a,block_w", [(1, 1), (128, 1), (128, 128)])
@pytest.mark.parametrize("M", [5, 200, 2100])
def test_scale_granularities(M, block_a, block_w):
    g = torch.Generator().manual_seed(5)
    N, K = 392, 1040
    x = torch.randn(M, K, generator=g) * torch.exp2(torch.randint(-5, 6, (M, 1), generator=g).float())
    w = torch.randn(N, K, generator=g) * torch.exp2(torch.randint(-5, 6, (N, 1), generator=g).float())
    a, wq = ops.fp8_quantize(x.cuda(), block_a), ops.fp8_quantize(w.cuda(), block_w)
    check(ops.gemm_fp8(a, wq), a, wq)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 13, 150, 2240])
@pytest.mark.parametrize("act", [ops.ACT_NONE, ops.ACT_SILU, ops.ACT_GELU_TANH])
def test_epilogue(M, act):
    N, K = 328, 400
    a, w, g = operands(M, N, K, spread=False)
    bias = torch.randn(N, generator=g).bfloat16().cuda()
    rows = (M + 1) // 2
    gate = (torch.randn(6, N, generator=g).bfloat16().cuda(), torch.randn(2, 6 * N, generator=g).bfloat16().cuda(), 2, rows)
    big = torch.randn(M, 2 * N, generator=g).bfloat16().cuda()
    check(ops.gemm_fp8(a, w, bias=bias, act=act), a, w, bias, act)
    check(ops.gemm_fp8(a, w, bias=bias, act=act, gate=gate, residual=big[:, N:]), a, w, bias, act, gate, big[:, N:])
    dst = torch.full((M + 2, 2 * N), 3.0, dtype=torch.bfloat16, device="cuda")
    ops.gemm_fp8(a, w, bias=bias, act=act, out=dst[1:M + 1, :N])  # a view: what surrounds it stays
    check(dst[1:M + 1, :N], a, w, bias, act)
    assert (dst[0] == 3).all() and (dst[-1] == 3).all() and (dst[:, N:] == 3).all()


@pytest.mark.gpu
@pytest.mark.parametrize("M", [3, 140, 2050])
def test_relu_columns_and_in_place_residual(M):
    a, w, g = operands(M, 256, 272, spread=False)
    y = ops.gemm_fp8(a, w, act=ops.ACT_RELU_COLS, relu_cols=100)
    z = ops.gemm_fp8(a, w)
    assert torch.equal(y[:, :100], z[:, :100].clamp(min=0)) and torch.equal(y[:, 100:], z[:, 100:])
    r = torch.randn(M, 256, generator=g).bfloat16().cuda()
    want = ops.gemm_fp8(a, w, residual=r)
    got = r.clone()
    ops.gemm_fp8(a, w, residual=got, out=got)
    assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [4, 40, 200, 2100])
def test_nan_reaches_its_row_and_column_only(M):
    N, K = 264, 288
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(2))
    w = torch.randn(N, K, generator=torch.Generator().manual_seed(3))
    x[M // 2, 200] = float("inf")
    w[77, 3] = float("nan")
    a, wq = ops.fp8_quantize(x.cuda()), ops.fp8_quantize(w.cuda(), 128)
    bad = torch.isnan(ops.gemm_fp8(a, wq))
    want = torch.zeros_like(bad)
    want[M // 2] = True
    want[:, 77] = True
    assert torch.equal(bad, want)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [8, 256, 4096])
def test_zero_rows_and_extreme_scales(M):
    N, K = 256, 384
    g = torch.Generator().manual_seed(9)
    x, w = torch.randn(M, K, generator=g) * 1e30, torch.randn(N, K, generator=g) * 1e-30
    x[1] = 0
    w[:, 128:256] = 0
    a, wq = ops.fp8_quantize(x.cuda()), ops.fp8_quantize(w.cuda(), 128)
    out = ops.gemm_fp8(a, wq)
    check(out, a, wq)
    assert (out[1] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 16, 40, 2100])
def test_a_scale_of_255_is_nan(M):
    """E8M0's NaN in a caller's own scales reaches exactly the outputs that its block enters."""
    K, N = 384, 144
    g = torch.Generator().manual_seed(3)
    a = ops.fp8_quantize(torch.randn(M, K, generator=g).to(torch.bfloat16).cuda())
    w = ops.fp8_quantize(torch.randn(N, K, generator=g).to(torch.bfloat16).cuda(), 128)
    sa, sw = a.scales.clone(), w.scales.clone()
    sa[M // 2, 1] = 255
    sw[1, 2] = 255  # rows 128 .. 143 of the weight
    out = ops.gemm_fp8(ops.Fp8Tensor(a.q, sa), ops.Fp8Tensor(w.q, sw, 128))
    want = torch.zeros(M, N, dtype=torch.bool, device="cuda")
    want[M // 2] = True
    want[:, 128:] = True
    assert torch.equal(out.isnan(), want)
    assert ops.Fp8Tensor(a.q, sa).dequantize().isnan().sum() == 128


@pytest.mark.gpu
@pytest.mark.parametrize("M", [5, 700, 3000])
def test_replays_from_a_graph_and_on_another_stream(M):
    N, K = 520, 1152
    g = torch.Generator().manual_seed(4)
    x = torch.randn(M, K, generator=g).bfloat16().cuda()
    w = ops.fp8_quantize(torch.randn(N, K, generator=g).bfloat16().cuda(), 128)
    want = ops.gemm_fp8(ops.fp8_quantize(x), w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.gemm_fp8(ops.fp8_quantize(x), w)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    graphs, outs = [], []
    for _ in range(2):  # two captured graphs side by side
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(ops.gemm_fp8(ops.fp8_quantize(x), w))
        graphs.append(gr)
    x.copy_(-x)
    for gr in graphs:
        gr.replay()
    assert torch.equal(outs[0], -want) and torch.equal(outs[1], -want)


def test_refusals_on_the_host():
    codes = torch.zeros(16, 256).to(torch.float8_e4m3fn)
    with pytest.raises(SanaLibraryError, match="CUDA"):
        ops.fp8_quantize(torch.zeros(4, 128))
    with pytest.raises(SanaLibraryError, match="codes"):
        ops.Fp8Tensor(codes.float(), torch.zeros(16, 2, dtype=torch.uint8))
    with pytest.raises(SanaLibraryError, match="codes"):
        ops.Fp8Tensor(codes[:, :128], torch.zeros(16, 1, dtype=torch.uint8))
    with pytest.raises(SanaLibraryError, match="scales"):
        ops.Fp8Tensor(codes, torch.zeros(16, 1, dtype=torch.uint8))
    with pytest.raises(SanaLibraryError, match="scales"):
        ops.Fp8Tensor(codes, torch.zeros(16, 2))
    with pytest.raises(SanaLibraryError, match="block_rows"):
        ops.Fp8Tensor(codes, torch.zeros(16, 2, dtype=torch.uint8), block_rows=64)
    t = ops.Fp8Tensor(codes, torch.zeros(16, 2, dtype=torch.uint8))
    assert t.scales.stride(0) == 4  # padded to whole words
    with pytest.raises(SanaLibraryError, match="K mismatch"):
        ops.gemm_fp8(t, ops.Fp8Tensor(codes[:, :128].contiguous(), torch.zeros(16, 1, dtype=torch.uint8)))


def test_refusals_of_the_c_entry_points(lib):
    import ctypes as C

    from sana_b200 import _lib
    p, bf = C.c_void_p(0x1000), _lib.SANA_BF16
    assert lib.sana_fp8_quantize(None, 128, p, p, 4, 8, 128, 1, bf, None) == -1
    assert lib.sana_fp8_quantize(p, 128, p, p, 4, 8, 120, 1, bf, None) == -1  # K % 16
    assert lib.sana_fp8_quantize(p, 128, p, p, 4, 8, 128, 2, bf, None) == -1  # block_rows
    assert lib.sana_fp8_quantize(p, 100, p, p, 4, 8, 128, 1, bf, None) == -1  # ld < K
    assert lib.sana_fp8_quantize(p, 132, p, p, 4, 8, 128, 1, bf, None) == -1  # rows not 16-byte aligned
    assert lib.sana_fp8_quantize(p, 256, p, p, 1, 8, 256, 1, bf, None) == -1  # ldsf < blocks
    assert lib.sana_fp8_quantize(p, 128, p, p, 4, 8, 128, 1, 9, None) == -1  # dtype
    assert lib.sana_fp8_quantize(C.c_void_p(0x1004), 128, p, p, 4, 8, 128, 1, bf, None) == -1
    ok = [p, p, 4, 1, p, p, 4, 128, p, 64, 8, 64, 128, None, None]

    def refused(i, v):
        a = list(ok)
        a[i] = v
        return lib.sana_gemm_fp8(*a) == -1

    assert refused(0, None) and refused(8, None)
    assert refused(2, 2) and refused(2, 6) and refused(6, 0)  # scale strides
    assert refused(1, C.c_void_p(0x1002)) and refused(3, 16) and refused(7, 0)
    assert refused(9, 56) and refused(9, 68) and refused(11, 60) and refused(12, 120) and refused(10, 0)
    assert refused(4, C.c_void_p(0x1008))
    ep = _lib.GemmEpilogue()
    ep.act = 9
    assert refused(13, C.byref(ep))
    assert lib.sana_gemm_fp8_take_device_status(None) == -1
