"""Where the outputs of the decaying linear attention may lie: in place of q; nowhere that another row still reads."""
import pytest
import torch

from sana_b200 import ops
from sana_b200._lib import SanaLibraryError

BF16, F32 = torch.bfloat16, torch.float32


def rows(n, H, D, dtype, Hk=None, device="cuda"):
    Hk = Hk or H
    qkv = torch.randn(n, (H + 2 * Hk) * D, generator=torch.Generator().manual_seed(n + H + D)).to(dtype).to(device)
    return qkv[:, :H * D], qkv[:, H * D:(H + Hk) * D], qkv[:, (H + Hk) * D:]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,N,H,Hk,D", [(2, 60, 3, 3, 48), (2, 333, 4, 2, 64), (1, 1500, 2, 1, 112), (3, 700, 2, 2, 128), (2, 500, 8, 4, 32)])
def test_outputs_in_place_of_q(dtype, B, N, H, Hk, D):
    q, k, v = rows(B * N, H, D, dtype, Hk)
    ld = -torch.rand(H).cuda()
    lengths = torch.tensor([N, N // 3, 0][:B], dtype=torch.int32).cuda()
    for kw in (dict(), dict(lengths=lengths), dict(relu=True, eps=1e-6)):
        want, st = ops.la_decay(q, k, v, ld, B, N, H, D, **kw)
        hold = torch.cat([q, k, v], 1)
        q2, k2, v2 = hold[:, :H * D], hold[:, H * D:(H + Hk) * D], hold[:, (H + Hk) * D:]
        out, st2 = ops.la_decay(q2, k2, v2, ld, B, N, H, D, out=q2, **kw)
        assert out.data_ptr() == q2.data_ptr() and torch.equal(out, want) and torch.equal(st, st2)
        assert torch.equal(k2, k) and torch.equal(v2, v)
    one = [t[:B].clone() for t in (q, k, v)]
    state = st.clone()
    want = ops.la_decay_step(*one, ld, st, H, D)
    got = ops.la_decay_step(*one, ld, state, H, D, out=one[0])
    assert torch.equal(got, want) and torch.equal(state, st)


def test_what_counts_as_an_overlap():
    buf = torch.zeros(20, 96)
    f = ops._rows_overlap
    assert not f(buf[:, :32], buf[:, 32:64]) and not f(buf[:, 64:], buf[:, :32])  # column blocks of one projection
    assert f(buf[:, :32], buf[:, 31:64]) and f(buf[:, 16:48], buf[:, 40:72]) and f(buf, buf[:, 5:6])
    assert not f(buf[:10], buf[10:]) and f(buf[:11], buf[10:]) and f(buf[:10, :32], buf[1:11, :32])
    assert not f(buf[:10, :32], buf[1:11, 32:64]) and not f(buf[1:11, :32], buf[:10, 64:])
    assert f(buf.view(10, 192)[:, :40], buf[:, :10])  # other strides in the same memory: taken to meet
    assert not f(torch.zeros(4, 8), torch.zeros(4, 8))
    assert not f(buf[3:4, :32], buf[3:4, 32:]) and f(buf[3:4, :33], buf[3:4, 32:])
    wrap = torch.zeros(200).as_strided((5, 30), (30, 1))
    assert not f(wrap[1:3], wrap[3:]) and f(wrap[1:3], wrap[2:])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_outputs_over_other_inputs_are_refused(dtype):
    B, N, H, D = 2, 40, 2, 32
    hold = torch.randn(B * N + 1, 3 * H * D, device="cuda").to(dtype)
    part = lambda r, c: hold[r:r + B * N, c * H * D:(c + 1) * H * D]
    q, k, v = part(0, 0), part(0, 1), part(0, 2)
    ld = -torch.rand(H).cuda()
    before = hold.clone()
    for out in (k, v, part(1, 0), part(1, 2), hold[:B * N, H * D // 2:H * D // 2 + H * D]):
        with pytest.raises(SanaLibraryError, match="overlap"):
            ops.la_decay(q, k, v, ld, B, N, H, D, out=out)
        with pytest.raises(SanaLibraryError, match="overlap"):
            ops.la_decay_step(q, k, v, ld, torch.zeros(B * N, H, D + 1, D, device="cuda"), H, D, out=out)
    one = torch.zeros(1, H * D, dtype=dtype, device="cuda").expand(B * N, H * D)
    with pytest.raises(SanaLibraryError):
        ops.la_decay(q, k, v, ld, B, N, H, D, out=one)
    assert torch.equal(hold, before)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_the_stride_of_a_single_row_is_not_looked_at(dtype):
    H, D = 2, 32
    odd = lambda n: torch.randn(1, n + 13, device="cuda").to(dtype)[:, :n]  # stride n + 13
    q, k, v, ld = odd(H * D), odd(H * D), odd(H * D), -torch.rand(H).cuda()
    want, st = ops.la_decay(q.contiguous(), k.contiguous(), v.contiguous(), ld, 1, 1, H, D)
    out, st2 = ops.la_decay(q, k, v, ld, 1, 1, H, D, out=odd(H * D))
    assert torch.equal(out, want) and torch.equal(st, st2)
    assert torch.equal(ops.la_decay_step(q, k, v, ld, st, H, D, out=odd(H * D)), ops.la_decay_step(q, k, v, ld, st2, H, D))
    x, w = odd(144), ops.fp8_quantize(torch.randn(24, 144, device="cuda").to(dtype), 128)
    a, b = ops.fp8_quantize(x), ops.fp8_quantize(x.contiguous())
    assert torch.equal(a.dequantize(), b.dequantize())
    o = torch.zeros(1, 37, dtype=BF16, device="cuda")[:, :24]
    r = torch.randn(1, 37, device="cuda").to(BF16)[:, :24]
    assert torch.equal(ops.gemm_fp8(a, w, residual=r, out=o), ops.gemm_fp8(b, w, residual=r.contiguous()))
