"""The normaliser of the decaying linear attention: the key sum carried from earlier tokens enters it with more than a
bf16 value's bits, in every kernel."""
import pytest
import torch

from sana_b200 import ops

BF16, F32 = torch.bfloat16, torch.float32


def carried(B, N, H, D, dtype):
    """q > 0, keys whose features are zeros, no decay: every output is (row of the state) / (key sum) = 1 / z.  1 / z is the
    bf16 value 1 - 2^-8, while z = 1.0039... lies next to the middle between two bf16 values (1 and 1 + 2^-7)."""
    g = torch.Generator().manual_seed(B + N + H + D)
    q = (torch.rand(B * N, H * D, generator=g) + 0.5).to(dtype).cuda()
    k = -torch.rand(B * N, H * D, generator=g).to(dtype).cuda() - 0.5
    v = torch.randn(B * N, H * D, generator=g).to(dtype).cuda()
    want = 1 - 2.0 ** -8
    prior = torch.ones(B, H, D + 1, D)
    prior[:, :, D] = 1 / want
    return q, k, v, torch.zeros(H, device="cuda"), prior.cuda(), want


def exactly(out, want, dtype):
    """bf16: the key sum as two terms is off by 2^-17 of it, the sums by D * 2^-23 <= 2^-16, and the value wanted is a bf16
    value, half a step (2^-9) from the next border: rounding has to return it.  fp32: the sums alone."""
    if dtype == BF16:
        assert (out == want).all(), out.float().flatten()[:4].tolist()
    else:
        assert ((out - want).abs() <= 2.0 ** -16).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("D", [16, 32, 48, 64, 80, 96, 112, 128])
@pytest.mark.parametrize("N", [1, 64, 65, 300])
def test_the_carried_key_sum_keeps_its_bits(dtype, D, N):
    q, k, v, ld, prior, want = carried(1, N, 3, D, dtype)
    out, state = ops.la_decay(q, k, v, ld, 1, N, 3, D, relu=True, eps=0.0, prior=prior)
    exactly(out, want, dtype)
    assert torch.equal(state, prior)
    if N == 1:
        exactly(ops.la_decay_step(q, k, v, ld, prior.clone(), 3, D, relu=True, eps=0.0), want, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("B,N,H,D", [(4, 200, 80, 32), (4, 200, 74, 64), (4, 200, 74, 112), (1, 1500, 2, 32), (1, 1500, 2, 64),
                                     (1, 1500, 2, 112), (1, 1500, 2, 128)])
def test_in_one_launch_and_in_segments(B, N, H, D):
    q, k, v, ld, prior, want = carried(B, N, H, D, BF16)
    out, state = ops.la_decay(q, k, v, ld, B, N, H, D, relu=True, eps=0.0, prior=prior)
    exactly(out, want, BF16)
    assert torch.equal(state, prior)
