"""The decayed scores of a prompt meet v with more than a bf16 value's bits: an output of a few tokens would feel their
rounding as much as its own."""
import pytest
import torch

from sana_b200 import ops


def check(B, N, H, Hk, D, relu, lengths=None):
    """No state comes in and N <= 128, so that an output is its scores times v.  With mag the sum of the absolute products,
    relative to it: two bf16 terms 2^-17, a score's D products 2^-15 (D 2^-22, truncated fp32 sums), the power and its
    product 2^-21, 2 N products with v 2^-14; 2^-13 together, once more for the normaliser, and half a step (2^-8) of the
    result for its own rounding.  Heads of 128 channels keep one term (2^-8 at most) for keys 64 and up."""
    g = torch.Generator().manual_seed(B + 3 * N + 5 * H + 7 * D + relu)
    q, k, v = (torch.randn(B * N, h * D, generator=g).bfloat16() for h in (H, Hk, Hk))
    log_decay = -torch.linspace(0, 1.5, H)
    out, _ = ops.la_decay(q.cuda(), k.cuda(), v.cuda(), log_decay.cuda(), B, N, H, D, relu=relu, eps=1e-6 if relu else None,
                          lengths=None if lengths is None else torch.tensor(lengths, dtype=torch.int32).cuda())
    out = out.double().cpu().view(B, N, H, D)
    f = (lambda x: x.clamp(min=0)) if relu else (lambda x: x)
    q, k, v = (x.double().view(B, N, h, D).repeat_interleave(H // h, 2) for x, h in ((f(q), H), (f(k), Hk), (v, Hk)))
    t = torch.arange(N)
    power = torch.exp(log_decay.double()[:, None, None] * (t[:, None] - t).clamp(min=0)) * (t[:, None] >= t)
    p = torch.einsum("bthd,bshd->bhts", q, k) * power
    pa = torch.einsum("bthd,bshd->bhts", q.abs(), k.abs()) * power
    want, mag = torch.einsum("bhts,bshd->bthd", p, v), torch.einsum("bhts,bshd->bthd", pa, v.abs())
    late = torch.einsum("bhts,bshd->bthd", p.abs() * (t >= 64), v.abs()) if D == 128 else torch.zeros_like(mag)
    bound = 2.0 ** -13 * mag + 2.0 ** -8 * late
    if relu:
        den = p.sum(-1).permute(0, 2, 1).unsqueeze(-1) + 1e-6
        want, bound = want / den, bound / den
        bound = bound + 2.0 ** -13 * want.abs()
    bound = bound + 2.0 ** -8 * want.abs() + 1e-30
    for b in range(B):
        m = N if lengths is None else lengths[b]
        worst = ((out[b, :m] - want[b, :m]).abs() / bound[b, :m]).max().item() if m else 0.0
        assert worst <= 1, f"sequence {b}: {worst:.2f} times the bound"
        assert (out[b, m:] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("D", [16, 32, 48, 64, 80, 96, 112, 128])
@pytest.mark.parametrize("N", [33, 64, 65, 77, 96, 128])
def test_scores_keep_their_bits(N, D, relu):
    check(1, N, 5, 5, D, relu)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [32, 64, 112, 128])
def test_shared_heads_and_padded_batches(D):
    check(4, 113, 6, 2, D, True, [113, 0, 1, 70])


@pytest.mark.gpu
@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("D", [16, 48, 64])
@pytest.mark.parametrize("N", [1, 64, 65, 128])
def test_the_carried_state_keeps_its_bits(N, D, relu):
    """Keys without features: an output is the state that came in times q.  Two bf16 terms of the state 2^-17 of the sum of the
    absolute products, D truncated fp32 sums of two products each 2^-15, the power 2^-21: 2^-14 together, and half a step
    (2^-8) of the result.  (Widths without room for a second term: see the header.)"""
    B, H = 2, 5
    g = torch.Generator().manual_seed(N + 7 * D + relu)
    q = torch.randn(B * N, H * D, generator=g).bfloat16()
    v = torch.randn(B * N, H * D, generator=g).bfloat16()
    prior = torch.randn(B, H, D + 1, D, generator=g)
    log_decay = -torch.linspace(0, 0.02, H)
    out, state = ops.la_decay(q.cuda(), torch.zeros_like(q).cuda(), v.cuda(), log_decay.cuda(), B, N, H, D, scale=1.0, relu=relu,
                              prior=prior.cuda())
    f = q.double().view(B, N, H, D)
    f = f.clamp(min=0) if relu else f
    power = torch.exp(log_decay.double() * torch.arange(1, N + 1)[:, None])[None, :, :, None]
    want = torch.einsum("bthd,bhed->bthe", f, prior[:, :, :D].double()) * power
    mag = torch.einsum("bthd,bhed->bthe", f.abs(), prior[:, :, :D].double().abs()) * power
    bound = 2.0 ** -14 * mag + 2.0 ** -8 * want.abs() + 1e-30
    worst = ((out.double().cpu().view(B, N, H, D) - want).abs() / bound).max().item()
    assert worst <= 1, f"{worst:.2f} times the bound"
