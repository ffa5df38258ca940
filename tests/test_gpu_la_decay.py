"""Causal linear attention with a decay for each head: prompts and single tokens against the recurrence in 64 bits."""
import math

import pytest
import torch

from sana_b200 import ops
from sana_b200._lib import SanaLibraryError

BF16, F32 = torch.bfloat16, torch.float32


def reference(q, k, v, log_decay, B, N, H, D, scale=1.0, relu=False, eps=None, prior=None, lengths=None):
    """(out, state, magnitude of out, magnitude of state) in fp64 from the definition, token by token.  The magnitudes are
    the same sums over absolute values, to which rounding errors are relative."""
    Hk = k.shape[1] // D
    q = q.double().cpu().reshape(B, N, H, D)
    k = k.double().cpu().reshape(B, N, Hk, D).repeat_interleave(H // Hk, 2)
    v = v.double().cpu().reshape(B, N, Hk, D).repeat_interleave(H // Hk, 2)
    if relu:
        q, k = q.clamp(min=0), k.clamp(min=0)
    v = torch.cat([v, torch.ones(B, N, H, 1, dtype=torch.float64)], -1)
    lam = torch.exp(log_decay.double().cpu())[:, None, None]
    S = prior.double().cpu().clone() if prior is not None else torch.zeros(B, H, D + 1, D, dtype=torch.float64)
    M = S.abs()
    out, mag = torch.zeros(B, N, H, D, dtype=torch.float64), torch.zeros(B, N, H, D, dtype=torch.float64)
    n = lengths.cpu().clamp(0, N).tolist() if lengths is not None else [N] * B
    for t in range(N):
        on = torch.tensor([t < x for x in n])
        if not on.any():
            break
        add = v[:, t, :, :, None] * k[:, t, :, None]
        S = torch.where(on[:, None, None, None], lam * S + add, S)
        M = torch.where(on[:, None, None, None], lam * M + add.abs(), M)
        o, a = (S @ q[:, t, :, :, None])[..., 0], (M @ q[:, t, :, :, None].abs())[..., 0]
        if eps is not None:
            den = o[..., D:] + eps
            o, a = o[..., :D] / den, a[..., :D] / den
        else:
            o, a = o[..., :D] * scale, a[..., :D] * abs(scale)
        out[:, t] = torch.where(on[:, None, None], o, out[:, t])
        mag[:, t] = torch.where(on[:, None, None], a, mag[:, t])
    return out.reshape(B * N, H * D), S, mag.reshape(B * N, H * D), M


def make(B, N, H, D, dtype, Hk=None, seed=0, prior=False, relu=False):
    Hk = Hk or H
    g = torch.Generator().manual_seed(seed + 1000 * B + 10 * N + H + D)
    qkv = torch.randn(B * N, (H + 2 * Hk) * D, generator=g).to(dtype).cuda()
    ld = -torch.exp2(-6 * torch.rand(H, generator=g)).cuda()
    p = None
    if prior:
        p = torch.randn(B, H, D + 1, D, generator=g)
        p = (p.abs() if relu else p).cuda()
    return qkv[:, :H * D], qkv[:, H * D:(H + Hk) * D], qkv[:, (H + Hk) * D:], ld, p


def close(got, want, mag, dtype, what, fp32_terms):
    """Rounding to the type (half a step of the value), plus what the sums may lose relative to their magnitudes:
    fp32: `fp32_terms` steps of 2^-24; bf16 outputs also one rounding of each score (2^-8 of it at most) and the state
    as two bf16 terms (2^-16)."""
    u = 2.0 ** -24
    tol = mag * (fp32_terms * u)
    if dtype == BF16:
        tol = tol + mag * (2.0 ** -8 + 2.0 ** -16) + want.abs() * 2.0 ** -8
    tol = tol * 1.01 + 1e-30
    d = (got.double().cpu() - want).abs()
    assert not torch.isnan(d).any(), what
    worst = (d / tol).max().item()
    assert worst <= 1, f"{what}: {worst} times the bound"


def state_tol(n_tokens, dtype):
    # three bf16 terms of a weighted v leave 2^-24 of it; powers from expf (2^-22 with the rounding of the exponent's
    # argument, up to 88 * 2^-24 for a power that has decayed to 2^-127 - those weigh nothing); sums of at most a chunk's
    # tokens and one multiply-add a chunk
    return 64 + 4 * math.ceil(n_tokens / 32)


def run_case(B, N, H, D, dtype, Hk=None, relu=False, eps=None, prior=False, lengths=None, scale=1.0, seed=0):
    q, k, v, ld, p = make(B, N, H, D, dtype, Hk, seed, prior, relu)
    n = torch.tensor(lengths, dtype=torch.int32).cuda() if lengths is not None else None
    out, st = ops.la_decay(q, k, v, ld, B, N, H, D, scale=scale, relu=relu, eps=eps, prior=p, lengths=n)
    ro, rs, mo, ms = reference(q, k, v, ld, B, N, H, D, scale, relu, eps, p, n)
    terms = state_tol(N, dtype) + 2 * D
    close(st, rs, ms, F32, "state", state_tol(N, dtype))
    close(out, ro, 2 * mo if eps is not None else mo, dtype, "out", terms)
    assert ops.take_la_decay_device_status() == 0
    if lengths is not None:
        for b, m in enumerate(lengths):
            assert (out[b * N + max(0, m):(b + 1) * N] == 0).all()
    return out, st


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("D", [16, 32, 48, 64, 80, 96, 112, 128])
@pytest.mark.parametrize("N", [1, 2, 15, 33, 64, 65, 130])
def test_widths_and_lengths(dtype, D, N):
    run_case(2, N, 3, D, dtype, prior=N % 2 == 1)
    run_case(1, N, 5, D, dtype, relu=True, eps=1e-6, prior=N % 2 == 0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("D,H,Hk", [(32, 6, 3), (64, 8, 2), (112, 4, 1), (16, 7, 7)])
def test_shared_key_value_heads_and_ragged_batches(dtype, D, H, Hk):
    run_case(5, 150, H, D, dtype, Hk=Hk, relu=True, eps=1e-8, prior=True, lengths=[0, 1, 150, 64, 97])
    run_case(4, 70, H, D, dtype, Hk=Hk, lengths=[70, 0, 500, -3], scale=D ** -0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("D,N", [(32, 3000), (64, 2111), (112, 1500), (128, 1025)])
def test_long_sequences_in_segments(dtype, D, N):
    assert ops._lib.load().sana_la_decay_workspace_bytes(1, N, 2, D, ops._dtype_code(dtype)) > 0  # cut into segments
    run_case(1, N, 2, D, dtype, relu=True, eps=1e-8, prior=True)
    run_case(2, N, 2, D, dtype, prior=True, lengths=[N // 3, N - 1], scale=0.25)


@pytest.mark.gpu
@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("B,N,H,Hk,D", [(4, 4096, 16, 8, 64), (4, 4096, 16, 16, 48), (2, 8192, 20, 20, 32), (8, 2048, 20, 20, 112)])
def test_many_segments_give_the_same_bits_every_time(B, N, H, Hk, D, relu):
    """More segments than multiprocessors, slow decays (nothing that goes wrong on the way is forgotten), and the chunks of
    a segment against single tokens: the state of a few heads in 64 bits."""
    q, k, v, _, p = make(B, N, H, D, BF16, Hk, prior=True, relu=relu)
    ld = -torch.exp2(-torch.linspace(4, 14, H)).cuda()
    lengths = torch.tensor([N - 77 * b for b in range(B)], dtype=torch.int32).cuda()
    kw = dict(relu=relu, eps=1e-8 if relu else None, prior=p)
    for n in (lengths, None):
        out, st = ops.la_decay(q, k, v, ld, B, N, H, D, lengths=n, **kw)
        for _ in range(8):
            o2, s2 = ops.la_decay(q, k, v, ld, B, N, H, D, lengths=n, **kw)
            assert torch.equal(o2, out) and torch.equal(s2, st)
        for b in (0, B - 1):
            m = int(lengths[b]) if n is not None else N
            for h in (0, H // 2, H - 1):
                hk = h // (H // Hk)
                rows = slice(b * N, b * N + m)
                f = k[rows, hk * D:(hk + 1) * D].double()
                f = f.clamp(min=0) if relu else f
                v1 = torch.cat([v[rows, hk * D:(hk + 1) * D].double(), torch.ones(m, 1, dtype=torch.float64, device="cuda")], 1)
                w = torch.exp(ld[h].double() * torch.arange(m - 1, -1, -1, device="cuda"))[:, None]
                whole = torch.exp(ld[h].double() * m)
                want, mag = v1.T @ (w * f) + whole * p[b, h].double(), v1.abs().T @ (w * f.abs()) + whole * p[b, h].double().abs()
                close(st[b, h], want.cpu(), mag.cpu(), F32, (b, h), state_tol(N, BF16))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("D", [32, 112])
def test_decays_from_none_to_total(dtype, D):
    B, N, H = 1, 200, 6
    q, k, v, _, p = make(B, N, H, D, dtype, prior=True, relu=True)
    ld = torch.tensor([0.0, -1e-4, -0.7, -12.0, -300.0, -float("inf")]).cuda()
    for kw in (dict(), dict(relu=True, eps=1e-8)):
        out, st = ops.la_decay(q, k, v, ld, B, N, H, D, prior=p, **kw)
        ro, rs, mo, ms = reference(q, k, v, ld, B, N, H, D, prior=p, **kw)
        close(st, rs, ms, F32, "state", state_tol(N, dtype))
        close(out, ro, 2 * mo if kw else mo, dtype, "out", state_tol(N, dtype) + 2 * D)


@pytest.mark.gpu
def test_without_decay_the_state_is_the_plain_one():
    B, N, H, D = 2, 333, 4, 32
    q, k, v, _, _ = make(B, N, H, D, BF16)
    _, st = ops.la_decay(q, k, v, torch.zeros(H, device="cuda"), B, N, H, D, relu=True, eps=1e-8)
    want = ops.la_state(k, v, B, N, H)
    kd, vd = k.double().abs().reshape(B, N, H, D), v.double().abs().reshape(B, N, H, D)
    mag = torch.cat([torch.einsum("bnhi,bnhj->bhij", vd, kd), kd.sum(1)[:, :, None]], 2)
    assert ((st - want).abs().double() <= mag * (2 * state_tol(N, BF16) * 2.0 ** -24)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_behind_a_sequence_are_not_read(dtype):
    B, N, H, D = 3, 100, 2, 64
    lens = [40, 0, 100]
    q, k, v, ld, p = make(B, N, H, D, dtype, prior=True, relu=True)
    n = torch.tensor(lens, dtype=torch.int32).cuda()
    a = ops.la_decay(q, k, v, ld, B, N, H, D, relu=True, eps=1e-8, prior=p, lengths=n)
    for t in (q, k, v):
        for b, m in enumerate(lens):
            t[b * N + m:(b + 1) * N] = float("nan")
    b_ = ops.la_decay(q, k, v, ld, B, N, H, D, relu=True, eps=1e-8, prior=p, lengths=n)
    assert torch.equal(a[0], b_[0]) and torch.equal(a[1], b_[1])
    assert torch.equal(a[1][1], p[1])  # an empty sequence hands its state on


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_non_finite_values_stay_behind_their_token(dtype, bad):
    B, N, H, D = 1, 256, 2, 32
    for which in range(3):
        q, k, v, ld, _ = make(B, N, H, D, dtype)
        clean, _ = ops.la_decay(q, k, v, ld, B, N, H, D)
        (q, k, v)[which][100, D + 3] = bad  # head 1
        out, st = ops.la_decay(q, k, v, ld, B, N, H, D)
        assert torch.equal(out[:, :D], clean[:, :D])  # the other head
        assert torch.equal(out[:85], clean[:85])
        assert not torch.isfinite(out[100, D:]).all()
        assert torch.isfinite(st[:, 0]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("D,N,at", [(16, 40, 20), (32, 64, 37), (48, 200, 131), (64, 300, 257), (96, 129, 128), (112, 2000, 1111), (128, 700, 5)])
def test_no_output_depends_on_a_later_token(dtype, D, N, at):
    B, H = 1, 2
    kw = dict(relu=True, eps=1e-8)
    q, k, v, ld, _ = make(B, N, H, D, dtype)
    clean, _ = ops.la_decay(q, k, v, ld, B, N, H, D, **kw)
    for value in (float("nan"), float("-inf"), 1e4):
        for t in (k, v):
            old = t[at:].clone()
            t[at:] = value
            out, st = ops.la_decay(q, k, v, ld, B, N, H, D, **kw)
            assert torch.equal(out[:at], clean[:at])
            assert math.isfinite(value) or not torch.isfinite(st).all() or t is k
            t[at:] = old
        # one channel of one token: its channel from there on, nothing else
        old = v[at, 3].clone()
        v[at, 3] = value
        out, st = ops.la_decay(q, k, v, ld, B, N, H, D, **kw)
        same = torch.ones_like(clean, dtype=torch.bool)
        same[at:, 3] = False
        assert torch.equal(out[same], clean[same])
        if not math.isfinite(value):
            live = (q[at:, :D].float().clamp(min=0) * k[at, :D].float().clamp(min=0)).sum(-1) > 0
            assert not torch.isfinite(out[at:, 3][live]).any() or dtype == F32
            assert torch.isfinite(st[0, 0, [i for i in range(D + 1) if i != 3]]).all() and torch.isfinite(st[0, 1]).all()
        v[at, 3] = old
    assert ops.take_la_decay_device_status() == 0


@pytest.mark.gpu
def test_zero_features_give_zero_outputs():
    B, N, H, D = 1, 90, 2, 48
    q, k, v, ld, _ = make(B, N, H, D, BF16)
    out, st = ops.la_decay(-q.abs(), k, v, ld, B, N, H, D, relu=True, eps=1e-15)
    assert (out == 0).all()
    out, st = ops.la_decay(q, -k.abs(), v, ld, B, N, H, D, relu=True, eps=1e-15)
    assert (out == 0).all() and (st == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_prompt_in_pieces_and_token_by_token(dtype):
    """A prompt cut anywhere, then tokens one at a time, against the whole prompt at once."""
    B, N, H, D, Hk = 2, 150, 4, 64, 2
    q, k, v, ld, _ = make(B, N, H, D, dtype, Hk)
    kw = dict(relu=True, eps=1e-8)
    ro, rs, mo, ms = reference(q, k, v, ld, B, N, H, D, **kw)
    part = lambda t, a, b: t.reshape(B, N, -1)[:, a:b].reshape(B * (b - a), -1)
    outs, st = [], None
    for a, b in ((0, 1), (1, 70), (70, 128)):
        o, st = ops.la_decay(part(q, a, b), part(k, a, b), part(v, a, b), ld, B, b - a, H, D, prior=st, **kw)
        outs.append(o.reshape(B, b - a, -1))
    for t in range(128, N):
        o = ops.la_decay_step(part(q, t, t + 1), part(k, t, t + 1), part(v, t, t + 1), ld, st, H, D, **kw)
        outs.append(o.reshape(B, 1, -1))
    close(torch.cat(outs, 1).reshape(B * N, -1), ro, 2 * mo, dtype, "out", state_tol(N, dtype) + 4 * N + 2 * D)
    close(st, rs, ms, F32, "state", state_tol(N, dtype) + 4 * N)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("D", [16, 32, 48, 64, 80, 96, 112, 128])
def test_step_with_slots(dtype, D):
    B, H, Hk, pool = 7, 4, 2, 12
    q, k, v, ld, _ = make(B, 1, H, D, dtype, Hk)
    g = torch.Generator().manual_seed(D)
    state = torch.randn(pool, H, D + 1, D, generator=g).abs().cuda()
    slots = torch.tensor([3, 11, -1, 0, 7, -1, 5], dtype=torch.int32).cuda()
    for kw in (dict(relu=True, eps=1e-6), dict(scale=0.3), dict(relu=True)):
        before = state.clone()
        out = ops.la_decay_step(q, k, v, ld, state, H, D, slots=slots, **kw)
        for b, s in enumerate(slots.tolist()):
            if s < 0:
                assert (out[b] == 0).all()
                continue
            ro, rs, mo, ms = reference(q[b:b + 1], k[b:b + 1], v[b:b + 1], ld, 1, 1, H, D, prior=before[s:s + 1], **kw)
            close(state[s:s + 1], rs, ms, F32, "state", 4)
            close(out[b:b + 1], ro, 2 * mo, dtype if dtype == F32 else BF16, "out", 2 * D + 8)
        rest = [s for s in range(pool) if s not in slots.tolist()]
        assert torch.equal(state[rest], before[rest])


@pytest.mark.gpu
def test_step_with_bad_or_repeated_slots():
    B, H, D, pool = 6, 2, 32, 4
    q, k, v, ld, _ = make(B, 1, H, D, BF16)
    state = torch.randn(pool, H, D + 1, D).cuda()
    before = state.clone()
    slots = torch.tensor([1, 4, 1, -2, 0, 2 ** 30], dtype=torch.int32).cuda()
    out = ops.la_decay_step(q, k, v, ld, state, H, D, slots=slots)
    for b in (1, 2, 3, 5):
        assert torch.isnan(out[b]).all()
    assert torch.isfinite(out[0]).all() and torch.isfinite(out[4]).all()
    assert torch.equal(state[2:], before[2:])
    once = before.clone()
    ops.la_decay_step(q[:1], k[:1], v[:1], ld, once, H, D, slots=slots[:1])
    assert torch.equal(state[1], once[1])  # the first row that names a slot takes its step


@pytest.mark.gpu
def test_strided_views_and_preallocated_outputs():
    B, N, H, D = 2, 77, 3, 48
    q, k, v, ld, _ = make(B, N, H, D, BF16)
    want = ops.la_decay(q, k, v, ld, B, N, H, D)
    big = torch.full((B * N + 2, 2 * H * D), 5.0, dtype=BF16, device="cuda")
    got = ops.la_decay(q.contiguous(), k, v, ld, B, N, H, D, out=big[1:-1, H * D:])
    assert torch.equal(big[1:-1, H * D:], want[0]) and torch.equal(got[1], want[1])
    assert (big[:, :H * D] == 5).all() and (big[0] == 5).all() and (big[-1] == 5).all()


@pytest.mark.gpu
def test_replays_from_graphs_and_on_another_stream():
    B, N, H, D = 1, 1500, 2, 112  # more than one segment: a workspace
    q, k, v, ld, p = make(B, N, H, D, BF16, prior=True, relu=True)
    kw = dict(relu=True, eps=1e-8, prior=p)
    want = ops.la_decay(q, k, v, ld, B, N, H, D, **kw)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.la_decay(q, k, v, ld, B, N, H, D, **kw)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graphs, res = [], []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            o, st = ops.la_decay(q, k, v, ld, B, N, H, D, **kw)
            o2 = ops.la_decay_step(q[:1], k[:1], v[:1], ld, st, H, D, relu=True, eps=1e-8)
        graphs.append(gr)
        res.append((o, st, o2))
    v.mul_(2)
    p[:, :, :D].mul_(2)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for gr, st in zip(graphs, streams):  # two captured graphs at once: each has its own workspace
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            gr.replay()
    torch.cuda.synchronize()
    assert torch.equal(res[0][0], want[0] * 2) and torch.equal(res[1][0], want[0] * 2)
    assert torch.equal(res[0][2], res[1][2]) and torch.equal(res[0][1], res[1][1])


def cpu_inputs(B=2, N=4, H=2, D=32):
    t = torch.zeros(B * N, H * D)
    return t, t, t, torch.zeros(H), B, N, H, D


def test_refusals_on_the_host():
    with pytest.raises(SanaLibraryError, match="CUDA"):
        ops.la_decay(*cpu_inputs())
    with pytest.raises(SanaLibraryError, match="CUDA"):
        q, k, v, ld, B, N, H, D = cpu_inputs(N=1)
        ops.la_decay_step(q, k, v, ld, torch.zeros(2, 2, 33, 32), H, D)
    chk = ops._decay_inputs
    t = torch.zeros(8, 64)
    ld = torch.zeros(2)
    assert chk("x", t, t, t, ld, 8, 2, 32, False, None) == (64, 64, 64, 2)
    assert chk("x", t, t[:, :32], t[:, 32:], ld, 8, 2, 32, False, None) == (64, 64, 64, 1)
    for bad in (dict(rows=7), dict(H=3), dict(D=24), dict(D=144), dict(k=t[:, :48]), dict(k=t[:4]), dict(v=t[:, :32]),
                dict(v=t.double()), dict(ld=ld.double()), dict(ld=torch.zeros(3)),
                dict(eps=1e-6), dict(relu=True, eps=-1.0), dict(relu=True, eps=float("nan")), dict(q=t.t())):
        a = dict(q=t, k=t, v=t, ld=ld, rows=8, H=2, D=32, relu=False, eps=None)
        a.update(bad)
        with pytest.raises(SanaLibraryError):
            chk("x", a["q"], a["k"], a["v"], a["ld"], a["rows"], a["H"], a["D"], a["relu"], a["eps"])
    with pytest.raises(SanaLibraryError, match="int32"):
        ops._int32_vector(torch.zeros(2, dtype=torch.int64), 2, "lengths")
    with pytest.raises(SanaLibraryError, match="int32"):
        ops._int32_vector(torch.zeros(3, dtype=torch.int32), 2, "lengths")


@pytest.mark.gpu
def test_refusals_with_device_tensors():
    q, k, v, ld, _ = make(2, 8, 2, 32, BF16)
    ok = lambda **kw: ops.la_decay(q, k, v, ld, 2, 8, 2, 32, **kw)
    for kw in (dict(prior=torch.zeros(2, 2, 32, 32).cuda()), dict(prior=torch.zeros(2, 2, 33, 32).double().cuda()),
               dict(lengths=torch.zeros(3, dtype=torch.int32).cuda()), dict(out=torch.zeros(16, 64).cuda()),
               dict(lengths=torch.zeros(2, dtype=torch.int32)), dict(eps=1e-8)):
        with pytest.raises(SanaLibraryError):
            ok(**kw)
    wide = torch.zeros(16, 65 * 3, dtype=BF16).cuda()
    with pytest.raises(SanaLibraryError, match="16-byte"):
        ops.la_decay(wide[:, 1:65], k, v, ld, 2, 8, 2, 32)
    with pytest.raises(SanaLibraryError, match="one entry"):
        ops.la_decay_step(q[:2], k[:2], v[:2], ld, torch.zeros(3, 2, 33, 32).cuda(), 2, 32)
    with pytest.raises(SanaLibraryError, match="state"):
        ops.la_decay_step(q[:2], k[:2], v[:2], ld, torch.zeros(2, 2, 33, 32).half().cuda(), 2, 32)


def test_refusals_of_the_c_entry_points(lib):
    import ctypes as C

    from sana_b200 import _lib
    p, p2, bf = C.c_void_p(0x1000), C.c_void_p(0x2000), _lib.SANA_BF16
    assert lib.sana_la_decay_workspace_bytes(0, 4, 2, 32, bf) == -1
    assert lib.sana_la_decay_workspace_bytes(1, 4, 2, 40, bf) == -1
    assert lib.sana_la_decay_workspace_bytes(1, 4, 2, 32, 7) == -1
    ok = [p, 64, p, 64, p, 64, p, None, None, p, p, 64, None, 0, 2, 4, 2, 2, 32, 1.0, 0, -1.0, bf, None]

    def refused(i, v):
        a = list(ok)
        a[i] = v
        return lib.sana_la_decay(*a) == -1

    for i, v in ((0, None), (6, None), (9, None), (10, None), (1, 60), (3, 56), (5, 32), (11, 32), (1, 68), (0, C.c_void_p(0x1008)),
                 (14, 0), (15, 0), (14, 70000), (16, 3), (18, 24), (21, 1e-6), (22, 5), (13, 4), (7, p), (12, C.c_void_p(0x1004))):
        assert refused(i, v), (i, v)
    ok = [p, 64, p, 64, p, 64, p, p2, 2, None, p, 64, 2, 2, 2, 32, 1.0, 0, -1.0, bf, None]

    def refused_step(i, v):
        a = list(ok)
        a[i] = v
        return lib.sana_la_decay_step(*a) == -1

    for i, v in ((0, None), (7, None), (10, None), (8, 1), (8, 0), (12, 0), (14, 3), (15, 8), (1, 48), (5, 60), (18, 0.0), (19, 4),
                 (7, C.c_void_p(0x2008))):
        assert refused_step(i, v), (i, v)
