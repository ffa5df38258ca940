"""The decaying linear attention and the 8-bit projections as they are used together: a causal layer over prompts and
single tokens, the Linear-DiT block with 8-bit projections, the torch custom operators."""
import pytest
import torch

import sana_b200
import sana_b200.torch_ops  # noqa: F401  (registers the operators)
from sana_b200 import ops, synthetic

BF16 = torch.bfloat16


def layer(heads=4, kv_heads=2, dim=64, in_dim=192, normalize=True, seed=0):
    torch.manual_seed(seed)
    m = sana_b200.DecayCausalAttention(in_dim, heads * dim, heads, kv_heads=kv_heads, normalize=normalize, use_bias=True)
    return m.to("cuda", BF16)


def test_layer_keeps_its_decays_in_fp32_and_refuses_what_the_kernels_lack():
    m = sana_b200.DecayCausalAttention(64, 64, 2)
    before = m.log_decay.clone()
    m = m.to(BF16)
    assert m.log_decay.dtype == torch.float32 and torch.equal(m.log_decay, before) and m.qkv.weight.dtype == BF16
    assert (m.log_decay < 0).all()
    assert set(m.state_dict()) == {"log_decay", "qkv.weight", "proj.weight", "proj.bias"}
    with torch.device("meta"):
        empty = sana_b200.DecayCausalAttention(64, 64, 2).to(BF16)
    empty = empty.to_empty(device="cpu")
    assert empty.log_decay.dtype == torch.float32 and empty.qkv.weight.dtype == BF16
    empty.load_state_dict(m.state_dict())
    assert torch.equal(empty.log_decay, before)
    for kw in (dict(heads=3), dict(heads=8), dict(heads=2, kv_heads=3)):
        with pytest.raises(NotImplementedError):
            sana_b200.DecayCausalAttention(64, 64, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("fp8", [False, True])
def test_prompt_then_tokens_equals_the_whole_prompt(normalize, fp8):
    """Rows of a projection are quantised on their own, so a prompt in one piece and the same tokens in pieces meet the
    same codes; what differs is the order of sums (and the kernel that multiplies): both are within rounding of the
    outputs, whose roundings to bf16 enter the output projection."""
    B, N = 3, 160
    m = layer(normalize=normalize)
    m.fp8 = fp8
    x = torch.randn(B, N, 192, generator=torch.Generator().manual_seed(1)).to(BF16).cuda()
    whole, st = m(x)
    first, state = m(x[:, :130])
    parts = [first]
    for t in range(130, N):
        parts.append(m.step(x[:, t], state)[:, None])
    got = torch.cat(parts, 1)
    # qkv may differ by one rounding (2^-8) between two kernels; q, k and v enter the attention, so an output moves by at
    # most about 3 of them, its own rounding and that of the scores; the projection's codes add 2^-4 of what moved
    tol = (6 + (2 if fp8 else 0)) * 2.0 ** -8
    assert (got.float() - whole.float()).norm() <= tol * whole.float().norm()
    assert (state - st).norm() <= tol * st.norm()


@pytest.mark.gpu
def test_layer_is_the_operators_in_a_row():
    m = layer()
    m.fp8 = True
    B, N, D, H, Hk = 2, 100, 64, 4, 2
    x = torch.randn(B, N, 192).to(BF16).cuda()
    y, st = m(x, lengths=torch.tensor([100, 33], dtype=torch.int32).cuda())
    q8 = lambda w: ops.fp8_quantize(w, 128)
    qkv = ops.gemm_fp8(ops.fp8_quantize(x.reshape(B * N, -1)), q8(m.qkv.weight), bias=m.qkv.bias)
    o, st2 = ops.la_decay(qkv[:, :H * D], qkv[:, H * D:(H + Hk) * D], qkv[:, (H + Hk) * D:], m.log_decay, B, N, H, D, relu=True,
                          eps=1e-8, lengths=torch.tensor([100, 33], dtype=torch.int32).cuda())
    want = ops.gemm_fp8(ops.fp8_quantize(o), q8(m.proj.weight), bias=m.proj.bias)
    assert torch.equal(y.reshape(B * N, -1), want) and torch.equal(st, st2)
    # a changed weight is quantised anew
    with torch.no_grad():
        m.proj.weight.mul_(2)
    y2, _ = m(x)
    assert not torch.equal(y2, y)


@pytest.mark.gpu
def test_serving_batch_with_slots_in_a_graph():
    """A decoding batch captured once: rows join and leave by rewriting the slots."""
    m = layer()
    pool, B = 6, 4
    x = torch.randn(B, 192).to(BF16).cuda()
    state = torch.rand(pool, 4, 65, 64).cuda()
    slots = torch.tensor([2, -1, 5, 0], dtype=torch.int32).cuda()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        m.step(x, state.clone(), slots)
    torch.cuda.current_stream().wait_stream(s)
    held = state.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = m.step(x, held, slots)
    held.copy_(state)
    want_state = state.clone()
    for new in ([2, -1, 5, 0], [1, 3, -1, 4]):
        slots.copy_(torch.tensor(new, dtype=torch.int32))
        x.normal_()
        g.replay()
        want = m.step(x, want_state, slots)
        assert torch.equal(y, want) and torch.equal(held, want_state)


@pytest.mark.gpu
def test_the_kept_weight_image_is_that_of_the_weight():
    m = layer()
    m.fp8 = True
    x = torch.randn(1, 70, 192).to(BF16).cuda()
    y = m(x)[0]
    for seed in (1, 2, 3):  # new weights of the same size, which the allocator would put where freed ones were
        m.qkv.weight = None
        m.qkv.weight = torch.nn.Parameter(layer(seed=seed).qkv.weight.detach().clone(), requires_grad=False)
        kept, fresh = m(x)[0], layer()
        fresh.load_state_dict(m.state_dict())
        fresh.fp8 = True
        assert torch.equal(kept, fresh(x)[0]) and not torch.equal(kept, y)
    with torch.inference_mode():  # changes of inference tensors are not counted
        n = layer()
        n.fp8 = True
        first = n(x)[0]
        n.proj.weight.mul_(2)
        assert not torch.equal(n(x)[0], first)


@pytest.mark.gpu
def test_a_capture_without_warm_up_keeps_nothing():
    m = layer()
    m.fp8 = True
    x = torch.randn(1, 70, 192).to(BF16).cuda()
    ops.gemm_fp8(ops.fp8_quantize(x[0]), ops.fp8_quantize(m.qkv.weight, 128))  # the library is loaded
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y, st = m(x)
    eager = m(x)  # before the first replay
    g.replay()
    assert torch.equal(y, eager[0]) and torch.equal(st, eager[1])
    with torch.no_grad():
        m.qkv.weight.mul_(0.5)
    g.replay()
    assert torch.equal(y, m(x)[0])


@pytest.mark.gpu
def test_a_captured_forward_follows_a_changed_weight():
    m = layer()
    m.fp8 = True
    x = torch.randn(1, 70, 192).to(BF16).cuda()
    before = m(x)[0]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y, _ = m(x)
    with torch.no_grad():
        m.proj.weight.mul_(-2)
    eager = m(x)[0]
    junk = [torch.full_like(m.proj.weight, 3.0) for _ in range(8)]  # would land in memory that had been freed
    g.replay()
    assert torch.equal(y, eager) and not torch.equal(y, before) and len(junk) == 8


@pytest.mark.gpu
def test_block_with_8_bit_projections():
    """Every operand is off by at most 2^-4 of itself (rms 2^-4 / sqrt 3), so a projection by sqrt 2 of that in norm; four
    projections follow one another in the block, and their branches' share of the output is at most all of it."""
    C, heads, L, HW = 256, 4, 20, (16, 16)
    shp = synthetic.BlockShape("fp8", C, heads, 2, HW, text_len=L)
    params = synthetic.make_block_params(C, shp.ffn_hidden, seed=0, std=0.05)
    x, y, t = synthetic.make_block_inputs(shp, seed=0, std=0.05, text_dim=64)
    blk = sana_b200.SanaMSBlock(C, heads, mlp_ratio=2.5, attn_type="linear", ffn_type="glumbconv").eval()
    blk.load_state_dict(params, strict=True)
    blk = blk.to("cuda", BF16)
    a = [v.to("cuda", BF16) for v in (x, y, t)]
    ref = blk(*a, None, HW).float()
    blk.set_fp8(True)
    got = blk(*a, None, HW).float()
    assert not torch.equal(got, ref)
    branch = (ref - a[0].float()).norm()
    assert (got - ref).norm() <= 4 * 2 ** 0.5 * 2.0 ** -4 / 3 ** 0.5 * branch
    blk.set_nvfp4(True)
    assert not blk.attn.fp8 and not blk.mlp.fp8
    blk.set_nvfp4(False)
    assert torch.equal(blk(*a, None, HW).float(), ref)
    blk.attn.fp8 = blk.attn.nvfp4 = True
    with pytest.raises(ValueError):
        blk(*a, None, HW)


def test_custom_operators_propagate_shapes_without_a_gpu():
    from torch._subclasses.fake_tensor import FakeTensorMode

    ns = torch.ops.sana_b200
    with FakeTensorMode():
        x = torch.empty(300, 272, dtype=BF16)
        c, s = ns.fp8_quantize(x, 1)
        assert c.shape == (300, 272) and c.dtype == torch.float8_e4m3fn and s.shape == (300, 3) and s.stride(0) == 4
        cw, sw = ns.fp8_quantize(torch.empty(136, 272, dtype=BF16), 128)
        assert sw.shape == (2, 3)
        y = ns.gemm_fp8(c, s, 1, cw, sw, 128, None, 0, 0, None, None, 0, 1, None)
        assert y.shape == (300, 136) and y.dtype == BF16
        q, k = torch.empty(2 * 50, 128, dtype=BF16), torch.empty(2 * 50, 64, dtype=BF16)
        o, st = ns.la_decay(q, k, k, torch.empty(4), 2, 50, 4, 32, 1.0, True, 1e-8, None, None)
        assert o.shape == (100, 128) and st.shape == (2, 4, 33, 32) and st.dtype == torch.float32
        assert ns.la_decay_step(q[:2], k[:2], k[:2], torch.empty(4), st, 4, 32, 1.0, False, None, None).shape == (2, 128)


@pytest.mark.gpu
def test_custom_operators_match_the_direct_path():
    ns = torch.ops.sana_b200
    x, w = torch.randn(70, 272).to(BF16).cuda(), torch.randn(136, 272).to(BF16).cuda()
    a, b = ops.fp8_quantize(x), ops.fp8_quantize(w, 128)
    ca, sa = ns.fp8_quantize(x, 1)
    cb, sb = ns.fp8_quantize(w, 128)
    assert torch.equal(ca.view(torch.uint8), a.q.view(torch.uint8)) and torch.equal(sb, b.scales)
    assert torch.equal(ns.gemm_fp8(ca, sa, 1, cb, sb, 128, None, ops.ACT_SILU, 0, None, None, 0, 1, None),
                       ops.gemm_fp8(a, b, act=ops.ACT_SILU))
    q = torch.randn(2 * 90, 3 * 64).to(BF16).cuda()
    ld = -torch.rand(2).cuda()
    args = (q[:, :64], q[:, 64:128], q[:, 128:], ld)
    o, st = ns.la_decay(*args, 2, 90, 2, 32, 1.0, True, 1e-8, None, None)
    o2, st2 = ops.la_decay(*args, 2, 90, 2, 32, relu=True, eps=1e-8)
    assert torch.equal(o, o2) and torch.equal(st, st2)
    row = tuple(v[:2] for v in args[:3]) + (ld,)
    y = ns.la_decay_step(*row, st, 2, 32, 1.0, True, 1e-8, None)
    assert torch.equal(y, ops.la_decay_step(*row, st2, 2, 32, relu=True, eps=1e-8)) and torch.equal(st, st2)
    m = layer()
    z = torch.randn(2, 80, 192).to(BF16).cuda()
    want = m(z)
    try:
        sana_b200.torch_ops.route_modules(True)
        got = m(z)
        y1 = m.step(z[:, 0], got[1])
    finally:
        sana_b200.torch_ops.route_modules(False)
    assert torch.equal(got[0], want[0])
    assert torch.equal(y1, m.step(z[:, 0], want[1])) and torch.equal(got[1], want[1])
