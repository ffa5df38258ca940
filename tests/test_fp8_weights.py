"""The 8-bit images of projection weights that modules keep: whose they are, who reads them, when they go."""
import copy
import gc
import io

import pytest
import torch

import sana_b200
from sana_b200 import ops, weight_pack

BF16 = torch.bfloat16


def layer(seed=0, heads=4, kv_heads=2, dim=64, in_dim=192):
    torch.manual_seed(seed)
    m = sana_b200.DecayCausalAttention(in_dim, heads * dim, heads, kv_heads=kv_heads)
    m.fp8 = True
    return m.to("cuda", BF16)


def inputs(n=70, in_dim=192):
    return torch.randn(1, n, in_dim, generator=torch.Generator().manual_seed(1)).to(BF16).cuda()


@pytest.mark.gpu
def test_a_view_of_the_weight_is_another_weight():
    m, x = layer(), inputs()
    before = m(x)[0]
    m.proj.weight = torch.nn.Parameter(m.proj.weight.t(), requires_grad=False)  # the same storage, shape and version
    fresh = layer()
    fresh.proj.weight = torch.nn.Parameter(m.proj.weight.detach().contiguous().clone(), requires_grad=False)
    after = m(x)[0]
    assert torch.equal(after, fresh(x)[0]) and not torch.equal(after, before)


@pytest.mark.gpu
def test_a_replaced_weight_does_not_reach_a_forward_that_is_under_way():
    """A forward queued on another stream multiplies with the weight it was called with."""
    m, x, side = layer(), inputs(), torch.cuda.Stream()
    weights = [m.proj.weight] + [torch.nn.Parameter(f * m.proj.weight.detach(), requires_grad=False) for f in (-2, 3)]
    want, got = [], []
    for w in weights:
        m.proj.weight = w
        want.append(m(x)[0])
    for _ in range(2):  # the first time round everything is loaded and allocated, which may wait for the GPU
        for w in weights:
            m.proj.weight = w
            m(x)
            torch.cuda.synchronize()
            with torch.cuda.stream(side):
                torch.cuda._sleep(100_000_000)  # about 50 ms
                got.append(m(x)[0])
    m.proj.weight = weights[0]
    m(x)  # while the last one is still under way
    torch.cuda.synchronize()
    assert all(torch.equal(g, w) for g, w in zip(got, want + want))


@pytest.mark.gpu
def test_a_captured_forward_keeps_the_image_it_reads():
    m, x = layer(), inputs()
    before = m(x)[0]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y, _ = m(x)
    old = m.proj  # the graph reads its bias
    m.proj = torch.nn.Linear(256, 512).to("cuda", BF16)
    assert m(x)[0].shape[-1] == 512
    image = 256 * 256
    junk = [torch.full((image,), 0x55, dtype=torch.uint8, device="cuda") for _ in range(64)]  # would land in freed memory
    g.replay()
    assert torch.equal(y, before) and len(junk) == 64 and old is not None


@pytest.mark.gpu
def test_a_moved_module_leaves_no_memory_behind():
    ops.gemm_fp8(ops.fp8_quantize(inputs()[0]), ops.fp8_quantize(torch.zeros(8, 192, dtype=BF16, device="cuda"), 128))
    gc.collect()
    torch.cuda.synchronize()
    start = torch.cuda.memory_allocated()
    m, x = layer(), inputs()
    first = m(x)[0].cpu()
    del x
    m.to("cpu")
    gc.collect()
    assert torch.cuda.memory_allocated() == start
    m.to("cuda")
    assert torch.equal(m(inputs())[0].cpu(), first)


@pytest.mark.gpu
def test_copies_of_a_module_have_images_of_their_own():
    m, x = layer(), inputs()
    want = m(x)[0]
    twin = copy.deepcopy(m)
    with torch.no_grad():
        twin.proj.weight.mul_(-2)
    moved = twin(x)[0]
    assert torch.equal(m(x)[0], want) and not torch.equal(moved, want)
    f = io.BytesIO()
    torch.save(m, f)
    f.seek(0)
    loaded = torch.load(f, weights_only=False)
    del m
    gc.collect()
    assert torch.equal(loaded(x)[0], want) and torch.equal(twin(x)[0], moved)


def pack_of(model):
    """A weight pack of the right names and shapes (its codes are zeros)."""
    pack = {}
    for name, module in model.named_modules():
        for key, w in weight_pack._projections(module):
            base = f"{name}.{key}.nvfp4"
            n, k = w.shape
            pack.update({base + ".q": torch.zeros(n, k // 2, dtype=torch.uint8), base + ".sf": torch.zeros(16, dtype=torch.uint8),
                         base + ".scales": torch.zeros(4), base + ".shape": torch.tensor([n, k])})
    return pack


def test_installed_nvfp4_weights_replace_the_8_bit_setting():
    blk = sana_b200.SanaMSBlock(64, 2, mlp_ratio=2.5, attn_type="linear", ffn_type="glumbconv")
    blk.set_fp8(True)
    assert sana_b200.load_nvfp4_weights(blk, pack_of(blk), enable=False) == 4
    assert blk.attn.fp8 and blk.mlp.fp8 and not blk.attn.nvfp4  # installed, not switched on
    sana_b200.load_nvfp4_weights(blk, pack_of(blk))
    assert blk.attn.nvfp4 and blk.mlp.nvfp4 and not blk.attn.fp8 and not blk.mlp.fp8
    blk.set_fp8(True)
    assert blk.attn.fp8 and blk.mlp.fp8 and not blk.attn.nvfp4 and not blk.mlp.nvfp4
