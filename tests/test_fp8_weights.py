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
