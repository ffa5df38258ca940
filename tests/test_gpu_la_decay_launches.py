"""How many kernels a call of the decaying attention launches, and the workspace it takes."""
import ctypes as C

import pytest
import torch

from sana_b200 import _lib, ops

BF16 = torch.bfloat16
CASES = [(8, 3355, 10, 112, BF16), (3, 3012, 26, 112, BF16), (2, 64, 4, 32, BF16), (2, 300, 2, 128, BF16), (1, 1001, 4, 32, torch.float32)]


def plan(lib, B, N, H, D, dtype, ragged):
    n = C.c_int(0)
    return lib.sana_la_decay_plan(B, N, H, D, ops._dtype_code(dtype), ragged, C.byref(n)), n.value


def test_a_workspace_goes_with_a_second_launch(lib):
    """The larger of the two plans is what sana_la_decay_workspace_bytes promises to be enough; where lengths make the
    difference, a call without them takes neither the workspace nor the launch."""
    differ = 0
    for B, N, H, D, dtype in CASES:
        plans = [plan(lib, B, N, H, D, dtype, r) for r in (0, 1)]
        assert max(b for b, _ in plans) == lib.sana_la_decay_workspace_bytes(B, N, H, D, ops._dtype_code(dtype))
        for b, n in plans:
            assert n == (2 if b > 0 else 1)
        differ += plans[0] != plans[1]
    assert differ >= 2
    assert lib.sana_la_decay_plan(0, 4, 2, 32, _lib.SANA_BF16, 0, None) == -1
    assert lib.sana_la_decay_plan(1, 4, 2, 32, _lib.SANA_BF16, 0, None) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("B,N,H,D,dtype", CASES)
def test_launches_are_counted_as_they_are_made(lib, B, N, H, D, dtype):
    q, k, v = (torch.randn(B * N, H * D, device="cuda").to(dtype) for _ in range(3))
    ld = -torch.rand(H).cuda()
    for lengths in (None, torch.full((B,), N, dtype=torch.int32, device="cuda")):
        want = plan(lib, B, N, H, D, dtype, 0 if lengths is None else 1)
        before = ops.counters.launches
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        held = torch.cuda.memory_stats()["requested_bytes.all.current"]  # as asked for, before the allocator rounds
        out, state = ops.la_decay(q, k, v, ld, B, N, H, D, lengths=lengths)
        assert ops.counters.launches - before == want[1]
        asked = torch.cuda.memory_stats()["requested_bytes.all.peak"] - held
        assert asked == out.numel() * out.element_size() + state.numel() * 4 + want[0]
