"""8-bit projections and decaying attention from two threads at once, each on a stream of its own."""
import threading

import pytest
import torch

import sana_b200
from sana_b200 import ops

BF16 = torch.bfloat16


def work(m, x, lengths):
    y, state = m(x, lengths=lengths)
    z = m.step(x[:, 0], state)
    return y, z, state


@pytest.mark.gpu
def test_two_threads_share_a_layer():
    """The layer's images are made by whichever thread comes first; results are those of one call after the other."""
    torch.manual_seed(0)
    m = sana_b200.DecayCausalAttention(256, 448, 4, kv_heads=2).to("cuda", BF16)
    m.fp8 = True
    g = torch.Generator().manual_seed(1)
    jobs = []
    for B, N in ((1, 40), (3, 333), (2, 1500), (5, 129), (1, 2500), (4, 640)):
        lengths = torch.randint(0, N + 1, (B,), generator=g).to(torch.int32).cuda()
        jobs.append((torch.randn(B, N, 256, generator=g).to(BF16).cuda(), lengths))
    got, failed = {}, []
    torch.cuda.synchronize()
    start = threading.Barrier(2)

    def run(who):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                start.wait(30)
                for rep in range(10):
                    for i in range(len(jobs)):
                        j = (i + 3 * who) % len(jobs)
                        got[who, rep, j] = work(m, *jobs[j])
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001  (told to the main thread)
            failed.append(e)

    threads = [threading.Thread(target=run, args=(w,)) for w in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(120)
    assert not failed and len(got) == 2 * 10 * len(jobs), failed
    torch.cuda.synchronize()
    for j, job in enumerate(jobs):
        want = work(m, *job)
        for who in range(2):
            for rep in range(10):
                assert all(torch.equal(a, b) for a, b in zip(got[who, rep, j], want)), (who, rep, j)
    assert ops.take_la_decay_device_status() == 0 and ops.take_gemm_fp8_device_status() == 0
