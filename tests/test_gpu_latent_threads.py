"""latent_attention from several threads: every call of every thread is counted, and what a thread raises is raised here."""
from concurrent.futures import ThreadPoolExecutor

import pytest
import torch

from test_gpu_latent_calls import _problem, _same

pytestmark = pytest.mark.gpu
ROUNDS = 20


def test_every_call_of_every_thread():
    import dsv3_b200
    problems = [_problem(60 + i, [1500 + 100 * i, 40], heads=16 if i % 2 else 128) for i in range(4)]
    want = [[t.clone() for t in f()] for f, _ in problems]
    torch.cuda.synchronize()

    def work(i):
        stream, right = torch.cuda.Stream(), 0
        with torch.cuda.stream(stream):
            for _ in range(ROUNDS):
                out = problems[i][0]()
                stream.synchronize()
                right += _same(out, want[i])
        return right

    with ThreadPoolExecutor(4) as pool:
        assert [r.result() for r in [pool.submit(work, i) for i in range(4)]] == [ROUNDS] * 4
    dsv3_b200.check_device_status()
