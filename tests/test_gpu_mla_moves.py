"""install_mla: a module that goes to the host and back goes on where it was; a cache made on one stream is there for the others."""
import threading

import pytest
import torch

from test_gpu_mla_seam import _bf16_default, _freqs, _model  # noqa: F401

pytestmark = pytest.mark.gpu


def _causal(n):
    return torch.full((n, n), float("-inf"), device="cuda").triu_(1)


def test_there_and_back():
    import dsv3_b200
    m, f = _model(4, 0), _freqs(200)
    x = torch.randn(2, 31, 256, device="cuda", dtype=torch.float32).bfloat16()
    m(x[:, :30], 0, f[:30], _causal(30))
    want = m(x[:, 30:], 30, f[30:31], None)
    m.kv_cache = m.kv_cache.cpu()
    assert dsv3_b200.mla_cache(m).pool.latent.device.type == "cpu"
    m.kv_cache = m.kv_cache.cuda()
    assert torch.equal(m(x[:, 30:], 30, f[30:31], None), want)


def test_first_calls_of_two_threads():
    """Each thread has a sequence of its own of one module's cache."""
    import dsv3_b200
    f = _freqs(200)
    x = torch.randn(2, 40, 256, device="cuda", dtype=torch.float32).bfloat16()
    want = _model(4, 0)(x, 0, f[:40], _causal(40))
    torch.cuda.synchronize()
    for _ in range(5):
        m, out, failed, together = _model(4, 0), [None, None], [], threading.Barrier(2)
        mask, starts = _causal(40), torch.tensor([0, 200], device="cuda")    # (a sequence that does not fit is not stored: each thread stores one)
        torch.cuda.synchronize()

        def work(i):
            try:
                torch.set_default_dtype(torch.bfloat16)
                stream = torch.cuda.Stream()
                with torch.cuda.stream(stream):
                    together.wait()
                    out[i] = m(x, starts if i == 0 else starts.flip(0), f[:40], mask)
                    stream.synchronize()
            except Exception as e:                                           # noqa: BLE001
                failed.append(e)

        threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert not failed
        cache = dsv3_b200.mla_cache(m)
        assert torch.isnan(out[0][1]).all() and torch.isnan(out[1][0]).all()
        for i in range(2):
            assert ((out[i][i].double() - want[i].double()).norm() / want[i].double().norm()).item() < 2.0 ** -9
        assert (cache.pool.scale.view(3, -1)[:2, :40] != 1).all()
