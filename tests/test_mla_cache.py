"""The cache of an MLA module: made once, whichever thread comes first, and on the device of the module's buffers."""
import threading
import time
import types

import torch


def _module(device="cpu"):
    return types.SimpleNamespace(kv_cache=torch.zeros(2, 70, 512, device=device))


def test_threads_that_come_at_once_get_one_cache(monkeypatch):
    import dsv3_b200 as d
    from dsv3_b200 import mla_seam
    made = []

    def slowly(*args):
        made.append(args)
        time.sleep(0.05)                                                    # (the others come meanwhile)
        return d.allocate_latent_cache(*args)

    monkeypatch.setattr(mla_seam, "allocate_latent_cache", slowly)
    module, got, together = _module(), [], threading.Barrier(6)

    def ask():
        together.wait()
        got.append(d.mla_cache(module))

    threads = [threading.Thread(target=ask) for _ in range(6)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(made) == 1 and len(got) == 6 and all(c is got[0] for c in got)


def test_a_module_that_moves_takes_its_tokens_along():
    import dsv3_b200 as d
    module = _module()
    cache = d.mla_cache(module)
    assert d.mla_cache(module) is cache
    module.kv_cache = module.kv_cache.to("meta")                            # (a second device that is there without a GPU)
    moved = d.mla_cache(module)
    assert all(t.device.type == "meta" for t in (*moved.pool, moved.block_table)) and moved[2:] == cache[2:]
    assert [t.shape for t in moved.pool] == [t.shape for t in cache.pool] and d.mla_cache(module) is moved
