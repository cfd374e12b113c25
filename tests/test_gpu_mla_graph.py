"""install_mla in a captured step: what a replay stores is its own, and what it attends to is what it stored."""
import math

import pytest
import torch

from test_gpu_mla_seam import _bf16_default, _freqs, _model  # noqa: F401

pytestmark = pytest.mark.gpu


def _bytes(m):
    import dsv3_b200
    return [t.view(torch.uint8).clone() for t in dsv3_b200.mla_cache(m).pool]


def test_a_replayed_step_stores_its_token():
    import dsv3_b200
    f = _freqs(200)
    g = torch.Generator(device="cuda").manual_seed(14)
    x = torch.randn(2, 68, 256, generator=g, device="cuda", dtype=torch.float32).bfloat16()
    prompt = torch.full((64, 64), -math.inf, device="cuda").triu_(1)
    m, plain = _model(16, 128, seed=4), _model(16, 128, seed=4)
    for one in (m, plain):
        one(x[:, :64], 0, f[:64], prompt)
    static = torch.zeros_like(x[:, 64:65])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = m(static, 64, f[64:65], None)
    cache = dsv3_b200.mla_cache(m)
    for i in range(64, 68):                                                 # another token each time, at the same position
        for b in range(2):
            slot = b * cache.first_page_slot + 64
            cache.pool.latent.view(torch.uint8).view(-1, 512)[slot] = 0
            cache.pool.scale.view(-1)[slot] = math.nan                      # (a step that stores nothing comes out as NaN)
        static.copy_(x[:, i:i + 1])
        graph.replay()
        want = plain(x[:, i:i + 1], 64, f[64:65], None)
        assert torch.equal(out, want) and not torch.isnan(out).any()
        assert all(torch.equal(a, b) for a, b in zip(_bytes(m), _bytes(plain)))
