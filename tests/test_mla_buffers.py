"""install_mla(release_buffers=True): the modules' bf16 buffers give their memory back."""
import types

import pytest
import torch


def _module(device="cpu", **buffers):
    m = torch.nn.Module()
    for name, shape in buffers.items():
        m.register_buffer(name, torch.zeros(shape, device=device, dtype=torch.bfloat16), persistent=False)
    return m


@pytest.mark.parametrize("shapes", [dict(kv_cache=(2, 70, 512), pe_cache=(2, 70, 64)), dict(k_cache=(2, 70, 4, 192), v_cache=(2, 70, 4, 128))])
def test_buffers_of_both_kinds(shapes):
    from dsv3_b200 import mla_cache, mla_seam
    m = _module(**shapes)
    mla_seam._release_buffers(m)
    for name, shape in shapes.items():
        b = getattr(m, name)
        assert b.shape == shape and b.dtype == torch.bfloat16 and b.untyped_storage().nbytes() == 2 and not b.any()
        with pytest.raises(RuntimeError):                                   # the old forward cannot store to it unnoticed
            b[:1, 3:5] = torch.ones_like(b[:1, 3:5])
        mla_seam._release_buffers(m)
        assert getattr(m, name) is b
    assert mla_cache(m).pool.scale.shape == (4, 64) and mla_cache(m).max_len == 70


@pytest.mark.parametrize("release", [False, True])
def test_only_where_it_is_asked_for(release, monkeypatch):
    from dsv3_b200 import mla_seam
    monkeypatch.setattr(mla_seam, "mla_forward", lambda self, *a, **k: self.kv_cache.untyped_storage().nbytes())
    model = types.SimpleNamespace(MLA=type("MLA", (torch.nn.Module,), {}))
    mla_seam.install_mla(model, release_buffers=True) if release else mla_seam.install_mla(model)
    m = model.MLA()
    m.kv_cache = torch.zeros(2, 70, 512, dtype=torch.bfloat16)
    assert m.forward(None, 0, None, None) == (2 if release else 2 * 70 * 512 * 2)


@pytest.mark.gpu
def test_memory_that_is_given_back_and_the_same_results():
    import dsv3_b200
    from test_gpu_mla_seam import _freqs, _model
    torch.set_default_dtype(torch.bfloat16)
    try:
        f = _freqs(200)
        x = torch.randn(2, 31, 256, device="cuda", dtype=torch.float32).bfloat16()
        mask = torch.full((30, 30), float("-inf"), device="cuda").triu_(1)
        plain = _model(4, 0)
        want = plain(x[:, :30], 0, f[:30], mask), plain(x[:, 30:], 30, f[30:31], None)
        m = _model(4, 0, batch=2, length=200)
        dsv3_b200.install_mla(types.SimpleNamespace(MLA=type(m), block_size=128), release_buffers=True)
        m.kv_cache = torch.zeros(64, 200, 512, device="cuda")
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        got = m(x[:, :30], 0, f[:30], mask), m(x[:, 30:], 30, f[30:31], None)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        del got
        cache = dsv3_b200.mla_cache(m)
        made = sum(t.untyped_storage().nbytes() for t in (*cache.pool, cache.block_table))
        assert cache.max_len == 200 and torch.cuda.memory_allocated() <= before - 64 * 200 * 1024 + made + (1 << 20)
    finally:
        torch.set_default_dtype(torch.float32)
        dsv3_b200.check_device_status()
