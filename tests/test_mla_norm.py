"""install_mla: which norms latent_cache_write may do in the place of kv_norm."""
import types

import pytest
import torch
import torch.nn.functional as F
from torch import nn


class Norm(nn.Module):
    """As the reference's, model.py:270-294."""

    def __init__(self, dim=512, eps=1e-6):
        super().__init__()
        self.dim, self.eps = dim, eps
        self.weight = nn.Parameter(torch.ones(dim))

    def forward(self, x):
        return F.rms_norm(x, (self.dim,), self.weight, self.eps)


class ByHand(Norm):
    def forward(self, x):
        y = x.float()
        return (y * torch.rsqrt(y.pow(2).mean(-1, keepdim=True) + self.eps)).type_as(x) * self.weight


class OnePlus(Norm):
    def forward(self, x):
        return F.rms_norm(x, (self.dim,), 1 + self.weight, self.eps)


class FixedEps(Norm):
    def forward(self, x):
        return F.rms_norm(x, (self.dim,), self.weight, 1e-5)


class Centred(Norm):
    def forward(self, x):
        return F.layer_norm(x, (self.dim,), self.weight, None, self.eps)


class Clamped(Norm):
    def forward(self, x):
        return F.rms_norm(x, (self.dim,), self.weight, self.eps).clamp(-1, 1)


class Counts(Norm):
    def forward(self, x):
        self.calls += 1
        return F.rms_norm(x, (self.dim,), self.weight, self.eps)


class Calls(Norm):
    def __call__(self, x):
        return 2 * super().__call__(x)


def _seam():
    from dsv3_b200 import mla_seam
    return mla_seam


@pytest.mark.parametrize("cls, plain", [(Norm, True), (ByHand, True), (OnePlus, False), (FixedEps, False), (Centred, False), (Clamped, False), (Counts, False), (Calls, False),
                                        (nn.RMSNorm, False)])
def test_classes(cls, plain):
    assert _seam()._is_rms_norm(cls(512)) is plain


def test_what_is_no_module():
    assert not _seam()._is_rms_norm(types.SimpleNamespace(weight=torch.ones(512), eps=1e-6))
    assert not _seam()._is_rms_norm(lambda x: x)


def test_hooks_and_forwards_of_their_own():
    plain = _seam()._is_rms_norm
    for change in (lambda m: m.register_forward_hook(lambda *a: None), lambda m: m.register_forward_pre_hook(lambda *a: None), lambda m: setattr(m, "forward", lambda x: x)):
        m = Norm()
        assert plain(m)
        change(m)
        assert not plain(m)
    handle = nn.modules.module.register_module_forward_hook(lambda *a: None)
    try:
        assert not plain(Norm())
    finally:
        handle.remove()
    assert plain(Norm())


def test_a_forward_that_is_replaced_on_the_class(monkeypatch):
    plain = _seam()._is_rms_norm
    assert plain(Norm())
    monkeypatch.setattr(Norm, "forward", OnePlus.forward)
    assert not plain(Norm())
    monkeypatch.undo()
    assert plain(Norm())


def test_random_numbers_stay_as_they_are():
    _seam()._known_norms.clear()
    torch.manual_seed(3)
    want = torch.rand(4)
    torch.manual_seed(3)
    assert _seam()._is_rms_norm(Norm())
    assert torch.equal(torch.rand(4), want)


RAN = []


def _kernel(x, weight, eps):
    RAN.append(x)                                                           # (would take the host's memory for the device's)
    return F.rms_norm(x, (x.size(-1),), weight, eps)


class CodeOfItsOwn(Norm):
    def forward(self, x):
        return _kernel(x, self.weight, self.eps)


class Imports(Norm):
    def forward(self, x):
        import test_mla_norm
        return test_mla_norm._kernel(x, self.weight, self.eps)


class Opens(Norm):
    def forward(self, x):
        RAN.append(open)
        return F.rms_norm(x, (self.dim,), self.weight, self.eps)


def _closed_over(kernel):
    class Closed(Norm):
        def forward(self, x):
            return kernel(x, self.weight, self.eps)
    return Closed


@pytest.mark.parametrize("cls", [CodeOfItsOwn, Imports, Opens, _closed_over(_kernel)])
def test_code_of_its_own_is_not_run(cls):
    RAN.clear()
    assert not _seam()._is_rms_norm(cls(512)) and not RAN
