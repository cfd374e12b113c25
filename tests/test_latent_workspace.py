"""The size of latent attention's workspace: the same under any budget of SMs, and one that is enough for all calls."""
import random

import pytest

from test_latent_refusals import _lib


@pytest.fixture
def size():
    lib, _ = _lib()
    lib.dsv3_set_num_sms(0)
    yield lib.dsv3_latent_attention_workspace_bytes
    lib.dsv3_set_num_sms(0)


def _shapes(n):
    rng = random.Random(5)
    for _ in range(n):
        seqs = round(2 ** rng.uniform(0, 9))
        yield seqs * round(2 ** rng.uniform(0, 6)), rng.choice([1, 5, 16, 17, 32, 40, 128, 1024]), seqs, round(2 ** rng.uniform(0, 17))


def test_the_budget_of_sms_does_not_change_it(size):
    lib, _ = _lib()
    shapes = list(_shapes(400))
    want = [size(*s) for s in shapes]
    assert any(w == 0 for w in want) and any(w > 0 for w in want)
    for sms in (2, 8, 37, 100, 147):
        lib.dsv3_set_num_sms(sms)
        assert [size(*s) for s in shapes] == want


def test_one_size_is_enough_for_all_calls(size):
    most = size(1, 32, 1, 1 << 30)
    assert most > 0 and all(size(*s) <= most for s in _shapes(2000))
    assert size(128, 8, 128, 1 << 14) < size(128, 8, 32, 1 << 14) <= most           # smaller for more sequences
