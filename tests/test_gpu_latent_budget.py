"""latent_attention while another thread sets the budget of SMs: every call is served, and its parts fit the workspace that was checked."""
import threading

import pytest
import torch

import latent_util as U
from test_gpu_latent_calls import SCALE, _problem

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lens, heads", [([5000, 900, 300], 16), ([3000] * 8, 128), ([384] * 60, 16), ([900] * 100, 16)])
def test_calls_while_the_budget_changes(lens, heads):
    import dsv3_b200
    from dsv3_b200 import _lib
    call, (q, cache, table, _) = _problem(50, lens, heads)
    want, want_lse, bound = U.attention(*q, cache, table, lens, [1] * len(lens), SCALE)
    stop = threading.Event()

    def change():
        while not stop.is_set():
            for n in (2, 0, 60, 0, 147, 0):
                _lib.lib.dsv3_set_num_sms(n)

    t = threading.Thread(target=change)
    t.start()
    outs = []
    try:
        for i in range(400):
            out = call()
            if i % 20 == 0:
                outs.append(out)
    finally:
        stop.set()
        t.join()
        dsv3_b200.set_num_sms(0)
    dsv3_b200.check_device_status()
    for out, lse in outs:
        U.assert_attention(out, lse, want, want_lse, bound)


@pytest.mark.parametrize("sms", [2, 3, 7, 64, 147])
@pytest.mark.parametrize("lens, heads, drafts", [([384] * 60, 16, 1), ([900] * 100, 16, 1), ([1100] * 140, 16, 1), ([700] * 12, 128, 1), ([620] * 9, 16, 15), ([90] * 300, 4, 1)])
def test_whole_and_cut_blocks_under_a_budget(sms, lens, heads, drafts):
    import dsv3_b200
    call, (q, cache, table, _) = _problem(51, lens, heads, drafts)
    want, want_lse, bound = U.attention(*q, cache, table, lens, [drafts] * len(lens), SCALE)
    dsv3_b200.set_num_sms(sms)
    try:
        out, lse = call()
        dsv3_b200.check_device_status()
    finally:
        dsv3_b200.set_num_sms(0)
    U.assert_attention(out, lse, want, want_lse, bound)
