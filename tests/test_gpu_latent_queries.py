"""latent_attention with queries of which one value is thousands of times the others."""
import pytest
import torch

import latent_util as U

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _status():
    yield
    import dsv3_b200
    dsv3_b200.check_device_status()


@pytest.mark.parametrize("heads", [16, 128])
@pytest.mark.parametrize("size", [1.0, 2.0 ** 12, 2.0 ** 13])
def test_queries_with_one_value_far_above_the_others(size, heads):
    """The others, between 1 and 2, decide the scores: no token holds anything in the large one's dimension.  They are 2^-6 or more where the row's largest is 256, so that
    the two e4m3 values that stand for a query are exactly it, and the bound is that of any other query."""
    g = torch.Generator(device="cuda").manual_seed(4)
    lens = [5, 300, 40]
    n_pages = 10
    cache = U.make_cache(g, n_pages, 64)
    cache.latent[:, :, 77] = 0
    table = U.block_table(g, lens, 64, n_pages)
    sign = torch.randint(0, 2, (3, heads, 512), generator=g, device="cuda") * 2.0 - 1.0
    ql = (sign * (1 + torch.rand(3, heads, 512, generator=g, device="cuda"))).bfloat16()
    ql[:, :, 77] = size
    qr = torch.randn(3, heads, 64, generator=g, device="cuda", dtype=torch.float32).bfloat16()
    scale = 0.25
    out, lse = U.dsv3().latent_attention(ql, qr, cache, table, U.i32(lens), scale, return_lse=True)
    U.assert_attention(out, lse, *U.attention(ql, qr, cache, table, lens, [1] * 3, scale))
