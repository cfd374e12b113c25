"""latent_attention where little things count: thousands of tokens that each weigh 2^-18 to 2^-21 of one, whose content follows their position.

A weight below a step of the grid is rounded up or down by an offset before it, so that its error lies in an interval of one step, 2^-18 of the row's largest weight
(2^-13 where the largest is 2^5), and has a mean of zero over the offsets.  The offsets of different tiles of 128 tokens are independent.  A dimension that n tokens hold, s of
them or fewer to a tile, adds up n / s or more independent errors within s steps each: off by more than 4 sqrt(s n) steps with a chance of 2 exp(-32) (Hoeffding: 2 exp(-2 t^2 / (T (s g)^2)) with
t = 4 s g sqrt(T), and T = n / s tiles).  With offsets that are the same in every tile the errors of a dimension add up to up to n / 2 steps instead."""
import math

import pytest
import torch

import latent_util as U

pytestmark = pytest.mark.gpu
TILE = 128


@pytest.fixture(autouse=True)
def _status():
    yield
    import dsv3_b200
    dsv3_b200.set_num_sms(0)
    dsv3_b200.check_device_status()


def _contents(n):
    """bool [512, n]: which tokens a dimension is set in, and how many of them there are at most to a tile."""
    p = torch.arange(n, device="cuda")
    sets = [p % TILE == r for r in range(TILE)]                                        # one place of every tile
    sets += [(p % TILE - r) % TILE < 16 for r in range(0, TILE, 2)]                    # sixteen places side by side
    sets += [p % every == every // 2 for every in range(1, 257)]                       # every so many tokens
    sets += [(p // TILE) % (2 + i) == 0 for i in range(32)]                            # every so many tiles
    sets += [p % (TILE * (2 + i)) == 7 * i for i in range(32)]                         # one token of those
    sets = torch.stack(sets)
    sets[:, 0] = False
    assert sets.shape == (512, n)
    per = [int(s.view(-1, TILE).sum(1).max()) for s in sets]
    return sets, torch.tensor(per, device="cuda", dtype=torch.float64)


@pytest.mark.parametrize("heads", [16, 32])
def test_many_tokens_of_small_weight_whose_content_follows_their_position(heads):
    """A first token 12.5 to 15 units of the exponent above 65535 others; two sequences of the same pages on two SMs, so that a row's weights are all relative to that token."""
    d = U.dsv3()
    n, page = 65536, 128
    sets, per_tile = _contents(n)
    latent = torch.where(sets.t(), 256.0, 0.0).to(torch.float8_e4m3fn).contiguous().view(n // page, page, 512)
    rope = torch.zeros(n // page, page, 64, dtype=torch.bfloat16, device="cuda")
    rope[0, 0, 0] = 256.0
    scale = torch.full((n // page, page), 2.0 ** -8, device="cuda", dtype=torch.float32)
    cache = d.LatentCache(latent, rope, scale)
    table = torch.arange(n // page, dtype=torch.int32, device="cuda").expand(2, -1)
    ql = torch.zeros(2, heads, 512, dtype=torch.bfloat16, device="cuda")
    qr = torch.zeros(2, heads, 64, dtype=torch.bfloat16, device="cuda")
    gap = 12.5 + 0.0625 * torch.arange(heads, device="cuda", dtype=torch.float64) * (32 // heads)
    qr[:, :, 0] = gap.bfloat16()
    assert torch.equal(qr[0, :, 0].double(), gap)
    d.set_num_sms(2)
    out = d.latent_attention(ql, qr, cache, table, U.i32([n, n]), 1.0)
    weight = torch.exp(-gap)[:, None]
    total = 1 + (n - 1) * weight
    count = sets.sum(1).double()
    want = count * weight / total
    bound = (2.0 ** -8 + 2.0 ** -12) * want + 4 * (per_tile * count).sqrt() * 2.0 ** -18 / total
    worst = ((out.double() - want).abs() / bound).amax(0).amax(0)
    assert worst.max().item() <= 1, (worst.max().item(), worst.argmax().item(), int((worst > 1).sum()))
