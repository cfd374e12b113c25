"""latent_attention where sequences share the pages of a prefix."""
import pytest
import torch

import latent_util as U

pytestmark = pytest.mark.gpu
SCALE = 192 ** -0.5


@pytest.fixture(autouse=True)
def _status():
    yield
    import dsv3_b200
    dsv3_b200.check_device_status()


@pytest.mark.parametrize("page, shared, seqs, drafts, heads", [(64, 14, 60, 1, 16), (16, 40, 9, 5, 16), (128, 3, 150, 1, 40)])
def test_sequences_that_share_the_pages_of_a_prefix(page, shared, seqs, drafts, heads):
    """Many sequences on one prompt, each with a page of its own behind it."""
    g = torch.Generator(device="cuda").manual_seed(3)
    cache = U.make_cache(g, shared + seqs, page, 4.0)
    prefix = torch.randperm(shared, generator=g, device="cuda").expand(seqs, -1)
    table = torch.cat([prefix, shared + torch.arange(seqs, device="cuda")[:, None]], 1).to(torch.int32)
    lens = [shared * page + drafts + i % (page - drafts) for i in range(seqs)]
    q = (torch.randn(seqs * drafts, heads, 512, generator=g, device="cuda", dtype=torch.float32).bfloat16(),
         torch.randn(seqs * drafts, heads, 64, generator=g, device="cuda", dtype=torch.float32).bfloat16())
    out, lse = U.dsv3().latent_attention(*q, cache, table, U.i32(lens), SCALE, cu_seqlens_q=U.offsets([drafts] * seqs), return_lse=True)
    U.assert_attention(out, lse, *U.attention(*q, cache, table, lens, [drafts] * seqs, SCALE))
    latent, rope = U.dsv3().latent_cache_read(cache, table, U.offsets(lens), sum(lens))
    for b, at in ((0, 0), (seqs - 1, sum(lens[:-1]))):
        c, k, _ = U.tokens_of(cache, table, b, lens[b])
        assert torch.equal(latent[at:at + lens[b]].double(), c.bfloat16().double()) and torch.equal(rope[at:at + lens[b]].double(), k.bfloat16().double())


def test_drafts_kept_behind_a_shared_prefix():
    """Each sequence's drafts lie in pages of its own; what it keeps of them leaves the shared pages, and the others', as they are."""
    d = U.dsv3()
    g = torch.Generator(device="cuda").manual_seed(4)
    page, shared, seqs = 16, 4, 5
    cache = U.make_cache(g, shared + 2 * seqs, page)
    table = torch.cat([torch.arange(shared, device="cuda").expand(seqs, -1), shared + torch.arange(2 * seqs, device="cuda").view(seqs, 2)], 1).to(torch.int32)
    before = [t.clone().view(torch.uint8) for t in cache]
    path = [[0, 2, 5, 19], [1], [3, 4, 20], [], [0, 1, 2]]
    padded = U.i32([p + [0] * (4 - len(p)) for p in path])
    d.latent_cache_keep(cache, table, U.i32([shared * page] * seqs), padded, U.i32([len(p) for p in path]))
    at = lambda b, p: int(table[b, p // page]) * page + p % page  # noqa: E731
    for plane, old in zip(cache, before):
        new, want = plane.view(torch.uint8).reshape(len(cache.scale.view(-1)), -1), old.reshape(len(cache.scale.view(-1)), -1).clone()
        source = want.clone()
        for b, p in enumerate(path):
            for j, node in enumerate(p):
                want[at(b, shared * page + j)] = source[at(b, shared * page + node)]
        assert torch.equal(new, want)
