"""latent_attention against its definition in 64 bits; the tolerances are derived in latent_util.attention."""
import math

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


def _queries(g, tokens, heads, size=1.0):
    return ((torch.randn(tokens, heads, 512, generator=g, device="cuda", dtype=torch.float32) * size).bfloat16(),
            torch.randn(tokens, heads, 64, generator=g, device="cuda", dtype=torch.float32).bfloat16())


def _setup(seed, lens, page, spread=4.0, spare_pages=3):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n_pages = sum(-(-n // page) for n in lens) + spare_pages
    cache = U.make_cache(g, n_pages, page, spread)
    table = U.block_table(g, lens, page, n_pages, spare=1)
    U.poison_rest(cache, table, lens)
    return g, cache, table


def _compare(q, cache, table, lens, counts, tree=None, scale=SCALE, packed=True):
    d = U.dsv3()
    out, lse = d.latent_attention(*q, cache, table, U.i32(lens), scale, cu_seqlens_q=U.offsets(counts) if packed else None, tree_mask=tree, return_lse=True)
    want, want_lse, bound = U.attention(*q, cache, table, lens, counts, scale, tree)
    U.assert_attention(out.view(want.shape), lse.view(want_lse.shape), want, want_lse, bound)
    return out, lse


@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 256, 257, 1000])
@pytest.mark.parametrize("heads", [1, 16, 128])
def test_one_token(n, heads):
    g, cache, table = _setup(n + heads, [n], 64)
    _compare(_queries(g, 1, heads), cache, table, [n], [1])


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("heads", [3, 5, 20, 32, 40, 64])
def test_heads_and_pages(page, heads):
    lens = [300, 1, 129]
    g, cache, table = _setup(page + heads, lens, page)
    _compare(_queries(g, 3, heads), cache, table, lens, [1, 1, 1], packed=False)


@pytest.mark.parametrize("drafts", [2, 3, 8, 33, 130])
@pytest.mark.parametrize("heads", [1, 5, 16, 40])
def test_chains_and_chunks(drafts, heads):
    lens = [drafts, drafts + 1, 200 + drafts, 700]
    g, cache, table = _setup(drafts + heads, lens, 32)
    counts = [drafts, 1, max(1, drafts - 1), drafts]
    _compare(_queries(g, sum(counts), heads), cache, table, lens, counts)


@pytest.mark.parametrize("nodes", [1, 2, 13, 31, 64])
@pytest.mark.parametrize("heads", [2, 16])
def test_trees(nodes, heads):
    cpu = torch.Generator().manual_seed(nodes)
    lens = [nodes, nodes + 3, 126 + nodes, 500]
    counts = [nodes, nodes, max(1, nodes // 2), nodes]
    g, cache, table = _setup(nodes + heads, lens, 16)
    tree = torch.tensor([b for n in counts for b in U.random_tree(cpu, n)], dtype=torch.int64, device="cuda")
    _compare(_queries(g, sum(counts), heads), cache, table, lens, counts, tree)


def test_a_chain_as_a_tree_is_the_chain():
    d = U.dsv3()
    lens, counts = [40, 300], [8, 8]
    g, cache, table = _setup(1, lens, 64)
    q = _queries(g, 16, 16)
    tree = torch.tensor([(2 << i) - 1 for i in range(8)] * 2, dtype=torch.int64, device="cuda")
    a = d.latent_attention(*q, cache, table, U.i32(lens), SCALE, cu_seqlens_q=U.offsets(counts))
    b = d.latent_attention(*q, cache, table, U.i32(lens), SCALE, cu_seqlens_q=U.offsets(counts), tree_mask=tree)
    assert torch.equal(a, b)


def test_queries_that_see_nothing():
    lens, counts = [3, 0, 5, 2], [3, 1, 2, 4]            # the last has more queries than tokens
    g, cache, table = _setup(2, lens, 16)
    tree = torch.tensor([0, 2, 0, 1, 0, 0, 0, 0, 4, 12], dtype=torch.int64, device="cuda")
    out, lse = _compare(_queries(g, 10, 5), cache, table, lens, counts, tree)
    assert not out[0].any() and not out[2].any() and not out[3].any() and not out[6].any()
    assert (lse[[0, 2, 3, 6]] == -math.inf).all()
    _compare(_queries(g, 10, 5), cache, table, lens, counts)


def test_sequences_without_queries_and_no_sequences():
    d = U.dsv3()
    lens, counts = [100, 50, 200, 1], [0, 2, 0, 0]
    g, cache, table = _setup(3, lens, 64)
    _compare(_queries(g, 2, 16), cache, table, lens, counts)
    q = _queries(g, 0, 16)
    assert d.latent_attention(*q, cache, table, U.i32(lens), SCALE, cu_seqlens_q=U.offsets([0] * 4)).shape == (0, 16, 512)
    assert d.latent_attention(*_queries(g, 2, 0), cache, table, U.i32(lens), SCALE, cu_seqlens_q=U.offsets(counts)).shape == (2, 0, 512)


def test_absent_pages_and_lengths_beyond_the_table():
    d = U.dsv3()
    g = torch.Generator(device="cuda").manual_seed(5)
    cache = U.make_cache(g, 8, 32)
    table = U.i32([[3, -1, 1, 5], [8, 2, 1 << 30, 0], [-1, -1, -1, -1]])
    lens = [120, 100, 70]
    _compare(_queries(g, 6, 16), cache, table, lens, [2, 2, 2])
    q = _queries(g, 3, 16)
    far = d.latent_attention(*q, cache, table, U.i32([4000, 128, -7]), SCALE)
    near = d.latent_attention(*q, cache, table, U.i32([128, 128, 0]), SCALE)
    assert torch.equal(far, near) and not far[2].any()


def test_strides_of_tokens_and_heads():
    d = U.dsv3()
    lens = [70, 300]
    g, cache, table = _setup(6, lens, 64)
    ql, qr = _queries(g, 6, 16)
    cu, lens_d = U.offsets([3, 3]), U.i32(lens)
    want = d.latent_attention(ql, qr, cache, table, lens_d, SCALE, cu_seqlens_q=cu)
    by_head = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (ql, qr)]
    assert torch.equal(d.latent_attention(*by_head, cache, table, lens_d, SCALE, cu_seqlens_q=cu), want)
    joined = torch.cat([ql, qr], -1)
    assert torch.equal(d.latent_attention(joined[..., :512], joined[..., 512:], cache, table, lens_d, SCALE, cu_seqlens_q=cu), want)
    batch = d.latent_attention(ql.view(2, 3, 16, 512), qr.view(2, 3, 16, 64), cache, table, lens_d, SCALE)
    assert batch.shape == (2, 3, 16, 512) and torch.equal(batch.view(6, 16, 512), want)
    turned = by_head[0].view(2, 3, 16, 512)                      # as an einsum over heads leaves it
    assert torch.equal(d.latent_attention(turned, qr.view(2, 3, 16, 64), cache, table, lens_d, SCALE).view(6, 16, 512), want)
    wide = torch.cat([table, table], 1)
    assert torch.equal(d.latent_attention(ql, qr, cache, wide[:, :table.shape[1]], lens_d, SCALE, cu_seqlens_q=cu), want)


def test_rows_behind_the_last_sequence_are_left():
    import ctypes
    from dsv3_b200 import _lib
    from test_latent_refusals import Cache, _lib as bind
    lib, _ = bind()
    lens, counts = [150, 33], [2, 1]
    g, cache, table = _setup(7, lens, 16)
    q = _queries(g, 5, 16)
    out, lse = torch.full((5, 16, 512), 3.0, dtype=torch.bfloat16, device="cuda"), torch.full((5, 16), 3.0, device="cuda", dtype=torch.float32)
    need = lib.dsv3_latent_attention_workspace_bytes(5, 16, 2, table.shape[1] * 16)
    ws = torch.full((max(need, 1),), 0xFF, dtype=torch.uint8, device="cuda")
    c = Cache(cache.latent.data_ptr(), cache.rope.data_ptr(), cache.scale.data_ptr(), cache.scale.shape[0], 16, table.data_ptr(), table.stride(0), table.shape[1], 2)
    lens_d, cu = U.i32(lens), U.offsets(counts)
    _lib.check(lib.dsv3_latent_attention(ctypes.byref(c), q[0].data_ptr(), 16 * 512, 512, q[1].data_ptr(), 16 * 64, 64, 5, 16, lens_d.data_ptr(), cu.data_ptr(),
                                         None, SCALE, out.data_ptr(), lse.data_ptr(), ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream))
    assert (out[3:] == 3).all() and (lse[3:] == 3).all()
    want, want_lse, bound = U.attention(q[0][:3], q[1][:3], cache, table, lens, counts, SCALE)
    U.assert_attention(out[:3], lse[:3], want, want_lse, bound)


def test_a_token_that_is_not_finite_reaches_only_who_sees_it():
    d = U.dsv3()
    lens, counts = [200], [6]
    g, cache, table = _setup(8, lens, 64)
    q = _queries(g, 6, 16)
    tree = torch.tensor([1, 3, 4, 13, 17, 32], dtype=torch.int64, device="cuda")
    kv = torch.zeros(1, 576, dtype=torch.bfloat16, device="cuda")
    kv[0, 9] = math.nan
    slot = table[0, 196 // 64].long() * 64 + 196 % 64                       # draft 2
    d.latent_cache_write(cache, kv, torch.ones(512, dtype=torch.bfloat16, device="cuda"), torch.ones(4, 32, dtype=torch.complex64, device="cuda"),
                         torch.zeros(1, dtype=torch.int64, device="cuda"), slot.view(1))
    out, lse = _compare(q, cache, table, lens, counts, tree)
    assert torch.isnan(out[[2, 3]]).all() and not torch.isnan(out[[0, 1, 4, 5]]).any()


def test_queries_that_are_not_finite_stay_in_their_row():
    d = U.dsv3()
    lens = [300, 40]
    g, cache, table = _setup(9, lens, 64)
    ql, qr = _queries(g, 2, 16)
    clean = d.latent_attention(ql, qr, cache, table, U.i32(lens), SCALE)
    ql[0, 3, 100], qr[1, 7, 5], ql[1, 2, 0] = math.nan, math.inf, -math.inf
    out = d.latent_attention(ql, qr, cache, table, U.i32(lens), SCALE)
    bad = torch.zeros(2, 16, dtype=torch.bool, device="cuda")
    bad[0, 3] = bad[1, 7] = bad[1, 2] = True
    assert torch.isnan(out[bad]).all() and torch.equal(out[~bad], clean[~bad])


@pytest.mark.parametrize("size", [0.0, 1e-3, 8.0, 60.0])
def test_flat_and_sharp_softmax(size):
    lens = [513, 129]
    g, cache, table = _setup(10, lens, 64, spread=64.0)
    ql, qr = _queries(g, 4, 16, size)
    _compare((ql, (qr * min(size, 1.0)).bfloat16()), cache, table, lens, [2, 2])


def test_one_token_draws_nearly_everything():
    """A first token 13 units of the exponent above 6000 others: each of them weighs 2e-6 of it, together 1.3 %, which must not be lost."""
    n = 6001
    g, cache, table = _setup(11, [n], 64, spread=1.0)
    ql = torch.zeros(1, 16, 512, dtype=torch.bfloat16, device="cuda")
    qr = torch.zeros(1, 16, 64, dtype=torch.bfloat16, device="cuda")
    qr[:, :, 0] = 13.0
    latent, rope, scale = cache
    rope[:, :, 0] = 0
    slot = int(table[0, 0]) * 64
    rope.view(-1, 64)[slot, 0] = (1.0 / scale.view(-1)[slot]).bfloat16()
    # all the others point the same way
    common = torch.ones(512, device="cuda")
    names = table[0][table[0] >= 0].long()
    latent[names] = (common / 2.0 ** -8).to(torch.float8_e4m3fn).expand(len(names), 64, 512)
    scale[names] = 2.0 ** -8
    rope[names] = 0
    rope.view(-1, 64)[slot, 0] = 2.0 ** 8
    latent.view(-1, 512)[slot] = 0
    U.poison_rest(cache, table, [n])
    out, _ = _compare((ql, qr), cache, table, [n], [1], scale=1.0)
    p = 6000 * math.exp(-13) / (1 + 6000 * math.exp(-13))
    assert abs(out.double().mean().item() - p) < p * 2.0 ** -7


def test_scales_of_tokens_far_apart():
    lens = [400]
    g, cache, table = _setup(12, lens, 64, spread=2.0 ** 24)
    _compare(_queries(g, 2, 16, 0.05), cache, table, lens, [2])


def test_small_latent_queries_beside_large_rotated_ones():
    lens = [260]
    g, cache, table = _setup(13, lens, 64)
    ql, qr = _queries(g, 3, 16)
    ql[0] *= 2.0 ** -50
    ql[1] = 0
    qr[2] = 0
    _compare((ql, qr), cache, table, lens, [3])


def test_many_sequences():
    lens = [(i * 37) % 290 + 1 for i in range(333)]
    g, cache, table = _setup(14, lens, 16)
    _compare(_queries(g, 333, 4), cache, table, lens, [1] * 333, packed=False)


@pytest.mark.parametrize("heads, drafts", [(5, 1), (12, 3), (40, 1)])
def test_more_sequences_than_threads(heads, drafts):
    """1400 sequences: the list of tiles is added up in several rounds.  One is long, some have no queries."""
    lens = [(i * 37) % 140 + 3 for i in range(1400)]
    lens[901] = 5000
    counts = [0 if i % 11 == 5 else drafts for i in range(1400)]
    g, cache, table = _setup(19 + heads, lens, 16)
    _compare(_queries(g, sum(counts), heads), cache, table, lens, counts)


@pytest.mark.parametrize("lens, heads, drafts", [([1100] * 140, 16, 1), ([1300] + [200] * 120, 8, 1), ([700, 650, 1100] * 12, 128, 1), ([620] * 9, 16, 15), ([4000, 3999], 16, 70)])
def test_blocks_left_whole_and_blocks_cut(lens, heads, drafts):
    """About as many blocks as SMs, equal and not, and far more: cut among CTAs or one to each, by what their lengths say."""
    g, cache, table = _setup(23 + heads, lens, 64)
    q = _queries(g, drafts * len(lens), heads)
    _compare(q, cache, table, lens, [drafts] * len(lens))


def test_a_wide_table_is_the_narrow_one():
    """Short sequences in a table for 40 times their length: whole blocks either way, and the same bits."""
    d = U.dsv3()
    lens = [300, 20, 129, 384]
    g, cache, table = _setup(22, lens, 16)
    q = _queries(g, 4, 16)
    wide = torch.full((4, 1000), -1, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    narrow = _compare(q, cache, table, lens, [1] * 4)
    out = d.latent_attention(*q, cache, wide, U.i32(lens), SCALE, return_lse=True)
    assert torch.equal(out[0], narrow[0]) and torch.equal(out[1], narrow[1])


def test_slots_whose_bytes_pass_32_bits():
    """A pool of 8.4 million tokens, of which one sequence uses pages at both ends: offsets in bytes pass 2^32."""
    d = U.dsv3()
    n_pages, page, n = 131200, 64, 300
    g = torch.Generator(device="cuda").manual_seed(20)
    small = U.make_cache(g, 5, page)
    cache = d.LatentCache(*(torch.empty(n_pages, *t.shape[1:], dtype=t.dtype, device="cuda") for t in small))
    names = [n_pages - 1, 0, n_pages - 40, 131071, 131072]
    assert names[3] * page * 512 < 1 << 32 <= names[4] * page * 512
    for big, few in zip(cache, small):
        for i, name in enumerate(names):
            big[name] = few[i]
    table, few = U.i32([names]), U.i32([list(range(5))])
    q = _queries(g, 2, 16)
    out = d.latent_attention(*q, cache, table, U.i32([n]), SCALE, return_lse=True)
    want = d.latent_attention(*q, small, few, U.i32([n]), SCALE, return_lse=True)
    assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
    for a, b in zip(d.latent_cache_read(cache, table, U.offsets([n]), n), d.latent_cache_read(small, few, U.offsets([n]), n)):
        assert torch.equal(a, b)
    kv = torch.randn(2, 576, generator=g, device="cuda", dtype=torch.float32).bfloat16()
    f, w = torch.ones(4, 32, dtype=torch.complex64, device="cuda"), torch.ones(512, dtype=torch.bfloat16, device="cuda")
    for c, slots in ((cache, [n_pages * page - 1, 131072 * page + 5]), (small, [63, 4 * page + 5])):
        d.latent_cache_write(c, kv, w, f, torch.arange(2, device="cuda"), torch.tensor(slots, device="cuda"))
    d.latent_cache_keep(cache, table, U.i32([60]), U.i32([[3, 200]]), U.i32([2]))
    d.latent_cache_keep(small, few, U.i32([60]), U.i32([[3, 200]]), U.i32([2]))
    for big, few_of in zip(cache, small):
        for i, name in enumerate(names):
            assert torch.equal(big[name].view(torch.uint8), few_of[i].view(torch.uint8))


@pytest.mark.parametrize("heads, drafts", [(16, 1), (16, 2), (128, 1)])
def test_one_long_among_many(heads, drafts):
    """A block cut among nearly all SMs, whose parts are joined in two steps, among others in few parts and whole ones."""
    lens = [100] * 40 + [16000] + [300, 129, 1] * 10
    g, cache, table = _setup(17 + heads + drafts, lens, 64)
    counts = [drafts if n > 1 else 1 for n in lens]
    q = _queries(g, sum(counts), heads)
    first = _compare(q, cache, table, lens, counts)
    for _ in range(3):                                                     # whichever CTA comes last
        again = U.dsv3().latent_attention(*q, cache, table, U.i32(lens), SCALE, cu_seqlens_q=U.offsets(counts), return_lse=True)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_long_sequence():
    lens, counts = [20011, 3], [2, 1]
    g, cache, table = _setup(15, lens, 128)
    _compare(_queries(g, 3, 16), cache, table, lens, counts)


def test_results_do_not_change_from_call_to_call():
    d = U.dsv3()
    lens = [3000, 17, 1200, 640]
    g, cache, table = _setup(16, lens, 64)
    q = _queries(g, 8, 16)
    first = d.latent_attention(*q, cache, table, U.i32(lens), SCALE, return_lse=True)
    for _ in range(5):
        again = d.latent_attention(*q, cache, table, U.i32(lens), SCALE, return_lse=True)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
