"""latent_cache_write, latent_cache_read and latent_cache_keep against their definitions in 64 bits.

Tolerances.  A stored latent is c / s in e4m3: half a step, 2^-4 of it, or 2^-10 where it is below the smallest normal (2^-6); c itself comes from fp32
arithmetic, 2^-20 of it (some ten roundings and the sum of 512 squares), which decides on which side of a tie it falls: one whole step there, which
the half-step bound plus that covers.  A rotated value is bf16: 2^-8 of it, plus the fp32 rotation's 2^-22 of the pair's length.  What read gives is the
exact product, and what keep moves is moved bit for bit."""
import math

import pytest
import torch

import latent_util as U

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _status():
    yield
    import dsv3_b200
    dsv3_b200.check_device_status()


def _inputs(n, seed, weight=torch.bfloat16, positions=512):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kv = (torch.randn(n, 576, generator=g, device="cuda", dtype=torch.float32) * 3).bfloat16()
    w = (1 + 0.2 * torch.randn(512, generator=g, device="cuda", dtype=torch.float32)).to(weight)
    angle = torch.rand(positions, 32, generator=g, device="cuda", dtype=torch.float32) * 6.2831853
    f = torch.polar(torch.ones_like(angle), angle)
    at = torch.randint(0, positions, (n,), generator=g, device="cuda")
    return g, kv, w, f, at


def _definition(kv, w, f, at, eps):
    x = kv.double()
    c = x[:, :512] / torch.sqrt(x[:, :512].square().mean(-1, keepdim=True) + eps) * w.double()
    z = torch.view_as_complex(x[:, 512:].reshape(len(x), 32, 2)) * f[at].to(torch.complex128)
    return c, torch.view_as_real(z).reshape(len(x), 64)


def _check(cache, slots, c, k):
    s = cache.scale.view(-1)[slots].double()
    top = c.abs().amax(-1).clamp_min(1e-4)
    want = U.least_power(top)
    border = (top / (448 * want) > 1 - 2.0 ** -20) | (top / (224 * want) < 1 + 2.0 ** -20)
    assert torch.equal(s[~border], want[~border])
    assert ((s == want) | (s == 2 * want) | (s * 2 == want)).all()
    q = cache.latent.view(-1, 512)[slots].double()
    v = c / s[:, None]
    assert ((q - v).abs() <= torch.maximum(v.abs() * 2.0 ** -4, torch.full_like(v, 2.0 ** -10)) + v.abs() * 2.0 ** -20).all()
    r = cache.rope.view(-1, 64)[slots].double() * s[:, None]
    length = k.reshape(len(k), 32, 2).norm(dim=-1).repeat_interleave(2, -1)
    assert ((r - k).abs() <= k.abs() * 2.0 ** -8 + length * 2.0 ** -22).all()


@pytest.mark.parametrize("n", [1, 7, 8, 9, 300])
@pytest.mark.parametrize("weight", [torch.bfloat16, torch.float32])
def test_write(n, weight):
    d = U.dsv3()
    g, kv, w, f, at = _inputs(n, n, weight)
    cache = U.make_cache(g, 11, 32)
    before = [p.clone() for p in cache]
    slots = torch.randperm(11 * 32, generator=g, device="cuda")[:n]
    d.latent_cache_write(cache, kv, w, f, at, slots, 1e-6)
    _check(cache, slots, *_definition(kv, w, f, at, 1e-6))
    rest = torch.ones(11 * 32, dtype=torch.bool, device="cuda")
    rest[slots] = False
    for old, new in zip(before, cache):                     # the other tokens are left as they were
        assert torch.equal(old.view(torch.uint8).reshape(11 * 32, -1)[rest], new.view(torch.uint8).reshape(11 * 32, -1)[rest])


def test_write_of_a_strided_view_and_of_a_batch():
    d = U.dsv3()
    g, kv, w, f, at = _inputs(24, 5)
    wide = torch.randn(24, 640, device="cuda", dtype=torch.float32).bfloat16()
    wide[:, 64:] = kv
    slots = torch.randperm(64, generator=g, device="cuda")[:24]
    caches = [d.allocate_latent_cache(4, 16) for _ in range(3)]
    d.latent_cache_write(caches[0], kv, w, f, at, slots)
    d.latent_cache_write(caches[1], wide[:, 64:], w, f, at, slots)
    d.latent_cache_write(caches[2], kv.view(2, 12, 576), w, f, at.view(2, 12), slots.view(2, 12))
    for other in caches[1:]:
        for a, b in zip(caches[0], other):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_slots_outside_the_pool_are_not_written():
    d = U.dsv3()
    g, kv, w, f, at = _inputs(6, 6)
    cache = d.allocate_latent_cache(2, 16)
    slots = torch.tensor([-1, 32, 3, -(1 << 40), 1 << 40, 31], device="cuda")
    d.latent_cache_write(cache, kv, w, f, at, slots)
    touched = cache.latent.view(torch.uint8).view(32, 512).any(-1)
    assert touched.nonzero().flatten().tolist() == [3, 31]
    _check(cache, slots[[2, 5]], *[t[[2, 5]] for t in _definition(kv, w, f, at, 1e-6)])


def test_values_at_the_ends_of_the_range():
    """Zeros, latents around the floor and ones whose largest is at a border of the scale."""
    d = U.dsv3()
    g, kv, w, f, at = _inputs(40, 7)
    w = torch.ones(512, device="cuda", dtype=torch.float32)
    kv[0] = 0
    kv[1, :512] = 0
    kv[2:10] *= 2.0 ** -60                       # eps decides: latents far below the floor
    kv[10:20] *= 2.0 ** 40
    kv[20, :512] = 0
    kv[20, 0] = 1.0                              # a single value: its latent is sqrt(512)
    cache = d.allocate_latent_cache(3, 16)
    slots = torch.arange(40, device="cuda")
    d.latent_cache_write(cache, kv, w, f, at, slots, 1e-6)
    _check(cache, slots, *_definition(kv, w, f, at, 1e-6))


def test_tokens_that_are_not_finite_are_stored_as_such():
    d = U.dsv3()
    g, kv, w, f, at = _inputs(8, 8)
    kv[1, 5] = math.nan
    kv[2, 100] = math.inf
    kv[3, 520] = math.nan
    kv[4, 575] = -math.inf
    at[5], at[6] = -1, 512
    cache = U.make_cache(g, 1, 16)
    d.latent_cache_write(cache, kv, w, f, at, torch.arange(8, device="cuda"))
    for t in range(1, 7):
        assert math.isnan(cache.scale[0, t].item())
        assert not cache.latent.view(torch.uint8)[0, t].any() and not cache.rope[0, t].any()
    good = torch.tensor([0, 7], device="cuda")
    _check(cache, good, *[t[good] for t in _definition(kv, w, f, at.clamp(0, 511), 1e-6)])


def test_write_agrees_with_act_quant():
    """The same latents through act_quant with blocks of 512 and power-of-two scales: where fp32's last bits do not decide, the same bytes."""
    d = U.dsv3()
    g, kv, w, f, at = _inputs(64, 9)
    cache = d.allocate_latent_cache(4, 16)
    d.latent_cache_write(cache, kv, w, f, at, torch.arange(64, device="cuda"))
    c, _ = _definition(kv, w, f, at, 1e-6)
    y, s = d.act_quant(c.bfloat16().contiguous(), 512, "ue8m0")
    assert (s.view(-1) == cache.scale.view(-1)).float().mean().item() > 0.95
    # bf16 on the way moves a value by 2^-8, a step is 2^-3: one in sixteen may change at most
    assert (y.view(torch.uint8) != cache.latent.view(64, 512).view(torch.uint8)).float().mean().item() < 1 / 16 + 0.05


@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("lens", [[1], [0], [17, 0, 0, 64, 1, 65], [300], [33] * 270])
def test_read(page, lens):
    d = U.dsv3()
    g = torch.Generator(device="cuda").manual_seed(len(lens) + page)
    n_pages = sum(-(-n // page) for n in lens) + 2
    cache = U.make_cache(g, n_pages, page, spread=2.0 ** 20)
    table = U.block_table(g, lens, page, n_pages)
    U.poison_rest(cache, table, lens)
    total = sum(lens)
    latent, rope = d.latent_cache_read(cache, table, U.offsets(lens), total)
    assert latent.shape == (total, 512) and rope.shape == (total, 64)
    row = 0
    for b, n in enumerate(lens):
        if n:
            c, k, _ = U.tokens_of(cache, table, b, n)
            assert torch.equal(latent[row:row + n].double(), c) and torch.equal(rope[row:row + n].double(), k)
        row += n


def test_read_of_absent_pages_and_rows_behind_the_last_sequence():
    import ctypes
    d = U.dsv3()
    from dsv3_b200 import _lib
    from test_latent_refusals import Cache, _lib as bind
    lib, _ = bind()
    g = torch.Generator(device="cuda").manual_seed(3)
    cache = U.make_cache(g, 4, 16)
    table = U.i32([[2, -1, 0], [7, 1, 1 << 30]])
    lens = [40, 37]
    latent, rope = d.latent_cache_read(cache, table, U.offsets(lens), 77)
    for b, lo in ((0, 0), (1, 40)):
        c, k, there = U.tokens_of(cache, table, b, lens[b])
        assert torch.equal(latent[lo:lo + lens[b]].double(), torch.where(there[:, None], c, 0.0))
        assert torch.equal(rope[lo:lo + lens[b]].double(), torch.where(there[:, None], k, 0.0))
    out, out2 = torch.full((80, 512), 7.0, dtype=torch.bfloat16, device="cuda"), torch.full((80, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    c = Cache(cache.latent.data_ptr(), cache.rope.data_ptr(), cache.scale.data_ptr(), 4, 16, table.data_ptr(), 3, 3, 2)
    cu = U.offsets(lens)
    _lib.check(lib.dsv3_latent_read(ctypes.byref(c), cu.data_ptr(), 80, out.data_ptr(), out2.data_ptr(), torch.cuda.current_stream().cuda_stream))
    assert torch.equal(out[:77], latent) and (out[77:] == 7).all() and (out2[77:] == 7).all()


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("drafts", [1, 8, 33, 64, 200])
def test_keep(page, drafts):
    d = U.dsv3()
    g = torch.Generator(device="cuda").manual_seed(drafts + page)
    cpu = torch.Generator().manual_seed(drafts)
    firsts = [0, 5, 16, 129, 40, 7]
    lens = [n + drafts for n in firsts]
    n_pages = sum(-(-n // page) for n in lens)
    cache = U.make_cache(g, n_pages, page, spread=4.0)
    table = U.block_table(g, lens, page, n_pages)
    counts = [0, 1, drafts, max(1, drafts // 2), max(1, drafts - 1), max(1, drafts // 3)]
    path = torch.zeros(6, drafts, dtype=torch.int32)
    for b, n in enumerate(counts):
        path[b, :n] = torch.sort(torch.randperm(drafts, generator=cpu)[:n]).values.int()
    want = [p.view(torch.uint8).reshape(n_pages * page, -1).clone() for p in cache]
    for b, n in enumerate(counts):
        slot = lambda p: int(table[b, p // page]) * page + p % page  # noqa: E731
        src = [slot(firsts[b] + int(path[b, j])) for j in range(n)]
        dst = [slot(firsts[b] + j) for j in range(n)]
        for w in want:
            w[dst] = w[src].clone()
    wide = torch.full((6, drafts + 3), -5, dtype=torch.int32, device="cuda")       # rows of the path further apart than they are long
    wide[:, :drafts] = path.cuda()
    d.latent_cache_keep(cache, table, U.i32(firsts), wide[:, :drafts], U.i32(counts))
    for p, w in zip(cache, want):
        assert torch.equal(p.view(torch.uint8).reshape(n_pages * page, -1), w)


def test_keep_leaves_alone_what_lies_in_no_page():
    d = U.dsv3()
    g = torch.Generator(device="cuda").manual_seed(4)
    cache = U.make_cache(g, 3, 16)
    before = [p.clone() for p in cache]
    table = U.i32([[0, -1], [1, 9]])
    d.latent_cache_keep(cache, table, U.i32([14, 20]), U.i32([[1, 3, 5], [0, 1, 2]]), U.i32([3, 3]))
    # sequence 0: draft 1 (position 15) moves to 14; the others come from an absent page.  Sequence 1 has nothing there at all.
    assert torch.equal(cache.latent.view(torch.uint8)[0, 14], before[0].view(torch.uint8)[0, 15])
    for p, b in zip(cache, before):
        p, b = p.view(torch.uint8).reshape(48, -1).clone(), b.view(torch.uint8).reshape(48, -1).clone()
        p[14] = b[14] = 0
        assert torch.equal(p, b)
