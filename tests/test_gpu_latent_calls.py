"""How the operators of the latent cache are called: graphs, streams, threads, many calls at once, a budget of SMs."""
import threading

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
    dsv3_b200.set_num_sms(0)


def _problem(seed, lens, heads=16, drafts=1, page=64):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n_pages = sum(-(-n // page) for n in lens) + 1
    cache = U.make_cache(g, n_pages, page)
    table = U.block_table(g, lens, page, n_pages)
    total = drafts * len(lens)
    q = (torch.randn(total, heads, 512, generator=g, device="cuda", dtype=torch.float32).bfloat16(),
         torch.randn(total, heads, 64, generator=g, device="cuda", dtype=torch.float32).bfloat16())
    lens_d = U.i32(lens)
    return lambda: U.dsv3().latent_attention(*q, cache, table, lens_d, SCALE, return_lse=True), (q, cache, table, lens_d)


def _same(a, b):
    return torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_lengths_that_change_between_replays():
    """A captured step whose lengths, table and queries live in device memory: each replay sees what they hold then."""
    call, (q, cache, table, lens) = _problem(1, [900, 300, 64])
    call()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = call()
    for now in ([900, 300, 64], [1, 2, 3], [128, 129, 0], [900, 1, 64]):
        lens.copy_(U.i32(now))
        want = [t.clone() for t in call()]
        graph.replay()
        torch.cuda.synchronize()
        assert _same(out, want)


def test_two_graphs_of_one_stream_and_an_eager_call_between():
    a, _ = _problem(2, [3000, 400])
    b, _ = _problem(3, [70] * 40, heads=32)
    want = [[t.clone() for t in f()] for f in (a, b)]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    for f in (a, b):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=stream):
            outs.append(f())
    for _ in range(3):
        graphs[1].replay()
        graphs[0].replay()
        eager = a()
        graphs[1].replay()
        torch.cuda.synchronize()
        assert _same(eager, want[0]) and _same(outs[0], want[0]) and _same(outs[1], want[1])


def test_calls_on_two_streams_at_once():
    problems = [_problem(10 + i, [2500, 600, 30], heads=16 if i % 2 else 128) for i in range(4)]
    want = [[t.clone() for t in f()] for f, _ in problems]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    for _ in range(3):
        outs = []
        for s, (f, _) in zip(streams, problems):
            with torch.cuda.stream(s):
                outs.append(f())
        torch.cuda.synchronize()
        assert all(_same(o, w) for o, w in zip(outs, want))


def test_threads_with_streams_of_their_own():
    problems = [_problem(20 + i, [1500 + 100 * i, 40]) for i in range(4)]
    want = [[t.clone() for t in f()] for f, _ in problems]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(20):
                out = problems[i][0]()
                s.synchronize()
                if not _same(out, want[i]):
                    bad.append(i)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


@pytest.mark.parametrize("sms", [2, 7, 100])
@pytest.mark.parametrize("heads", [16, 128])
def test_a_budget_of_sms(sms, heads):
    call, (q, cache, table, lens) = _problem(30, [1000, 200, 129, 64], heads)
    want, want_lse, bound = U.attention(*q, cache, table, [1000, 200, 129, 64], [1] * 4, SCALE)
    U.dsv3().set_num_sms(sms)
    out, lse = call()
    U.assert_attention(out, lse, want, want_lse, bound)


def test_write_attend_keep_and_read_in_a_row():
    """A prompt, a tree of drafts, what is kept of it, the next token: on one stream, with nothing waiting in between."""
    d = U.dsv3()
    g = torch.Generator(device="cuda").manual_seed(40)
    cache = d.allocate_latent_cache(12, 32)
    table = U.i32([[7, 2, 9, 0], [1, 11, 4, 5]])
    angle = torch.rand(128, 32, generator=g, device="cuda", dtype=torch.float32)
    freqs, weight = torch.polar(torch.ones_like(angle), angle), torch.ones(512, device="cuda", dtype=torch.float32)
    slot = lambda b, p: int(table[b, p // 32]) * 32 + p % 32  # noqa: E731

    def write(kv, seqs, positions, depths):
        slots = torch.tensor([slot(b, p) for b, p in zip(seqs, positions)], device="cuda")
        d.latent_cache_write(cache, kv, weight, freqs, torch.tensor(depths, device="cuda"), slots)
    prompt = torch.randn(2 * 60, 576, generator=g, device="cuda", dtype=torch.float32).bfloat16()
    write(prompt, [0] * 60 + [1] * 60, list(range(60)) * 2, list(range(60)) * 2)
    drafts = torch.randn(8, 576, generator=g, device="cuda", dtype=torch.float32).bfloat16()
    write(drafts, [0] * 4 + [1] * 4, [60, 61, 62, 63] * 2, [60, 60, 61, 62] * 2)
    tree = torch.tensor([1, 2, 6, 14] * 2, device="cuda")
    q = (torch.randn(8, 16, 512, generator=g, device="cuda", dtype=torch.float32).bfloat16(), torch.randn(8, 16, 64, generator=g, device="cuda", dtype=torch.float32).bfloat16())
    out, lse = d.latent_attention(*q, cache, table, U.i32([64, 64]), SCALE, cu_seqlens_q=U.offsets([4, 4]), tree_mask=tree, return_lse=True)
    want = U.attention(*q, cache, table, [64, 64], [4, 4], SCALE, tree)
    d.latent_cache_keep(cache, table, U.i32([60, 60]), U.i32([[1, 2, 3], [0, 0, 0]]), U.i32([3, 1]))
    nxt, nxt_lse = d.latent_attention(q[0][:2], q[1][:2], cache, table, U.i32([63, 61]), SCALE, return_lse=True)
    latent, rope = d.latent_cache_read(cache, table, U.offsets([63, 61]), 124)
    U.assert_attention(out, lse, *want)
    U.assert_attention(nxt, nxt_lse, *U.attention(q[0][:2], q[1][:2], cache, table, [63, 61], [1, 1], SCALE))
    other = d.allocate_latent_cache(12, 32)
    d.latent_cache_write(other, drafts[1:4], weight, freqs, torch.tensor([60, 61, 62], device="cuda"), torch.arange(3, device="cuda"))
    for j in range(3):                                                      # the branch of nodes 1, 2, 3 now follows the prompt
        s = slot(0, 60 + j)
        assert torch.equal(cache.latent.view(torch.uint8).view(-1, 512)[s], other.latent.view(torch.uint8).view(-1, 512)[j])
        assert torch.equal(latent[60 + j].double(), other.latent.view(-1, 512)[j].double() * other.scale.view(-1)[j].double())
