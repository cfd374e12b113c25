"""install_mla: sequences of a batch that are of different lengths, as after drafts of which different numbers were kept."""
import pytest
import torch

import latent_util as U
from test_gpu_mla_seam import _bf16_default, _cached, _freqs, _model, _off  # noqa: F401

pytestmark = pytest.mark.gpu
# Two runs of one sequence, in batches of their own, differ by how projections and attention are cut: roundings to bf16 at queries, result and output, 2^-9 RMS each, and the
# same for tokens whose latents go to another e4m3 value by a last bit of a projection.
CLOSE = 2.0 ** -7


def _causal(n):
    return torch.full((n, n), float("-inf"), device="cuda").triu_(1)


def _tokens(batch, n, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(batch, n, 256, generator=g, device="cuda", dtype=torch.float32).bfloat16()


@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
def test_a_batch_goes_on_after_drafts_of_which_different_numbers_are_kept(kind):
    import dsv3_b200
    m, f = _model(16, 128), _freqs(200)
    x, drafts, after = _tokens(3, 50, 7), _tokens(3, 6, 8), _tokens(3, 4, 9)
    m(x, 0, f[:50], _causal(50))
    parent = [-1, -1, 0, 1, 3, 4]
    words, depth = [], []
    for i, p in enumerate(parent):
        words.append((words[p] if p >= 0 else 0) | 1 << i)
        depth.append(depth[p] + 1 if p >= 0 else 0)
    m(drafts, 50, f[50 + torch.tensor(depth, device="cuda")], torch.tensor([words] * 3, device="cuda"))
    kept = [[1, 3, 4, 5], [0, 2], [1]]
    cache = dsv3_b200.mla_cache(m)
    path = torch.zeros(3, 6, dtype=torch.int32, device="cuda")
    for b, nodes in enumerate(kept):
        path[b, :len(nodes)] = U.i32(nodes)
    dsv3_b200.latent_cache_keep(cache.pool, cache.block_table, U.i32([50] * 3), path, U.i32([len(k) for k in kept]))
    at = torch.tensor([50 + len(k) for k in kept], device="cuda", dtype=kind)
    step = m(after[:, :1], at, f[at.long()][:, None], None)
    tree = torch.tensor([[1, 2, 5]] * 3, device="cuda")
    nodes = torch.tensor([0, 0, 1], device="cuda")
    more = m(after[:, 1:], at + 1, f[(at.long() + 1)[:, None] + nodes], tree)
    chunk = m(after[:, 1:], at + 1, f[(at.long() + 1)[:, None] + torch.arange(3, device="cuda")], _causal(3))
    for b, nodes_kept in enumerate(kept):                                   # the same sequence, alone and never drafted
        one, n = _model(16, 128), 50 + len(kept[b])
        one(x[b:b + 1], 0, f[:50], _causal(50))
        one(drafts[b:b + 1, nodes_kept], 50, f[50:n], _causal(len(nodes_kept)))
        assert _off(step[b:b + 1], one(after[b:b + 1, :1], n, f[n:n + 1], None)) < CLOSE
        assert _off(more[b:b + 1], one(after[b:b + 1, 1:], n + 1, f[n + 1 + nodes], tree[:1])) < CLOSE
        assert _off(chunk[b:b + 1], one(after[b:b + 1, 1:], n + 1, f[n + 1:n + 4], _causal(3))) < CLOSE


def test_one_start_for_all_as_a_number_and_as_a_tensor():
    m, f, x = _model(4, 0), _freqs(200), _tokens(2, 61, 10)
    m(x[:, :60], 0, f[:60], _causal(60))
    want = m(x[:, 60:], 60, f[60:61], None)
    tokens = [t.clone() for t in _cached(m, 2, 61)]
    at = torch.tensor([60, 60], device="cuda")
    for freqs in (f[60:61], f[at][:, None]):
        assert _off(m(x[:, 60:], at, freqs, None), want) < 2.0 ** -9           # (a wider table: the work may be cut another way)
        assert all(torch.equal(a, b) for a, b in zip(_cached(m, 2, 61), tokens))


def test_a_captured_step_that_goes_on():
    m, plain, f, x = _model(16, 0), _model(16, 0), _freqs(200), _tokens(2, 70, 11)
    for one in (m, plain):
        one(x[:, :60], 0, f[:60], _causal(60))
    at, token, angles = torch.tensor([60, 60], device="cuda"), x[:, 60:61].clone(), f[60:61].repeat(2, 1)[:, None].clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = m(token, at, angles, None)
    for n in range(60, 70):
        at.fill_(n)
        token.copy_(x[:, n:n + 1])
        angles.copy_(f[n])
        graph.replay()
        assert _off(out, plain(x[:, n:n + 1], n, f[n:n + 1], None)) < 2.0 ** -9
    assert all(torch.equal(a, b) for a, b in zip(_cached(m, 2, 70), _cached(plain, 2, 70)))


def test_sequences_that_are_full_and_starts_that_are_none():
    m, f, x = _model(4, 0), _freqs(210), _tokens(3, 40, 12)
    m(x, 0, f[:40], _causal(40))
    before = [t.clone() for t in _cached(m, 3, 200)]
    at = torch.tensor([200, 40, -1], device="cuda")
    out = m(x[:, :1], at, f[at.clamp_min(0)][:, None], None)
    assert torch.isnan(out[[0, 2]]).all() and not torch.isnan(out[1]).any()
    after = _cached(m, 3, 200)
    for a, b in zip(after, before):
        assert torch.equal(a[[0, 2]], b[[0, 2]]) and torch.equal(a[1, :40], b[1, :40]) and not torch.equal(a[1, 40], b[1, 40])
    at = torch.tensor([198, 40, 197], device="cuda")                        # three tokens: the first sequence holds two of them
    out = m(x[:, :3], at, f[at[:, None] + torch.arange(3, device="cuda")], _causal(3))
    assert torch.isnan(out[0]).all() and not torch.isnan(out[1:]).any()
    window = _causal(3)
    window[2, 0] = -1.0
    assert torch.isnan(m(x[:, :3], at, f[at[:, None] + torch.arange(3, device="cuda")], window)).all()


def test_starts_that_are_refused():
    m, f, x = _model(4, 0), _freqs(200), _tokens(2, 1, 13)
    for bad in (torch.tensor([1, 2, 3], device="cuda"), torch.tensor([1.0, 2.0], device="cuda"), torch.tensor([1, 2])):
        with pytest.raises(ValueError, match="start_pos"):
            m(x, bad, f[:1], None)
    with pytest.raises(ValueError, match="do not fit"):
        m(x, -1, f[:1], None)


@pytest.mark.parametrize("shape", [(8, 32), (2, 32), (3, 32), (1, 4, 32), (3, 4, 32), (2, 8, 32), (2, 4, 16), (4, 64), (2, 2, 4, 32)])
def test_angles_of_other_shapes_are_refused(shape):
    """Of two sequences of four tokens; eight rows would do for both, but the second sequence's are not the first's."""
    m, x = _model(4, 0), _tokens(2, 4, 15)
    with pytest.raises(ValueError, match="freqs_cis"):
        m(x, 0, torch.ones(shape, dtype=torch.complex64, device="cuda"), _causal(4))
