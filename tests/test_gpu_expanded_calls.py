"""Calls of expanded attention, its joins and rotary positions as a serving program makes them: graphs, streams, threads, rows that belong to nobody, one operator behind another."""
import ctypes
import threading

import pytest
import torch

from expanded_util import SCALE, check, inputs, offsets, reference
from test_expanded_refusals import Args, _lib

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _status():
    yield
    import dsv3_b200
    dsv3_b200.check_device_status()


def _c_args(q_nope, q_rope, k_nope, k_rope, v, out, lse, cu_q, cu_k, n_seqs, causal=1):
    t = lambda x: x.data_ptr()  # noqa: E731
    return Args(t(q_nope), q_nope.stride(0), q_nope.stride(1), t(q_rope), q_rope.stride(0), q_rope.stride(1), t(k_nope), k_nope.stride(0), k_nope.stride(1), t(k_rope), k_rope.stride(0),
                t(v), v.stride(0), v.stride(1), q_nope.shape[0], k_nope.shape[0], q_nope.shape[1], n_seqs, t(cu_q), t(cu_k), causal, SCALE, t(out), t(lse))


@pytest.mark.parametrize("q, k, heads", [([100, 40], [130, 70], 2), ([3, 2], [3000, 2000], 2), ([300], [300], 130)])
def test_rows_that_belong_to_no_sequence_are_left_as_they_are(q, k, heads):
    """Through the C entry point, into memory that holds something: rows before the first sequence and behind the last one."""
    lib, names = _lib()
    front, back = 5, 300
    args = inputs([front] + q + [back], [7] + k + [9], heads)
    for t in args:
        t[:4], t[-9:] = float("nan"), float("nan")
    cu_q, cu_k = offsets([front] + q)[1:].contiguous(), offsets([7] + k)[1:].contiguous()
    tokens = front + sum(q) + back
    out = torch.full((tokens, heads, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    lse = torch.full((tokens, heads), 7.0, device="cuda")
    need = lib.dsv3_expanded_attention_workspace_bytes(tokens, args[2].shape[0], heads, len(q), 1, 1)
    ws = torch.full((max(need, 1),), 0xFF, dtype=torch.uint8, device="cuda")
    c = _c_args(*args, out, lse, cu_q, cu_k, len(q))
    assert lib.dsv3_expanded_attention(ctypes.byref(c), ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream) == names.OK
    here = slice(front, front + sum(q))
    keys = slice(7, 7 + sum(k))
    want, want_lse, bound, lse_bound = reference(args[0][here], args[1][here], args[2][keys], args[3][keys], args[4][keys], q, k)
    check(out[here], want, bound)
    check(lse[here], want_lse, lse_bound)
    for t in (out, lse):
        assert bool((t[:front] == 7).all()) and bool((t[front + sum(q):] == 7).all())


def test_offsets_that_lead_out_of_the_tensors_are_cut_off():
    from dsv3_b200 import expanded_attention
    args = inputs([100], [150], 2)
    out = expanded_attention(*args, SCALE, torch.tensor([0, 1000], dtype=torch.int32, device="cuda"), torch.tensor([-5, 1 << 30], dtype=torch.int32, device="cuda"))
    want, _, bound, _ = reference(*args, [100], [150])
    check(out, want, bound)


@pytest.mark.parametrize("sequences", [3, 5, 50])
def test_offsets_that_do_not_ascend_end(sequences):
    """Sequences over one another, more blocks than there are queries for: results are anything, but of the keys, and the call ends without an error."""
    from dsv3_b200 import expanded_attention
    args = inputs([700], [900], 3)
    cu = lambda n: torch.tensor([n * (i % 2) for i in range(sequences + 1)], dtype=torch.int32, device="cuda")  # noqa: E731
    expanded_attention(*args, SCALE, cu(700), cu(900))
    want, _, bound, _ = reference(*args, [700], [900])
    check(expanded_attention(*args, SCALE, offsets([700]), offsets([900])), want, bound)


@pytest.mark.parametrize("tokens, keys, heads", [(400, 900, 4), (30, 5000, 2)])
def test_a_captured_call_follows_the_lengths(tokens, keys, heads):
    """One graph, other lengths at every replay; beside another graph and eager calls."""
    from dsv3_b200 import expanded_attention
    args = inputs([tokens], [keys], heads)
    cu_q, cu_k = offsets([tokens, 0, 0]), offsets([keys, 0, 0])
    expanded_attention(*args, SCALE, cu_q, cu_k, return_lse=True)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            graphs.append((graph, expanded_attention(*args, SCALE, cu_q, cu_k, return_lse=True)))
    for q, k in (([tokens, 0, 0], [keys, 0, 0]), ([tokens - 20, 15, 5], [keys - 600, 500, 100]), ([0, tokens - 7, 7], [0, keys - 7, 7]), ([1, 1, 1], [1, 200, 300])):
        cu_q.copy_(offsets(q)), cu_k.copy_(offsets(k))
        for graph, _ in graphs:
            graph.replay()
        eager = expanded_attention(*args, SCALE, cu_q, cu_k, return_lse=True)
        torch.cuda.synchronize()
        n, m = sum(q), sum(k)
        want, want_lse, bound, lse_bound = reference(args[0][:n], args[1][:n], args[2][:m], args[3][:m], args[4][:m], q, k)
        for out, lse in [r for _, r in graphs] + [eager]:
            check(out[:n], want, bound)
            check(lse[:n], want_lse, lse_bound)


def test_streams_and_threads():
    """Calls of several threads on streams of their own, with workspaces and without, give what they give alone."""
    from dsv3_b200 import attention_join, expanded_attention, rotary, rotary_table
    shapes = [([300, 20], [500, 20], 4), ([5], [4000], 3), ([700], [700], 2), ([64, 64], [1000, 64], 8)]
    cases = [(inputs(q, k, h, seed=i), offsets(q), offsets(k)) for i, (q, k, h) in enumerate(shapes)]
    table = rotary_table(1000, 64, factor=4.0)
    torch.cuda.synchronize()

    def work(i):
        args, cu_q, cu_k = cases[i]
        turned = rotary(args[1], table[:len(args[1])])
        out, lse = expanded_attention(args[0], turned, *args[2:], SCALE, cu_q, cu_k, return_lse=True)
        return attention_join([out, out], [lse, lse], return_lse=True)

    want = [work(i) for i in range(4)]
    torch.cuda.synchronize()
    wrong, errors = [], []

    def run(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(30):
                    got = work(i)
                    stream.synchronize()
                    if not (torch.equal(got[0], want[i][0]) and torch.equal(got[1], want[i][1])):
                        wrong.append(i)
        except BaseException as e:
            errors.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors and not wrong, (errors, wrong)


def test_calls_behind_one_another():
    """Launches that overlap the kernel before them: what a call writes the next one reads."""
    from dsv3_b200 import expanded_attention
    args = inputs([260], [260], 3)
    x = args[0].contiguous()
    for _ in range(20):
        x = expanded_attention(x, args[1], args[2], args[3], args[4], SCALE)
    torch.cuda.synchronize()
    y = args[0].contiguous()
    for _ in range(20):
        y = expanded_attention(y, args[1], args[2], args[3], args[4], SCALE)
        torch.cuda.synchronize()
    assert torch.equal(x, y)


def test_a_stream_that_is_not_the_tensors_own():
    from dsv3_b200 import expanded_attention
    args = inputs([200], [3000], 2)
    want = expanded_attention(*args, SCALE, offsets([200]), offsets([3000]))
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        got = expanded_attention(*args, SCALE, offsets([200]), offsets([3000]))
    stream.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("shape", [(0, 2), (3, 0)])
def test_empty_batches(shape):
    from dsv3_b200 import attention_join, expanded_attention, rotary
    tokens, heads = shape
    args = inputs([tokens], [5], heads)
    out, lse = expanded_attention(*args, SCALE, return_lse=True)
    assert out.shape == (tokens, heads, 128) and lse.shape == shape
    assert attention_join([out], [lse]).shape == out.shape
    assert rotary(args[1], torch.zeros(9, 32, dtype=torch.complex64, device="cuda")).shape == args[1].shape


def test_a_long_sequence_of_one_head():
    """More tiles than a part's counters would hold by accident: 200 thousand keys, one query and 300."""
    for q in (1, 300):
        args = inputs([q], [200000], 1, seed=q)
        from dsv3_b200 import expanded_attention
        out, lse = expanded_attention(*args, SCALE, offsets([q]), offsets([200000]), return_lse=True)
        want, want_lse, bound, lse_bound = reference(*args, [q], [200000])
        check(out, want, bound)
        check(lse, want_lse, lse_bound)


def test_refusals_that_need_a_gpu():
    from dsv3_b200 import attention_join, expanded_attention, rotary
    args = inputs([4], [4], 2)
    with pytest.raises(AssertionError, match="sequences"):
        expanded_attention(*args, SCALE, offsets([4]), offsets([2, 2]))
    with pytest.raises(AssertionError, match="batch"):
        expanded_attention(*args, SCALE, offsets([2, 2]))
    with pytest.raises(AssertionError, match="int32"):
        expanded_attention(*args, SCALE, offsets([4]).long(), offsets([4]))
    with pytest.raises(NotImplementedError):
        expanded_attention(args[0].half(), *args[1:], SCALE)
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError):
            expanded_attention(*args, scale)
    lse = torch.zeros(4, 2, device="cuda")
    with pytest.raises(AssertionError):
        attention_join([args[4].contiguous()], [lse[:3]])
    with pytest.raises(NotImplementedError):
        attention_join([args[4].float()], [lse])
    with pytest.raises(NotImplementedError):
        attention_join([args[4].contiguous()] * 33, [lse] * 33)
    x, f = torch.zeros(4, 3, 64, device="cuda"), torch.zeros(4, 32, dtype=torch.complex64, device="cuda")
    with pytest.raises(AssertionError, match="row"):
        rotary(x, f[:3])
    with pytest.raises(AssertionError, match="overlap"):
        rotary(x[:2], f, out=x[1:3])
    with pytest.raises(AssertionError, match="one place"):
        rotary(x, f, out=x[:, :1].expand(-1, 3, -1))
    with pytest.raises(AssertionError):
        rotary(x, f, out=torch.zeros(4, 3, 64, device="cuda", dtype=torch.bfloat16))
    with pytest.raises(AssertionError):
        rotary(x, f, positions=torch.zeros(4, dtype=torch.int32, device="cuda"))
    with pytest.raises(NotImplementedError):
        rotary(x.double(), f)
