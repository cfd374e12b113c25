"""Attention over expanded keys and values against its definition in 64 bits."""
import math

import pytest
import torch

from expanded_util import NOPE, ROPE, SCALE, VALUE, check, inputs, offsets, reference

pytestmark = pytest.mark.gpu


def _run(args, q_counts, k_counts, causal=True, scale=SCALE):
    from dsv3_b200 import check_device_status, expanded_attention
    out, lse = expanded_attention(*args, scale, offsets(q_counts), offsets(k_counts), causal=causal, return_lse=True)
    check_device_status()
    return out, lse


def _compare(args, q_counts, k_counts, causal=True, scale=SCALE):
    out, lse = _run(args, q_counts, k_counts, causal, scale)
    want, want_lse, bound, lse_bound = reference(*args, q_counts, k_counts, causal, scale)
    check(out, want, bound)
    check(lse, want_lse, lse_bound, "lse")
    return out, lse


@pytest.mark.parametrize("queries", [1, 2, 31, 63, 64, 65, 127, 128, 129, 255, 256, 257, 383, 385, 511, 513, 700])
@pytest.mark.parametrize("before", [0, 1, 127, 300])
def test_one_prompt(queries, before):
    q, k = [queries], [before + queries]
    _compare(inputs(q, k, 3, seed=queries), q, k)


@pytest.mark.parametrize("heads", [1, 5, 16, 128])
@pytest.mark.parametrize("causal", [True, False])
def test_heads(heads, causal):
    q, k = [130, 7], [200, 150]
    _compare(inputs(q, k, heads, seed=heads), q, k, causal)


@pytest.mark.parametrize("q, k", [([300, 1, 0, 77, 513], [300, 40, 9, 77, 900]), ([1] * 33, [(7 * i) % 300 + 1 for i in range(33)]), ([0, 0, 5], [0, 3, 5]),
                                  ([256, 256, 256], [256, 512, 256]), ([3, 257, 129], [1025, 257, 130])])
@pytest.mark.parametrize("causal", [True, False])
def test_batches(q, k, causal):
    _compare(inputs(q, k, 4, seed=len(q)), q, k, causal)


@pytest.mark.parametrize("causal", [True, False])
def test_queries_that_see_nothing(causal):
    """More queries than keys: the first ones have none before them; and sequences without keys."""
    q, k = [300, 10, 200, 140], [40, 0, 199, 1]
    out, lse = _compare(inputs(q, k, 2), q, k, causal)
    if causal:
        assert not out[:260].any() and bool((lse[:260] == -math.inf).all())
    assert not out[300:310].any() and bool((lse[300:310] == -math.inf).all())


def test_no_keys_at_all():
    q, k = [5, 300], [0, 0]
    out, lse = _run(inputs(q, k, 2), q, k)
    assert not out.any() and bool((lse == -math.inf).all())


@pytest.mark.parametrize("q, k, heads", [([1], [5000], 2), ([1], [5000], 16), ([37], [4000], 4), ([1, 1, 1], [3000, 100, 2000], 3), ([200], [6000], 1), ([129], [2049], 3)])
@pytest.mark.parametrize("causal", [True, False])
def test_few_queries_over_many_keys(q, k, heads, causal):
    """The keys are cut in parts, which are joined."""
    _compare(inputs(q, k, heads, seed=k[0]), q, k, causal)


def test_more_sequences_than_lanes():
    q = [(5 * i) % 7 for i in range(1000)]
    k = [n + (11 * i) % 60 for i, n in enumerate(q)]
    _compare(inputs(q, k, 2), q, k)


def test_long_sequences_in_a_large_batch():
    q = [600 if i == 50 else 20 for i in range(70)]
    _compare(inputs(q, q, 2), q, q)


def _rising(tokens, heads, step, seed=0):
    """Keys that score higher from tile to tile, so that the running reference has to move."""
    q_nope, q_rope, k_nope, k_rope, v = (t.clone() for t in inputs([tokens], [tokens], heads, seed))
    lead = torch.randn(heads, NOPE, generator=torch.Generator(device="cuda").manual_seed(seed + 1), device="cuda")
    lead /= lead.square().mean(-1, keepdim=True).sqrt()
    q_nope += lead.bfloat16()
    k_nope += (lead * (torch.arange(tokens, device="cuda") * step)[:, None, None]).bfloat16()
    return q_nope, q_rope, k_nope, k_rope, v


@pytest.mark.parametrize("step", [0.001, 0.01, -0.01, 0.1])
def test_scores_that_rise_and_fall(step):
    _compare(_rising(900, 2, step), [900], [900])


@pytest.mark.parametrize("scale", [1e-4, 1.0, 4.0])
def test_scales(scale):
    _compare(inputs([333], [500], 2), [333], [500], True, scale)


def test_heads_in_front_and_keys_that_heads_share():
    """Layouts [heads, tokens, ...], and one head's keys for all by a stride of zero."""
    tokens, heads = 270, 3
    q_nope, q_rope, k_nope, k_rope, v = inputs([tokens], [tokens], heads)
    fronted = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q_nope, q_rope, k_nope, v)]
    _compare((fronted[0], fronted[1], fronted[2], k_rope, fronted[3]), [tokens], [tokens])
    wide = torch.zeros(tokens, 128, dtype=torch.bfloat16, device="cuda")
    wide[:, 64:] = k_rope
    _compare((q_nope, q_rope, k_nope[:, :1].expand(-1, heads, -1), wide[:, 64:], v[:, 1:2].expand(-1, heads, -1)), [tokens], [tokens])


def test_batches_in_front():
    from dsv3_b200 import expanded_attention
    b, s, t, heads = 3, 140, 200, 2
    args = inputs([s] * b, [t] * b, heads)
    want = _run(args, [s] * b, [t] * b)
    shaped = [x.reshape(b, -1, *x.shape[1:]) for x in args]
    out, lse = expanded_attention(*shaped, SCALE, return_lse=True)
    assert out.shape == (b, s, heads, VALUE) and lse.shape == (b, s, heads)
    assert torch.equal(out.flatten(0, 1), want[0]) and torch.equal(lse.flatten(0, 1), want[1])
    # one sequence without either
    one = expanded_attention(*(x[0] for x in shaped), SCALE)
    check(one, *[r for i, r in enumerate(reference(*(x[0] for x in shaped), [s], [t])) if i in (0, 2)])


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_what_lies_behind_a_sequence_does_not_matter(value):
    """Keys and values of other sequences, and of nobody, that are not finite."""
    q, k = [100, 40], [130, 70]
    args = [t.clone() for t in inputs(q, k, 2)]
    want = reference(*args, q, k)
    args = [torch.cat([t, t[:60]]) if i >= 2 else t for i, t in enumerate(args)]
    for t in args[2:]:
        t[200:] = value
    for causal in (True, False):
        out, lse = _run(args, q, k, causal)
        want = reference(*[t[:200] if i >= 2 else t for i, t in enumerate(args)], q, k, causal)
        check(out, want[0], want[2])
        check(lse, want[1], want[3])
    # the second sequence spoils itself alone
    for t in args[2:]:
        t[130:] = value
    out, _ = _run(args, q, k)
    want = reference(*[t[:130] if i >= 2 else t[:100] for i, t in enumerate(args)], q[:1], k[:1])
    check(out[:100], want[0], want[2])


@pytest.mark.parametrize("which", ["k_nope", "k_rope", "v"])
@pytest.mark.parametrize("queries, before, bad", [(300, 0, 133), (300, 0, 0), (300, 50, 349), (300, 200, 100), (60, 3, 30), (513, 0, 260)])
def test_a_key_that_is_not_finite_reaches_only_those_that_see_it(which, queries, before, bad):
    q, k = [queries], [before + queries]
    args = [t.clone() for t in inputs(q, k, 2)]
    want, _, bound, _ = reference(*args, q, k)
    t = args[["q_nope", "q_rope", "k_nope", "k_rope", "v"].index(which)]
    t[bad, ..., 5] = math.nan
    out, _ = _run(args, q, k)
    sees = torch.arange(queries, device="cuda") + before >= bad
    check(out[~sees], want[~sees], bound[~sees])
    assert bool(out[sees][..., 5].isnan().all())                     # (a key spoils all of a result, a value its own dimension at least)


def test_results_do_not_change():
    args = inputs([700, 30], [900, 2000], 8)
    first = _run(args, [700, 30], [900, 2000])
    for _ in range(5):
        again = _run(args, [700, 30], [900, 2000])
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("sms", [8, 60, 146])
def test_a_budget_of_sms_changes_nothing(sms):
    from dsv3_b200 import set_num_sms
    q, k = [700, 30, 300], [900, 30, 1300]
    args = inputs(q, k, 8)
    want = _run(args, q, k)
    set_num_sms(sms)
    try:
        got = _run(args, q, k)
    finally:
        set_num_sms(0)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])


@pytest.mark.parametrize("q, k, heads, causal", [([1700], [2600], 40, True), ([1536, 1400, 1000], [6000, 1400, 7000], 24, True), ([512, 700], [3000, 4001], 37, False), ([2100], [5000], 9, True),
                                                 ([1000], [8000], 3, True), ([1024], [1300], 1, False),
                                                 ([1000], [8000], 16, True), ([700], [5000], 33, False)])
@pytest.mark.parametrize("sms", [0, 7, 60])
def test_long_chunks_over_many_keys(q, k, heads, causal, sms):
    """What CTAs work on in pairs: several blocks to a pair, blocks of fewer queries than a pair has room for among them, and keys that are cut."""
    from dsv3_b200 import set_num_sms
    args = inputs(q, k, heads, seed=sms)
    set_num_sms(sms)
    try:
        out, lse = _run(args, q, k, causal)
    finally:
        set_num_sms(0)
    for b in range(len(q)):
        rows, keys = slice(sum(q[:b]), sum(q[:b + 1])), slice(sum(k[:b]), sum(k[:b + 1]))
        for h in range(0, heads, 4):
            part = [args[0][rows, h:h + 4], args[1][rows, h:h + 4], args[2][keys, h:h + 4], args[3][keys], args[4][keys, h:h + 4]]
            want, want_lse, bound, lse_bound = reference(*part, q[b:b + 1], k[b:b + 1], causal)
            check(out[rows, h:h + 4], want, bound)
            check(lse[rows, h:h + 4], want_lse, lse_bound, "lse")


def test_long_sequences_among_those_that_see_little():
    """Blocks of a pair, some of which have no tiles at all, or only one half of them has."""
    q, k, heads = [1500, 1500, 700, 1300, 900], [4000, 0, 6000, 100, 1700], 24
    args = inputs(q, k, heads)
    first, first_lse = _run(args, q, k)
    for b in range(len(q)):
        rows, keys = slice(sum(q[:b]), sum(q[:b + 1])), slice(sum(k[:b]), sum(k[:b + 1]))
        for h in range(0, heads, 8):
            part = [args[0][rows, h:h + 8], args[1][rows, h:h + 8], args[2][keys, h:h + 8], args[3][keys], args[4][keys, h:h + 8]]
            want, want_lse, bound, lse_bound = reference(*part, q[b:b + 1], k[b:b + 1], True)
            check(first[rows, h:h + 8], want, bound)
            check(first_lse[rows, h:h + 8], want_lse, lse_bound, "lse")
    for _ in range(20):
        out, lse = _run(args, q, k)
        assert torch.equal(out, first) and torch.equal(lse, first_lse)


@pytest.mark.parametrize("heads", [2, 24])
def test_values_that_are_not_finite_in_a_pairs_tiles(heads):
    """Either CTA of a pair looks at half of the values' dimensions; what one finds both know."""
    q, k = [1536], [6000]
    for column in (5, 100):
        for bad in (4600, 5990):
            args = [t.clone() for t in inputs(q, k, heads)]
            args[4][bad, 1, column] = math.inf
            out, _ = _run(args, q, k)
            sees = torch.arange(1536, device="cuda") + 6000 - 1536 >= bad
            assert bool(out[:, 0].isfinite().all()) and bool(out[~sees].isfinite().all()) and not out[sees][:, 1, column].isfinite().any()


def test_offsets_beyond_32_bits():
    """Keys whose last sequence begins more than 2^31 values, and 2^32 bytes, behind the first."""
    heads, tokens = 128, 70000
    kv = torch.zeros(tokens, heads, NOPE + VALUE, dtype=torch.bfloat16, device="cuda")
    k_rope = torch.zeros(tokens, ROPE, dtype=torch.bfloat16, device="cuda")
    q, k = [2, 40], [tokens - 150, 150]
    small = inputs([42], [150], heads)
    kv[-150:, :, :NOPE], kv[-150:, :, NOPE:], k_rope[-150:] = small[2], small[4], small[3]
    out, _ = _run((small[0], small[1], kv[..., :NOPE], k_rope, kv[..., NOPE:]), q, k)
    assert not out[:2].any()
    want = reference(small[0][2:], small[1][2:], *small[2:], [40], [150])
    check(out[2:], want[0], want[2])
