"""Expanded attention with keys whose scores are infinite, against the definition in 64 bits: a score of -inf weighs nothing, one of +inf makes the query's results NaN."""
import math

import pytest
import torch

from expanded_util import check, inputs, reference
from test_gpu_expanded_attention import _run

pytestmark = pytest.mark.gpu

SHAPES = [(300, 350, 2), (300, 300, 2), (60, 900, 2), (5, 4000, 3), (1100, 2000, 24)]      # two halves, a first query that sees one key, one half, cut keys, pairs


def _compare(out, lse, args, queries, keys, causal, rows):
    for h in range(0, out.shape[1], 4):
        part = [args[0][:, h:h + 4], args[1][:, h:h + 4], args[2][:, h:h + 4], args[3], args[4][:, h:h + 4]]
        want, want_lse, bound, lse_bound = reference(*part, [queries], [keys], causal)
        here = rows[:, h:h + 4]
        check(out[:, h:h + 4][here], want[here], bound[here])
        check(lse[:, h:h + 4][here], want_lse[here], lse_bound[here], "lse")


@pytest.mark.parametrize("queries, keys, heads", SHAPES)
@pytest.mark.parametrize("which", ["k_nope", "k_rope"])
@pytest.mark.parametrize("value", [math.inf, -math.inf])
@pytest.mark.parametrize("causal", [True, False])
def test_a_key_of_infinite_scores(queries, keys, heads, which, value, causal):
    """The first key (without it a causal query sees as many as before less one): queries whose score it makes +inf are NaN, others are as if it were not there."""
    args = [t.clone() for t in inputs([queries], [keys], heads, seed=queries)]
    t = args[2] if which == "k_nope" else args[3]
    t[0, ..., 5] = value
    out, lse = _run(args, [queries], [keys], causal)
    score = (args[0] if which == "k_nope" else args[1])[..., 5].double() * value
    assert bool((score == math.inf).any()) and bool((score == -math.inf).any()) and not score.isnan().any()
    spoilt = score == math.inf
    if causal and keys == queries:                          # (the first query sees this key alone)
        assert bool((spoilt | (score == -math.inf)).all())
    assert bool(out[spoilt].isnan().all()) and bool(lse[spoilt].isnan().all())
    _compare(out, lse, [x[1:] if i >= 2 else x for i, x in enumerate(args)], queries, keys - 1, causal, ~spoilt)


@pytest.mark.parametrize("queries, keys, heads", SHAPES)
def test_queries_all_of_whose_scores_are_minus_infinity(queries, keys, heads):
    """As if they saw nothing."""
    args = [t.clone() for t in inputs([queries], [keys], heads)]
    args[2][..., 7] = -math.inf
    out, lse = _run(args, [queries], [keys])
    nothing = args[0][..., 7] > 0
    assert not out[nothing].any() and bool((lse[nothing] == -math.inf).all())
    assert bool(out[~nothing].isnan().all()) and bool(lse[~nothing].isnan().all())


def test_a_key_that_is_not_a_number_or_both_infinities():
    args = [t.clone() for t in inputs([300], [350], 2)]
    args[2][0, :, 5], args[2][0, :, 6] = math.inf, -math.inf
    out, _ = _run(args, [300], [350])
    both = (args[0][..., 5] > 0) == (args[0][..., 6] > 0)   # inf - inf
    plus = (args[0][..., 5] > 0) & (args[0][..., 6] < 0)
    assert bool(out[both | plus].isnan().all()) and bool(out[~(both | plus)].isfinite().all())
