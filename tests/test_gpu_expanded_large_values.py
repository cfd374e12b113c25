"""Expanded attention of values near the largest that its fp32 sums hold: finite inputs, finite results."""
import pytest
import torch

from expanded_util import check, reference
from test_gpu_expanded_attention import _rising, _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("queries, keys, heads", [(900, 900, 2), (60, 900, 2), (1, 4000, 2), (1100, 2000, 24)])
@pytest.mark.parametrize("rise", [0, 4, 8, 15, 20, -15])
def test_scores_that_rise_over_large_values(queries, keys, heads, rise):
    """Scores rise by `rise` (in e-folds) from the first key to the last: the running reference lags behind by up to 2^8, and what it lags by the sums are larger.  One CTA's blocks of two halves and of
    one, keys that are cut, and blocks of a pair."""
    args = [t.clone() for t in _rising(keys, heads, rise / keys / (128 * 192 ** -0.5), seed=rise)]
    args[0], args[1] = args[0][-queries:], args[1][-queries:]
    args[4] = args[4].clamp(-4, 4) * 2.0 ** 105
    assert float(args[4].abs().max()) <= 2.0 ** 119 / keys
    out, lse = _run(args, [queries], [keys])
    for h in range(0, heads, 4):
        part = [args[0][:, h:h + 4], args[1][:, h:h + 4], args[2][:, h:h + 4], args[3], args[4][:, h:h + 4]]
        want, want_lse, bound, lse_bound = reference(*part, [queries], [keys])
        check(out[:, h:h + 4], want, bound)
        check(lse[:, h:h + 4], want_lse, lse_bound, "lse")
