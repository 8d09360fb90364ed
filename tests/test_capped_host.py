"""CPU: the bound of capped rows rejects results of wrong scores."""
import numpy as np
import pytest

from capped_common import capped_rows, telling_values

CASES = [  # cap, scale, the queries' size
    (0.003, 128 ** -0.5, 6.0), (0.003, 128 ** -0.5, 1500.0), (0.003, 128 ** -0.5, 0.01),
    (0.125, 4.0, 0.003), (0.125, 4.0, 1500.0), (1.0, 4.0, 0.02), (1.0, 4.0, 6.0), (0.125, 128 ** -0.5, 0.2),
]
WRONG = {"zero": lambda s: 0 * s, "negated": lambda s: -s, "other_rows": lambda s: np.roll(s, 1, 0),
         "other_keys": lambda s: np.roll(s, 1, 1)}


@pytest.mark.parametrize("keys", [33, 257, 900])
@pytest.mark.parametrize("cap,scale,spread", CASES)
def test_wrong_scores_are_rejected(cap, scale, spread, keys):
    rng = np.random.default_rng(keys)
    q, K = rng.standard_normal((5, 128)) * spread, rng.standard_normal((keys, 128))
    V = telling_values(q, K, scale, cap, rng)
    seen = np.ones((5, keys), bool)
    out, bound = capped_rows(q, K, V, scale, cap, seen)
    for name, f in WRONG.items():
        bad, _ = capped_rows(q, K, V, scale, cap, seen, wrong=f)
        assert (np.abs(bad - out) > bound).any(1).all(), name  # in every row
    if np.abs(q @ K.T * scale).mean() < 2 * cap and cap > 0.1:  # a factor off shows where the cap does not flatten
        bad, _ = capped_rows(q, K, V, scale, cap, seen, wrong=lambda s: s / 2)
        assert (np.abs(bad - out) > bound).any(1).all()
