"""The oracle's greedy rows of nothing but -inf, as masks and bans leave them: no draw. An argmax has an id for them."""
import numpy as np

import oracle


def test_greedy_rows_of_nothing():
    x = np.full(100, -np.inf, dtype=np.float32)
    for p in (dict(temperature=0.0), dict(temperature=1.0, top_k=1)):
        assert oracle.sample(x, oracle.params(**p), 0.5).status == oracle.ERR_NONFINITE
        y = x.copy()
        y[40] = -7.0
        drawn = oracle.sample(y, oracle.params(**p), 0.5)
        assert drawn.status == oracle.OK and drawn.token == 40
        drawn = oracle.sample(np.full(100, np.nan, dtype=np.float32), oracle.params(**p), 0.5)
        assert drawn.status == oracle.OK and drawn.token == 0
    assert oracle.argmax(x) == 0
