"""Eviction where many tokens' weights are NaN, as after attention from a
query that holds one, against the 64-bit reference."""
import numpy as np
import pytest

from test_gpu_kv_cache import Pair, _evict

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lengths", [[500, 300, 90], [9000]])
@pytest.mark.parametrize("least", [0.01, 0.3])
@pytest.mark.parametrize("part", [0.3, 0.9])
def test_evict_more_nan_weights_than_stay(uh, gpu, lengths, least, part):
    """The last token that stays is one of NaN, and the others' weights are
    not 0."""
    p = Pair(uh, gpu, lengths, dim=64, bt=32, seed=int(100 * least + 10 * part), extra=20)
    rows = sum(lengths)
    w = (least + p.rs.random((rows, 2))).astype(np.float32)
    w[p.rs.random((rows, 2)) < part] = np.nan
    p.append(lengths, weights=w)
    _evict(p, 60, 3, 10)


def test_evict_after_a_query_of_nan(uh, gpu):
    """Every token that a NaN query saw has a weight of NaN, those after it
    have finite ones."""
    p = Pair(uh, gpu, [300], heads=2, bt=64, seed=5, extra=12)
    p.fill()
    q = p.random(40, 8)
    q[7] = float("nan")                     # at position 267
    args = (p.dev([300]), p.dev(p.tables))
    p.cache.attend(q, *args, accumulate=True)
    w = p.cache.gather_weights(*args, 300).cpu().numpy()
    assert np.isnan(w[:268]).all() and (w[268:] > 0).all()
    p.ref.append(*p.ref.gather([300], p.tables, [300])[:2], [300], p.tables, [300], w)
    _evict(p, 128, 4, 20)
