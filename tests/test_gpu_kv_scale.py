"""The largest scales of attention."""
import pytest
import torch

from test_gpu_kv_cache import Pair

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [1, 300])
def test_scales_whose_base_2_form_overflows_are_refused(uh, gpu, rows):
    """Scores are kept in units of log2: a scale past FLT_MAX / log2(e) made
    NaN of a score of 0."""
    p = Pair(uh, gpu, [300], heads=2, bt=64, seed=1)
    p.fill()
    q = torch.zeros_like(p.random(rows, 8))
    args = (q, p.dev([300]), p.dev(p.tables))
    for scale in (2.37e38, -3.4e38):
        for call in (p.cache.attend, p.cache.attend_plan):
            with pytest.raises(uh.HipError, match="scale"):
                call(*args, scale=scale)
    want = p.cache.attend(*args, scale=1.0)               # queries of 0: the mean
    assert torch.equal(p.cache.attend(*args, scale=2.35e38), want)
