"""Attention whose output takes the place of its queries."""
import pytest
import torch

from test_gpu_kv_cache import Pair

pytestmark = pytest.mark.gpu
WIDE = 4160  # tokens of tables that the kernel of many rows is chosen for


@pytest.mark.parametrize("counts,spare", [([1, 1], 0), ([3, 40], 0), ([200, 300], WIDE // 64),
                                          ([500, 30], 0)])
@pytest.mark.parametrize("layout", ["plain", "slice", "heads_first"])
def test_output_over_the_queries(uh, gpu, counts, spare, layout):
    p = Pair(uh, gpu, [1500, 700], heads=2, bt=64, seed=sum(counts), spare=spare)
    p.fill()
    rows = sum(counts)
    if layout == "slice":
        q = p.random(rows, 12)[:, 2:10]
    elif layout == "heads_first":
        q = p.random(8, rows).transpose(0, 1)
    else:
        q = p.random(rows, 8)
    args = (p.dev(p.lengths), p.dev(p.tables))
    want = p.cache.attend(q, *args, starts=p.starts(counts))
    assert p.cache.attend(q, *args, starts=p.starts(counts), out=q).data_ptr() == q.data_ptr()
    assert torch.equal(q, want)


def test_refused_where_the_queries_are_read_again(uh, gpu):
    """The weights that tokens receive come from a second pass over the queries
    in some calls: no call that adds them up takes its queries as output."""
    p = Pair(uh, gpu, [300], heads=2, bt=64, seed=1)
    p.fill()
    args = (p.dev([300]), p.dev(p.tables))
    for rows in (1, 300):
        q = p.random(rows, 8)
        keep = q.clone()
        with pytest.raises(uh.HipError, match="out must not be q") as e:
            p.cache.attend(q, *args, out=q, accumulate=True)
        assert e.value.status == uh.Status.INVALID_ARGUMENT
        torch.cuda.synchronize()
        assert torch.equal(q, keep)
    assert not p.cache.gather_weights(*args, 300).any()


def test_refused_with_other_strides(uh, gpu):
    p = Pair(uh, gpu, [90], heads=2, bt=64, seed=2)
    p.fill()
    buf = p.random(90, 8)
    other = buf.view(8, 90, 128).transpose(0, 1)
    with pytest.raises(uh.HipError, match="strides"):
        p.cache.attend(buf, p.dev([90]), p.dev(p.tables), out=other)
