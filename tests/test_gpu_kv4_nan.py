"""Values of NaN in the 4-bit cache's attention: the result of a row that sees one
is NaN; its log-sum and the weights that its tokens receive are of scores alone
and stay numbers, in small and in large tiles, whole and split.

Tolerances are those of RefCache4.attend."""
import numpy as np
import pytest
import torch

from test_gpu_kv4_cache import Pair
from test_gpu_kv_cache import f64
from test_gpu_kv_calls import WIDE

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")


def spoil(p, v, at):
    """NaN or an infinity in the values' (row, head) pairs of `at`, one dim of each."""
    for i, (row, head) in enumerate(at):
        v[row, head, (17 * i) % p.dim] = (NAN, INF, -INF)[i % 3]
    return v


def check(p, counts, heads, kernel, window=0, bad_rows=True):
    out, lse = p.check_attend(counts, heads, window=window, accumulate=True, kernel=kernel)
    nan = out.isnan()
    assert not lse.isnan().any()
    assert bool(nan.any()) == bad_rows and not nan.all()
    assert torch.equal(nan.any(-1), nan.all(-1))     # a value is NaN as a whole
    return out, lse


@pytest.mark.parametrize("dim,bt,group,rows,window", [
    (128, 64, 4, 150, 0), (128, 32, 1, 150, 0), (64, 128, 7, 150, 0), (64, 32, 2, 150, 0),
    (128, 64, 4, 300, 90), (64, 32, 7, 300, 1),
    (128, 64, 4, 3, 0), (128, 32, 1, 3, 90), (64, 128, 7, 3, 200), (64, 32, 2, 3, 1)])
def test_values_of_nan(uh, gpu, dim, bt, group, rows, window):
    """In chunks that rows see whole, in part and not at all; two in one chunk, at
    its first and last tokens, in several heads."""
    many, lengths = rows > 3, [310, 305]
    p = Pair(uh, gpu, lengths, heads=8, dim=dim, bt=bt, seed=window + dim + group,
             spare=WIDE // bt if many else 0)
    v = spoil(p, p.random(615, 8), [
        (310 - rows + 1, 0), (309, 0), (310 - rows, 1), (255, 2), (224, 3), (255, 3),
        (309, 4), (310 + 304, 0), (310 + 305 - rows // 2, 5), (310, 6)])
    p.append(lengths, v=v)
    kernel = uh.KV_KERNEL_MANY_ROWS if many else uh.KV_KERNEL_FEW_ROWS
    check(p, [rows, rows], 8 * group, kernel, window)
    # The bound is that of one call's additions: the reference goes on from what the
    # first call left in the cache.
    w = p.cache.gather_weights(p.dev(lengths), p.dev(p.tables), 615, starts=p.starts(lengths))
    for b, first in ((0, 0), (1, 310)):
        for t in range(lengths[b]):
            p.ref.w[p.tables[b, t // bt], :, t % bt] = f64(w[first + t])
    check(p, [rows, 1], 8 * group, None, window)


@pytest.mark.parametrize("rows", [3, 150])
def test_hidden_values_of_nan(uh, gpu, rows):
    """Past a sequence's end and in blocks out of the pool."""
    p = Pair(uh, gpu, [400], heads=8, bt=64, seed=3, spare=WIDE // 64 if rows > 3 else 0)
    p.append([400], v=spoil(p, p.random(400, 8), [(70, 1), (130, 2), (395, 3), (390, 4)]))
    p.tables[0, 1], p.tables[0, 2] = -1, p.blocks
    p.lengths = [390]
    out, lse = p.check_attend([rows], 32, accumulate=True, kernel=uh.KV_KERNEL_MANY_ROWS
                              if rows > 3 else uh.KV_KERNEL_FEW_ROWS)
    assert out.isfinite().all() and lse.isfinite().all()


@pytest.mark.parametrize("rows", [60, 300])
@pytest.mark.parametrize("at", [10, 1650, 1990])
def test_values_of_nan_in_one_part(uh, gpu, rows, at):
    """A split call: one part of a row's tokens has the NaN, the join the row."""
    p = Pair(uh, gpu, [2000], heads=1, dim=64, bt=128, seed=at, spare=WIDE // 128)
    p.append([2000], v=spoil(p, p.random(2000, 1), [(at, 0)]))
    q = p.random(rows, 14)
    plan = p.cache.attend_plan(q, p.dev([2000]), p.dev(p.tables), starts=p.starts([rows]))
    assert plan.kernel == (uh.KV_KERNEL_FEW_ROWS if rows == 60 else uh.KV_KERNEL_MANY_ROWS)
    assert plan.part_tokens < 2000
    out, lse = p.check_attend([rows], 14, q=q, accumulate=True)
    assert not lse.isnan().any()
    sees = np.arange(2000 - rows, 2000) >= at
    assert np.array_equal(out.isnan().all(-1).all(-1).cpu().numpy(), sees)
    assert np.array_equal(out.isnan().any(-1).any(-1).cpu().numpy(), sees)


def test_long_prompt_with_a_value_of_nan(uh, gpu):
    """Tiles that walk through more blocks than a workgroup holds: the log-sums and
    weights are those of finite values.  One token's part of a sum is made with
    another scale (within 2^-18 of it), and the sum rounded otherwise: 1270 additions
    after each other by 2^-24 on either side, under 2^-12 in all; of the weights'
    sums twice that."""
    n, rows, at = 40064, 12800, 40064 - 700
    g = torch.Generator(device=gpu).manual_seed(6)
    k, v = (torch.randn((n, 1, 64), generator=g, device=gpu).bfloat16() for _ in range(2))
    q = torch.randn((rows, 4, 64), generator=g, device=gpu).bfloat16()
    length = torch.tensor([n], dtype=torch.int32, device=gpu)
    c = uh.KvCache(-(-n // 32), 1, 64, block_tokens=32, track_weights=True, bits=4)
    table = torch.randperm(-(-n // 32), generator=g, device=gpu).int().view(1, -1)
    got = []
    for value in (v[at, 0, 7].item(), NAN):
        v[at, 0, 7] = value
        c.append(k, v, length, table)
        p = c.attend_plan(q, length, table)
        assert p.kernel == uh.KV_KERNEL_MANY_ROWS and p.part_tokens > 512 * 32
        lse = torch.empty((rows, 4), device=gpu)
        out = c.attend(q, length, table, lse=lse, accumulate=True)
        got.append((out, lse, c.gather_weights(length, table, n)))
    (out, lse, w), (out_nan, lse_nan, w_nan) = got
    assert out.isfinite().all() and lse_nan.isfinite().all() and w_nan.isfinite().all()
    first = rows - 700                                # the query at the token's position
    assert torch.equal(out_nan.isnan().all(-1).all(-1),
                       torch.arange(rows, device=gpu) >= first)
    assert out_nan[:first].isfinite().all()
    assert ((lse_nan - lse).abs() <= 2.0 ** -12).all()
    assert ((w_nan - w).abs() <= 2.0 ** -11 * w.abs()).all()


def test_eviction_after_values_of_nan(uh, gpu):
    """Weights that stay numbers choose the tokens that stay: those of a twin whose
    values are finite, but where two weights are within rounding."""
    p, twin = (Pair(uh, gpu, [600], heads=8, bt=64, seed=9, spare=WIDE // 64) for _ in range(2))
    k, v = p.random(600, 8), p.random(600, 8)
    twin.append([600], k=k, v=v)
    p.append([600], k=k, v=spoil(p, v.clone(), [(520, h) for h in range(8)]))
    q = p.random(200, 32)
    kept = []
    for c in (p, twin):
        lens, table = c.dev([600]), c.dev(c.tables)
        assert c.cache.attend_plan(q, lens, table, accumulate=True).kernel == \
            uh.KV_KERNEL_MANY_ROWS
        c.cache.attend(q, lens, table, accumulate=True)
        w = c.cache.gather_weights(lens, table, 600)
        assert w.isfinite().all()
        spare = c.dev(np.array(c.free[:2]))[None]
        kept.append((c.cache.evict(lens, table, spare, 100)[1], w))
    (one, w), (two, _) = kept
    for h in range(8):
        a, b = (set(x[0, h].tolist()) for x in (one, two))
        edge = w[sorted(b), h].min()
        for t in a ^ b:
            assert abs(float(w[t, h] - edge)) <= 2.0 ** -11 * float(edge)
