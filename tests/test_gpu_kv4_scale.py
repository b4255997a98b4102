"""The scale of the 4-bit cache's scores at the end of its range, and scores so
large that their rounding shows.  Tolerances are those of RefCache4.attend."""
import numpy as np
import pytest
import torch

from kv_attention64 import within
from test_gpu_kv4_cache import Pair
from test_gpu_kv4_calls import calls  # noqa: F401  (a fixture)
from test_gpu_kv_cache import f64
from test_gpu_kv_calls import WIDE

pytestmark = pytest.mark.gpu

END = 2.0 ** 100 / 1.4426950408889634     # scale * log2(e) = 2^100


@pytest.mark.parametrize("name", ["attend", "attend_plan"])
def test_the_end_of_the_scale(calls, name):  # noqa: F811
    """2^-22 to either side, four steps of f32; the refusal names the bound."""
    for sign in (1, -1):
        assert calls.call(name, scale=sign * END * (1 - 2.0 ** -22))[0] == "OK"
        st, text = calls.call(name, scale=sign * END * (1 + 2.0 ** -22))
        assert st == "INVALID_ARGUMENT" and "scale" in text and "2^100" in text
    torch.cuda.synchronize()


@pytest.mark.parametrize("rows", [2, 200])
def test_scores_of_zero_at_the_end_of_the_scale(uh, gpu, rows):
    p = Pair(uh, gpu, [300], heads=8, bt=64, seed=31, spare=WIDE // 64)
    size = torch.exp2(torch.randint(-6, 7, (300, 1, 1), device=gpu).float())
    p.append([300], v=(p.random(300, 8).float() * size).bfloat16())
    for scale in (END * (1 - 2.0 ** -22), -END * (1 - 2.0 ** -22)):
        p.check_attend([rows], 32, q=torch.zeros_like(p.random(rows, 32)), scale=scale,
                       kernel=uh.KV_KERNEL_FEW_ROWS if rows == 2 else uh.KV_KERNEL_MANY_ROWS)


@pytest.mark.parametrize("rows", [2, 200])
@pytest.mark.parametrize("scale", [0.1, 1.0, 20.0, -20.0])
def test_equal_keys_of_large_scores(uh, gpu, rows, scale):
    """Sixty tokens share each key and have values of scales 2^20 apart: their
    weights are equal but for the rounding of a score, to which large tiles add log2
    of the value's scale."""
    p = Pair(uh, gpu, [300], heads=8, bt=64, seed=32, spare=WIDE // 64)
    k = p.random(5, 8, 8.0).repeat(60, 1, 1)
    size = torch.exp2(torch.randint(-10, 11, (300, 1, 1), device=gpu).float())
    p.append([300], k=k, v=(p.random(300, 8).float() * size).bfloat16())
    q = p.random(rows, 32, 8.0)
    p.check_attend([rows], 32, q=q, scale=scale,
                   kernel=uh.KV_KERNEL_FEW_ROWS if rows == 2 else uh.KV_KERNEL_MANY_ROWS)
    # The weights that the tokens receive, some far below what f32 holds: a power under
    # 2^-126 counts as 0, in each of the 800 rows of a head at most.
    lens, table = p.dev([300]), p.dev(p.tables)
    p.cache.attend(q, lens, table, scale=scale, accumulate=True)
    tol = p.ref.attend(f64(q), [300], p.tables, [rows], scale, 0, True)[4]
    got = p.cache.gather_weights(lens, table, 300)
    slots = [(p.tables[0, t // 64], slice(None), t % 64) for t in range(300)]
    want, tol = (torch.tensor(np.array([x[at] for at in slots])) for x in (p.ref.w, tol))
    within(got.cpu(), want, tol + 800 * 2.0 ** -126, "weights")
