"""The scale of the 4-bit cache's scores at the end of its range."""
import pytest
import torch

from test_gpu_kv4_cache import Pair
from test_gpu_kv4_calls import calls  # noqa: F401  (a fixture)
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
