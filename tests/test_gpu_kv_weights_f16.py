"""The precision of the softmax weights in the product with the values: two
tokens of opposite values and nearly equal weights, where a row's result is
what the weights' rounding leaves."""
import pytest
import torch

from kv_attention64 import attention64, within


def _pairs(rows, heads, dim, device, seed):
    """Tokens t and t + 1 of values v and -v; scores that differ by up to 0.05."""
    g = torch.Generator(device="cpu").manual_seed(seed)
    k = torch.randn((rows + 1, 1, dim), generator=g) * 0.25
    v = torch.randn((1, 1, dim), generator=g).expand(rows + 1, 1, dim) * \
        (1 - 2 * (torch.arange(rows + 1) % 2))[:, None, None]
    q = torch.randn((rows, heads, dim), generator=g) * 0.1
    return [t.bfloat16().to(device) for t in (q, k, v)]


def _rounded(q, k, v, positions, scale, to):
    """The result with weights of a type, 2^11 for the largest of a row."""
    s = torch.stack([scale * (q[:, h].double() @ k[:, 0].double().T) for h in range(q.shape[1])], 1)
    tok = torch.arange(k.shape[0])
    pos = torch.tensor(positions)[:, None, None]
    s = torch.where((tok <= pos) & (tok > pos - 2), s, -torch.inf)
    p = torch.exp(s - s.amax(2, keepdim=True)) * 2.0 ** 11
    return (p.to(to).double() @ v[:, 0].double() / p.sum(2, keepdim=True)).bfloat16()


def test_the_bound_tells_f16_from_bf16():
    """On the CPU: weights of f16 keep the bound, those of bf16 do not."""
    q, k, v = _pairs(300, 2, 64, "cpu", 1)
    at = list(range(1, 301))
    ref, tol, _, _, _, _ = attention64(q, k, v, at, 0.125, 2)
    within(_rounded(q, k, v, at, 0.125, torch.float16), ref, tol, "f16")
    with pytest.raises(AssertionError, match="over the bound"):
        within(_rounded(q, k, v, at, 0.125, torch.bfloat16), ref, tol, "bf16")


@pytest.mark.gpu
@pytest.mark.parametrize("rows,heads,few", [(1, 8, True), (16, 4, True), (4200, 4, False)])
@pytest.mark.parametrize("dim", [64, 128])
def test_weights_enter_in_f16(uh, gpu, rows, heads, few, dim):
    for seed in range(40 if rows < 100 else 1):
        q, k, v = _pairs(rows, heads, dim, gpu, seed)
        n = torch.tensor([rows + 1], dtype=torch.int32, device=gpu)
        cache = uh.KvCache(-(-(rows + 1) // 64), 1, dim)
        table = torch.arange(cache.blocks, dtype=torch.int32, device=gpu).view(1, -1)
        cache.append(k, v, n, table)
        k, v = cache.gather(n, table, rows + 1)
        kernel = uh.KV_KERNEL_FEW_ROWS if few else uh.KV_KERNEL_MANY_ROWS
        assert cache.attend_plan(q, n, table, window=2).kernel == kernel
        out = cache.attend(q, n, table, window=2, scale=0.125)
        ref, tol, _, _, _, _ = attention64(q, k, v, list(range(1, rows + 1)), 0.125, 2)
        within(out, ref, tol, "out")
