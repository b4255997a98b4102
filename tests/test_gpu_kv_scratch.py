"""Received weights of calls whose tables are far wider than their sequences."""
import pytest
import torch

from kv_attention64 import attention64, within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("batch,columns", [(256, 2048), (4, 2048)])
def test_scratch_of_wide_tables_is_bounded(uh, gpu, batch, columns):
    """Stored scores would take 4.3 GB for tables of 131072 tokens, whatever
    the sequences hold."""
    n, heads, dim = 150, 32, 64
    g = torch.Generator(device=gpu).manual_seed(batch)
    cache = uh.KvCache(4, 8, dim, track_weights=True)
    table = torch.full((1, columns), -1, dtype=torch.int32, device=gpu)
    table[0, :3] = torch.tensor([2, 0, 3])
    length = torch.tensor([n], dtype=torch.int32, device=gpu)
    k, v = (torch.randn((n, 8, dim), generator=g, device=gpu).bfloat16() for _ in range(2))
    cache.append(k, v, length, table)
    k, v = cache.gather(length, table, n)
    # All sequences share the blocks and end at places of their own.
    lengths = torch.tensor([n - b % 9 for b in range(batch)], dtype=torch.int32, device=gpu)
    tables = table.expand(batch, -1).contiguous()
    q = torch.randn((batch, heads, dim), generator=g, device=gpu).bfloat16()
    plan = cache.attend_plan(q, lengths, tables, accumulate=True)
    assert plan.workspace_bytes <= 2 ** 31 + 2 ** 28
    out = cache.attend(q, lengths, tables, accumulate=True)
    ref, tol, _, _, p, ptol = attention64(q, k, v, [m - 1 for m in lengths.tolist()], dim ** -0.5)
    within(out, ref, tol, "out")
    shape = (batch, 8, heads // 8, n)
    added, bound = (x.view(shape).sum((0, 2)).T for x in (p, ptol))
    w = cache.gather_weights(length, table, n)
    within(w, added, bound + batch * 2.0 ** -23 * added, "weights")
