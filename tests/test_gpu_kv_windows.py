"""Windows as long as a part of a sequence can be, which start anywhere in a
block, against the definition in 64 bits."""
import pytest
import torch

from kv_attention64 import attention64, within

pytestmark = pytest.mark.gpu


class Sequence:
    """One stored sequence, whose last tokens have the largest values, so that
    a group of tokens taken for another one shows."""

    def __init__(self, uh, gpu, length, bt, kv_heads, dim, seed, last=2048):
        g = torch.Generator(device=gpu).manual_seed(seed)
        self.gpu, self.length, self.g = gpu, length, g
        blocks = -(-length // bt)
        k, v = (torch.randn((length, kv_heads, dim), generator=g, device=gpu) for _ in range(2))
        v[-last:] *= 64
        self.cache = uh.KvCache(blocks, kv_heads, dim, block_tokens=bt, track_weights=True)
        self.table = torch.randperm(blocks, generator=g, device=gpu).int().view(1, -1)
        n = torch.tensor([length], dtype=torch.int32, device=gpu)
        self.cache.append(k.bfloat16(), v.bfloat16(), n, self.table)
        self.k, self.v = self.cache.gather(n, self.table, length)

    def queries(self, rows, heads):
        return torch.randn((rows, heads, self.k.shape[2]), generator=self.g,
                           device=self.gpu).bfloat16()


@pytest.mark.parametrize("bt,window,rows", [(64, 32683, 2048), (64, 32704, 2048),
                                            (128, 65440, 1024), (128, 65400, 2048)])
def test_window_of_many_rows_over_all_held_blocks(uh, gpu, bt, window, rows):
    """Parts of 512 blocks' tokens that touch one block more."""
    kv_heads = 8 if rows == 2048 else 16
    s = Sequence(uh, gpu, window + rows + 333, bt, kv_heads, 64, window)
    n = torch.tensor([s.length], dtype=torch.int32, device=gpu)
    q = s.queries(rows, 4 * kv_heads)
    plan = s.cache.attend_plan(q, n, s.table, window=window)
    assert plan.kernel == uh.KV_KERNEL_MANY_ROWS and plan.parts == 1
    assert 511 * bt < plan.part_tokens <= 512 * bt
    lse = torch.empty((rows, 4 * kv_heads), device=gpu)
    out = s.cache.attend(q, n, s.table, window=window, lse=lse)
    assert out.isfinite().all()
    # The first and last row of tiles that start at every place in a block.
    at = torch.tensor([32 * i + e for i in (0, 1, 2, 3, rows // 32 - 1) for e in (0, 31)],
                      device=gpu)
    ref, tol, rlse, ltol, _, _ = attention64(q[at], s.k, s.v, s.length - rows + at,
                                             64 ** -0.5, window)
    within(out[at], ref, tol, "out")
    within(lse[at], rlse, ltol, "lse")


@pytest.mark.parametrize("bt,window,dim,batch,rows", [
    (64, 4096, 128, 40, 1), (64, 8192, 128, 17, 1), (128, 8192, 64, 40, 1),
    (128, 8100, 64, 40, 1), (32, 4096, 64, 40, 1), (64, 4096, 64, 20, 4)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_window_of_few_rows_over_all_looked_up_blocks(uh, gpu, bt, window, dim, batch, rows,
                                                      accumulate):
    """Parts of 64 blocks' tokens that touch one block more: sequences that
    share one table and end at every place in a block."""
    heads, kv_heads = 32, 8
    s = Sequence(uh, gpu, window + 640, bt, kv_heads, dim, window + bt + rows, last=800)
    lengths = torch.tensor([s.length - 15 * i for i in range(batch)], dtype=torch.int32,
                           device=gpu)
    tables = s.table.expand(batch, -1).contiguous()
    q = s.queries(batch * rows, heads)
    plan = s.cache.attend_plan(q, lengths, tables, window=window, accumulate=accumulate)
    assert plan.kernel == uh.KV_KERNEL_FEW_ROWS
    lse = torch.empty((batch * rows, heads), device=gpu)
    out = s.cache.attend(q, lengths, tables, window=window, accumulate=accumulate, lse=lse)
    added, bound = 0, 0
    for b, n in enumerate(lengths.tolist()):
        at = slice(b * rows, (b + 1) * rows)
        ref, tol, rlse, ltol, p, ptol = attention64(
            q[at], s.k, s.v, list(range(n - rows, n)), dim ** -0.5, window)
        within(out[at], ref, tol, "out")
        within(lse[at], rlse, ltol, "lse")
        shape = (rows, kv_heads, heads // kv_heads, s.length)
        added = added + p.view(shape).sum((0, 2)).T
        bound = bound + ptol.view(shape).sum((0, 2)).T
    if accumulate:
        w = s.cache.gather_weights(lengths[:1], s.table, s.length)
        within(w, added, bound + batch * 2.0 ** -23 * added, "weights")
