"""Values of blocks whose exponents are far apart, and blocks that a row does
not see, against the definition in 64 bits: each element of a result keeps the
documented relative error of its own values."""
import pytest
import torch

from kv_attention64 import attention64, within

pytestmark = pytest.mark.gpu
WIDE = 4160  # tokens of tables that the kernel of many rows is chosen for


def _attend(uh, cache, q, length, table, kernel, **kw):
    rows, heads, _ = q.shape
    n = torch.tensor([length], dtype=torch.int32, device=q.device)
    assert cache.attend_plan(q, n, table, scale=0.125, **kw).kernel == kernel
    lse = torch.empty((rows, heads), device=q.device)
    return cache.attend(q, n, table, scale=0.125, lse=lse, **kw), lse


def _case(uh, gpu, stds, rows, few, dim=128, bt=64, seed=0, absent=(), window=0, first=0,
          change=None):
    """A sequence with values of `stds[j]` in block j, in one head dimension of
    two alone where they are large; attention of `rows` queries of 8 heads over
    2, compared row by row."""
    g = torch.Generator(device=gpu).manual_seed(seed)
    length = len(stds) * bt
    k, v = (torch.randn((length, 2, dim), generator=g, device=gpu) for _ in range(2))
    scale = torch.tensor(stds, dtype=torch.float32, device=gpu).repeat_interleave(bt)[:, None, None]
    v = torch.where(scale.abs() > 2, v * scale * (torch.arange(dim, device=gpu) % 2 == 0), v * scale)
    if change is not None:
        change(v)
    columns = len(stds) if few else max(len(stds), -(-WIDE // bt))
    cache = uh.KvCache(len(stds) + 1, 2, dim, block_tokens=bt, track_weights=True)
    table = torch.full((1, columns), -1, dtype=torch.int32, device=gpu)
    table[0, :len(stds)] = torch.arange(1, len(stds) + 1)
    n = torch.tensor([length], dtype=torch.int32, device=gpu)
    cache.append(k.bfloat16(), v.bfloat16(), n, table)
    k, v = cache.gather(n, table, length)
    # The pool's first block, which the sequence does not own.
    other = torch.tensor([[0]], dtype=torch.int32, device=gpu)
    huge = torch.full((bt, 2, dim), 1e36, dtype=torch.bfloat16, device=gpu)
    cache.append(huge, huge, torch.tensor([bt], dtype=torch.int32, device=gpu), other)
    gone = torch.zeros(length, dtype=torch.bool, device=gpu)
    for j in absent:
        table[0, j] = -1
        gone[j * bt:(j + 1) * bt] = True
    q = torch.randn((rows, 8, dim), generator=g, device=gpu).bfloat16()
    kernel = uh.KV_KERNEL_FEW_ROWS if few else uh.KV_KERNEL_MANY_ROWS
    out, lse = _attend(uh, cache, q, length, table, kernel, window=window)
    ref, tol, rlse, ltol, _, _ = attention64(q, k, v, list(range(length - rows, length)), 0.125,
                                             window, gone)
    within(lse, rlse, ltol, "lse")
    within(out[first:], ref[first:], tol[first:], "out")


SHAPES = [(1, True), (40, True), (200, False)]


@pytest.mark.parametrize("rows,few", SHAPES)
@pytest.mark.parametrize("dim,bt", [(128, 64), (64, 32), (64, 128)])
def test_absent_blocks_leave_no_trace(uh, gpu, rows, few, dim, bt):
    """A table entry that names no block, while the pool's first one holds
    values of 2^120."""
    _case(uh, gpu, [1.0] * 9, rows, few, dim, bt, seed=1, absent=(0, 3, 7))


@pytest.mark.parametrize("rows,few", SHAPES)
@pytest.mark.parametrize("stds", [
    [1.0, 2.0 ** 60, 1.0, 1.0, 1.0, 1.0], [2.0 ** 60, 1.0, 2.0 ** -20, 1.0, 2.0 ** -14, 1.0],
    [1.0, 2.0 ** 17, 1.0, 2.0 ** 34, 1.0, 2.0 ** 51], [2.0 ** -60, 2.0 ** -30, 1.0, 2.0 ** 16,
                                                       2.0 ** 15, 2.0 ** 14],
    [1.0, 0.0, 1.0, 0.0, 2.0 ** -16, 1.0]])
def test_large_values_in_some_dimensions(uh, gpu, rows, few, stds):
    """What one block holds in some dimensions takes nothing from the others'
    dimensions, which it is zero in."""
    _case(uh, gpu, stds, rows, few, seed=2)
    _case(uh, gpu, stds, rows, few, dim=64, bt=128, seed=3)


# With a short window the kernel of many rows takes calls of 1024 tiles of 16.
WINDOWS = [(1, True), (40, True), (2100, False)]


@pytest.mark.parametrize("rows,few", WINDOWS)
@pytest.mark.parametrize("window", [70, 192])
def test_large_values_out_of_the_window(uh, gpu, rows, few, window):
    """A block of 2^60 times the others' values that some rows of a tile see
    and the next ones do not."""
    if few:
        _case(uh, gpu, [1.0, 1.0, 1.0, 2.0 ** 60, 1.0, 1.0], rows, few, seed=4, window=window)
    else:
        _case(uh, gpu, [1.0, 2.0 ** 60, 1.0, 1.0, 1.0, 1.0], rows, few, seed=4, window=window)


@pytest.mark.parametrize("rows,few", WINDOWS)
def test_large_tokens_of_a_block_that_is_seen_in_part(uh, gpu, rows, few):
    """The block's exponent is that of a token out of every row's window."""
    def change(v):
        v[128] = 2.0 ** 60

    _case(uh, gpu, [1.0] * 6, rows, few, seed=5, window=60 if rows > 1 else 200, change=change)
