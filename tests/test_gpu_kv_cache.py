"""GPU parity of the 8-bit key/value cache (append, gather, attend, evict)
through the Python mirror, against the 64-bit reference of kv_reference.py.

Stored values are compared bit for bit.  Attention is compared within a bound
that the reference computes for each element from the documented arithmetic
(RefCache.attend), fixed before any run."""
import numpy as np
import pytest
import torch

from kv_reference import RefCache

pytestmark = pytest.mark.gpu


def f64(t):
    return t.detach().float().cpu().numpy().astype(np.float64)


def same(a, b):
    return np.array_equal(np.nan_to_num(a, nan=1e300), np.nan_to_num(b, nan=1e300))


class Pair:
    """A cache and its reference, with tables over shuffled blocks."""

    def __init__(self, uh, gpu, lengths, heads=2, dim=128, bt=64, seed=0, extra=4, spare=0):
        self.uh, self.gpu, self.bt, self.dim, self.heads = uh, gpu, bt, dim, heads
        self.rs = np.random.default_rng(seed)
        need = [-(-int(n) // bt) for n in lengths]
        self.columns = max(1, max(need)) + spare
        self.blocks = sum(need) + extra
        self.free = list(self.rs.permutation(self.blocks))
        # Columns past a sequence's blocks name no block.
        self.tables = np.full((len(lengths), self.columns), -1, np.int32)
        for b, n in enumerate(need):
            self.tables[b, :n] = [self.free.pop() for _ in range(n)]
        self.lengths = list(lengths)
        self.cache = uh.KvCache(self.blocks, heads, dim, block_tokens=bt, track_weights=True)
        self.ref = RefCache(self.blocks, heads, dim, bt)

    def dev(self, a, dtype=torch.int32):
        return torch.tensor(np.asarray(a), dtype=dtype, device=self.gpu)

    def random(self, rows, heads, std=1.0):
        x = self.rs.standard_normal((rows, heads, self.dim)) * std
        return torch.tensor(x, dtype=torch.float32, device=self.gpu).bfloat16()

    def starts(self, counts):
        return self.dev(np.concatenate([[0], np.cumsum(counts)]))

    def append(self, counts, lengths=None, k=None, v=None, weights=None):
        lengths = self.lengths if lengths is None else lengths
        rows = int(sum(counts))
        k = self.random(rows, self.heads) if k is None else k
        v = self.random(rows, self.heads) if v is None else v
        self.cache.append(k, v, self.dev(lengths), self.dev(self.tables),
                          starts=self.starts(counts),
                          weights=None if weights is None else self.dev(weights, torch.float32))
        self.ref.append(f64(k), f64(v), lengths, self.tables, counts, weights)
        return k, v

    def fill(self, weights=False):
        rows = int(sum(self.lengths))
        w = np.exp(self.rs.standard_normal((rows, self.heads))).astype(np.float32) \
            if weights else None
        return self.append(self.lengths, weights=w)

    def check_stored(self, tables=None, lengths=None):
        tables = self.tables if tables is None else tables
        lengths = self.lengths if lengths is None else lengths
        counts = [max(int(n), 0) for n in lengths]
        k, v = self.cache.gather(self.dev(lengths), self.dev(tables), sum(counts),
                                 starts=self.starts(counts))
        w = self.cache.gather_weights(self.dev(lengths), self.dev(tables), sum(counts),
                                      starts=self.starts(counts))
        rk, rv, rw = self.ref.gather(lengths, tables, counts)
        assert same(f64(k), rk) and same(f64(v), rv)
        return f64(w), rw

    def check_attend(self, counts, heads, q=None, scale=None, window=0, accumulate=False,
                     lengths=None, starts=True, kernel=None, out=None):
        lengths = self.lengths if lengths is None else lengths
        rows = int(sum(counts))
        q = self.random(rows, heads) if q is None else q
        lse = torch.full((rows, heads), 7.0, device=self.gpu)
        args = (q, self.dev(lengths), self.dev(self.tables))
        kw = dict(starts=self.starts(counts) if starts else None, scale=scale, window=window,
                  accumulate=accumulate)
        if kernel is not None:
            assert self.cache.attend_plan(*args, **kw).kernel == kernel
        got = self.cache.attend(*args, lse=lse, out=out, **kw)
        ref, tol, rlse, ltol, wtol = self.ref.attend(
            f64(q), lengths, self.tables, counts,
            self.dim ** -0.5 if scale is None else scale, window, accumulate)
        compare(f64(got), ref, tol, "out")
        compare(f64(lse), rlse, ltol, "lse")
        if accumulate:
            counts = [int(n) for n in lengths]
            w = self.cache.gather_weights(self.dev(lengths), self.dev(self.tables), sum(counts),
                                          starts=self.starts(counts))
            rw = self.ref.gather(lengths, self.tables, counts)[2]
            keep = self.ref.w
            self.ref.w = wtol
            tol = self.ref.gather(lengths, self.tables, counts)[2]
            self.ref.w = keep
            compare(f64(w), rw, tol, "weights")
        return got, lse


def compare(got, ref, tol, what):
    fine = np.isfinite(ref)
    assert np.array_equal(np.isnan(got), np.isnan(ref)), what
    assert np.array_equal(got[~fine & ~np.isnan(ref)], ref[~fine & ~np.isnan(ref)]), what
    over = np.abs(got[fine] - ref[fine]) - tol[fine]
    worst = float(over.max()) if over.size else 0.0
    assert worst <= 0, f"{what}: over the bound"


# ------------------------------------------------------------------- storing

@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("bt", [32, 64, 128])
def test_append_prompts_and_single_tokens(uh, gpu, dim, bt):
    p = Pair(uh, gpu, [0, 1, 31, 33, 64, 97, 129], dim=dim, bt=bt, seed=bt + dim, spare=1)
    p.fill()
    p.check_stored()
    # Single tokens until every kind of place in a block was written, the
    # sequence that was empty among them.
    grown = [n + 3 for n in p.lengths]
    for b, n in enumerate(grown):
        for j in range(-(-n // bt)):
            if p.tables[b, j] < 0 and p.free:
                p.tables[b, j] = p.free.pop()
    for step in range(1, 4):
        lengths = [n + step for n in p.lengths]
        p.append([1] * len(lengths), lengths)
    p.lengths = grown
    p.check_stored()


def test_append_raises_exponents_of_begun_blocks(uh, gpu):
    p = Pair(uh, gpu, [40, 40], bt=64, seed=1)
    small = p.random(20, 2, 2.0 ** -9)
    p.append([10, 10], [10, 10], k=small, v=small)
    # Larger tokens move the earlier ones towards and below the subnormals.
    for step, std in enumerate((1.0, 37.0, 2.0 ** 13)):
        x = p.random(20, 2, std)
        p.append([10, 10], [20 + 10 * step] * 2, k=x, v=-x)
        p.check_stored(lengths=[20 + 10 * step] * 2)


def test_append_starts_a_reused_block_anew(uh, gpu):
    p = Pair(uh, gpu, [70], bt=64, seed=2)
    big = p.random(70, 2, 1e20)
    p.append([70], k=big, v=big)
    p.fill()          # over the same blocks: the old exponents must not stay
    p.check_stored()
    x = p.random(40, 2, 1e-3)
    p.append([40], [104 - 64 + 30], k=x, v=x)   # positions 30 .. 69, exponents of block 0 stay
    p.check_stored()


def test_append_extremes(uh, gpu):
    p = Pair(uh, gpu, [64, 64, 64, 64], bt=64, seed=3)
    x = p.random(256, 2)
    y = p.random(256, 2)
    x[3, 0, 5], x[4, 1, 6], x[5, 0, 7] = float("inf"), float("-inf"), float("nan")
    y[9, 0, 0] = float("nan")
    x[64:128] = 3.38e38 * torch.sign(x[64:128].float())   # the top of bf16: saturates
    y[64:128] = 0
    x[128:192] = (x[128:192].float() * 1e-38).bfloat16()  # the bottom: flushed
    x[192, 0, 0] = 3.38e38                                # the rest becomes zero
    x[200:, 1] = float("nan")                             # no finite element in the rows
    p.append([64] * 4, k=x, v=y)
    p.check_stored()
    z = p.random(4, 2)
    p.append([1] * 4, k=z, v=z)                           # rewrites the last token
    p.check_stored()


@pytest.mark.parametrize("layout", ["slice", "heads_first", "odd"])
def test_append_strides(uh, gpu, layout):
    p = Pair(uh, gpu, [37, 90], heads=3, dim=64, bt=32, seed=4)
    rows = 127
    if layout == "slice":       # columns of a wider projection output
        buf = p.random(rows, 12)
        k, v = buf[:, 4:7], buf[:, 8:11]
    elif layout == "heads_first":
        k = p.random(rows, 3).transpose(0, 1).contiguous().transpose(0, 1)
        v = p.random(rows, 3).transpose(0, 1).contiguous().transpose(0, 1)
    else:                       # rows on odd addresses
        flat = p.random(rows + 1, 3).reshape(-1)
        k = torch.as_strided(flat, (rows, 3, 64), (193, 64, 1), 1)[:100]
        k = torch.cat([k, k[:27]]).reshape(-1)
        odd = torch.empty(rows * 193 + 1, dtype=torch.bfloat16, device=gpu)
        v = torch.as_strided(odd, (rows, 3, 64), (193, 64, 1), 1)
        v.copy_(k.view(rows, 3, 64))
        k = v
    p.append(p.lengths, k=k, v=v)
    p.check_stored()


def test_rows_without_a_place(uh, gpu):
    """Negative positions, blocks out of the pool, lengths past the table and
    starts out of range: nothing is written out of place."""
    p = Pair(uh, gpu, [5, 100, 64], bt=32, seed=5)
    p.tables[1, 1] = -1
    p.tables[1, 2] = p.blocks
    p.append([9, 100, 64], [5, 100, 64])       # 4 rows of the first are before it
    p.check_stored()
    p.append([2, 2, 2], [5, 100, 10 ** 6])     # the last is taken as the table's end
    p.check_stored(lengths=[5, 100, 128])
    k = p.random(10, 2)
    bad = p.dev([-7, 4, 2, 400])               # sequences: 0..3, none, 2..9
    p.cache.append(k, k, p.dev([5, 100, 64]), p.dev(p.tables), starts=bad)
    kk = f64(k)
    p.ref.append(kk[:4], kk[:4], [5], p.tables[:1], [4])
    p.ref.append(kk[2:], kk[2:], [64], p.tables[2:], [8])
    p.check_stored()


def test_gather_and_append_restore_a_sequence(uh, gpu):
    p = Pair(uh, gpu, [150, 77], bt=64, seed=6, extra=8)
    p.fill(weights=True)
    counts = [150, 77]
    args = (p.dev(p.lengths), p.dev(p.tables), 227)
    k, v = p.cache.gather(*args, starts=p.starts(counts))
    w = p.cache.gather_weights(*args, starts=p.starts(counts))
    other = p.tables.copy()
    for b in range(2):
        for j in range(-(-counts[b] // 64)):
            other[b, j] = p.free.pop()
    p.cache.append(k, v, p.dev(p.lengths), p.dev(other), starts=p.starts(counts), weights=w)
    k2, v2 = p.cache.gather(p.dev(p.lengths), p.dev(other), 227, starts=p.starts(counts))
    w2 = p.cache.gather_weights(p.dev(p.lengths), p.dev(other), 227, starts=p.starts(counts))
    assert torch.equal(k, k2) and torch.equal(v, v2) and torch.equal(w, w2)
    rw = p.ref.gather(p.lengths, p.tables, counts)[2]
    assert np.array_equal(f64(w), rw)


# ----------------------------------------------------------------- attention

LENGTHS = [1, 2, 31, 32, 33, 64, 65, 200, 0]


@pytest.mark.parametrize("dim,bt,heads,kv_heads", [(128, 64, 8, 2), (128, 32, 2, 2), (64, 32, 7, 1),
                                                   (64, 128, 40, 2), (128, 128, 19, 1)])
@pytest.mark.parametrize("window", [0, 1, 40])
def test_decode(uh, gpu, dim, bt, heads, kv_heads, window):
    p = Pair(uh, gpu, LENGTHS, heads=kv_heads, dim=dim, bt=bt, seed=heads + window)
    p.fill()
    p.check_attend([1] * len(LENGTHS), heads, window=window, starts=False)


@pytest.mark.parametrize("dim,heads,kv_heads", [(128, 8, 2), (64, 7, 1), (128, 4, 4)])
@pytest.mark.parametrize("window", [0, 17])
@pytest.mark.parametrize("accumulate", [False, True])
def test_ragged_rows(uh, gpu, dim, heads, kv_heads, window, accumulate):
    lengths = [1, 5, 64, 130, 0, 77, 33]
    p = Pair(uh, gpu, lengths, heads=kv_heads, dim=dim, bt=32, seed=window + heads)
    p.fill(weights=True)
    # More rows than tokens, none, all and some of them.
    p.check_attend([3, 5, 0, 9, 2, 77, 20], heads, window=window, accumulate=accumulate)


@pytest.mark.parametrize("length,rows", [(700, 700), (1500, 130), (333, 64)])
@pytest.mark.parametrize("dim,heads,kv_heads", [(128, 8, 2), (64, 14, 2)])
@pytest.mark.parametrize("window", [0, 100])
def test_prompts_and_chunks(uh, gpu, length, rows, dim, heads, kv_heads, window):
    p = Pair(uh, gpu, [length, 65], heads=kv_heads, dim=dim, bt=64, seed=length + dim)
    p.fill(weights=True)
    p.check_attend([rows, 65], heads, window=window, accumulate=window == 0)


def test_long_single_rows(uh, gpu):
    p = Pair(uh, gpu, [5000, 4097, 1, 2048], heads=2, bt=64, seed=9)
    p.fill(weights=True)
    p.check_attend([1] * 4, 8, starts=False, accumulate=True)
    p.check_attend([1] * 4, 8, starts=False, window=3000)


def test_large_scores_and_scales(uh, gpu):
    p = Pair(uh, gpu, [90, 300], heads=2, bt=64, seed=10)
    k = p.random(390, 2, 8.0)
    p.append(p.lengths, k=k)
    q = p.random(2, 4, 8.0)
    p.check_attend([1, 1], 4, q=q)                       # one weight near 1
    p.check_attend([1, 1], 4, scale=0.0)                 # the mean
    p.check_attend([1, 1], 4, scale=-0.05)
    q[0] = 0
    q[1, 0, 5:] *= 2.0 ** -20                            # elements far below the largest
    p.check_attend([1, 1], 4, q=q)


def test_values_of_very_different_blocks(uh, gpu):
    p = Pair(uh, gpu, [256], heads=1, bt=64, seed=11)
    v = p.random(256, 1)
    for i, std in enumerate((2.0 ** -30, 1.0, 2.0 ** 25, 0.0)):
        v[64 * i:64 * i + 64] = (v[64 * i:64 * i + 64].float() * std).bfloat16()
    p.append([256], v=v)
    p.check_attend([1], 2)
    p.check_attend([200], 2)


@pytest.mark.parametrize("rows", [1, 100])
def test_nan_and_infinity_stay_with_the_rows_that_see_them(uh, gpu, rows):
    lengths = [150, 130]
    p = Pair(uh, gpu, lengths, heads=1, bt=64, seed=12)
    k, v = p.random(280, 1), p.random(280, 1)
    k[100, 0, 3] = float("nan")        # hidden from the first queries of the chunk
    v[120, 0, 7] = float("inf")
    v[149, 0, 9] = float("nan")
    p.append(lengths, k=k, v=v)
    p.check_attend([rows, rows], 4)
    p.check_attend([rows, rows], 4, window=20)
    q = p.random(2 * rows, 4)
    q[0, 1, 0], q[rows, 2, 1] = float("inf"), float("nan")
    p.check_attend([rows, rows], 4, q=q, accumulate=False)


def test_stale_tokens_are_not_seen(uh, gpu):
    """Blocks hold NaN past the sequence's end, from what they held before."""
    p = Pair(uh, gpu, [128, 128], heads=1, bt=64, seed=13)
    bad = torch.full((256, 1, 128), float("nan"), dtype=torch.bfloat16, device=gpu)
    p.append([128, 128], k=bad, v=bad)
    p.append([70, 1], [70, 1])
    p.check_attend([1, 1], 4, lengths=[70, 1])
    p.check_attend([40, 1], 4, lengths=[70, 1], accumulate=True)


def test_blocks_out_of_the_pool_are_not_seen(uh, gpu):
    p = Pair(uh, gpu, [200, 64], heads=1, bt=64, seed=14)
    p.fill(weights=True)
    p.tables[0, 1], p.tables[1, 0] = -1, p.blocks
    p.check_attend([1, 1], 4, accumulate=True)
    p.check_attend([150, 64], 4)
    p.check_attend([1, 1], 4, lengths=[10 ** 6, 64])     # taken as the table's end


@pytest.mark.parametrize("rows", [3, 150])
def test_query_and_output_strides(uh, gpu, rows):
    p = Pair(uh, gpu, [160, 170], heads=2, bt=64, seed=15)
    p.fill()
    wide = p.random(2 * rows, 12)
    out = torch.zeros((2 * rows, 12, 128), dtype=torch.bfloat16, device=gpu)
    p.check_attend([rows, rows], 4, q=wide[:, 3:7], out=out[:, 5:9])
    assert not out[:, :5].any() and not out[:, 9:].any()
    by_head = torch.zeros((4, 2 * rows, 128), dtype=torch.bfloat16, device=gpu)
    p.check_attend([rows, rows], 4, q=p.random(4, 2 * rows).transpose(0, 1),
                   out=by_head.transpose(0, 1))
    odd = torch.zeros(2 * rows * 4 * 128 + 1, dtype=torch.bfloat16, device=gpu)[1:]
    q = odd.view(2 * rows, 4, 128)
    q.copy_(p.random(2 * rows, 4))
    o = torch.zeros_like(torch.empty(2 * rows * 4 * 128 + 1, dtype=torch.bfloat16, device=gpu))
    p.check_attend([rows, rows], 4, q=q, out=o[1:].view(2 * rows, 4, 128))
    assert o[0] == 0


def test_offsets_past_32_bits(uh, gpu):
    """A pool of 9 GiB, with the sequence in its last blocks."""
    blocks = 9 * 2 ** 30 // (8 * 2 * 128 * 128)
    cache = uh.KvCache(blocks, 8, 128, block_tokens=128, track_weights=True)
    assert cache.info().device_bytes > 9 * 2 ** 30
    ids = [blocks - 1, 3, blocks - 2, blocks // 2 + 1]
    p = Pair(uh, gpu, [500], heads=8, bt=128, seed=16, extra=0)
    p.fill(weights=True)
    table = torch.tensor([ids], dtype=torch.int32, device=gpu)
    lens = p.dev([500])
    k, v = p.cache.gather(lens, p.dev(p.tables), 500)
    w = p.cache.gather_weights(lens, p.dev(p.tables), 500)
    cache.append(k, v, lens, table, weights=w)
    for rows in (1, 300):
        q = p.random(rows, 32)
        assert torch.equal(cache.attend(q, lens, table, accumulate=True),
                           p.cache.attend(q, lens, p.dev(p.tables), accumulate=True))
    got = cache.gather_weights(lens, table, 500)
    assert torch.equal(got, p.cache.gather_weights(lens, p.dev(p.tables), 500))
    new = torch.tensor([[blocks - 3, 1]], dtype=torch.int32, device=gpu)
    n, kept = cache.evict(lens, table, new, 200)
    k2, _ = cache.gather(n, new, 200)
    assert torch.equal(k2, torch.stack([k[kept[0, h].long(), h] for h in range(8)], 1))
    cache.destroy()


def test_shared_blocks_collect_weights_of_all_sequences(uh, gpu):
    p = Pair(uh, gpu, [100, 100], heads=2, bt=64, seed=17)
    p.tables[1] = p.tables[0]
    p.append([100, 0])
    p.check_attend([1, 1], 4, accumulate=True)


def test_repeated_calls_give_the_same_bits(uh, gpu):
    p = Pair(uh, gpu, [3000, 900, 17], heads=2, bt=64, seed=18)
    p.fill()
    for counts in ([1, 1, 1], [500, 3, 17]):
        q = p.random(sum(counts), 8)
        args = (q, p.dev(p.lengths), p.dev(p.tables))
        first = p.cache.attend(*args, starts=p.starts(counts)).clone()
        for _ in range(3):
            assert torch.equal(p.cache.attend(*args, starts=p.starts(counts)), first)


def test_other_streams_and_workspaces(uh, gpu):
    p = Pair(uh, gpu, [4000, 300], heads=2, bt=64, seed=19)
    p.fill()
    for counts, acc in (([1, 1], False), ([200, 300], True)):
        q = p.random(sum(counts), 8)
        args = (q, p.dev(p.lengths), p.dev(p.tables))
        kw = dict(starts=p.starts(counts), accumulate=acc)
        ref = p.cache.attend(*args, **kw)
        need = p.cache.attend_plan(*args, **kw).workspace_bytes
        ws = torch.full((need + 256,), 0xff, dtype=torch.uint8, device=gpu)
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            got = p.cache.attend(*args, workspace=ws[:need], **kw)
            again = p.cache.attend(*args, stream=side, **kw)
        side.synchronize()
        assert torch.equal(got, ref) and torch.equal(again, ref)
        assert (ws[need:] == 0xff).all()
        if need > 0:
            with pytest.raises(uh.HipError) as e:
                p.cache.attend(*args, workspace=ws[:need - 1], **kw)
            assert e.value.status == uh.Status.BUFFER_TOO_SMALL


def test_decode_steps_under_a_graph(uh, gpu):
    """Append and attend captured once; every replay is a step of its own."""
    p = Pair(uh, gpu, [200, 90], heads=2, bt=64, seed=20)
    twin = Pair(uh, gpu, [200, 90], heads=2, bt=64, seed=20)
    k0, v0 = p.random(230, 2), p.random(230, 2)
    for c in (p, twin):
        c.cache.append(k0, v0, c.dev([160, 70]), c.dev(c.tables), starts=c.starts([160, 70]))
    lens, table = p.dev([160, 70]), p.dev(p.tables)
    q, k, v = p.random(2, 8), p.random(2, 2), p.random(2, 2)
    out = torch.empty_like(q)

    def step():
        lens.add_(1)
        p.cache.append(k, v, lens, table)
        p.cache.attend(q, lens, table, out=out, accumulate=True)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()                              # warm-up, and the twin's first step
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    expect = [161, 71]
    twin.cache.append(k, v, twin.dev(expect), twin.dev(twin.tables))
    twin.cache.attend(q, twin.dev(expect), twin.dev(twin.tables), accumulate=True)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        step()
    for i in range(5):
        q.copy_(p.random(2, 8))
        k.copy_(p.random(2, 2))
        v.copy_(p.random(2, 2))
        torch.randn(1 << 16, device=gpu).sum()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        expect = [n + 1 for n in expect]
        tl = twin.dev(expect)
        twin.cache.append(k, v, tl, twin.dev(twin.tables))
        ref = twin.cache.attend(q, tl, twin.dev(twin.tables), accumulate=True)
        assert torch.equal(out, ref), i
    w = p.cache.gather_weights(lens, table, sum(expect), starts=p.starts(expect))
    w2 = twin.cache.gather_weights(twin.dev(expect), twin.dev(twin.tables), sum(expect),
                                   starts=twin.starts(expect))
    assert torch.equal(w, w2)


# ------------------------------------------------------------------ eviction

def _evict(p, keep, sink, recent):
    columns = -(-keep // p.bt)
    new = np.full((len(p.lengths), columns), -1, np.int32)
    for b, n in enumerate(p.lengths):
        for j in range(-(-min(max(n, 0), keep) // p.bt)):
            new[b, j] = p.free.pop()
    lens, kept = p.cache.evict(p.dev(p.lengths), p.dev(p.tables), p.dev(new), keep, sink, recent)
    rkept, rlens = p.ref.evict(p.lengths, p.tables, new, keep, sink, recent)
    assert lens.tolist() == rlens
    assert np.array_equal(kept.cpu().numpy(), rkept)
    w, rw = p.check_stored(tables=new, lengths=rlens)
    assert same(w, rw)
    p.check_stored()                        # the old blocks are as they were


@pytest.mark.parametrize("dim,bt", [(64, 32), (128, 64), (128, 128)])
@pytest.mark.parametrize("keep,sink,recent", [(1, 0, 0), (1, 1, 0), (40, 4, 9), (64, 0, 64),
                                              (100, 3, 0), (130, 1, 1)])
def test_evict(uh, gpu, dim, bt, keep, sink, recent):
    p = Pair(uh, gpu, [0, 1, 40, 41, 130, 300], dim=dim, bt=bt, seed=keep, extra=40)
    p.fill(weights=True)
    _evict(p, keep, sink, recent)


def test_evict_ties_and_odd_weights(uh, gpu):
    p = Pair(uh, gpu, [257, 2100], bt=64, seed=21, extra=40)
    w = p.rs.integers(0, 3, (2357, 2)).astype(np.float32)    # long ties
    w[5, 0], w[250, 0], w[6, 1] = np.nan, np.nan, np.inf
    w[7, 1], w[8, 1], w[9, 0], w[10, 0] = -1.0, -np.inf, -0.0, 1e-45
    p.append(p.lengths, weights=w)
    _evict(p, 100, 2, 30)


def test_evict_equal_weights_keep_the_first(uh, gpu):
    p = Pair(uh, gpu, [1500], bt=32, seed=22, extra=60)
    p.append(p.lengths)                     # all weights 0
    _evict(p, 1030, 0, 5)


def test_evict_blocks_of_different_exponents(uh, gpu):
    p = Pair(uh, gpu, [256], bt=64, seed=23, extra=8)
    k, v = p.random(256, 2), p.random(256, 2)
    for i, std in enumerate((1e-30, 1.0, 3e30, 1e3)):
        k[64 * i:64 * i + 64] = (k[64 * i:64 * i + 64].float() * std).bfloat16()
    v[:64], v[64:128] = float("nan"), 0
    k[130, 0, 3] = float("inf")
    w = p.rs.random((256, 2)).astype(np.float32)
    p.append([256], k=k, v=v, weights=w)
    _evict(p, 128, 0, 0)


def test_evict_after_attention(uh, gpu):
    """The weights that attention added decide, and attention goes on in the
    new blocks."""
    p = Pair(uh, gpu, [400, 350], heads=2, bt=64, seed=24, extra=20)
    p.fill()
    p.check_attend([64, 64], 8, accumulate=True)
    counts = [400, 350]
    w = p.cache.gather_weights(p.dev(p.lengths), p.dev(p.tables), 750, starts=p.starts(counts))
    # The reference continues from the device's weights: their last bits order tokens.
    p.ref.append(*p.ref.gather(p.lengths, p.tables, counts)[:2], p.lengths, p.tables, counts,
                 f64(w))
    _evict(p, 150, 4, 50)
