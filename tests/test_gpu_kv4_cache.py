"""GPU parity of the 4-bit key/value cache (append, gather, attend, evict)
through the Python mirror, against the 64-bit reference of kv_reference4.py.

Stored values are compared bit for bit.  Attention is compared within a bound
that the reference computes for each element from the documented arithmetic
(RefCache4.attend), fixed before any run."""
import numpy as np
import pytest
import torch

import test_gpu_kv_cache as T
from kv_attention64 import attention64, within
from kv_reference4 import RefCache4
from test_gpu_kv_cache import f64, same

pytestmark = pytest.mark.gpu


class Pair(T.Pair):
    """A cache of 4 bits and its reference."""

    def __init__(self, uh, gpu, lengths, **kw):
        super().__init__(uh, gpu, lengths, **kw)
        self.cache.destroy()
        self.cache = uh.KvCache(self.blocks, self.heads, self.dim, block_tokens=self.bt,
                                track_weights=True, bits=4)
        self.ref = RefCache4(self.blocks, self.heads, self.dim, self.bt)


# ------------------------------------------------------------------- storing

@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("bt", [32, 64, 128])
def test_append_prompts_and_single_tokens(uh, gpu, dim, bt):
    p = Pair(uh, gpu, [0, 1, 31, 33, 64, 97, 129], dim=dim, bt=bt, seed=bt + dim, spare=1)
    p.fill()
    p.check_stored()
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


def test_every_place_of_a_chunk(uh, gpu):
    """Pieces of every length from every place on leave the others alone."""
    p = Pair(uh, gpu, [96], dim=64, bt=32, seed=1)
    p.fill()
    for first in range(0, 96, 5):
        for n in (1, 2, 7, 31, 33):
            if first + n <= 96:
                p.append([n], [first + n])
    p.check_stored()


def test_scales_of_every_size(uh, gpu):
    """Largest elements at and beside every border of a scale: each bf16
    significand over several binades, as largest element of a key's 32 and a
    value, among others that fall on the borders of codes."""
    p = Pair(uh, gpu, [2048], heads=1, dim=64, bt=128, seed=2)
    r = np.random.default_rng(3)
    top = np.array([(128 + i % 128) / 128 * 2.0 ** (i // 128 % 16 - 8) for i in range(2048)])
    border = np.array([0, 0.25, 0.5, 0.75, 1, 1.25, 1.75, 2.5, 3.5, 5, 6, 5.5])
    x = border[r.integers(0, len(border), (2048, 64))] * r.choice([-1, 1], (2048, 64))
    k = x * (2.0 ** np.floor(np.log2(top / 6)))[:, None]
    k[:, 3], k[:, 40] = top, -top
    v = x * (top / 6)[:, None]
    v[:, 17] = top
    dev = [torch.tensor(y, device=gpu).bfloat16()[:, None] for y in (k, v)]
    p.append([2048], k=dev[0], v=dev[1])
    p.check_stored()


def test_append_extremes(uh, gpu):
    p = Pair(uh, gpu, [64, 64, 64, 64], bt=64, seed=3)
    x, y = p.random(256, 2), p.random(256, 2)
    x[3, 0, 5], x[4, 1, 36], x[5, 0, 127] = float("inf"), float("-inf"), float("nan")
    y[9, 0, 0], y[10, 1, 100] = float("nan"), float("inf")
    x[64:128] = 3.38e38 * torch.sign(x[64:128].float())   # the top of bf16: saturates
    y[64:96] = 0
    y[96:128] = (y[96:128].float() * 1e30).bfloat16()     # past the largest scale
    x[128:192] = (x[128:192].float() * 1e-38).bfloat16()  # the bottom: flushed
    y[128:160] = (y[128:160].float() * 2.0 ** -18).bfloat16()
    y[160:192] = (y[160:192].float() * 2.0 ** -60).bfloat16()
    y[192, 0], y[193, 0], y[194, 0] = 387072.0, 389120.0, 2.0 ** -17   # ends of the scales
    x[195, 1] = 0
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
        odd = torch.empty(rows * 193 + 1, dtype=torch.bfloat16, device=gpu)
        v = torch.as_strided(odd, (rows, 3, 64), (193, 64, 1), 1)
        v.copy_(p.random(rows, 3))
        k = v
    p.append(p.lengths, k=k, v=v)
    p.check_stored()


def test_rows_without_a_place(uh, gpu):
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


@pytest.mark.parametrize("rows", [1, 200])
def test_values_of_very_different_scales(uh, gpu, rows):
    """Scales over their whole range, token by token, in both orders; and a
    token of most of the weight beside ones with most of the result."""
    p = Pair(uh, gpu, [256], heads=1, bt=64, seed=11)
    v = p.random(256, 1)
    power = torch.tensor([2.0 ** (i % 34 - 19) for i in range(256)], device=gpu)
    for order in (power, power.flip(0)):
        x = (v.float() * order[:, None, None]).bfloat16()
        p.append([256], v=x)
        p.check_attend([rows], 2)
    k = p.random(256, 1) * 0.01
    k[5, 0] = 3.0                                        # scores near 200 with q of ones
    x = v.clone()
    x[5] = (x[5].float() * 2.0 ** -15).bfloat16()
    p.append([256], k=k, v=x)
    p.check_attend([rows], 2, q=torch.ones((rows, 2, 128), dtype=torch.bfloat16, device=gpu) * 0.3)


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


def test_rows_that_see_nan_alone(uh, gpu):
    """One token whose value is NaN: its result is, its log-sum is the score."""
    p = Pair(uh, gpu, [1, 40], heads=1, bt=32, seed=13)
    v = p.random(41, 1)
    v[0, 0, 1] = float("nan")
    v[1:] = float("nan")
    p.append([1, 40], v=v)
    for counts in ([1, 1], [1, 40]):
        p.check_attend(counts, 4)


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


@pytest.mark.parametrize("length,rows,dim,heads,kv_heads,window", [
    (20000, 1, 128, 32, 8, 0), (9000, 16, 64, 14, 2, 0), (9000, 40, 128, 8, 1, 5000),
    (6000, 1200, 128, 8, 2, 0), (5000, 900, 64, 14, 2, 700), (33000, 300, 128, 8, 8, 0)])
def test_long_sequences(uh, gpu, length, rows, dim, heads, kv_heads, window):
    """Lengths that the reference above is too slow for, against torch in 64
    bits over the gathered values."""
    torch.manual_seed(length)
    cache = uh.KvCache(-(-length // 64) + 2, kv_heads, dim, bits=4)
    table = torch.randperm(cache.blocks, device=gpu, dtype=torch.int32)[None, :-(-length // 64)]
    k, v = (torch.randn((length, kv_heads, dim), device=gpu).bfloat16() for _ in "kv")
    n = torch.tensor([length], dtype=torch.int32, device=gpu)
    cache.append(k, v, n, table.contiguous())
    kk, vv = cache.gather(n, table.contiguous(), length)
    q = torch.randn((rows, heads, dim), device=gpu).bfloat16()
    lse = torch.empty((rows, heads), device=gpu)
    out = cache.attend(q, n, table.contiguous(), window=window, lse=lse)
    pick = torch.arange(0, rows, max(1, rows // 37), device=gpu)
    ref, tol, rlse, ltol, _, _ = attention64(q[pick], kk, vv, length - rows + pick, dim ** -0.5,
                                             window)
    within(out[pick], ref, tol, "out")
    within(lse[pick], rlse, ltol, "lse")


def test_offsets_past_32_bits(uh, gpu):
    """A pool of 9 GiB, with the sequence in its last blocks."""
    blocks = 9 * 2 ** 30 // (8 * 4 * 4288)
    cache = uh.KvCache(blocks, 8, 128, block_tokens=128, track_weights=True, bits=4)
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


def test_rows_of_no_sequence_are_left_alone(uh, gpu):
    p = Pair(uh, gpu, [50, 60], heads=2, bt=32, seed=20)
    p.fill()
    q = p.random(9, 4)
    out = torch.full((9, 4, 128), 3.0, dtype=torch.bfloat16, device=gpu)
    lse = torch.full((9, 4), 5.0, device=gpu)
    starts = p.dev([2, 4, 6])
    p.cache.attend(q, p.dev(p.lengths), p.dev(p.tables), starts=starts, out=out, lse=lse)
    for rest in (slice(0, 2), slice(6, 9)):
        assert (out[rest] == 3).all() and (lse[rest] == 5).all()
    assert not (out[2:6] == 3).all()


# ------------------------------------------------------------------ eviction

@pytest.mark.parametrize("dim,bt", [(64, 32), (128, 64), (128, 128)])
@pytest.mark.parametrize("keep,sink,recent", [(1, 0, 0), (1, 1, 0), (40, 4, 9), (64, 0, 64),
                                              (100, 3, 0), (130, 1, 1)])
def test_evict(uh, gpu, dim, bt, keep, sink, recent):
    p = Pair(uh, gpu, [0, 1, 40, 41, 130, 300], dim=dim, bt=bt, seed=keep, extra=40)
    p.fill(weights=True)
    T._evict(p, keep, sink, recent)


def test_evict_odd_tokens(uh, gpu):
    """NaN, zeros and scales of both ends move as they are; tokens of blocks
    out of the pool become zeros."""
    p = Pair(uh, gpu, [257], bt=64, seed=21, extra=40)
    k, v = p.random(257, 2), p.random(257, 2)
    k[3, 0, 40], v[5, 1, 2] = float("nan"), float("inf")
    v[:64] = (v[:64].float() * 2.0 ** -19).bfloat16()
    v[64:100] = (v[64:100].float() * 2.0 ** 14).bfloat16()
    k[100:130] = 0
    w = p.rs.random((257, 2)).astype(np.float32)
    p.append([257], k=k, v=v, weights=w)
    T._evict(p, 200, 2, 30)
    p.tables[0, 2] = -1
    T._evict(p, 230, 0, 0)


def test_evict_after_attention(uh, gpu):
    p = Pair(uh, gpu, [400, 350], heads=2, bt=64, seed=24, extra=20)
    p.fill()
    p.check_attend([64, 64], 8, accumulate=True)
    counts = [400, 350]
    w = p.cache.gather_weights(p.dev(p.lengths), p.dev(p.tables), 750, starts=p.starts(counts))
    # The reference continues from the device's weights: their last bits order tokens.
    p.ref.append(*p.ref.gather(p.lengths, p.tables, counts)[:2], p.lengths, p.tables, counts,
                 f64(w))
    T._evict(p, 150, 4, 50)


def test_bytes(uh, gpu):
    for dim, per in ((64, 68), (128, 134)):
        c = uh.KvCache(10, 3, dim, block_tokens=64, bits=4)
        info = c.info()
        assert info.device_bytes == 10 * 3 * 64 * per and info.flags == uh.KV_CACHE_4_BITS
        c.destroy()
