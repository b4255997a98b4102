"""Rotary positions on the way into caches of 8 and 4 bits, against 64-bit
rotation with exactly reduced angles (kv_reference4.py).

Stored keys are compared bit for bit: they are rounded once from the rotation
in 64 bits, whose error of some 2^-52 meets a border of two codes with a
probability of some 2^-40 for an element.  Queries x, y are rotated in f32: the
cosine, the sine, one product and the sum are each rounded by 2^-24 of at most
|x| + |y|, and the result to bf16 by 2^-8 of itself."""
import numpy as np
import pytest
import torch

import test_gpu_kv4_cache as T4
import test_gpu_kv_cache as T8
from kv_reference4 import rotate
from test_gpu_kv_cache import f64, same

pytestmark = pytest.mark.gpu


def same_queries(got, q, positions, f, axes=None, interleaved=False):
    """Whether the rotated queries are within their bound; whole where not finite."""
    q, f = f64(q), f64(f)
    ref = rotate(q, positions, f, axes, interleaved)
    size = np.abs(q)
    with np.errstate(invalid="ignore"):
        turned = rotate(size, positions, np.zeros_like(f), axes, interleaved)
    half = len(f)
    order = np.arange(q.shape[-1])
    if interleaved:
        order[:2 * half] = order[:2 * half] ^ 1
    else:
        order[:2 * half] = (order[:2 * half] + half) % (2 * half)
    size = turned + size[..., order]
    got = f64(got)
    # Past the largest bf16 and half a step results are infinite.
    ref = np.where(np.abs(ref) >= 2.0 ** 128 * (1 - 2.0 ** -9), np.copysign(np.inf, ref), ref)
    fine = np.isfinite(ref)
    tol = 2.0 ** -22 * size[fine]
    tol = tol + 2.0 ** -8 * (np.abs(ref[fine]) + tol) + 2.0 ** -133
    return np.array_equal(np.isnan(got), np.isnan(ref)) and \
        np.array_equal(got[np.isinf(ref)], ref[np.isinf(ref)]) and \
        bool((np.abs(got[fine] - ref[fine]) <= tol).all())


def pair(bits, *a, **kw):
    return (T4 if bits == 4 else T8).Pair(*a, **kw)


def freqs(gpu, half, base=10000.0):
    return torch.tensor([base ** (-j / half) for j in range(half)], dtype=torch.float32, device=gpu)


def places(lengths, counts, columns, bt):
    return np.concatenate([min(max(n, 0), columns * bt) - c + np.arange(c)
                           for n, c in zip(lengths, counts)]).astype(np.int64)


def check(p, counts, heads, f, lengths=None, positions=None, axes=None, interleaved=False, q=None,
          k=None, v=None, out=None, weights=None, starts=None, stored=True):
    """One append_rotary against the reference: queries, then all that is stored."""
    lengths = p.lengths if lengths is None else lengths
    rows = int(sum(counts))
    q = p.random(rows, heads) if q is None and heads else q
    k = p.random(rows, p.heads) if k is None else k
    v = p.random(rows, p.heads) if v is None else v
    at = places(lengths, counts, p.columns, p.bt)[None] if positions is None else \
        np.atleast_2d(positions)
    rk = rotate(f64(k), at, f64(f), axes, interleaved)
    got = p.cache.append_rotary(
        q, k, v, p.dev(lengths), p.dev(p.tables), f,
        starts=p.starts(counts) if starts is None else starts,
        positions=None if positions is None else p.dev(positions),
        pair_axes=None if axes is None else p.dev(axes, torch.uint8), interleaved=interleaved,
        out=out, weights=None if weights is None else p.dev(weights, torch.float32))
    p.ref.append(rk, f64(v), lengths, p.tables, counts, weights)
    if heads:
        assert same_queries(got, q, at, f, axes, interleaved)
    else:
        assert got is None
    if stored:
        w, rw = p.check_stored(lengths=[max(n, 0) for n in lengths])
        assert same(w, rw)
    return got


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dim,bt", [(64, 32), (64, 128), (128, 32), (128, 64), (128, 128)])
def test_prompts_then_single_tokens(uh, gpu, bits, dim, bt):
    p = pair(bits, uh, gpu, [0, 1, 31, 33, 64, 97, 130], dim=dim, bt=bt, seed=bt + dim, spare=1)
    f = freqs(gpu, dim // 2)
    check(p, p.lengths, 4, f)
    for b, n in enumerate(p.lengths):
        for j in range(-(-(n + 2) // bt)):
            if p.tables[b, j] < 0 and p.free:
                p.tables[b, j] = p.free.pop()
    for step in (1, 2):
        check(p, [1] * 7, 6, f, lengths=[n + step for n in p.lengths])
    check(p, [3, 0, 7, 1, 0, 50, 2], 0, f, lengths=[n + 2 for n in p.lengths])


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rotary", [(128, 128), (128, 64), (128, 32), (128, 42), (128, 2),
                                        (128, 126), (64, 64), (64, 16), (64, 34)])
def test_parts_of_heads_and_pairings(uh, gpu, bits, interleaved, dim, rotary):
    p = pair(bits, uh, gpu, [45, 70], dim=dim, bt=64, seed=rotary)
    check(p, p.lengths, 2, freqs(gpu, rotary // 2), interleaved=interleaved)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("interleaved", [False, True])
def test_axes(uh, gpu, bits, interleaved):
    p = pair(bits, uh, gpu, [90, 40], dim=128, bt=64, seed=3)
    r = np.random.default_rng(1)
    for axes in (1, 2, 3, 4):
        at = r.integers(-50, 5000, (axes, 130)).astype(np.int32)
        of = r.integers(0, axes + 2, 48).astype(np.uint8)     # some past the last axis
        check(p, p.lengths, 2, freqs(gpu, 48), positions=at, axes=of, interleaved=interleaved)
    # Sections, and positions of one axis without an axis of its own.
    check(p, p.lengths, 4, freqs(gpu, 64), positions=at[:3], axes=np.repeat([0, 1, 2], [16, 24, 24]))
    check(p, p.lengths, 4, freqs(gpu, 64), positions=at[0])
    check(p, p.lengths, 4, freqs(gpu, 64), positions=at[1:2])


@pytest.mark.parametrize("bits", [4, 8])
def test_far_positions(uh, gpu, bits):
    p = pair(bits, uh, gpu, [64], dim=128, bt=64, seed=4)
    at = np.array([0, 1, -1, 2 ** 31 - 1, -2 ** 31, 2 ** 31 - 2, 10 ** 6, 10 ** 9] * 8, np.int64)
    f = torch.tensor([1.0, 3.0, 1e4, 6.2831855, 1e-9, 0.0, 0.1, -0.5] * 8, device=gpu)
    check(p, [64], 2, f, positions=at)


@pytest.mark.parametrize("bits", [4, 8])
def test_strides_and_in_place(uh, gpu, bits):
    """Thirds of a projection's output, heads outermost, odd addresses; and the
    queries rotated where they are."""
    p = pair(bits, uh, gpu, [37, 90], heads=2, dim=64, bt=32, seed=5)
    rows, f = 127, freqs(gpu, 32)
    qkv = p.random(rows, 8)
    keep = qkv.clone()
    check(p, p.lengths, 4, f, q=qkv[:, :4], k=qkv[:, 4:6], v=qkv[:, 6:])
    assert torch.equal(qkv, keep)
    buf = qkv.clone()
    at = places(p.lengths, p.lengths, p.columns, 32)[None]
    got = p.cache.append_rotary(buf[:, :4], buf[:, 4:6], buf[:, 6:], p.dev(p.lengths),
                                p.dev(p.tables), f, starts=p.starts(p.lengths), out=buf[:, :4])
    assert got.data_ptr() == buf.data_ptr() and same_queries(buf[:, :4], keep[:, :4], at, f)
    assert torch.equal(buf[:, 4:], keep[:, 4:])
    p.check_stored()
    by_head = torch.zeros((4, rows, 64), dtype=torch.bfloat16, device=gpu)
    check(p, p.lengths, 4, f, q=p.random(4, rows).transpose(0, 1).contiguous().view(rows, 4, 64),
          out=by_head.transpose(0, 1))
    odd = torch.empty(rows * 193 + 1, dtype=torch.bfloat16, device=gpu)
    x = torch.as_strided(odd, (rows, 2, 64), (193, 64, 1), 1)
    x.copy_(p.random(rows, 2))
    o = torch.zeros(rows * 2 * 64 + 1, dtype=torch.bfloat16, device=gpu)
    for interleaved in (False, True):
        check(p, p.lengths, 2, f, q=x, k=x, v=x, out=o[1:].view(rows, 2, 64),
              interleaved=interleaved)
    assert o[0] == 0


@pytest.mark.parametrize("bits", [4, 8])
def test_rows_without_a_place_have_their_queries_rotated(uh, gpu, bits):
    p = pair(bits, uh, gpu, [5, 100, 0], bt=32, seed=6)
    p.tables[1, 1] = -1
    p.tables[1, 2] = p.blocks
    f = freqs(gpu, 64)
    check(p, [9, 100, 2], 4, f)                       # before the first token, of no block
    check(p, [70, 2, 1], 4, f, lengths=[5, 10 ** 6, -3], stored=False)
    # Rows of no sequence: as they were.
    q, k = p.random(10, 4), p.random(10, 2)
    out = torch.full((10, 4, 128), 3.0, dtype=torch.bfloat16, device=gpu)
    p.cache.append_rotary(q, k, k, p.dev([5, 100, 0]), p.dev(p.tables), f, starts=p.dev([2, 4, 6, 6]),
                          out=out)
    assert (out[:2] == 3).all() and (out[6:] == 3).all()
    assert same_queries(out[2:6], q[2:6], np.array([[3, 4, 98, 99]]), f)


@pytest.mark.parametrize("bits", [4, 8])
def test_extremes(uh, gpu, bits):
    p = pair(bits, uh, gpu, [64, 64], bt=64, seed=7)
    f = freqs(gpu, 32)                                # half of the dims
    q, k = p.random(128, 2), p.random(128, 2)
    for x in (q, k):
        x[3, 0, 5], x[4, 1, 40], x[5, 0, 127] = float("inf"), float("-inf"), float("nan")
        x[6, 0, 100] = float("inf")                   # a dim that is not rotated
        x[10:20] = (3.38e38 * torch.sign(x[10:20].float())).bfloat16()
        x[20:30] = (x[20:30].float() * 1e-38).bfloat16()
        x[30:40] = 0
        x[64, 0, 0], x[64, 0, 32] = float("inf"), 1.0  # position 0: cosine 1, sine 0
    with np.errstate(invalid="ignore", over="ignore"):
        check(p, [64, 64], 2, f, q=q, k=k)


@pytest.mark.parametrize("bits", [4, 8])
def test_weights_come_along(uh, gpu, bits):
    p = pair(bits, uh, gpu, [40, 3], bt=32, seed=8)
    w = np.exp(p.rs.standard_normal((43, 2))).astype(np.float32)
    check(p, [40, 3], 2, freqs(gpu, 64), weights=w)
    check(p, [2, 1], 2, freqs(gpu, 64))               # zeros again


def test_8_bit_blocks_follow_the_largest_rotated_key(uh, gpu):
    """Exponents of begun blocks grow with rotated keys, and pairs whose
    rotation reaches past both elements count as rotated."""
    p = T8.Pair(uh, gpu, [40], bt=64, seed=9)
    f = freqs(gpu, 64)
    for step, std in enumerate((2.0 ** -9, 1.0, 37.0, 2.0 ** 13)):
        x = p.random(10, 2, std)
        check(p, [10], 2, f, lengths=[10 + 10 * step], k=x, v=-x)
    k = torch.full((1, 2, 128), 448.0, dtype=torch.bfloat16, device=gpu)
    check(p, [1], 2, torch.full((64,), 0.785398, device=gpu), lengths=[40], k=k, positions=[1])


@pytest.mark.parametrize("bits", [4, 8])
def test_without_rotation_it_is_append(uh, gpu, bits):
    """Position 0 turns nothing: the same codes, the same queries."""
    p, twin = (pair(bits, uh, gpu, [100, 33], bt=64, seed=10) for _ in range(2))
    k, v, q = p.random(133, 2), p.random(133, 2), p.random(133, 4)
    got = p.cache.append_rotary(q, k, v, p.dev(p.lengths), p.dev(p.tables), freqs(gpu, 64),
                                starts=p.starts(p.lengths), positions=p.dev(np.zeros(133)))
    twin.append(twin.lengths, k=k, v=v)
    assert torch.equal(got, q)
    args = (p.dev(p.lengths), p.dev(p.tables), 133)
    for a, b in zip(p.cache.gather(*args, starts=p.starts([100, 33])),
                    twin.cache.gather(*args, starts=p.starts([100, 33]))):
        assert torch.equal(a, b)


@pytest.mark.parametrize("bits", [4, 8])
def test_many_sequences(uh, gpu, bits):
    p = pair(bits, uh, gpu, [3 + i % 40 for i in range(150)], heads=1, dim=64, bt=32, seed=11)
    f = freqs(gpu, 32)
    check(p, p.lengths, 2, f)
    check(p, [i % 3 for i in range(150)], 1, f)
    check(p, [1] * 150, 2, f)


@pytest.mark.parametrize("bits", [4, 8])
def test_rotate_store_attend_under_a_graph(uh, gpu, bits):
    """A decode step of a layer, captured once, on a stream of its own: each
    replay is a step, as the eager calls of a twin are."""
    p, twin = (pair(bits, uh, gpu, [200, 90], heads=2, bt=64, seed=12) for _ in range(2))
    f = freqs(gpu, 64)
    k0, v0 = p.random(230, 2), p.random(230, 2)
    for c in (p, twin):
        c.cache.append_rotary(None, k0, v0, c.dev([160, 70]), c.dev(c.tables), f,
                              starts=c.starts([160, 70]))
    lens, table = p.dev([160, 70]), p.dev(p.tables)
    q, k, v = p.random(2, 8), p.random(2, 2), p.random(2, 2)
    turned, out = torch.empty_like(q), torch.empty_like(q)

    def step():
        lens.add_(1)
        p.cache.append_rotary(q, k, v, lens, table, f, out=turned)
        p.cache.attend(turned, lens, table, out=out, accumulate=True)

    def eager(expect):
        tl = twin.dev(expect)
        turn = twin.cache.append_rotary(q, k, v, tl, twin.dev(twin.tables), f)
        return twin.cache.attend(turn, tl, twin.dev(twin.tables), accumulate=True)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()                              # warm-up, and the twin's first step
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    expect = [161, 71]
    eager(expect)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        step()
    for i in range(5):
        for x in (q, k, v):
            x.copy_(p.random(2, x.shape[1]))
        torch.randn(1 << 16, device=gpu).sum()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        expect = [n + 1 for n in expect]
        assert torch.equal(out, eager(expect)), i
    for one, two in zip(p.cache.gather(lens, table, sum(expect), starts=p.starts(expect)),
                        twin.cache.gather(lens, twin.dev(twin.tables), sum(expect),
                                          starts=p.starts(expect))):
        assert torch.equal(one, two)
