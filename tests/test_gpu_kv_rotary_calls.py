"""Calls of the rotating append that a server makes around it: rows of no
sequence, lengths past the tables, other streams, strides past 32 bits, two
graphs over one cache."""
import numpy as np
import pytest
import torch

from kv_reference4 import rotate
from test_gpu_kv_cache import f64, same
from test_gpu_kv_rotary import check, freqs, pair, same_queries

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [4, 8])
def test_rows_of_no_sequence_are_left_alone(uh, gpu, bits):
    p = pair(bits, uh, gpu, [50, 60], heads=2, bt=32, seed=1)
    f = freqs(gpu, 64)
    p.fill()
    q, k, v = p.random(9, 4), p.random(9, 2), p.random(9, 2)
    out = torch.full_like(q, 3.0)
    p.cache.append_rotary(q, k, v, p.dev(p.lengths), p.dev(p.tables), f,
                          starts=p.dev([2, 4, 6]), out=out)
    at = np.array([48, 49, 58, 59])
    assert same_queries(out[2:6], q[2:6], at[None], f)
    assert (out[:2] == 3).all() and (out[6:] == 3).all()
    p.ref.append(rotate(f64(k[2:6]), at[None], f64(f)), f64(v[2:6]), p.lengths, p.tables, [2, 2])
    p.check_stored()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dim,bt", [(64, 32), (64, 128), (128, 32), (128, 64), (128, 128)])
def test_the_same_number_of_rows_each(uh, gpu, bits, dim, bt):
    """Without starts: on both sides of where each pair of a sequence's rows has a
    thread of its own, across the ends of chunks and blocks, before the first
    token and in places of no block, against the same call with starts."""
    lengths = [0, 1, 3, 33, bt, bt + 2, 200]
    p, twin = (pair(bits, uh, gpu, lengths, heads=2, dim=dim, bt=bt, seed=6, spare=1)
               for _ in range(2))
    p.tables[6, 0] = twin.tables[6, 0] = -1
    f = freqs(gpu, dim // 2)
    for i, each in enumerate((1, 2, 4, 5, 8, 9, 16)):
        now = [n + i for n in lengths]
        q, k, v = p.random(7 * each, 6), p.random(7 * each, 2), p.random(7 * each, 2)
        at = p.rs.integers(0, 10 ** 6, (2, 7 * each))
        axes = np.arange(dim // 2) % 2
        kw = dict(positions=at, axes=axes, interleaved=True) if i % 2 else {}
        want = check(twin, [each] * 7, 6, f, lengths=now, q=q, k=k, v=v, stored=False, **kw)
        got = p.cache.append_rotary(
            q, k, v, p.dev(now), p.dev(p.tables), f, interleaved=bool(i % 2),
            positions=p.dev(at) if i % 2 else None,
            pair_axes=p.dev(axes, torch.uint8) if i % 2 else None)
        assert torch.equal(got, want), each
        twin.check_stored(lengths=now)
        for a, b in zip(*(c.cache.gather(c.dev(now), c.dev(c.tables), sum(now),
                                         starts=c.starts(now)) for c in (p, twin))):
            assert torch.equal(a, b), each


@pytest.mark.parametrize("bits", [4, 8])
def test_no_rows(uh, gpu, bits):
    """Tensors without rows have no address."""
    p = pair(bits, uh, gpu, [50, 60], heads=2, bt=32, seed=7)
    p.fill()
    q, k = p.random(0, 4), p.random(0, 2)
    for positions in (None, np.zeros((1, 0)), np.zeros((3, 0))):
        got = p.cache.append_rotary(
            q, k, k, p.dev(p.lengths), p.dev(p.tables), freqs(gpu, 64), starts=p.dev([0, 0, 0]),
            positions=None if positions is None else p.dev(positions),
            pair_axes=p.dev(np.arange(64) % 3, torch.uint8))
        assert got.shape == (0, 4, 128)
    p.check_stored()


@pytest.mark.parametrize("bits", [4, 8])
def test_lengths_past_the_tables(uh, gpu, bits):
    """They are taken as the tables' end, places too."""
    p = pair(bits, uh, gpu, [64, 128], heads=1, dim=64, bt=64, seed=2, spare=0)
    p.fill()
    check(p, [3, 5], 2, freqs(gpu, 32), lengths=[64, 1000], stored=False)
    p.lengths = [64, 128]
    p.check_stored()


@pytest.mark.parametrize("bits", [4, 8])
def test_streams(uh, gpu, bits):
    """On torch's current stream, or on one that is named."""
    p, twin = (pair(bits, uh, gpu, [300, 77], heads=2, bt=64, seed=3) for _ in range(2))
    f = freqs(gpu, 64)
    q, k, v = p.random(377, 8), p.random(377, 2), p.random(377, 2)
    args = (q, k, v, p.dev(p.lengths), p.dev(p.tables), f)
    want = twin.cache.append_rotary(*args, starts=p.starts([300, 77]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = torch.zeros_like(q)
    side.wait_stream(torch.cuda.current_stream())
    starts = p.starts([300, 77])
    torch.cuda.synchronize()
    p.cache.append_rotary(*args, starts=starts, out=got, stream=side)
    with torch.cuda.stream(side):
        again = p.cache.append_rotary(*args, starts=starts)
        kv = p.cache.gather(args[3], args[4], 377, starts=starts)
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(again, want)
    for a, b in zip(kv, twin.cache.gather(args[3], args[4], 377, starts=starts)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("odd", [0, 1])
def test_strides_past_32_bits(uh, gpu, bits, odd):
    """Rows of q, k, v and of the result 2^31 elements and more apart."""
    far = 2 ** 31 + 64 + odd
    flat = torch.empty(2 * far + 4096, dtype=torch.bfloat16, device=gpu)
    p = pair(bits, uh, gpu, [40], heads=2, bt=32, seed=4)
    p.fill()

    def view(heads, at):
        return flat.as_strided((3, heads, 128), (far, 128, 1), at)
    q, k, v, out = view(4, 0), view(2, 512), view(2, 768), view(4, 1024)
    for x in (q, k, v):
        x.copy_(p.random(3, x.shape[1]))
    check(p, [3], 4, freqs(gpu, 64), q=q, k=k, v=v, out=out)
    near = p.cache.attend(out.contiguous(), p.dev([40]), p.dev(p.tables))
    assert torch.equal(p.cache.attend(out, p.dev([40]), p.dev(p.tables)), near)


@pytest.mark.parametrize("bits", [4, 8])
def test_two_graphs_over_one_cache(uh, gpu, bits):
    """A step of one sequence and of another, captured apart and replayed in turn
    on one stream, against eager steps of a twin."""
    both = [pair(bits, uh, gpu, [120, 90], heads=2, bt=32, seed=5) for _ in range(2)]
    f = freqs(gpu, 64)
    lens = [[c.dev([60]), c.dev([40])] for c in both]
    tables = [[c.dev(c.tables[b:b + 1]) for b in (0, 1)] for c in both]
    q, k, v = both[0].random(1, 8), both[0].random(1, 2), both[0].random(1, 2)
    outs = [torch.empty_like(q) for _ in range(2)]

    def step(c, b, out):
        n, t = lens[c][b], tables[c][b]
        n.add_(1)
        turned = both[c].cache.append_rotary(q, k, v, n, t, f)
        return both[c].cache.attend(turned, n, t, out=out, accumulate=True)

    start = [both[0].random(n, 2) for n in (60, 40)]
    for c in (0, 1):
        for b in (0, 1):
            both[c].cache.append(start[b], start[b], lens[c][b], tables[c][b])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for b in (0, 1):
            step(0, b, outs[b])
    torch.cuda.synchronize()
    for b in (0, 1):
        step(1, b, None)
    graphs = []
    for b in (0, 1):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            step(0, b, outs[b])
        graphs.append(g)
    for i in range(6):
        b = i % 3 % 2
        for x in (q, k, v):
            x.copy_(both[0].random(1, x.shape[1]))
        torch.cuda.synchronize()
        graphs[b].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[b], step(1, b, None)), i
    for b in (0, 1):
        rows = int(lens[0][b][0])
        assert rows == int(lens[1][b][0])
        for a, w in zip(both[0].cache.gather(lens[0][b], tables[0][b], rows),
                        both[1].cache.gather(lens[1][b], tables[1][b], rows)):
            assert torch.equal(a, w)
        w = [f64(c.cache.gather_weights(lens[i][b], tables[i][b], rows))
             for i, c in enumerate(both)]
        assert same(*w)
