"""The 4-bit cache and the rotating append on a live handle: what they refuse,
the kernels that calls of different sizes take, large tiles, and calls that
share a stream's workspace."""
import ctypes

import numpy as np
import pytest
import torch

import test_gpu_kv4_cache as T4
import test_gpu_kv_calls as C
from test_gpu_kv4_cache import Pair
from test_gpu_kv_calls import WIDE

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ refusals

class Calls(C.Calls):
    """The calls of a cache of 4 bits, and append_rotary into both kinds."""

    def __init__(self, uh, gpu):
        super().__init__(uh, gpu)
        self.eight = self.track
        self.track = uh.KvCache(8, 2, 128, track_weights=True, bits=4)
        self.plain = uh.KvCache(8, 2, 128, bits=4)

    def rotary(self, cache="track", seqs=None, reserved=0, **over):
        uh = self.uh
        fields = dict(q=self.at(2), q_out=self.at(4), k=self.at(6), v=self.at(7), heads=8,
                      inv_freq=self.at(8), rotary_dims=128, axes=1)
        handle = cache if isinstance(cache, uh.KvCache) else getattr(self, cache)
        d = uh.new(uh.KvAppendRotaryDesc, cache=handle.handle,
                   seqs=uh.KvSequences(**{**self.seqs, **(seqs or {})}), **{**fields, **over})
        d.reserved[3] = reserved
        s = uh._Sink()
        st = uh.Status(uh.lib().ullm_kv_cache_append_rotary(ctypes.byref(d), s.ref))
        return st.name, s.text()


@pytest.fixture(scope="module")
def calls(uh, gpu):
    return Calls(uh, gpu)


@pytest.mark.parametrize("name,over,status,word", C.REFUSED)
def test_refusals(calls, name, over, status, word):
    st, text = calls.call(name, **over)
    assert st == status and word in text, (st, text)


ROTARY = C.ANY + C.ROWS + [
    ({"k": 0}, "INVALID_ARGUMENT", "null"), ({"v": 0}, "INVALID_ARGUMENT", "null"),
    ({"inv_freq": 0}, "INVALID_ARGUMENT", "null"), ({"q": 0}, "INVALID_ARGUMENT", "null"),
    ({"q_out": 0}, "INVALID_ARGUMENT", "null"), ({"heads": 3}, "INVALID_ARGUMENT", "heads"),
    ({"heads": 1 << 30}, "UNSUPPORTED", "heads"), ({"flags": 2}, "INVALID_ARGUMENT", "flags"),
    ({"rotary_dims": 0}, "INVALID_ARGUMENT", "rotary_dims"),
    ({"rotary_dims": 31}, "INVALID_ARGUMENT", "rotary_dims"),
    ({"rotary_dims": 130}, "INVALID_ARGUMENT", "rotary_dims"),
    ({"axes": 0}, "INVALID_ARGUMENT", "axes"), ({"axes": 5}, "INVALID_ARGUMENT", "axes"),
    ({"axes": 2}, "INVALID_ARGUMENT", "positions"),
    ({"axes": 2, "positions": 4096, "position_stride": 3}, "INVALID_ARGUMENT", "position_stride"),
    ({"k_row_stride": 127}, "INVALID_ARGUMENT", "stride"),
    ({"v_head_stride": 64}, "INVALID_ARGUMENT", "stride"),
    ({"q_head_stride": 64}, "INVALID_ARGUMENT", "stride"),
    ({"q_out_row_stride": 1}, "INVALID_ARGUMENT", "stride"),
    ({"q_out_row_stride": 256}, "INVALID_ARGUMENT", "overlap")]


@pytest.mark.parametrize("cache", ["track", "eight"])
@pytest.mark.parametrize("over,status,word", ROTARY)
def test_rotary_refusals(calls, cache, over, status, word):
    st, text = calls.rotary(cache, **over)
    assert st == status and word in text, (st, text)


def test_rotary_refusals_of_weights_and_places(calls):
    st, text = calls.rotary("plain", weights=4096)
    assert st == "INVALID_ARGUMENT" and "track" in text
    st, text = calls.rotary(q_out=calls.at(2), q_row_stride=2048)
    assert st == "INVALID_ARGUMENT" and "in place" in text


def test_calls_without_work(calls):
    for cache in ("track", "eight"):
        for seqs in ({"rows": 0}, {"batch": 0, "rows": 0}):
            assert calls.rotary(cache, seqs=seqs)[0] == "OK"
        assert calls.rotary(cache, heads=0, q=0, q_out=0)[0] == "OK"    # lengths of 0: no place
        assert calls.rotary(cache)[0] == "OK"
    torch.cuda.synchronize()


@pytest.mark.parametrize("bits", [4, 8])
def test_appends_refuse_more_workgroups_than_a_launch_has(calls, uh, bits):
    """65535 sequences of 512 heads, by the checks on the host alone (the
    pointers name a megabyte): two spans for each are over 2^32 threads."""
    c = uh.KvCache(1, 512, 64, block_tokens=128, bits=bits)
    seqs = dict(batch=65535, rows=65535, starts=calls.at(9), max_blocks=1, table_stride=1)
    st, text = calls.rotary(c, seqs=seqs, heads=0, rotary_dims=64)
    assert st == "UNSUPPORTED" and "spans" in text
    if bits == 4:
        d = uh.new(uh.KvAppendDesc, cache=c.handle, k=calls.at(6), v=calls.at(7),
                   seqs=uh.KvSequences(**{**calls.seqs, **seqs}))
        s = uh._Sink()
        st = uh.Status(uh.lib().ullm_kv_cache_append(ctypes.byref(d), s.ref))
        assert st == uh.Status.UNSUPPORTED and "spans" in s.text()


@pytest.mark.parametrize("name", ["attend", "attend_plan"])
def test_the_scale_of_scores(calls, name):
    for scale in (1e30, -1e30, 3e38):
        st, text = calls.call(name, scale=scale)
        assert st == "INVALID_ARGUMENT" and "scale" in text
        assert calls.call(name, cache="eight", scale=1e30)[0] == "OK"
    for scale in (6e29, -6e29, 0.0, 1e-38):
        assert calls.call(name, scale=scale)[0] == "OK"
    torch.cuda.synchronize()


@pytest.mark.parametrize("rows", [2, 200])
def test_scales_of_scores_at_their_ends(uh, gpu, rows):
    """Scores of 0 whatever the scale, and scores that are all alike."""
    p = Pair(uh, gpu, [300], heads=8, bt=64, seed=22, spare=WIDE // 64)
    size = torch.exp2(torch.randint(-6, 7, (300, 1, 1), device=gpu).float())
    p.append([300], v=(p.random(300, 8).float() * size).bfloat16())
    for scale in (6e29, -6e29, 0.0, 1e-38):
        q = p.random(rows, 32)
        p.check_attend([rows], 32, q=torch.zeros_like(q) if scale else q, scale=scale,
                       kernel=uh.KV_KERNEL_FEW_ROWS if rows == 2 else uh.KV_KERNEL_MANY_ROWS)


@pytest.mark.parametrize("rows", [2, 200])
@pytest.mark.parametrize("size", [2.0 ** -14, 1.0, 2.0 ** 12])
def test_log_sums_of_small_and_large_values(uh, gpu, rows, size):
    """The values' scales are in the references of the powers, not in the log-sum."""
    p = Pair(uh, gpu, [300, 200], heads=8, bt=64, seed=23, spare=WIDE // 64)
    p.append([300, 200], v=p.random(500, 8, std=size))
    for scale in (None, 0.0, -0.2):
        p.check_attend([rows, 1], 32, scale=scale, kernel=uh.KV_KERNEL_FEW_ROWS if rows == 2
                       else uh.KV_KERNEL_MANY_ROWS)
        p.check_attend([1, 1], 16, scale=scale)


# --------------------------------------------------------------------- plans

@pytest.mark.parametrize("counts,heads,lengths,few,parts", [
    ([1], 8, [333], True, 1),
    ([1], 8, [5000], True, 2),
    ([16], 8, [5000], True, 2),
    ([17], 8, [5000], True, 2),               # all small tiles run at once
    ([150, 12], 8, [400, 90], True, 1),
    ([150], 8, [5000], True, 2),
    ([400], 8, [5000], False, 2),
    # (51 + 3 tiles) x 2 heads x 2 parts: 216 run at once; (68 + 4) x 2 x 2 do not.
    ([17, 17, 17], 32, [5000, 4200, 90], True, 2),
    ([17, 17, 17, 17], 32, [5000, 4200, 90, 400], False, 2),
    ([1500, 700], 16, [1500, 700], False, 1)])
def test_plans_and_their_results(uh, gpu, counts, heads, lengths, few, parts):
    p = Pair(uh, gpu, lengths, heads=2, seed=sum(counts))
    p.fill()
    q = p.random(sum(counts), heads)
    plan = p.cache.attend_plan(q, p.dev(lengths), p.dev(p.tables), starts=p.starts(counts))
    kernel = uh.KV_KERNEL_FEW_ROWS if few else uh.KV_KERNEL_MANY_ROWS
    assert plan.kernel == kernel and plan.row_tile == (16 if few else 128)
    assert (plan.parts > 1) == (parts > 1)
    assert plan.part_tokens * plan.parts >= max(lengths)
    p.check_attend(counts, heads, q=q, kernel=kernel)


# --------------------------------------------------------------- large tiles

def test_tiles_of_many_sequences(uh, gpu):
    rs = np.random.default_rng(3)
    counts = [int(n) for n in rs.integers(0, 60, 70)]
    counts[5], counts[69] = 0, 200
    lengths = [n + int(m) for n, m in zip(counts, rs.integers(0, 40, 70))]
    p = Pair(uh, gpu, lengths, heads=1, bt=32, dim=64, seed=4, spare=WIDE // 32)
    p.fill()
    p.check_attend(counts, 4, kernel=uh.KV_KERNEL_MANY_ROWS, accumulate=True)


@pytest.mark.parametrize("counts", [[1, 300, 0, 129, 40], [300, 1], [0, 0, 500], [128, 128]])
def test_tiles_of_ragged_prompts(uh, gpu, counts):
    lengths = [n + 7 * i for i, n in enumerate(counts)]
    p = Pair(uh, gpu, lengths, heads=8, seed=5, spare=WIDE // 64)
    p.fill()
    p.check_attend(counts, 16, kernel=uh.KV_KERNEL_MANY_ROWS, accumulate=True)


@pytest.mark.parametrize("case", [
    lambda *g: T4.test_ragged_rows(*g, 128, 8, 2, 0, True),
    lambda *g: T4.test_ragged_rows(*g, 64, 7, 1, 0, False),
    lambda *g: T4.test_prompts_and_chunks(*g, 700, 700, 128, 8, 2, 0),
    lambda *g: T4.test_prompts_and_chunks(*g, 1500, 130, 64, 14, 2, 0),
    lambda *g: T4.test_values_of_very_different_scales(*g, 200),
    lambda *g: T4.test_nan_and_infinity_stay_with_the_rows_that_see_them(*g, 100),
    lambda *g: T4.test_stale_tokens_are_not_seen(*g),
    lambda *g: T4.test_blocks_out_of_the_pool_are_not_seen(*g),
    lambda *g: T4.test_query_and_output_strides(*g, 150),
    lambda *g: T4.test_repeated_calls_give_the_same_bits(*g),
    lambda *g: T4.test_other_streams_and_workspaces(*g)])
def test_with_wide_tables(uh, gpu, monkeypatch, case):
    """Tests of small tiles with tables that the large ones are chosen for."""
    init, attend, kernels = Pair.__init__, uh.KvCache.attend, set()

    def wide(self, uh, gpu, lengths, bt=64, spare=0, **kw):
        # 64 parts of small tiles at least: more than run at once.
        init(self, uh, gpu, lengths, bt=bt, spare=spare + 64 * 64, **kw)

    def watched(self, q, lengths, tables, out=None, lse=None, workspace=None, **kw):
        kernels.add(self.attend_plan(q, lengths, tables, **kw).kernel)
        return attend(self, q, lengths, tables, out=out, lse=lse, workspace=workspace, **kw)

    monkeypatch.setattr(Pair, "__init__", wide)
    monkeypatch.setattr(uh.KvCache, "attend", watched)
    case(uh, gpu)
    assert uh.KV_KERNEL_MANY_ROWS in kernels


@pytest.mark.parametrize("dim,group,rows", [(128, 4, 520), (64, 7, 300), (128, 1, 2100)])
@pytest.mark.parametrize("window", [0, 1, 17, 300])
def test_windows_of_large_tiles(uh, gpu, dim, group, rows, window):
    p = Pair(uh, gpu, [rows + 90, 80], heads=8, dim=dim, bt=32, seed=window)
    p.fill()
    p.check_attend([rows, 1], 8 * group, window=window, accumulate=True,
                   kernel=uh.KV_KERNEL_MANY_ROWS)


def test_large_scores_of_large_tiles(uh, gpu):
    """Maxima that grow all along, scores of both signs, scales of all kinds."""
    p = Pair(uh, gpu, [900], heads=8, seed=12, spare=WIDE // 64)
    ramp = torch.arange(900, device=gpu).view(900, 1, 1) / 60
    p.append([900], k=p.random(900, 8).float().mul(ramp).bfloat16())
    for scale in (None, 1.0, -0.3, 0.0, 1e-30, 50.0):
        p.check_attend([150], 32, scale=scale, kernel=uh.KV_KERNEL_MANY_ROWS)


@pytest.mark.parametrize("nan", [False, True])
def test_long_prompt_of_small_blocks(uh, gpu, nan):
    """A prompt whose tiles walk through more blocks than a workgroup holds,
    against the same tokens in larger blocks: stored values are equal, and what
    is made of them too."""
    n, rows = 40064, 12800
    g = torch.Generator(device=gpu).manual_seed(5)
    k, v = (torch.randn((n, 1, 64), generator=g, device=gpu).bfloat16() for _ in range(2))
    q = torch.randn((rows, 4, 64), generator=g, device=gpu).bfloat16()
    if nan:
        v[n - 10, 0, 7] = float("nan")
    length = torch.tensor([n], dtype=torch.int32, device=gpu)
    got = []
    for bt in (128, 32):
        c = uh.KvCache(-(-n // bt), 1, 64, block_tokens=bt, track_weights=True, bits=4)
        table = torch.randperm(-(-n // bt), generator=g, device=gpu).int().view(1, -1)
        c.append(k, v, length, table)
        p = c.attend_plan(q, length, table)
        assert p.kernel == uh.KV_KERNEL_MANY_ROWS and p.parts == 2 and p.part_tokens > 512 * 32
        lse = torch.empty((rows, 4), device=gpu)
        got.append((*c.gather(length, table, n),
                    c.attend(q, length, table, lse=lse, accumulate=True), lse,
                    c.gather_weights(length, table, n)))
    for a, b in zip(*got):
        assert torch.equal(a.isnan(), b.isnan())
        assert torch.equal(a.nan_to_num(), b.nan_to_num())
    out = got[1][2]
    assert out[:-10].isfinite().all() and bool(out[-10:].isnan().all()) == nan


# ------------------------------------------------------------- shared scratch

def test_graphs_and_calls_that_share_a_workspace(uh, gpu):
    """Two captured calls of different splits on one stream, replayed in turn
    with eager ones between them."""
    p = Pair(uh, gpu, [6000, 300], heads=2, bt=64, seed=21)
    p.fill()
    table, lens = p.dev(p.tables), p.dev(p.lengths)
    qs = [p.random(n, 8) for n in (2, 300)]
    starts = [p.starts(c) for c in ([1, 1], [200, 100])]
    outs = [torch.empty_like(q) for q in qs]

    def run(i):
        return p.cache.attend(qs[i], lens, table, starts=starts[i], out=outs[i])

    want = [run(i).clone() for i in (0, 1)]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        run(0), run(1)                          # the stream's workspace, outside of a capture
    stream.synchronize()
    graphs = []
    for i in (0, 1):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            run(i)
        graphs.append(g)
    for _ in range(3):
        for i in (0, 1):
            outs[i].zero_()
            with torch.cuda.stream(stream):
                stream.wait_stream(torch.cuda.default_stream())
                graphs[i].replay()
                run(1 - i)
            torch.cuda.synchronize()
            assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
            torch.randn(1 << 16, device=gpu).sum()
