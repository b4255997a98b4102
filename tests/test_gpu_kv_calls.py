"""The key/value cache's entry points on a live handle: what they refuse, the
kernels that calls of different sizes take, lengths that the tests of the
numerics do not reach, and the decode stack that runs them together."""
import ctypes
import math

import numpy as np
import pytest
import torch

from kv_reference import encode, exponent
import test_gpu_kv_cache as T
from test_gpu_kv_cache import Pair, f64

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ refusals

class Calls:
    """A tracking and a plain cache of 8 blocks of 64 tokens, 2 heads of 128,
    and descriptors of valid calls on them: 2 sequences of 3 blocks."""

    def __init__(self, uh, gpu):
        self.uh = uh
        self.track = uh.KvCache(8, 2, 128, track_weights=True)
        self.plain = uh.KvCache(8, 2, 128)
        self.mem = torch.zeros(1 << 20, dtype=torch.uint8, device=gpu)
        self.seqs = dict(batch=2, rows=4, tables=self.at(0), table_stride=3, max_blocks=3,
                         lengths=self.at(1), starts=0)

    def at(self, slot):
        return self.mem.data_ptr() + slot * 65536

    def call(self, name, cache="track", seqs=None, reserved=0, **over):
        uh = self.uh
        cls = {"append": uh.KvAppendDesc, "gather": uh.KvGatherDesc, "attend": uh.KvAttendDesc,
               "attend_plan": uh.KvAttendDesc, "evict": uh.KvEvictDesc}[name]
        fields = {"append": dict(k=self.at(2), v=self.at(3)),
                  "gather": dict(k=self.at(2), v=self.at(3)),
                  "attend": dict(q=self.at(2), out=self.at(4), heads=8, scale=1.0),
                  "evict": dict(new_tables=self.at(5), new_lengths=self.at(6),
                                kept=self.at(7), keep=64)}[name.replace("_plan", "")]
        rows = dict(rows=0) if name == "evict" else {}
        d = uh.new(cls, cache=getattr(self, cache).handle,
                   seqs=uh.KvSequences(**{**self.seqs, **rows, **(seqs or {})}),
                   **{**fields, **over})
        d.reserved[3] = reserved
        s = uh._Sink()
        fn = getattr(uh.lib(), "ullm_kv_cache_" + name)
        args = (ctypes.byref(uh.new(uh.KvAttendPlan)),) if name == "attend_plan" else ()
        st = uh.Status(fn(ctypes.byref(d), *args, s.ref))
        return st.name, s.text()


@pytest.fixture(scope="module")
def calls(uh, gpu):
    return Calls(uh, gpu)


ANY = [
    ({"reserved": 1}, "RESERVED_NONZERO", "reserved"),
    ({"seqs": {"batch": 65536, "rows": 0}}, "UNSUPPORTED", "65535"),
    ({"seqs": {"max_blocks": 1 << 25, "table_stride": 0}}, "UNSUPPORTED", "max_blocks"),
    ({"seqs": {"table_stride": 2}}, "INVALID_ARGUMENT", "table_stride"),
    ({"seqs": {"max_blocks": 0}}, "INVALID_ARGUMENT", "max_blocks"),
    ({"seqs": {"tables": 0}}, "INVALID_ARGUMENT", "tables"),
    ({"seqs": {"lengths": 0}}, "INVALID_ARGUMENT", "lengths")]
ROWS = [
    ({"seqs": {"rows": 5}}, "INVALID_ARGUMENT", "multiple of batch"),
    ({"seqs": {"rows": 1 << 31}}, "UNSUPPORTED", "rows")]
REFUSED = [(n, *c) for n in ("append", "gather", "attend", "attend_plan") for c in ANY + ROWS] + \
    [("evict", *c) for c in ANY] + [
    ("append", {"k": 0}, "INVALID_ARGUMENT", "null"),
    ("append", {"v": 0}, "INVALID_ARGUMENT", "null"),
    ("append", {"k_row_stride": 127}, "INVALID_ARGUMENT", "stride"),
    ("append", {"v_head_stride": 64}, "INVALID_ARGUMENT", "stride"),
    ("append", {"cache": "plain", "weights": 4096}, "INVALID_ARGUMENT", "track"),
    ("gather", {"k": 0, "v": 0}, "INVALID_ARGUMENT", "null"),
    ("gather", {"k": 4104}, "INVALID_ARGUMENT", "aligned"),
    ("gather", {"cache": "plain", "weights": 4096}, "INVALID_ARGUMENT", "track"),
    ("attend", {"heads": 0}, "INVALID_ARGUMENT", "heads"),
    ("attend", {"heads": 7}, "INVALID_ARGUMENT", "heads"),
    ("attend", {"flags": 2}, "INVALID_ARGUMENT", "flags"),
    ("attend", {"flags": 1, "cache": "plain"}, "INVALID_ARGUMENT", "track"),
    ("attend", {"scale": math.inf}, "INVALID_ARGUMENT", "finite"),
    ("attend", {"scale": math.nan}, "INVALID_ARGUMENT", "finite"),
    ("attend", {"q_row_stride": 64}, "INVALID_ARGUMENT", "stride"),
    ("attend", {"out_head_stride": 64}, "INVALID_ARGUMENT", "stride"),
    ("attend", {"out_row_stride": 256}, "INVALID_ARGUMENT", "overlap"),
    ("attend", {"q": 0}, "INVALID_ARGUMENT", "null"),
    ("attend", {"out": 0}, "INVALID_ARGUMENT", "null"),
    ("attend_plan", {"heads": 7}, "INVALID_ARGUMENT", "heads"),
    ("evict", {"seqs": {"rows": 2}}, "INVALID_ARGUMENT", "no rows"),
    ("evict", {"seqs": {"starts": 4096}}, "INVALID_ARGUMENT", "no rows"),
    ("evict", {"cache": "plain"}, "INVALID_ARGUMENT", "track"),
    ("evict", {"keep": 0}, "INVALID_ARGUMENT", "keep"),
    ("evict", {"keep": 1 << 31}, "UNSUPPORTED", "keep"),
    ("evict", {"sink": 65}, "INVALID_ARGUMENT", "sink"),
    ("evict", {"sink": 32, "recent": 33}, "INVALID_ARGUMENT", "sink"),
    ("evict", {"sink": 1 << 63, "recent": 1 << 63}, "INVALID_ARGUMENT", "sink"),
    ("evict", {"keep": 129, "new_table_stride": 2}, "INVALID_ARGUMENT", "new_table_stride"),
    ("evict", {"new_tables": 0}, "INVALID_ARGUMENT", "null"),
    ("evict", {"new_lengths": 0}, "INVALID_ARGUMENT", "null"),
    ("evict", {"kept": 0}, "INVALID_ARGUMENT", "null")]


@pytest.mark.parametrize("name,over,status,word", REFUSED)
def test_refusals(calls, name, over, status, word):
    """Before any launch: pointers that a call would read are never followed."""
    st, text = calls.call(name, **over)
    assert st == status and word in text, (st, text)


def test_attend_refuses_more_tiles_than_a_launch_has(calls, uh):
    """2^31 - 1 rows of one head: 2^24 tiles of 128, by the checks on the host
    alone (the pointers name a megabyte)."""
    one = uh.KvCache(4, 1, 128)
    d = uh.new(uh.KvAttendDesc, cache=one.handle, q=calls.at(2), out=calls.at(4), heads=1,
               scale=1.0, seqs=uh.KvSequences(batch=1, rows=2 ** 31 - 1, tables=calls.at(0),
                                              max_blocks=1, lengths=calls.at(1)))
    s = uh._Sink()
    st = uh.Status(uh.lib().ullm_kv_cache_attend(ctypes.byref(d), s.ref))
    assert st == uh.Status.UNSUPPORTED and "tiles" in s.text()


def test_evict_refuses_its_own_tables(calls):
    for over in ({"new_tables": calls.at(0)}, {"new_lengths": calls.at(1)}):
        st, text = calls.call("evict", **over)
        assert st == "INVALID_ARGUMENT" and "old ones" in text


def test_attend_checks_its_workspace(calls, uh, gpu):
    c = uh.KvCache(64, 2, 128, track_weights=True)
    q = torch.zeros((1, 8, 128), dtype=torch.bfloat16, device=gpu)
    n = torch.tensor([4000], dtype=torch.int32, device=gpu)
    t = torch.arange(64, dtype=torch.int32, device=gpu).view(1, 64)
    need = c.attend_plan(q, n, t).workspace_bytes
    assert need > 0
    ws = torch.zeros(need + 32, dtype=torch.uint8, device=gpu)
    with pytest.raises(uh.HipError, match="workspace needs"):
        c.attend(q, n, t, workspace=ws[:need - 16])
    with pytest.raises(uh.HipError, match="aligned"):
        c.attend(q, n, t, workspace=ws[8:])
    assert not c.attend(q, n, t, workspace=ws[:need]).any()


def test_calls_without_work(calls, uh, gpu):
    for name in ("append", "gather", "attend", "attend_plan"):
        for seqs in ({"rows": 0}, {"batch": 0, "rows": 0}):
            assert calls.call(name, seqs=seqs)[0] == "OK"
    assert calls.call("evict", seqs={"batch": 0})[0] == "OK"
    calls.track.destroy()
    assert calls.call("attend", cache="plain")[0] == "OK"     # lengths of 0: zeros
    torch.cuda.synchronize()


# --------------------------------------------------------------------- plans

WIDE = 4160  # tokens of tables that the large tiles are chosen for


@pytest.mark.parametrize("counts,heads,lengths,few,parts", [
    ([1], 8, [333], True, 1),
    ([1], 8, [5000], True, 2),
    ([16], 8, [5000], True, 2),              # 64 rows for each sequence and head
    ([17], 8, [5000], False, 2),
    ([150, 12], 8, [400, 90], True, 1),      # few tokens
    ([150], 8, [5000], False, 2),
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


def test_tiles_of_many_sequences(uh, gpu):
    """More sequences than a wave has lanes, some without rows, in tiles of
    128 rows."""
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
    p = Pair(uh, gpu, lengths, heads=2, seed=5, spare=WIDE // 64)
    p.fill()
    p.check_attend(counts, 4, kernel=uh.KV_KERNEL_MANY_ROWS, accumulate=True)


@pytest.mark.parametrize("case", [
    lambda *g: T.test_ragged_rows(*g, 128, 8, 2, 0, True),
    lambda *g: T.test_ragged_rows(*g, 64, 7, 1, 0, False),
    lambda *g: T.test_prompts_and_chunks(*g, 700, 700, 128, 8, 2, 0),
    lambda *g: T.test_prompts_and_chunks(*g, 1500, 130, 64, 14, 2, 0),
    lambda *g: T.test_values_of_very_different_blocks(*g),
    lambda *g: T.test_nan_and_infinity_stay_with_the_rows_that_see_them(*g, 100),
    lambda *g: T.test_stale_tokens_are_not_seen(*g),
    lambda *g: T.test_blocks_out_of_the_pool_are_not_seen(*g),
    lambda *g: T.test_query_and_output_strides(*g, 150),
    lambda *g: T.test_repeated_calls_give_the_same_bits(*g),
    lambda *g: T.test_other_streams_and_workspaces(*g)])
def test_with_wide_tables(uh, gpu, monkeypatch, case):
    """Tests of small tiles with tables that the large ones are chosen for."""
    init, attend, kernels = Pair.__init__, uh.KvCache.attend, set()

    def wide(self, uh, gpu, lengths, bt=64, spare=0, **kw):
        init(self, uh, gpu, lengths, bt=bt, spare=spare + WIDE // bt, **kw)

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
    p = Pair(uh, gpu, [900], heads=2, seed=12, spare=WIDE // 64)
    ramp = torch.arange(900, device=gpu).view(900, 1, 1) / 60
    p.append([900], k=p.random(900, 2).float().mul(ramp).bfloat16())
    for scale in (None, 1.0, -0.3, 0.0, 1e-30, 50.0):
        p.check_attend([120], 8, scale=scale, kernel=uh.KV_KERNEL_MANY_ROWS)


@pytest.mark.parametrize("nan", [False, True])
def test_long_prompt_of_small_blocks(uh, gpu, nan):
    """A prompt whose tiles walk through more blocks than a workgroup holds,
    against the same values in larger blocks: the stored values are equal
    (read back from the larger blocks, whose exponents reach further), the
    products and sums too, up to powers of two."""
    n, rows = 40064, 12800
    g = torch.Generator(device=gpu).manual_seed(5)
    k, v = (torch.randn((n, 1, 64), generator=g, device=gpu).bfloat16() for _ in range(2))
    q = torch.randn((rows, 4, 64), generator=g, device=gpu).bfloat16()
    if nan:
        v[n - 10, 0, 7] = float("nan")
    length = torch.tensor([n], dtype=torch.int32, device=gpu)
    got = []
    for bt in (128, 32):
        c = uh.KvCache(-(-n // bt), 1, 64, block_tokens=bt, track_weights=True)
        table = torch.randperm(-(-n // bt), generator=g, device=gpu).int().view(1, -1)
        c.append(k, v, length, table)
        k, v = c.gather(length, table, n)
        p = c.attend_plan(q, length, table)
        assert p.kernel == uh.KV_KERNEL_MANY_ROWS and p.parts == 2 and p.part_tokens > 512 * 32
        lse = torch.empty((rows, 4), device=gpu)
        got.append((c.attend(q, length, table, lse=lse, accumulate=True), lse,
                    c.gather_weights(length, table, n)))
    for a, b in zip(*got):
        assert torch.equal(a.isnan(), b.isnan())
        assert torch.equal(a.nan_to_num(), b.nan_to_num())
    out = got[1][0]
    assert out[:-10].isfinite().all()
    assert bool(out[-10:, :, 7].isnan().all()) == nan and out[-10:, :, :7].isfinite().all()


@pytest.mark.parametrize("n,keep", [(9000, 700), (40000, 2500)])
def test_evict_long_sequences(uh, gpu, n, keep):
    """More tokens than a thread holds keys of, and than a workgroup does."""
    p = Pair(uh, gpu, [n, n - 4321], heads=2, bt=128, dim=64, seed=6)
    rows = sum(p.lengths)
    w = np.exp(3 * p.rs.standard_normal((rows, 2))).astype(np.float32)
    w[::7] = w[3]                                   # ties across waves and spans
    p.append(p.lengths, weights=w)
    cols = -(-keep // 128)
    new = np.arange(2 * cols, dtype=np.int32).reshape(2, cols)
    # The new blocks must not be the old ones: a cache of their own side.
    big = uh.KvCache(p.blocks + 2 * cols, 2, 64, block_tokens=128, track_weights=True)
    k, v = p.cache.gather(p.dev(p.lengths), p.dev(p.tables), rows, starts=p.starts(p.lengths))
    big.append(k, v, p.dev(p.lengths), p.dev(p.tables + 2 * cols), starts=p.starts(p.lengths),
               weights=p.dev(w, torch.float32))
    lens, kept = big.evict(p.dev(p.lengths), p.dev(p.tables + 2 * cols), p.dev(new), keep,
                           sink=4, recent=30)
    assert lens.tolist() == [keep, keep]
    start = 0
    for b, m in enumerate(p.lengths):
        for h in range(2):
            x = w[start:start + m, h]
            middle = sorted(range(4, m - 30), key=lambda t: (-x[t], t))[:keep - 34]
            want = list(range(4)) + sorted(middle) + list(range(m - 30, m))
            assert kept[b, h].tolist() == want
        start += m
    gk, gv = big.gather(lens, p.dev(new), 2 * keep)
    for b in range(2):
        for h in range(2):
            at = kept[b, h].long() + sum(p.lengths[:b])
            for x, got in ((k, gk), (v, gv)):
                got = f64(got[b * keep:(b + 1) * keep, h])
                for j in range(0, keep, 128):   # as if appended to the new block
                    moved = f64(x[at[j:j + 128], h])
                    assert np.array_equal(got[j:j + 128], encode(moved, exponent(moved)))


# ------------------------------------------------------------- decode stack

def small_stack(uh, gpu, **more):
    import stack
    return stack.DecodeStack(uh, torch, gpu, batch=3, layers=2, hidden=512, qkv=768, ffn=1024,
                             vocab=1000, seed=3, **more)


def chain(st, x, starts, caches, lengths, accumulate):
    """The stack's layers written out: logits of every row, last attention."""
    rows = x.shape[0]
    for ws, cache in zip(st.weights, caches):
        qkv = ws["qkv"].forward(x, alpha=st.alpha_h)
        q, k, v = (t.reshape(rows, -1, 128) for t in (qkv[:, :512], qkv[:, 512:640],
                                                      qkv[:, 640:]))
        cache.append(k, v, lengths, st.tables, starts=starts)
        a = cache.attend(q, lengths, st.tables, starts=starts, scale=1.0, accumulate=accumulate)
        o = ws["o"].forward(a.view(rows, 512), alpha=st.alpha_h)
        up = ws["gate_up"].forward(o, alpha=st.alpha_h)
        x = ws["down"].forward(up[:, :1024].contiguous(), alpha=st.alpha_f)
    return x, (q, k, v, a)


def test_stack_attends_over_its_cache(uh, gpu):
    st = small_stack(uh, gpu, context=400, evict_to=130)
    other = [uh.KvCache(c.blocks, 1, 128, track_weights=True) for c in st.caches]
    g = torch.Generator(device=gpu).manual_seed(1)
    counts = [200, 1, 97]
    h = torch.randn((298, 512), generator=g, device=gpu).bfloat16()
    logits = st.prompt(h, counts).clone()
    assert st.lengths.tolist() == counts
    starts = torch.tensor([0, 200, 201, 298], dtype=torch.int32, device=gpu)
    x, _ = chain(st, h, starts, other, st.lengths, True)
    last = x[[199, 200, 297]].contiguous()
    assert torch.equal(logits, st.lm_head.forward(last, alpha=st.alpha_h))
    assert torch.isfinite(logits.float()).all()
    assert 0.2 < float(x.float().pow(2).mean().sqrt()) < 5.0

    for step in range(3):
        st.h0.copy_(torch.randn((3, 512), generator=g, device=gpu))
        logits = st.step().clone()
        x, (q, _, _, a) = chain(st, st.h0, None, other, st.lengths, True)
        assert torch.equal(logits, st.lm_head.forward(x, alpha=st.alpha_h))
        assert torch.equal(a.view(3, 512), st.attn)
    assert st.lengths.tolist() == [n + 3 for n in counts]
    # The last attention against its definition in 64 bits, within f16 weights,
    # a bf16 result and f32 scores of sums of 128 products.
    for b, n in enumerate(st.lengths.tolist()):
        k, v = st.caches[1].gather(st.lengths[b:b + 1], st.tables[b:b + 1], n)
        k, v, qb = f64(k)[:, 0], f64(v)[:, 0], f64(q)[b]
        s = qb @ k.T
        p = np.exp(s - s.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        eps = 2.0 ** -20 * (np.abs(qb) @ np.abs(k).T).max(1, keepdims=True)
        part = (2.0 ** -10 + 2.0 ** -17 + 2 * eps) * (p @ np.abs(v))
        err = np.abs(f64(a)[b] - p @ v) - part - 2.0 ** -8 * (np.abs(p @ v) + part)
        assert err.max() <= 0

    before = [st.caches[1].gather(st.lengths[b:b + 1], st.tables[b:b + 1], n)[0]
              for b, n in enumerate(st.lengths.tolist())]
    old = st.tables.clone()
    st.evict(sink=2, recent=16)
    assert st.lengths.tolist() == [130, 4, 100]
    ids = torch.cat([st.tables.flatten(), st.spare.flatten()])
    assert sorted(ids.tolist()) == list(range(len(ids))) and not torch.equal(old, st.tables)
    k = st.caches[1].gather(st.lengths[:1], st.tables[:1], 130)[0]
    rows = {tuple(r.tolist()) for r in before[0][:, 0].float()}
    assert torch.equal(k[:2], before[0][:2]) and torch.equal(k[-16:], before[0][-16:])
    assert all(tuple(r.tolist()) in rows for r in k[:, 0].float())
    for b in (1, 2):
        n = st.lengths.tolist()[b]
        assert torch.equal(st.caches[1].gather(st.lengths[b:b + 1], st.tables[b:b + 1], n)[0],
                           before[b])
    st.step()
    st.evict(sink=2, recent=16)
    assert torch.isfinite(st.step().float()).all()
    assert st.lengths.tolist() == [131, 6, 102]
    st.destroy()


def test_stack_steps_under_a_graph(uh, gpu):
    a, b = small_stack(uh, gpu, context=300), small_stack(uh, gpu, context=300)
    h = torch.randn((9, 512), device=gpu).bfloat16()
    for st in (a, b):
        st.prompt(h, [2, 3, 4])
        st.h0.copy_(h[:3])
        st.step()                                    # workspaces, outside of the capture
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b.step()
        a.step()
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        a.step()
    for _ in range(70):                              # across the end of a block
        g.replay()
        torch.cuda.synchronize()
        want = b.step()
        torch.cuda.synchronize()
        assert torch.equal(a.logits, want)
    assert torch.equal(a.lengths, b.lengths)
    a.destroy()
    b.destroy()


def test_stack_refuses(uh, gpu):
    plain = small_stack(uh, gpu)
    h = torch.zeros((3, 512), dtype=torch.bfloat16, device=gpu)
    with pytest.raises(ValueError):
        plain.prompt(h, [1, 1, 1])
    with pytest.raises(ValueError):
        plain.evict()
    with pytest.raises(ValueError):
        small_stack(uh, gpu, context=64, evict_to=65)
    st = small_stack(uh, gpu, context=64)
    for counts in ([1, 2], [1, 2, 0], [1, 1, 2]):
        with pytest.raises(ValueError):
            st.prompt(h, counts)
    plain.destroy()
    st.destroy()
