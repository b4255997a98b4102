"""The decode stack with rotary positions, over caches of 8 and of 4 bits: the
rotating append, the attention and the eviction as a model runs them."""
import numpy as np
import pytest
import torch

from kv_attention64 import attention64, within
from test_gpu_kv_calls import small_stack
from test_gpu_kv_cache import f64
from test_gpu_kv_rotary import same_queries

pytestmark = pytest.mark.gpu


def chain(st, x, starts, caches, positions):
    """The stack's layers written out; what the last attention saw and gave."""
    rows, f = x.shape[0], st.inv_freq
    for ws, cache in zip(st.weights, caches):
        qkv = ws["qkv"].forward(x, alpha=st.alpha_h)
        q, k, v = (t.reshape(rows, -1, 128).contiguous()
                   for t in (qkv[:, :512], qkv[:, 512:640], qkv[:, 640:]))
        turned = cache.append_rotary(q, k, v, st.lengths, st.tables, f, starts=starts,
                                     positions=positions)
        a = cache.attend(turned, st.lengths, st.tables, starts=starts, scale=1.0,
                         accumulate=True)
        o = ws["o"].forward(a.view(rows, 512), alpha=st.alpha_h)
        up = ws["gate_up"].forward(o, alpha=st.alpha_h)
        x = ws["down"].forward(up[:, :1024].contiguous(), alpha=st.alpha_f)
    return x, (q, turned, a, f)


@pytest.mark.parametrize("bits", [4, 8])
def test_stack_rotates_and_attends(uh, gpu, bits):
    st = small_stack(uh, gpu, context=400, evict_to=130, kv_bits=bits, rope_base=10000.0)
    assert all(c.bits == bits for c in st.caches)
    # Frequencies: rounded once from 64 bits, whose power is within 2^-50.
    want = 10000.0 ** (-np.arange(64) / 64)
    assert np.abs(f64(st.inv_freq) / want - 1).max() <= 2.0 ** -24 + 2.0 ** -49
    other = [uh.KvCache(c.blocks, 1, 128, track_weights=True, bits=bits) for c in st.caches]
    g = torch.Generator(device=gpu).manual_seed(1)
    counts = [200, 1, 97]
    h = torch.randn((298, 512), generator=g, device=gpu).bfloat16()
    logits = st.prompt(h, counts).clone()
    starts = torch.tensor([0, 200, 201, 298], dtype=torch.int32, device=gpu)
    x, _ = chain(st, h, starts, other, None)          # places are the positions yet
    last = x[[199, 200, 297]].contiguous()
    assert torch.equal(logits, st.lm_head.forward(last, alpha=st.alpha_h))
    assert torch.isfinite(logits.float()).all()
    assert 0.2 < float(x.float().pow(2).mean().sqrt()) < 5.0

    given = np.array(counts)
    for step in range(6):
        if step == 3:
            st.evict(sink=2, recent=16)
            for c in other:                           # on the old tables, before they are swapped
                c.destroy()
            other = [uh.KvCache(c.blocks, 1, 128, track_weights=True, bits=bits)
                     for c in st.caches]
            rows = int(st.lengths.sum())
            counts = st.lengths.tolist()
            at = torch.tensor([0, *np.cumsum(counts)], dtype=torch.int32, device=gpu)
            for c, mine in zip(other, st.caches):
                k, v = mine.gather(st.lengths, st.tables, rows, starts=at)
                c.append(k, v, st.lengths, st.tables, starts=at,
                         weights=mine.gather_weights(st.lengths, st.tables, rows, starts=at))
            assert counts == [130, 4, 100]
        st.h0.copy_(torch.randn((3, 512), generator=g, device=gpu))
        logits = st.step().clone()
        positions = torch.tensor(given, dtype=torch.int32, device=gpu)
        given = given + 1
        x, (q, turned, a, f) = chain(st, st.h0, None, other, positions)
        if bits == 4 or step < 3:
            assert torch.equal(logits, st.lm_head.forward(x, alpha=st.alpha_h))
            assert torch.equal(a.view(3, 512), st.attn)
        assert same_queries(turned, q, f64(positions)[None], f)
        # The last attention against its definition in 64 bits.
        for b, n in enumerate(st.lengths.tolist()):
            k, v = other[1].gather(st.lengths[b:b + 1], st.tables[b:b + 1], n)
            ref, tol, _, _, _, _ = attention64(turned[b:b + 1], k, v,
                                               torch.tensor([n - 1], device=gpu), 1.0, 0)
            within(a[b:b + 1], ref, tol, "out")
    assert st.lengths.tolist() == [133, 7, 103] and st.given.tolist() == [206, 7, 103]

    # A prompt goes on from where its sequence is.
    h = torch.randn((4, 512), generator=g, device=gpu).bfloat16()
    logits = st.prompt(h, [2, 1, 1]).clone()
    starts = torch.tensor([0, 2, 3, 4], dtype=torch.int32, device=gpu)
    positions = torch.tensor([206, 207, 7, 103], dtype=torch.int32, device=gpu)
    x, _ = chain(st, h, starts, other, positions)
    if bits == 4:
        assert torch.equal(logits, st.lm_head.forward(x[[1, 2, 3]].contiguous(),
                                                      alpha=st.alpha_h))
    st.destroy()


@pytest.mark.parametrize("bits", [4, 8])
def test_stack_steps_under_a_graph(uh, gpu, bits):
    a, b = (small_stack(uh, gpu, context=300, kv_bits=bits, rope_base=500000.0) for _ in range(2))
    h = torch.randn((9, 512), device=gpu).bfloat16()
    for st in (a, b):
        st.prompt(h, [2, 3, 4])
        st.h0.copy_(h[:3])
        st.step()
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
        a.replayed()
        g.replay()
        torch.cuda.synchronize()
        want = b.step()
        torch.cuda.synchronize()
        assert torch.equal(a.logits, want)
    assert a.given.tolist() == b.given.tolist() == [74, 75, 76]
    for st in (a, b):
        st.destroy()


def test_positions_change_what_is_attended(uh, gpu):
    """The same rows without a rotation give other logits; a single token, which
    sees itself alone, the same."""
    a, b = (small_stack(uh, gpu, context=64, rope_base=r) for r in (0.0, 10000.0))
    h = torch.randn((42, 512), device=gpu).bfloat16()
    one, two = (st.prompt(h, [40, 1, 1]).clone() for st in (a, b))
    assert torch.equal(one[1:], two[1:]) and not torch.equal(one[0], two[0])
    for st in (a, b):
        st.destroy()


@pytest.mark.parametrize("over", [{"rope_base": -1.0, "context": 64}, {"rope_base": 10000.0},
                                  {"kv_bits": 4}, {"kv_bits": 5, "context": 64}])
def test_stack_refuses(uh, gpu, over):
    with pytest.raises(ValueError, match="rope_base|bits"):
        small_stack(uh, gpu, **over)
