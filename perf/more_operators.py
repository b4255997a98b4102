"""Workloads of a 4-bit key/value cache and of rotary positions, as a program that serves a model calls them.

Two operators.  ``attend`` is softmax attention over a paged cache that holds
keys and values in 4 bits (E2M1 codes; a power of two for each 32 dims of a
key, one scale for each value).  ``append`` rotates the queries and keys of new
tokens by their positions (one axis, or several as for images) and stores keys
and values in a cache of 4 or 8 bits, whose blocks a table assigns to each
sequence.  Head layouts are the Llama-3-8B ones of ``stack.py`` (32 query heads
and 8 key/value heads of 128) and generic ones.

``own = False`` computes an operator in elementary torch operations on pools of
codes; ``own = True`` calls the framework's cache.
"""
import json
import math
import random
import sys
from pathlib import Path

import torch

own = False

DEV = torch.device("cuda:0")
LARGEST_CACHE = 131072 * 8 * 128    # tokens x heads x dim of the largest listed cache
LARGEST_PAIRS = 32 * 128 * (4096 * 4097 // 2 + 3001 * 3002 // 2)   # of the largest prompt
LARGEST_APPEND = 16000 * 40 * 128   # new tokens x query and key heads x dim


# op:       "attend" or "append"
# bits:     of the cache's codes
# heads, kv_heads, dim: query heads, key/value heads, head dimension
# block:    tokens of a cache block
# batch:    sequences; length: tokens of the longest, with the new ones
# rows:     new tokens (queries) of a sequence, at most; -1: all its tokens
# ragged:   lengths, and row counts above one, differ from sequence to sequence
# idle:     the last slot of the batch holds no sequence (length 0)
# window:   a query sees that many tokens (0: all up to its own)
# track:    attend adds the weights that tokens receive to the cache's
# rotary:   dims that are rotated (0: none), the first of each head
# pairs:    "halves" rotates dims j and j + rotary / 2, "neighbours" 2j and 2j + 1
# base:     frequencies are base ** (-2j / rotary)
# axes:     axes of a position; 3: time, height and width, images between text
# far:      position of a sequence's first cached token


def _attend(name, heads, kv_heads, dim, block, batch, length, rows, ragged=False,
            idle=False, window=0, track=False):
    return _named(name, {"op": "attend", "bits": 4, "heads": heads, "kv_heads": kv_heads,
                         "dim": dim, "block": block, "batch": batch, "length": length,
                         "rows": rows, "ragged": ragged, "idle": idle, "window": window,
                         "track": track})


def _append(name, bits, heads, kv_heads, dim, block, batch, length, rows, ragged=False,
            idle=False, rotary=0, pairs="halves", base=500000.0, axes=1, far=0):
    return _named(name, {"op": "append", "bits": bits, "heads": heads, "kv_heads": kv_heads,
                         "dim": dim, "block": block, "batch": batch, "length": length,
                         "rows": rows, "ragged": ragged, "idle": idle, "rotary": rotary,
                         "pairs": pairs, "base": base, "axes": axes, "far": far})


def _named(name, case):
    return dict(case, name=name) if name else case


def listed():
    return [
        # One sequence decoding, early in its answer: the smallest launch of a layer.
        _attend("decode1_len333", 32, 8, 128, 64, 1, 333, 1),
        # A continuous batch of 16 slots, one of them free, ragged to 8192 tokens.
        _attend("decode16_ragged_8k", 32, 8, 128, 64, 16, 8192, 1, ragged=True, idle=True),
        # One sequence decoding over a long document.
        _attend("decode1_len131072", 32, 8, 128, 128, 1, 131072, 1),
        # A few proposed tokens checked at once, in a small model with heads of 64, 7
        # query heads to a key/value head and a sliding window.
        _attend("verify6_window_dim64", 28, 4, 64, 32, 24, 3001, 6, ragged=True, window=1024),
        # Two prompts of different lengths.
        _attend("prompt_4096_3001", 32, 8, 128, 64, 2, 4096, -1, ragged=True),
        # A chunk of a long prompt over what is cached already, tracking weights.
        _attend("chunk509_track_16k", 32, 8, 128, 64, 1, 15873, 509, track=True),
        # A decode batch rotates and stores a token each, somewhere inside their blocks.
        _append("rotate_decode64_4bit", 4, 32, 8, 128, 64, 64, 2048, 1, ragged=True, idle=True,
                rotary=128),
        # The same into an 8-bit cache, the sequences far into a conversation of which the
        # cache holds the last tokens.
        _append("rotate_decode16_8bit_far", 8, 32, 8, 128, 64, 16, 1501, 1, ragged=True,
                rotary=128, far=1000000),
        # Prompts on their way from the projections into a 4-bit and an 8-bit cache.
        _append("rotate_prompts_4bit", 4, 32, 8, 128, 64, 4, 4096, -1, ragged=True, rotary=128),
        _append("rotate_prompts_8bit", 8, 32, 8, 128, 64, 4, 4096, -1, ragged=True, rotary=128),
        # Prompts with images: positions of three axes, half of a head rotated, pairs of
        # neighbours, heads of 64.
        _append("rotate_images_dim64", 4, 28, 4, 64, 32, 3, 2777, -1, ragged=True, rotary=32,
                pairs="neighbours", base=10000.0, axes=3),
        # Chunks of prompts that need no rotation, behind what is cached already.
        _append("store_chunks_4bit", 4, 0, 8, 128, 128, 8, 5000, 1013, ragged=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attend"] * 6 + ["append"] * 6)
    heads, kv_heads, dim = rng.choice([(32, 8, 128), (32, 8, 128), (28, 4, 64), (8, 8, 128),
                                       (16, 1, 128), (40, 8, 128), (14, 2, 64)])
    block = rng.choice([32, 64, 128])
    batch = _log(rng, 1, 48)
    ragged = rng.random() < 0.6
    idle = ragged and rng.random() < 0.3
    if op == "append":
        if rng.random() < 0.5:
            length, rows = _log(rng, 1, 4096), rng.choice([1, 1, rng.randint(2, 8)])
        else:
            length, rows = _log(rng, 16, 4096), rng.choice([-1, _log(rng, 9, 1024)])
        while (batch * length * kv_heads * dim > LARGEST_CACHE // 8 or
               batch * length * (heads + kv_heads) * dim > LARGEST_APPEND):
            batch, length = max(1, batch // 2), max(1, length // 2)
        rotary = rng.choice([dim, dim, dim // 2, 2 * rng.randint(1, dim // 2)])
        bits = rng.choice([4, 4, 8])
        if bits == 4 and rng.random() < 0.2:
            heads, rotary = 0, 0
        return _append(None, bits, heads, kv_heads, dim, block, batch, length, min(rows, length),
                       ragged, idle, rotary, rng.choice(["halves", "halves", "neighbours"]),
                       rng.choice([10000.0, 500000.0, 1000000.0]),
                       rng.choice([1, 1, 3]), rng.choice([0, 0, _log(rng, 10, 1000000)]))
    kind = rng.choice(["decode", "decode", "few", "prompt", "chunk"])
    window = rng.choice([0, 0, 0, rng.randint(1, 2000)])
    track = rng.random() < 0.25
    if kind == "decode":
        length, rows = _log(rng, 1, 131072), 1
    elif kind == "few":
        length, rows = _log(rng, 8, 32768), rng.randint(2, 16)
    elif kind == "prompt":
        length, rows = _log(rng, 2, 4096), -1
    else:
        length = _log(rng, 600, 16384)
        rows = _log(rng, 20, min(1024, length))
    while (batch * length * kv_heads * dim > LARGEST_CACHE // 2 or
           batch * length * (length if rows < 0 else rows) * heads * dim > LARGEST_PAIRS):
        if batch > 1:
            batch //= 2
        else:
            length = max(1, length // 2)
            rows = min(rows, length)
    return _attend(None, heads, kv_heads, dim, block, batch, length, rows, ragged, idle,
                   window, track)


def _layout(case):
    """Lengths and row counts of the sequences: part of the case, not of its data."""
    r = random.Random(json.dumps({k: v for k, v in case.items() if k != "name"}, sort_keys=True))
    batch, length, rows = case["batch"], case["length"], case["rows"]
    if case["op"] == "attend" and (batch, length, rows) == (2, 4096, -1):
        lengths = [4096, 3001]
    else:
        lengths = [length] + [r.randint((length + 1) // 2, length) if case["ragged"] else length
                              for _ in range(batch - 1)]
    if case["idle"] and batch > 1:
        lengths[-1] = 0
    if rows < 0:
        counts = list(lengths)
    elif rows == 1 or not case["ragged"]:
        counts = [rows] * batch
    else:
        counts = [min(r.randint(1, rows), n) for n in lengths]
    return lengths, counts


def _seen(length, count, window):
    """(pairs of a query and a token it sees, tokens that any query sees) of a sequence."""
    first = length - count
    w = window or length
    pairs = sum(min(p + 1, w) for p in range(max(first, 0), length))
    return pairs, length - max(0, max(first, 0) + 1 - w) if length else 0


def _span(length, count, block):
    """First token of the blocks that an append touches."""
    return max(length - count, 0) // block * block


def _token_bytes(case):
    """Bytes of a cached token and head: codes, exponents and scales."""
    d = case["dim"]
    return 2 * d if case["bits"] == 8 else d + d // 32 + 2


def work(case):
    lengths, counts = _layout(case)
    hkv, d = case["kv_heads"], case["dim"]
    token = _token_bytes(case)
    if case["op"] == "attend":
        seen = [_seen(n, c, case["window"]) for n, c in zip(lengths, counts)]
        pairs, tokens = sum(s[0] for s in seen), sum(s[1] for s in seen)
        nbytes = token * hkv * tokens + sum(counts) * case["heads"] * (4 * d + 4)
        if case["track"]:
            nbytes += 8 * hkv * sum(lengths)
        return {"bytes": nbytes, "flops": 4 * d * case["heads"] * pairs}
    new = sum(min(c, n) for n, c in zip(lengths, counts))
    back = sum(n - _span(n, c, case["block"]) for n, c in zip(lengths, counts))
    return {"bytes": hkv * ((4 * d + token) * new + 4 * d * back) + 4 * d * case["heads"] * new,
            "flops": 6 * case["rotary"] * (case["heads"] + hkv) // 2 * new}


# ------------------------------------------------------------------ the codes

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _exponents(amax, top, low, high):
    """Smallest e from low to high with amax <= top * 2^e, top in [1, 2) * 2^n; amax not negative."""
    m, e = torch.frexp(amax.double())
    n = math.frexp(top)
    e = e - n[1] + (m > n[0]).int()
    return torch.where(amax == 0, low, e).clamp(low, high).int()


def _power_of_two(exponents):
    """2^e for whole e, in 64 bits."""
    return ((exponents.long() + 1023) << 52).view(torch.float64)


def _scales(amax):
    """Smallest numbers of 6 significant bits from 2^-19 to 63 * 2^10 whose 6-fold reaches amax, in 64 bits."""
    m, e = torch.frexp(amax.double() / 6)
    return (torch.ceil(m * 64) * _power_of_two(e - 6)).clamp(2.0 ** -19, 63 * 2.0 ** 10)


def _to_e4m3(y):
    """E4M3 codes of values in 64 bits, nearest, ties to even: rounded once, before the conversion."""
    a = y.abs()
    quantum = _power_of_two(torch.frexp(a.clamp_min(2.0 ** -6)).exponent - 4)
    r = (torch.round(a / quantum) * quantum).clamp_max(448)
    return torch.copysign(r, y).float().to(torch.float8_e4m3fn).view(torch.uint8)


def _encode4(y):
    """Values over their scale to E2M1 codes: nearest, ties to even."""
    a = y.abs()
    quantum = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    r = (torch.round(a / quantum) * quantum).clamp_max(6)
    code = torch.where(r < 2, 2 * r, torch.where(r < 4, r + 2, r / 2 + 4)).to(torch.uint8)
    return code + torch.signbit(y).to(torch.uint8) * 8


def _pack(codes):
    return codes[..., 0::2] | codes[..., 1::2] << 4


def _decode4(packed, dtype=torch.float32):
    """E2M1 values of packed codes, [..., dim]."""
    table = torch.tensor(E2M1 + tuple(-x for x in E2M1), dtype=dtype, device=DEV)
    both = torch.stack((packed & 15, packed >> 4), -1).flatten(-2)
    return table[both.int()]


def _keys4(x):
    """Packed codes and exponents of keys [..., dim]."""
    g = x.unflatten(-1, (-1, 32))
    e = _exponents(g.abs().amax(-1), 6.0, -100, 119)
    return _pack(_encode4((g.double() / _power_of_two(e)[..., None]).flatten(-2))), e.to(torch.int8)


def _values4(x):
    """Packed codes and scales of values [..., dim]."""
    s = _scales(x.abs().amax(-1))
    return _pack(_encode4(x.double() / s[..., None])), s.half()


def _read_keys(p, at):
    """Keys of 4 bits in f32, at an index of the pool's leading axes."""
    power = _power_of_two(p["ke"][at]).float()
    return (_decode4(p["k"][at]).unflatten(-1, (-1, 32)) * power[..., None]).flatten(-2)


def _read_values(p, at):
    return _decode4(p["v"][at]) * p["ve"][at].float()[..., None]


# ------------------------------------------------------------------ the inputs

def _ids(counts):
    """(sequence, index within it) of every row, for row counts of the sequences."""
    c = torch.tensor(counts, device=DEV)
    seq = torch.repeat_interleave(torch.arange(len(counts), device=DEV), c)
    first = torch.cumsum(c, 0) - c
    return seq, torch.arange(int(sum(counts)), device=DEV) - first[seq]


def _starts(counts):
    """Row offsets of the sequences; None where all have the same number of rows."""
    if len(set(counts)) == 1:
        return None
    return torch.tensor([0] + [sum(counts[:i + 1]) for i in range(len(counts))],
                        dtype=torch.int32, device=DEV)


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _positions(case, lengths, counts):
    """Positions [axes][rows] of the rows; None where they are the tokens' places in the cache."""
    if case["axes"] == 1 and not case["far"]:
        return None
    seq, i = _ids(counts)
    at = (_int32(lengths) - _int32(counts))[seq] + i
    if case["axes"] == 1:
        return (at + case["far"]).int()[None].contiguous()
    # Text of 100 tokens, then an image of 24 x 30 patches, and so on: a patch has the
    # time of the image's start, and its row and column from there.
    period, wide, tall = 100 + 24 * 30, 30, 24
    step, inside = at // period, at % period
    start = case["far"] + step * (100 + wide) + 100
    patch = (inside - 100).clamp_min(0)
    text = start - 100 + inside
    image = torch.stack([start, start + patch // wide % tall, start + patch % wide])
    return torch.where(inside < 100, text[None], image).int().contiguous()


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    lengths, counts = _layout(case)
    op, hkv, d, bt = case["op"], case["kv_heads"], case["dim"], case["block"]
    batch, width = case["batch"], max(1, -(-max(lengths) // bt))
    # Blocks are handed out in no order, as after some hours of serving.
    need = [-(-n // bt) for n in lengths]
    blocks = sum(need) + 3
    order = torch.randperm(blocks, generator=g, device=DEV, dtype=torch.int32)
    tables, at = torch.zeros((batch, width), dtype=torch.int32, device=DEV), 0
    for b, n in enumerate(need):
        tables[b, :n] = order[at:at + n]
        at += n
    # What is cached before the call: all of it, or what an append has before it.
    old = [max(n - c, 0) for n, c in zip(lengths, counts)] if op == "append" else lengths
    total = sum(old)
    seq, pos = _ids(old)
    channel = torch.exp(0.5 * torch.randn((hkv, d), generator=g, device=DEV))
    k = (torch.randn((total, hkv, d), generator=g, device=DEV) * channel).bfloat16()
    v = torch.randn((total, hkv, d), generator=g, device=DEV).bfloat16()
    weights = torch.exp(2 * torch.randn((total, hkv), generator=g, device=DEV))
    block, slot = tables.long()[seq, pos // bt], pos % bt
    # The pool: of 8 bits, codes [block][head][token][dim] and exponents [block][head];
    # of 4 bits, codes [block][head][token][dim / 2] with exponents [..., dim / 32] of keys and scales of
    # values.  Weights [block][head][token].
    p, flat = {"w": torch.zeros((blocks, hkv, bt), device=DEV)}, []
    p["w"][block, :, slot] = weights
    if case["bits"] == 4:
        shape = (blocks, hkv, bt)
        p["k"], p["v"] = (torch.zeros(shape + (d // 2,), dtype=torch.uint8, device=DEV) for _ in "kv")
        p["ke"] = torch.zeros(shape + (d // 32,), dtype=torch.int8, device=DEV)
        p["ve"] = torch.ones(shape, dtype=torch.float16, device=DEV)
        for lo in range(0, total, 16384):      # in pieces: the work is in 64 bits
            part = slice(lo, lo + 16384)
            where = (block[part], slice(None), slot[part])
            p["k"][where], p["ke"][where] = _keys4(k[part])
            p["v"][where], p["ve"][where] = _values4(v[part])
            if own:
                flat.append((_read_keys(p, where).bfloat16(), _read_values(p, where).bfloat16()))
        if own and total:
            flat = [torch.cat([f[i] for f in flat]) for i in (0, 1)]
    else:
        key = (block[:, None] * hkv + torch.arange(hkv, device=DEV)).reshape(-1)
        for name, x in (("k", k), ("v", v)):
            amax = torch.zeros(blocks * hkv, device=DEV)
            amax.scatter_reduce_(0, key, x.float().abs().amax(2).reshape(-1), "amax")
            e = _exponents(amax, 448.0, -100, 119).view(blocks, hkv)
            pool = torch.zeros((blocks, hkv, bt, d), dtype=torch.uint8, device=DEV)
            power = _power_of_two(e[block])[:, :, None]
            codes = _to_e4m3(x / power)
            pool[block, :, slot] = codes
            p[name], p[name + "s"] = pool, e
            flat.append((codes.view(torch.float8_e4m3fn).double() * power).bfloat16())
    s = {"case": case, "pools": p, "tables": tables, "counts": counts, "lengths_list": lengths,
         "lengths": _int32(lengths), "starts": _starts(counts), "whole": _starts(lengths),
         "width": width}
    rows = sum(counts)
    if op == "attend":
        s["q"] = torch.randn((rows, case["heads"], d), generator=g, device=DEV).bfloat16()
        s["scale"] = 1 / math.sqrt(d)
    else:
        s["k"] = (torch.randn((rows, hkv, d), generator=g, device=DEV) * channel).bfloat16()
        s["v"] = torch.randn((rows, hkv, d), generator=g, device=DEV).bfloat16()
        s["span"] = [n - _span(n, c, bt) for n, c in zip(lengths, counts)]
        s["span_starts"] = _starts(s["span"])
    if op == "append" and case["rotary"]:
        half = case["rotary"] // 2
        s["q"] = torch.randn((rows, case["heads"], d), generator=g, device=DEV).bfloat16()
        s["inv_freq"] = torch.tensor([case["base"] ** (-j / half) for j in range(half)],
                                     dtype=torch.float32, device=DEV)
        s["positions"] = _positions(case, lengths, counts)
        # Of three axes the first third of the pairs turns with the time, and so on.
        s["axis"] = None if case["axes"] == 1 else \
            torch.tensor([3 * j // half for j in range(half)], dtype=torch.uint8, device=DEV)
    if own:
        pkg = str(Path(__file__).resolve().parents[1] / "ullm-project_amd")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        import ullm_hip as uh
        s["cache"] = uh.KvCache(blocks, hkv, d, block_tokens=bt, track_weights=True,
                                bits=case["bits"])
        if total:
            s["cache"].append(flat[0], flat[1], _int32(old), tables, starts=_starts(old),
                              weights=weights.contiguous())
        s["pools"] = None
    return s


# ------------------------------------------------------------- the operators

def run(s):
    if s["case"]["op"] == "attend":
        return _own_attend(s) if own else _plain_attend(s)
    return _own_append(s) if own else _plain_append(s)


def _own_attend(s):
    c, cache = s["case"], s["cache"]
    lse = torch.empty(s["q"].shape[:2], dtype=torch.float32, device=DEV)
    out = cache.attend(s["q"], s["lengths"], s["tables"], starts=s["starts"],
                       scale=s["scale"], window=c["window"], accumulate=c["track"], lse=lse)
    if not c["track"]:
        return {"out": out, "lse": lse}
    w = cache.gather_weights(s["lengths"], s["tables"], sum(s["lengths_list"]),
                             starts=s["whole"])
    return {"out": out, "lse": lse, "weights": w}


def _own_append(s):
    c, cache, got = s["case"], s["cache"], {}
    if c["rotary"]:
        got["q"] = cache.append_rotary(s["q"], s["k"], s["v"], s["lengths"], s["tables"],
                                       s["inv_freq"], starts=s["starts"],
                                       positions=s["positions"], pair_axes=s["axis"],
                                       interleaved=c["pairs"] == "neighbours")
    else:
        cache.append(s["k"], s["v"], s["lengths"], s["tables"], starts=s["starts"])
    k, v = cache.gather(s["lengths"], s["tables"], sum(s["span"]), starts=s["span_starts"])
    return dict(got, k=k, v=v)


def _plain_attend(s):
    c, p = s["case"], s["pools"]
    hq, hkv, d, bt, batch = c["heads"], c["kv_heads"], c["dim"], c["block"], c["batch"]
    group, n, length = hq // hkv, max(s["counts"]), s["width"] * bt
    tables, lengths = s["tables"].long(), s["lengths"].long()
    seq, i = _ids(s["counts"])
    q = torch.zeros((batch, n, hq, d), device=DEV)
    q[seq, i] = s["q"].float()
    q = q.view(batch, n, hkv, group, d).permute(0, 2, 3, 1, 4).reshape(batch, hkv, group * n, d)

    def whole(x):                # [batch][blocks][head][token][dim]
        return x.permute(0, 2, 1, 3, 4).reshape(batch, hkv, length, d)

    token = torch.arange(length, device=DEV)
    counts = torch.tensor(s["counts"], device=DEV)
    place = (lengths - counts)[:, None] + torch.arange(n, device=DEV)
    sees = (token <= place[..., None]) & (torch.arange(n, device=DEV) < counts[:, None])[..., None]
    if c["window"]:
        sees &= token > place[..., None] - c["window"]
    keys = whole(_read_keys(p, tables)).transpose(2, 3).contiguous()
    x = torch.matmul(q, keys) * s["scale"]
    x = x.view(batch, hkv, group, n, length).masked_fill(~sees[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    x = torch.exp(x - top.clamp_min(torch.finfo(torch.float32).min))
    total = x.sum(-1, keepdim=True)
    lse = top + torch.log(total)
    x = x / total.clamp_min(torch.finfo(torch.float32).tiny)
    out = torch.matmul(x.view(batch, hkv, group * n, length), whole(_read_values(p, tables)))
    out = out.view(batch, hq, n, d).permute(0, 2, 1, 3)[seq, i]
    lse = lse.view(batch, hq, n).permute(0, 2, 1)[seq, i]
    got = {"out": out.bfloat16(), "lse": lse}
    if c["track"]:
        mine, at = _ids(s["lengths_list"])
        block, slot = tables[mine, at // bt], at % bt
        added = x.sum((2, 3)).permute(0, 2, 1)[mine, at]
        p["w"][block, :, slot] += added
        got["weights"] = p["w"][block, :, slot]
    return got


def _rotated(x, s, place):
    """x [rows][heads][dim] rotated in 64 bits by its rows' positions; `place`: those in the cache."""
    r, x = s["case"]["rotary"], x.double()
    at = place[None] if s["positions"] is None else s["positions"]
    axis = torch.zeros(r // 2, dtype=torch.long, device=DEV) if s["axis"] is None else s["axis"].long()
    angle = at.double()[axis].T * s["inv_freq"].double()
    cos, sin = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    if s["case"]["pairs"] == "halves":
        a, b = x[..., :r // 2], x[..., r // 2:r]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., r:]], -1)
    a, b = x[..., 0:r:2], x[..., 1:r:2]
    turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([turned, x[..., r:]], -1)


def _store8(p, x, name, block, slot, fresh, hkv):
    """Codes of new tokens x [n][hkv][d] into their blocks; `fresh`: blocks whose first token is new."""
    e = p[name + "s"]
    blocks = e.shape[0]
    key = (block[:, None] * hkv + torch.arange(hkv, device=DEV)).reshape(-1)
    amax = torch.zeros(blocks * hkv, dtype=torch.float64, device=DEV)
    amax.scatter_reduce_(0, key, x.abs().amax(2).reshape(-1), "amax")
    new = _exponents(amax, 448.0, -100, 119).view(blocks, hkv)
    new = torch.where(fresh[:, None], new, torch.maximum(new, e))
    touched = torch.unique(block)
    power = _power_of_two(e[touched])[..., None, None]
    values = p[name][touched].view(torch.float8_e4m3fn).double() * power
    p[name][touched] = _to_e4m3(values / _power_of_two(new[touched])[..., None, None])
    p[name][block, :, slot] = _to_e4m3(x / _power_of_two(new[block])[:, :, None])
    e[touched] = new[touched]


def _plain_append(s):
    c, p = s["case"], s["pools"]
    bt, hkv = c["block"], c["kv_heads"]
    seq, i = _ids(s["counts"])
    place = (s["lengths"].long() - torch.tensor(s["counts"], device=DEV))[seq] + i
    k, got = s["k"].double(), {}
    if c["rotary"]:
        k = _rotated(s["k"], s, place)
        got["q"] = _rotated(s["q"], s, place).bfloat16()
    there = place >= 0
    seq, at, k, v = seq[there], place[there], k[there], s["v"].double()[there]
    block, slot = s["tables"].long()[seq, at // bt], at % bt
    if c["bits"] == 4:
        p["k"][block, :, slot], p["ke"][block, :, slot] = _keys4(k)
        p["v"][block, :, slot], p["ve"][block, :, slot] = _values4(v)
    else:
        fresh = torch.zeros(p["w"].shape[0], dtype=torch.bool, device=DEV)
        fresh[block[slot == 0]] = True
        _store8(p, k, "k", block, slot, fresh, hkv)
        _store8(p, v, "v", block, slot, fresh, hkv)
    p["w"][block, :, slot] = 0
    # Read back from the start of the blocks that were touched.
    seq, i = _ids(s["span"])
    at = s["lengths"].long()[seq] - torch.tensor(s["span"], device=DEV)[seq] + i
    block, slot = s["tables"].long()[seq, at // bt], at % bt
    if c["bits"] == 4:
        where = (block, slice(None), slot)
        return dict(got, k=_read_keys(p, where).bfloat16(), v=_read_values(p, where).bfloat16())
    k, v = ((p[x][block, :, slot].view(torch.float8_e4m3fn).float() *
             _power_of_two(p[x + "s"][block]).float()[..., None]).bfloat16() for x in "kv")
    return dict(got, k=k, v=v)


# ------------------------------------------------------------ the definition

def exact(case, seed):
    """The outputs from the definitions, sequence by sequence and head by head, in 64 bits."""
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return _exact_attend(s) if case["op"] == "attend" else _exact_append(s)


def _e4m3_values():
    """The 256 values of E4M3FN from its definition (bias 7, no infinities), in 64 bits."""
    v = []
    for code in range(256):
        e, m = code >> 3 & 15, code & 7
        x = math.nan if e == 15 and m == 7 else math.ldexp(m, -9) if e == 0 else math.ldexp(8 + m, e - 10)
        v.append(-x if code & 128 else x)
    return torch.tensor(v, dtype=torch.float64, device=DEV)


def _e2m1_values():
    """The 16 values of E2M1 from its definition (bias 1), in 64 bits."""
    v = [math.ldexp(c & 1, -1) if c < 2 else math.ldexp(2 + (c & 1), (c >> 1) - 2) for c in range(8)]
    return torch.tensor(v + [-x for x in v], dtype=torch.float64, device=DEV)


def _powers(exponents):
    """2^e for whole e from -100 to 119, in 64 bits."""
    table = [math.ldexp(1.0, e) for e in range(-100, 120)]
    return torch.tensor(table, dtype=torch.float64, device=DEV)[exponents.long() + 100]


def _exact_tokens(s, name, b, h, n):
    """[n][d] of head h of sequence b's first n tokens."""
    c, p = s["case"], s["pools"]
    ids = s["tables"][b, :-(-n // c["block"])].long()
    codes = p[name][ids, h]
    if c["bits"] == 8:
        x = _e4m3_values()[codes.long()] * _powers(p[name + "s"][ids, h])[:, None, None]
    else:
        x = torch.empty(codes.shape[:2] + (c["dim"],), dtype=torch.float64, device=DEV)
        x[..., 0::2], x[..., 1::2] = (_e2m1_values()[y.long()] for y in (codes % 16, codes // 16))
        if name == "k":
            x = x * _powers(p["ke"][ids, h]).repeat_interleave(32, -1)
        else:
            x = x * p["ve"][ids, h].double()[..., None]
    return x.reshape(-1, c["dim"])[:n]


def _exact_attend(s):
    c = s["case"]
    group = c["heads"] // c["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device=DEV)
    weights, row = [], 0
    for b, (n, count) in enumerate(zip(s["lengths_list"], s["counts"])):
        mine = []
        place = torch.arange(n - count, n, device=DEV)[:, None]
        token = torch.arange(n, device=DEV)
        hidden = token > place
        if c["window"]:
            hidden |= token <= place - c["window"]
        for h in range(c["kv_heads"] if n else 0):
            k, v = _exact_tokens(s, "k", b, h, n), _exact_tokens(s, "v", b, h, n)
            got = torch.zeros(n, dtype=torch.float64, device=DEV)
            for j in range(h * group, (h + 1) * group):
                x = s["q"][row:row + count, j].double() @ k.T * s["scale"]
                x[hidden] = -math.inf
                one = torch.logsumexp(x, 1)
                x = torch.exp(x - one[:, None])
                x[torch.isinf(one)] = 0
                out[row:row + count, j], lse[row:row + count, j] = x @ v, one
                got += x.sum(0)
            ids = s["tables"][b, :-(-n // c["block"])].long()
            mine.append(s["pools"]["w"][ids, h].reshape(-1)[:n].double() + got)
        if n:
            weights.append(torch.stack(mine, 1))
        row += count
    return dict({"out": out, "lse": lse}, **({"weights": torch.cat(weights)} if c["track"] else {}))


def _turn(x, s, at):
    """x [n][heads][dim] at positions `at` [n][pair], pair by pair as complex numbers."""
    r = s["case"]["rotary"]
    first = torch.arange(r // 2, device=DEV)
    first, second = (first, first + r // 2) if s["case"]["pairs"] == "halves" else (2 * first, 2 * first + 1)
    z = torch.complex(x[..., first], x[..., second])
    one = torch.ones((), dtype=torch.float64, device=DEV)
    z = z * torch.polar(one, at * s["inv_freq"].double())[:, None]
    y = x.clone()
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _nearest(x, power, bits):
    """x over power, rounded to the nearest E4M3 or E2M1 value (ties to the even code), times power."""
    y = (x / power).abs()
    least, below = ((2.0 ** -6, 4) if bits == 8 else (1.0, 2))
    # frexp's mantissa is in [0.5, 1): a normal value's quantum is 2^(its exponent - below).
    quantum = _powers(torch.frexp(y.clamp_min(least)).exponent - below)
    y = torch.minimum(torch.round(y / quantum) * quantum, torch.full_like(y, 448 if bits == 8 else 6))
    return torch.sign(x) * y * power


def _power(amax, top):
    """Smallest power of two whose `top`-fold reaches amax."""
    e = torch.full_like(amax, -100.0)
    for k in range(-40, 40):
        e = torch.where(amax > top * 2.0 ** (k - 1), float(k), e)
    return _powers(e)


def _scale(amax):
    """Smallest of the numbers n * 2^k, n = 32 .. 63, k = -24 .. 10, whose 6-fold reaches amax."""
    every = torch.tensor([n * 2.0 ** k for k in range(-24, 11) for n in range(32, 64)],
                         dtype=torch.float64, device=DEV)
    return every[torch.searchsorted(6 * every, amax.contiguous()).clamp_max(len(every) - 1)]


def _exact_append(s):
    c, bt = s["case"], s["case"]["block"]
    got, row = {"k": [], "v": []}, 0
    if c["rotary"]:
        got["q"] = []
    for b, (n, count) in enumerate(zip(s["lengths_list"], s["counts"])):
        first, mine = n - count, slice(row, row + count)
        row += count
        new = {x: s[x][mine].double() for x in ("k", "v")}
        if c["rotary"]:
            at = torch.arange(first, n, device=DEV)[None] if s["positions"] is None else \
                s["positions"][:, mine]
            axis = [0] * (c["rotary"] // 2) if s["axis"] is None else s["axis"].tolist()
            at = at.double()[axis].T
            new["k"] = _turn(new["k"], s, at)
            got["q"].append(_turn(s["q"][mine].double(), s, at))
        new = {x: y[max(0, -first):] for x, y in new.items()}
        first = max(first, 0)
        for block in range(first // bt, -(-n // bt)) if n else ():
            lo, hi = max(first, block * bt), min(n, (block + 1) * bt)
            begun, where = lo - block * bt, s["tables"][b, block].long()
            for x in ("k", "v"):
                y = new[x][lo - first:hi - first]
                before = [torch.stack([_exact_tokens(s, x, b, h, lo)[block * bt:]
                                       for h in range(c["kv_heads"])], 1)] if begun else []
                if c["bits"] == 8:
                    power = _power(y.abs().amax((0, 2)), 448.0)
                    if begun:
                        power = torch.maximum(power, _powers(s["pools"][x + "s"][where]))
                    y = _nearest(torch.cat(before + [y]), power[:, None], 8)
                elif x == "k":
                    z = y.unflatten(-1, (-1, 32))
                    z = _nearest(z, _power(z.abs().amax(-1), 6.0)[..., None], 4).flatten(-2)
                    y = torch.cat(before + [z])
                else:
                    y = torch.cat(before + [_nearest(y, _scale(y.abs().amax(-1))[..., None], 4)])
                got[x].append(y)
    return {x: torch.cat(v) for x, v in got.items()}
