"""The 4-bit cache and the rotating append without a GPU: the headers against
the Python mirror, what the C entry points refuse, the layout of a chunk, the
arithmetic of a rotation as it is compiled for the host, and the reference that
the GPU's tests compare with."""
import ctypes
import math
import subprocess
from fractions import Fraction
from pathlib import Path

import numpy as np
import pytest

import abi_parse as A
import kv_reference4 as R
from test_kv_cache_host import _call, _create

ROOT = Path(__file__).resolve().parents[1]
SRC = ROOT / "ullm-project_amd" / "src"
STRUCT = "ullm_kv_cache_append_rotary_desc_t"


def _headers():
    return "".join((ROOT / "include" / "ullm" / n).read_text()
                   for n in ("kv_cache4.h", "kv_rotary.h"))


def test_python_mirrors_the_headers(uh, tmp_path):
    text = _headers()
    consts = A.c_constants(text)
    assert consts == {"ULLM_KV_CACHE_4_BITS": uh.KV_CACHE_4_BITS,
                      "ULLM_KV_ROTARY_INTERLEAVED": uh.KV_ROTARY_INTERLEAVED}
    structs = A.c_structs(text, consts)
    assert list(structs) == [STRUCT]
    assert [f[0] for f in structs[STRUCT]] == [f[0] for f in uh.KvAppendRotaryDesc._fields_]
    lines = [f'printf("size %zu\\n", sizeof({STRUCT}));'] + \
        [f'printf("{f[0]} %zu\\n", offsetof({STRUCT}, {f[0]}));' for f in structs[STRUCT]]
    src = tmp_path / "probe.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "ullm/ullm.h"\n'
                   "int main(void) {" + "".join(lines) + "return 0;}\n")
    exe = tmp_path / "probe"
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Wextra", "-Wpedantic", "-Werror",
                    f"-I{ROOT / 'include'}", str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout
    t = uh.KvAppendRotaryDesc
    for line in out.splitlines():
        f, value = line.split()
        assert (ctypes.sizeof(t) if f == "size" else getattr(t, f).offset) == int(value), line


def test_packed_descriptor_equals_the_ctypes_one(uh):
    p = uh._Packed(uh.KvAppendRotaryDesc)
    count = len(p.format.unpack(bytes(p.format.size))) - 2
    p.fill(*range(3, 3 + count))
    assert (p.desc.struct_size, p.desc.abi_version) == (ctypes.sizeof(uh.KvAppendRotaryDesc), 1)
    got = []
    for name, t in uh.KvAppendRotaryDesc._fields_[2:]:
        v = getattr(p.desc, name)
        if name == "seqs":
            got += [getattr(v, f) for f, _ in t._fields_]
        elif name == "reserved":
            assert list(v) == [0] * 4
        else:
            got.append(v)
    assert got == list(range(3, 3 + count))


@pytest.mark.parametrize("flags", [4, 5])
def test_create_takes_the_flag(uh, flags):
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is visible")
    assert _create(uh, flags=flags)[0] == uh.Status.HIP_UNAVAILABLE


@pytest.mark.parametrize("flags", [8, 6, 12])
def test_create_refuses_other_flags(uh, flags):
    st, text = _create(uh, flags=flags)
    assert st == uh.Status.INVALID_ARGUMENT and "flags" in text


@pytest.mark.parametrize("over,status", [
    (None, "INVALID_ARGUMENT"), ({"struct_size": 256}, "INVALID_ARGUMENT"),
    ({"abi_version": 9}, "INVALID_ABI_VERSION"), ({"reserved": 1}, "RESERVED_NONZERO"),
    ({}, "INVALID_ARGUMENT"), ({"cache": 0x1000}, "HIP_INVALID_HANDLE")])
def test_append_rotary_checks_its_handle(uh, over, status):
    d = uh.new(uh.KvAppendRotaryDesc)
    for k, v in (over or {}).items():
        if k == "reserved":
            d.reserved[2] = v
        else:
            setattr(d, k, v)
    st, text = _call(uh, uh.lib().ullm_kv_cache_append_rotary,
                     None if over is None else ctypes.byref(d))
    assert st.name == status and text


# ------------------------------------------------------- what Python refuses

@pytest.fixture
def cache(uh, monkeypatch):
    monkeypatch.setattr(uh, "_raw_stream", lambda: 0)
    c = uh.KvCache.__new__(uh.KvCache)
    c.handle, c.kv_heads, c.head_dim, c.block_tokens, c.device = None, 2, 128, 64, -1
    return c


def _rotary_args():
    import torch
    q = torch.zeros((2, 4, 128), dtype=torch.bfloat16)
    return dict(q=q, k=q[:, :2], v=q[:, 2:], lengths=torch.zeros(2, dtype=torch.int32),
                tables=torch.zeros((2, 3), dtype=torch.int32), inv_freq=torch.zeros(64))


def _bad_rotary_args():
    import torch
    q = torch.zeros((2, 4, 128), dtype=torch.bfloat16)
    i = torch.zeros((3, 2), dtype=torch.int32)
    return [({"q": q[0]}, "q must be"), ({"q": q.float()}, "q must be"),
            ({"q": q[:, :, :64]}, "q must be"), ({"q": q[:1]}, "rows"), ({"q": q[:, :0]}, "heads"),
            ({"out": q[:1]}, "rows"), ({"out": q[:, :2]}, "out must be"),
            ({"q": None, "out": q}, "out needs q"),
            ({"k": q}, "k must be"), ({"v": q[:1, :2]}, "rows"),
            ({"weights": torch.zeros(2, 3)}, "weights"),
            ({"inv_freq": torch.zeros(2, 32)}, "inv_freq"),
            ({"inv_freq": torch.zeros(64, dtype=torch.float64)}, "inv_freq"),
            ({"inv_freq": torch.zeros(128)[::2]}, "inv_freq"),
            ({"positions": i[0].long()}, "positions"), ({"positions": i[0, :1]}, "positions"),
            ({"positions": i[None]}, "positions"), ({"positions": i.t()}, "positions"),
            ({"positions": i[:1].expand(3, 2)}, "positions"),
            ({"pair_axes": torch.zeros(64, dtype=torch.int32)}, "pair_axes"),
            ({"pair_axes": torch.zeros(32, dtype=torch.uint8)}, "pair_axes"),
            ({"lengths": torch.zeros(3, dtype=torch.int32)}, "lengths"),
            ({"tables": torch.zeros(3, dtype=torch.int32)}, "tables"),
            ({"starts": torch.zeros(2, dtype=torch.int32)}, "starts"), ({"stream": -1}, "field")]


@pytest.mark.parametrize("i", range(25))
def test_python_refusals_name_the_argument(cache, i):
    assert len(_bad_rotary_args()) == 25
    over, word = _bad_rotary_args()[i]
    with pytest.raises(ValueError, match=word):
        cache.append_rotary(**{**_rotary_args(), **over})


def test_valid_arguments_reach_the_library(uh, cache):
    import torch
    i = torch.zeros((3, 2), dtype=torch.int32)
    a = _rotary_args()
    for over in ({}, {"q": None}, {"out": a["q"]}, {"positions": i[0]}, {"interleaved": True},
                 {"positions": i, "pair_axes": torch.zeros(64, dtype=torch.uint8)}):
        with pytest.raises(uh.HipError, match="handle is null"):
            cache.append_rotary(**{**a, **over})


def test_tensors_of_another_device_are_refused(cache):
    import torch

    class Other(torch.Tensor):
        def get_device(self):
            return 0

    a = {**_rotary_args(), "starts": torch.zeros(3, dtype=torch.int32),
         "positions": torch.zeros(2, dtype=torch.int32), "out": torch.zeros_like(_rotary_args()["q"]),
         "pair_axes": torch.zeros(64, dtype=torch.uint8), "weights": torch.zeros(2, 2)}
    for name in a:
        with pytest.raises(ValueError, match="on GPU"):
            cache.append_rotary(**{**a, name: a[name].as_subclass(Other)})


@pytest.mark.parametrize("bits", [0, 2, 16, None])
def test_bits(uh, bits):
    with pytest.raises(ValueError, match="bits"):
        uh.KvCache(4, 2, 128, bits=bits)


# ---------------------------------------------------------------- the layout

HOST = "#define __device__\n#define __host__\n#define __forceinline__ inline\n" \
       "#include <cmath>\n#include <cstdint>\n#include <cstdio>\n#include <cstring>\n" \
       "using namespace std;\n"


def _host_program(d, body, args=(), stdin=None):
    (d / "p.cpp").write_text(HOST + body)
    subprocess.run(["g++", "-std=c++17", "-O1", "-ffp-contract=off", str(d / "p.cpp"), "-o",
                    str(d / "p")], check=True)
    return subprocess.run([str(d / "p"), *args], input=stdin, capture_output=True, text=True,
                          check=True).stdout.split()


@pytest.mark.parametrize("dim", [64, 128])
def test_every_byte_of_a_chunk_has_one_owner(tmp_path, dim):
    """33 * dim + 64 bytes: two dims to a byte of the keys, a dword for 8 tokens
    of a value's dim, a byte for each exponent, two for each scale."""
    text = (SRC / "kv_cache4.hpp").read_text()
    places = text[text.index("// Byte of (token t of 32, dim d) of the keys"):
                  text.index("constexpr uint32_t kKv4ExpNan")]
    out = _host_program(tmp_path, places + f"""
int main() {{
  for (uint32_t t = 0; t < 32; ++t)
    for (uint32_t d = 0; d < {dim}; ++d)
      printf("k%u v%u.%u e%u s%u\\n", kv4_key_byte<{dim}>(t, d),
             kv4_value_dword(kv4_value_group(t), d), kv4_value_slot(t), kv4_exp_byte(t, d),
             kv4_scale_byte(t));
}}
""")
    count = {}
    for w in out:
        count[w] = count.get(w, 0) + 1
    side = 16 * dim
    assert {w: n for w, n in count.items() if w[0] == "k"} == {f"k{b}": 2 for b in range(side)}
    assert {w: n for w, n in count.items() if w[0] == "v"} == \
        {f"v{4 * b}.{j}": 1 for b in range(side // 4) for j in range(8)}
    assert {w: n for w, n in count.items() if w[0] == "e"} == {f"e{b}": 32 for b in range(dim)}
    assert {w: n for w, n in count.items() if w[0] == "s"} == {f"s{2 * b}": dim for b in range(32)}
    assert "kBytes = kScales + 64" in text and "return 33 * uint64_t(dim) + 64;" in text


# -------------------------------------------------------------- the rotation

@pytest.fixture(scope="module")
def turns(tmp_path_factory):
    """turn_of and to_odd of the header, compiled."""
    text = (SRC / "kv_rotary.hpp").read_text()
    parts = text[text.index("struct Turn {"):text.index("// The dims of pair j")]
    parts = parts.replace("__builtin_bit_cast(uint64_t, v)", "bits_of(v)")
    body = """
static float bits_f32(uint32_t b) { float f; memcpy(&f, &b, 4); return f; }
static uint64_t bits_of(double v) { uint64_t b; memcpy(&b, &v, 8); return b; }
""" + parts + """
int main(int, char **v) {
  double a, b;
  while (scanf("%lf %lf", &a, &b) == 2) {
    if (v[1][0] == 't') {
      const Turn t = turn_of(int32_t(a), float(b));
      printf("%.17g %.17g\\n", t.c, t.s);
    } else {
      printf("%.17g\\n", double(to_odd(a)));
    }
  }
}
"""
    d = tmp_path_factory.mktemp("turns")

    def run(kind, pairs):
        out = _host_program(d, body, [kind], "\n".join(f"{a!r} {b!r}" for a, b in pairs))
        return np.array([float(x) for x in out])
    return run


def test_turns_are_exact_at_every_position(turns):
    """Within 2^-49: the reduced angle of the header is within 2^-50 (three
    roundings of at most 2^-54 of a turn, times 2 pi, one of 2^-54 and two
    series' ends of 2^-53), the reference's angle is rounded by 2^-52."""
    rs = np.random.default_rng(0)
    ps = [0, 1, -1, 2, 2 ** 31 - 1, -2 ** 31, 710, 355, 103993, 2 ** 24 + 1] + \
        [int(x) for x in rs.integers(-2 ** 31, 2 ** 31, 60)] + \
        [int(x) for x in rs.integers(0, 200000, 60)]
    fs = np.float32([1, 0, 1e-4, 0.5, 3.1415927, 1e-7, -1, 65535, 0.31622776, 1.5707964, 1e-30])
    pairs = [(p, float(f)) for p in ps for f in fs]
    got = turns("t", pairs).reshape(-1, 2)
    want = np.array([(math.cos(a), math.sin(a)) for a in (R.angle(p, f) for p, f in pairs)])
    assert np.abs(got - want).max() <= 2.0 ** -49
    assert (got[[p == 0 or f == 0 for p, f in pairs]] == [1, 0]).all()


def test_to_odd_rounds_on_as_the_whole_value(turns):
    """Rounded on to bf16, the float goes where the double does; it is exact
    where the double is a float."""
    rs = np.random.default_rng(1)
    x = rs.standard_normal(400) * np.exp2(rs.integers(-90, 120, 400))
    b = np.float64(np.float32(x).view(np.uint32).__and__(0xffff0000).view(np.float32))
    mid = b * (1 + 2.0 ** -8)                      # near the middle of two bf16
    edge = np.concatenate([x, b, np.float64(np.float32(x))] +
                          [mid * (1 + s * 2.0 ** -50) for s in (-1, 0, 1)])
    got = turns("o", [(float(v), 0.0) for v in edge])

    def down(v):
        """v to bf16, to nearest, ties to even, by fractions."""
        m, e = math.frexp(v)
        return math.ldexp(round(Fraction(m) * 256), e - 8)    # 8 bits; round() ties to even
    assert [down(g) for g in got] == [down(float(v)) for v in edge]
    assert (got[400:1200] == edge[400:1200]).all()
    top = float(np.finfo(np.float32).max)
    special = [1e300, -1e300, 1e-300, 0.0, math.inf, -math.inf, 2.0 ** 128]
    assert list(turns("o", [(v, 0.0) for v in special])) == \
        [top, -top, 0.0, 0.0, math.inf, -math.inf, top]
    assert np.isnan(turns("o", [(math.nan, 0.0)])).all()


# -------------------------------------------------------------- the reference

def test_reference_rounds_to_the_nearest_even_code():
    y = np.array([0, 0.25, 0.26, 0.75, 0.74, 1.25, 1.75, 2.5, 2.51, 3.5, 5.0, 5.01, 6, 7, 1e30])
    want = np.array([0, 0, 0.5, 1, 0.5, 1, 2, 2, 3, 4, 4, 6, 6, 6, 6])
    assert (R.round_e2m1(y) == want).all() and (R.round_e2m1(-y) == -want).all()


def test_reference_scales_are_the_smallest_that_reach():
    rs = np.random.default_rng(2)
    for top in np.exp2(rs.uniform(-30, 20, 300)):
        s = R.value_scale(top)
        smaller = R.SCALES[R.SCALES < s]
        assert 6 * s >= top or s == 64512
        assert not len(smaller) or 6 * smaller[-1] < top
        assert float(np.float16(s)) == s
    for e in range(-99, 119):
        assert R.key_exponent(6 * 2.0 ** e) == e
        assert R.key_exponent(np.nextafter(6 * 2.0 ** e, np.inf)) == e + 1
    assert R.key_exponent(0.0) == -100 and R.key_exponent(3e38) == 119


@pytest.mark.parametrize("encode", [R.encode_keys4, R.encode_values4])
def test_reference_stores_stored_values_unchanged(encode):
    x = np.random.default_rng(3).standard_normal((200, 128)) * \
        np.exp2(np.random.default_rng(4).integers(-40, 30, (200, 1)))
    y = encode(x)
    assert (encode(y) == y).all() and np.abs(y - x).max() > 0
    x[3, 40], x[9, 1] = np.inf, np.nan
    bad = np.isnan(encode(x))
    if encode is R.encode_keys4:
        assert bad[3, 32:64].all() and bad[9, :32].all() and bad.sum() == 64
    else:
        assert bad[3].all() and bad[9].all() and bad.sum() == 256


def test_reference_rotation():
    """Against complex numbers where the angle needs no reduction."""
    rs = np.random.default_rng(5)
    x, f = rs.standard_normal((9, 3, 64)), np.float32([0.3, 0.01] * 8)
    p = np.arange(9)
    y = R.rotate(x, p[None], f)
    z = (x[..., :16] + 1j * x[..., 16:32]) * np.exp(1j * (p[:, None] * np.float64(f)))[:, None]
    assert np.abs(y[..., :16] - z.real).max() < 1e-13
    assert np.abs(y[..., 16:32] - z.imag).max() < 1e-13
    assert (y[..., 32:] == x[..., 32:]).all()
    y = R.rotate(x, np.stack([p, 2 * p]), f, [0, 1] * 8, True)
    at = np.where(np.arange(16) % 2 == 1, 2, 1) * p[:, None]
    z = (x[..., :32:2] + 1j * x[..., 1:32:2]) * np.exp(1j * at * np.float64(f))[:, None]
    assert np.abs(y[..., :32:2] - z.real).max() < 1e-13
    assert np.abs(y[..., 1:32:2] - z.imag).max() < 1e-13
