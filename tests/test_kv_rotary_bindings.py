"""rust/ullm-hip-sys/src/kv_rotary_bindings.rs against include/ullm/kv_cache4.h
and kv_rotary.h: every constant, struct field, layout and signature, and the
module that the patch of the crate gives it (CPU only; no Rust toolchain exists
here)."""
import re
from pathlib import Path

import abi_parse as A

ROOT = Path(__file__).resolve().parent.parent


def _header(*names):
    return "".join((ROOT / "include" / "ullm" / n).read_text() for n in names)


def _rust(name):
    return (ROOT / "rust" / "ullm-hip-sys" / "src" / name).read_text()


OWN = ("kv_cache4.h", "kv_rotary.h")


def test_constants():
    assert A.rust_constants(_rust("kv_rotary_bindings.rs")) == A.c_constants(_header(*OWN))


def test_structs():
    header, rust = _header(*OWN), _rust("kv_rotary_bindings.rs")
    c, r = A.c_structs(header, A.c_constants(header)), A.rust_structs(rust)
    assert r == c and list(c) == ["ullm_kv_cache_append_rotary_desc_t"]
    both = _header("kv_cache.h", *OWN)
    every = A.c_structs(both, A.c_constants(both))
    sizes = re.findall(r"/// (\d+) bytes\.\n(?:#.*\n)+pub struct (\w+)", rust)
    assert {n: int(s) for s, n in sizes} == {n: A.size_align(n, every)[0] for n in c}


def test_functions():
    assert A.rust_functions(_rust("kv_rotary_bindings.rs")) == A.c_functions(_header(*OWN))


def test_the_patch_includes_the_module():
    patch = (ROOT / "rust" / "patches" / "ullm-hip-sys.patch").read_text()
    assert '+    include!("kv_rotary_bindings.rs");\n' in patch
    # The types that it takes from its neighbour are there.
    theirs = set(A.rust_structs(_rust("kv_cache_bindings.rs")))
    used = re.search(r"use crate::kv_cache::\{([^}]*)\}", _rust("kv_rotary_bindings.rs")).group(1)
    assert {n.strip() for n in used.split(",")} <= theirs


def test_the_integration_guide_names_every_function():
    doc = (ROOT / "INTEGRATION.md").read_text()
    assert "rust/ullm-hip-sys/src/kv_rotary_bindings.rs" in doc
    assert not [f for f in A.c_functions(_header(*OWN)) if f not in doc]
