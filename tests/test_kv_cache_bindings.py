"""rust/ullm-hip-sys/src/kv_cache_bindings.rs against include/ullm/kv_cache.h:
every constant, struct field, layout and signature, and the place that the
patch of the crate gives it (CPU only; no Rust toolchain exists here)."""
import re
from pathlib import Path

import abi_parse as A

ROOT = Path(__file__).resolve().parent.parent


def _header():
    return (ROOT / "include" / "ullm" / "kv_cache.h").read_text()


def _rust():
    return (ROOT / "rust" / "ullm-hip-sys" / "src" / "kv_cache_bindings.rs").read_text()


def test_constants():
    assert A.rust_constants(_rust()) == A.c_constants(_header())


def test_structs():
    header, rust = _header(), _rust()
    c, r = A.c_structs(header, A.c_constants(header)), A.rust_structs(rust)
    assert r.pop("ullm_kv_cache_t") == [("_private", ("array", "u8", 0))]
    assert r == c
    sizes = re.findall(r"/// (\d+) bytes\.\n(?:#.*\n)+pub struct (\w+)", rust)
    assert {n: int(s) for s, n in sizes} == {n: A.size_align(n, c)[0] for n in c}


def test_functions():
    assert A.rust_functions(_rust()) == A.c_functions(_header())


def test_the_patch_includes_the_module_and_counts_its_lines():
    patch = (ROOT / "rust" / "patches" / "ullm-hip-sys.patch").read_text()
    assert '+    include!("kv_cache_bindings.rs");\n' in patch
    hunks = re.finditer(r"^(@@ .*)\n((?:[ +\-].*\n|\n)*?)(?=^@@|^--- |\Z)", patch, flags=re.M)
    for head, body in (m.groups() for m in hunks):
        old, new = map(int, re.search(r"-\d+,(\d+) \+\d+,(\d+)", head).groups())
        lines = body.split("\n")[:-1]
        assert sum(l[:1] != "+" for l in lines) == old, head
        assert sum(l[:1] != "-" for l in lines) == new, head


def test_the_integration_guide_names_every_function():
    doc = (ROOT / "INTEGRATION.md").read_text()
    assert "rust/ullm-hip-sys/src/kv_cache_bindings.rs" in doc
    assert not [f for f in A.c_functions(_header()) if f not in doc]
