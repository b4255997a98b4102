"""The cut of a range of weight keys into bins, by which eviction finds the
last token that stays, on the CPU: no key outside of the range is ever counted
(a key of 0 is a token that is no candidate)."""
import subprocess
from pathlib import Path

import numpy as np
import pytest

HEADER = Path(__file__).resolve().parents[1] / "ullm-project_amd" / "src" / "kv_cache.hpp"

MAIN = """
// Reads want and keys; prints the key of the last token that stays and how many
// of that key do, in the order of the kernel's steps.
int main() {
  uint32_t want, n;
  if (std::scanf("%u %u", &want, &n) != 2) return 1;
  std::vector<uint32_t> keys(n);
  for (uint32_t &k : keys) if (std::scanf("%u", &k) != 1) return 1;
  uint32_t least = ~0u, most = 0;
  for (uint32_t k : keys) { least = std::min(least, k - 1u); most = std::max(most, k); }
  KvKeyRange cut{least + 1, most - (least + 1)};
  uint32_t last, passes = 0;
  for (;;) {
    last = cut.from;
    if (cut.width == 0) break;
    if (++passes > 8) return 2;
    const uint32_t shift = kv_bin_shift(cut);
    std::vector<uint32_t> hist(1u << kKvBinBits);
    for (uint32_t k : keys) if (k - cut.from <= cut.width) hist.at((k - cut.from) >> shift)++;
    uint32_t bin = hist.size() - 1;
    while (hist[bin] < want) { want -= hist[bin]; if (bin-- == 0) return 3; }
    cut = kv_bin_keys(cut, shift, bin);
    if (want == hist[bin]) { last = cut.from - 1; want = 0; break; }
  }
  std::printf("%u %u", last, want);
}
"""


@pytest.fixture(scope="module")
def select(tmp_path_factory):
    text = HEADER.read_text()
    body = text[text.index("struct KvKeyRange {"):text.index("inline uint64_t kv_slots(")]
    d = tmp_path_factory.mktemp("select")
    (d / "select.cpp").write_text(
        "#include <algorithm>\n#include <cstdint>\n#include <cstdio>\n#include <vector>\n"
        "#define __host__\n#define __device__\n" + body + MAIN)
    subprocess.run(["g++", "-std=c++17", str(d / "select.cpp"), "-o", str(d / "select")],
                   check=True)

    def run(keys, want):
        r = subprocess.run([str(d / "select")], input=f"{want} {len(keys)} " +
                           " ".join(map(str, keys)), capture_output=True, text=True)
        assert r.returncode == 0, r.returncode
        return [int(x) for x in r.stdout.split()]
    return run


def key(weights):
    """Weights as keys of their order, NaN the largest."""
    b = np.asarray(weights, np.float32).view(np.uint32)
    k = np.where(b >> 31 != 0, ~b, b | np.uint32(1 << 31))
    return np.where(np.isnan(weights), np.uint32(0xffffffff), k)


def check(select, keys, want):
    last, ties = select(keys, want)
    chosen = np.sort(keys[keys > 0])[::-1][:want]
    assert (keys > last).sum() + ties == want
    assert np.array_equal(np.sort(np.concatenate([keys[keys > last], np.repeat(last, ties)]))[::-1],
                          chosen)


@pytest.mark.parametrize("least", [0.0, 1e-30, 0.01, 0.3, 1.0, 7.7e8])
@pytest.mark.parametrize("want", [1, 40, 99, 100, 101, 150])
def test_nan_weights_beside_finite_ones(select, least, want):
    """100 tokens of NaN, 100 finite ones, and as many as a wave that are no
    candidates."""
    w = np.concatenate([np.full(100, np.nan), least + np.linspace(0, 1, 100)])
    check(select, np.concatenate([np.zeros(64, np.uint32), key(w)]), want)


@pytest.mark.parametrize("seed", range(20))
def test_keys_of_any_kind(select, seed):
    rs = np.random.default_rng(seed)
    w = np.exp(rs.standard_normal(300) * rs.choice([0.01, 1, 20])).astype(np.float32)
    w[rs.random(300) < 0.3] = rs.choice([0.0, np.inf, np.nan, -np.inf, w[0]])
    k = key(w)
    k[rs.random(300) < rs.choice([0, 0.2])] = 1          # tokens of no block
    k[rs.random(300) < 0.3] = 0                          # no candidates
    check(select, k, int(rs.integers(1, (k > 0).sum())))
