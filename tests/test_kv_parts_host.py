"""Parts of a sequence's tokens against the blocks that a workgroup holds
numbers of, wherever a part starts (without a GPU)."""
import re
import subprocess
from pathlib import Path

import pytest

SRC = Path(__file__).resolve().parents[1] / "ullm-project_amd" / "src"


def _function(text, start):
    """The source of one function that begins with `start`."""
    at = text.index(start)
    return text[at:text.index("\n}", at) + 2]


@pytest.fixture(scope="module")
def limit(tmp_path_factory):
    """kv_part_limit(blocks, shift, window) of the header, compiled."""
    body = _function((SRC / "kv_cache.hpp").read_text(), "constexpr uint64_t kv_part_limit(")
    d = tmp_path_factory.mktemp("parts")
    (d / "limit.cpp").write_text(
        "#include <cstdint>\n#include <cstdio>\n#include <cstdlib>\n" + body + """
int main(int, char **v) {
  std::printf("%llu", (unsigned long long)kv_part_limit(std::atoi(v[1]), std::atoi(v[2]),
                                                        std::atoi(v[3])));
}
""")
    subprocess.run(["g++", "-std=c++17", str(d / "limit.cpp"), "-o", str(d / "limit")], check=True)
    return lambda *a: int(subprocess.run([str(d / "limit"), *map(str, a)], capture_output=True,
                                         text=True, check=True).stdout)


def _touched(start, tokens, bt):
    return (start + tokens - 1) // bt - start // bt + 1


def _constant(name, file):
    m = re.search(rf"\b{name} = (\d+)", (SRC / file).read_text())
    return int(m.group(1))


@pytest.mark.parametrize("shift", [5, 6, 7])
@pytest.mark.parametrize("blocks", [64, 512])
def test_a_part_touches_no_more_blocks_than_its_limit(limit, shift, blocks):
    bt = 1 << shift
    # With a window the first part starts at any 32-token group.
    most = limit(blocks, shift, 1)
    assert all(_touched(start, most // 64 * 64, bt) <= blocks for start in range(0, 4 * bt, 32))
    assert most > (blocks - 1) * bt
    # Without one parts start at multiples of their size, a multiple of 64.
    most = limit(blocks, shift, 0)
    for tokens in range(64, most + 1, 64):
        assert all(_touched(p * tokens, tokens, bt) <= blocks for p in range(5))


@pytest.mark.parametrize("bt,window,rows,length", [
    (64, 32683, 2048, 140033), (64, 32704, 2048, 40000), (128, 65440, 1024, 140000),
    (128, 65400, 2048, 140000), (64, 32600, 2048, 140033), (32, 16300, 2048, 140033)])
def test_many_rows_hold_every_block_of_a_part(limit, bt, window, rows, length):
    """A workgroup of many rows that keeps one set of block entries looks at
    none past them: 4 heads of a group, one part to a tile of 128 rows."""
    held, shift = _constant("kManyBlocks", "kv_attend.hip"), bt.bit_length() - 1
    span = window + 128 // 4 + 32
    part = -(-span // 64) * 64
    longer = part > limit(held, shift, window)
    most = 0
    for first in range(0, rows, 32):
        low = length - rows + first
        begin = max(low - window + 1, 0) // 32 * 32
        most = max(most, _touched(begin, min(part, low + 32 - begin), bt))
    assert longer or most <= held
    # The entries are replaced on the way only where a part needs it.
    assert not longer or part + bt > held * bt
