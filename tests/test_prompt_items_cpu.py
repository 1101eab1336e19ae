"""The prompt kernel's search for an item's sequence (csrc/prompt_items.cuh), compiled for the host: row tiles asked for in
any order are found where a search from the start finds them."""
import ctypes
import random
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "qwen-mtp-mac_b200" / "csrc"

# the kernel's loop over 32 sequences a step, lane by lane
SOURCE = """
#include "prompt_items.cuh"
extern "C" void search(const int* tiles, int B, const long long* asked, int n, int* found, long long* inside) {
  qmtp::ItemCursor at;
  for (int i = 0; i < n; ++i) {
    found[i] = -1;
    inside[i] = -1;
    at.seek(asked[i]);
    while (at.seq < B && found[i] < 0) {
      long long sum = 0;
      for (int lane = 0; lane < 32 && at.seq + lane < B; ++lane) {
        const long long place = asked[i] - at.before - sum;
        if (place >= 0 && place < tiles[at.seq + lane]) {
          found[i] = at.seq + lane;
          inside[i] = place;
        }
        sum += tiles[at.seq + lane];
      }
      if (found[i] < 0) at.pass(32, sum);
    }
  }
}
"""


@pytest.fixture(scope="module")
def search(tmp_path_factory):
    out = tmp_path_factory.mktemp("items")
    (out / "items.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-I", str(CSRC), "-o", str(out / "items.so"),
                    str(out / "items.cpp")], check=True)
    fn = ctypes.CDLL(str(out / "items.so")).search

    def run(tiles, asked):
        found, inside = (ctypes.c_int * len(asked))(), (ctypes.c_longlong * len(asked))()
        fn((ctypes.c_int * len(tiles))(*tiles), len(tiles), (ctypes.c_longlong * len(asked))(*asked), len(asked), found, inside)
        return list(zip(found, inside))

    return run


@pytest.mark.parametrize("order", ["rising", "falling", "any"])
@pytest.mark.parametrize("B", [1, 31, 32, 33, 100, 1000])
def test_items_are_found_in_any_order(search, B, order):
    rng = random.Random(B)
    tiles = [rng.choice((0, 0, 1, 2, 7)) for _ in range(B)]
    want = [(b, i) for b, n in enumerate(tiles) for i in range(n)]
    asked = list(range(len(want) + 5))  # beyond the last tile: no sequence
    if order == "falling":
        asked.reverse()
    elif order == "any":
        asked = rng.choices(asked, k=3 * len(asked))
    assert search(tiles, asked) == [want[t] if t < len(want) else (-1, -1) for t in asked]
