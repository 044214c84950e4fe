"""Tile plan of the window attention kernels (csrc/window_plan.h), compiled for the host and checked against the definition."""
import os
import random
import shutil
import subprocess

import pytest

import train_large_model_from_scratch_b200 as pkg

SRC = os.path.join(os.path.dirname(pkg.__file__), "csrc")
HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("no host compiler")
    exe = str(tmp_path_factory.mktemp("plan") / "plan")
    subprocess.run(["g++", "-O2", "-std=c++17", "-I", SRC, os.path.join(HERE, "window_plan_host_test.cpp"), "-o", exe], check=True)
    return exe


def test_pieces_of_many_sink_tiles_stay_few(tmp_path):
    """A piece of a sink tile leaves 128 rows of partial sums: 256 pieces in all while there are fewer tiles, else one a tile."""
    if shutil.which("g++") is None:
        pytest.skip("no host compiler")
    src, exe = tmp_path / "far.cpp", str(tmp_path / "far")
    src.write_text('#include <cstdio>\n#include "window_plan.h"\nint main() { int T, W, S; while (std::scanf("%d %d %d", &T, &W, &S) == 3) '
                   '{ const tlm::WinFar f = tlm::win_far(T, W, S); std::printf("%d %d\\n", f.tiles, f.chunks); } }\n')
    subprocess.run(["g++", "-O2", "-std=c++17", "-I", SRC, str(src), "-o", exe], check=True)
    cases = [(T, W, S) for T in (4096, 32768, 131072, 1 << 20, 1 << 29) for W in (1, 1024) for S in (1, 129, 1000, T // 8, T // 2, T)]
    out = subprocess.run([exe], input="".join("%d %d %d\n" % c for c in cases), capture_output=True, text=True, check=True).stdout.split()
    for (T, W, S), tiles, chunks in zip(cases, map(int, out[::2]), map(int, out[1::2])):
        assert chunks >= 1 and 1 <= tiles <= -(-S // 128) and tiles * chunks <= max(256, tiles) and chunks <= 64, (T, W, S, tiles, chunks)


def test_blocks_without_a_mask_have_nothing_to_hide(tmp_path):
    """The backward's 32 x 32 blocks: where one is taken without a mask all its pairs are visible; where not, the columns that a row
    sees are those of the definition."""
    if shutil.which("g++") is None:
        pytest.skip("no host compiler")
    src, exe = tmp_path / "block.cpp", str(tmp_path / "block")
    src.write_text("""#include <cstdio>
#include "window_plan.h"
int main() {
  int T, W, S;
  while (std::scanf("%d %d %d", &T, &W, &S) == 3) {
    const int n = (T + 127) / 128;
    int bad = 0;
    for (int j = 0; j < n; ++j)
      for (int qi = j; qi < n; ++qi)
        for (int block = 0; block < 16; ++block) {
          const int k0 = j * 128 + block / 4 * 32, q0 = qi * 128 + block % 4 * 32;
          const bool partial = tlm::win_block_partial(j, k0 - q0, W, S);
          for (int k = k0; k < k0 + 32; ++k)
            for (int i = 0; i < 32; ++i) {
              const bool seen = k <= q0 + i && (q0 + i - k < W || k < S);
              const bool kept = (unsigned)(i - (k - q0)) < (k < S ? 0x80000000u : (unsigned)W);
              bad += partial ? kept != seen : !seen;
            }
        }
    std::printf("%d\\n", bad);
  }
}
""")
    subprocess.run(["g++", "-O2", "-std=c++17", "-I", SRC, str(src), "-o", exe], check=True)
    cases = [(T, W, S) for T in (1, 100, 128, 400, 700) for W in (1, 2, 31, 32, 33, 63, 64, 65, 100, 127, 128, 129, 160, 300, 700) if W <= T
             for S in (0, 1, 4, 31, 32, 127, 128, 129, 300) if S <= T]
    out = subprocess.run([exe], input="".join("%d %d %d\n" % c for c in cases), capture_output=True, text=True, check=True).stdout.split()
    assert len(out) == len(cases) and not [c for c, o in zip(cases, out) if o != "0"]


def test_rows_without_a_rest_see_a_tile_of_keys(tmp_path):
    if shutil.which("g++") is None:
        pytest.skip("no host compiler")
    src, exe = tmp_path / "rest.cpp", str(tmp_path / "rest")
    src.write_text('#include <cstdio>\n#include "window_plan.h"\nint main() { int T, W, S; while (std::scanf("%d %d %d", &T, &W, &S) == 3) '
                   '{ std::printf("%d %d\\n", tlm::win_rest_rows(T, W, S), (int)tlm::win_few(T, W, S)); } }\n')
    subprocess.run(["g++", "-O2", "-std=c++17", "-I", SRC, str(src), "-o", exe], check=True)
    cases = [(T, W, S) for T in (1, 2, 127, 128, 129, 300, 1000) for W in (1, 2, 64, 127, 128, 129, 300, 1000) if W <= T
             for S in (0, 1, 63, 64, 126, 127, 128, 300) if S <= T]
    out = subprocess.run([exe], input="".join("%d %d %d\n" % c for c in cases), capture_output=True, text=True, check=True).stdout.split()
    for (T, W, S), rows, few in zip(cases, map(int, out[::2]), map(int, out[1::2])):
        keys = [sum(1 for j in range(i + 1) if i - j < W or j < S) for i in range(min(T, 400))]
        assert rows <= T and (rows == T or rows == 128) and all(n >= 128 for n in keys[rows:]), (T, W, S, rows)
        assert not few or max(keys) < 128, (T, W, S)


def test_every_visible_pair_is_met_once(plan):
    rng = random.Random(0)
    sizes = [1, 2, 127, 128, 129, 255, 256, 257, 640, 1001]
    cases = [(T, W, S) for T in sizes for W in sizes if W <= T for S in (0, 1, 4, 127, 128, 129, 300, 1001) if S <= T]
    for _ in range(100):
        T = rng.randint(1, 2000)
        cases.append((T, rng.randint(1, T), rng.choice([0, rng.randint(0, min(T, 20)), rng.randint(0, T)])))
    cases += [(4000, 1, 1), (4000, 128, 4), (4000, 1000, 500)]
    out = subprocess.run([plan], input="".join("%d %d %d\n" % c for c in cases), capture_output=True, text=True, check=True).stdout.split("\n")
    bad = [(c, o) for c, o in zip(cases, out) if o != "ok"]
    assert len(out) == len(cases) + 1 and not bad, bad[:5]
