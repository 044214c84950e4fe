// Every visible (query, key) pair is met exactly once, by the forward's walk over KV tiles and by the backward's blocks; tiles that
// are taken without a mask have nothing to hide. Reads "T W S" lines, prints the first failure of a line or "ok".
#include <cstdio>
#include <vector>

#include "window_plan.h"

using namespace tlm;

static bool visible(int q, int k, int W, int S) { return k <= q && (q - k < W || k < S); }

static const char* check(int T, int W, int S) {
  const int n = (T + WIN_TILE - 1) / WIN_TILE;
  std::vector<unsigned char> seen((size_t)T * T);
  auto tile = [&](int qt, int t, bool masked, int keys_below) -> const char* {
    for (int q = qt * WIN_TILE; q < (qt + 1) * WIN_TILE && q < T; ++q)
      for (int k = t * WIN_TILE; k < (t + 1) * WIN_TILE && k < T; ++k) {
        const bool v = visible(q, k, W, S);
        if (!v && !masked) return "a hidden pair in a tile without mask";
        if (v && k >= keys_below) return "a visible pair that its block drops";
        if (v && seen[(size_t)q * T + k]++) return "a pair met twice";
      }
    return nullptr;
  };
  auto all = [&]() -> const char* {
    for (int q = 0; q < T; ++q)
      for (int k = 0; k < T; ++k)
        if (visible(q, k, W, S) != (seen[(size_t)q * T + k] == 1)) return "a visible pair not met";
    return nullptr;
  };
  const char* e;
  for (int qt = 0; qt < n; ++qt) {
    const int first = win_first_tile(qt, W), steps = qt - first + 1 + win_sink_tiles(first, S);
    if (win_kv_tile(0, qt, first) != qt) return "the diagonal is not first";
    for (int s = 0; s < steps; ++s) {
      const int t = win_kv_tile(s, qt, first);
      if (t < 0 || t > qt) return "a tile out of range";
      if ((e = tile(qt, t, win_partial(qt, t, W, S), T))) return e;
    }
  }
  if ((e = all())) return e;
  std::fill(seen.begin(), seen.end(), 0);
  const WinFar f = win_far(T, W, S);
  // as the kernel decides it, for whole tiles
  auto masked = [&](int qi, int j) { return qi == j || ((qi - j) * WIN_TILE + WIN_TILE - 1 >= W && (j + 1) * WIN_TILE > S); };
  for (int j = 0; j < n; ++j)
    for (int qi = j; qi <= win_last_q(j, W, n); ++qi)
      if ((e = tile(qi, j, masked(qi, j), T))) return e;
  if (f.chunks > 64) return "too many pieces";
  for (int j = 0; j < f.tiles; ++j)
    for (int c = 0; c < f.chunks; ++c) {
      int from, to;
      win_far_range(f, j, c, W, n, from, to);
      for (int qi = from; qi < to; ++qi)
        if ((e = tile(qi, j, masked(qi, j), S))) return e;
    }
  return all();
}

int main() {
  int T, W, S;
  while (std::scanf("%d %d %d", &T, &W, &S) == 3) {
    const char* e = check(T, W, S);
    std::printf("%s\n", e ? e : "ok");
  }
}
