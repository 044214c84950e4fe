// Which 128-row tiles meet under a causal sliding window with sinks, written once for the attention kernels and for a host test
// (tests/window_plan_host_test.cpp). Key k is visible to query q iff k <= q and (q - k < W or k < S); 1 <= W <= T, 0 <= S <= T.
#pragma once

#include "tile_order.h"

namespace tlm {

constexpr int WIN_TILE = 128;

// ---- forward: the KV tiles of query tile qt, the diagonal first (every row sees itself, so its running maximum is finite from
// then on), then down to the window's first tile, then the sink tiles in front of that.
TLM_TILE_HD int win_first_tile(int qt, int W) {
  const int lo = qt * WIN_TILE - W + 1;
  return lo > 0 ? lo / WIN_TILE : 0;
}
TLM_TILE_HD int win_sink_tiles(int first, int S) {
  const int n = (S + WIN_TILE - 1) / WIN_TILE;
  return n < first ? n : first;
}
TLM_TILE_HD int win_kv_tile(int step, int qt, int first) {
  const int in_window = qt - first + 1;
  return step < in_window ? qt - step : step - in_window;
}
// Does some (query, key) pair of query tile qt and KV tile t not see each other? Rows past the end of the sequence count as rows.
TLM_TILE_HD bool win_partial(int qt, int t, int W, int S) {
  return t == qt || (t * WIN_TILE < (qt + 1) * WIN_TILE - W && (t + 1) * WIN_TILE > S);
}

// No row sees a tile's worth of keys
TLM_TILE_HD bool win_few(int T, int W, int S) { return T < WIN_TILE || W < WIN_TILE - S; }
// Rows of which the backward wants o more exactly than bf16 holds it (AttnFwdParams::o_rest), because they see few keys: all of them, or
// those of the first tile: behind it every row sees 128 keys or more.
TLM_TILE_HD int win_rest_rows(int T, int W, int S) { return win_few(T, W, S) ? T : WIN_TILE; }

// ---- backward: a block takes KV tile j and the query tiles of its window, j .. win_last_q. What sees the tile only as sinks, the
// query tiles after that ("far"), is cut into pieces of `chunk` query tiles that are blocks of their own: one tile with all of
// them would take as long as the sequence is.
TLM_TILE_HD int win_last_q(int j, int W, int n_tiles) {
  const int last = (j * WIN_TILE + WIN_TILE - 2 + W) / WIN_TILE;
  return last < n_tiles - 1 ? last : n_tiles - 1;
}

// A warp of the backward takes 32 keys of KV tile j by 32 queries; `ahead` is how far its first key lies behind its first query's own place
// (negative: in front of it). Query i of key k's row is seen iff ahead + k <= i < ahead + k + W (or whatever, for sinks). Is one hidden?
TLM_TILE_HD bool win_block_partial(int j, int ahead, int W, int S) {
  return ahead > -31 || (ahead + W < 32 && (j + 1) * WIN_TILE > S);
}

struct WinFar {
  int tiles;           // sink tiles that have far query tiles
  int chunk, chunks;   // query tiles a piece, pieces of tile 0 (which has the most)
};
// A piece is as long as a block's share of the window, but not below 8 query tiles (a block costs about 5 steps beside its steps).
// There are at most 64 of a tile, which are added up one by one, and 256 in all, or one a tile: each holds its tile's rows in memory. In
// us, 64 of every tile / 256 / 64 in all (16 / 8 heads of 64): 32768 keys and 16384 sinks, window 1024 6908 / 5426 / 5345 and 1.9 GB /
// 201 / 134 MB, 1000 sinks 1020 / 978 / 936; 8192 keys, 2000 sinks, window 256, 4 / 1 heads 87 / 89 / 102.
TLM_TILE_HD WinFar win_far(int T, int W, int S) {
  const int n_tiles = (T + WIN_TILE - 1) / WIN_TILE, far0 = S > 0 ? n_tiles - 1 - win_last_q(0, W, n_tiles) : 0;
  WinFar f{0, 1, 0};
  if (far0 <= 0) return f;
  f.tiles = (S + WIN_TILE - 1) / WIN_TILE;
  while (win_last_q(f.tiles - 1, W, n_tiles) >= n_tiles - 1) --f.tiles;       // tile 0 has far0 > 0
  const int most = f.tiles < 4 ? 64 : f.tiles < 256 ? 256 / f.tiles : 1, share = 1 + (WIN_TILE - 2 + W) / WIN_TILE;
  f.chunk = share < 8 ? 8 : share;
  if (f.chunk < (far0 + most - 1) / most) f.chunk = (far0 + most - 1) / most;
  f.chunks = (far0 + f.chunk - 1) / f.chunk;
  return f;
}
// Query tiles [from, to) of piece c of sink tile j (none where from >= to)
TLM_TILE_HD void win_far_range(const WinFar& f, int j, int c, int W, int n_tiles, int& from, int& to) {
  from = win_last_q(j, W, n_tiles) + 1 + c * f.chunk;
  to = from + f.chunk < n_tiles ? from + f.chunk : n_tiles;
}

}  // namespace tlm
