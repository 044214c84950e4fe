// What the window attention's forward (attention_fwd.cu) and backward (attention_bwd.cu) share.
#pragma once
#include "common.cuh"
#include "window_plan.h"

namespace tlm {

// 4-D map over a [B, T, heads, hd] tensor with rows of hd contiguous elements; strides (batch, token, head) in elements, positive
// multiples of 8; boxes of box_rows tokens.
inline int make_bthd_map(CUtensorMap* map, const void* base, const long long* strides, int B, int T, int heads, int hd, int box_rows) {
  if (!aligned16(base)) return -7;
  for (int i = 0; i < 3; ++i) if (strides[i] <= 0 || strides[i] % 8 != 0 || strides[i] >= (1LL << 39)) return -7;
  uint64_t dims[4] = {(uint64_t)hd, (uint64_t)heads, (uint64_t)T, (uint64_t)B};
  uint64_t bytes[3] = {(uint64_t)strides[2] * 2, (uint64_t)strides[1] * 2, (uint64_t)strides[0] * 2};
  uint32_t box[4] = {hd == 32 ? 32u : 64u, 1, (uint32_t)box_rows, 1};
  return make_tmap_bf16(map, base, 4, dims, bytes, box);
}

}  // namespace tlm
