// Causal GQA flash attention, backward, on tcgen05 / TMEM.
//
// Inputs: packed qkv[B,T,Hq+2Hkv,hd], o[B,T,Hq,hd], do[B,T,Hq,hd] (bf16),
// lse[B,Hq,T] (fp32). Output: dqkv[B,T,Hq+2Hkv,hd] (bf16) in the packed layout,
// so the QKV projection's dgrad/wgrad GEMMs consume one tensor.
//
// Three launches:
//   1. delta[b,h,t] = sum_d do*o; the dQ accumulator is zeroed on the way (few rows: by a memset)
//   2. main kernel: one CTA per (128-row KV tile, batch, KV head). The CTA walks over every query head of the group and
//      every query tile at or below the diagonal. Per step five products run on the tensor cores, scores transposed:
//                      S^T = K Q^T,  dP^T = V dO^T       (TMEM, fp32; rows = keys, columns = queries)
//                      dV += P^T dO,  dK += dS^T Q       (TMEM accumulators; P^T / dS^T are TMEM operands)
//                      dQ  = dS K                        (TMEM, flushed per step)
//      so P never leaves tensor memory and only dS goes through shared memory, as the [kv][q] bf16 tile that dQ reads
//      MN-major. Q / dO / K / V tiles are used as loaded.
//      Warps: 0 loads (Q, dO by TMA; -lse log2 e and -delta of the step's rows by the warp), 1 issues the products,
//      2 - 17 softmax (32 keys x 32 queries each: P, dS), 18 - 21 take dQ out: tiles are added to an fp32 buffer with TMA
//      reduce-add tile stores because several KV tiles contribute to one query row.
//      With few KV tiles a cluster of CTAs shares a tile's steps (SPLIT, see split_for).
//   3. dq (fp32, [B,Hq,T,hd]) -> bf16 into dqkv; with RoPE tables this pass also applies the transposed rotation to
//      dQ (from the fp32 accumulator) and to the dK slots the main kernel wrote, so the packed gradient that leaves
//      is the gradient of the UN-rotated q and k and no separate RoPE pass runs.
// A second instantiation of the main kernel (SCATTER) serves Ulysses sequence parallelism: its dK / dV epilogue
// rotates dK itself and stores the rows straight into the sequence owners' packed gradient buffers, and the
// conversion pass does the same for dQ.
// A third one (WIN) takes a sliding window with sinks (window_plan.h) and q, k, v and their gradients as tensors of their own: a block
// walks over the query tiles of its KV tile's window; the query tiles that see a tile only as sinks are further blocks, whose
// dV | dK rows meet the tile's own in an fp32 buffer that the conversion pass adds up in fixed order. A step costs what it does in
// the causal form; what a short window adds is a block's start and end, about 4 steps of 16 + 4 at B 8, T 4096, 16 / 8 heads of 64,
// window 1024: 491 us with delta and conversion passes (32 / 4 of 32, window 512 505; B 2, 16 / 4 of 128, window 2048 364).
// Every wait is bounded; on a timeout the CTA records a status code, leaves its
// loops and still releases its tensor memory.
#include "attention_window.h"
#include <cstdlib>

namespace tlm {

constexpr int AB_TILE = 128, AB_THREADS = 704, AB_MAX_DST = 8;

struct AttnBwdDst {
  __nv_bfloat16* p[AB_MAX_DST];
  int n, rows, heads;
};

struct AttnBwdParams {
  __nv_bfloat16* dqkv;
  float* dq_acc;            // [B,Hq,T,hd] fp32, zeroed before the main kernel
  const __nv_bfloat16* qkv;
  const float* lse;
  const float* delta;
  int B, T, Hq, Hkv;
  float scale, scale_log2;
  unsigned int* status;
  int hd;                   // head dim in memory; the SCATTER form runs 32 on its HD = 64 kernel with zero-filled upper columns
  // Transposed RoPE on the way out (tables cos / sin [T, hd], fp32, row = position; nullptr: off):
  //   dx[j] = dy[j] c[j] + dy[j+h] s[j+h],  dx[j+h] = dy[j+h] c[j+h] - dy[j] s[j]   (h = hd / 2).
  const float* cosT;
  const float* sinT;
  // SCATTER instantiation only: head -> sequence return of the packed gradient (Ulysses backward). Row t of local
  // head slot s is stored into
  //   dst[t / dst_rows][b, t % dst_rows, head(s), :]     (bf16 [B, dst_rows, dst_heads, hd] per rank)
  // with head(s) = dst_q0 + s for q slots, dst_k0 + s for k, dst_v0 + s for v (peer-mapped addresses, plain
  // 16-byte stores).
  __nv_bfloat16* dst[AB_MAX_DST];
  int n_dst, dst_rows, dst_heads, dst_q0, dst_k0, dst_v0;
  int split;               // SPLIT instantiation: CTAs of the cluster that share one KV tile's steps
  int head_group;          // (batch, KV head) pairs per group of the heavy-first block order (see heavy_first_decode)
  // WIN instantiation only
  int window, sinks;       // in [1, T], [0, T]
  WinFar far;
  float* part;             // far.chunks > 0: [B Hkv][1 + far.chunks][sinks][dV HD | dK HD], of tiles below far.tiles; slot 0: the window's
  const __nv_bfloat16 *k, *v;
  __nv_bfloat16 *dk, *dv;
  long long ks[3], vs[3], dks[3], dvs[3];      // batch, token, head strides in elements
};

// WIN: q [.., Hq, hd], k and v [.., Hkv, hd]; else one map over the packed tensor
template <bool WIN> struct AttnBwdMaps { CUtensorMap qkv, dout, dq; };
template <> struct AttnBwdMaps<true> { CUtensorMap q, k, v, dout, dq; };

// delta[b, h, t] = sum_c o[b, t, h, c] * dout[b, t, h, c]. One block per (b, 32 consecutive t): that slab of o
// and dout is contiguous, hd / 8 lanes share a row with 16-byte loads (four rows in flight per lane), the row sums
// are staged in shared memory so that the [B, Hq, T] output is written as whole 128-byte lines.
constexpr int DELTA_T = 32, DELTA_THREADS = 256;

// REST: o + o_rest in place of o in the first rest_rows rows, which are all or whole blocks (see AttnFwdParams).
template <bool REST>
__global__ void __launch_bounds__(DELTA_THREADS)
attn_delta_kernel(const __nv_bfloat16* o, const __nv_bfloat16* o_rest, const __nv_bfloat16* dout,
                  float* __restrict__ delta, float* __restrict__ dq_acc, int B, int T, int Hq, int hd, int rest_rows) {
  griddep_wait();
  griddep_launch();
  extern __shared__ float delta_s[];                       // [Hq][DELTA_T + 1]
  const int tiles_t = (T + DELTA_T - 1) / DELTA_T;
  const int b = blockIdx.x / tiles_t, t0 = (blockIdx.x % tiles_t) * DELTA_T;
  const int nt = min(DELTA_T, T - t0);
  const int lpr = hd >> 3;                                 // lanes per row: 4, 8 or 16
  const int sub = threadIdx.x % lpr, slot = threadIdx.x / lpr, slots = DELTA_THREADS / lpr;
  const int rows = nt * Hq;                                // row rr = tl * Hq + h
  const long long base = ((long long)b * T + t0) * Hq * hd;
  // this slab of the dQ accumulator starts at zero: stores that nothing waits for, beside the loads of the row sums
  const int vec_h = nt * hd / 4;                           // float4 of one head: its nt rows are contiguous
  for (int h = 0; dq_acc != nullptr && h < Hq; ++h) {
    float4* z = reinterpret_cast<float4*>(dq_acc + (((long long)b * Hq + h) * T + t0) * hd);
    for (int i = threadIdx.x; i < vec_h; i += DELTA_THREADS) z[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  const uint4* op = reinterpret_cast<const uint4*>(o + base) + sub;
  const uint4* dp = reinterpret_cast<const uint4*>(dout + base) + sub;
  const bool rest = REST && t0 < rest_rows;
  const uint4* rp = rest ? reinterpret_cast<const uint4*>(o_rest + ((long long)b * rest_rows + t0) * Hq * hd) + sub : nullptr;
  for (int rb = 0; rb < rows; rb += 4 * slots) {          // trip count is uniform: the shuffles below need whole warps
    const int r0 = rb + slot;
    uint4 a[4], d[4], e[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int rr = r0 + u * slots;
      if (rr < rows) { a[u] = op[(long long)rr * lpr]; d[u] = dp[(long long)rr * lpr]; }
      else { a[u] = make_uint4(0, 0, 0, 0); d[u] = a[u]; }
      if (rest) e[u] = rr < rows ? rp[(long long)rr * lpr] : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const uint32_t aw[4] = {a[u].x, a[u].y, a[u].z, a[u].w}, dw[4] = {d[u].x, d[u].y, d[u].z, d[u].w};
      float acc = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 x = unpack_bf16(aw[k]), y = unpack_bf16(dw[k]);
        acc = fmaf(x.x, y.x, fmaf(x.y, y.y, acc));
      }
      if (rest) {
        const uint32_t ew[4] = {e[u].x, e[u].y, e[u].z, e[u].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 x = unpack_bf16(ew[k]), y = unpack_bf16(dw[k]);
          acc = fmaf(x.x, y.x, fmaf(x.y, y.y, acc));
        }
      }
      for (int off = lpr >> 1; off > 0; off >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, off);
      const int rr = r0 + u * slots;
      if (sub == 0 && rr < rows) delta_s[(rr % Hq) * (DELTA_T + 1) + rr / Hq] = acc;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < Hq * DELTA_T; i += DELTA_THREADS) {
    const int h = i / DELTA_T, tl = i % DELTA_T;
    if (tl < nt) delta[((long long)b * Hq + h) * T + t0 + tl] = delta_s[h * (DELTA_T + 1) + tl];
  }
}

// dq_acc (fp32 [B, Hq, T, hd]) * scale -> bf16 q-head slots of dqkv, 8 low columns and their 8 partner columns
// (j + hd / 2) per thread so that the transposed rotation (see AttnBwdParams) can be applied on the way.
// `rot_k` (only without a head -> sequence return): the Hkv k-head slots of dqkv, written as bf16 by the main kernel, are
// rotated in place by further work items (heads Hq .. Hq + Hkv - 1).
// Index: 32 bits while the items fit (three 64-bit divisions per item took longer than the item's 64 bytes).
template <typename Index>
__global__ void attn_dq_convert_kernel(const float* dq_acc, __nv_bfloat16* __restrict__ dqkv, int B, int T,
                                       int Hq, int heads_total, int hd, float scale, const float* cosT,
                                       const float* sinT, const AttnBwdDst d, int dst_q0, int rot_k) {
  griddep_wait();
  griddep_launch();
  const int half = hd / 2, vec_log = hd == 32 ? 1 : hd == 64 ? 2 : 3;          // hd / 16 items per row
  const int heads = Hq + rot_k;
  const Index total = ((Index)B * heads * T) << vec_log, step = (Index)gridDim.x * blockDim.x;
  for (Index i = blockIdx.x * (Index)blockDim.x + threadIdx.x; i < total; i += step) {
    const int j = (int)(i & ((1 << vec_log) - 1)) * 8;
    Index r = i >> vec_log;
    const Index bh = r / (Index)T;
    const int t = (int)(r - bh * (Index)T);
    const long long b = (long long)(bh / (Index)heads);
    const int h = (int)(bh - (Index)b * heads);
    float lo[8], hi[8];
    if (h < Hq) {
      const float* src = dq_acc + (((long long)b * Hq + h) * T + t) * hd + j;
      *reinterpret_cast<float4*>(lo) = *reinterpret_cast<const float4*>(src);
      *reinterpret_cast<float4*>(lo + 4) = *reinterpret_cast<const float4*>(src + 4);
      *reinterpret_cast<float4*>(hi) = *reinterpret_cast<const float4*>(src + half);
      *reinterpret_cast<float4*>(hi + 4) = *reinterpret_cast<const float4*>(src + half + 4);
#pragma unroll
      for (int k = 0; k < 8; ++k) { lo[k] *= scale; hi[k] *= scale; }
    } else {                                             // a k head: bf16 in, rotated bf16 out, same place
      const __nv_bfloat16* src = dqkv + ((b * T + t) * heads_total + h) * (long long)hd + j;
      const uint4 a = *reinterpret_cast<const uint4*>(src), c = *reinterpret_cast<const uint4*>(src + half);
      const uint32_t aw[4] = {a.x, a.y, a.z, a.w}, cw[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 x = unpack_bf16(aw[k]), y = unpack_bf16(cw[k]);
        lo[2 * k] = x.x; lo[2 * k + 1] = x.y; hi[2 * k] = y.x; hi[2 * k + 1] = y.y;
      }
    }
    if (cosT != nullptr) {
      const float* c = cosT + (long long)t * hd + j;
      const float* sn = sinT + (long long)t * hd + j;
      float cl[8], ch[8], sl[8], sh[8];
      *reinterpret_cast<float4*>(cl) = *reinterpret_cast<const float4*>(c);
      *reinterpret_cast<float4*>(cl + 4) = *reinterpret_cast<const float4*>(c + 4);
      *reinterpret_cast<float4*>(ch) = *reinterpret_cast<const float4*>(c + half);
      *reinterpret_cast<float4*>(ch + 4) = *reinterpret_cast<const float4*>(c + half + 4);
      *reinterpret_cast<float4*>(sl) = *reinterpret_cast<const float4*>(sn);
      *reinterpret_cast<float4*>(sl + 4) = *reinterpret_cast<const float4*>(sn + 4);
      *reinterpret_cast<float4*>(sh) = *reinterpret_cast<const float4*>(sn + half);
      *reinterpret_cast<float4*>(sh + 4) = *reinterpret_cast<const float4*>(sn + half + 4);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float a = lo[k], bb = hi[k];
        lo[k] = a * cl[k] + bb * sh[k];
        hi[k] = bb * ch[k] - a * sl[k];
      }
    }
    __nv_bfloat16* dst;
    if (d.n > 0) {
      const int owner = t / d.rows, tl = t - owner * d.rows;
      if (owner >= d.n) continue;
      dst = d.p[owner] + ((b * d.rows + tl) * d.heads + dst_q0 + h) * (long long)hd + j;
    } else {
      dst = dqkv + ((b * T + t) * heads_total + h) * (long long)hd + j;
    }
    *reinterpret_cast<uint4*>(dst) = make_uint4(pack_bf16(lo[0], lo[1]), pack_bf16(lo[2], lo[3]), pack_bf16(lo[4], lo[5]), pack_bf16(lo[6], lo[7]));
    *reinterpret_cast<uint4*>(dst + half) = make_uint4(pack_bf16(hi[0], hi[1]), pack_bf16(hi[2], hi[3]), pack_bf16(hi[4], hi[5]), pack_bf16(hi[6], hi[7]));
  }
}

// The window's conversion: rows of dQ (fp32 accumulator * scale -> bf16), with a rotation its transposed form on the way, and what the
// main kernel has not finished of dK and dV: with a rotation all rows of dK (bf16, in place), and the sink rows of both, whose fp32
// parts are added up slot by slot. An item is 8 low columns and their 8 partners (j + hd / 2) of a row. The sums have blocks of
// their own: beside the conversion, one item after the other, 28 slots of 16 rows took 15 us longer than everything else (T 32768).
struct AttnWinFinish {
  const float* dq_acc;
  const float* part;                 // see AttnBwdParams
  __nv_bfloat16 *dq, *dk, *dv;
  long long dqs[3], dks[3], dvs[3];
  const float *cosT, *sinT;
  int B, T, Hq, Hkv, hd;
  int sinks, slots, slot_rows;       // rows whose sums are in `part`, its slots and a slot's rows
  int sum_blocks;                    // the first blocks of the grid
  float scale;
};
constexpr int WIN_FINISH_THREADS = 256;

// kind: 0 dQ, 1 dK, 2 dV
__device__ __forceinline__ void win_finish_item(const AttnWinFinish& p, int kind, __nv_bfloat16* dst, int t, int j, float* lo, float* hi) {
  const int half = p.hd / 2;
  if (p.cosT != nullptr && kind < 2) {
    const float *c = p.cosT + (long long)t * p.hd + j, *sn = p.sinT + (long long)t * p.hd + j;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float a = lo[k], bb = hi[k];
      lo[k] = a * c[k] + bb * sn[half + k];
      hi[k] = bb * c[half + k] - a * sn[k];
    }
  }
  *reinterpret_cast<uint4*>(dst) = make_uint4(pack_bf16(lo[0], lo[1]), pack_bf16(lo[2], lo[3]), pack_bf16(lo[4], lo[5]), pack_bf16(lo[6], lo[7]));
  *reinterpret_cast<uint4*>(dst + half) = make_uint4(pack_bf16(hi[0], hi[1]), pack_bf16(hi[2], hi[3]), pack_bf16(hi[4], hi[5]), pack_bf16(hi[6], hi[7]));
}

__global__ void __launch_bounds__(WIN_FINISH_THREADS)
attn_window_finish_kernel(const AttnWinFinish p) {
  griddep_wait();
  griddep_launch();
  const int half = p.hd / 2;
  if ((int)blockIdx.x < p.sum_blocks) {
    // a row of dV | dK: hd / 2 threads take 16 bytes of it each, as many groups of them as there are take slots in turn
    __shared__ float4 sums[WIN_FINISH_THREADS];
    const int vecs = p.hd / 2, groups = WIN_FINISH_THREADS / vecs, vec = threadIdx.x % vecs, group = threadIdx.x / vecs;
    for (int r = blockIdx.x; r < p.B * p.Hkv * p.sinks; r += p.sum_blocks) {
      const int bh = r / p.sinks, t = r - bh * p.sinks, b = bh / p.Hkv, h = bh - b * p.Hkv;
      const float4* src = reinterpret_cast<const float4*>(p.part + ((long long)bh * p.slots * p.slot_rows + t) * (2 * p.hd)) + vec;
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
      for (int n = group; n < p.slots; n += groups) {
        const float4 x = src[(long long)n * p.slot_rows * (p.hd / 2)];
        a.x += x.x; a.y += x.y; a.z += x.z; a.w += x.w;
      }
      sums[threadIdx.x] = a;
      __syncthreads();
      if (group == 0) {
        for (int n = 1; n < groups; ++n) {
          const float4 x = sums[n * vecs + vec];
          a.x += x.x; a.y += x.y; a.z += x.z; a.w += x.w;
        }
        sums[vec] = a;
      }
      __syncthreads();
      if ((int)threadIdx.x < p.hd / 8) {                 // hd / 16 items of dV, then of dK
        const int kind = (int)threadIdx.x < p.hd / 16 ? 2 : 1, j = threadIdx.x % (p.hd / 16) * 8;
        const float* row = reinterpret_cast<const float*>(sums) + (kind == 1 ? p.hd : 0) + j;
        const float osc = kind == 1 ? p.scale : 1.f;
        float lo[8], hi[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) { lo[k] = row[k] * osc; hi[k] = row[half + k] * osc; }
        __nv_bfloat16* dst = kind == 1 ? p.dk + b * p.dks[0] + t * p.dks[1] + h * p.dks[2] : p.dv + b * p.dvs[0] + t * p.dvs[1] + h * p.dvs[2];
        win_finish_item(p, kind, dst + j, t, j, lo, hi);
      }
      __syncthreads();
    }
    return;
  }
  const int vec_log = p.hd == 32 ? 1 : p.hd == 64 ? 2 : 3;          // hd / 16 items per row
  const int k_rows = p.cosT != nullptr ? p.T - p.sinks : 0;         // finished rows of dK, to be rotated
  const long long q_rows = (long long)p.B * p.Hq * p.T, total = (q_rows + (long long)p.B * p.Hkv * k_rows) << vec_log;
  const long long step = (long long)(gridDim.x - p.sum_blocks) * WIN_FINISH_THREADS;
  for (long long i = (blockIdx.x - p.sum_blocks) * (long long)WIN_FINISH_THREADS + threadIdx.x; i < total; i += step) {
    const int j = (int)(i & ((1 << vec_log) - 1)) * 8;
    long long r = i >> vec_log;
    const int kind = r < q_rows ? 0 : 1;
    if (kind == 1) r -= q_rows;
    const int rows = kind == 0 ? p.T : k_rows, heads = kind == 0 ? p.Hq : p.Hkv;
    const int bh = (int)(r / rows), t = (int)(r - (long long)bh * rows) + (kind == 0 ? 0 : p.sinks), b = bh / heads, h = bh - b * heads;
    __nv_bfloat16* dst = (kind == 0 ? p.dq + b * p.dqs[0] + t * p.dqs[1] + h * p.dqs[2] : p.dk + b * p.dks[0] + t * p.dks[1] + h * p.dks[2]) + j;
    float lo[8], hi[8];
    if (kind == 0) {
      const float* src = p.dq_acc + ((long long)bh * p.T + t) * p.hd + j;
#pragma unroll
      for (int k = 0; k < 8; k += 4) {
        *reinterpret_cast<float4*>(lo + k) = *reinterpret_cast<const float4*>(src + k);
        *reinterpret_cast<float4*>(hi + k) = *reinterpret_cast<const float4*>(src + half + k);
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) { lo[k] *= p.scale; hi[k] *= p.scale; }
    } else {
      const uint4 a = *reinterpret_cast<const uint4*>(dst), c = *reinterpret_cast<const uint4*>(dst + half);
      const uint32_t aw[4] = {a.x, a.y, a.z, a.w}, cw[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 x = unpack_bf16(aw[k]), y = unpack_bf16(cw[k]);
        lo[2 * k] = x.x; lo[2 * k + 1] = x.y; hi[2 * k] = y.x; hi[2 * k + 1] = y.y;
      }
    }
    win_finish_item(p, kind, dst, t, j, lo, hi);
  }
}

// What a step consists of, and what bounds it. Every step is taken in two halves of 64 query columns, each with its own eight
// softmax warps and barriers: while one half's exponentials run, the other half's products do. For head dims 32 and 64 there
// are three score tiles for the two halves, so a half's scores of its next step are there before its warps ask for them
// (two tiles: 1048 us against 974 at the first shape below); dP^T of the next step is issued as soon as a half has published
// P^T and dS^T, and its warps come to it only after their exponentials. Head dim 128 (WIDE) has 256 tensor-memory columns
// beside dV and dK: scores of both halves, and dP^T in turns with dQ; a step's chain is dQ -> its way out, beside dV, dK and
// the next scores -> dP^T -> dS, and the exponentials of the next step run beside the last link.
// Cycles per 128 x 128 step, head dim 64 / 32 / 128: products 1664 / 832 / 2560, exponentials 1024 (16 a cycle); shared memory
// moves 300 / 184 KB at head dim 64 / 32, 128 B a cycle. By ncu (B 8, T 4096, 16 / 8 heads: 457 steps and 14 blocks an SM) 2750 / 2630 / 5190, what
// surrounds a block's steps included, about five steps each; tensor pipe 48 / 25 / 51 %, exponential unit 45 / 46 / 23 %, shared
// memory 47 / 26 / 39 % of its cycles. Long runs are under the power cap at 1.5 - 1.7 GHz, so what counts is energy: without the dQ
// reductions to L2 head dim 64 would take 8 % less, without any other part 2 - 4 %.
// In us with the delta and conversion passes, in sequence, against the form before (scores [q][kv], P and dS through shared
// memory, eight softmax warps that also flushed dQ, products issued by one lane's own code, a smaller last group of heads):
//   B 8, T 4096, 16 / 8 heads of 64: 1098 -> 930     B 1, T 32768, the same: 7400 -> 6040
//   B 8, T 4096, 32 / 4 heads of 32: 2055 -> 1350    B 2, T 4096, 24 / 8 heads of 128: 929 -> 667
// The parts were not timed one by one. What was measured is that a step's products, issued by one lane's own code, took 76 cycles
// each whatever their size (see umma_bf16_w), more than those of 64 columns run.
template <int HD>
struct AttnBwdCfg {
  static constexpr bool WIDE = HD == 128;
  static constexpr int KB = WIDE ? 2 : 1;                     // 64-wide blocks of a tile (HD 32: one of 32)
  static constexpr int STAGES = WIDE ? 2 : 3;                 // Q / lse / delta ring
  static constexpr int DO_STAGES = WIDE ? 1 : 3;
  static constexpr int DS_BUFS = WIDE ? 1 : 2;
  static constexpr int NS = WIDE ? 2 : 3;                     // score tiles (half steps)
  static constexpr bool KV_TMEM = HD == 32;                   // K and V as operands in tensor memory
  static constexpr int TILE_BYTES = AB_TILE * HD * 2;
  static constexpr int OFF_K = 0;
  static constexpr int OFF_V = OFF_K + TILE_BYTES;
  static constexpr int OFF_Q = OFF_V + (KV_TMEM ? 0 : TILE_BYTES);
  static constexpr int OFF_DO = OFF_Q + STAGES * TILE_BYTES;
  static constexpr int OFF_DS = OFF_DO + DO_STAGES * TILE_BYTES;   // buffers of [2 query halves][128 kv][64 q] bf16
  static constexpr int DS_BYTES = AB_TILE * AB_TILE * 2;
  static constexpr int OFF_DQS = OFF_DS + DS_BUFS * DS_BYTES;  // dQ staging: [32 rows][32 fp32] boxes of the four flush warps
  static constexpr int BOXES = WIDE ? 2 : 1;
  static constexpr int OFF_ROW = OFF_DQS + 4 * BOXES * 4096;
  static constexpr int OFF_BAR = OFF_ROW + STAGES * 2 * AB_TILE * 4;
  static constexpr int TOTAL = OFF_BAR + 256;
  static_assert(TOTAL <= 232448, "shared memory of one block");
  static constexpr int PART_PITCH = 2 * HD + 4;                // SPLIT: floats per row of this CTA's dV | dK, from OFF_Q on
  static_assert(AB_TILE * PART_PITCH * 4 <= (WIDE ? OFF_ROW : OFF_DS) - OFF_Q, "the partial dV | dK fits behind K and V");
  // tensor memory: NS tiles of S^T (a half step's P^T and dS^T replace them as bf16), two of dP^T, dV, dK, dQ, K and V.
  // WIDE: dQ takes turns with dP^T.
  static constexpr uint32_t S_COL = 0, DP_COL = NS * 64, DV_COL = DP_COL + 128, DK_COL = DV_COL + HD, DQ_COL = WIDE ? DP_COL : DK_COL + HD;
  static constexpr uint32_t K_COL = DQ_COL + HD, V_COL = K_COL + HD / 2;
  static_assert((WIDE ? DK_COL + HD : KV_TMEM ? V_COL + HD / 2 : DQ_COL + HD) <= 512, "tensor memory");
  static constexpr int OUT_COLS = HD / 4;                      // columns of dV and of dK one softmax warp carries out
};

// P of 32 query columns of one KV row: scores from tensor memory, -lse of the columns from shared memory; columns below
// `masked` come before the row (DIAG).
// WIN (with DIAG): columns [masked, masked + width) are seen.
template <bool DIAG, bool WIN = false>
__device__ __forceinline__ void attn_bwd_p(uint32_t t_s, const float* nlse, float2 sc2, int masked, float2* pr, uint32_t width = 0) {
#pragma unroll
  for (int c = 0; c < 32; c += 16) {
    uint32_t sv[16];
    tmem_ld16(t_s + c, sv);
    tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const float4 nl = *reinterpret_cast<const float4*>(nlse + c + i);
      const float2 x = ffma2(make_float2(__uint_as_float(sv[i]), __uint_as_float(sv[i + 1])), sc2, make_float2(nl.x, nl.y));
      const float2 y = ffma2(make_float2(__uint_as_float(sv[i + 2]), __uint_as_float(sv[i + 3])), sc2, make_float2(nl.z, nl.w));
      float2* o = pr + ((c + i) >> 1);
      o[0] = make_float2(ex2_approx(x.x), ex2_approx(x.y));
      o[1] = make_float2(ex2_approx(y.x), ex2_approx(y.y));
      if (WIN) {
        if ((uint32_t)(c + i - masked) >= width) o[0].x = 0.f;
        if ((uint32_t)(c + i + 1 - masked) >= width) o[0].y = 0.f;
        if ((uint32_t)(c + i + 2 - masked) >= width) o[1].x = 0.f;
        if ((uint32_t)(c + i + 3 - masked) >= width) o[1].y = 0.f;
      } else if (DIAG) {
        if (c + i < masked) o[0].x = 0.f;
        if (c + i + 1 < masked) o[0].y = 0.f;
        if (c + i + 2 < masked) o[1].x = 0.f;
        if (c + i + 3 < masked) o[1].y = 0.f;
      }
    }
  }
}

// Does some thread of the warp have a NaN among its 32 packed dS? A hidden pair's P is zero, but zero times dP - delta is NaN where do * v of
// the pair or do * o of the row overflow; hidden pairs are cleared then. Looked for behind the stores of dS, while they are on their way,
// and by warps that have hidden pairs only. In us with delta and conversion passes, without it / so / in front of the stores, in all
// warps of such tiles / as a select for each of their columns: 8 x 4096, 32 / 4 heads of 32, window 512 499 / 505 / 515 / 524; 16 / 8 of 64,
// window 1024 489 / 491 / 499 / 501; 2 x 4096, 16 / 4 of 128, window 2048 362 / 364 / 373 / 375.
__device__ __forceinline__ bool attn_bwd_any_nan(const uint32_t* dd) {
  const __nv_bfloat162* d = reinterpret_cast<const __nv_bfloat162*>(dd);
  const __nv_bfloat162 zero = __floats2bfloat162_rn(0.f, 0.f);
  __nv_bfloat162 a = d[0], b = d[1];
#pragma unroll
  for (int i = 2; i < 16; i += 2) { a = __hfma2(d[i], zero, a); b = __hfma2(d[i + 1], zero, b); }      // a, or NaN
  const float2 s = __bfloat1622float2(__hfma2(a, zero, b));
  return __any_sync(0xffffffffu, s.x != s.x || s.y != s.y);
}

// SPLIT: a cluster of p.split CTAs works on one KV tile, each on its share of the (query head, query tile) steps; every CTA
// leaves its fp32 dV | dK in its own shared memory and the cluster adds them up, in fixed order. See split_for.
template <int HD, bool SCATTER, bool SPLIT, bool WIN>
__global__ void __launch_bounds__(AB_THREADS, 1)
attn_bwd_kernel(const __grid_constant__ AttnBwdMaps<WIN> tm, const AttnBwdParams p) {
  static_assert(!(WIN && SCATTER), "the window has no head -> sequence return");
  using C = AttnBwdCfg<HD>;
  constexpr uint32_t TMEM_COLS = 512;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t sbase = smem_u32(smem_raw);
  uint8_t* sal = smem_raw;
  if (sbase & 1023u) {                                // swizzled tiles need a 1024-byte aligned base
    griddep_wait();
    if (threadIdx.x == 0) report_status(p.status, (20u << 8) | 2u);
    return;
  }
  const uint32_t bar0 = sbase + C::OFF_BAR;
  // barriers; [n] of a half, buffer, stage or score tile
  enum { KV_FULL = 0, KV_TMEM = 1, DP_FULL = 2 /* [2] */, PDS = 4 /* [2]: P^T, dS^T published */, DQ_FULL = 6 /* [2] */, DQ_FREE = 8,
         RING_FULL = 9 /* [3] */, RING_EMPTY = 12 /* [3] */, S_FULL = 15 /* [3] */, DO_FULL = 18, DO_EMPTY = 19, ALL_DONE = 20, N_BARS = 21 };
  auto bar = [&](int i) { return bar0 + 8u * i; };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sal + C::OFF_BAR + 192);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int n_tiles = (p.T + AB_TILE - 1) / AB_TILE;
  int j, bh;                                                  // KV tile (tile 0 has the most query tiles), (batch, KV head)
  const int split = SPLIT ? p.split : 1, rank = SPLIT ? (int)cluster_ctarank() : 0;
  int q_from, q_to, part = -1;                                // query tiles; slot of `part` that this block's sink rows go to
  if constexpr (WIN) {
    // A head's far pieces come in front of its tiles: they are as long, and what they read is read again by the group's tiles
    const int far_items = p.far.tiles * p.far.chunks;
    int rank;
    heavy_first_decode((int)blockIdx.x / split, n_tiles + far_items, p.B * p.Hkv, p.head_group, rank, bh);
    if (rank < far_items) {
      const int c = rank / p.far.tiles;
      j = rank - c * p.far.tiles;
      win_far_range(p.far, j, c, p.window, n_tiles, q_from, q_to);
      part = 1 + c;
    } else {
      j = rank - far_items;
      q_from = j;
      q_to = win_last_q(j, p.window, n_tiles) + 1;
      if (j < p.far.tiles) part = 0;
    }
  } else {
    heavy_first_decode((int)blockIdx.x / split, n_tiles, p.B * p.Hkv, p.head_group, j, bh);
    q_from = j;                                               // query tiles j..n_tiles-1
    q_to = n_tiles;
  }
  const int b = bh / p.Hkv, kvh = bh % p.Hkv;
  const int rep = p.Hq / p.Hkv;
  const int per_head = WIN && q_to < q_from ? 0 : q_to - q_from;
  const int it0 = SPLIT ? rep * per_head * rank / split : 0;                                       // this CTA's steps
  const int n_it = SPLIT ? rep * per_head * (rank + 1) / split - it0 : rep * per_head;             // (SPLIT: may be none)
  const int heads_total = p.Hq + 2 * p.Hkv;
  // query head and query tile of this CTA's first step; a step further is the next tile, behind the last one the next head's first
  const int hq0 = kvh * rep + (n_it > 0 ? it0 / per_head : 0), qi0 = q_from + (n_it > 0 ? it0 % per_head : 0);
  auto advance = [&](int& hq, int& qi) { if (++qi == q_to) { qi = q_from; ++hq; } };
  const CUtensorMap *tm_q, *tm_k, *tm_v;
  int k_head = kvh, v_head = kvh;
  if constexpr (WIN) { tm_q = &tm.q; tm_k = &tm.k; tm_v = &tm.v; }
  else { tm_q = tm_k = tm_v = &tm.qkv; k_head += p.Hq; v_head += p.Hq + p.Hkv; }
  // fp32 row of slot `part` for key t (dV, then dK)
  auto part_row = [&](int t) { return p.part + (((long long)bh * (1 + p.far.chunks) + part) * p.sinks + t) * (2 * HD); };

  if (threadIdx.x == 0) {
    for (int i = 0; i < N_BARS; ++i)
      mbar_init(bar(i), i == KV_TMEM ? 16 : (i == PDS || i == PDS + 1) ? 8 : i == DQ_FREE ? 4 : (i >= RING_FULL && i < RING_EMPTY) ? 2 : 1);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(tm_q);
    if (WIN) { tma_prefetch_desc(tm_k); tma_prefetch_desc(tm_v); }
    tma_prefetch_desc(&tm.dout);
    tma_prefetch_desc(&tm.dq);
  }
  if (warp == 1) { tmem_alloc(smem_u32(tmem_slot), TMEM_COLS); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  griddep_wait();

  if (warp == 0) {
    // ---------------------------------------------------------------- producer: Q, dO by TMA; -lse, -delta by the warp
    if (lane == 0) {
      mbar_expect_tx(bar(KV_FULL), (C::KV_TMEM ? 1 : 2) * C::TILE_BYTES);
#pragma unroll
      for (int kb = 0; kb < C::KB; ++kb) {
        tma_load_4d(sbase + C::OFF_K + kb * 16384, tm_k, bar(KV_FULL), kb * 64, k_head, j * AB_TILE, b);
        if (!C::KV_TMEM) tma_load_4d(sbase + C::OFF_V + kb * 16384, tm_v, bar(KV_FULL), kb * 64, v_head, j * AB_TILE, b);
      }
    }
    for (int it = 0, hq = hq0, qi = qi0; it < n_it; ++it, advance(hq, qi)) {
      const int st = it % C::STAGES;
      if (!mbar_wait_warp(bar(RING_EMPTY + st), ((uint32_t)(it / C::STAGES) & 1u) ^ 1u, 21, abort_flag, p.status)) break;
      if (lane == 0) {
        mbar_expect_tx(bar(RING_FULL + st), (C::WIDE ? 1 : 2) * C::TILE_BYTES);
#pragma unroll
        for (int kb = 0; kb < C::KB; ++kb)
          tma_load_4d(sbase + C::OFF_Q + st * C::TILE_BYTES + kb * 16384, tm_q, bar(RING_FULL + st), kb * 64, hq, qi * AB_TILE, b);
        if (!C::WIDE) tma_load_4d(sbase + C::OFF_DO + st * C::TILE_BYTES, &tm.dout, bar(RING_FULL + st), 0, hq, qi * AB_TILE, b);
      }
      constexpr float LOG2E = 1.4426950408889634f;
      const long long r0 = ((long long)b * p.Hq + hq) * p.T;
      float* rows = reinterpret_cast<float*>(sal + C::OFF_ROW) + st * 2 * AB_TILE;
      float l[4], d[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int t = qi * AB_TILE + 32 * k + lane;
        l[k] = t < p.T ? p.lse[r0 + t] * -LOG2E : -INFINITY;               // rows past the end: P = 0
        d[k] = t < p.T ? -p.delta[r0 + t] : 0.f;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) { rows[32 * k + lane] = l[k]; rows[AB_TILE + 32 * k + lane] = d[k]; }
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(RING_FULL + st));
      if constexpr (C::WIDE) {
        if (!mbar_wait_warp(bar(DO_EMPTY), ((uint32_t)it & 1u) ^ 1u, 35, abort_flag, p.status)) break;
        if (lane == 0) {
          mbar_expect_tx(bar(DO_FULL), C::TILE_BYTES);
#pragma unroll
          for (int kb = 0; kb < C::KB; ++kb)
            tma_load_4d(sbase + C::OFF_DO + kb * 16384, &tm.dout, bar(DO_FULL), kb * 64, hq, qi * AB_TILE, b);
        }
      }
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA issuer
    const uint32_t el = elect_one();
    constexpr uint32_t idesc_s = umma_idesc_bf16(AB_TILE, 64, 0, 0);          // S^T, dP^T of one half: B K-major
    constexpr uint32_t idesc_t = umma_idesc_bf16(AB_TILE, HD, 0, 1);          // dV, dK: A from tensor memory, B MN-major
    constexpr uint32_t idesc_q = umma_idesc_bf16(AB_TILE, HD, 1, 1);          // dQ    : A, B MN-major
    const uint64_t dk_mn = attn_desc_mn<HD>(sbase + C::OFF_K);
    // Half step h = 2 it + s: query columns 64 s .. 64 s + 63 of step it, scores in tile h % NS. Which tile and which ring stage
    // is carried along instead of computed from h, and s is a constant of the unrolled body: both keep the operands uniform.
    const uint64_t dk_k = attn_desc_k<HD>(sbase + C::OFF_K), dv_k = attn_desc_k<HD>(sbase + C::OFF_V);
    const uint64_t q_k = attn_desc_k<HD>(sbase + C::OFF_Q), do_k = attn_desc_k<HD>(sbase + C::OFF_DO);
    const uint64_t q_mn = attn_desc_mn<HD>(sbase + C::OFF_Q), do_mn = attn_desc_mn<HD>(sbase + C::OFF_DO);
    auto issue_sp = [&](uint32_t d, uint32_t a_tmem, uint64_t a_smem, uint64_t db) {
#pragma unroll
      for (int t = 0; t < HD / 16; ++t) {
        if constexpr (C::KV_TMEM) umma_bf16_ts_w(el, d, a_tmem + t * 8, umma_desc_advance(db, t * 32), idesc_s, t > 0);
        else umma_bf16_w(el, d, umma_desc_advance(a_smem, t * 32), umma_desc_advance(db, t * 32), idesc_s, t > 0);
      }
    };
    auto ring = [&](int it, int st) -> bool {
      const bool r = mbar_wait_warp(bar(RING_FULL + st), (uint32_t)(it / C::STAGES) & 1u, 22, abort_flag, p.status);
      tc_fence_after();
      return r;
    };
    auto issue_s = [&](int sb, int st, int s) {
      issue_sp(tmem + C::S_COL + sb * 64, tmem + C::K_COL, dk_k, umma_desc_advance(q_k, st * C::TILE_BYTES + s * (C::TILE_BYTES / 2)));
      umma_commit_w(el, bar(S_FULL + sb));
    };
    auto issue_dp = [&](int st, int s) {
      issue_sp(tmem + C::DP_COL + s * 64, tmem + C::V_COL, dv_k, umma_desc_advance(do_k, st * C::TILE_BYTES + s * (C::TILE_BYTES / 2)));
      umma_commit_w(el, bar(DP_FULL + s));
    };
    bool ok = mbar_wait_warp(bar(KV_FULL), 0, 23, abort_flag, p.status);
    if (ok && C::KV_TMEM) ok = mbar_wait_warp(bar(KV_TMEM), 0, 34, abort_flag, p.status);
    tc_fence_after();
    if constexpr (C::WIDE) {
      // One order of five products a step; S^T and dP^T of both halves in one piece (half the reads of K and V).
      constexpr uint32_t idesc_w = umma_idesc_bf16(AB_TILE, AB_TILE, 0, 0);
      auto issue_kk = [&](uint32_t d, uint64_t a, uint64_t bm) {
#pragma unroll
        for (int t = 0; t < HD / 16; ++t) {
          const uint32_t off = (t >> 2) * 16384 + (t & 3) * 32;
          umma_bf16_w(el, d, umma_desc_advance(a, off), umma_desc_advance(bm, off), idesc_w, t > 0);
        }
      };
      auto issue_dp_w = [&](int it) -> bool {
        if (!mbar_wait_warp(bar(DO_FULL), (uint32_t)it & 1u, 36, abort_flag, p.status)) return false;
        tc_fence_after();
        issue_kk(tmem + C::DP_COL, dv_k, do_k);
        umma_commit_w(el, bar(DP_FULL));
        return true;
      };
      const uint64_t dds_mn = umma_smem_desc(sbase + C::OFF_DS, 16384, 1024);
      if (ok && n_it > 0 && (ok = ring(0, 0))) {
        issue_kk(tmem + C::S_COL, dk_k, q_k);
        umma_commit_w(el, bar(S_FULL));
        ok = issue_dp_w(0);
      }
      for (int it = 0; it < n_it && ok; ++it) {
        const int st = it & 1;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          if (!(ok = mbar_wait_warp(bar(PDS + s), (uint32_t)it & 1u, 26, abort_flag, p.status))) break;
          tc_fence_after();
          if (s == 1) {                                 // first, so that its way out runs beside the products after it
#pragma unroll
            for (int t = 0; t < AB_TILE / 16; ++t)
              umma_bf16_w(el, tmem + C::DQ_COL, umma_desc_advance(dds_mn, t * 2048), umma_desc_advance(dk_mn, t * 2048), idesc_q, t > 0);
            umma_commit_w(el, bar(DQ_FULL));
          }
          const uint64_t dq = umma_desc_advance(q_mn, st * C::TILE_BYTES + s * 8192), ddo = umma_desc_advance(do_mn, s * 8192);
          const uint32_t t_s = tmem + C::S_COL + s * 64;
#pragma unroll
          for (int t = 0; t < 4; ++t)
            umma_bf16_ts_w(el, tmem + C::DV_COL, t_s + (t >> 1) * 32 + (t & 1) * 8, umma_desc_advance(ddo, t * 2048), idesc_t, (it > 0) | (s > 0) | (t > 0));
          if (s == 1) umma_commit_w(el, bar(DO_EMPTY));
#pragma unroll
          for (int t = 0; t < 4; ++t)
            umma_bf16_ts_w(el, tmem + C::DK_COL, t_s + 16 + (t >> 1) * 32 + (t & 1) * 8, umma_desc_advance(dq, t * 2048), idesc_t, (it > 0) | (s > 0) | (t > 0));
        }
        if (!ok) break;
        umma_commit_w(el, bar(RING_EMPTY + st));
        if (it + 1 < n_it) {
          if (!(ok = ring(it + 1, st ^ 1))) break;
          issue_kk(tmem + C::S_COL, dk_k, umma_desc_advance(q_k, (st ^ 1) * C::TILE_BYTES));
          umma_commit_w(el, bar(S_FULL));
          if (!(ok = mbar_wait_warp(bar(DQ_FREE), (uint32_t)it & 1u, 27, abort_flag, p.status))) break;     // dQ(it) is out of the dP columns
          if (!(ok = issue_dp_w(it + 1))) break;
        }
      }
    } else {
      if (ok && n_it > 0 && (ok = ring(0, 0))) {
        issue_s(0, 0, 0);
        issue_dp(0, 0);
        issue_s(1, 0, 1);
        issue_dp(0, 1);
        if (n_it > 1 && (ok = ring(1, 1))) issue_s(2, 1, 0);
      }
      int st = 0, sb = 0;
      for (int it = 0; it < n_it && ok; ++it) {
        const int st1 = st == C::STAGES - 1 ? 0 : st + 1, st2 = st1 == C::STAGES - 1 ? 0 : st1 + 1;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          if (!(ok = mbar_wait_warp(bar(PDS + s), (uint32_t)it & 1u, 26, abort_flag, p.status))) break;
          tc_fence_after();
          if (it + 1 < n_it) issue_dp(st1, s);           // needed first; its columns were read before P^T and dS^T were published
          const uint64_t dq = umma_desc_advance(q_mn, st * C::TILE_BYTES + s * (C::TILE_BYTES / 2));
          const uint64_t ddo = umma_desc_advance(do_mn, st * C::TILE_BYTES + s * (C::TILE_BYTES / 2));
          const uint32_t t_s = tmem + C::S_COL + sb * 64;
#pragma unroll
          for (int t = 0; t < 4; ++t)
            umma_bf16_ts_w(el, tmem + C::DV_COL, t_s + (t >> 1) * 32 + (t & 1) * 8, umma_desc_advance(ddo, t * attn_mn_step<HD>()), idesc_t, (it > 0) | (s > 0) | (t > 0));
#pragma unroll
          for (int t = 0; t < 4; ++t)
            umma_bf16_ts_w(el, tmem + C::DK_COL, t_s + 16 + (t >> 1) * 32 + (t & 1) * 8, umma_desc_advance(dq, t * attn_mn_step<HD>()), idesc_t, (it > 0) | (s > 0) | (t > 0));
          // the tensor pipe works in order: these scores replace the P^T / dS^T that were just read
          if (s == 0) {
            if (it + 1 < n_it) issue_s(sb, st1, 1);
          } else if (it + 2 < n_it) {
            if (!(ok = ring(it + 2, st2))) break;
            issue_s(sb, st2, 0);
          }
          sb = sb == C::NS - 1 ? 0 : sb + 1;
        }
        if (!ok) break;
        if (it > 0 && !(ok = mbar_wait_warp(bar(DQ_FREE), ((uint32_t)it & 1u) ^ 1u, 27, abort_flag, p.status))) break;     // dQ(it-1) is in registers
        tc_fence_after();
        const uint64_t dds_mn = umma_smem_desc(sbase + C::OFF_DS + (it & 1) * C::DS_BYTES, 16384, 1024);
#pragma unroll
        for (int t = 0; t < AB_TILE / 16; ++t)
          umma_bf16_w(el, tmem + C::DQ_COL, umma_desc_advance(dds_mn, t * 2048), umma_desc_advance(dk_mn, t * attn_mn_step<HD>()), idesc_q, t > 0);
        umma_commit_w(el, bar(DQ_FULL + (it & 1)));       // dQ ready, this dS buffer free
        umma_commit_w(el, bar(RING_EMPTY + st));
        st = st1;
      }
    }
    if (ok && n_it > 0) umma_commit_w(el, bar(ALL_DONE));
    griddep_launch();
  } else if (warp < 18) {
    // ---------------------------------------------------------------- softmax warps: 32 query columns of 32 KV rows each
    const int q4 = warp & 3, g = (warp - 2) >> 2, s = g >> 1;
    const int row = q4 * 32 + lane;                           // row of the KV tile
    const int t_row = j * AB_TILE + row;
    const uint32_t t_lane = tmem + ((uint32_t)(q4 * 32) << 16);
    bool ok = true;
    if constexpr (C::KV_TMEM) {   // K (warps of half 0) and V (half 1) rows become tensor-memory operands, half a row per warp
      static_assert(HD == 32, "half a row is 16 columns, 8 words; p.hd is HD (the scatter form has wider tiles)");
      const int c0 = (g & 1) * 16;
      const __nv_bfloat16* src = WIN ? (s == 0 ? p.k + b * p.ks[0] + t_row * p.ks[1] + kvh * p.ks[2] : p.v + b * p.vs[0] + t_row * p.vs[1] + kvh * p.vs[2]) + c0
                                     : p.qkv + (((long long)b * p.T + t_row) * heads_total + p.Hq + s * p.Hkv + kvh) * HD + c0;
      uint32_t w[8];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const uint4 v = t_row < p.T ? reinterpret_cast<const uint4*>(src)[c] : make_uint4(0, 0, 0, 0);
        w[4 * c] = v.x; w[4 * c + 1] = v.y; w[4 * c + 2] = v.z; w[4 * c + 3] = v.w;
      }
      tmem_st8(t_lane + (s == 0 ? C::K_COL : C::V_COL) + c0 / 2, w);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(KV_TMEM));
    }
    const float2 sc2 = make_float2(p.scale_log2, p.scale_log2);
    const int col0 = (g & 1) * 32;                             // of the half's 64 query columns
    for (int it = 0, hq = hq0, qi = qi0; it < n_it; ++it, advance(hq, qi)) {
      const int st = it % C::STAGES;
      const float* rows = reinterpret_cast<const float*>(sal + C::OFF_ROW) + st * 2 * AB_TILE + s * 64 + col0;
      uint8_t* drow = sal + C::OFF_DS + (C::WIDE ? 0 : it & 1) * C::DS_BYTES + s * 16384 + row * 128;
      if (!mbar_wait_warp(bar(RING_FULL + st), (uint32_t)(it / C::STAGES) & 1u, 28, abort_flag, p.status)) { ok = false; break; }
      const int h = 2 * it + s, sb = C::WIDE ? 0 : h % C::NS;
      const uint32_t t_s = t_lane + C::S_COL + (C::WIDE ? s : sb) * 64 + col0, t_dp = t_lane + C::DP_COL + s * 64 + col0;
      if (!mbar_wait_warp(bar(S_FULL + sb), (uint32_t)(C::WIDE ? it : h / C::NS) & 1u, 29, abort_flag, p.status)) { ok = false; break; }
      tc_fence_after();
      float2 pr[16];
      // two copies: the compare and select of the diagonal tiles doubled the instructions of a pair in all the others
      // WIN: columns [first, first + width) of a row are seen; `masked`: not all of them in all of this warp's rows
      const int first0 = (j - qi) * AB_TILE + q4 * 32 - s * 64 - col0, first = first0 + lane;
      const bool masked = WIN && win_block_partial(j, first0, p.window, p.sinks);
      const uint32_t width = t_row < p.sinks ? 0x80000000u : (uint32_t)p.window;
      if constexpr (WIN) {
        if (masked) attn_bwd_p<true, true>(t_s, rows, sc2, first, pr, width);
        else attn_bwd_p<false>(t_s, rows, sc2, 0, pr);
      } else if (qi == j) attn_bwd_p<true>(t_s, rows, sc2, row - s * 64 - col0, pr);
      else attn_bwd_p<false>(t_s, rows, sc2, 0, pr);
      {
        uint32_t pp[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) pp[i] = pack_bf16(pr[i].x, pr[i].y);
        tmem_st16(t_s, pp);
      }
      if (!mbar_wait_warp(bar(DP_FULL + (C::WIDE ? 0 : s)), (uint32_t)it & 1u, 33, abort_flag, p.status)) { ok = false; break; }
      tc_fence_after();
      uint32_t dd[16];
#pragma unroll
      for (int c = 0; c < 32; c += 16) {
        uint32_t dp[16];
        tmem_ld16(t_dp + c, dp);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
          const float4 nd = *reinterpret_cast<const float4*>(rows + AB_TILE + c + i);
          // dS = P (dP - delta); the softmax scale is applied once, when dQ and dK leave their accumulators
          const float2 d0 = fmul2(pr[(c + i) >> 1], fadd2(make_float2(__uint_as_float(dp[i]), __uint_as_float(dp[i + 1])), make_float2(nd.x, nd.y)));
          const float2 d1 = fmul2(pr[((c + i) >> 1) + 1], fadd2(make_float2(__uint_as_float(dp[i + 2]), __uint_as_float(dp[i + 3])), make_float2(nd.z, nd.w)));
          dd[(c + i) >> 1] = pack_bf16(d0.x, d0.y);
          dd[((c + i) >> 1) + 1] = pack_bf16(d1.x, d1.y);
        }
      }
      tmem_st16(t_s + 16, dd);
      if (!C::WIDE && it > 1 && !mbar_wait_warp(bar(DQ_FULL + (it & 1)), ((uint32_t)(it >> 1) & 1u) ^ 1u, 30, abort_flag, p.status)) { ok = false; break; }
      auto store_ds = [&] {
#pragma unroll
        for (int ch = 0; ch < 4; ++ch)
          *reinterpret_cast<uint4*>(drow + ((((col0 >> 3) + ch) ^ (row & 7)) << 4)) = make_uint4(dd[4 * ch], dd[4 * ch + 1], dd[4 * ch + 2], dd[4 * ch + 3]);
      };
      store_ds();
      if (masked && attn_bwd_any_nan(dd)) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          if ((uint32_t)(2 * i - first) >= width) dd[i] &= 0xffff0000u;
          if ((uint32_t)(2 * i + 1 - first) >= width) dd[i] &= 0x0000ffffu;
        }
        __syncwarp();
        tmem_st_wait();                                        // the first stores; nothing orders two to the same place
        tmem_st16(t_s + 16, dd);
        store_ds();
      }
      fence_proxy_async_smem();
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(PDS + s));
    }
    if (ok && n_it > 0) ok = mbar_wait_warp(bar(ALL_DONE), 0, 31, abort_flag, p.status);
    tc_fence_after();
    constexpr int W = C::OUT_COLS;
    const int out0 = g * W;                                    // first of this warp's columns of dV and dK
    auto load_out = [&](uint32_t col, uint32_t* r) {
      if constexpr (W == 8) tmem_ld8(t_lane + col, r);
      else if constexpr (W == 16) tmem_ld16(t_lane + col, r);
      else tmem_ld32(t_lane + col, r);
      tmem_ld_wait();
    };
    if (ok && !SPLIT && !WIN) {
      // dV, dK accumulators -> bf16 rows of the packed gradient tensor
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        const float osc = which == 0 ? 1.f : p.scale;
        __nv_bfloat16* dst = p.dqkv + (((long long)b * p.T + t_row) * heads_total + (which == 0 ? p.Hq + p.Hkv : p.Hq) + kvh) * p.hd + out0;
        bool dst_ok = t_row < p.T && out0 < p.hd;
        if (SCATTER && p.n_dst > 0) {
          const int owner = t_row / p.dst_rows, tl = t_row - owner * p.dst_rows;
          dst_ok = dst_ok && owner < p.n_dst;
          if (dst_ok)
            dst = p.dst[owner] + (((long long)b * p.dst_rows + tl) * p.dst_heads + (which == 0 ? p.dst_v0 : p.dst_k0) + kvh) * p.hd + out0;
        }
        uint32_t r[W];
        load_out((which == 0 ? C::DV_COL : C::DK_COL) + out0, r);
        if (SCATTER && which == 1 && p.cosT != nullptr && out0 < p.hd) {
          // transposed RoPE on dK (fp32): column j pairs with j +- hd / 2 (the condition is the warp's, as the load needs)
          const bool low = out0 < p.hd / 2;
          const int pc = low ? out0 + p.hd / 2 : out0 - p.hd / 2;      // partner's first column
          uint32_t q2[W];
          load_out(C::DK_COL + pc, q2);
          if (t_row < p.T) {
            const float* cr = p.cosT + (long long)t_row * p.hd;
            const float* sr = p.sinT + (long long)t_row * p.hd;
#pragma unroll
            for (int i = 0; i < W; ++i) {
              const float a = __uint_as_float(r[i]), bb = __uint_as_float(q2[i]);
              r[i] = __float_as_uint(low ? a * cr[out0 + i] + bb * sr[pc + i] : a * cr[out0 + i] - bb * sr[pc + i]);
            }
          }
        }
        if (dst_ok) {
#pragma unroll
          for (int i = 0; i < W; i += 8) {
            uint4 v;
            v.x = pack_bf16(__uint_as_float(r[i]) * osc, __uint_as_float(r[i + 1]) * osc);
            v.y = pack_bf16(__uint_as_float(r[i + 2]) * osc, __uint_as_float(r[i + 3]) * osc);
            v.z = pack_bf16(__uint_as_float(r[i + 4]) * osc, __uint_as_float(r[i + 5]) * osc);
            v.w = pack_bf16(__uint_as_float(r[i + 6]) * osc, __uint_as_float(r[i + 7]) * osc);
            *reinterpret_cast<uint4*>(dst + i) = v;
          }
        }
      }
    }
    if constexpr (WIN && !SPLIT) {
      // dV and dK as bf16 through shared memory (where dS was; every MMA that reads it is done), so that a row leaves in one piece: written
      // from the accumulators' layout, 16 bytes of 32 rows at a time, it took 3100 cycles. Rows whose sums go to `part` leave as fp32.
      constexpr int PASSES = C::WIDE ? 2 : 1, CHUNKS = 2 * HD / PASSES / 8;      // 16-byte chunks of a row of the stage
      uint8_t* stage = sal + C::OFF_DS;
      const bool summed = part >= 0 && t_row < p.sinks;
#pragma unroll
      for (int pass = 0; pass < PASSES; ++pass) {
#pragma unroll
        for (int w = 0; w < 2 / PASSES; ++w) {
          const int which = PASSES == 2 ? pass : w;
          const float osc = which == 0 ? 1.f : p.scale;
          uint32_t r[W];
          load_out((which == 0 ? C::DV_COL : C::DK_COL) + out0, r);
          if (summed) {
            uint4* d = reinterpret_cast<uint4*>(part_row(t_row) + which * HD + out0);
#pragma unroll
            for (int i = 0; i < W; i += 4) d[i / 4] = n_it > 0 ? make_uint4(r[i], r[i + 1], r[i + 2], r[i + 3]) : make_uint4(0, 0, 0, 0);
          }
#pragma unroll
          for (int i = 0; i < W; i += 8) {
            uint4 v;
            v.x = pack_bf16(__uint_as_float(r[i]) * osc, __uint_as_float(r[i + 1]) * osc);
            v.y = pack_bf16(__uint_as_float(r[i + 2]) * osc, __uint_as_float(r[i + 3]) * osc);
            v.z = pack_bf16(__uint_as_float(r[i + 4]) * osc, __uint_as_float(r[i + 5]) * osc);
            v.w = pack_bf16(__uint_as_float(r[i + 6]) * osc, __uint_as_float(r[i + 7]) * osc);
            *reinterpret_cast<uint4*>(stage + row * (CHUNKS * 16) + (((w * HD + out0 + i) / 8 ^ (row & 7)) << 4)) = v;
          }
        }
        __syncwarp();
        asm volatile("bar.sync 2, 512;" ::: "memory");            // the softmax warps; all of them come here, on an error too
        if (ok && part <= 0) {
          for (int i = threadIdx.x - 64; i < AB_TILE * CHUNKS; i += 512) {
            const int r = i / CHUNKS, ch = i % CHUNKS, t = j * AB_TILE + r, which = PASSES == 2 ? pass : ch * 8 / HD;
            if (t >= p.T || (part == 0 && t < p.sinks)) continue;
            __nv_bfloat16* dst = which == 0 ? p.dv + b * p.dvs[0] + t * p.dvs[1] + kvh * p.dvs[2] : p.dk + b * p.dks[0] + t * p.dks[1] + kvh * p.dks[2];
            *reinterpret_cast<uint4*>(dst + ch * 8 % HD) = *reinterpret_cast<const uint4*>(stage + r * (CHUNKS * 16) + ((ch ^ (r & 7)) << 4));
          }
        }
        if (pass + 1 < PASSES) {
          __syncwarp();
          asm volatile("bar.sync 2, 512;" ::: "memory");
        }
      }
    }
    if constexpr (SPLIT) {
      // this CTA's dV | dK, over the Q / dO ring: every MMA and every row of the ring has been read (WIDE: over the dQ boxes too)
      if (C::WIDE) {
        __syncwarp();
        asm volatile("bar.sync 1, 640;" ::: "memory");
      }
      float* part = reinterpret_cast<float*>(sal + C::OFF_Q) + row * C::PART_PITCH + out0;
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        uint32_t r[W];
        load_out((which == 0 ? C::DV_COL : C::DK_COL) + out0, r);
#pragma unroll
        for (int i = 0; i < W; i += 4)
          *reinterpret_cast<uint4*>(part + which * HD + i) =
              n_it > 0 ? make_uint4(r[i], r[i + 1], r[i + 2], r[i + 3]) : make_uint4(0, 0, 0, 0);      // no step: nothing was accumulated
      }
    }
  } else {
    // ---------------------------------------------------------------- dQ of every step -> fp32 accumulator in global memory
    const int q4 = warp & 3;
    const uint32_t t_lane = tmem + ((uint32_t)(q4 * 32) << 16);
    const int box0 = C::OFF_DQS + q4 * C::BOXES * 4096;
    for (int it = 0, hq = hq0, qi = qi0; it < n_it; ++it, advance(hq, qi)) {
      const int y0 = qi * AB_TILE + q4 * 32;                  // first of this warp's 32 query rows
      if (!mbar_wait_warp(bar(DQ_FULL + (C::WIDE ? 0 : it & 1)), (uint32_t)(C::WIDE ? it : it >> 1) & 1u, 32, abort_flag, p.status)) break;
      tc_fence_after();
      constexpr int COLS = HD < 64 ? HD : 64;                 // in registers at a time
#pragma unroll
      for (int c0 = 0; c0 < HD; c0 += COLS) {
        uint32_t r[COLS];
#pragma unroll
        for (int c = 0; c < COLS; c += 32) tmem_ld32(t_lane + C::DQ_COL + c0 + c, r + c);
        tmem_ld_wait();
        if (c0 + COLS == HD) {                                // all of it has been read: the columns are free
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(DQ_FREE));
        }
#pragma unroll
        for (int c = 0; c < COLS; c += 32 * C::BOXES) {
          if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");      // staging boxes free again
          __syncwarp();
#pragma unroll
          for (int x = 0; x < C::BOXES; ++x) {
            uint8_t* rowp = sal + box0 + x * 4096 + lane * 128;
            const uint32_t* v = r + c + 32 * x;
#pragma unroll
            for (int ch = 0; ch < 8; ++ch)
              *reinterpret_cast<uint4*>(rowp + ((ch ^ (lane & 7)) << 4)) = make_uint4(v[4 * ch], v[4 * ch + 1], v[4 * ch + 2], v[4 * ch + 3]);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
#pragma unroll
            for (int x = 0; x < C::BOXES; ++x)
              if (y0 < p.T && c0 + c + 32 * x < p.hd)
                asm volatile("cp.reduce.async.bulk.tensor.3d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3, %4}], [%1];"
                             ::"l"((uint64_t)&tm.dq), "r"(sbase + box0 + x * 4096), "r"(c0 + c + 32 * x), "r"(y0), "r"(b * p.Hq + hq) : "memory");
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          }
        }
      }
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");      // dQ reductions have left shared memory and landed
    if (SPLIT && C::WIDE) {
      __syncwarp();
      asm volatile("bar.sync 1, 640;" ::: "memory");
    }
  }
  if constexpr (SPLIT) {
    __syncwarp();
    tc_fence_before();
    cluster_sync_all();
    // rows [128 rank / split, 128 (rank + 1) / split) of the sum, in place (nobody else reads these rows of this CTA's part)
    float* base = reinterpret_cast<float*>(sal + C::OFF_Q);
    const int rows = AB_TILE / split, r0 = rank * rows;
    for (int i = threadIdx.x; i < rows * (HD / 2); i += AB_THREADS) {
      const int r = r0 + i / (HD / 2), c = (i % (HD / 2)) * 4;
      const uint32_t off = sbase + C::OFF_Q + (uint32_t)(r * C::PART_PITCH + c) * 4u;
      float4 a[8];
#pragma unroll
      for (int q = 0; q < 8; ++q)
        if (q < split) a[q] = ld_cluster_f4(mapa_shared(off, (uint32_t)q));
#pragma unroll
      for (int q = 1; q < 8; ++q)
        if (q < split) { a[0].x += a[q].x; a[0].y += a[q].y; a[0].z += a[q].z; a[0].w += a[q].w; }
      *reinterpret_cast<float4*>(base + r * C::PART_PITCH + c) = a[0];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < rows * (HD / 4); i += AB_THREADS) {
      const int r = r0 + i / (HD / 4), c = (i % (HD / 4)) * 8, t_row = j * AB_TILE + r;
      if (t_row >= p.T) continue;
      const bool is_k = c >= HD;
      const float osc = is_k ? p.scale : 1.f;
      const float* v = base + r * C::PART_PITCH + c;
      if constexpr (WIN) {
        if (part >= 0 && t_row < p.sinks) {
          float* d = part_row(t_row) + c;                       // dV | dK, as they lie here
          *reinterpret_cast<float4*>(d) = *reinterpret_cast<const float4*>(v);
          *reinterpret_cast<float4*>(d + 4) = *reinterpret_cast<const float4*>(v + 4);
          continue;
        }
        if (part > 0) continue;
      }
      uint4 o;
      o.x = pack_bf16(v[0] * osc, v[1] * osc); o.y = pack_bf16(v[2] * osc, v[3] * osc);
      o.z = pack_bf16(v[4] * osc, v[5] * osc); o.w = pack_bf16(v[6] * osc, v[7] * osc);
      __nv_bfloat16* dst;
      if constexpr (WIN) dst = is_k ? p.dk + b * p.dks[0] + t_row * p.dks[1] + kvh * p.dks[2] : p.dv + b * p.dvs[0] + t_row * p.dvs[1] + kvh * p.dvs[2];
      else dst = p.dqkv + (((long long)b * p.T + t_row) * heads_total + (is_k ? p.Hq : p.Hq + p.Hkv) + kvh) * p.hd;
      *reinterpret_cast<uint4*>(dst + (c - (is_k ? HD : 0))) = o;
    }
    cluster_sync_all();                // no CTA leaves while another may still read its part
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) { tc_fence_after(); tmem_dealloc(tmem, TMEM_COLS); }
}

// CTAs per KV tile. One CTA per KV tile walks over all its query heads and tiles, so the tile with the most steps bounds the
// launch from below however idle the chip is. A cluster divides that, but every CTA of a cluster costs about 5.4 steps
// (start-up and the exchange of dV and dK while its SM has no other CTA). The estimate is the longer of a CTA's own time and the
// work per SM; its pick was within 1 % of the fastest of 1, 2, 4, 8 on seventeen measured shapes of all head dims. With delta and
// conversion passes, in us, unsplit -> picked: 1 x 8192, 8 / 1 heads of 64 680 -> 194; 4 x 777, 16 / 2 94 -> 51; 3 x 1001, 12 / 4
// 50 -> 40; 1 x 1074, 8 / 2 of 128 108 -> 41; 2 x 256, 8 / 2 of 32 20 -> 14.
// `heaviest`: steps of the longest block, `tiles`: blocks, `total`: steps of all.
static int split_for(double heaviest, double tiles, double total) {
  const char* v = getenv("TLM_ATTN_BWD_SPLIT");          // 1, 2, 4 or 8: for tests and measurements
  const int forced = v != nullptr ? atoi(v) : 0;
  if (forced == 1 || forced == 2 || forced == 4 || forced == 8) return forced;
  const double sms = num_sms();
  int best = 1;
  double best_cost = heaviest > total / sms ? heaviest : total / sms;
  for (int s = 2; s <= 8; s *= 2) {
    const double own = heaviest / s + 3.0, shared = (total + 5.4 * tiles * s) / sms, cost = own > shared ? own : shared;
    if (cost < best_cost) { best_cost = cost; best = s; }
  }
  return best;
}

template <int HD, bool SCATTER, bool SPLIT = false, bool WIN = false>
static int launch_bwd(const AttnBwdMaps<WIN>& maps, const AttnBwdParams& p, cudaStream_t st) {
  constexpr int smem = AttnBwdCfg<HD>::TOTAL;
  auto kern = attn_bwd_kernel<HD, SCATTER, SPLIT, WIN>;
  static SmemConfigured configured;
  if (const int e = configured.set(kern, smem)) return e;
  const int grid = ((p.T + AB_TILE - 1) / AB_TILE + (WIN ? p.far.tiles * p.far.chunks : 0)) * p.B * p.Hkv;
  return launch_overlapped(kern, dim3((unsigned)(grid * (SPLIT ? p.split : 1))), dim3(AB_THREADS), smem, st, SPLIT ? p.split : 1, maps, p);
}

// fp32 [B*Hq, T, hd] accumulator, box 32 x 32 x 1
static int make_dq_map(CUtensorMap* map, const float* dq_acc, int B, int T, int Hq, int hd) {
  uint64_t dims[3] = {(uint64_t)hd, (uint64_t)T, (uint64_t)B * Hq};
  uint64_t strides[2] = {(uint64_t)hd * 4, (uint64_t)T * hd * 4};
  uint32_t box[3] = {32, 32, 1};
  return make_tmap_f32(map, dq_acc, 3, dims, strides, box);
}

// delta [B, Hq, T] and a dQ accumulator of zeros
static int launch_delta(const void* o, const void* o_rest, int rest_rows, const void* dout, float* delta, float* dq_acc, int B, int T, int Hq, int hd,
                        cudaStream_t st) {
  // Few blocks would take longer over the zeroes than a memset (48 heads of 64, 16 rows: one block, 3 us more)
  const int delta_blocks = B * ((T + DELTA_T - 1) / DELTA_T);
  const bool fused_zero = delta_blocks >= num_sms();
  if (!fused_zero) {
    const cudaError_t ce = cudaMemsetAsync(dq_acc, 0, (size_t)B * T * Hq * hd * 4, st);
    if (ce != cudaSuccess) return (int)ce;
  }
  return launch_overlapped(o_rest != nullptr ? attn_delta_kernel<true> : attn_delta_kernel<false>, dim3(delta_blocks), dim3(DELTA_THREADS),
      (size_t)Hq * (DELTA_T + 1) * 4, st, 1, (const __nv_bfloat16*)o, (const __nv_bfloat16*)o_rest, (const __nv_bfloat16*)dout, delta, fused_zero ? dq_acc : nullptr, B, T, Hq, hd, rest_rows);
}

}  // namespace tlm

using namespace tlm;

// dq_acc: fp32 scratch [B,Hq,T,hd]; delta: fp32 scratch [B,Hq,T]. Both are owned by the caller.
// cosT / sinT (optional, fp32 [T, hd]): the transposed RoPE is applied to dQ and dK on the way out.
// dst_ptrs (optional, n_dst > 0): head -> sequence return, see AttnBwdParams; dqkv may then be null.
static int attn_bwd_impl(const void* qkv, const void* o, const void* dout, const float* lse, void* dqkv,
                         float* dq_acc, float* delta, int B, int T, int Hq, int Hkv, int hd, float scale,
                         const float* cosT, const float* sinT, void* const* dst_ptrs, int n_dst, int dst_rows,
                         int dst_heads, int dst_q0, int dst_k0, int dst_v0, cudaStream_t st) {
  if (hd != 32 && hd != 64 && hd != 128) return -4;
  if (Hq % Hkv != 0) return -5;
  if ((size_t)Hq * (DELTA_T + 1) * 4 > 48 * 1024) return -6;
  const int le = launch_delta(o, nullptr, 0, dout, delta, dq_acc, B, T, Hq, hd, st);
  if (le) return le;
  AttnBwdMaps<false> maps;
  const int box_cols = hd == 32 && n_dst == 0 ? 32 : 64;
  int e = make_qkv_map(&maps.qkv, qkv, B, T, Hq + 2 * Hkv, hd, AB_TILE, box_cols);
  if (e) return e;
  e = make_qkv_map(&maps.dout, dout, B, T, Hq, hd, AB_TILE, box_cols);
  if (e) return e;
  if ((cosT == nullptr) != (sinT == nullptr)) return -6;
  if (n_dst < 0 || n_dst > AB_MAX_DST || (n_dst > 0 && (dst_ptrs == nullptr || dst_rows <= 0 || (long long)dst_rows * n_dst < T)))
    return -6;
  if (n_dst == 0 && dqkv == nullptr) return -6;
  AttnBwdParams p{};
  p.qkv = (const __nv_bfloat16*)qkv; p.dqkv = (__nv_bfloat16*)dqkv; p.dq_acc = dq_acc; p.lse = lse; p.delta = delta; p.B = B; p.T = T; p.Hq = Hq; p.Hkv = Hkv;
  p.scale = scale; p.scale_log2 = scale * 1.4426950408889634f; p.status = status_word(); p.hd = hd; p.cosT = cosT; p.sinT = sinT;
  p.n_dst = n_dst; p.dst_rows = dst_rows; p.dst_heads = dst_heads; p.dst_q0 = dst_q0; p.dst_k0 = dst_k0; p.dst_v0 = dst_v0;
  // per (batch, KV head): Q, dO, dQ (fp32 accumulator + bf16 result) of its query heads, K, V, dK, dV. In us with the delta and
  // conversion passes: B 8, T 4096, 16 / 8 heads of 64: 910 - 925 with groups of 4 - 16, 957 with 32, 1055 with all 64.
  // What is left for the last group counts (even_group): 24 / 8 heads of 128, B 2, T 4096, 4 x 4 650, 5 + 5 + 5 + 1 730, 6 + 6 + 4 720,
  // 2 x 8 650; 32 / 4 heads of 32, B 8, 4 x 8 1345, 10 + 10 + 10 + 2 1515, 5 x 6 + 2 1478, 2 x 16 1367
  p.head_group = attn_head_group("TLM_ATTN_BWD_GROUP", (long long)T * hd * (10LL * (Hq / Hkv) + 8), 112LL << 20, B * Hkv);
  AttnBwdDst dd{};
  dd.n = n_dst; dd.rows = dst_rows; dd.heads = dst_heads;
  for (int i = 0; i < n_dst; ++i) { p.dst[i] = (__nv_bfloat16*)dst_ptrs[i]; dd.p[i] = p.dst[i]; }
  e = make_dq_map(&maps.dq, dq_acc, B, T, Hq, hd);
  if (e) return e;
  if (n_dst > 0) e = hd == 128 ? launch_bwd<128, true>(maps, p, st) : launch_bwd<64, true>(maps, p, st);
  else {
    const double n_tiles = (T + AB_TILE - 1) / AB_TILE, rep = Hq / Hkv;
    p.split = split_for(rep * n_tiles, n_tiles * B * Hkv, rep * n_tiles * (n_tiles + 1) / 2 * B * Hkv);
    if (p.split > 1) e = hd == 128 ? launch_bwd<128, false, true>(maps, p, st) : hd == 64 ? launch_bwd<64, false, true>(maps, p, st)
                                                                                           : launch_bwd<32, false, true>(maps, p, st);
    else e = hd == 128 ? launch_bwd<128, false>(maps, p, st) : hd == 64 ? launch_bwd<64, false>(maps, p, st) : launch_bwd<32, false>(maps, p, st);
  }
  if (e) return e;
  // without a return scatter the main kernel has written un-rotated dK into dqkv: this pass rotates it in place
  const int rot_k = (n_dst == 0 && cosT != nullptr) ? Hkv : 0;
  const long long items = (long long)B * T * (Hq + rot_k) * (hd / 16);
  int cb = (int)((items + 255) / 256 < num_sms() * 16 ? (items + 255) / 256 : num_sms() * 16);
  auto conv = items + 256LL * cb < (1LL << 32) ? attn_dq_convert_kernel<unsigned> : attn_dq_convert_kernel<long long>;
  return launch_overlapped(conv, dim3(cb), dim3(256), 0, st, 1, (const float*)dq_acc, (__nv_bfloat16*)dqkv, B, T, Hq, Hq + 2 * Hkv, hd, scale, cosT, sinT,
                           dd, dst_q0, rot_k);
}

TLM_API int tlm_attn_bwd(const void* qkv, const void* o, const void* dout, const float* lse, void* dqkv,
                         float* dq_acc, float* delta, int B, int T, int Hq, int Hkv, int hd, float scale,
                         const float* cosT, const float* sinT, cudaStream_t st) {
  return attn_bwd_impl(qkv, o, dout, lse, dqkv, dq_acc, delta, B, T, Hq, Hkv, hd, scale, cosT, sinT, nullptr, 0, 0, 0, 0, 0, 0, st);
}

// Attention backward whose gradient rows leave for the sequence owners' packed buffers (see AttnBwdParams):
// dst_ptrs[r]: bf16 [B, dst_rows, dst_heads, hd] on rank r; q slot s -> head dst_q0 + s, k -> dst_k0 + s, v -> dst_v0 + s.
TLM_API int tlm_attn_bwd_scatter(const void* qkv, const void* o, const void* dout, const float* lse, float* dq_acc,
                                 float* delta, int B, int T, int Hq, int Hkv, int hd, float scale, const float* cosT,
                                 const float* sinT, void* const* dst_ptrs, int n_dst, int dst_rows, int dst_heads,
                                 int dst_q0, int dst_k0, int dst_v0, cudaStream_t st) {
  if (n_dst < 1) return -6;
  return attn_bwd_impl(qkv, o, dout, lse, nullptr, dq_acc, delta, B, T, Hq, Hkv, hd, scale, cosT, sinT, dst_ptrs, n_dst,
                       dst_rows, dst_heads, dst_q0, dst_k0, dst_v0, st);
}

// Floats of `part` that tlm_attn_window_bwd needs (0: none).
TLM_API long long tlm_attn_window_part_floats(int B, int T, int Hkv, int hd, int window, int sinks) {
  if (T <= 0 || T > (1 << 29)) return 0;
  const int S = sinks < T ? sinks : T;
  const WinFar f = win_far(T, window > 0 && window < T ? window : T, S);
  return f.chunks > 0 ? (long long)B * Hkv * (1 + f.chunks) * S * 2 * hd : 0;
}

// Backward of tlm_attn_window_fwd. strides[9] and o_rest (may be null) as there; out_strides[9]: of dq, dk and dv (rows of 16-byte aligned addresses). o, dout
// [B, T, Hq, hd] and lse contiguous. Scratch owned by the caller: dq_acc, delta as for tlm_attn_bwd, part (see above; may be null
// where it takes no floats). cosT / sinT (optional, fp32 [T, hd]): the transposed rotation of dQ and dK on the way out.
TLM_API int tlm_attn_window_bwd(const void* q, const void* k, const void* v, const long long* strides, const void* o, const void* o_rest, const void* dout,
                                const float* lse, void* dq, void* dk, void* dv, const long long* out_strides, float* dq_acc, float* delta,
                                float* part, int B, int T, int Hq, int Hkv, int hd, float scale, const float* cosT, const float* sinT,
                                int window, int sinks, cudaStream_t st) {
  if (hd != 32 && hd != 64 && hd != 128) return -4;
  if (Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0) return -5;
  if ((size_t)Hq * (DELTA_T + 1) * 4 > 48 * 1024) return -6;
  if (B < 0 || T < 0 || T > (1 << 29) || sinks < 0 || (cosT == nullptr) != (sinT == nullptr)) return -6;
  if (B == 0 || T == 0) return 0;
  if (!aligned16(dq) || !aligned16(dk) || !aligned16(dv)) return -7;
  for (int i = 0; i < 9; ++i) if (out_strides[i] % 8 != 0) return -7;
  AttnBwdParams p{};
  p.window = window > 0 && window < T ? window : T;
  p.sinks = sinks < T ? sinks : T;
  p.far = win_far(T, p.window, p.sinks);
  if (p.far.chunks > 0 && part == nullptr) return -6;
  const double n_tiles = (T + AB_TILE - 1) / AB_TILE, bh = (double)B * Hkv, rep = Hq / Hkv;
  if ((n_tiles + (double)p.far.tiles * p.far.chunks) * bh * 8 > 2147483647.) return -6;
  AttnBwdMaps<true> maps;
  const long long o_strides[3] = {(long long)T * Hq * hd, (long long)Hq * hd, hd};
  int e = make_bthd_map(&maps.q, q, strides, B, T, Hq, hd, AB_TILE);
  if (!e) e = make_bthd_map(&maps.k, k, strides + 3, B, T, Hkv, hd, AB_TILE);
  if (!e) e = make_bthd_map(&maps.v, v, strides + 6, B, T, Hkv, hd, AB_TILE);
  if (!e) e = make_bthd_map(&maps.dout, dout, o_strides, B, T, Hq, hd, AB_TILE);
  if (!e) e = make_dq_map(&maps.dq, dq_acc, B, T, Hq, hd);
  if (e) return e;
  e = launch_delta(o, o_rest, win_rest_rows(T, p.window, p.sinks), dout, delta, dq_acc, B, T, Hq, hd, st);
  if (e) return e;
  p.dq_acc = dq_acc; p.lse = lse; p.delta = delta; p.B = B; p.T = T; p.Hq = Hq; p.Hkv = Hkv; p.hd = hd;
  p.scale = scale; p.scale_log2 = scale * 1.4426950408889634f; p.status = status_word(); p.part = part;
  p.k = (const __nv_bfloat16*)k; p.v = (const __nv_bfloat16*)v; p.dk = (__nv_bfloat16*)dk; p.dv = (__nv_bfloat16*)dv;
  AttnWinFinish f{};
  for (int i = 0; i < 3; ++i) {
    p.ks[i] = strides[3 + i]; p.vs[i] = strides[6 + i];
    f.dqs[i] = out_strides[i]; p.dks[i] = f.dks[i] = out_strides[3 + i]; p.dvs[i] = f.dvs[i] = out_strides[6 + i];
  }
  p.head_group = attn_head_group("TLM_ATTN_BWD_GROUP", (long long)T * hd * (10LL * (Hq / Hkv) + 8), 112LL << 20, B * Hkv);
  // steps: the window's query tiles of every KV tile (fewer at the end), and the far ones of the sink tiles
  const double wt = win_last_q(0, p.window, (int)n_tiles) + 1, far_items = (double)p.far.tiles * p.far.chunks;
  const double steps = n_tiles * wt - wt * (wt - 1) / 2 + p.far.tiles * (n_tiles - wt), longest = p.far.chunks > 0 && p.far.chunk > wt ? p.far.chunk : wt;
  p.split = split_for(rep * longest, (n_tiles + far_items) * bh, rep * steps * bh);
  if (p.split > 1) e = hd == 128 ? launch_bwd<128, false, true, true>(maps, p, st) : hd == 64 ? launch_bwd<64, false, true, true>(maps, p, st)
                                                                                               : launch_bwd<32, false, true, true>(maps, p, st);
  else e = hd == 128 ? launch_bwd<128, false, false, true>(maps, p, st) : hd == 64 ? launch_bwd<64, false, false, true>(maps, p, st)
                                                                                    : launch_bwd<32, false, false, true>(maps, p, st);
  if (e) return e;
  f.dq_acc = dq_acc; f.part = p.far.chunks > 0 ? part : nullptr; f.dq = (__nv_bfloat16*)dq; f.dk = p.dk; f.dv = p.dv;
  f.cosT = cosT; f.sinT = sinT; f.B = B; f.T = T; f.Hq = Hq; f.Hkv = Hkv; f.hd = hd; f.scale = scale; f.slots = 1 + p.far.chunks;
  f.slot_rows = p.sinks;                        // but only those of tiles with far query tiles are in use
  f.sinks = p.sinks < p.far.tiles * AB_TILE ? p.sinks : p.far.tiles * AB_TILE;
  const long long rows = (long long)B * Hkv * f.sinks, items = ((long long)B * Hq * T + (cosT != nullptr ? (long long)B * Hkv * (T - f.sinks) : 0)) * (hd / 16);
  const long long blocks = (items + WIN_FINISH_THREADS - 1) / WIN_FINISH_THREADS;
  f.sum_blocks = (int)(rows < num_sms() ? rows : num_sms());
  const int cb = f.sum_blocks + (int)(blocks < num_sms() * 16 ? blocks : num_sms() * 16);
  return launch_overlapped(attn_window_finish_kernel, dim3(cb), dim3(WIN_FINISH_THREADS), 0, st, 1, f);
}
