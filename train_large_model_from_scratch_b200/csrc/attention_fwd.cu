// Causal GQA flash attention, forward, on tcgen05 / TMEM.
//
// Input is the packed projection output  qkv[B, T, Hq + 2*Hkv, hd]  (bf16):
// heads [0,Hq) are queries, [Hq,Hq+Hkv) keys, [Hq+Hkv,Hq+2Hkv) values; query
// head h reads KV head h / (Hq/Hkv) in place, nothing is expanded or transposed.
// Output o[B, T, Hq, hd] (bf16) and lse[B, Hq, T] (fp32, natural log).
//
// One CTA owns 128 query rows of one (batch, head) and walks over 128-row KV
// tiles up to the diagonal:
//   warp 0     TMA: Q once, then K / V tiles into a 2-deep ring (128B swizzle)
//   warp 1     issues  S = Q K^T  (M128 N128) into TMEM, and after the
//              softmax warps have published P:  O_j = P V  (M128 N=hd; V is
//              consumed as an MN-major operand straight from its row-major tile)
//   warps 2-5  one thread per query row: tcgen05.ld S, running max / sum with
//              exp2, P written back to tensor memory as packed bf16 pairs (the A
//              operand of the P V MMA). O accumulates in TMEM across KV tiles; it is only
//              rescaled (ld / multiply / st) when the row maximum grew by more
//              than 2^8, and S of tile j+1 is issued while tile j's softmax runs
// Shared memory is 80 KB and tensor memory 256 columns (hd 64), so two CTAs share an
// SM and one CTA's softmax overlaps the other's MMAs. All waits are bounded.
//
// WIN, a second instantiation: a sliding window with sinks (see window_plan.h), q, k and v as tensors of their own. The tiles are those
// that the window and the sinks leave, the row's own first: its maximum is then finite, whatever is hidden later. Hidden scores become
// -infinity before anything looks at them. What bounds it is the way from tile to tile of the two blocks an SM has room for (tensor
// memory, registers): scores 460 cycles, maximum 670, exponentials 1580, P V 260, and 6500 around a block's tiles. B 8, T 4096, 16 / 8
// heads of 64, window 1024 228 us (530 TF of what is seen), 32 / 4 of 32, window 512 314 us, B 2, 16 / 4 of 128, window 2048 116 us
// (889 TF). P is rounded to bf16 where the tensor core takes it, as in the causal form: 2^-9 of a probability on average.
// FEW, a third one, where no row sees a tile's worth of keys: o more exactly. Its rest, for the gradients of q and k, is kept there for all
// rows, elsewhere for those of the first tile.
#include "attention_window.h"

namespace tlm {

constexpr int AT_BQ = 128, AT_BKV = 128, AT_THREADS = 192, AT_KV_STAGES = 2;

constexpr int AT_MAX_DST = 8;

struct AttnFwdParams {
  __nv_bfloat16* o;
  float* lse;
  int B, T, Hq, Hkv;
  float scale_log2;        // softmax scale * log2(e)
  float scale;             // softmax scale
  unsigned int* status;
  // Optional second copy of the output for sequence parallelism (head -> sequence exchange done by
  // this kernel's epilogue): row t of head h also goes to
  //   o_dst[t / dst_rows][b, t % dst_rows, dst_head0 + h, :]   (bf16 [B, dst_rows, dst_heads, hd] per rank;
  // peer-mapped addresses, plain 16-byte stores). n_dst == 0 disables it.
  __nv_bfloat16* o_dst[AT_MAX_DST];
  int n_dst, dst_rows, dst_heads, dst_head0;
  int hd;                  // head dim of the tensors in memory (= the kernel's HD)
  int head_group;          // heads per group of the heavy-first block order (see heavy_first_decode)
  int window, sinks;       // WIN: keys a query sees, itself included (at most T), and first keys that stay visible
  // WIN, optional, [B, rest_rows, Hq, hd]: what o, divided by the sum of the probabilities as they were rounded, lost when it was rounded
  // to bf16, for the first rest_rows rows of a sequence (win_rest_rows). The backward's delta = sum do * o is compared with do * v of
  // single keys; where a row sees few keys they nearly cancel, and half a bf16 step of o is then much of the gradient of q and k.
  __nv_bfloat16* o_rest;
  int rest_rows;
};

// WIN: q [.., Hq, hd], k and v [.., Hkv, hd]; else one map over the packed tensor
template <bool WIN> struct AttnFwdMaps { CUtensorMap qkv; };
template <> struct AttnFwdMaps<true> { CUtensorMap q, k, v; };

// The first n of 128 positions, as the word with positions 32 w .. 32 w + 31
__device__ __forceinline__ uint32_t first_bits(int n, int w) {
  n -= 32 * w;
  return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u;
}

// ALIAS: P takes the place of S in tensor memory and K and V have one stage each, so that two blocks share an SM at head dim 128 too.
// The next scores then wait for P V, a longer way from tile to tile, but the other block's exponentials run beside it: B 2, T 4096,
// 16 / 4 heads of 128, window 2048 134 us with one block an SM, 120 with two.
template <int HD, bool ALIAS = false>
struct AttnFwdSmem {
  static constexpr int STAGES = ALIAS ? 1 : AT_KV_STAGES;
  static constexpr int KB = HD == 128 ? 2 : 1;         // blocks along hd (64 wide; HD 32: one of 32)
  static constexpr int Q_BYTES = AT_BQ * HD * 2;
  static constexpr int KV_BYTES = AT_BKV * HD * 2;
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_K = OFF_Q + Q_BYTES;
  static constexpr int OFF_V = OFF_K + STAGES * KV_BYTES;
  static constexpr int OFF_BAR = OFF_V + STAGES * KV_BYTES;
  static constexpr int TOTAL = OFF_BAR + 256;          // + barriers; 2 CTAs (hd 64) must fit in 228 KB
};

// Thread `row` owns one query row: running reference max `m_ref`, running sum `l_run`.
// The exponent reference is only moved (and O rescaled in TMEM) when the tile
// maximum exceeds it by more than RESCALE_LOG2 in the log2 domain, so most tiles
// do no rescaling; the result is exact either way because the same reference
// is used for P and for the final normalisation.
constexpr float RESCALE_LOG2 = 8.0f;

// 2^x for x <= 127 on the FMA pipe: x = n + f with n the nearest integer (the sum with 1.5 * 2^23 + 127 leaves n + 127 in the low bits), a
// polynomial of degree 3 for 2^f on [-1/2, 1/2] (minimax, off by 7.5e-5, a fiftieth of half a bf16 step), times 2^n. The row's sum adds up
// what P V is given, so it and lse are off by at most as much (7.5e-5, where such a pair holds all of a row's weight).
// Below -126, -infinity included, that is 0.99993 * 2^-126; less 2^-126 it is nearer to zero than to any bf16, and so a hidden key's
// probability is. NaN stays NaN.
__device__ __forceinline__ float2 ex2_poly(float2 x) {
  asm("max.NaN.f32 %0, %0, 0fC2FC0000;" : "+f"(x.x));      // -126
  asm("max.NaN.f32 %0, %0, 0fC2FC0000;" : "+f"(x.y));
  const float2 magic = make_float2(12583039.f, 12583039.f);
  const float2 t = fadd2(x, magic), f = fadd2(x, fadd2(magic, make_float2(-t.x, -t.y)));
  float2 q = ffma2(f, make_float2(0.05517166f, 0.05517166f), make_float2(0.24261112f, 0.24261112f));
  q = ffma2(f, q, make_float2(0.69326099f, 0.69326099f));
  q = ffma2(f, q, make_float2(0.99992807f, 0.99992807f));
  const float2 two_n = make_float2(__int_as_float(__float_as_int(t.x) << 23), __int_as_float(__float_as_int(t.y) << 23));
  return ffma2(q, two_n, make_float2(-1.17549435e-38f, -1.17549435e-38f));
}

template <int HD, bool WIN = false, bool FEW = false>
__global__ void __launch_bounds__(AT_THREADS, HD <= 64 || WIN ? 2 : 1)
attn_fwd_kernel(const __grid_constant__ AttnFwdMaps<WIN> tm, const AttnFwdParams p) {
  constexpr bool ALIAS = WIN && HD == 128;
  using L = AttnFwdSmem<HD, ALIAS>;
  constexpr int KB = L::KB;
  // tensor-memory columns: S (128 fp32), O (HD fp32) and the probabilities as packed bf16 pairs (64 columns),
  // which the P V MMA reads as its A operand straight from tensor memory (P never touches shared memory)
  constexpr uint32_t S_COL = 0, O_COL = 128, P_COL = ALIAS ? S_COL : 128 + HD;
  constexpr uint32_t TMEM_COLS = HD == 128 && !ALIAS ? 512 : 256;
  // stage of step j's K and V, and how often it has been used before
  auto stage = [](int j) { return ALIAS ? 0 : j & 1; };
  auto uses = [](int j) { return (uint32_t)(ALIAS ? j : j >> 1); };
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t sbase = smem_u32(smem_raw);
  uint8_t* sal = smem_raw;
  if (sbase & 1023u) {                                // swizzled tiles need a 1024-byte aligned base
    griddep_wait();
    if (threadIdx.x == 0) report_status(p.status, (10u << 8) | 2u);
    return;
  }
  const uint32_t bar0 = sbase + L::OFF_BAR;
  // barriers: 0 q_full, 1..2 k_full, 3..4 v_full, 5..6 v_empty, 7 s_full, 8 p_full, 9 o_done, 10 s_consumed,
  //           11..12 k_empty. A K stage is free as soon as its S = Q K^T has run, long before the stage's V is
  //           consumed, so K tiles are loaded one step ahead of V tiles and their latency stays hidden.
  auto bar = [&](int i) { return bar0 + 8u * i; };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sal + L::OFF_BAR + 128);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int n_q_tiles = (p.T + AT_BQ - 1) / AT_BQ;
  int tile_rank, bh;
  heavy_first_decode((int)blockIdx.x, n_q_tiles, p.B * p.Hq, p.head_group, tile_rank, bh);
  const int qt = n_q_tiles - 1 - tile_rank;           // heavy (late) tiles first
  const int b = bh / p.Hq, h = bh % p.Hq;
  const int kvh = h / (p.Hq / p.Hkv);
  const int q0 = qt * AT_BQ;
  const int first = WIN ? win_first_tile(qt, p.window) : 0;
  const int n_kv = WIN ? qt - first + 1 + win_sink_tiles(first, p.sinks) : qt + 1;      // causal: KV tiles 0..qt
  // keys of step j that anybody sees, in whole 16s: of a sink tile the sinks only, and its products are that much smaller
  auto kv_keys = [&](int j) {
    if (!WIN || j <= qt - first) return AT_BKV;
    const int n = p.sinks - win_kv_tile(j, qt, first) * AT_BKV;
    return n < AT_BKV ? (n + 15) & ~15 : AT_BKV;
  };
  auto kv_row = [&](int j) { return (WIN ? win_kv_tile(j, qt, first) : j) * AT_BKV; };
  const CUtensorMap *tm_q, *tm_k, *tm_v;
  int k_head = kvh, v_head = kvh;
  if constexpr (WIN) { tm_q = &tm.q; tm_k = &tm.k; tm_v = &tm.v; }
  else { tm_q = tm_k = tm_v = &tm.qkv; k_head += p.Hq; v_head += p.Hq + p.Hkv; }

  if (threadIdx.x == 0) {
    for (int i = 0; i < 13; ++i) mbar_init(bar(i), (i == 8 || i == 10) ? 4 : 1);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(tm_q);
    if (WIN) { tma_prefetch_desc(tm_k); tma_prefetch_desc(tm_v); }
  }
  if (warp == 1) { tmem_alloc(smem_u32(tmem_slot), TMEM_COLS); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  griddep_wait();

  if (warp == 0) {
    if (lane == 0) {
      mbar_expect_tx(bar(0), L::Q_BYTES);
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) tma_load_4d(sbase + L::OFF_Q + kb * 16384, tm_q, bar(0), kb * 64, h, q0, b);
      auto load_k = [&](int j) -> bool {
        const int st = stage(j);
        if (!mbar_wait(bar(11 + st), (uses(j) & 1u) ^ 1u, 11, abort_flag, p.status)) return false;
        mbar_expect_tx(bar(1 + st), L::KV_BYTES);
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
          tma_load_4d(sbase + L::OFF_K + st * L::KV_BYTES + kb * 16384, tm_k, bar(1 + st), kb * 64, k_head, kv_row(j), b);
        return true;
      };
      bool ok = load_k(0);
      for (int j = 0; j < n_kv && ok; ++j) {
        const int st = stage(j);
        if (!ALIAS && j + 1 < n_kv && !load_k(j + 1)) break;
        if (!mbar_wait(bar(5 + st), (uses(j) & 1u) ^ 1u, 20, abort_flag, p.status)) break;
        mbar_expect_tx(bar(3 + st), L::KV_BYTES);
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
          tma_load_4d(sbase + L::OFF_V + st * L::KV_BYTES + kb * 16384, tm_v, bar(3 + st), kb * 64, v_head, kv_row(j), b);
        if (ALIAS && j + 1 < n_kv && !load_k(j + 1)) break;
      }
    }
  } else if (warp == 1) {
    // The warp stays together and one lane issues (see umma_bf16_w): as one lane's own code a tile's 12 MMAs took 76 cycles each
    // to issue, longer than they run. Long runs, in us: B 8, T 4096, 16 heads of 64 452 -> 424, 32 heads of 32 832 -> 780; B 2, 24
    // heads of 128 269 -> 268. By ncu (B 8, 16 / 8 heads) the exponential unit is busy 65 / 68 / 43 % of the cycles at head dim
    // 64 / 32 / 128, the tensor pipe 32 / 17 / 42 %.
    // Descriptors are built once per tile and advanced with one add per MMA.
    const uint32_t el = elect_one();
    constexpr uint32_t idesc_s = umma_idesc_bf16(AT_BQ, AT_BKV, 0, 0);
    constexpr uint32_t idesc_o = umma_idesc_bf16(AT_BQ, HD, 0, 1);
    const uint64_t dq = attn_desc_k<HD>(sbase + L::OFF_Q);
    auto issue_s = [&](int j) -> bool {
      const int st = stage(j);
      if (!mbar_wait_warp(bar(1 + st), uses(j) & 1u, 13, abort_flag, p.status)) return false;
      tc_fence_after();
      const uint64_t dk = attn_desc_k<HD>(sbase + L::OFF_K + st * L::KV_BYTES);
      const uint32_t idesc = WIN ? umma_idesc_bf16(AT_BQ, kv_keys(j), 0, 0) : idesc_s;
#pragma unroll
      for (int t = 0; t < HD / 16; ++t) {
        const uint32_t off = (t >> 2) * 16384 + (t & 3) * 32;
        umma_bf16_w(el, tmem + S_COL, umma_desc_advance(dq, off), umma_desc_advance(dk, off), idesc, t > 0);
      }
      umma_commit_w(el, bar(7));
      umma_commit_w(el, bar(11 + st));                              // K stage free
      return true;
    };
    bool ok = mbar_wait_warp(bar(0), 0, 12, abort_flag, p.status);
    if (ok) ok = issue_s(0);
    for (int j = 0; j < n_kv && ok; ++j) {
      const int st = stage(j);
      const uint32_t par = (uint32_t)j & 1u;
      if (!ALIAS && j + 1 < n_kv) {                                     // S of the next tile overlaps this tile's softmax
        if (!mbar_wait_warp(bar(10), par, 18, abort_flag, p.status)) break;
        if (!issue_s(j + 1)) break;
      }
      if (!mbar_wait_warp(bar(8), par, 14, abort_flag, p.status)) break;                        // P written
      if (!mbar_wait_warp(bar(3 + st), uses(j) & 1u, 15, abort_flag, p.status)) break;   // V landed
      tc_fence_after();
      const uint64_t dv = attn_desc_mn<HD>(sbase + L::OFF_V + st * L::KV_BYTES);   // MN-major: 16 kv rows per step
      const int keys = kv_keys(j);
#pragma unroll
      for (int t = 0; t < AT_BKV / 16; ++t) {                 // 16 kv = 8 columns of packed pairs per step
        if (WIN && t * 16 >= keys) break;
        umma_bf16_ts_w(el, tmem + O_COL, tmem + P_COL + t * 8, umma_desc_advance(dv, t * attn_mn_step<HD>()), idesc_o, (j > 0) | (t > 0));
      }
      umma_commit_w(el, bar(9));                                    // O updated, P free
      umma_commit_w(el, bar(5 + st));                               // V stage free
      if (ALIAS && j + 1 < n_kv && !issue_s(j + 1)) break;          // behind P V, which reads what these scores replace
    }
    griddep_launch();
  } else {
    const int q = warp & 3;
    const int row = q * 32 + lane;                              // row inside the tile == TMEM lane
    const uint32_t t_lane = tmem + ((uint32_t)(q * 32) << 16);
    const float tau = RESCALE_LOG2 / p.scale_log2;              // threshold in raw-score units
    float m_ref = -INFINITY, l_run = 0.f;
    // FEW: the sum of the probabilities as they are rounded for P V. Divided by it o is a weighted mean of values that are there, and
    // delta (see o_rest) the same mean of their products with do.
    float l_round = 0.f;
    bool ok = true;
    for (int j = 0; j < n_kv; ++j) {
      const uint32_t par = (uint32_t)j & 1u;
      if (!mbar_wait_warp(bar(7), par, 16, abort_flag, p.status)) { ok = false; break; }
      tc_fence_after();
      const bool diag = !WIN && j == qt;
      // ---- the whole S row (128 fp32) moves to registers in one go; S may then be overwritten by the next
      // tile's Q K^T, which therefore overlaps all of this tile's softmax
      uint32_t sr[AT_BKV];
#pragma unroll
      for (int c = 0; c < AT_BKV; c += 32) tmem_ld32(t_lane + S_COL + c, sr + c);
      tmem_ld_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(10));
      if constexpr (WIN) {
        const int t = win_kv_tile(j, qt, first);
        if (win_partial(qt, t, p.window, p.sinks)) {            // hidden scores become -infinity: probability 0, whatever they were
          const int last = (qt - t) * AT_BKV + row;             // this row's own position in the tile
          uint32_t seen[4];
#pragma unroll
          for (int w = 0; w < 4; ++w)
            seen[w] = first_bits(last + 1, w) & (~first_bits(last + 1 - p.window, w) | first_bits(p.sinks - t * AT_BKV, w));
#pragma unroll
          for (int i = 0; i < AT_BKV; ++i)
            if (!((seen[i >> 5] >> (i & 31)) & 1u)) sr[i] = 0xff800000u;
        }
      }
      // ---- row maximum
      float mx0 = -INFINITY, mx1 = -INFINITY, mx2 = -INFINITY, mx3 = -INFINITY;
      if (!diag) {
#pragma unroll
        for (int i = 0; i < AT_BKV; i += 4) {
          mx0 = fmaxf(mx0, __uint_as_float(sr[i]));     mx1 = fmaxf(mx1, __uint_as_float(sr[i + 1]));
          mx2 = fmaxf(mx2, __uint_as_float(sr[i + 2])); mx3 = fmaxf(mx3, __uint_as_float(sr[i + 3]));
        }
      } else {
#pragma unroll
        for (int i = 0; i < AT_BKV; ++i) if (i <= row) mx0 = fmaxf(mx0, __uint_as_float(sr[i]));
      }
      const float mx = fmaxf(fmaxf(mx0, mx1), fmaxf(mx2, mx3));
      // ---- the reference only moves when the maximum grew a lot (O is then rescaled below)
      const bool grow = j > 0 && mx > m_ref + tau;
      float alpha = 1.f;
      if (j == 0) m_ref = mx;
      else if (grow) { alpha = ex2_approx((m_ref - mx) * p.scale_log2); m_ref = mx; }
      const float neg_m = -m_ref * p.scale_log2;
      // ---- probabilities as packed bf16 pairs, still in registers (they take the place of the S row)
      // WIN takes every seventh pair of probabilities this way: the exponential unit takes 1024 cycles for a tile, two warps share it, and the
      // rest of a warp's way from tile to tile is too short to hide that (at best 58 % of its cycles were in use). In us, no pair / every
      // eighth / seventh / fifth: B 8, T 4096, 16 / 8 heads of 64, window 1024 248 / 230 / 228 / 231; 32 / 4 of 32, window 512 331 / 316 / 313 /
      // 317; B 2, 16 / 4 of 128, window 2048 120 / 118 / 116 / 118.
      float2 l2 = make_float2(0.f, 0.f);
      const float2 sc2 = make_float2(p.scale_log2, p.scale_log2), nm2 = make_float2(neg_m, neg_m);
      uint32_t pk[AT_BKV / 2];
#pragma unroll
      for (int i = 0; i < AT_BKV; i += 2) {
        const float2 x = ffma2(make_float2(__uint_as_float(sr[i]), __uint_as_float(sr[i + 1])), sc2, nm2);
        float2 pp = WIN && (i >> 1) % 7 == 6 ? ex2_poly(x) : make_float2(ex2_approx(x.x), ex2_approx(x.y));
        if (diag) { if (i > row) pp.x = 0.f; if (i + 1 > row) pp.y = 0.f; }
        l2 = fadd2(l2, pp);
        pk[i >> 1] = pack_bf16(pp.x, pp.y);
      }
      // ---- only now is the previous tile's P V needed to be complete (P is overwritten, O may be rescaled):
      // by this time it is, so the wait costs nothing
      if (j > 0) {
        if (!mbar_wait_warp(bar(9), par ^ 1u, 17, abort_flag, p.status)) { ok = false; break; }
        tc_fence_after();
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
          for (int c = 0; c < HD; c += 8) {                    // rare path; narrow chunks keep registers free
            uint32_t r[8];
            tmem_ld8(t_lane + O_COL + c, r);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 8; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * alpha);
            tmem_st8(t_lane + O_COL + c, r);
          }
        }
      }
      l_run = fmaf(l_run, alpha, l2.x + l2.y);
      if constexpr (FEW) {
        l2 = make_float2(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < AT_BKV / 2; ++i) l2 = fadd2(l2, unpack_bf16(pk[i]));
        l_round = fmaf(l_round, alpha, l2.x + l2.y);
      }
#pragma unroll
      for (int c = 0; c < AT_BKV; c += 32)
        tmem_st16(t_lane + P_COL + (c >> 1), pk + (c >> 1));    // word i of the row = probabilities 2i, 2i+1
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(8));
    }
    if (ok) ok = mbar_wait_warp(bar(9), (uint32_t)(n_kv - 1) & 1u, 19, abort_flag, p.status);
    const int t_row = q0 + row;
    if (ok) {
      tc_fence_after();
      const float inv = 1.f / (FEW ? l_round : l_run);
      __nv_bfloat16* out = p.o + (((long long)b * p.T + t_row) * p.Hq + h) * p.hd;
      __nv_bfloat16* out2 = nullptr;
      if (p.n_dst > 0 && t_row < p.T) {
        const int dest = t_row / p.dst_rows, tl = t_row - dest * p.dst_rows;
        if (dest < p.n_dst) out2 = p.o_dst[dest] + (((long long)b * p.dst_rows + tl) * p.dst_heads + p.dst_head0 + h) * p.hd;
      }
#pragma unroll
      for (int c = 0; c < HD; c += 32) {
        uint32_t r[32];
        tmem_ld32(t_lane + O_COL + c, r);
        tmem_ld_wait();
        if (t_row < p.T && c < p.hd) {
#pragma unroll
          for (int i = 0; i < 32; i += 8) {
            uint4 v;
            v.x = pack_bf16(__uint_as_float(r[i]) * inv, __uint_as_float(r[i + 1]) * inv);
            v.y = pack_bf16(__uint_as_float(r[i + 2]) * inv, __uint_as_float(r[i + 3]) * inv);
            v.z = pack_bf16(__uint_as_float(r[i + 4]) * inv, __uint_as_float(r[i + 5]) * inv);
            v.w = pack_bf16(__uint_as_float(r[i + 6]) * inv, __uint_as_float(r[i + 7]) * inv);
            *reinterpret_cast<uint4*>(out + c + i) = v;
            if (out2 != nullptr) *reinterpret_cast<uint4*>(out2 + c + i) = v;
          }
        }
      }
      if (t_row < p.T) p.lse[((long long)b * p.Hq + h) * p.T + t_row] = m_ref * p.scale + __logf(l_run);
      if constexpr (WIN) {
        if (p.o_rest != nullptr && (FEW || qt == 0)) {
          float inv_rest = inv;
          if (!FEW) {
            // The first tile is its rows' only one, so its probabilities, as they were rounded, still lie where P V read them. Their sum in the
            // loop over tiles took 75 us of 313 (8 x 4096, 32 / 8 heads of 32, window 1024), this and the stores 3.
            float2 l2 = make_float2(0.f, 0.f);
#pragma unroll
            for (int c = 0; c < AT_BKV / 2; c += 32) {
              uint32_t r[32];
              tmem_ld32(t_lane + P_COL + c, r);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 32; ++i) l2 = fadd2(l2, unpack_bf16(r[i]));
            }
            inv_rest = 1.f / (l2.x + l2.y);
          }
          __nv_bfloat16* dst = p.o_rest + (((long long)b * p.rest_rows + t_row) * p.Hq + h) * p.hd;
#pragma unroll
          for (int c = 0; c < HD; c += 32) {
            uint32_t r[32];
            tmem_ld32(t_lane + O_COL + c, r);
            tmem_ld_wait();
            auto rest = [&](int k) {                            // o is rounded again, as it left
              const float x = __uint_as_float(r[k]), y = __uint_as_float(r[k + 1]);
              const float2 left = unpack_bf16(pack_bf16(x * inv, y * inv));
              return pack_bf16(fmaf(x, inv_rest, -left.x), fmaf(y, inv_rest, -left.y));
            };
            if (t_row < p.T) {
#pragma unroll
              for (int i = 0; i < 32; i += 8) *reinterpret_cast<uint4*>(dst + c + i) = make_uint4(rest(i), rest(i + 2), rest(i + 4), rest(i + 6));
            }
          }
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) { tc_fence_after(); tmem_dealloc(tmem, TMEM_COLS); }
}

// 4-D map over the packed tensor: dims (hd, heads, T, B); box (cols, 1, rows, 1). A box wider than hd = 32 is
// filled with zeros (loads) or clipped (stores) there.
int make_qkv_map(CUtensorMap* map, const void* base, int B, int T, int heads, int hd, int box_rows, int box_cols) {
  uint64_t dims[4] = {(uint64_t)hd, (uint64_t)heads, (uint64_t)T, (uint64_t)B};
  uint64_t strides[3] = {(uint64_t)hd * 2, (uint64_t)heads * hd * 2, (uint64_t)T * heads * hd * 2};
  uint32_t box[4] = {(uint32_t)box_cols, 1, (uint32_t)box_rows, 1};
  return make_tmap_bf16(map, base, 4, dims, strides, box);
}

template <int HD, bool WIN = false, bool FEW = false>
static int launch_fwd(const AttnFwdMaps<WIN>& maps, const AttnFwdParams& p, cudaStream_t st) {
  using L = AttnFwdSmem<HD, WIN && HD == 128>;
  static SmemConfigured configured;
  if (const int e = configured.set(attn_fwd_kernel<HD, WIN, FEW>, L::TOTAL)) return e;
  const int grid = ((p.T + AT_BQ - 1) / AT_BQ) * p.B * p.Hq;
  return launch_overlapped(attn_fwd_kernel<HD, WIN, FEW>, dim3(grid), dim3(AT_THREADS), L::TOTAL, st, 1, maps, p);
}

}  // namespace tlm

using namespace tlm;

static int attn_fwd_impl(const void* qkv, void* o, float* lse, int B, int T, int Hq, int Hkv, int hd, float scale,
                         void* const* o_dst, int n_dst, int dst_rows, int dst_heads, int dst_head0, cudaStream_t st) {
  if (hd != 32 && hd != 64 && hd != 128) return -4;
  if (Hq % Hkv != 0) return -5;
  if (n_dst < 0 || n_dst > AT_MAX_DST || (n_dst > 0 && (dst_rows <= 0 || (long long)dst_rows * n_dst < T))) return -6;
  AttnFwdMaps<false> map;
  int e = make_qkv_map(&map.qkv, qkv, B, T, Hq + 2 * Hkv, hd, AT_BQ, hd == 32 ? 32 : 64);
  if (e) return e;
  AttnFwdParams p{};
  p.o = (__nv_bfloat16*)o; p.lse = lse; p.B = B; p.T = T; p.Hq = Hq; p.Hkv = Hkv;
  p.scale_log2 = scale * 1.4426950408889634f; p.scale = scale; p.status = status_word();
  p.n_dst = n_dst; p.dst_rows = dst_rows; p.dst_heads = dst_heads; p.dst_head0 = dst_head0; p.hd = hd;
  for (int i = 0; i < n_dst; ++i) p.o_dst[i] = (__nv_bfloat16*)o_dst[i];
  // a head's Q, K, V and O rows, groups within 64 MB of them. B 8, T 4096, 16 heads of 64: 435 us with groups of 22 - 43, 459 with
  // each head's tiles adjacent; all 128 heads at once are no better alone and lose to L2 misses in a step. Against 48 MB, 16 heads
  // of 64: T 28000 2224 us (groups of 4) and 2327 (3), T 30000 2550 and 2662, T 32768 3031 and 3137; but T 36000 3762 (3) and 3687
  // (2), T 40000 4635 and 4410; T 24000 1653 either way (4; 6: 1646, 8: 1632). 16 of 128: T 16384 1166 (4) and 1201 (3), T 18000 1446
  // (3) and 1406 (2). So it is groups of three that lose, five and a rest of one, wherever the budget puts them (see even_group).
  p.head_group = attn_head_group("TLM_ATTN_FWD_GROUP", 8LL * T * hd, 64LL << 20, B * Hq);
  return hd == 128 ? launch_fwd<128>(map, p, st) : hd == 64 ? launch_fwd<64>(map, p, st) : launch_fwd<32>(map, p, st);
}

TLM_API int tlm_attn_fwd(const void* qkv, void* o, float* lse, int B, int T, int Hq, int Hkv, int hd, float scale,
                         cudaStream_t st) {
  return attn_fwd_impl(qkv, o, lse, B, T, Hq, Hkv, hd, scale, nullptr, 0, 0, 0, 0, st);
}

// Same, and the epilogue also stores every output row into the memory of the rank that owns the
// row's sequence chunk (see AttnFwdParams): the head -> sequence exchange of Ulysses sequence parallelism.
TLM_API int tlm_attn_fwd_scatter(const void* qkv, void* o, float* lse, int B, int T, int Hq, int Hkv, int hd,
                                 float scale, void* const* o_dst, int n_dst, int dst_rows, int dst_heads,
                                 int dst_head0, cudaStream_t st) {
  return attn_fwd_impl(qkv, o, lse, B, T, Hq, Hkv, hd, scale, o_dst, n_dst, dst_rows, dst_heads, dst_head0, st);
}

// Causal attention over a sliding window with sinks (window_plan.h) on q [B, T, Hq, hd], k and v [B, T, Hkv, hd]; strides[9]: batch,
// token and head strides of q, k and v in elements. window <= 0 or above T: no window. o [B, T, Hq, hd], lse [B, Hq, T] contiguous;
// o_rest: null or, for the backward, [B, rows, Hq, hd] of tlm_attn_window_rest_rows rows (see AttnFwdParams).
TLM_API int tlm_attn_window_rest_rows(int T, int window, int sinks) {
  return T <= 0 ? 0 : win_rest_rows(T, window > 0 && window < T ? window : T, sinks < T ? sinks : T);
}
TLM_API int tlm_attn_window_fwd(const void* q, const void* k, const void* v, const long long* strides, void* o, void* o_rest, float* lse, int B, int T,
                                int Hq, int Hkv, int hd, float scale, int window, int sinks, cudaStream_t st) {
  if (hd != 32 && hd != 64 && hd != 128) return -4;
  if (Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0) return -5;
  if (B < 0 || T < 0 || T > (1 << 29) || sinks < 0 || (long long)((T + AT_BQ - 1) / AT_BQ) * B * Hq > 0x7fffffffLL) return -6;
  if (B == 0 || T == 0) return 0;
  AttnFwdMaps<true> maps;
  int e = make_bthd_map(&maps.q, q, strides, B, T, Hq, hd, AT_BQ);
  if (!e) e = make_bthd_map(&maps.k, k, strides + 3, B, T, Hkv, hd, AT_BKV);
  if (!e) e = make_bthd_map(&maps.v, v, strides + 6, B, T, Hkv, hd, AT_BKV);
  if (e) return e;
  AttnFwdParams p{};
  p.o = (__nv_bfloat16*)o; p.lse = lse; p.B = B; p.T = T; p.Hq = Hq; p.Hkv = Hkv;
  p.scale_log2 = scale * 1.4426950408889634f; p.scale = scale; p.status = status_word(); p.hd = hd;
  p.window = window > 0 && window < T ? window : T;
  p.sinks = sinks < T ? sinks : T;
  p.o_rest = (__nv_bfloat16*)o_rest;
  // FEW where no row sees a tile's worth of keys. Errors of dq and dk relative to 64 bits, without and with it, median (worst): 0.0042
  // (0.42) and 0.0024 (0.0044) for 2 keys, 0.0035 (0.017) and 0.0025 (0.0039) for 4, 0.0027 (0.0033) and 0.0024 (0.0030) for 64, 0.0025
  // (0.0026) and 0.0024 (0.0025) for a window of 200. Taken everywhere it cost 75 us of 313 forward and 14 of 499 backward
  // (8 x 4096, 32 / 8 heads of 32, window 1024).
  const bool few = win_few(T, p.window, p.sinks);
  p.rest_rows = win_rest_rows(T, p.window, p.sinks);
  p.head_group = attn_head_group("TLM_ATTN_FWD_GROUP", 8LL * T * hd, 64LL << 20, B * Hq);
  if (few)
    return hd == 128 ? launch_fwd<128, true, true>(maps, p, st) : hd == 64 ? launch_fwd<64, true, true>(maps, p, st)
                                                                           : launch_fwd<32, true, true>(maps, p, st);
  return hd == 128 ? launch_fwd<128, true>(maps, p, st) : hd == 64 ? launch_fwd<64, true>(maps, p, st) : launch_fwd<32, true>(maps, p, st);
}
