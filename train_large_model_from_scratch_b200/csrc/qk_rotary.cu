// Rotary positions on the heads of [B, T, H, hd] (bf16), alone or behind an RMS norm of every head.
//
//   u = x, or with weights  u = w * x * rstd,  rstd = 1 / sqrt(mean(x^2) + eps)   (w: one vector for heads < n_q, one for the others)
//   pair i < n_freq:  angle = position * inv_freq[i],  (y_a, y_b) = m (u_a cos - u_b sin, u_b cos + u_a sin)
//   with (a, b) = (i, i + n_freq) in the half layout, (2 i, 2 i + 1) interleaved; the rest of the head passes through.
//
// Backward:  du = transposed rotation of dy,  dw = sum over rows of du * xhat,  g = du * w,  dx = rstd (g - xhat mean(g xhat)),
// with xhat = x rstd recomputed from x. All sums are fp32; what leaves is rounded once.
//
// Bound by memory at best (each element read and written once: x, and dy in the backward), by instruction issue in practice. B 8,
// T 4096, cold: norm and rotation of 16 + 8 heads of 64 39 us forward (31 at the measured bandwidth), 64 backward (46) and about 5 for
// the weights' sums; rotation of 32 + 4 heads of 32 33 us (23), of 20 heads of 128, 32768 tokens, 57 us (51).
#include "common.cuh"

namespace tlm {

constexpr int QR_THREADS = 256;

// A [B, T, H, hd] tensor whose rows of hd elements are contiguous; strides in elements.
struct QrTensor {
  __nv_bfloat16* p;
  long long sb, st, sh;
};

struct QrParams {
  QrTensor x, in, out;            // in: forward x, backward dy. out: forward y, backward dx (may be `in`: a row is read before it is written)
  const long long* pos;           // [T] or [B, T]
  long long pos_sb;               // 0 or T
  const double* inv_freq;         // [n_freq]
  const __nv_bfloat16* w[2];      // of heads < n_q, of the others
  float* part;                    // backward with weights: [gridDim.x][2][hd]
  int tokens, T, H, n_q, hd, n_freq;
  int hps_log;                    // log2 of the row slots that one token gets
  float eps, m, sign;             // sign -1: transposed rotation
};

// Sixteen elements of a row are one lane's: eight pairs (8 l + i), the rotated ones first, then what passes through, paired up in
// the same way. In registers the first and second elements of the pairs are four packed fp32 pairs each (a, b): two lanes of
// arithmetic an issue slot: B 8, T 4096, 16 + 8 heads of 64 took 56 us forward and 73 backward with scalar arithmetic, weights
// selected in registers and addresses worked out row by row (1146 instructions a token and warp).
struct Packed { uint32_t w[8]; };                       // as they lie in memory: half layout 4 words of a, 4 of b; interleaved (a, b) each
struct Pairs { float2 a[4], b[4]; };

template <bool INTER>
__device__ __forceinline__ Pairs unpack(const Packed& r) {
  Pairs v;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 x = unpack_bf16(r.w[INTER ? 2 * j : j]), y = unpack_bf16(r.w[INTER ? 2 * j + 1 : j + 4]);
    v.a[j] = INTER ? make_float2(x.x, y.x) : x;
    v.b[j] = INTER ? make_float2(x.y, y.y) : y;
  }
  return v;
}
template <bool INTER>
__device__ __forceinline__ Packed pack(const Pairs& v) {
  Packed r;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    r.w[INTER ? 2 * j : j] = INTER ? pack_bf16(v.a[j].x, v.b[j].x) : pack_bf16(v.a[j].x, v.a[j].y);
    r.w[INTER ? 2 * j + 1 : j + 4] = INTER ? pack_bf16(v.a[j].y, v.b[j].y) : pack_bf16(v.b[j].x, v.b[j].y);
  }
  return r;
}

template <bool INTER>
__device__ __forceinline__ void pair_at(int pair, int hd, int n_freq, int& a, int& b) {
  if (INTER) { a = 2 * pair; b = 2 * pair + 1; }
  else if (pair < n_freq) { a = pair; b = pair + n_freq; }
  else { a = n_freq + pair; b = a + (hd - 2 * n_freq) / 2; }      // 2 n_freq + (pair - n_freq)
}

// Where a lane's elements lie. VEC: two 16-byte pieces at a and b; else element by element (odd widths, strides, addresses).
template <bool INTER, bool VEC>
struct RowMap {
  int a, b, l, hd, n_freq;
  bool any;                                             // this lane has elements
  __device__ RowMap(int lane_of_row, int hd_, int n_freq_) : l(lane_of_row), hd(hd_), n_freq(n_freq_) {
    pair_at<INTER>(8 * l, hd, n_freq, a, b);
    if (INTER) b = a + 8;
    any = 16 * l < hd;
  }
  __device__ __forceinline__ Packed load(const __nv_bfloat16* row, bool ok) const {
    Packed r;
    if (VEC) {
      uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
      if (ok && any) { lo = *reinterpret_cast<const uint4*>(row + a); hi = *reinterpret_cast<const uint4*>(row + b); }
      r.w[0] = lo.x; r.w[1] = lo.y; r.w[2] = lo.z; r.w[3] = lo.w; r.w[4] = hi.x; r.w[5] = hi.y; r.w[6] = hi.z; r.w[7] = hi.w;
    } else {
      unsigned short e[16];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        int x, y;
        pair_at<INTER>(8 * l + i, hd, n_freq, x, y);
        const bool in = ok && 2 * (8 * l + i) < hd;
        e[INTER ? 2 * i : i] = in ? reinterpret_cast<const unsigned short*>(row)[x] : 0;
        e[INTER ? 2 * i + 1 : i + 8] = in ? reinterpret_cast<const unsigned short*>(row)[y] : 0;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) r.w[k] = e[2 * k] | ((uint32_t)e[2 * k + 1] << 16);
    }
    return r;
  }
  __device__ __forceinline__ void store(__nv_bfloat16* row, const Packed& r) const {
    if (VEC) {
      if (!any) return;
      *reinterpret_cast<uint4*>(row + a) = make_uint4(r.w[0], r.w[1], r.w[2], r.w[3]);
      *reinterpret_cast<uint4*>(row + b) = make_uint4(r.w[4], r.w[5], r.w[6], r.w[7]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (2 * (8 * l + i) >= hd) continue;
        int x, y;
        pair_at<INTER>(8 * l + i, hd, n_freq, x, y);
        const int k = INTER ? 2 * i : i, m = INTER ? 2 * i + 1 : i + 8;
        reinterpret_cast<unsigned short*>(row)[x] = (unsigned short)(r.w[k >> 1] >> (16 * (k & 1)));
        reinterpret_cast<unsigned short*>(row)[y] = (unsigned short)(r.w[m >> 1] >> (16 * (m & 1)));
      }
    }
  }
};

// Eight floats of shared memory that belong to a lane, as packed pairs
__device__ __forceinline__ void four_pairs(const float* s, float2* out) {
  const float4 x = reinterpret_cast<const float4*>(s)[0], y = reinterpret_cast<const float4*>(s)[1];
  out[0] = make_float2(x.x, x.y); out[1] = make_float2(x.z, x.w);
  out[2] = make_float2(y.x, y.y); out[3] = make_float2(y.z, y.w);
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }
__device__ __forceinline__ void scale_by(Pairs& v, float s) {
#pragma unroll
  for (int j = 0; j < 4; ++j) { v.a[j] = fmul2(v.a[j], both(s)); v.b[j] = fmul2(v.b[j], both(s)); }
}
// sum of x * y over a lane's sixteen
__device__ __forceinline__ float dot16(const Pairs& x, const Pairs& y) {
  float2 s = fmul2(x.a[0], y.a[0]), t = fmul2(x.b[0], y.b[0]);
#pragma unroll
  for (int j = 1; j < 4; ++j) { s = ffma2(x.a[j], y.a[j], s); t = ffma2(x.b[j], y.b[j], t); }
  s = fadd2(s, t);
  return s.x + s.y;
}
template <int LPR>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Where a lane stands: LPR lanes share a row; a warp's 32 / LPR row slots take one token's heads, or those of several tokens where a
// token has fewer heads.
template <int LPR>
struct QrLane {
  int lane, warp, l, hps, tpw, h0, tslot;
  __device__ explicit QrLane(const QrParams& p)
      : lane(threadIdx.x & 31), warp(threadIdx.x >> 5), l(lane % LPR), hps(1 << p.hps_log), tpw((32 / LPR) >> p.hps_log),
        h0((lane / LPR) & (hps - 1)), tslot((lane / LPR) >> p.hps_log) {}
};

// m cos and m sin of a warp's tokens, worked out once for all their heads: [token of the warp][a row's LPR * 8 pairs], (1, 0) for what
// passes through. The product of position and frequency keeps 64 bits until whole turns are taken off: at position 2^20 a 32-bit
// product is off by 0.06 radians.
template <int LPR>
struct QrAngles {
  float cos[256], sin[256];                             // 32 / LPR tokens at most

  __device__ void clear(int lane) {
    for (int k = lane; k < 256; k += 32) { cos[k] = 1.f; sin[k] = 0.f; }
  }
  // `pos`: the position of the lane's own token
  __device__ __forceinline__ void set(const QrParams& p, const QrLane<LPR>& me, double pos) {
    __syncwarp();                                       // the last tokens' have been read
    for (int ts = 0; ts < me.tpw; ++ts) {
      const double at = __shfl_sync(0xffffffffu, pos, (ts << p.hps_log) * LPR);
      for (int pair = me.lane; pair < p.n_freq; pair += 32) {
        const double turns = at * (p.inv_freq[pair] * 0.15915494309189533577);      // 1 / (2 pi)
        float s, c;
        sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
        cos[ts * LPR * 8 + pair] = p.m * c;
        sin[ts * LPR * 8 + pair] = p.m * p.sign * s;
      }
    }
    __syncwarp();
  }
  __device__ __forceinline__ void rotate(Pairs& v, const QrLane<LPR>& me) const {
    const int at = (me.tslot * LPR + me.l) * 8;
    float2 c[4], s[4];
    four_pairs(cos + at, c);
    four_pairs(sin + at, s);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 a = v.a[j], b = v.b[j], n = fmul2(s[j], both(-1.f));
      v.a[j] = ffma2(a, c[j], fmul2(b, n));
      v.b[j] = ffma2(b, c[j], fmul2(a, s[j]));
    }
  }
};

// The two weights in 32 bits, in the lanes' order: [of q, of others][a, b][a row's LPR * 8 pairs]
template <int LPR, bool INTER, bool VEC>
struct QrWeights {
  float w[2][2][LPR * 8];

  __device__ void fill(const QrParams& p) {
    for (int i = threadIdx.x; i < 2 * LPR * 8; i += QR_THREADS) {
      const int which = i / (LPR * 8), pair = i % (LPR * 8);
      int a, b;
      pair_at<INTER>(pair, p.hd, p.n_freq, a, b);
      const bool in = 2 * pair < p.hd;
      w[which][0][pair] = in ? __bfloat162float(p.w[which][a]) : 0.f;
      w[which][1][pair] = in ? __bfloat162float(p.w[which][b]) : 0.f;
    }
    __syncthreads();
  }
  __device__ __forceinline__ void times(Pairs& v, int which, int l) const {
    float2 x[4];
    four_pairs(w[which][0] + l * 8, x);
#pragma unroll
    for (int j = 0; j < 4; ++j) v.a[j] = fmul2(v.a[j], x[j]);
    four_pairs(w[which][1] + l * 8, x);
#pragma unroll
    for (int j = 0; j < 4; ++j) v.b[j] = fmul2(v.b[j], x[j]);
  }
};

// The lane's token: batch entry, place, and whether there is one
struct QrToken {
  int b, t;
  bool in;
  __device__ __forceinline__ QrToken(const QrParams& p, long long tok) {
    in = tok < p.tokens;
    b = in ? (int)tok / p.T : 0;
    t = in ? (int)tok - b * p.T : 0;
  }
  __device__ __forceinline__ __nv_bfloat16* in_tensor(const QrTensor& x, int h) const { return x.p + b * x.sb + t * x.st + h * x.sh; }
  __device__ __forceinline__ double position(const QrParams& p) const { return in ? (double)p.pos[b * p.pos_sb + t] : 0.; }
};

// One row is worked on while the next is on its way, the next token's first one included, and its position. (Four rows requested at
// once, each processed from registers, needed 80 registers and 130 bytes of spills.)
template <int LPR, bool INTER, bool VEC, bool NORM>
__global__ void __launch_bounds__(QR_THREADS, VEC ? 4 : 2)
qk_rotary_fwd_kernel(const QrParams p) {
  griddep_wait();
  griddep_launch();
  __shared__ __align__(16) QrAngles<LPR> turn_all[QR_THREADS / 32];
  __shared__ __align__(16) QrWeights<NORM ? LPR : 1, INTER, VEC> weights;
  const QrLane<LPR> me(p);
  const RowMap<INTER, VEC> map(me.l, p.hd, p.n_freq);
  QrAngles<LPR>& turn = turn_all[me.warp];
  turn.clear(me.lane);
  if constexpr (NORM) weights.fill(p);
  const float inv_hd = 1.f / (float)p.hd;
  const long long ahead = (long long)p.in.sh * me.hps;
  const int step = gridDim.x * (QR_THREADS / 32) * me.tpw;
  long long tok0 = (long long)(blockIdx.x * (QR_THREADS / 32) + me.warp) * me.tpw;
  QrToken now(p, tok0 + me.tslot);
  const __nv_bfloat16* x = now.in_tensor(p.in, me.h0);
  Packed raw = map.load(x, now.in && me.h0 < p.H);
  double pos = now.position(p);
  for (; tok0 < p.tokens; tok0 += step) {
    const QrToken next(p, tok0 + step + me.tslot);
    const __nv_bfloat16* x_next = next.in_tensor(p.in, me.h0);
    __nv_bfloat16* y = now.in_tensor(p.out, me.h0);
    turn.set(p, me, pos);
    pos = next.position(p);
#pragma unroll 1
    for (int h = me.h0; h - me.h0 < p.H; h += me.hps) {
      Pairs v = unpack<INTER>(raw);
      x += ahead;
      const bool more = h - me.h0 + me.hps < p.H;       // of the whole warp
      raw = map.load(more ? x : x_next, more ? now.in && h + me.hps < p.H : next.in && me.h0 < p.H);
      if constexpr (NORM) {
        const float rstd = rsqrtf(row_sum<LPR>(dot16(v, v)) * inv_hd + p.eps);
        weights.times(v, h < p.n_q ? 0 : 1, me.l);
        scale_by(v, rstd);
      }
      turn.rotate(v, me);
      if (now.in && h < p.H) map.store(y, pack<INTER>(v));
      y += p.out.sh * me.hps;
    }
    now = next;
    x = x_next;
  }
}

// Every block leaves its sums for the weights in `part`; qk_norm_dw_kernel adds them up in a fixed order.
template <int LPR, bool INTER, bool VEC>
__global__ void __launch_bounds__(QR_THREADS, VEC ? 2 : 1)
qk_norm_rotary_bwd_kernel(const QrParams p) {
  griddep_wait();
  griddep_launch();
  __shared__ __align__(16) QrAngles<LPR> turn_all[QR_THREADS / 32];
  __shared__ __align__(16) QrWeights<LPR, INTER, VEC> weights;
  __shared__ float sums[QR_THREADS / 32][2][LPR * 16];
  const QrLane<LPR> me(p);
  const RowMap<INTER, VEC> map(me.l, p.hd, p.n_freq);
  QrAngles<LPR>& turn = turn_all[me.warp];
  turn.clear(me.lane);
  weights.fill(p);
  const float inv_hd = 1.f / (float)p.hd;
  Pairs dq, dk;
#pragma unroll
  for (int j = 0; j < 4; ++j) dq.a[j] = dq.b[j] = dk.a[j] = dk.b[j] = make_float2(0.f, 0.f);
  const int step = gridDim.x * (QR_THREADS / 32) * me.tpw;
  long long tok0 = (long long)(blockIdx.x * (QR_THREADS / 32) + me.warp) * me.tpw;
  QrToken now(p, tok0 + me.tslot);
  const __nv_bfloat16 *x = now.in_tensor(p.x, me.h0), *dy = now.in_tensor(p.in, me.h0);
  Packed rx = map.load(x, now.in && me.h0 < p.H), rg = map.load(dy, now.in && me.h0 < p.H);
  double pos = now.position(p);
  for (; tok0 < p.tokens; tok0 += step) {
    const QrToken next(p, tok0 + step + me.tslot);
    const __nv_bfloat16 *x_next = next.in_tensor(p.x, me.h0), *dy_next = next.in_tensor(p.in, me.h0);
    __nv_bfloat16* dx = now.in_tensor(p.out, me.h0);
    turn.set(p, me, pos);
    pos = next.position(p);
#pragma unroll 1
    for (int h = me.h0; h - me.h0 < p.H; h += me.hps) {
      const Pairs v = unpack<INTER>(rx);
      Pairs g = unpack<INTER>(rg);
      x += p.x.sh * me.hps;
      dy += p.in.sh * me.hps;
      const bool more = h - me.h0 + me.hps < p.H;       // of the whole warp
      const bool ok = more ? now.in && h + me.hps < p.H : next.in && me.h0 < p.H;
      rx = map.load(more ? x : x_next, ok);
      rg = map.load(more ? dy : dy_next, ok);
      const bool there = now.in && h < p.H;
      // a row that is not there adds zeros to the weights' sums: its own rstd is infinite where eps is 0
      const float mean = row_sum<LPR>(dot16(v, v)) * inv_hd + p.eps, rstd = there ? rsqrtf(mean) : 0.f;
      turn.rotate(g, me);
      // du * xhat, for the weights
      if (h < p.n_q) {
#pragma unroll
        for (int j = 0; j < 4; ++j) { dq.a[j] = ffma2(fmul2(g.a[j], both(rstd)), v.a[j], dq.a[j]); dq.b[j] = ffma2(fmul2(g.b[j], both(rstd)), v.b[j], dq.b[j]); }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) { dk.a[j] = ffma2(fmul2(g.a[j], both(rstd)), v.a[j], dk.a[j]); dk.b[j] = ffma2(fmul2(g.b[j], both(rstd)), v.b[j], dk.b[j]); }
      }
      weights.times(g, h < p.n_q ? 0 : 1, me.l);
      // dx = rstd (g - xhat mean(g xhat)); the factors of x in an order that cannot overflow: (rstd x) has mean square 1
      const float back = -row_sum<LPR>(dot16(g, v)) * rstd * inv_hd;
      Pairs out;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        out.a[j] = ffma2(fmul2(v.a[j], both(rstd)), both(back), g.a[j]);
        out.b[j] = ffma2(fmul2(v.b[j], both(rstd)), both(back), g.b[j]);
      }
      scale_by(out, rstd);
      if (there) map.store(dx, pack<INTER>(out));
      dx += p.out.sh * me.hps;
    }
    now = next;
    x = x_next;
    dy = dy_next;
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) {                        // pair i % 8, first elements then second ones
    float2 &fq = i < 8 ? dq.a[i / 2] : dq.b[i / 2 - 4], &fk = i < 8 ? dk.a[i / 2] : dk.b[i / 2 - 4];
    float sq = i & 1 ? fq.y : fq.x, sk = i & 1 ? fk.y : fk.x;
#pragma unroll
    for (int o = LPR; o < 32; o <<= 1) {
      sq += __shfl_xor_sync(0xffffffffu, sq, o);
      sk += __shfl_xor_sync(0xffffffffu, sk, o);
    }
    if (me.lane < LPR) { sums[me.warp][0][me.l * 16 + i] = sq; sums[me.warp][1][me.l * 16 + i] = sk; }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * LPR * 16; i += QR_THREADS) {
    const int which = i / (LPR * 16), at = i % (LPR * 16), pair = 8 * (at / 16) + at % 8;
    if (2 * pair >= p.hd) continue;
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < QR_THREADS / 32; ++w) s += sums[w][which][at];
    int a, b;
    pair_at<INTER>(pair, p.hd, p.n_freq, a, b);
    p.part[((long long)blockIdx.x * 2 + which) * p.hd + (at % 16 < 8 ? a : b)] = s;
  }
}

// dw[which][c] += sum over blocks of part[block][which][c]; 8 columns a block, 32 runs of blocks each (with 32 columns and eight runs
// 592 blocks took 33 us, one load after the other). One thread adds to both weights, which may be the same.
__global__ void __launch_bounds__(256)
qk_norm_dw_kernel(const float* part, int blocks, int hd, float* dwq, float* dwk) {
  griddep_wait();
  griddep_launch();
  __shared__ float s[32][2][8];
  const int col = threadIdx.x & 7, c = blockIdx.x * 8 + col, run = threadIdx.x >> 3;
  float a = 0.f, b = 0.f;
  if (c < hd) {
#pragma unroll 4
    for (int i = run; i < blocks; i += 32) {
      a += part[(long long)i * 2 * hd + c];
      b += part[(long long)i * 2 * hd + hd + c];
    }
  }
  s[run][0][col] = a;
  s[run][1][col] = b;
  __syncthreads();
  if (run == 0 && c < hd) {
#pragma unroll
    for (int i = 1; i < 32; ++i) { a += s[i][0][col]; b += s[i][1][col]; }
    dwq[c] += a;
    dwk[c] += b;
  }
}

static int qr_blocks(const QrParams& p, int lpr, int per_sm) {
  const int per_block = (QR_THREADS / 32) * ((32 / lpr) >> p.hps_log);
  const long long need = ((long long)p.tokens + per_block - 1) / per_block;
  return (int)(need < (long long)num_sms() * per_sm ? need : (long long)num_sms() * per_sm);
}

constexpr int QR_FWD_PER_SM = 4, QR_BWD_PER_SM = 2;

template <int LPR, bool INTER, bool VEC>
static int qr_launch(const QrParams& p, bool norm, bool bwd, float* dwq, float* dwk, cudaStream_t st) {
  if (!bwd) {
    const int grid = qr_blocks(p, LPR, QR_FWD_PER_SM);
    return launch_overlapped(norm ? qk_rotary_fwd_kernel<LPR, INTER, VEC, true> : qk_rotary_fwd_kernel<LPR, INTER, VEC, false>,
                             dim3(grid), dim3(QR_THREADS), 0, st, 1, p);
  }
  const int grid = qr_blocks(p, LPR, QR_BWD_PER_SM);
  const int e = launch_overlapped(qk_norm_rotary_bwd_kernel<LPR, INTER, VEC>, dim3(grid), dim3(QR_THREADS), 0, st, 1, p);
  if (e) return e;
  return launch_overlapped(qk_norm_dw_kernel, dim3((p.hd + 7) / 8), dim3(256), 0, st, 1, (const float*)p.part, grid, p.hd, dwq, dwk);
}

template <bool INTER, bool VEC>
static int qr_width(const QrParams& p, bool norm, bool bwd, float* dwq, float* dwk, int lpr, cudaStream_t st) {
  switch (lpr) {
    case 1: return qr_launch<1, INTER, VEC>(p, norm, bwd, dwq, dwk, st);
    case 2: return qr_launch<2, INTER, VEC>(p, norm, bwd, dwq, dwk, st);
    case 4: return qr_launch<4, INTER, VEC>(p, norm, bwd, dwq, dwk, st);
    case 8: return qr_launch<8, INTER, VEC>(p, norm, bwd, dwq, dwk, st);
    case 16: return qr_launch<16, INTER, VEC>(p, norm, bwd, dwq, dwk, st);
  }
  return -4;
}

static bool vec_ok(const QrTensor& t) { return aligned16(t.p) && t.sb % 8 == 0 && t.st % 8 == 0 && t.sh % 8 == 0; }

static int qr_run(QrParams& p, int B, bool norm, bool bwd, int interleaved, float* dwq, float* dwk, cudaStream_t st) {
  if (B < 0 || p.T < 0 || p.H < 0 || p.n_q < 0 || p.n_q > p.H) return -6;
  if (p.hd < 2 || p.hd > 256 || p.hd % 2 != 0 || p.n_freq < 1 || 2 * p.n_freq > p.hd) return -4;
  if ((long long)B * p.T > 0x7fffff00LL) return -6;
  p.tokens = B * p.T;
  if (p.tokens == 0 || p.H == 0) return 0;
  int lpr = 1;
  while (lpr * 16 < p.hd) lpr *= 2;
  p.hps_log = 0;
  while ((1 << p.hps_log) < p.H && (1 << p.hps_log) < 32 / lpr) ++p.hps_log;
  // 16-byte pieces: half layout needs both halves, of the rotated part and of the rest, to be whole pieces
  const bool vec = p.hd % 16 == 0 && (interleaved || p.n_freq % 8 == 0) && vec_ok(p.in) && vec_ok(p.out) && (!bwd || vec_ok(p.x)) &&
                   (!norm || (aligned16(p.w[0]) && aligned16(p.w[1])));
  if (interleaved) return vec ? qr_width<true, true>(p, norm, bwd, dwq, dwk, lpr, st) : qr_width<true, false>(p, norm, bwd, dwq, dwk, lpr, st);
  return vec ? qr_width<false, true>(p, norm, bwd, dwq, dwk, lpr, st) : qr_width<false, false>(p, norm, bwd, dwq, dwk, lpr, st);
}

}  // namespace tlm

using namespace tlm;

// Tensors as in QrParams; `strides`: of x (and, backward, dy and dx) over batch, token, head, in elements. pos_sb: 0 where all
// sequences share positions [T]. wq / wk null: rotation alone, `inverse` then applies the transposed one (its backward).
TLM_API int tlm_qk_rotary(const void* x, const long long* x_strides, void* y, const long long* y_strides, const long long* pos,
                          long long pos_sb, const double* inv_freq, int n_freq, const void* wq, const void* wk, int B, int T, int H,
                          int n_q, int hd, float eps, float m, int interleaved, int inverse, cudaStream_t st) {
  if ((wq == nullptr) != (wk == nullptr) || (wq != nullptr && inverse)) return -6;
  QrParams p{};
  p.in = {(__nv_bfloat16*)x, x_strides[0], x_strides[1], x_strides[2]};
  p.out = {(__nv_bfloat16*)y, y_strides[0], y_strides[1], y_strides[2]};
  p.pos = pos; p.pos_sb = pos_sb; p.inv_freq = inv_freq; p.n_freq = n_freq;
  p.w[0] = (const __nv_bfloat16*)wq; p.w[1] = (const __nv_bfloat16*)wk;
  p.T = T; p.H = H; p.n_q = n_q; p.hd = hd; p.eps = eps; p.m = m; p.sign = inverse ? -1.f : 1.f;
  return qr_run(p, B, wq != nullptr, false, interleaved, nullptr, nullptr, st);
}

// Floats of `work` that tlm_qk_norm_rotary_bwd writes at most.
TLM_API int tlm_qk_norm_work_floats(int hd) { return num_sms() * QR_BWD_PER_SM * 2 * hd; }

// dwq / dwk: fp32 [hd], added to. dx may be dy (same strides).
TLM_API int tlm_qk_norm_rotary_bwd(const void* x, const long long* x_strides, const void* dy, const long long* dy_strides, void* dx,
                                   const long long* dx_strides, const long long* pos, long long pos_sb, const double* inv_freq,
                                   int n_freq, const void* wq, const void* wk, float* dwq, float* dwk, float* work, int B, int T, int H,
                                   int n_q, int hd, float eps, float m, int interleaved, cudaStream_t st) {
  if (wq == nullptr || wk == nullptr || dwq == nullptr || dwk == nullptr || work == nullptr) return -6;
  QrParams p{};
  p.x = {(__nv_bfloat16*)x, x_strides[0], x_strides[1], x_strides[2]};
  p.in = {(__nv_bfloat16*)dy, dy_strides[0], dy_strides[1], dy_strides[2]};
  p.out = {(__nv_bfloat16*)dx, dx_strides[0], dx_strides[1], dx_strides[2]};
  p.pos = pos; p.pos_sb = pos_sb; p.inv_freq = inv_freq; p.n_freq = n_freq;
  p.w[0] = (const __nv_bfloat16*)wq; p.w[1] = (const __nv_bfloat16*)wk; p.part = work;
  p.T = T; p.H = H; p.n_q = n_q; p.hd = hd; p.eps = eps; p.m = m; p.sign = -1.f;
  return qr_run(p, B, true, true, interleaved, dwq, dwk, st);
}
