// Rotary positions on the heads of [B, T, H, hd] (bf16), alone or behind an RMS norm of every head.
//
//   u = x, or with weights  u = w * x * rstd,  rstd = 1 / sqrt(mean(x^2) + eps)   (w: one vector for heads < n_q, one for the others)
//   pair i < n_freq:  angle = position * inv_freq[i],  (y_a, y_b) = m (u_a cos - u_b sin, u_b cos + u_a sin)
//   with (a, b) = (i, i + n_freq) in the half layout, (2 i, 2 i + 1) interleaved; the rest of the head passes through.
//
// Backward:  du = transposed rotation of dy,  dw = sum over rows of du * xhat,  g = du * w,  dx = rstd (g - xhat mean(g xhat)),
// with xhat = x rstd recomputed from x. All sums are fp32; what leaves is rounded once.
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
// the same way. v[va(i)], v[vb(i)] are pair i. VEC: two 16-byte pieces; else element by element (odd widths, strides, addresses).
template <bool INTER> __device__ __forceinline__ constexpr int va(int i) { return INTER ? 2 * i : i; }
template <bool INTER> __device__ __forceinline__ constexpr int vb(int i) { return INTER ? 2 * i + 1 : i + 8; }

template <bool INTER>
__device__ __forceinline__ void pair_at(int pair, int hd, int n_freq, int& a, int& b) {
  if (INTER) { a = 2 * pair; b = 2 * pair + 1; }
  else if (pair < n_freq) { a = pair; b = pair + n_freq; }
  else { a = n_freq + pair; b = a + (hd - 2 * n_freq) / 2; }      // 2 n_freq + (pair - n_freq)
}

template <bool INTER, bool VEC>
__device__ __forceinline__ void load_row(const __nv_bfloat16* row, int l, int hd, int n_freq, bool ok, float* v) {
  if (VEC) {
    int a, b;
    pair_at<INTER>(8 * l, hd, n_freq, a, b);
    if (INTER) b = a + 8;
    ok = ok && 16 * l < hd;
    const uint4 z = make_uint4(0, 0, 0, 0);
    const uint4 lo = ok ? *reinterpret_cast<const uint4*>(row + a) : z, hi = ok ? *reinterpret_cast<const uint4*>(row + b) : z;
    const uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
    for (int k = 0; k < 8; ++k) { const float2 f = unpack_bf16(w[k]); v[2 * k] = f.x; v[2 * k + 1] = f.y; }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      int a, b;
      pair_at<INTER>(8 * l + i, hd, n_freq, a, b);
      const bool in = ok && 2 * (8 * l + i) < hd;
      v[va<INTER>(i)] = in ? __bfloat162float(row[a]) : 0.f;
      v[vb<INTER>(i)] = in ? __bfloat162float(row[b]) : 0.f;
    }
  }
}

template <bool INTER, bool VEC>
__device__ __forceinline__ void store_row(__nv_bfloat16* row, int l, int hd, int n_freq, const float* v) {
  if (VEC) {
    if (16 * l >= hd) return;
    int a, b;
    pair_at<INTER>(8 * l, hd, n_freq, a, b);
    if (INTER) b = a + 8;
    *reinterpret_cast<uint4*>(row + a) = make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
    *reinterpret_cast<uint4*>(row + b) = make_uint4(pack_bf16(v[8], v[9]), pack_bf16(v[10], v[11]), pack_bf16(v[12], v[13]), pack_bf16(v[14], v[15]));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (2 * (8 * l + i) >= hd) continue;
      int a, b;
      pair_at<INTER>(8 * l + i, hd, n_freq, a, b);
      row[a] = __float2bfloat16(v[va<INTER>(i)]);
      row[b] = __float2bfloat16(v[vb<INTER>(i)]);
    }
  }
}

// m cos and m sin of this lane's eight pairs. The product of position and frequency keeps 64 bits until whole turns are taken off:
// at position 2^20 a 32-bit product is off by 0.06. Pairs that pass through turn by nothing.
__device__ __forceinline__ void angles(const QrParams& p, double pos, int l, float* cs, float* sn) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int pair = 8 * l + i;
    cs[i] = 1.f;
    sn[i] = 0.f;
    if (pair < p.n_freq) {
      const double turns = pos * (p.inv_freq[pair] * 0.15915494309189533577);      // 1 / (2 pi)
      float s, c;
      sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
      cs[i] = p.m * c;
      sn[i] = p.m * p.sign * s;
    }
  }
}

template <bool INTER>
__device__ __forceinline__ void rotate(float* v, const float* cs, const float* sn) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float a = v[va<INTER>(i)], b = v[vb<INTER>(i)];
    v[va<INTER>(i)] = a * cs[i] - b * sn[i];
    v[vb<INTER>(i)] = b * cs[i] + a * sn[i];
  }
}

template <int LPR>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// LPR lanes share a row. A warp's 32 / LPR row slots take one token's heads, or those of several tokens where a token has fewer
// heads: a lane computes its angles once for all heads of its token.
template <int LPR, bool INTER, bool VEC, bool NORM>
__global__ void __launch_bounds__(QR_THREADS)
qk_rotary_fwd_kernel(const QrParams p) {
  griddep_wait();
  griddep_launch();
  const int lane = threadIdx.x & 31, l = lane % LPR, slot = lane / LPR;
  const int hps = 1 << p.hps_log, tpw = (32 / LPR) >> p.hps_log;
  const int h0 = slot & (hps - 1), tslot = slot >> p.hps_log;
  const int step = gridDim.x * (QR_THREADS / 32) * tpw;
  float wq[NORM ? 16 : 1], wk[NORM ? 16 : 1];
  if (NORM) {
    load_row<INTER, VEC>(p.w[0], l, p.hd, p.n_freq, true, wq);
    load_row<INTER, VEC>(p.w[1], l, p.hd, p.n_freq, true, wk);
  }
  for (long long tok0 = (long long)(blockIdx.x * (QR_THREADS / 32) + (threadIdx.x >> 5)) * tpw; tok0 < p.tokens; tok0 += step) {
    const int tok = (int)tok0 + tslot;
    const bool in = tok < p.tokens;
    const int b = in ? tok / p.T : 0, t = in ? tok - b * p.T : 0;
    float cs[8], sn[8];
    angles(p, (double)p.pos[b * p.pos_sb + t], l, cs, sn);
    const __nv_bfloat16* x = p.in.p + b * p.in.sb + t * p.in.st;
    __nv_bfloat16* y = p.out.p + b * p.out.sb + t * p.out.st;
    for (int hb = 0; hb < p.H; hb += hps) {
      const int h = hb + h0;
      const bool ok = in && h < p.H;
      float v[16];
      load_row<INTER, VEC>(x + h * p.in.sh, l, p.hd, p.n_freq, ok, v);
      if (NORM) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) ss = fmaf(v[i], v[i], ss);
        const float rstd = rsqrtf(row_sum<LPR>(ss) / (float)p.hd + p.eps);
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] *= rstd * (h < p.n_q ? wq[i] : wk[i]);
      }
      rotate<INTER>(v, cs, sn);
      if (ok) store_row<INTER, VEC>(y + h * p.out.sh, l, p.hd, p.n_freq, v);
    }
  }
}

// Every block leaves its sums for the weights in `part`; qk_norm_dw_kernel adds them up in a fixed order.
template <int LPR, bool INTER, bool VEC>
__global__ void __launch_bounds__(QR_THREADS)
qk_norm_rotary_bwd_kernel(const QrParams p) {
  griddep_wait();
  griddep_launch();
  __shared__ float sums[QR_THREADS / 32][2][LPR * 16];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l = lane % LPR, slot = lane / LPR;
  const int hps = 1 << p.hps_log, tpw = (32 / LPR) >> p.hps_log;
  const int h0 = slot & (hps - 1), tslot = slot >> p.hps_log;
  const int step = gridDim.x * (QR_THREADS / 32) * tpw;
  float wq[16], wk[16], dq[16], dk[16];
  load_row<INTER, VEC>(p.w[0], l, p.hd, p.n_freq, true, wq);
  load_row<INTER, VEC>(p.w[1], l, p.hd, p.n_freq, true, wk);
#pragma unroll
  for (int i = 0; i < 16; ++i) dq[i] = dk[i] = 0.f;
  for (long long tok0 = (long long)(blockIdx.x * (QR_THREADS / 32) + warp) * tpw; tok0 < p.tokens; tok0 += step) {
    const int tok = (int)tok0 + tslot;
    const bool in = tok < p.tokens;
    const int b = in ? tok / p.T : 0, t = in ? tok - b * p.T : 0;
    float cs[8], sn[8];
    angles(p, (double)p.pos[b * p.pos_sb + t], l, cs, sn);
    const __nv_bfloat16* x = p.x.p + b * p.x.sb + t * p.x.st;
    const __nv_bfloat16* dy = p.in.p + b * p.in.sb + t * p.in.st;
    __nv_bfloat16* dx = p.out.p + b * p.out.sb + t * p.out.st;
    for (int hb = 0; hb < p.H; hb += hps) {
      const int h = hb + h0;
      const bool ok = in && h < p.H, is_q = h < p.n_q;
      float v[16], g[16];
      load_row<INTER, VEC>(x + h * p.x.sh, l, p.hd, p.n_freq, ok, v);
      load_row<INTER, VEC>(dy + h * p.in.sh, l, p.hd, p.n_freq, ok, g);
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) ss = fmaf(v[i], v[i], ss);
      const float rstd = rsqrtf(row_sum<LPR>(ss) / (float)p.hd + p.eps);
      rotate<INTER>(g, cs, sn);
      float dot = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        v[i] *= rstd;
        const float d = g[i] * v[i];                       // rows that are not there add zeros
        if (is_q) dq[i] += d; else dk[i] += d;
        g[i] *= is_q ? wq[i] : wk[i];
        dot = fmaf(g[i], v[i], dot);
      }
      dot = row_sum<LPR>(dot) / (float)p.hd;
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = rstd * (g[i] - v[i] * dot);
      if (ok) store_row<INTER, VEC>(dx + h * p.out.sh, l, p.hd, p.n_freq, v);
    }
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) {
#pragma unroll
    for (int o = LPR; o < 32; o <<= 1) {
      dq[i] += __shfl_xor_sync(0xffffffffu, dq[i], o);
      dk[i] += __shfl_xor_sync(0xffffffffu, dk[i], o);
    }
    if (slot == 0) { sums[warp][0][l * 16 + i] = dq[i]; sums[warp][1][l * 16 + i] = dk[i]; }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * LPR * 16; i += QR_THREADS) {
    const int which = i / (LPR * 16), at = i % (LPR * 16), lane_of = at / 16, k = at % 16;
    const int pair = 8 * lane_of + (INTER ? k / 2 : k % 8);
    if (2 * pair >= p.hd) continue;
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < QR_THREADS / 32; ++w) s += sums[w][which][at];
    int a, bb;
    pair_at<INTER>(pair, p.hd, p.n_freq, a, bb);
    const bool second = INTER ? (k & 1) : k >= 8;
    p.part[((long long)blockIdx.x * 2 + which) * p.hd + (second ? bb : a)] = s;
  }
}

// dw[which][c] += sum over blocks of part[block][which][c]; 32 columns a block, eight runs of blocks each. One thread adds to both
// weights, which may be the same.
__global__ void qk_norm_dw_kernel(const float* part, int blocks, int hd, float* dwq, float* dwk) {
  griddep_wait();
  griddep_launch();
  __shared__ float s[8][2][32];
  const int col = threadIdx.x & 31, c = blockIdx.x * 32 + col, run = threadIdx.x >> 5;
  float a = 0.f, b = 0.f;
  if (c < hd)
    for (int i = run; i < blocks; i += 8) {
      a += part[(long long)i * 2 * hd + c];
      b += part[(long long)i * 2 * hd + hd + c];
    }
  s[run][0][col] = a;
  s[run][1][col] = b;
  __syncthreads();
  if (run == 0 && c < hd) {
#pragma unroll
    for (int i = 1; i < 8; ++i) { a += s[i][0][col]; b += s[i][1][col]; }
    dwq[c] += a;
    dwk[c] += b;
  }
}

static int qr_blocks(const QrParams& p, int lpr, int per_sm) {
  const int per_block = (QR_THREADS / 32) * ((32 / lpr) >> p.hps_log);
  const long long need = ((long long)p.tokens + per_block - 1) / per_block;
  return (int)(need < (long long)num_sms() * per_sm ? need : (long long)num_sms() * per_sm);
}

constexpr int QR_BWD_PER_SM = 4;

template <int LPR, bool INTER, bool VEC>
static int qr_launch(const QrParams& p, bool norm, bool bwd, float* dwq, float* dwk, cudaStream_t st) {
  if (!bwd) {
    const int grid = qr_blocks(p, LPR, 16);
    return launch_overlapped(norm ? qk_rotary_fwd_kernel<LPR, INTER, VEC, true> : qk_rotary_fwd_kernel<LPR, INTER, VEC, false>,
                             dim3(grid), dim3(QR_THREADS), 0, st, 1, p);
  }
  const int grid = qr_blocks(p, LPR, QR_BWD_PER_SM);
  const int e = launch_overlapped(qk_norm_rotary_bwd_kernel<LPR, INTER, VEC>, dim3(grid), dim3(QR_THREADS), 0, st, 1, p);
  if (e) return e;
  return launch_overlapped(qk_norm_dw_kernel, dim3((p.hd + 31) / 32), dim3(256), 0, st, 1, (const float*)p.part, grid, p.hd, dwq, dwk);
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
