// RMS norm of every query and key head with the rotation of its position in the same pass, forward and backward.
//
// A head x of D channels of a qkv row at position p, its weight w (one of D channels for all query heads, one for all key
// heads), r = 1 / sqrt(mean(x^2) + eps):
//   y = R(p) (x r w),   R(p): the pairs (i, i + D / 2) turned by the table's angle of p and i.
// Backward, dy the gradient of y:
//   dn = R(p)^T dy,  g = w dn,  dx = r g - x r^3 mean(g x),  dw = sum over heads and rows of dn x r.
// x is read again and r formed anew, so nothing is kept between the passes but the rows themselves.
//
// Both are bound by memory: every row is read and every head written once (backward: rows and gradients read, gradients
// written).  A thread has 8 pairs of one head (two pieces of 16 bytes), D / 16 neighbouring threads a head, whose sums
// go by lane swaps.  Sums and products are f32; each output is rounded once.  4,096 rows of 48 heads of 128, forward 21 us (101 MB,
// 4.8 TB/s), backward 28 (143 MB, 5.1) and 4 for the weights' sums; 8,192 rows of 80 heads 57 us (5.8) and 104 + 4 (4.7).  Plain copies of
// as much run at 5.9 and 6.2 TB/s, sums of two arrays at 5.9.
#include "common.h"

namespace mx {

// sum over the N (2, 4, 8) neighbouring lanes of a head, in all of them
template <int N>
__device__ __forceinline__ float head_sum(float v) {
  v = lane_sum<1>(v);
  if constexpr (N >= 4) v = lane_sum<2>(v);
  if constexpr (N >= 8) v += __uint_as_float(lane_dpp<0x141>(__float_as_uint(v)));  // row_half_mirror: the other four
  return v;
}

__device__ __forceinline__ void load8(const uint16_t* p, float (&x)[8]) {
  const u16x8 v = *reinterpret_cast<const u16x8*>(p);
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = bf2f(v[j]);
}
__device__ __forceinline__ void load8(const float* p, float (&x)[8]) {
  const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
  for (int j = 0; j < 4; ++j) x[j] = a[j], x[j + 4] = b[j];
}
__device__ __forceinline__ void store8(uint16_t* p, const float (&x)[8]) {
  u16x8 v;
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = f2bf(x[j]);
  *reinterpret_cast<u16x8*>(p) = v;
}
// the table's row of a position; one outside the table turns what it is used for into NaN
__device__ __forceinline__ void load_turn(const float* cosb, const float* sinb, int pos, int rows, int half, int c,
                                          float (&cs)[8], float (&sn)[8]) {
  const bool in = (unsigned)pos < (unsigned)rows;
  const int64_t at = (int64_t)(in ? pos : 0) * half + c;
  load8(cosb + at, cs);
  load8(sinb + at, sn);
  if (!in) {
#pragma unroll
    for (int j = 0; j < 8; ++j) cs[j] = sn[j] = __builtin_nanf("");
  }
}

template <int D>
__global__ void __launch_bounds__(256)
    qk_norm_rope_kernel(const uint16_t* __restrict__ qkv, int64_t ld, const uint16_t* __restrict__ wq,
                        const uint16_t* __restrict__ wk, const float* __restrict__ cosb, const float* __restrict__ sinb,
                        const int32_t* __restrict__ positions, int rows, uint16_t* __restrict__ q,
                        uint16_t* __restrict__ k, uint16_t* __restrict__ v, int T, int S, int Hq, int Hkv, float eps) {
  constexpr int HALF = D / 2, CPH = D / 16;
  const int NH = Hq + 2 * Hkv;
  const uint32_t n = (uint32_t)T * NH;
  const uint32_t at = blockIdx.x * (256 / CPH) + threadIdx.x / CPH, th = min(at, n - 1);  // (lanes past the end help with sums)
  const uint32_t head = th % NH, t = th / NH, s = t % S, b = t / S;
  const int c = (threadIdx.x % CPH) * 8;
  const uint16_t* src = qkv + t * ld + head * D;
  float x1[8], x2[8];
  load8(src + c, x1);
  load8(src + HALF + c, x2);
  uint16_t* dst;
  if (head < (uint32_t)Hq) dst = q + (((int64_t)b * Hq + head) * S + s) * D;
  else if (head < (uint32_t)(Hq + Hkv)) dst = k + (((int64_t)b * Hkv + (head - Hq)) * S + s) * D;
  else dst = v + (((int64_t)b * Hkv + (head - Hq - Hkv)) * S + s) * D;
  const bool turned = head < (uint32_t)(Hq + Hkv);
  float cs[8], sn[8], w1[8], w2[8];
  load_turn(cosb, sinb, positions ? positions[t] : (int)s, rows, HALF, c, cs, sn);
  const uint16_t* w = head < (uint32_t)Hq ? wq : wk;
  load8(w + c, w1);
  load8(w + HALF + c, w2);
  float ss = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) ss += x1[j] * x1[j] + x2[j] * x2[j];
  const float r = rsqrtf(head_sum<CPH>(ss) * (1.f / D) + eps);
  if (turned) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float a = x1[j] * r * w1[j], e = x2[j] * r * w2[j];
      x1[j] = rope_lo(a, e, cs[j], sn[j]);
      x2[j] = rope_hi(a, e, cs[j], sn[j]);
    }
  }
  if (at < n) {
    store8(dst + c, x1);
    store8(dst + HALF + c, x2);
  }
}

// What a workgroup of the backward has: query, key or value heads (roles 0, 1, 2), every `blocks`-th group of them.
// G: type of the gradients, [B, H, S, D]; those of keys and values as `rep` summands a head, consecutive heads.
// part: f32 [blocks of q and k, D], the workgroup's sum of dn x r; the value heads are only moved.
template <int D, typename G>
__global__ void __launch_bounds__(256)
    qk_norm_rope_bwd_kernel(const G* __restrict__ dq, const G* __restrict__ dk, const G* __restrict__ dv, int rep,
                            const uint16_t* __restrict__ qkv, int64_t ld, const uint16_t* __restrict__ wq,
                            const uint16_t* __restrict__ wk, const float* __restrict__ cosb,
                            const float* __restrict__ sinb, const int32_t* __restrict__ positions, int rows,
                            uint16_t* __restrict__ dqkv, int64_t ldo, float* __restrict__ part, int T, int S, int Hq,
                            int Hkv, float eps, int nbq, int nbk, int nbv) {
  constexpr int HALF = D / 2, CPH = D / 16, HPB = 256 / CPH;
  __shared__ float sums[4][D];
  const int blk = blockIdx.x;
  const int role = blk < nbq ? 0 : blk < nbq + nbk ? 1 : 2;
  const int H = role ? Hkv : Hq, off = role == 0 ? 0 : role == 1 ? Hq : Hq + Hkv;
  const int first = role == 0 ? blk : role == 1 ? blk - nbq : blk - nbq - nbk, step = role == 0 ? nbq : role == 1 ? nbk : nbv;
  const G* grad = role == 0 ? dq : role == 1 ? dk : dv;
  const int nsum = role ? rep : 1;
  const int c = (threadIdx.x % CPH) * 8;
  const int64_t n = (int64_t)T * H;
  float w1[8], w2[8], dw1[8], dw2[8];
  const uint16_t* w = role ? wk : wq;
  load8(w + c, w1);
  load8(w + HALF + c, w2);
#pragma unroll
  for (int j = 0; j < 8; ++j) dw1[j] = dw2[j] = 0.f;
  for (int64_t base = (int64_t)first * HPB; base < n; base += (int64_t)step * HPB) {  // the same turns in every thread
    const bool on = base + threadIdx.x / CPH < n;
    const uint32_t th = (uint32_t)min(base + threadIdx.x / CPH, n - 1);
    const uint32_t h = th % H, t = th / H, s = t % S, b = t / S;
    float a1[8], a2[8];
    const G* g = grad + (((int64_t)b * H + h) * nsum * S + s) * D;
    load8(g + c, a1);
    load8(g + HALF + c, a2);
    for (int i = 1; i < nsum; ++i) {
      float e1[8], e2[8];
      load8(g + (int64_t)i * S * D + c, e1);
      load8(g + (int64_t)i * S * D + HALF + c, e2);
#pragma unroll
      for (int j = 0; j < 8; ++j) a1[j] += e1[j], a2[j] += e2[j];
    }
    uint16_t* dst = dqkv + t * ldo + (off + h) * D;
    if (role < 2) {
      float x1[8], x2[8], cs[8], sn[8];
      const uint16_t* src = qkv + t * ld + (off + h) * D;
      load8(src + c, x1);
      load8(src + HALF + c, x2);
      load_turn(cosb, sinb, positions ? positions[t] : (int)s, rows, HALF, c, cs, sn);
      float ss = 0.f, gx = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float lo = __builtin_fmaf(a1[j], cs[j], a2[j] * sn[j]), hi = __builtin_fmaf(a2[j], cs[j], -(a1[j] * sn[j]));
        a1[j] = lo, a2[j] = hi;
        ss += x1[j] * x1[j] + x2[j] * x2[j];
        gx += lo * w1[j] * x1[j] + hi * w2[j] * x2[j];
      }
      ss = head_sum<CPH>(ss);
      gx = head_sum<CPH>(gx);
      const float r = rsqrtf(ss * (1.f / D) + eps), f = r * r * (gx * (1.f / D)), live = on ? r : 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        dw1[j] += on ? a1[j] * x1[j] * live : 0.f;  // (a lane past the end holds another's head, NaN with it)
        dw2[j] += on ? a2[j] * x2[j] * live : 0.f;
        a1[j] = r * (a1[j] * w1[j] - x1[j] * f);
        a2[j] = r * (a2[j] * w2[j] - x2[j] * f);
      }
    }
    if (on) {
      store8(dst + c, a1);
      store8(dst + HALF + c, a2);
    }
  }
  if (role == 2) return;
  // the heads of a wave, then its four waves, always in the same order
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float x = half ? dw2[j] : dw1[j];
      x = lane_sum<8>(lane_sum<16>(lane_sum<32>(x)));
      if constexpr (CPH <= 4) x = lane_sum<4>(x);
      if constexpr (CPH <= 2) x = lane_sum<2>(x);
      if (lane < CPH) sums[wave][half * HALF + c + j] = x;
    }
  }
  __syncthreads();
  for (int d = threadIdx.x; d < D; d += 256) part[(int64_t)blk * D + d] = sums[0][d] + sums[1][d] + sums[2][d] + sums[3][d];
}

// columns of part [nbq + nbk, D] -> dwq (blockIdx.y 0: the first nbq rows), dwk (1): 16 channels a workgroup
__global__ void __launch_bounds__(256) qk_norm_dw_kernel(const float* __restrict__ part, int nbq, int nbk, int D,
                                                         void* __restrict__ dwq, void* __restrict__ dwk, int f32) {
  __shared__ float sums[64][17];
  const int c = blockIdx.x * 16 + (threadIdx.x & 3) * 4, r0 = threadIdx.x >> 2;
  const int n = blockIdx.y ? nbk : nbq;
  const float* p = part + (blockIdx.y ? (int64_t)nbq * D : 0) + c;
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int r = r0; r < n; r += 64) s += *reinterpret_cast<const f32x4*>(p + (int64_t)r * D);
#pragma unroll
  for (int j = 0; j < 4; ++j) sums[r0][(threadIdx.x & 3) * 4 + j] = s[j];
  __syncthreads();
  if (threadIdx.x >= 16) return;
  float x = 0.f;
#pragma unroll 8
  for (int r = 0; r < 64; ++r) x += sums[r][threadIdx.x];
  void* out = blockIdx.y ? dwk : dwq;
  const int d = blockIdx.x * 16 + threadIdx.x;
  if (f32) reinterpret_cast<float*>(out)[d] = x;
  else reinterpret_cast<uint16_t*>(out)[d] = f2bf(x);
}

// workgroups of a role: its share of four a CU (all there at once; eight 102.0 -> 99.9 us for 8,192 rows of 80 heads of 128), no more
// than its heads fill
static int bwd_blocks(int64_t heads, int H, int NH, int D) {
  const int64_t per = 256 / (D / 16), all = (heads + per - 1) / per, most = (int64_t)1024 * H / NH;
  return (int)(all < most ? all : most < 1 ? 1 : most);
}

}  // namespace mx

using namespace mx;

// qkv rows of stride ld; q [B, Hq, S, D], k, v [B, Hkv, S, D]; the table has `rows` positions
extern "C" int mx_qk_norm_rope(const uint16_t* qkv, int64_t ld, const uint16_t* wq, const uint16_t* wk, const float* cosb,
                               const float* sinb, const int32_t* positions, int rows, uint16_t* q, uint16_t* k,
                               uint16_t* v, int B, int S, int Hq, int Hkv, int D, float eps, hipStream_t stream) {
  const int64_t heads = (int64_t)B * S * (Hq + 2 * Hkv);
  if (heads <= 0) return 0;
  if (heads > INT32_MAX / 16 * 15) return -1;
#define FWD(DD)                                                                                                     \
  qk_norm_rope_kernel<DD><<<(unsigned)((heads + 256 / (DD / 16) - 1) / (256 / (DD / 16))), 256, 0, stream>>>(       \
      qkv, ld, wq, wk, cosb, sinb, positions, rows, q, k, v, B * S, S, Hq, Hkv, eps)
  if (D == 128) FWD(128);
  else if (D == 64) FWD(64);
  else if (D == 32) FWD(32);
  else return -1;
#undef FWD
  return (int)hipGetLastError();
}

extern "C" int mx_qk_norm_rope_bwd_parts(int B, int S, int Hq, int Hkv, int D) {
  const int64_t T = (int64_t)B * S;
  return bwd_blocks(T * Hq, Hq, Hq + 2 * Hkv, D) + bwd_blocks(T * Hkv, Hkv, Hq + 2 * Hkv, D);
}

// f32 gradients: g32 != 0; dwq, dwk null: the weights' gradients are not wanted; dw32: they are f32, else bf16
extern "C" int mx_qk_norm_rope_bwd(const void* dq, const void* dk, const void* dv, int g32, int rep, const uint16_t* qkv,
                                   int64_t ld, const uint16_t* wq, const uint16_t* wk, const float* cosb,
                                   const float* sinb, const int32_t* positions, int rows, uint16_t* dqkv, int64_t ldo,
                                   float* part, void* dwq, void* dwk, int dw32, int B, int S, int Hq, int Hkv, int D,
                                   float eps, hipStream_t stream) {
  const int64_t T = (int64_t)B * S;
  if (T <= 0) return 0;
  if (T * (Hq + 2 * Hkv) > INT32_MAX / 16 * 15) return -1;
  const int NH = Hq + 2 * Hkv;
  const int nbq = bwd_blocks(T * Hq, Hq, NH, D), nbk = bwd_blocks(T * Hkv, Hkv, NH, D), nbv = nbk;
#define BWD(DD, GG)                                                                                                      \
  qk_norm_rope_bwd_kernel<DD, GG><<<nbq + nbk + nbv, 256, 0, stream>>>(                                                  \
      (const GG*)dq, (const GG*)dk, (const GG*)dv, rep, qkv, ld, wq, wk, cosb, sinb, positions, rows, dqkv, ldo, part,   \
      (int)T, S, Hq, Hkv, eps, nbq, nbk, nbv)
  if (g32) {
    if (D == 128) BWD(128, float);
    else if (D == 64) BWD(64, float);
    else if (D == 32) BWD(32, float);
    else return -1;
  } else {
    if (D == 128) BWD(128, uint16_t);
    else if (D == 64) BWD(64, uint16_t);
    else if (D == 32) BWD(32, uint16_t);
    else return -1;
  }
#undef BWD
  const int rc = (int)hipGetLastError();
  if (rc || !dwq) return rc;
  qk_norm_dw_kernel<<<dim3(D / 16, 2), 256, 0, stream>>>(part, nbq, nbk, D, dwq, dwk, dw32);
  return (int)hipGetLastError();
}
