// Keys and values into a paged cache of 8 bits (kv8.h), rotated on the way and normed where weights are given; and out again.
//
//   n = x r w (with weights; r = 1 / sqrt(mean(x^2) + eps)),  y = R(p) n of query and key heads,  v as it is
//   e(token) = the least exponent byte with amax <= 448 2^(e - 127), over a head's numbers
//   e(group) = the largest of its new tokens', and of what the group had where rows of it were held before
//   code = e4m3(y 2^(127 - e)), rounded once from f32; rows held before are rounded again where e grew.
//
// Keys are normed and turned in 64 bits and reach their codes by one rounding (odd_f32): a code is then the nearest of the key's own
// value, the same wherever and in whatever company it was computed.  In f32 a few keys of a million lie so near a border
// that the sums' order decides (6 of 4.2 million normed ones); 64 bits cost nothing that is seen, a key head in six.
//
// A row held before is one ahead of the newest row that is not written now: the group's first row alone starts a group
// afresh, whatever a page held for its last owner.  Rows behind the newest stay as they are.
//
// Bound by memory (prompts) and by a few dependent loads (single tokens).  A wave has one group of one head: 16 rows of four
// lanes, each with D / 8 pairs (i, i + D / 2), so the rotation needs no neighbour, a norm two lane swaps, and the group's
// largest value one fold of the wave.  4,096 rows of 48 heads of 128 behind 1,003 positions, normed: 26.5 us (109 MB, 4.1 TB/s; a copy
// of as much runs at 5.9), read back 6.4 (25 MB).  64 single tokens of 80 heads of 128 6.6 us, one of 48 heads of 64 3.9.
#include "kv8.h"

namespace mx {

// A lane's P numbers of a head's half are pieces of 8 (4 where P is 4), of neighbouring lanes side by side: the second piece is
// four pieces further.
__device__ __forceinline__ constexpr int piece(int i) { return i / 8 * 32 + i % 8; }

template <int P>
__device__ __forceinline__ void load_bf(const uint16_t* p, float (&x)[P]) {
  if constexpr (P == 4) {
    const u16x4 v = *reinterpret_cast<const u16x4*>(p);
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = bf2f(v[j]);
  } else {
#pragma unroll
    for (int i = 0; i < P; i += 8) {
      const u16x8 v = *reinterpret_cast<const u16x8*>(p + piece(i));
#pragma unroll
      for (int j = 0; j < 8; ++j) x[i + j] = bf2f(v[j]);
    }
  }
}
template <int P>
__device__ __forceinline__ void store_bf(uint16_t* p, const float (&x)[P]) {
  if constexpr (P == 4) {
    u16x4 v;
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = f2bf(x[j]);
    *reinterpret_cast<u16x4*>(p) = v;
  } else {
#pragma unroll
    for (int i = 0; i < P; i += 8) {
      u16x8 v;
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = f2bf(x[i + j]);
      *reinterpret_cast<u16x8*>(p + piece(i)) = v;
    }
  }
}
template <int P>
__device__ __forceinline__ void load_f32(const float* p, float (&x)[P]) {
#pragma unroll
  for (int i = 0; i < P; i += 4) {
    const f32x4 v = *reinterpret_cast<const f32x4*>(p + piece(i));
#pragma unroll
    for (int j = 0; j < 4; ++j) x[i + j] = v[j];
  }
}
typedef uint32_t u32x2c __attribute__((ext_vector_type(2)));
template <int P>
__device__ __forceinline__ void store_codes(uint8_t* p, const float (&x)[P], int s) {
  if constexpr (P == 4) *reinterpret_cast<uint32_t*>(p) = kv8_code4(x[0], x[1], x[2], x[3], s);
  else {
#pragma unroll
    for (int i = 0; i < P; i += 8)
      *reinterpret_cast<u32x2c*>(p + piece(i)) = u32x2c{kv8_code4(x[i], x[i + 1], x[i + 2], x[i + 3], s),
                                                        kv8_code4(x[i + 4], x[i + 5], x[i + 6], x[i + 7], s)};
  }
}
template <int P>
__device__ __forceinline__ void load_codes(const uint8_t* p, float (&x)[P], int s) {
  if constexpr (P == 4) kv8_value4(*reinterpret_cast<const uint32_t*>(p), s, x);
  else {
#pragma unroll
    for (int i = 0; i < P; i += 8) {
      const u32x2c w = *reinterpret_cast<const u32x2c*>(p + piece(i));
      kv8_value4(w[0], s, x + i);
      kv8_value4(w[1], s, x + i + 4);
    }
  }
}
// x by the nearest f32 with an odd last bit where f32 does not hold it: rounded to fewer bits afterwards, as x itself would be
__device__ __forceinline__ float odd_f32(double x) {
  const float f = (float)x;
  uint32_t b = __float_as_uint(f);
  if ((double)f != x && !(b & 1)) b += fabs((double)f) < fabs(x) ? 1 : -1;
  return __uint_as_float(b);
}
template <int O>
__device__ __forceinline__ double lane_sum(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  constexpr int C = O == 2 ? 0x4E : 0xB1;  // quad_perm: lane ^ O
  static_assert(O == 1 || O == 2, "within four lanes");
  const uint64_t other = ((uint64_t)lane_dpp<C>((uint32_t)(b >> 32)) << 32) | lane_dpp<C>((uint32_t)b);
  return v + __builtin_bit_cast(double, other);
}
// a, b: the pairs' halves; n = x r w (w null: x), turned by the angles of cos, sin; T: float or double.  N pairs at a time, the
// next ones' angles and weights not asked for before these are done (the compiler would put the products off until all
// are there, 152 registers, 244 with 16 pairs at a time): 122 registers, four waves a SIMD, with 128 channels, 74 and six with
// 64.  4,096 rows of 48 heads of 128 26.3 us (16 pairs at a time 31.6, 4 27.5), six prompts of 17 to 901 rows of 48 heads of 64 9.1
// (8 at a time 10.0).
template <typename T, int P>
__device__ __forceinline__ void norm_turn(float (&a)[P], float (&b)[P], const uint16_t* w, int half, const float* cosb,
                                          const float* sinb, T eps) {
  constexpr int N = P < 16 ? 4 : 8;
  static_assert(P % N == 0 && (N % 8 == 0 || P <= 8), "whole pieces, or parts of the only one");
  T r = 1;
  if (w) {
    T ss = 0;
#pragma unroll
    for (int j = 0; j < P; ++j) ss += (T)a[j] * (T)a[j] + (T)b[j] * (T)b[j];
    ss = lane_sum<2>(lane_sum<1>(ss)) * (T)(1.0 / (2 * half)) + eps;
    if constexpr (sizeof(T) == 8) r = 1.0 / sqrt(ss);
    else r = rsqrtf(ss);
    if constexpr (sizeof(T) == 8) {  // (made 64 bits anew below: kept, they are 4 P registers)
#pragma unroll
      for (int j = 0; j < P; ++j) asm volatile("" : "+v"(a[j]), "+v"(b[j]));
    }
  }
#pragma unroll
  for (int p = 0; p < P; p += N) {
    float cs[N], sn[N], w1[N], w2[N];
    load_f32<N>(cosb + piece(p), cs);
    load_f32<N>(sinb + piece(p), sn);
    if (w) {
      load_bf<N>(w + piece(p), w1);
      load_bf<N>(w + half + piece(p), w2);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) w1[j] = w2[j] = 1.f;
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const T x = (T)a[p + j] * r * (T)w1[j], y = (T)b[p + j] * r * (T)w2[j], c = cs[j], s = sn[j];
      if constexpr (sizeof(T) == 8) {
        a[p + j] = odd_f32(x * c - y * s);
        b[p + j] = odd_f32(y * c + x * s);
      } else {
        a[p + j] = rope_lo(x, y, c, s);
        b[p + j] = rope_hi(x, y, c, s);
      }
    }
    if constexpr (P > N) {
#pragma unroll
      for (int j = 0; j < N; ++j) asm volatile("" : "+v"(a[p + j]), "+v"(b[p + j]));
    }
  }
}
// |x| where it is a number
__device__ __forceinline__ float number(float x) {
  x = fabsf(x);
  return x <= 3.4028234663852886e38f ? x : 0.f;
}

// index: RUNS: runs int4 [n] = (first row, rows, slot, first position), rows of one sequence within one group of positions;
// else the positions of n rows, slots theirs (null: the row's number).
// q: RUNS [Hq, T, D], with kout, vout [Hkv, T, D]; else [n, Hq, D].
template <int D, bool RUNS>
__global__ void __launch_bounds__(256)
    kv8_append_kernel(const uint16_t* __restrict__ qkv, int64_t ld, const float* __restrict__ cosb,
                      const float* __restrict__ sinb, int turns, const int32_t* __restrict__ index,
                      const int32_t* __restrict__ slots, int n, int T, const uint16_t* __restrict__ wq,
                      const uint16_t* __restrict__ wk, double eps, uint16_t* __restrict__ q, uint16_t* __restrict__ kout,
                      uint16_t* __restrict__ vout, Kv8Pages pg, int Hq) {
  constexpr int P = D / 8, HALF = D / 2;
  const int Hkv = pg.Hkv, NH = Hq + 2 * Hkv;
  int64_t item = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, row = lane >> 2, c = (P < 8 ? P : 8) * (lane & 3);
  const int cap = (int)min((int64_t)pg.maxp * pg.block, (int64_t)turns);  // positions that a sequence can have
  if constexpr (!RUNS) {
    // single tokens: the first waves have 16 query heads each, of whatever rows, the others a key or value head of a row
    const int64_t heads = (int64_t)n * Hq, first = (heads + kUnit - 1) / kUnit;
    if (item < first) {
      const int64_t h = min(item * kUnit + row, heads - 1);  // (lanes past the end help with the sums of a norm)
      const int at = (int)(h / Hq), head = (int)(h % Hq), p = index[at], s = slots ? slots[at] : at;
      const bool place = (unsigned)p < (unsigned)cap && (unsigned)s < (unsigned)pg.slots;  // else its queries are zero
      const uint16_t* src = qkv + at * ld + head * D + c;
      float a[P], b[P];
      load_bf<P>(src, a);
      load_bf<P>(src + HALF, b);
      const int64_t turn = (int64_t)(place ? p : 0) * HALF + c;
      norm_turn<float, P>(a, b, wq ? wq + c : nullptr, HALF, cosb + turn, sinb + turn, (float)eps);
#pragma unroll
      for (int j = 0; j < P; ++j) a[j] = place ? a[j] : 0.f, b[j] = place ? b[j] : 0.f;
      if (item * kUnit + row < heads) {
        uint16_t* dst = q + h * D + c;
        store_bf<P>(dst, a);
        store_bf<P>(dst + HALF, b);
      }
      return;
    }
    item -= first;
  }
  const int H = RUNS ? NH : 2 * Hkv;  // heads of a row here
  if (item >= (int64_t)n * H) return;
  const int at = (int)(item / H), head = (int)(item % H) + (RUNS ? 0 : Hq);
  int p0, slot, tk = -1;  // tk: the row of qkv of this lane's position, -1: none
  if constexpr (RUNS) {
    const int4 r = reinterpret_cast<const int4*>(index)[at];
    p0 = r.w, slot = r.z;
    if (r.x < 0 || r.y < 1 || r.y > kUnit || r.x > T - r.y || p0 < 0 || p0 > cap - r.y || (p0 % kUnit) + r.y > kUnit ||
        (unsigned)slot >= (unsigned)pg.slots)
      return;
    const int i = row - p0 % kUnit;
    if (i >= 0 && i < r.y) tk = r.x + i;
  } else {
    p0 = index[at], slot = slots ? slots[at] : at;
    if ((unsigned)p0 >= (unsigned)cap || (unsigned)slot >= (unsigned)pg.slots) return;
    // rows of the same group in this call belong to the first of them (of the same position the last one stays)
    bool found = false;
    for (int i0 = 0; i0 < n; i0 += 64) {
      const int i = i0 + lane;
      const int p = i < n ? index[i] : -1, s = i < n ? (slots ? slots[i] : i) : -1;
      uint64_t same = __ballot(s == slot && p >= 0 && p / kUnit == p0 / kUnit && p < cap);
      if (!same) continue;
      if (!found && i0 + __ffsll((unsigned long long)same) - 1 != at) return;
      found = true;
      for (; same; same &= same - 1) {
        const int l = __ffsll((unsigned long long)same) - 1;
        if (row == __builtin_amdgcn_readlane(p, l) % kUnit) tk = i0 + l;
      }
    }
  }
  const int group = p0 / kUnit;
  const bool isq = RUNS && head < Hq, isv = head >= Hq + Hkv, on = tk >= 0;
  float a[P], b[P];
#pragma unroll
  for (int j = 0; j < P; ++j) a[j] = b[j] = 0.f;
  if (on) {
    const uint16_t* src = qkv + tk * ld + head * D + c;
    load_bf<P>(src, a);
    load_bf<P>(src + HALF, b);
  }
  int64_t unit = -1;
  int old = 0;
  uint8_t *codes = nullptr, *exps = nullptr;
  if (!isq) {
    unit = kv8_unit(pg, slot, group, head - (isv ? Hq + Hkv : Hq));
    codes = (isv ? pg.v : pg.k) + unit * kUnit * D + row * D + c;
    exps = (isv ? pg.ve : pg.ke) + unit;
    if (unit >= 0) old = *exps;
  }
  if (!isv) {
    const int64_t turn = (int64_t)(on ? group * kUnit + row : 0) * HALF + c;
    if (isq) norm_turn<float, P>(a, b, wq ? wq + c : nullptr, HALF, cosb + turn, sinb + turn, (float)eps);
    else norm_turn<double, P>(a, b, wk ? wk + c : nullptr, HALF, cosb + turn, sinb + turn, eps);
  }
  if (RUNS && on) {
    uint16_t* dst = isq ? q + ((int64_t)head * T + tk) * D
                        : (isv ? vout : kout) + ((int64_t)(head - (isv ? Hq + Hkv : Hq)) * T + tk) * D;
    store_bf<P>(dst + c, a);
    store_bf<P>(dst + HALF + c, b);
  }
  if (isq || unit < 0) return;
  float top = 0.f;
#pragma unroll
  for (int j = 0; j < P; ++j) top = fmaxf(top, on ? fmaxf(number(a[j]), number(b[j])) : 0.f);
  int e = kv8_exponent(wave_max(top));
  const uint64_t fresh = __ballot(on);
  const int newest = (63 - __clzll((unsigned long long)fresh)) >> 2;
  const bool held = !on && row < newest;
  if (__ballot(held)) {
    if (e > old) {
      if (held) {
        float x[P], y[P];
        load_codes<P>(codes, x, old - e);
        load_codes<P>(codes + HALF, y, old - e);
        store_codes<P>(codes, x, 0);
        store_codes<P>(codes + HALF, y, 0);
      }
    } else {
      e = old;
    }
  }
  if (on) {
    store_codes<P>(codes, a, 127 - e);
    store_codes<P>(codes + HALF, b, 127 - e);
  }
  if (lane == 0) *exps = (uint8_t)e;
}

// Positions starts[b] + i, i < n, of slot slots[b] as bf16 [B, Hkv, n, D] (blockIdx.y 0: keys, 1: values): zero at ends[b] and
// behind it, NaN where the table names no page of the pool.
template <int D>
__global__ void __launch_bounds__(256)
    kv8_read_kernel(Kv8Pages pg, const int32_t* __restrict__ slots, const int32_t* __restrict__ starts,
                    const int32_t* __restrict__ ends, uint16_t* __restrict__ k, uint16_t* __restrict__ v, int B, int n) {
  constexpr int P = D / 8, HALF = D / 2;
  const uint32_t per = (n + kUnit - 1) / kUnit;
  const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (item >= (int64_t)B * pg.Hkv * per) return;
  const int i = (int)(item % per) * kUnit + ((threadIdx.x & 63) >> 2), c = (P < 8 ? P : 8) * (threadIdx.x & 3);
  const int hk = (int)(item / per % pg.Hkv), b = (int)(item / per / pg.Hkv);
  if (i >= n) return;
  const int slot = slots ? slots[b] : b;
  const int64_t p = (int64_t)starts[b] + i;
  float x[P], y[P];
#pragma unroll
  for (int j = 0; j < P; ++j) x[j] = y[j] = 0.f;
  if (p >= 0 && p < min((int64_t)ends[b], (int64_t)pg.maxp * pg.block) && (unsigned)slot < (unsigned)pg.slots) {
    const int64_t unit = kv8_unit(pg, slot, (int)(p / kUnit), hk);
    if (unit >= 0) {
      const uint8_t* codes = (blockIdx.y ? pg.v : pg.k) + (unit * kUnit + p % kUnit) * D + c;
      const int s = (int)(blockIdx.y ? pg.ve : pg.ke)[unit] - 127;
      load_codes<P>(codes, x, s);
      load_codes<P>(codes + HALF, y, s);
    } else {
#pragma unroll
      for (int j = 0; j < P; ++j) x[j] = y[j] = __builtin_nanf("");
    }
  }
  uint16_t* dst = (blockIdx.y ? v : k) + (((int64_t)b * pg.Hkv + hk) * n + i) * D + c;
  store_bf<P>(dst, x);
  store_bf<P>(dst + HALF, y);
}

}  // namespace mx

using namespace mx;

// runs != 0: index int32 [n, 4], q, kout, vout head-major; else index int32 [n] (n = T rows)
extern "C" int mx_kv8_append(const uint16_t* qkv, int64_t ld, const float* cosb, const float* sinb, int turns, int runs,
                             const int32_t* index, const int32_t* slots, int n, int T, const uint16_t* wq,
                             const uint16_t* wk, double eps, uint16_t* q, uint16_t* kout, uint16_t* vout, const Kv8Pages* cache,
                             int Hq, int D, hipStream_t stream) {
  if (n <= 0) return 0;
  const int64_t waves = runs ? (int64_t)n * (Hq + 2 * cache->Hkv)
                             : ((int64_t)n * Hq + kUnit - 1) / kUnit + (int64_t)n * 2 * cache->Hkv;
  const int64_t blocks = (waves + 3) / 4;
  if (blocks > INT32_MAX) return -1;
#define APPEND(DD, RR)                                                                                                \
  kv8_append_kernel<DD, RR><<<(unsigned)blocks, 256, 0, stream>>>(qkv, ld, cosb, sinb, turns, index, slots, n, T, wq, \
                                                                  wk, eps, q, kout, vout, *cache, Hq)
#define APPENDS(DD)               \
  do {                            \
    if (runs) APPEND(DD, true);   \
    else APPEND(DD, false);       \
  } while (0)
  if (D == 128) APPENDS(128);
  else if (D == 64) APPENDS(64);
  else if (D == 32) APPENDS(32);
  else return -1;
#undef APPENDS
#undef APPEND
  return (int)hipGetLastError();
}

extern "C" int mx_kv8_read(const Kv8Pages* cache, const int32_t* slots, const int32_t* starts, const int32_t* ends, uint16_t* k,
                           uint16_t* v, int B, int n, int D, hipStream_t stream) {
  const int64_t blocks = ((int64_t)B * cache->Hkv * ((n + kUnit - 1) / kUnit) + 3) / 4;
  if (blocks <= 0) return 0;
  if (blocks > INT32_MAX) return -1;
  const dim3 grid((unsigned)blocks, 2);
  if (D == 128) kv8_read_kernel<128><<<grid, 256, 0, stream>>>(*cache, slots, starts, ends, k, v, B, n);
  else if (D == 64) kv8_read_kernel<64><<<grid, 256, 0, stream>>>(*cache, slots, starts, ends, k, v, B, n);
  else if (D == 32) kv8_read_kernel<32><<<grid, 256, 0, stream>>>(*cache, slots, starts, ends, k, v, B, n);
  else return -1;
  return (int)hipGetLastError();
}
