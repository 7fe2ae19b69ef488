// Attention of one token of each sequence over a paged cache of 8 bits (kv8.h):
//   o = softmax(q k^T scale) v over positions 0 .. pos, queries of a group of heads sharing a key/value head.
//
// Bound by memory: a key and a value of a head are 2 D bytes, half of a bf16 cache's, each read once for all query heads of the
// group.  8 sequences of 16,384 keys (8 heads of 128, 269 MB) 48 us, of which the merge 4.5; a linear read of as much takes 39.
//
//   S^T[key][head] = 2^(ek - 127) scale log2(e) (K . Q^T),  O^T[d][head] += (2^(ev - 127) V^T) . P
// by v_mfma_f32_16x16x32_bf16 on codes that become bf16 in registers, where they are exact, the units' (16 positions) powers of
// two in the scores and in the conversion of values.  Sums and outputs are f32; a weight is the sum of two numbers of bf16, off by
// 2^-16 of it, so an output is as near to 64 bits as its own rounding leaves it (1.66e-3 of its norm; with one number 2.3e-3, and 1
// to 4 % less time: 32 rows of 100 .. 2000 keys of 128 15.5 us, 15.9 with two, 8 of 16,384 47.6 and 47.8, 64 of 2048 .. 4096 68.7
// and 69.8).  (Scores on the codes themselves, queries as sums of two e4m3 codes under v_mfma_scale_f32_16x16x128_f8f6f4, save
// 32 conversions a tile and no time, and that product drops what is 2^-13 of its largest summand.)
//
// A wave works on tiles of two units, 32 keys and values.  They come to its own part of LDS by loads of 1 KB, whole rows, that
// are not kept in the caches, the next tile's while this one is worked on, and nothing waits for another wave.  A lane (c, g)
// then takes row c of each unit, pieces of 16 bytes 64 h + 16 g (a dot product does not mind the order of channels, and queries
// are laid out alike), and of eight value rows its D / 16 channels, whose bytes are put together row by row as the product
// reads them.  Us with what was there before (a weight was one number then, parts lay by row), memory's caches cold / as three calls
// in turn leave them:
//   a lane's rows straight to registers, kept in the caches    32 x 100 .. 2000 of 128 19.6 / 16.6, 8 x 16384 54.9 / 54.6
//   the same, not kept (rows of half a line: 40 x 1000 .. 4000 of 64 18.2 -> 19.7)      20.6 / 20.0,            49.8 / 49.3
//   whole rows by LDS, not kept                                                        18.2 / 17.4,            49.8 / 48.9
//   and the next tile on its way                                                       16.1 / 15.4,            47.8 / 47.3
// and 64 x 2048 .. 4096 78.3 -> 71.9 -> 69.1 -> 66.7 cold (now 70, 5.9 TB/s; a linear read of as much 59); one of 700 keys does not
// mind.  (Keys of the tile after next asked for as soon as a tile's are read, values alike, was 2 to 8 % slower.)
//
// Rows are whole (a workgroup each, nothing to merge) or cut: the units of all sequences in a row are dealt in equal
// shares, one a workgroup of a KV head, whose waves share what it has of a sequence, and sequences that were cut are merged by a
// second launch.  Where a row is cut follows from the lengths of all, so the last bits of an output may
// differ from batch to batch (the same call has the same bits).
//
// Waves and parts hand on means, sum of w v over sum of w, which are no larger than the values are; a wave's own sums, of weights up
// to 2^8, are held in units of 2^32 as soon as a unit of its keys has values that could take them past the end of f32 (kFar).
#include "kv8.h"

namespace mx {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4v __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2v __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(1))) const void* gptr_t;
typedef __attribute__((address_space(3))) void* lptr_t;
constexpr int kNt = 2;  // of a load: read once
// The exponent byte of values from which on a wave's sums are in units of 2^32: below it 2^21 weights of 2^8 of values up to
// 448 * 2^80 stay under 2^127.  (Beside values of 2^81 and more those under 2^-86 count for up to that much.)
constexpr int kFar = 208, kFarBy = 32;

__device__ __forceinline__ f32x4 mfma16(const u32x4v& a, const u16x8& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0,
                                                 0, 0);
}
__device__ __forceinline__ uint32_t pair_bf16(uint32_t w, float scale, bool high) {
  return high ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true))
              : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false));
}

template <int E>
struct VPiece {
  typedef uint32_t type;
};
template <>
struct VPiece<8> {
  typedef u32x2v type;
};
__device__ __forceinline__ uint32_t word(u32x2v v, int i) { return v[i]; }
__device__ __forceinline__ uint32_t word(uint32_t v, int) { return v; }

// channel of k-step s of lane group g
template <int D>
__device__ __forceinline__ int chan(int s, int g) {
  return D == 32 ? 8 * g : 64 * (s >> 1) + 16 * g + 8 * (s & 1);
}

// Products of queries and codes come ahead of the codes' power of two, so the queries of a head (that of four lanes) that could
// take their sum past f32 are divided by 2^qe = 2^32 (else 1); true: some head's are.  128 products of 2^96 and codes up to 448
// stay under 2^112.
template <int KS>
__device__ __forceinline__ bool shrink_queries(u16x8 (&q)[KS], int& qe) {
  constexpr uint16_t kBig = (127 + 96) << 7;
  uint16_t top = 0;
#pragma unroll
  for (int s = 0; s < KS; ++s) {
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, (uint16_t)(q[s][j] & 0x7fff));
  }
  qe = 0;
  if (!__ballot(top >= kBig)) return false;
  if (lane_max<32>(lane_max<16>(bf2f(top))) >= 0x1p96f) {
    qe = 32;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
#pragma unroll
      for (int j = 0; j < 8; ++j) q[s][j] = f2bf(bf2f(q[s][j]) * 0x1p-32f);
    }
  }
  return true;
}

template <int D>
struct Kv8State {  // of one wave
  static constexpr int E = D / 16, KS = D / 32;
  float m, l;   // reference of the exponents of head c; l: this lane's keys
  f32x4 o[E];   // [e][i]: channel E (4 g + i) + e of head c
  int qe;       // the power of two that the queries of head c were divided by
  bool big;     // some head's were (the same in all lanes)
  bool far;     // o is in units of 2^kFarBy (the same in all lanes)

  __device__ __forceinline__ void clear() {
    m = -INFINITY, l = 0.f, qe = 0, big = far = false;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  // 16-byte piece `ch` of key `row` (of the tile's 32) in LDS: pieces of a row change places so that rows that start in the
  // same bank do not meet
  static __device__ __forceinline__ int place(int row, int ch) {
    constexpr int N = D / 16;  // pieces of a row
    return row * D + 16 * (ch ^ (N == 8 ? row & 7 : N == 4 ? (row >> 2) & 3 : 0));
  }
  // LDS addresses of a lane: of its pieces of a key (h: 64 channels further), of its channels of four value rows; units of a tile
  // are 16 D apart, values 32 D behind keys
  struct Places {
    uint32_t k[D == 128 ? 2 : 1], v[4];

    __device__ __forceinline__ Places(const char* lds, int c, int g) {
      const uint32_t base = lds_addr(lds);
      if constexpr (D == 32) k[0] = base + place(c, g >> 1) + 8 * (g & 1);
      else {
#pragma unroll
        for (int h = 0; h < D / 64; ++h) k[h] = base + place(c, 4 * h + g);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = base + 32 * D + place(4 * g + i, E * c / 16) + E * c % 16;
    }
  };

  // A unit's keys or values (16 rows) to LDS; ALL: every row of it is there; else lim: its last one (less than 0: none), and rows
  // behind it are read as that row.  As the products want them, a lane a row, a load would ask for 64 pieces of as many lines;
  // so it has whole rows, 1 KB.
  template <bool ALL>
  static __device__ __forceinline__ void load(char* lds, const uint8_t* unit, int lim, int lane) {
    constexpr int N = D / 16, ROWS = 64 / N;  // pieces of a row, rows of a load
    static_assert(D >= 64, "a load of one unit");
    const int r = lane / N, at = 16 * ((place(r, lane % N) - r * D) / 16);  // (the exchange is its own inverse)
    if constexpr (ALL) {
      asm("" : "+s"(unit));  // (a base for all lanes, not added to each one's offset)
      __builtin_amdgcn_global_load_lds((gptr_t)(unit + (uint32_t)(r * D + at)), (lptr_t)lds, 16, 0, kNt);
      if constexpr (ROWS == 8)  // rows 8 further change places alike
        __builtin_amdgcn_global_load_lds((gptr_t)(unit + (uint32_t)(r * D + at)), (lptr_t)lds, 16, 1024, kNt);
    } else {
      const int z = max(lim, 0);
#pragma unroll
      for (int i = 0; i < 16 / ROWS; ++i)
        __builtin_amdgcn_global_load_lds((gptr_t)(unit + (uint32_t)(min(ROWS * i + r, z) * D + at)), (lptr_t)(lds + 1024 * i),
                                         16, 0, kNt);
    }
  }
  // Both units of a tile, keys and values (rows of 32 bytes: a load has both units')
  template <bool ALL>
  static __device__ __forceinline__ void load_tile(char* lds, const uint8_t* k0, const uint8_t* k1, const uint8_t* v0,
                                                   const uint8_t* v1, int lim0, int lim1, int lane) {
    if constexpr (D == 32) {
      const int row = lane / 2, z = max(lane < 32 ? lim0 : lim1, 0);
      const uint32_t off = (ALL ? row & 15 : min(row & 15, z)) * D + 16 * (lane % 2);
      __builtin_amdgcn_global_load_lds((gptr_t)((lane < 32 ? k0 : k1) + off), (lptr_t)lds, 16, 0, kNt);
      __builtin_amdgcn_global_load_lds((gptr_t)((lane < 32 ? v0 : v1) + off), (lptr_t)(lds + 1024), 16, 0, kNt);
    } else {
      load<ALL>(lds, k0, lim0, lane);
      load<ALL>(lds + 16 * D, k1, lim1, lane);
      load<ALL>(lds + 32 * D, v0, lim0, lane);
      load<ALL>(lds + 48 * D, v1, lim1, lane);
    }
  }

  // off: the tile's half; ks: what the units' scores are multiplied by (NaN: the units are none), where `big` the powers of two
  // beside sl; vs: powers of two of their values; all: every row is there, else up to lim0, lim1
  __device__ __forceinline__ void take(const Places& from, uint32_t off, const u16x8 (&qf)[KS], float ks0, float ks1,
                                       float vs0, float vs1, float sl, bool all, int lim0, int lim1, int c, int g) {
    Places at = from;
#pragma unroll
    for (uint32_t& x : at.k) x += off;
#pragma unroll
    for (uint32_t& x : at.v) x += off;
    f32x4 sc[2];
    typename VPiece<E>::type v[8];  // slot s: row 4 g + (s & 3) of unit s >> 2, channels E c ..
    // (one block of reads and their wait: the compiler would wait for the next tile, which is on its way to the other half)
#define KV8_V(OP)                                                                                       \
  OP " %[v0], %[b0]\n\t" OP " %[v1], %[b1]\n\t" OP " %[v2], %[b2]\n\t" OP " %[v3], %[b3]\n\t"             \
  OP " %[v4], %[b0] offset:%[p]\n\t" OP " %[v5], %[b1] offset:%[p]\n\t" OP " %[v6], %[b2] offset:%[p]\n\t" \
  OP " %[v7], %[b3] offset:%[p]\n\ts_waitcnt lgkmcnt(0)"
#define KV8_V_OUT                                                                                             \
  [v0] "=&v"(v[0]), [v1] "=&v"(v[1]), [v2] "=&v"(v[2]), [v3] "=&v"(v[3]), [v4] "=&v"(v[4]), [v5] "=&v"(v[5]), \
      [v6] "=&v"(v[6]), [v7] "=&v"(v[7])
#define KV8_V_IN [b0] "v"(at.v[0]), [b1] "v"(at.v[1]), [b2] "v"(at.v[2]), [b3] "v"(at.v[3]), [p] "i"(16 * D)
    if constexpr (D == 32) {
      u32x2v w0, w2;
      asm volatile("ds_read_b64 %[w0], %[a0]\n\tds_read_b64 %[w2], %[a0] offset:%[p]\n\t" KV8_V("ds_read_u16")
                   : [w0] "=&v"(w0), [w2] "=&v"(w2), KV8_V_OUT : [a0] "v"(at.k[0]), KV8_V_IN : "memory");
      sc[0] = mfma16(__builtin_bit_cast(u32x4v, dequant8(w0[0], w0[1])), qf[0], f32x4{0.f, 0.f, 0.f, 0.f});
      sc[1] = mfma16(__builtin_bit_cast(u32x4v, dequant8(w2[0], w2[1])), qf[0], f32x4{0.f, 0.f, 0.f, 0.f});
    } else {
      u32x4v w0, w1, w2, w3;
      if constexpr (D == 128)
        asm volatile("ds_read_b128 %[w0], %[a0]\n\tds_read_b128 %[w2], %[a0] offset:%[p]\n\t"
                     "ds_read_b128 %[w1], %[a1]\n\tds_read_b128 %[w3], %[a1] offset:%[p]\n\t" KV8_V("ds_read_b64")
                     : [w0] "=&v"(w0), [w1] "=&v"(w1), [w2] "=&v"(w2), [w3] "=&v"(w3), KV8_V_OUT
                     : [a0] "v"(at.k[0]), [a1] "v"(at.k[1]), KV8_V_IN
                     : "memory");
      else
        asm volatile("ds_read_b128 %[w0], %[a0]\n\tds_read_b128 %[w2], %[a0] offset:%[p]\n\t" KV8_V("ds_read_b32")
                     : [w0] "=&v"(w0), [w2] "=&v"(w2), KV8_V_OUT : [a0] "v"(at.k[0]), KV8_V_IN : "memory");
      sc[0] = mfma16(__builtin_bit_cast(u32x4v, dequant8(w0[0], w0[1])), qf[0], f32x4{0.f, 0.f, 0.f, 0.f});
      sc[1] = mfma16(__builtin_bit_cast(u32x4v, dequant8(w2[0], w2[1])), qf[0], f32x4{0.f, 0.f, 0.f, 0.f});
      sc[0] = mfma16(__builtin_bit_cast(u32x4v, dequant8(w0[2], w0[3])), qf[1], sc[0]);
      sc[1] = mfma16(__builtin_bit_cast(u32x4v, dequant8(w2[2], w2[3])), qf[1], sc[1]);
      if constexpr (D == 128) {
        sc[0] = mfma16(__builtin_bit_cast(u32x4v, dequant8(w1[0], w1[1])), qf[2], sc[0]);
        sc[1] = mfma16(__builtin_bit_cast(u32x4v, dequant8(w3[0], w3[1])), qf[2], sc[1]);
        sc[0] = mfma16(__builtin_bit_cast(u32x4v, dequant8(w1[2], w1[3])), qf[3], sc[0]);
        sc[1] = mfma16(__builtin_bit_cast(u32x4v, dequant8(w3[2], w3[3])), qf[3], sc[1]);
      }
    }
#undef KV8_V
#undef KV8_V_OUT
#undef KV8_V_IN
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = sc[i >> 2][i & 3] * (i < 4 ? ks0 : ks1);
    if (big) {  // ks is small, down to where f32 has few bits, where queries are so large: powers of two by themselves
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float k = i < 4 ? ks0 : ks1;
        x[i] = k == k ? __builtin_ldexpf(sc[i >> 2][i & 3] * sl, (int)k + qe) : k;
      }
    }
    if (!all) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = 4 * g + (i & 3) <= (i < 4 ? lim0 : lim1) ? x[i] : -INFINITY;
    }
    // The exponents' reference is a maximum that may be behind by 2^8: weights up to there cost no precision, and the sums are
    // multiplied again in a few of the tiles only
    float top = x[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) top = fmaxf(top, x[i]);
    if (__ballot(top > m + 8.f)) {
      const float now = fmaxf(m, lane_max<32>(lane_max<16>(top))), f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - now);
      m = now;
      l *= f;
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] *= f;
    }
    const float mref = m == -INFINITY ? 0.f : m;
    u16x8 pb, rest;  // a weight as two numbers of bf16
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float p = __builtin_amdgcn_exp2f(x[i] - mref);
      l += p;
      pb[i] = f2bf(p);
      rest[i] = f2bf(p - bf2f(pb[i]));
    }
    // bytes 0, 1 or 2, 3 of the words of two rows side by side, as pairs of rows of one channel each
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      u32x4v a0, a1;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t w = __builtin_amdgcn_perm(word(v[2 * i + 1], e >> 2), word(v[2 * i], e >> 2),
                                                 e & 2 ? 0x07030602u : 0x05010400u);
        a0[i] = pair_bf16(w, i < 2 ? vs0 : vs1, false), a1[i] = pair_bf16(w, i < 2 ? vs0 : vs1, true);
      }
      o[e] = mfma16(a0, pb, o[e]);
      o[e + 1] = mfma16(a1, pb, o[e + 1]);
      o[e] = mfma16(a0, rest, o[e]);
      o[e + 1] = mfma16(a1, rest, o[e + 1]);
    }
  }
};

// a row's output: zero without keys; keys that all score -inf have no softmax
__device__ __forceinline__ float kv8_output(float mean, float sum, int units) {
  return units == 0 ? 0.f : sum == 0.f ? __builtin_nanf("") : mean;
}
// keys of a row: none where its slot is none of the table's
__device__ __forceinline__ int kv8_len(int pos, int slot, const Kv8Pages& pg, int cap) {
  return (unsigned)slot < (unsigned)pg.slots ? min(max(pos, -1), cap - 1) + 1 : 0;
}
__device__ __forceinline__ int kv8_units(int len) { return (len + kUnit - 1) / kUnit; }
// Units that a row is dealt as: its own and `pad` for what a workgroup spends on a row beside its keys (48 KB of them), none where no
// workgroup has parts of two rows (B up to 64: a lane has a row's units), so that shares that are whole turns of the waves stay
// so.  Us with 6 always, with 6 / 12 / 24 / 48 where rows meet: 1 sequence (8 heads of 128) of 4,096 keys 9.6, 8.8 all; 2 of 4,096 11.7,
// 10.0; 8 of 16,384 48.5, 47.9;  4 of 20000 .. 30000 37.5, 38.3 / 37.8 / 38.4 / 38.0;  8 (heads of 64) of 4000 .. 8192 16.5, 17.3 / 17.1 / 16.9
// / 16.6;  32 of 2 heads of 32 of 4096 .. 8192 13.5, 13.9 / 13.8 / 13.4 / 12.8.
constexpr int kLeast = 8;
constexpr int kv8_pads(int D) { return 48 * 32 / D; }
__device__ __forceinline__ int kv8_dealt(int units, int pad) { return units ? units + pad : 0; }
__device__ __forceinline__ int kv8_share(int total, int W) { return max((total + W - 1) / W, kLeast); }
template <int D>
__device__ __forceinline__ int kv8_pad(int units, int B, int W) {
  return B > 64 || (B > 1 && __ballot(units % kv8_share(wave_sum(units), W))) ? kv8_pads(D) : 0;
}

// Where workgroup x of W leaves what it has of a row that was cut: it has at most one that began before its share (part > 0) and one
// that goes on behind it (part 0), so 2 W places a query head hold the parts of any batch.  By row, parts would take B times what
// one row can be cut into (1,024 rows of up to 32,768 keys of one head of 128, 16 query heads: 2.2 GB for 4 MB).
__device__ __forceinline__ int64_t kv8_place(int head, int x, int part, int W) { return ((int64_t)head * 2 + (part ? 0 : 1)) * W + x; }

// EVEN: grid (W, Hkv), shares of all rows' units; else (Hkv, B), a workgroup a row.
template <int D, int WAVES, bool EVEN>
__global__ void __launch_bounds__(64 * WAVES, 2)
    kv8_attn_kernel(const int32_t* __restrict__ pos, const int32_t* __restrict__ slots, const int32_t* __restrict__ table,
                    const uint16_t* __restrict__ q, uint8_t* __restrict__ keys, uint8_t* __restrict__ values,
                    uint8_t* __restrict__ key_exps, uint8_t* __restrict__ value_exps, int nslots, int maxp, int block,
                    int pages, int Hkv, float* __restrict__ part_ml, float* __restrict__ part_o,
                    uint16_t* __restrict__ out, int B, int Hq, int cap, float sl) {
  const Kv8Pages pg{keys, values, key_exps, value_exps, table, nslots, maxp, block, pages, Hkv};
  typedef Kv8State<D> State;
  constexpr int E = State::E, KS = State::KS, ROW = D + 8;  // (rows of whole pieces of 32 bytes)
  typedef float orow_t __attribute__((ext_vector_type(E)));
  // of a wave: two tiles on their way, then its outputs
  constexpr int PART = 128 * D > 64 * ROW ? 128 * D : 64 * ROW;
  __shared__ __attribute__((aligned(32))) char smem[WAVES * PART];
  __shared__ float mls[WAVES][2][16];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, g = lane >> 4, rep = Hq / pg.Hkv;
  const int hk = EVEN ? blockIdx.y : blockIdx.x;
  int b = EVEN ? 0 : blockIdx.y, start = 0, from_unit = 0, end = 0, share = 1;
  int i0 = 0, lens = 0, at_slot = 0, pad = 0;  // EVEN: lane i has row i0 + i
  const auto window = [&](int from) {
    i0 = from;
    at_slot = from + lane < B ? (slots ? slots[from + lane] : from + lane) : -1;
    lens = from + lane < B ? kv8_len(pos[from + lane], at_slot, pg, cap) : 0;
    return kv8_dealt(kv8_units(lens), pad);
  };
  if constexpr (EVEN) {
    int total = 0, mine = window(0);
    pad = __builtin_amdgcn_readfirstlane(kv8_pad<D>(mine, B, gridDim.x));
    for (int f = 64 * ((B - 1) / 64); f > 0; f -= 64) total += window(f);
    total += mine = B > 64 ? window(0) : kv8_dealt(mine, pad);  // (the first rows stay)
    total = __builtin_amdgcn_readfirstlane(wave_sum(total));
    share = kv8_share(total, gridDim.x);
    from_unit = blockIdx.x * share;
    end = min(total, from_unit + share);
    if (from_unit >= end) return;
    while (true) {  // the row that holds unit `from_unit`: start <= it < start + its units
      const int upto = (int)wave_scan((uint32_t)mine);
      const uint64_t past = __ballot(start + upto > from_unit);
      if (past) {
        const int first = __ffsll((unsigned long long)past) - 1;
        b = __builtin_amdgcn_readfirstlane(i0 + first);
        start = __builtin_amdgcn_readlane(start + upto - mine, first);
        break;
      }
      start = __builtin_amdgcn_readlane(start + upto, 63);
      mine = window(i0 + 64);
    }
  }
  while (true) {
    int len, slot, u0 = 0, u1, from = 0, n;
    if constexpr (EVEN) {
      if (b - i0 >= 64) window(i0 + 64);
      len = __builtin_amdgcn_readlane(lens, b - i0);
      slot = __builtin_amdgcn_readlane(at_slot, b - i0);
      n = kv8_units(len);
      if (n == 0) {  // (units are left, so a later row has them)
        ++b;
        continue;
      }
      from = start + pad;  // of its keys
      u0 = max(from_unit - from, 0), u1 = min(end - from, n);
      if (u1 <= 0) return;  // its keys begin in the next share
    } else {
      slot = slots ? slots[b] : b;
      len = kv8_len(pos[b], slot, pg, cap);
      n = u1 = kv8_units(len);
    }
    u16x8 qf[KS];
    const uint16_t* qrow = q + ((int64_t)b * Hq + hk * rep + min(c, rep - 1)) * D;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      qf[s] = *reinterpret_cast<const u16x8*>(qrow + chan<D>(s, g));
      if (c >= rep) qf[s] = u16x8{0, 0, 0, 0, 0, 0, 0, 0};
    }
    State st;
    st.clear();
    char* const kl = smem + w * PART;
    const typename State::Places at(kl, c, g);
    // tiles of two units, dealt to the waves in turn (side by side: 8 x WAVES KB in a row of keys, and of values); a lane finds one
    // of the wave's next 64 units: where it lies, and its powers of two (NaN where it lies nowhere)
    for (int t0 = u0 + 2 * w; t0 < u1; t0 += 64 * WAVES) {
      const int mine = t0 + 2 * WAVES * (lane >> 1) + (lane & 1);
      const int64_t unit = kv8_unit(pg, slot, min(mine, u1 - 1), hk);
      const int where = (int)max(unit, (int64_t)0);
      const int ke = pg.ke[where];
      float ks = unit < 0 ? __builtin_nanf("") : sl * __uint_as_float((uint32_t)ke << 23);
      int ve = pg.ve[where];
      const int tiles = min(32, (u1 - t0 + 2 * WAVES - 1) / (2 * WAVES));  // of this wave, here
      const int whole = min(u1, len / kUnit);                                // units before this one have all their rows
      const auto fetch = [&](int i, int half) {
        const int64_t a0 = (int64_t)__builtin_amdgcn_readlane(where, 2 * i) * (kUnit * D);
        const int64_t a1 = (int64_t)__builtin_amdgcn_readlane(where, 2 * i + 1) * (kUnit * D);
        const int u = t0 + 2 * WAVES * i, lim = len - 1 - kUnit * u, lim1 = u + 1 < u1 ? lim - kUnit : -1;
        char* to = kl + half * (64 * D);
        if (u + 2 <= whole) State::template load_tile<true>(to, pg.k + a0, pg.k + a1, pg.v + a0, pg.v + a1, 15, 15, lane);
        else State::template load_tile<false>(to, pg.k + a0, pg.k + a1, pg.v + a0, pg.v + a1, lim, lim1, lane);
      };
      const auto of = [](float x, int l) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), l)); };
      constexpr int LOADS = D / 16;  // of a tile
      fetch(0, 0);
      // (behind the first fetch, which waits neither for queries nor for exponents)
      if (t0 == u0 + 2 * w) st.big = shrink_queries<KS>(qf, st.qe);
      if (st.big && unit >= 0) ks = (float)(ke - 127);
      if (!st.far && __ballot(ve >= kFar)) {
        st.far = true;
#pragma unroll
        for (int e = 0; e < E; ++e) st.o[e] *= 0x1p-32f;
      }
      if (st.far) ve = max(ve - kFarBy, 1);
      const float vs = __uint_as_float((uint32_t)ve << 23);
      for (int i = 0; i < tiles; ++i) {
        if (i + 1 < tiles) {
          fetch(i + 1, (i + 1) & 1);
          __builtin_amdgcn_s_waitcnt(0x0F70 | LOADS);  // the older tile has landed (only this wave reads it)
        } else {
          __builtin_amdgcn_s_waitcnt(0x0F70);
        }
        const int u = t0 + 2 * WAVES * i, lim = len - 1 - kUnit * u, lim1 = u + 1 < u1 ? lim - kUnit : -1;
        st.take(at, (i & 1) * (64 * D), qf, of(ks, 2 * i), of(ks, 2 * i + 1), of(vs, 2 * i), of(vs, 2 * i + 1), sl,
                u + 2 <= whole, lim, lim1, c, g);
      }
    }
    st.l = lane_sum<32>(lane_sum<16>(st.l));
    const float inv = st.l == 0.f ? 1.f : __builtin_amdgcn_rcpf(st.l), up = st.far ? 0x1p32f : 1.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      orow_t y;
#pragma unroll
      for (int e = 0; e < E; ++e) y[e] = st.o[e][i] * inv * up;
      *reinterpret_cast<orow_t*>(reinterpret_cast<float*>(smem + w * PART) + c * ROW + E * (4 * g + i)) = y;
    }
    if (g == 0) mls[w][0][c] = st.m, mls[w][1][c] = st.l;
    __syncthreads();
    const int part = EVEN ? (int)blockIdx.x - from / share : 0, last = EVEN ? (from + n - 1) / share - from / share : 0;
    for (int idx = tid; idx < rep * D; idx += 64 * WAVES) {
      const int h = idx / D, d = idx % D;
      float M = -INFINITY, L = 0.f, acc = 0.f, f[WAVES];
#pragma unroll
      for (int x = 0; x < WAVES; ++x) M = fmaxf(M, mls[x][0][h]);
#pragma unroll
      for (int x = 0; x < WAVES; ++x) {  // (a wave whose scores are NaN has no maximum, and its sum carries them)
        const float mw = mls[x][0][h];
        f[x] = (mw == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mw - M)) * mls[x][1][h];
        L += f[x];
      }
      const float all = L == 0.f ? 0.f : __builtin_amdgcn_rcpf(L);
#pragma unroll
      for (int x = 0; x < WAVES; ++x) acc += f[x] * all * reinterpret_cast<const float*>(smem + x * PART)[h * ROW + d];
      const int64_t bh = (int64_t)b * Hq + hk * rep + h;
      if (last == 0) {  // the row's only part is its output
        out[bh * D + d] = f2bf(kv8_output(acc, L, n));
      } else {
        const int64_t at = kv8_place(hk * rep + h, blockIdx.x, part, gridDim.x);
        part_o[at * D + d] = acc;
        if (d == 0) part_ml[at * 2] = M, part_ml[at * 2 + 1] = L;
      }
    }
    if constexpr (!EVEN) return;
    from_unit = start = from + n;
    if (from_unit >= end) return;
    ++b;
    __syncthreads();  // the sums are read
  }
}

// The parts of rows that were cut, and the zeros of rows without keys; W: workgroups of a KV head.  A workgroup has C channels of a
// row, and G groups of its threads share the parts; a lane has the maximum and the sum of one of 64 parts.  Where the parts
// lie follows from the lengths; what comes from memory after them comes at once.
template <int D, int C, int G>
__global__ void __launch_bounds__(C* G)
    kv8_merge_kernel(const float* __restrict__ part_ml, const float* __restrict__ part_o, Kv8Pages pg,
                     const int32_t* __restrict__ pos, const int32_t* __restrict__ slots, uint16_t* __restrict__ out, int B,
                     int Hq, int W, int cap) {
  constexpr int AHEAD = G >= 8 ? 2 : G >= 4 ? 3 : 4;
  __shared__ float sums[G][C];
  const int64_t bh = blockIdx.x / (D / C);
  const int b = (int)(bh / Hq), head = (int)(bh % Hq), lane = threadIdx.x & 63, grp = threadIdx.x / C;
  const int d = C * (blockIdx.x % (D / C)) + threadIdx.x % C;
  const auto units = [&](int i) { return kv8_units(kv8_len(pos[i], slots ? slots[i] : i, pg, cap)); };
  const int n = units(b), mine = lane < B ? units(lane) : 0, pad = kv8_pad<D>(mine, B, W);
  int total = kv8_dealt(mine, pad), start = lane < b ? total : 0;
  for (int i = lane + 64; i < B; i += 64) {
    const int u = kv8_dealt(units(i), pad);
    total += u;
    if (i < b) start += u;
  }
  total = wave_sum(total), start = wave_sum(start);
  const int share = kv8_share(total, W), from = start + pad, x0 = from / share;
  const int parts = n > 0 ? (from + n - 1) / share - x0 + 1 : 0;
  if (parts == 1) return;  // written by its workgroup
  const auto ml = [&](int p) { return reinterpret_cast<const float2*>(part_ml)[kv8_place(head, x0 + p, p, W)]; };
  const auto po = [&](int p) { return part_o[kv8_place(head, x0 + p, p, W) * D + d]; };
  float2 first = {0.f, 0.f};
  float ahead[AHEAD] = {};
  if (parts) {
    first = ml(min(lane, parts - 1));
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) ahead[i] = po(min(grp + i * G, parts - 1));
  }
  float M = -INFINITY, L = 0.f, acc = 0.f;
  for (int p0 = 0; p0 < parts; p0 += 64) {
    const bool on = p0 + lane < parts;
    const float2 x = p0 ? ml(min(p0 + lane, parts - 1)) : first;
    const float m = on ? x.x : -INFINITY, top = fmaxf(M, wave_max(m));
    const float was = M == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(M - top), f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);
    const float kept = L * was, fl = on ? f * x.y : 0.f;
    L = kept + wave_sum(fl);
    const float inv = L == 0.f ? 0.f : __builtin_amdgcn_rcpf(L), share_of = fl * inv;
    acc *= kept * inv;
    M = top;
    const int end = min(64, parts - p0);
    const auto weight = [&](int s) { return __shfl(share_of, s); };  // (of this wave's groups)
    int i = 0;
    if (p0 == 0) {
#pragma unroll
      for (; i < AHEAD; ++i) {
        const int s = grp + i * G;
        const float wgt = weight(min(s, 63));
        if (s < end) acc += wgt * ahead[i];
      }
    }
#pragma unroll 8
    for (; i * G < end; ++i) {  // (every lane takes the same turns)
      const int s = grp + i * G;
      const float wgt = weight(min(s, 63)), y = po(p0 + min(s, end - 1));
      if (s < end) acc += wgt * y;
    }
  }
  if constexpr (G > 1) {
    sums[grp][threadIdx.x % C] = acc;
    __syncthreads();
    if (threadIdx.x >= C) return;
    acc = 0.f;
#pragma unroll
    for (int i = 0; i < G; ++i) acc += sums[i][threadIdx.x];
  }
  out[bh * D + d] = f2bf(kv8_output(acc, L, n));
}

}  // namespace mx

using namespace mx;

// Waves of a workgroup that takes a whole row, 0: rows are cut.  A row takes a workgroup 4.5 us for 256 KB of heads of 128 (a CU's
// 60 GB/s, however many waves); cutting costs a merge and more ends, 2 to 11 us.  The bounds are in keys whatever D is: a workgroup's
// time goes by its tiles of 32 as much as by their bytes (2,048 keys 14.5 us of 128, 10.7 of 64).  Rows that leave no CU alone are
// better off by four waves or within 3 % of it, where a CU has the next row's workgroup beside this one's end.  Us, cold, of a call
// in a graph (1.5 of it between launches), with whole rows of 4 / 8 waves, and cut:
//   heads of 128: 8 rows of 700 keys 8.9 / 8.7, 9.8; of 1,024 10.4 / 9.7, 10.1; of 2,048 15.8 / 14.5, 10.3;  32 of 1,500 13.2 / 12.4, 12.1;
//     64 of 1000 .. 2000 14.8 / 13.9, 16.0; of 16,384 96.1 / 87.3, 50.4;  128 of 1000 .. 2000 15.7 / 15.3, 21.3; of 2000 .. 4096 25.9 / 25.4,
//     27.8;  192 of 100 .. 4096 27.7 / 27.7, 29.2;  256 of 100 .. 2000 17.6 / 17.7, 22.3; of 100 .. 4096 31.2 / 31.6, 34.3;  512 of 30 .. 512
//     11.8 / 14.5, 21.5; of 2048 .. 4096 70.1 / 69.8, 71.6
//   of 64: 8 of 700 7.7 / 6.9, 9.2; of 2,048 13.0 / 10.7, 9.3;  64 of 1000 .. 3000 16.3 / 13.0, 13.3 (cut, its bound being 2,048);  128 of 500 ..
//     2000 12.8 / 10.7, 15.5; of 1000 .. 6000 31.0 / 22.7, 20.2;  192 of 100 .. 4000 21.6 / 17.1, 20.3;  320 of 1000 .. 8000 48.6 / 49.1, 39.0;
//     384 of 100 .. 2000 16.0 / 16.0, 21.5;  512 of 2048 .. 4096 38.0 / 38.9, 42.1
//   of 32: 64 of 4096 .. 8192 33.9 / 22.8, 14.4;  512 of 1000 .. 8000 41.6 / 36.9, 39.4 (cut);  1,024 of 30 .. 512 8.9 / 9.4, 22.2
// Rows of few keys beside a long one are what whole rows are worst at: the bounds keep that within some 12 us.
static int kv8_waves(int64_t rows, int64_t cap, int D) {
  if (cap > (rows >= 128 ? 4096 : rows >= 32 ? 32 * rows : 1024)) return 0;
  return rows >= (D == 128 ? 128 : D == 64 ? 384 : 1024) ? 4 : 8;
}
// Workgroups of a KV head where keys are dealt evenly: one a CU of 256, of four waves with heads of 128, of eight with smaller ones.
// Us with 512 of four waves, 256 of eight, 256 of four: 8 rows (a sequence of 8 heads) of 128 of 4,096 keys 9.8, 8.9, 8.9, of 32,768 19.0,
// 17.7, 17.4; 64 of 16,384 48.0, 48.7, 47.9; 512 of 500 .. 8192 97.9, 99.2, 95.2;  8 of 64 of 16,384 11.4, 10.3, 10.3; 64 of 4000 .. 8192 15.6,
// 16.5, 16.4;  64 of 32 of 4096 .. 8192 12.7, 12.7, 14.3.  (768 of four waves 23.8 and 54.5 where 512 have 19.0 and 48.0.)
static int kv8_shares(int Hkv) { return Hkv < 256 ? (256 + Hkv - 1) / Hkv : 1; }

// places for parts that a query head has (of part_ml [Hq, places, 2], part_o [Hq, places, D]); 0: rows are whole
extern "C" int mx_kv8_attn_parts(int B, int Hkv, int D, int cap) {
  return kv8_waves((int64_t)B * Hkv, cap, D) ? 0 : 2 * kv8_shares(Hkv);
}

namespace {

struct Launch {
  const uint16_t* q;
  Kv8Pages pg;
  const int32_t *pos, *slots;
  float *part_ml, *part_o;
  uint16_t* out;
  int B, Hq, cap;
  float sl;
  hipStream_t stream;
};

template <int D, int WAVES>
void launch_whole(const Launch& a) {
  kv8_attn_kernel<D, WAVES, false><<<dim3(a.pg.Hkv, a.B), 64 * WAVES, 0, a.stream>>>(
      a.pos, a.slots, a.pg.table, a.q, a.pg.k, a.pg.v, a.pg.ke, a.pg.ve, a.pg.slots, a.pg.maxp, a.pg.block, a.pg.pages,
      a.pg.Hkv, nullptr, nullptr, a.out, a.B, a.Hq, a.cap, a.sl);
}

template <int D>
void launch(const Launch& a) {
  const int Hkv = a.pg.Hkv, W = kv8_shares(Hkv), waves = kv8_waves((int64_t)a.B * Hkv, a.cap, D);
  if (waves) {
    if (waves == 4) launch_whole<D, 4>(a);
    else launch_whole<D, 8>(a);
    return;
  }
  constexpr int WAVES = D == 128 ? 4 : 8;
  kv8_attn_kernel<D, WAVES, true><<<dim3(W, Hkv), 64 * WAVES, 0, a.stream>>>(
      a.pos, a.slots, a.pg.table, a.q, a.pg.k, a.pg.v, a.pg.ke, a.pg.ve, a.pg.slots, a.pg.maxp, a.pg.block, a.pg.pages, Hkv,
      a.part_ml, a.part_o, a.out, a.B, a.Hq, a.cap, a.sl);
  const int rows = a.B * a.Hq;
  if (rows <= 512)  // few rows are waited for part by part: 1 x 4096 keys 15.2 -> 8.8 us, 1 x 32768 23.8 -> 17.5 (8 x 16384, of four parts a
                    // row, 47.1 -> 48.1; 64 x 500 .. 8192, 4,096 rows, would be 95 -> 107)
    kv8_merge_kernel<D, 32, 8><<<rows * (D / 32), 256, 0, a.stream>>>(a.part_ml, a.part_o, a.pg, a.pos, a.slots, a.out, a.B,
                                                                      a.Hq, W, a.cap);
  else
    kv8_merge_kernel<D, D, D < 128 ? 128 / D : 1><<<rows, 128, 0, a.stream>>>(a.part_ml, a.part_o, a.pg, a.pos, a.slots,
                                                                              a.out, a.B, a.Hq, W, a.cap);
}

}  // namespace

// q [B, Hq, D]; keys 0 .. pos[b], below cap, of slot slots[b] (null: b); out [B, Hq, D]
extern "C" int mx_kv8_attn(const uint16_t* q, const Kv8Pages* cache, const int32_t* pos, const int32_t* slots,
                           float* part_ml, float* part_o, uint16_t* out, int B, int Hq, int D, int cap, float scale,
                           hipStream_t stream) {
  if (B <= 0) return 0;
  const Kv8Pages pg = *cache;
  if (pg.Hkv <= 0 || Hq % pg.Hkv || Hq / pg.Hkv > 16 || B > 65535 || pg.Hkv > 65535 || cap < 1 ||
      (int64_t)B * (cap / kUnit + 1 + kv8_pads(D)) > INT32_MAX || (int64_t)B * Hq * (D / 32) > INT32_MAX || !(scale > 0.f))
    return -1;
  const Launch a{q, pg, pos, slots, part_ml, part_o, out, B, Hq, cap, scale * 1.4426950408889634f, stream};
  if (D == 128) launch<128>(a);
  else if (D == 64) launch<64>(a);
  else if (D == 32) launch<32>(a);
  else return -1;
  return (int)hipGetLastError();
}
