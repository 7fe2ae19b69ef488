// Attention of one token of each sequence over a paged cache of 8 bits (kv8.h):
//   o = softmax(q k^T scale) v over positions 0 .. pos, queries of a group of heads sharing a key/value head.
//
// Bound by memory: a key and a value of a head are 2 D bytes and half of a bf16 cache's, each read once for all query heads of
// the group.  Codes become bf16 in registers, where they are exact; the powers of two of a unit (16 positions) go
// into its scores and its weights, so they cost a product a score and a weight:
//   S^T[key][head] = 2^(ek - 127) scale log2(e) (K . Q^T),  O^T[d][head] += V^T . (2^(ev - 127) P)
// by v_mfma_f32_16x16x32_bf16.  Maxima, sums and outputs are f32; a weight is rounded once to bf16 (2^-9 of it, in a sum of
// many) where the product takes it, while the sum under it takes what was not rounded.
//
// The operands: a lane (c, g) of K has row c of a unit and the channels 64 (s / 2) + 16 g + 8 (s % 2) .. of step s (a dot
// product does not mind the order, so a lane takes whole pieces of 16 bytes; Q is laid out alike), of V eight rows and D / 16
// neighbouring channels, whose bytes are put together row by row as the product reads them.  No tile goes through LDS.
//
// Keys are dealt evenly: the units of all sequences in a row are cut into equal shares, one a workgroup of a KV head, whose four
// waves share what it has of a sequence; sequences that were cut are merged by a second launch.
#include "kv8.h"

namespace mx {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f32x4 mfma16(const u16x8& a, const u16x8& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0,
                                                 0, 0);
}
__device__ __forceinline__ uint32_t pair_bf16(uint32_t w, bool high) {
  return high ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, true))
              : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, false));
}
// channel of k-step s of lane group g
template <int D>
__device__ __forceinline__ int chan(int s, int g) {
  return D == 32 ? 8 * g : 64 * (s >> 1) + 16 * g + 8 * (s & 1);
}

template <int E>
struct VPiece {
  typedef uint32_t type;
};
template <>
struct VPiece<8> {
  typedef uint2 type;
};
template <>
struct VPiece<2> {
  typedef uint16_t type;
};
__device__ __forceinline__ uint32_t word(uint2 v, int i) { return i ? v.y : v.x; }
__device__ __forceinline__ uint32_t word(uint32_t v, int) { return v; }
__device__ __forceinline__ uint32_t word(uint16_t v, int) { return v; }

template <int D>
struct Kv8State {  // of one wave
  static constexpr int E = D / 16, KS = D / 32;
  float m, l;   // of head c; l: this lane's keys
  f32x4 o[E];   // [e][i]: channel E (4 g + i) + e of head c

  __device__ __forceinline__ void clear() {
    m = -INFINITY, l = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  // two units; k0, v0 / k1, v1: their rows, ks / vs: what their scores / weights are multiplied by, lim: their last row that is
  // there (-1: none; rows behind it are read as that row, and count nothing)
  __device__ __forceinline__ void take(const uint8_t* __restrict__ k0, const uint8_t* __restrict__ k1,
                                       const uint8_t* __restrict__ v0, const uint8_t* __restrict__ v1, float ks0, float ks1,
                                       float vs0, float vs1, int lim0, int lim1, const u16x8 (&qf)[KS], int c, int g) {
    uint32_t k[2][2 * KS];  // words of the lane's channels, in the order of the k-steps
    typename VPiece<E>::type v[8];  // slot s: row 4 g + (s & 3) of unit s >> 2, channels E c ..
    const int z0 = max(lim0, 0), z1 = max(lim1, 0);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint8_t* p = (j ? k1 : k0) + (uint32_t)(min(c, j ? z1 : z0) * D);
      if constexpr (D == 32) {
        const uint2 w = *reinterpret_cast<const uint2*>(p + 8 * g);
        k[j][0] = w.x, k[j][1] = w.y;
      } else {
#pragma unroll
        for (int h = 0; h < D / 64; ++h) {
          const uint4 w = *reinterpret_cast<const uint4*>(p + 64 * h + 16 * g);
          k[j][4 * h] = w.x, k[j][4 * h + 1] = w.y, k[j][4 * h + 2] = w.z, k[j][4 * h + 3] = w.w;
        }
      }
    }
#pragma unroll
    for (int s = 0; s < 8; ++s)
      v[s] = *reinterpret_cast<const typename VPiece<E>::type*>((s < 4 ? v0 : v1) +
                                                                (uint32_t)(min(4 * g + (s & 3), s < 4 ? z0 : z1) * D + E * c));
    __builtin_amdgcn_sched_barrier(0);  // every load is in flight before the first product waits
    f32x4 sc[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      sc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < KS; ++s) sc[j] = mfma16(dequant8(k[j][2 * s], k[j][2 * s + 1]), qf[s], sc[j]);
    }
    float mx = m;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = 4 * g + i <= (j ? lim1 : lim0) ? sc[j][i] * (j ? ks1 : ks0) : -INFINITY;
        sc[j][i] = x;
        mx = fmaxf(mx, x);
      }
    mx = lane_max<32>(lane_max<16>(mx));
    const float mref = mx == -INFINITY ? 0.f : mx, f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mref);
    m = mx;
    l *= f;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] *= f;
    u16x8 pb;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float p = __builtin_amdgcn_exp2f(sc[j][i] - mref);
        l += p;
        pb[4 * j + i] = f2bf(p * (j ? vs1 : vs0));
      }
    // bytes 0, 1 (lo) or 2, 3 (hi) of the words of two rows side by side, as pairs of rows of one channel each
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
      u32x4 a0, a1;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t w = __builtin_amdgcn_perm(word(v[2 * i + 1], e >> 2), word(v[2 * i], e >> 2),
                                                 e & 2 ? 0x07030602u : 0x05010400u);
        a0[i] = pair_bf16(w, false), a1[i] = pair_bf16(w, true);
      }
      o[e] = mfma16(__builtin_bit_cast(u16x8, a0), pb, o[e]);
      o[e + 1] = mfma16(__builtin_bit_cast(u16x8, a1), pb, o[e + 1]);
    }
  }
};

// keys of row b: none where its slot is none of the table's
__device__ __forceinline__ int kv8_len(const int32_t* pos, const int32_t* slots, const Kv8Pages& pg, int cap, int b) {
  const int slot = slots ? slots[b] : b;
  return (unsigned)slot < (unsigned)pg.slots ? min(max(pos[b], -1), cap - 1) + 1 : 0;
}
// units that row b is dealt as: its own and kPad for what a workgroup spends on a row beside its keys
constexpr int kPad = 6, kLeast = 8;
__device__ __forceinline__ int kv8_dealt(const int32_t* pos, const int32_t* slots, const Kv8Pages& pg, int cap, int b) {
  const int n = (kv8_len(pos, slots, pg, cap, b) + kUnit - 1) / kUnit;
  return n ? n + kPad : 0;
}
__device__ __forceinline__ int kv8_share(int total, int W) { return max((total + W - 1) / W, kLeast); }

// EVEN: grid (W, Hkv), shares of all rows' units; else (Hkv, B), a workgroup a row.
template <int D, int WAVES, bool EVEN>
__global__ void __launch_bounds__(64 * WAVES)
    kv8_attn_kernel(const uint16_t* __restrict__ q, Kv8Pages pg, const int32_t* __restrict__ pos,
                    const int32_t* __restrict__ slots, float* __restrict__ part_ml, float* __restrict__ part_o,
                    uint16_t* __restrict__ out, int B, int Hq, int cap, int nparts, float sl) {
  typedef Kv8State<D> State;
  constexpr int E = State::E, KS = State::KS, ROW = D + 8;  // (rows of whole pieces of 32 bytes)
  typedef float orow_t __attribute__((ext_vector_type(E)));
  __shared__ __attribute__((aligned(32))) float so[WAVES * 16 * ROW];
  __shared__ float mls[WAVES][2][16];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, g = lane >> 4, rep = Hq / pg.Hkv;
  const int hk = EVEN ? blockIdx.y : blockIdx.x;
  int b = EVEN ? 0 : blockIdx.y, start = 0, at = 0, end = 0, share = 1;
  if constexpr (EVEN) {
    int total = 0;
    for (int i = lane; i < B; i += 64) total += kv8_dealt(pos, slots, pg, cap, i);
    total = __builtin_amdgcn_readfirstlane(wave_sum(total));
    share = kv8_share(total, gridDim.x);
    at = blockIdx.x * share;
    end = min(total, at + share);
    if (at >= end) return;
    for (int i0 = 0;; i0 += 64) {  // the row that holds unit `at`: start <= at < start + its units
      const int n = i0 + lane < B ? kv8_dealt(pos, slots, pg, cap, i0 + lane) : 0;
      const int upto = (int)wave_scan((uint32_t)n);
      const uint64_t past = __ballot(start + upto > at);
      if (past) {
        const int first = __ffsll((unsigned long long)past) - 1;
        b = __builtin_amdgcn_readfirstlane(i0 + first);
        start = __builtin_amdgcn_readlane(start + upto - n, first);
        break;
      }
      start = __builtin_amdgcn_readlane(start + upto, 63);
    }
  }
  while (true) {
    const int len = kv8_len(pos, slots, pg, cap, b), n = (len + kUnit - 1) / kUnit;
    int u0 = 0, u1 = n, from = 0;
    if constexpr (EVEN) {
      if (n == 0) {  // (units are left, so a later row has them)
        ++b;
        continue;
      }
      from = start + kPad;  // of its keys
      u0 = max(at - from, 0), u1 = min(end - from, n);
      if (u1 <= 0) return;  // its keys begin in the next share
    }
    const int per = (u1 - u0 + WAVES - 1) / WAVES;
    const int ua = u0 + per * w, ub = min(u1, ua + per);
    const int slot = slots ? slots[b] : b;
    u16x8 qf[KS];
    const uint16_t* qrow = q + ((int64_t)b * Hq + hk * rep + min(c, rep - 1)) * D;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      qf[s] = *reinterpret_cast<const u16x8*>(qrow + chan<D>(s, g));
      if (c >= rep) qf[s] = u16x8{0, 0, 0, 0, 0, 0, 0, 0};
    }
    State st;
    st.clear();
    for (int v0 = ua; v0 < ub; v0 += 64) {
      // a lane finds one unit: where it lies, and its powers of two (NaN where it lies nowhere)
      const int m = min(64, ub - v0);
      const int64_t unit = kv8_unit(pg, slot, v0 + min(lane, m - 1), hk);
      const int where = (int)max(unit, (int64_t)0);
      const float ks = unit < 0 ? __builtin_nanf("") : sl * __uint_as_float((uint32_t)pg.ke[where] << 23);
      const float vs = __uint_as_float((uint32_t)pg.ve[where] << 23);
      for (int j = 0; j < m; j += 2) {
        const int j1 = min(j + 1, m - 1);
        const int64_t a0 = (int64_t)__builtin_amdgcn_readlane(where, j) * (kUnit * D);
        const int64_t a1 = (int64_t)__builtin_amdgcn_readlane(where, j1) * (kUnit * D);
        const auto of = [](float x, int l) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), l)); };
        const int lim = len - 1 - kUnit * (v0 + j);
        st.take(pg.k + a0, pg.k + a1, pg.v + a0, pg.v + a1, of(ks, j), of(ks, j1), of(vs, j), of(vs, j1), lim,
                j1 > j ? lim - kUnit : -1, qf, c, g);
      }
    }
    st.l = lane_sum<32>(lane_sum<16>(st.l));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      orow_t y;
#pragma unroll
      for (int e = 0; e < E; ++e) y[e] = st.o[e][i];
      *reinterpret_cast<orow_t*>(so + (w * 16 + c) * ROW + E * (4 * g + i)) = y;
    }
    if (g == 0) mls[w][0][c] = st.m, mls[w][1][c] = st.l;
    __syncthreads();
    const int part = EVEN ? (int)blockIdx.x - from / share : 0, last = EVEN ? (from + n - 1) / share - from / share : 0;
    for (int idx = tid; idx < rep * D; idx += 64 * WAVES) {
      const int h = idx / D, d = idx % D;
      float M = -INFINITY, L = 0.f, acc = 0.f;
#pragma unroll
      for (int x = 0; x < WAVES; ++x) M = fmaxf(M, mls[x][0][h]);
#pragma unroll
      for (int x = 0; x < WAVES; ++x) {  // (a wave whose scores are NaN has no maximum, and its sum carries them)
        const float mw = mls[x][0][h], f = mw == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mw - M);
        L += f * mls[x][1][h];
        acc += f * so[(x * 16 + h) * ROW + d];
      }
      const int64_t bh = (int64_t)b * Hq + hk * rep + h;
      if (last == 0) {  // the row's only part is its output
        out[bh * D + d] = f2bf(L == 0.f ? 0.f : acc / L);
      } else {
        part_o[(bh * nparts + part) * D + d] = acc;
        if (d == 0) part_ml[(bh * nparts + part) * 2] = M, part_ml[(bh * nparts + part) * 2 + 1] = L;
      }
    }
    if constexpr (!EVEN) return;
    at = start = from + n;
    if (at >= end) return;
    ++b;
    __syncthreads();  // the sums are read
  }
}

// the parts of rows that were cut, and the zeros of rows without keys; W: workgroups of a KV head
template <int D>
__global__ void __launch_bounds__(D < 64 ? 64 : D)
    kv8_merge_kernel(const float* __restrict__ part_ml, const float* __restrict__ part_o, Kv8Pages pg,
                     const int32_t* __restrict__ pos, const int32_t* __restrict__ slots, uint16_t* __restrict__ out, int B,
                     int Hq, int W, int cap, int nparts) {
  const int64_t bh = blockIdx.x;
  const int b = (int)(bh / Hq), d = threadIdx.x, lane = d & 63;
  const float* ml = part_ml + bh * nparts * 2;
  const float* po = part_o + bh * nparts * D + min(d, D - 1);
  const int n = (kv8_len(pos, slots, pg, cap, b) + kUnit - 1) / kUnit;
  int total = 0, start = 0;
  for (int i = lane; i < B; i += 64) {
    const int u = kv8_dealt(pos, slots, pg, cap, i);
    total += u;
    if (i < b) start += u;
  }
  total = wave_sum(total), start = wave_sum(start);
  const int share = kv8_share(total, W), from = start + kPad;
  const int parts = n > 0 ? (from + n - 1) / share - from / share + 1 : 0;
  if (parts == 1) return;  // written by its workgroup
  float M = -INFINITY, L = 0.f, acc = 0.f;
  for (int s = 0; s < parts; ++s) M = fmaxf(M, ml[2 * s]);
  for (int s = 0; s < parts; ++s) {
    const float m = ml[2 * s], f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - M);
    L += f * ml[2 * s + 1];
    acc += f * po[(int64_t)s * D];
  }
  if (d < D) out[bh * D + d] = f2bf(L == 0.f ? 0.f : acc / L);
}

}  // namespace mx

using namespace mx;

// workgroups of a KV head where keys are dealt evenly: two a CU of 256
static int kv8_shares(int Hkv) { return Hkv < 512 ? (512 + Hkv - 1) / Hkv : 1; }
// whether a workgroup takes a whole row: up to 512 keys, where a launch to merge would cost more than it saves
static bool kv8_whole(int cap) { return cap <= 512; }

// parts that a row of up to `cap` keys can be cut into (of part_ml [B, Hq, parts, 2], part_o [B, Hq, parts, D])
extern "C" int mx_kv8_attn_parts(int Hkv, int cap) {
  if (kv8_whole(cap)) return 0;
  const int W = kv8_shares(Hkv), most = (cap / kUnit + 1) / kLeast + 2;
  return W < most ? W : most;
}

// q [B, Hq, D]; keys 0 .. pos[b], below cap, of slot slots[b] (null: b); out [B, Hq, D]
extern "C" int mx_kv8_attn(const uint16_t* q, const Kv8Pages* cache, const int32_t* pos, const int32_t* slots,
                           float* part_ml, float* part_o, uint16_t* out, int B, int Hq, int D, int cap, float scale,
                           hipStream_t stream) {
  if (B <= 0) return 0;
  const Kv8Pages pg = *cache;
  if (pg.Hkv <= 0 || Hq % pg.Hkv || Hq / pg.Hkv > 16 || B > 65535 || pg.Hkv > 65535 || cap < 1 ||
      (int64_t)B * (cap / kUnit + 1 + kPad) > INT32_MAX)
    return -1;
  const float sl = scale * 1.4426950408889634f;
  const int nparts = mx_kv8_attn_parts(pg.Hkv, cap), W = kv8_shares(pg.Hkv);
#define ATTN(DD)                                                                                                         \
  do {                                                                                                                   \
    if (kv8_whole(cap)) {                                                                                                \
      kv8_attn_kernel<DD, 8, false><<<dim3(pg.Hkv, B), 512, 0, stream>>>(q, pg, pos, slots, nullptr, nullptr, out, B,    \
                                                                         Hq, cap, 0, sl);                                \
    } else {                                                                                                             \
      kv8_attn_kernel<DD, 4, true><<<dim3(W, pg.Hkv), 256, 0, stream>>>(q, pg, pos, slots, part_ml, part_o, out, B, Hq,  \
                                                                        cap, nparts, sl);                                \
      kv8_merge_kernel<DD><<<B * Hq, DD < 64 ? 64 : DD, 0, stream>>>(part_ml, part_o, pg, pos, slots, out, B, Hq, W,     \
                                                                     cap, nparts);                                       \
    }                                                                                                                    \
  } while (0)
  if (D == 128) ATTN(128);
  else if (D == 64) ATTN(64);
  else if (D == 32) ATTN(32);
  else return -1;
#undef ATTN
  return (int)hipGetLastError();
}
