// 64-key steps of the 16-bit attention kernels (prompt.hip, shared.hip): keys and values
// row-major in LDS as 16-bit elements, products by v_mfma_f32_32x32x16 with a wave's 32 query
// rows as columns:
//   S^T[key, row] = K Q^T,   O^T[d, row] += V^T P^T.
// Lane (j = lane % 32, hh = lane / 32) holds column j. Register i of a 32-key S^T accumulator is
// key 8 (i / 4) + 4 hh + i % 4, so registers 8 u .. 8 u + 7 are the lane's share of a 16-key
// contraction of O^T: no exchange, as long as V^T's operand lists the keys in that order. It is
// read from the row-major values by the transposing LDS read (ds_read_b64_tr_b16): of 16
// lanes, lane a addresses four channels 4 (a % 4) of row a / 4, and lane i receives channel i of
// the four rows.
#pragma once

#include "args.h"

namespace ek {

typedef float f16v_t __attribute__((ext_vector_type(16)));
typedef __bf16 b8_t __attribute__((ext_vector_type(8)));
typedef short s4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u4_t __attribute__((ext_vector_type(4)));

// Fragments are kept as bits: h8_t whatever the type.
template <bool BF>
__device__ __forceinline__ f16v_t mma(const h8_t a, const h8_t b, const f16v_t c) {
  if constexpr (BF)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8_t, a), __builtin_bit_cast(b8_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// Two floats rounded to the 16-bit type, as bits.
template <bool BF>
__device__ __forceinline__ uint32_t pack2(float x, float y) {
  if constexpr (BF) {
    typedef __bf16 b2_t __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, b2_t{(__bf16)x, (__bf16)y});
  } else {
    return __builtin_bit_cast(uint32_t, h2_t{(_Float16)x, (_Float16)y});
  }
}

// LDS rows are unpadded; 16-byte slots are permuted by row. K: 32 rows are read at one slot of
// each. V: the transposing read takes four neighbouring rows at 32 bytes of each, next to
// another 16 lanes at the next 32 bytes.
template <int D>
__device__ __forceinline__ int k_swz(int key) {
  return D == 64 ? (key >> 1) & 7 : key & 15;
}
template <int D>
__device__ __forceinline__ int v_swz(int key) {
  return D == 64 ? 4 * ((key >> 1) & 1) : 4 * (key & 3);
}

// max / sum of x over the two half-waves (lanes l and l ^ 32).
__device__ __forceinline__ float halves_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float halves_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

__device__ __forceinline__ const uint8_t* uniform_ptr(const uint8_t* p) {
  const uint64_t u = (uint64_t)p;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)u);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(u >> 32));
  return (const uint8_t*)(((uint64_t)hi << 32) | lo);
}

// 16 bytes per lane from base + off to LDS [lds, lds + 1024) in lane order.
__device__ __forceinline__ void dma16(const uint8_t* base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\tglobal_load_lds_dwordx4 %0, %2" ::"v"(off), "s"(__builtin_amdgcn_readfirstlane(lds)),
               "s"(base)
               : "memory", "m0");
}

template <class T>
using lds_t = __attribute__((address_space(3))) T;

// K fragment (A operand of S^T): key rows 32 kb + j, channels 16 s + 8 hh .. + 8. k_at: the
// lane's byte offset in the step's keys, k_read: the fragment at an LDS address made of it.
template <int D>
__device__ __forceinline__ uint32_t k_at(int s, int j, int hh) {
  return (uint32_t)(j * (2 * D) + 16 * ((2 * s + hh) ^ k_swz<D>(j)));  // k_swz has period 32
}
template <int D>
__device__ __forceinline__ h8_t k_read(uint32_t at, int kb) {
  return *(const lds_t<h8_t>*)(at + kb * 64 * D);
}

// V^T fragment (A operand of O^T): channels 32 db + j, keys 16 ks + {4 hh .. + 3, 8 + 4 hh .. + 3}.
template <int D>
__device__ __forceinline__ uint32_t v_at(int db, int lane) {
  const int a = lane & 15, hh = lane >> 5, g = (lane >> 4) & 1;
  const int key = 4 * hh + (a >> 2), slot = 4 * db + 2 * g + ((a & 3) >> 1);  // v_swz has period 4
  return (uint32_t)(key * (2 * D) + 16 * (slot ^ v_swz<D>(key)) + 8 * (a & 1));
}
template <int D>
__device__ __forceinline__ h8_t v_read(uint32_t at, int ks) {
  s4_t x[2];
#pragma unroll
  for (int u = 0; u < 2; ++u)
    x[u] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t<s4_t>*)(at + (16 * ks + 8 * u) * 2 * D));
  return __builtin_bit_cast(h8_t, __builtin_shufflevector(x[0], x[1], 0, 1, 2, 3, 4, 5, 6, 7));
}

// One wave's 32 rows over steps of 32 NKB keys. The loop is skewed by a step so that matrix and
// vector instructions run side by side in one wave (apart, a wave's products wait for its
// exponentials and back, and two waves a SIMD did not fill the gaps): the exponentials of step i
// go between the score products of step i + 1, whose maxima go between the value products of
// step i. Scheduling fences hold that order.
//
// PARTS: keys as one matrix or as hi + lo, `SIDE` bytes apart. QLO: the queries as hi + lo too, PLO:
// the weights as float16 hi + lo, VLO: the values as hi + lo like the keys (the product of the two low
// parts, 2^-22 of theirs, is left out).
template <int D, bool BF, int NKB, int PARTS, bool QLO, bool PLO = false, bool VLO = false>
struct Rows {
  static constexpr int NS = D / 16, NDB = D / 32;
  static constexpr int NP = 8 * NKB;  // pairs of scores a lane
  static constexpr int NW = 2 * NKB;  // words of 16 keys' weights, their low parts behind them
  static constexpr int PW = PLO ? 2 * NW : NW;
  static constexpr float kShift = BF ? 0.f : 6.f;  // float16 weights are 2^6 times the softmax's: small ones keep their bits
  static constexpr float kInf = __builtin_inff();
  h8_t q[NS], ql[QLO ? NS : 1];
  f16v_t acc[NDB];
  float m, l;      // running maximum (log2 units), this lane's share of the sum
  float scale;     // softmax scale in log2 units, positive

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int db = 0; db < NDB; ++db) acc[db] = f16v_t{};
    m = -kInf;
    l = 0.f;
  }
  // Scores are scaled inside the exponent and their maximum is taken before, which needs the scale
  // positive: a negative one flips the query's sign (the caller's), a zero one becomes 2^-100.
  __device__ __forceinline__ void set_scale(float s) {
    constexpr float kTiny = 7.8886090522101181e-31f;
    scale = fabsf(s) < kTiny ? kTiny : fabsf(s);  // NaN stays
  }

  // Fragments are requested AHEAD products before theirs, into a ring.
  static constexpr int UNITS = NS * PARTS * NKB, RING = 4, AHEAD = RING - 1;
  template <int SIDE>
  __device__ __forceinline__ h8_t k_load(uint32_t k, int u) const {
    const int c = u / (PARTS * NKB), part = u / NKB % PARTS, kb = u % NKB;
    return k_read<D>((k ^ 32 * c) + part * SIDE, kb);
  }
  __device__ __forceinline__ void k_mma(int u, const h8_t f, f16v_t* s) const {
    const int c = u / (PARTS * NKB), part = u / NKB % PARTS, kb = u % NKB;
    s[kb] = mma<BF>(f, q[c], s[kb]);
    if constexpr (QLO) {
      if (part == 0) s[kb] = mma<BF>(f, ql[c], s[kb]);
    }
  }
  // Scores of the keys at LDS address k (k_at's lane offset included).
  template <int SIDE>
  __device__ __forceinline__ void scores(uint32_t k, f16v_t* s) const {
#pragma unroll
    for (int kb = 0; kb < NKB; ++kb) s[kb] = f16v_t{};
    h8_t f[RING];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) f[u] = k_load<SIDE>(k, u);
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      if (u + AHEAD < UNITS) f[(u + AHEAD) % RING] = k_load<SIDE>(k, u + AHEAD);
      k_mma(u, f[u % RING], s);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  __device__ __forceinline__ float top(const f16v_t* s) const {  // largest scaled score of the lane's column
    float x = -kInf;
#pragma unroll
    for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) x = fmaxf(x, s[kb][i]);
    return halves_max(x) * scale;
  }
  // The running maximum moves only when a row's passes it by more than 2^8: weights stay below
  // 2^8 meanwhile.
  __device__ __forceinline__ void rescale(float mt) {
    if (__builtin_amdgcn_ballot_w64(mt > m + 8.f)) {
      const float m_new = fmaxf(m, mt);
      const float alpha = m_new == -kInf ? 1.f : __builtin_amdgcn_exp2f(m - m_new);
      l *= alpha;
#pragma unroll
      for (int db = 0; db < NDB; ++db) acc[db] *= alpha;
      m = m_new;
    }
  }
  // Scores to rounded weights (p[ks]: 16 keys), and with NEXT the next step's scores. Pair n's
  // exponentials are one slot ahead of its sum and rounding.
  template <bool NEXT, int SIDE>
  __device__ __forceinline__ void weights(const f16v_t* s, u4_t* p, uint32_t k, f16v_t* next) {
    const float ms = m == -kInf ? 0.f : m - kShift;
    float sum[2] = {0.f, 0.f}, x[2][2];
    auto ex = [&](int n) {
#pragma unroll
      for (int e = 0; e < 2; ++e)
        x[n & 1][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n / 8][2 * (n % 8) + e], scale, -ms));
    };
    auto put = [&](int n) {
      sum[0] += x[n & 1][0];
      sum[1] += x[n & 1][1];
      p[n / 4][n % 4] = pack2<BF>(x[n & 1][0], x[n & 1][1]);
      if constexpr (PLO) {
        const h2_t hi = __builtin_bit_cast(h2_t, (uint32_t)p[n / 4][n % 4]);
        p[NW + n / 4][n % 4] = pack2<false>(x[n & 1][0] - (float)hi[0], x[n & 1][1] - (float)hi[1]);
      }
    };
    if constexpr (NEXT) {
#pragma unroll
      for (int kb = 0; kb < NKB; ++kb) next[kb] = f16v_t{};
      h8_t f[RING];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) f[u] = k_load<SIDE>(k, u);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int u = 0; u < UNITS; ++u) {
        if (u + AHEAD < UNITS) f[(u + AHEAD) % RING] = k_load<SIDE>(k, u + AHEAD);
        k_mma(u, f[u % RING], next);
#pragma unroll
        for (int n = u * (NP + 1) / UNITS; n < (u + 1) * (NP + 1) / UNITS; ++n) {
          if (n < NP) ex(n);
          if (n > 0) put(n - 1);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
#pragma unroll
      for (int n = 0; n < NP; ++n) {
        ex(n);
        put(n);
      }
    }
    asm volatile("" : "+v"(sum[0]), "+v"(sum[1]));  // made here, not where l is used: 32 registers
    l += sum[0] + sum[1];
  }
  // O^T += V^T P^T over the values at LDS address v (v_at's lane offset included); returns top() of
  // `next`, taken along.
  template <bool NEXT, int SIDE = 0>
  __device__ __forceinline__ float values(const u4_t* p, uint32_t v, const f16v_t* next) {
    constexpr int VP = VLO ? 2 : 1, VU = 2 * NKB * NDB * VP;  // 16 keys x 32 channels of a part each
    auto load = [&](int u) { return v_read<D>((v ^ 64 * (u / VP % NDB)) + u % VP * SIDE, u / VP / NDB); };
    h8_t f[RING];
    float x = -kInf;
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) f[u] = load(u);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < VU; ++u) {
      if (u + AHEAD < VU) f[(u + AHEAD) % RING] = load(u + AHEAD);
      const int db = u / VP % NDB, ks = u / VP / NDB;
      acc[db] = mma<BF>(f[u % RING], __builtin_bit_cast(h8_t, p[ks]), acc[db]);
      if constexpr (PLO) {
        if (u % VP == 0) acc[db] = mma<BF>(f[u % RING], __builtin_bit_cast(h8_t, p[NW + ks]), acc[db]);
      }
      if constexpr (NEXT) {
#pragma unroll
        for (int n = u * NP / VU; n < (u + 1) * NP / VU; ++n)
          x = fmaxf(fmaxf(x, next[n / 8][2 * (n % 8)]), next[n / 8][2 * (n % 8) + 1]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    return NEXT ? halves_max(x) * scale : 0.f;
  }
};

typedef float f4_any_t __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u4_any_t __attribute__((ext_vector_type(4), aligned(2)));

// A lane's O^T column as a 16-bit row at `row` (any element alignment): the half-waves exchange
// their channels of two groups of eight, so that each lane stores 16 consecutive bytes. Both
// lanes of a column take part.
template <int NDB, bool BF>
__device__ __forceinline__ void store16(uint8_t* row, const f16v_t* acc, int hh) {
#pragma unroll
  for (int db = 0; db < NDB; ++db)
#pragma unroll
    for (int g = 0; g < 4; g += 2) {
      u4_any_t o;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint32_t x = pack2<BF>(acc[db][4 * g + 2 * e], acc[db][4 * g + 2 * e + 1]);
        const uint32_t y = pack2<BF>(acc[db][4 * g + 4 + 2 * e], acc[db][4 * g + 5 + 2 * e]);
        const auto z = __builtin_amdgcn_permlane32_swap(x, y, false, false);
        o[e] = z[0];
        o[2 + e] = z[1];
      }
      *(u4_any_t*)(row + 64 * db + 16 * g + 16 * hh) = o;
    }
}

}  // namespace ek
