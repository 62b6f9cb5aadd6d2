// Causal attention of packed prompts on 16-bit matrix instructions: float16 or bfloat16 rows of
// head size 64, 128 or 256 (attend_any.hip takes every other case).
//
// One workgroup per (query tile, KV head): 32 query rows per wave, rows are (token, GQA head)
// pairs of one KV head, so its heads share every key and value that is read. The tile's keys
// stream in steps of 64 through a ring in LDS, keys and values row-major as they lie in memory
// (direct global-to-LDS loads of 16 bytes a lane, rows past the sequence clamped to its last
// one), and each wave runs S^T, an online softmax and O^T per step (tiles.h). Scores and sums are
// float32; the weights are rounded to the inputs' type for the value product (half a step of it,
// 2^-8 or 2^-11, relative to each weight), float16 ones times 2^6 so that small ones keep their
// bits.
//
// A value that is infinite or NaN must not reach rows that do not see its key (their weight is
// 0, and 0 x inf is NaN). Steps with a causal edge look for one; a wave that finds one computes
// its rows again, with such values out of the products and added where they are seen.
//
// Four waves of 32 rows and two workgroups a CU: a wave's exponentials and a step's barrier leave
// the matrix cores to the other workgroup's waves. Bound by the matrix cores on long prompts: one of
// 16384 tokens (8 KV heads of GQA 4, D 128, bf16) takes 1.95 to 2.0 ms, 1.10 to 1.13 PFLOP/s of
// causal products (a library product of 8192^3: 1.205), MFMA busy 65 % of the cycles, no LDS bank
// conflicts; six packed prompts of 100 to 2600 tokens 146 us (876 TFLOP/s: short tiles start and
// end more often). Few tiles are bound by the longest one's chain of steps: 1500 tokens take 32 us,
// 24 steps of 1.3. The keys of a tile are not split over workgroups: its rows then have the same
// bits whatever else the step holds.
#include "tiles.h"

namespace ek {
namespace {

constexpr int kKeys = 64;
constexpr int kWaves = 4;
constexpr int kSlots = 2;  // steps in LDS: two workgroups fit a CU up to head size 128
constexpr float kInf = __builtin_inff();

template <int D>
struct Ring {
  static constexpr int SIDE = kKeys * D * 2;  // bytes of a step's keys (its values take as many)
  static constexpr int NDMA = SIDE / 1024 / kWaves;
};

}  // namespace

template <int D, bool BF>
__global__ __launch_bounds__(64 * kWaves, D == 256 ? 1 : 2) void prompt_kernel(PromptArgs a) {
  using R = Ring<D>;
  constexpr int NS = D / 16, NDB = D / 32, NDMA = R::NDMA;
  constexpr uint32_t kTop = BF ? 0x7f80u : 0x7c00u;  // infinity's bits
  extern __shared__ __attribute__((aligned(1024))) uint8_t ring[];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int j = lane & 31, hh = lane >> 5;
  const int h = (int)(blockIdx.x % a.H);  // heads fastest: with 8 of them an XCD's L2 holds one head's rows
  // Tiles come longest first, and a CU's second workgroup is the 256th after its first. Where that
  // is all there are, the second half goes shortest first, so that the longest tile shares its CU
  // with the shortest. us plainly / so, 8 KV heads of GQA 4, D 128: 1500 tokens (376 workgroups)
  // 32.2 / 31.7, 2000 (504) 43.7 / 42.0, 5 x 300 (400) 13.6 / 12.7; 2500 (632), were it so there
  // too, 59.7 / 65.8.
  int tile = (int)(blockIdx.x / a.H);
  if constexpr (D <= 128) {
    const int first = 256 / a.H;
    if (tile >= first && a.n_tiles <= 2 * first) tile = a.n_tiles - 1 - (tile - first);
  }
  const int32_t* td = a.tiles + 4 * (long)tile;
  const long row0 = td[0];
  const int seq = td[1], t0 = td[2], n_rows = td[3] * a.gqa;
  const int kv_end = min(seq, t0 + td[3]);
  const int n_steps = (kv_end + kKeys - 1) / kKeys;

  const int r = 32 * wave + j;
  const bool live = r < n_rows;
  const bool active = 32 * wave < n_rows;
  const int rc = live ? r : n_rows - 1;
  const int pos = t0 + rc / a.gqa, qh = h * a.gqa + rc % a.gqa;
  const int first_pos = t0 + 32 * wave / a.gqa;                              // the wave's first row's
  const int last_pos = t0 + min(32 * wave + 31, n_rows - 1) / a.gqa;  // and last row's position

  // LDS: the keys of two steps, then the values of two. This lane's share of a step's loads: byte
  // offsets from the step's first row. The permutation of LDS slots is made on the memory side,
  // since LDS fills in lane order.
  const uint8_t* kbase = (const uint8_t*)a.k + 2 * (row0 * a.k_s0 + (long)h * a.k_s1);
  const uint8_t* vbase = (const uint8_t*)a.v + 2 * (row0 * a.v_s0 + (long)h * a.v_s1);
  const uint32_t ring0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)ring);
  auto issue = [&](int step, bool val) {
    const int kb = step * kKeys, last = kv_end - 1 - kb;
    const uint32_t stride = (uint32_t)(val ? a.v_s0 : a.k_s0) * 2;
    const uint8_t* from = uniform_ptr((val ? vbase : kbase) + (long)kb * stride);
    const uint32_t to = ring0 + (uint32_t)(((val ? kSlots : 0) + step % kSlots) * R::SIDE + 1024 * NDMA * wave);
#pragma unroll
    for (int i = 0; i < NDMA; ++i) {
      const int q = 1024 * (NDMA * wave + i) + 16 * lane;
      const int key = q / (2 * D), slot = q % (2 * D) / 16;
      const uint32_t off = (uint32_t)min(key, last) * stride + 16 * (slot ^ (val ? v_swz<D>(key) : k_swz<D>(key)));
      dma16(from, off, to + 1024 * i);
    }
  };
  issue(0, false);
  issue(0, true);
  if (n_steps > 1) issue(1, false);

  // Query fragments (B operand): row r, channels 16 s + 8 hh .. + 8.
  Rows<D, BF, 2, 1, false> w;
  w.set_scale(a.scale_log2);
  {
    const uint16_t* src = (const uint16_t*)a.q + (row0 + pos) * a.q_s0 + (long)qh * a.q_s1 + 8 * hh;
#pragma unroll
    for (int s = 0; s < NS; ++s) w.q[s] = *(const h8_t*)(src + 16 * s);
    if (a.scale_log2 < 0.f) {
#pragma unroll
      for (int s = 0; s < NS; ++s)
        w.q[s] = __builtin_bit_cast(h8_t, __builtin_bit_cast(u4_t, w.q[s]) ^ 0x80008000u);
    }
  }

  // Scores of keys behind the row's position: -inf. `edge`: some row does not see the whole step.
  auto mask = [&](int kb0, f16v_t* s) {
    int left = pos - kb0 - 4 * hh;
    asm volatile("" : "+v"(left));  // keeps the compares in this branch
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[kb][i] = 32 * kb + 8 * (i >> 2) + (i & 3) > left ? -kInf : s[kb][i];
  };
  auto edge_of = [&](int step) { return (step + 1) * kKeys > first_pos + 1; };

  w.clear();
  const uint32_t k_lane = ring0 + k_at<D>(0, j, hh), v_lane = ring0 + kSlots * R::SIDE + v_at<D>(0, lane);
  const int my_steps = active ? last_pos / kKeys + 1 : 0;  // steps that some row of the wave sees
  bool odd = false;  // a step with an edge holds an infinite value or NaN
  // This wave's loads have landed, with the barrier every wave's: the keys of `step` + 1 and the
  // values of `step`. They were made a step ago; the next ones go to the slots that every wave has
  // left.
  auto advance = [&](int step) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (step + 2 < n_steps) issue(step + 2, false);
    if (step + 1 < n_steps) issue(step + 1, true);
  };
  auto vslot = [&](int step) { return (uint32_t)(step % kSlots * R::SIDE); };
  auto look = [&](int step) {
    if (!edge_of(step)) return;
    typedef unsigned short us2_t __attribute__((ext_vector_type(2)));
    us2_t m = {0, 0};
    const uint32_t vt = ring0 + kSlots * R::SIDE + vslot(step) + 16 * lane;
#pragma unroll 4
    for (int i = 0; i < R::SIDE / 1024; ++i) {
      const u4_t x = *(const lds_t<u4_t>*)(vt + 1024 * i);
#pragma unroll
      for (int e = 0; e < 4; ++e) m = __builtin_elementwise_max(m, __builtin_bit_cast(us2_t, x[e] & 0x7fff7fffu));
    }
    odd = odd || __builtin_amdgcn_ballot_w64(m[0] >= kTop || m[1] >= kTop);
  };
  f16v_t s0[2], s1[2];
  float mt = -kInf;
  // A step's weights and values beside the next step's scores (tiles.h).
  auto body = [&](int step, f16v_t* cur, f16v_t* nxt) {
    advance(step);
    look(step);
    w.rescale(mt);
    u4_t p[4];
    w.template weights<true, R::SIDE>(cur, p, k_lane + (uint32_t)((step + 1) % kSlots * R::SIDE), nxt);
    mt = w.template values<true>(p, v_lane + vslot(step), nxt);
    if (edge_of(step + 1)) {
      mask((step + 1) * kKeys, nxt);
      mt = w.top(nxt);
    }
  };
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  int step = 0;
  if (my_steps > 0) {
    w.template scores<R::SIDE>(k_lane, s0);
    if (edge_of(0)) mask(0, s0);
    mt = w.top(s0);
    for (; step + 2 < my_steps; step += 2) {
      body(step, s0, s1);
      body(step + 1, s1, s0);
    }
    if (step + 1 < my_steps) {
      body(step++, s0, s1);
      s0[0] = s1[0];
      s0[1] = s1[1];
    }
    advance(step);
    look(step);
    w.rescale(mt);
    u4_t p[4];
    w.template weights<false, R::SIDE>(s0, p, 0, s0);
    w.template values<false>(p, v_lane + vslot(step), s0);
    ++step;
  }
  for (; step < n_steps; ++step) advance(step);  // steps of the workgroup's later rows

  // Rare: the wave's rows once more, from memory. The products leave infinite values and NaN out;
  // which of them a row sees is a product of its own, of 0 / 1 weights with 1 for +inf, 2^7 for
  // -inf and 2^14 for NaN (at most 64 of each a step: the sum tells them apart).
  if (odd) {
    w.clear();
#pragma unroll 1
    for (int kb0 = 0; kb0 <= last_pos; kb0 += kKeys) {
      f16v_t x2[2] = {f16v_t{}, f16v_t{}};
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        const uint8_t* row = kbase + 2 * (long)min(kb0 + 32 * kb + j, kv_end - 1) * a.k_s0 + 16 * hh;
#pragma unroll
        for (int c = 0; c < NS; ++c) x2[kb] = mma<BF>(*(const h8_t*)(row + 32 * c), w.q[c], x2[kb]);
      }
      mask(kb0, x2);
      w.rescale(w.top(x2));
      u4_t p[4];
      w.template weights<false, R::SIDE>(x2, p, 0, x2);
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        uint32_t seen[4];
        const uint16_t* row[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int key = kb0 + 16 * ks + 8 * (e >> 2) + 4 * hh + (e & 3);
          row[e] = (const uint16_t*)(vbase + 2 * (long)min(key, kv_end - 1) * a.v_s0) + j;
          if (!(e & 1)) seen[e >> 1] = pack2<BF>(key <= pos ? 1.f : 0.f, key + 1 <= pos ? 1.f : 0.f);
        }
#pragma unroll
        for (int db = 0; db < NDB; ++db) {
          u4_t val, kinds;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint32_t x[2], k[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              x[u] = row[2 * e + u][32 * db];
              const bool bad = (x[u] & 0x7fffu) >= kTop;
              k[u] = pack2<BF>((x[u] & 0x7fffu) > kTop ? 16384.f : x[u] & 0x8000u ? 128.f : 1.f, 0.f);
              k[u] = bad ? k[u] : 0;
              x[u] = bad ? 0 : x[u];
            }
            val[e] = x[0] | x[1] << 16;
            kinds[e] = k[0] | k[1] << 16;
          }
          w.acc[db] = mma<BF>(__builtin_bit_cast(h8_t, val), __builtin_bit_cast(h8_t, p[ks]), w.acc[db]);
          f16v_t found = f16v_t{};
          found = mma<BF>(__builtin_bit_cast(h8_t, kinds), __builtin_bit_cast(h8_t, u4_t{seen[0], seen[1], seen[2], seen[3]}),
                          found);
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int n = (int)found[i];
            float x = n & 127 ? kInf : 0.f;
            x = n >> 7 & 127 ? (n & 127 ? __builtin_nanf("") : -kInf) : x;
            w.acc[db][i] += n >> 14 ? __builtin_nanf("") : x;
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
  }

  const float l = halves_sum(w.l);
  if (!live) return;
  const long row = row0 + pos, lr = row * a.hq + qh;
  float inv = l == 0.f ? 0.f : 1.f / l, lse = l == 0.f ? -kInf : w.m - w.kShift + __log2f(l), wp = 0.f;
  if (a.part) {
    const float pl = a.part_lse[lr], mx = fmaxf(pl, lse);
    if (mx != -kInf) {
      const float ep = __builtin_amdgcn_exp2f(pl - mx), eo = __builtin_amdgcn_exp2f(lse - mx), sum = ep + eo;
      wp = ep / sum;
      inv *= eo / sum;
      lse = mx + __log2f(sum);
    }
  }
  if (a.lse && hh == 0) a.lse[lr] = lse;
#pragma unroll
  for (int db = 0; db < NDB; ++db) w.acc[db] *= inv;
  if (wp != 0.f) {
    const float* src = a.part + row * a.p_s0 + (long)qh * a.p_s1 + 4 * hh;
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f4_t x = *(const f4_any_t*)(src + 32 * db + 8 * g);
#pragma unroll
        for (int e = 0; e < 4; ++e) w.acc[db][4 * g + e] = __builtin_fmaf(wp, x[e], w.acc[db][4 * g + e]);
      }
  }
  const long ob = row * a.o_s0 + (long)qh * a.o_s1;
  if (a.out_dtype == ECHOKV_F32) {
    float* dst = (float*)a.out + ob + 4 * hh;
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *(f4_any_t*)(dst + 32 * db + 8 * g) = f4_t{w.acc[db][4 * g], w.acc[db][4 * g + 1], w.acc[db][4 * g + 2], w.acc[db][4 * g + 3]};
  } else if (a.out_dtype == ECHOKV_BF16) {
    store16<NDB, true>((uint8_t*)a.out + 2 * ob, w.acc, hh);
  } else {
    store16<NDB, false>((uint8_t*)a.out + 2 * ob, w.acc, hh);
  }
}

bool prompt_mfma(const PromptArgs& a) {
  if (a.dtype == ECHOKV_F32 || (a.D != 64 && a.D != 128 && a.D != 256)) return false;
  // Rows aligned for 16-byte loads; a step's rows within 31 bits of bytes.
  auto rows_ok = [](const void* p, long s0, long s1) {
    return (uintptr_t)p % 16 == 0 && s0 % 8 == 0 && s1 % 8 == 0 && s0 >= 0 && s0 < (1L << 30) / kKeys;
  };
  return a.gqa <= kPromptRows && rows_ok(a.q, 0, 0) && a.q_s0 % 8 == 0 && a.q_s1 % 8 == 0 && rows_ok(a.k, a.k_s0, a.k_s1) &&
         rows_ok(a.v, a.v_s0, a.v_s1);
}

template <int D, bool BF>
static hipError_t launch_t(const PromptArgs& a, hipStream_t s) {
  using R = Ring<D>;
  constexpr int lds = 2 * kSlots * R::SIDE;
  static std::atomic<uint64_t> attr_done{0};
  const hipError_t e = ensure_lds_limit((const void*)prompt_kernel<D, BF>, lds, &attr_done);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((prompt_kernel<D, BF>), dim3((unsigned)((long)a.n_tiles * a.H)), dim3(64 * kWaves), lds, s, a);
  return hipGetLastError();
}

template <int D>
static hipError_t launch_d(const PromptArgs& a, hipStream_t s) {
  return a.dtype == ECHOKV_BF16 ? launch_t<D, true>(a, s) : launch_t<D, false>(a, s);
}

hipError_t launch_prompt(const PromptArgs& a, hipStream_t s) {
  if (a.D == 64) return launch_d<64>(a, s);
  if (a.D == 128) return launch_d<128>(a, s);
  if (a.D == 256) return launch_d<256>(a, s);
  return hipErrorInvalidValue;
}

}  // namespace ek
