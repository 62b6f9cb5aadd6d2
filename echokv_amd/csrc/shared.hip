// Attention of many query rows over one cached block list on 16-bit matrix instructions (head
// sizes 64, 128 and 256, layouts whose items sit in one group; attend_any.hip takes the others).
//
// One workgroup per (32 query rows per wave, KV head, range of keys): rows are (entry, GQA head)
// pairs, whatever sequence they belong to, so a key is dequantized once for all of them. Keys are
// held as a float16 hi + lo pair (2^-22 of the value together). Each wave runs S^T, an online softmax
// and O^T over a step's keys (tiles.h).
//
// Decode into float16 or float32 holds weights and values as hi + lo pairs too (PLO, VLO), what the
// paged decode it stands for holds: a float16 rounding of each is 2^-11 of weight x |value|, more than
// 2e-3 where outlier channels reach 40. Into bfloat16, whose own rounding is eight times that, both are
// float16. us a decode with one part / two: 4 sequences behind 512 28.7 / 29.9, 64 behind 4096 (GQA 4,
// INT4) 63.9 / 65.3, 24 behind 8192 (GQA 8, INT2) 58.5 / 62.5, 256 behind 16384 (INT8) 204 / 258.
// Prompts behind a prefix (float32 rows for prompt.hip to join) take values in float16, one rounding,
// as prefill.hip, and weights in float16 for bfloat16 queries, hi + lo for float16 and float32 ones:
// both roundings at once made float16 outputs 1.6 times as far off as their own rounding does, values
// alone 1.3 times (the low parts cost 1 to 7 % of a call).
//
// prefix_kernel dequantizes each step into LDS itself: a thread takes items of four keys x eight
// channels, of K in the first four waves and of V in the others (four waves: of both), its loads a
// chain spread over the steps (an item's codes are requested a step before they are needed, its
// page header two and its block id three).
//
// With many rows the same keys would be dequantized again for every 256 of them:
// prefix_pack_kernel dequantizes the prefix once into a workspace, in 64-key tiles laid out as
// LDS holds them, and prefix_flash_kernel streams those by direct global-to-LDS loads, the loop of
// prompt.hip. The workspace holds 128 MiB of tiles at most; a longer prefix goes through it slab by
// slab, each slab the next part of every range, and a row goes on from the unnormalized output,
// maximum and sum that the slab before left in its workspace row.
//
// Measured (8 KV heads of GQA 4, D 128): 64 sequences (256 rows) behind 4096 INT4 keys 23 us in
// prefix_kernel (27 with VLO), of which 16 ranges' partial rows (17 MB) are 3 at the rate of a copy and the loads'
// chain (block id, header, codes) with four steps the rest. 8065 bfloat16 rows behind 8192: pack 16
// us, then flash 1.36 to 1.44 ms, bound by the matrix cores: 0.76 to 0.80 PFLOP/s of the formula's
// products, 1.14 to 1.19 of those made (a key's two parts make the scores twice the work), MFMA
// busy 70 % of the cycles, no LDS bank conflicts. 256 sequences behind 16384 INT8 keys: pack 27 us
// (134 MB, 4.9 TB/s, a copy's rate), flash 99 us (1.04 PFLOP/s made).
#include "items.h"
#include "tiles.h"

namespace ek {
namespace {

constexpr float kInf = __builtin_inff();

// An item's words: each row's eight codes in the 8 bytes at or before them.
struct Raw {
  uint2 k[4], v[4];
  uint4 ks, km;  // float16 scale / min of the eight channels (the quad's K group)
  uint16_t vs[4], vm[4];
  int rg;   // K group of the block's residual slot (if it has one)
  bool ok;  // the item's keys can be read
};

struct Head {
  uint4 h;
  int blk, rs;  // rs: the low word (slots are small, -1: none)
};

// Items of the keys [k_begin, k_end) of head h in steps of KEYS: a thread's item of a step is four
// keys x eight channels. Nothing loaded is looked at before the step that needs it, and no load
// sits in a branch (addresses are clamped instead): the wave would wait for it there.
template <int D, int KEYS, bool VLO>
struct Items {
  static constexpr int OCTS = D / 8, SIDE = KEYS * D * 2;  // bytes of a step's K hi, K lo or V (VLO: V hi, V lo)
  static constexpr int STEP = (VLO ? 4 : 3) * SIDE;
  const PrefixArgs& a;
  const int h, k_begin, k_end, oct, quad;

  __device__ __forceinline__ Items(const PrefixArgs& args, int head, int begin, int end, int id)
      : a(args), h(head), k_begin(begin), k_end(end), oct(id % OCTS), quad(id / OCTS) {}
  __device__ __forceinline__ int key(int step) const { return k_begin + step * KEYS + 4 * quad; }
  __device__ __forceinline__ int off(int step) const { return key(step) & (a.L.BS - 1); }
  __device__ __forceinline__ int load_blk(int step) const {
    const int kp = key(step);
    return a.blocks[(kp < k_end - 1 ? kp : k_end - 1) >> a.bs_shift];
  }
  __device__ __forceinline__ long page_of(int blk) const { return (unsigned)blk < (unsigned long)a.L.nb ? (long)blk : 0l; }
  __device__ __forceinline__ Head load_head(int blk) const {
    const long b = page_of(blk);
    return Head{*(const uint4*)(a.pages + b * a.L.stride), blk, *(const int32_t*)(a.block_res + b)};
  }
  // keys, values (wave-uniform): what of the item this thread takes; values alone use w.k.
  __device__ __forceinline__ void load(int step, const Head& x, Raw& w, bool keys, bool values, bool both) const {
    const Lay& L = a.L;
    const int rs = (unsigned)x.rs < (unsigned)a.res.rows ? x.rs : 0;
    w.rg = *(const int32_t*)(a.res_group + rs);  // the low word: groups are small
    const int ch = 8 * oct, G = D / L.VG, o = off(step), bits = tier_of(x.h.x & 0xffu);
    const int tpc_shift = a.bs_shift + 1 - (bits == 8 ? 3 : bits == 4 ? 2 : 1);
    const int c = o >> tpc_shift;
    long cb = page_of(x.blk) * L.stride + L.o_data;
    bool ok = (unsigned)x.blk < (unsigned long)L.nb && key(step) < k_end;
    if (c > 0) {
      const Hdr hd{x.h.x & 0xffu, (int32_t)x.h.y, (int32_t)x.h.z, (int32_t)x.h.w};
      const uint32_t id = (uint32_t)hd.id(c - 1);
      const uint32_t page = a.kc_mul ? __umulhi(id, a.kc_mul) : id;
      const bool there = (int)id >= 0 && (long)page < L.nb;
      cb = there ? (long)page * L.stride + L.o_data + (long)(id - page * (uint32_t)L.KC) * L.cb : cb;
      ok = ok && there;
    }
    w.ok = ok;
    const int rowb = L.H * (D / 4) * bits;
    const uint8_t* pg = a.pages + page_of(x.blk) * L.stride;
    // An item that cannot be read takes its page's first bytes instead (dequantized to zero).
    const uint8_t* kp = ok ? a.pages + cb + (long)(o & ((1 << tpc_shift) - 1)) * rowb + ((h * D + ch) * bits / 8 & ~7) : pg;
    const int step_b = ok ? rowb : 0;
    if (keys) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w.k[i] = *(const uint2*)(kp + i * step_b);
      const int se = ((o >> a.kg_shift) * L.H + h) * D + ch;
      w.ks = *(const uint4*)(pg + L.o_ks + 2 * se);
      w.km = *(const uint4*)(pg + L.o_km + 2 * se);
    }
    if (values) {
      const int ve = (o * L.H + h) * G + ch / L.VG;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        (both ? w.v : w.k)[i] = *(const uint2*)(kp + i * step_b + step_b / 2);
        w.vs[i] = *(const uint16_t*)(pg + L.o_vs + 2 * (ve + i * L.H * G));
        w.vm[i] = *(const uint16_t*)(pg + L.o_vm + 2 * (ve + i * L.H * G));
      }
    }
  }
  // Eight channels as float16 hi + lo, at `buf` + `at` and SIDE behind it. CLAMP: statistics rounded
  // up can take the largest float16 value past its type (65504 in INT4 to 65536); lo holds the rest.
  template <bool CLAMP = false>
  __device__ __forceinline__ void put2(uint8_t* buf, int at, const float* x8) const {
    u4_t hi, lo;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      auto first = [](float x) { return (_Float16)(CLAMP ? __builtin_amdgcn_fmed3f(x, -65504.f, 65504.f) : x); };
      const h2_t p = {first(x8[2 * e]), first(x8[2 * e + 1])};
      hi[e] = __builtin_bit_cast(uint32_t, p);
      lo[e] = pack2<false>(x8[2 * e] - (float)p[0], x8[2 * e + 1] - (float)p[1]);
    }
    *(u4_t*)(buf + at) = hi;
    *(u4_t*)(buf + SIDE + at) = lo;
  }
  __device__ __forceinline__ void put_k(uint8_t* buf, int i, const float* x8) const {
    const int k = 4 * quad + i;
    put2(buf, k * (2 * D) + 16 * (oct ^ k_swz<D>(k)), x8);
  }
  __device__ __forceinline__ int v_slot(int i) const {
    const int k = 4 * quad + i;
    return k * (2 * D) + 16 * (oct ^ v_swz<D>(k));
  }
  __device__ __forceinline__ void put_v(uint8_t* buf, int i, const u4_t x) const { *(u4_t*)(buf + 2 * SIDE + v_slot(i)) = x; }
  // The item dequantized into a step's sides at `buf` (LDS or memory; keys past the range and
  // blocks that cannot be read: zeros).
  __device__ __forceinline__ void store(uint8_t* buf, int step, const Head& x, const Raw& w, bool keys, bool values,
                                        bool both) const {
    const Lay& L = a.L;
    const int kp = key(step), o = off(step), bits = tier_of(x.h.x & 0xffu), ch = 8 * oct;
    const int sh = 8 * (((h * D + ch) * bits / 8) & 7);
    auto rows = [&](auto width) __attribute__((always_inline)) {
      constexpr int B = decltype(width)::value;
      const uint32_t sw[4] = {w.ks.x, w.ks.y, w.ks.z, w.ks.w}, mw[4] = {w.km.x, w.km.y, w.km.z, w.km.w};
      if (keys) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          h2_t c[4];
          code_pairs<B>(w.k[i], sh, c);
          float x8[8];
#pragma unroll
          for (int e = 0; e < 8; ++e)
            x8[e] = __builtin_fmaf((float)c[e >> 1][e & 1], (float)u2h(sw[e >> 1])[e & 1], (float)u2h(mw[e >> 1])[e & 1]);
          put_k(buf, i, x8);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      if (values) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          h2_t c[4];
          code_pairs<B>((both ? w.v : w.k)[i], sh, c);
          const h2_t vs = u2h(w.vs[i] * 0x10001u), vm = u2h(w.vm[i] * 0x10001u);
          if constexpr (VLO) {
            float x8[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x8[e] = __builtin_fmaf((float)c[e >> 1][e & 1], (float)vs[0], (float)vm[0]);
            put2<true>(buf + 2 * SIDE, v_slot(i), x8);
          } else {
            u4_t v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(c[e], vs, vm));
            put_v(buf, i, v);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    };
    if (bits == 4) rows(std::integral_constant<int, 4>{});
    else if (bits == 2) rows(std::integral_constant<int, 2>{});
    else rows(std::integral_constant<int, 8>{});
    const int n_live = w.ok ? k_end - kp : 0;
    if (n_live < 4) {  // rare: past the range's end, or a block that cannot be read
      const float z8[8] = {};
#pragma unroll 1
      for (int i = n_live > 0 ? n_live : 0; i < 4; ++i) {
        if (keys) put_k(buf, i, z8);
        if (values) put_v(buf, i, u4_t{});
        if (VLO && values) put_v(buf + SIDE, i, u4_t{});
      }
    }
    if (keys && w.ok && (unsigned)x.rs < (unsigned)a.res.rows && w.rg == o >> a.kg_shift) {  // rare: an open K group
#pragma unroll 1
      for (int i = 0; i < 4 && kp + i < k_end; ++i) {
        float x8[8];
        ld_n<8>(a.res.ptr, a.res.dtype, x.rs * a.res.s0 + (long)((o + i) & (L.KG - 1)) * a.res.s1 + h * a.res.s2 + ch, x8);
        put_k(buf, i, x8);
      }
    }
  }
};

// A lane's query row: row r of the (entry, GQA head) pairs of KV head h. A sequence shorter than
// the prefix (graph padding) is not asked for its row index, which may be any: it computes with
// query row 0 into its workspace rows, and the join leaves them.
struct Row {
  int t, qh;
  long q_row;
  bool live;
};
__device__ __forceinline__ Row row_of(const PrefixArgs& a, int h, int r) {
  const bool live = r < (int)a.n * a.gqa;  // below 2^25, checked on the host
  const int t = live ? (int)((unsigned)r / (unsigned)a.gqa) : 0;
  const long len = a.lens ? a.lens[t] : a.len, q_row = a.q_rows ? a.q_rows[t] : t;
  return Row{t, h * a.gqa + (live ? r - t * a.gqa : 0), len < a.len ? 0 : q_row, live};
}

// The row's query as fragments: 16 bytes at a time, all requested together.
template <int D, int NKB, bool QLO, bool PLO, bool VLO>
__device__ __forceinline__ void load_query(Rows<D, false, NKB, 2, QLO, PLO, VLO>& w, const PrefixArgs& a, const Row& row, int hh) {
  constexpr int NS = D / 16, QW = QLO ? 2 : 1;
  w.set_scale(a.scale_log2);
  const uint8_t* src = (const uint8_t*)a.q + (row.q_row * a.q_s0 + (long)row.qh * a.q_s1 + 8 * hh) * (2 * QW);
  const uint32_t flip = a.scale_log2 < 0.f ? (QLO ? 0x80000000u : 0x80008000u) : 0u;
  u4_t x[NS][QW];
#pragma unroll
  for (int s = 0; s < NS; ++s)
#pragma unroll
    for (int i = 0; i < QW; ++i) x[s][i] = *(const u4_any_t*)(src + 32 * QW * s + 16 * i) ^ flip;
  const bool bf = a.q_dtype == ECHOKV_BF16;
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    if constexpr (QLO) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float y = __uint_as_float(x[s][e >> 2][e & 3]);
        w.q[s][e] = (_Float16)y;
        w.ql[s][e] = (_Float16)(y - (float)w.q[s][e]);
      }
    } else {
      u4_t y;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        y[e] = pack2<false>(__uint_as_float(x[s][0][e] << 16), __uint_as_float(x[s][0][e] & 0xffff0000u));
      w.q[s] = __builtin_bit_cast(h8_t, bf ? y : x[s][0]);
    }
  }
}

// Scores of a step's keys from `left` on: -inf.
template <int NKB>
__device__ __forceinline__ void mask_tail(f16v_t* s, int left, int hh) {
  left -= 4 * hh;
  asm volatile("" : "+v"(left));  // keeps the compares in the caller's branch
#pragma unroll
  for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
    for (int i = 0; i < 16; ++i) s[kb][i] = 32 * kb + 8 * (i >> 2) + (i & 3) < left ? s[kb][i] : -kInf;
}

// The wave's rows out: range z's partial ones, or normalized ones with their log-sum-exp.
template <int D, int NKB, bool QLO, bool PLO, bool VLO>
__device__ __forceinline__ void write_rows(Rows<D, false, NKB, 2, QLO, PLO, VLO>& w, const PrefixArgs& a, int h, int r, int z, int hh) {
  const float l = halves_sum(w.l);
  asm volatile("" : "+v"(r));  // the row's place is found again, not kept through the loop
  const Row row = row_of(a, h, r);
  if (!row.live) return;
  const bool direct = a.part != nullptr;
  const long pr = ((long)z * a.n + row.t) * a.hq + row.qh;
  if (hh == 0) {
    if (direct) a.lse[row.q_row * a.hq + row.qh] = l == 0.f ? -kInf : w.m - w.kShift + __log2f(l);
    else *(float2*)(a.ml + 2 * pr) = float2{w.m - w.kShift, l};
  }
  const float inv = !direct ? 1.f : l == 0.f ? 0.f : 1.f / l;
  float* dst = (direct ? a.part + row.q_row * a.p_s0 + (long)row.qh * a.p_s1 : a.acc + pr * D) + 4 * hh;
#pragma unroll
  for (int db = 0; db < D / 32; ++db) {
    if (direct) w.acc[db] *= inv;
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *(f4_any_t*)(dst + 32 * db + 8 * g) =
          f4_t{w.acc[db][4 * g], w.acc[db][4 * g + 1], w.acc[db][4 * g + 2], w.acc[db][4 * g + 3]};
  }
}

// The wave's rows as range z's partial ones in the workspace are: what write_rows left there.
template <int D, int NKB, bool QLO, bool PLO, bool VLO>
__device__ __forceinline__ void resume_rows(Rows<D, false, NKB, 2, QLO, PLO, VLO>& w, const PrefixArgs& a, int h, int r, int z, int hh) {
  const Row row = row_of(a, h, r);
  if (!row.live) return;
  const long pr = ((long)z * a.n + row.t) * a.hq + row.qh;
  const float2 ml = *(const float2*)(a.ml + 2 * pr);
  w.m = ml.x + w.kShift;
  w.l = hh == 0 ? ml.y : 0.f;  // the half-waves' shares are added at the end
  const float* src = a.acc + pr * D + 4 * hh;
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const f4_t x = *(const f4_any_t*)(src + 32 * db + 8 * g);
#pragma unroll
      for (int e = 0; e < 4; ++e) w.acc[db][4 * g + e] = x[e];
    }
}

// Decode: the lengths behind the prefix, for the kernels that follow.
__device__ __forceinline__ void write_suffix(const PrefixArgs& a) {
  if (!a.suffix) return;
  for (int t = (int)(blockIdx.x * blockDim.x + threadIdx.x); t < a.n; t += (int)(gridDim.x * blockDim.x)) {
    const long x = a.lens[t] - a.len;
    a.suffix[t] = x > 0 ? x : 0;
  }
}

}  // namespace

template <int D, bool QLO, int WAVES, bool PLO, bool VLO>
__global__ __launch_bounds__(64 * WAVES, D == 256 || (QLO && D == 128) ? 1 : 2) void prefix_kernel(PrefixArgs a) {
  static_assert(WAVES == 4 || WAVES == 8, "a thread takes its items' K and V, or one of them");
  constexpr bool BOTH = WAVES == 4;
  constexpr int KEYS = 8192 / D;           // keys per step: 256 items
  constexpr int NKB = KEYS >= 64 ? 2 : 1;  // 32-key blocks per softmax update
  using I = Items<D, KEYS, VLO>;
  constexpr int SIDE = I::SIDE;
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];

  write_suffix(a);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int j = lane & 31, hh = lane >> 5;
  // Heads fastest, then row tiles: those of one head and range run together and on one XCD
  // (with 8 heads), which reads the range's pages once.
  const int h = (int)(blockIdx.x % (unsigned)a.L.H), tile = (int)(blockIdx.x / (unsigned)a.L.H), z = blockIdx.y;
  const int k_begin = z * a.per, k_end = z == a.ranges - 1 ? a.len : min(a.len, k_begin + a.per);
  const int n_steps = k_end > k_begin ? (k_end - k_begin + KEYS - 1) / KEYS : 0;
  const bool keys = BOTH || wave < 4, values = BOTH || wave >= 4;  // wave-uniform
  const I it(a, h, k_begin, k_end, (int)threadIdx.x % 256);
  Raw raw;
  Head head{}, head1{};
  int blk2 = 0;
  if (n_steps > 0) {
    head = it.load_head(it.load_blk(0));
    head1 = it.load_head(it.load_blk(1));
    blk2 = it.load_blk(2);
    it.load(0, head, raw, keys, values, BOTH);
  }
  const int r = (tile * WAVES + wave) * 32 + j;
  const bool active = (tile * WAVES + wave) * 32 < (int)a.n * a.gqa;
  Rows<D, false, NKB, 2, QLO, PLO, VLO> w;
  load_query(w, a, row_of(a, h, r), hh);
  w.clear();
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)lds);
  const uint32_t k_lane = lds0 + k_at<D>(0, j, hh), v_lane = lds0 + 2 * SIDE + v_at<D>(0, lane);

  // The words of step `step` requested.
  auto fetch = [&](int step) __attribute__((always_inline)) {
    if (step >= n_steps) return;
    head = head1;
    it.load(step, head, raw, keys, values, BOTH);
    head1 = it.load_head(blk2);
    blk2 = it.load_blk(step + 2);
  };
  // Eight waves: two steps in LDS, the next one is written while this one is computed.
  if (!BOTH && n_steps > 0) {
    it.store(lds, 0, head, raw, keys, values, BOTH);
    fetch(1);
  }
  for (int step = 0; step < n_steps; ++step) {
    __syncthreads();  // every wave is done with the step before (eight waves: and this one is there)
    const int put = BOTH ? step : step + 1;
    const uint32_t buf = BOTH ? 0u : (uint32_t)((step & 1) * I::STEP);
    if (put < n_steps) {
      it.store(lds + (BOTH ? 0 : (put & 1) * I::STEP), put, head, raw, keys, values, BOTH);
      if (BOTH) __syncthreads();
      fetch(put + 1);
    }
    if (!active) continue;
#pragma unroll 1
    for (int sb = 0; sb < KEYS; sb += 32 * NKB) {
      const int left = k_end - (k_begin + step * KEYS + sb);  // keys of this block that there are
      if (left <= 0) break;
      f16v_t s[NKB];
      u4_t p[w.PW];
      w.template scores<SIDE>(k_lane + buf + sb * 2 * D, s);
      if (left < 32 * NKB) mask_tail<NKB>(s, left, hh);
      w.rescale(w.top(s));
      w.template weights<false, SIDE>(s, p, 0, s);
      w.template values<false, SIDE>(p, v_lane + buf + sb * 2 * D, s);
    }
  }
  write_rows(w, a, h, r, z, hh);
}

// Range z's keys: [begin, end).
__device__ __forceinline__ int range_begin(const PrefixArgs& a, int z) { return z * a.per; }
__device__ __forceinline__ int range_end(const PrefixArgs& a, int z) {
  return z == a.ranges - 1 ? a.len : min(a.len, (z + 1) * a.per);
}

// One workgroup per (64-key tile of the slab, KV head, range): its sides into the workspace. A range's
// tiles of the slab lie behind one another. Bound by memory: 64 registers, eight waves a SIMD.
template <int D, bool VLO>
__global__ __launch_bounds__(256, 8) void prefix_pack_kernel(PrefixArgs a) {
  using I = Items<D, kPackKeys, VLO>;
  write_suffix(a);
  const int h = (int)(blockIdx.x % (unsigned)a.L.H), tile = (int)(blockIdx.x / (unsigned)a.L.H);
  const int z = blockIdx.y, begin = range_begin(a, z) + a.slab * a.seg + tile * kPackKeys, end = range_end(a, z);
  if (begin >= end) return;
  const I it(a, h, begin, end - begin < kPackKeys ? end : begin + kPackKeys, (int)threadIdx.x);
  if (4 * it.quad >= kPackKeys) return;  // head size 64: half of the threads
  Raw raw;
  const Head head = it.load_head(it.load_blk(0));
  it.load(0, head, raw, true, true, true);
  it.store(a.pack + ((long)(z * (a.seg / kPackKeys) + tile) * a.L.H + h) * I::STEP, 0, head, raw, true, true, true);
}

template <int D, bool PLO, bool VLO>
__global__ __launch_bounds__(512, 2) void prefix_flash_kernel(PrefixArgs a) {
  constexpr int WAVES = 8, KEYS = kPackKeys, NKB = 2, SIDE = KEYS * D * 2;
  constexpr int VSIDE = (VLO ? 2 : 1) * SIDE, STEP = 2 * SIDE + VSIDE;
  constexpr int KDMA = 2 * SIDE / 1024 / WAVES, VDMA = VSIDE / 1024 / WAVES;
  // LDS: the keys (hi, lo) of two steps, then the values of two.
  constexpr int V0 = 4 * SIDE;
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int j = lane & 31, hh = lane >> 5;
  const int h = (int)(blockIdx.x % (unsigned)a.L.H), tile = (int)(blockIdx.x / (unsigned)a.L.H), z = blockIdx.y;
  const int k_begin = range_begin(a, z) + a.slab * a.seg, z_end = range_end(a, z);
  const int k_end = z_end - k_begin < a.seg ? z_end : k_begin + a.seg;  // this slab's keys of the range
  const int n_steps = k_end > k_begin ? (k_end - k_begin + KEYS - 1) / KEYS : 0;
  if (a.slab > 0 && n_steps == 0) return;  // the rows are as the slabs before left them
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)lds);
  const uint8_t* tiles = a.pack + ((long)z * (a.seg / KEYS) * a.L.H + h) * STEP;
  auto issue = [&](int step, bool val) __attribute__((always_inline)) {
    const int n = val ? VDMA : KDMA;
    const uint8_t* from = uniform_ptr(tiles + (long)step * a.L.H * STEP + (val ? 2 * SIDE : 0) + 1024 * n * wave);
    const uint32_t to = lds0 + (uint32_t)((val ? V0 + (step & 1) * VSIDE : (step & 1) * 2 * SIDE) + 1024 * n * wave);
#pragma unroll
    for (int i = 0; i < n; ++i) dma16(from, 1024 * i + 16 * lane, to + 1024 * i);
  };
  if (n_steps > 0) {
    issue(0, false);
    issue(0, true);
    if (n_steps > 1) issue(1, false);
  }
  const int r = (tile * WAVES + wave) * 32 + j;
  const bool active = (tile * WAVES + wave) * 32 < (int)a.n * a.gqa;
  Rows<D, false, NKB, 2, false, PLO, VLO> w;
  load_query(w, a, row_of(a, h, r), hh);
  w.clear();
  if (a.slab > 0) resume_rows<D>(w, a, h, r, z, hh);
  const uint32_t k_lane = lds0 + k_at<D>(0, j, hh), v_lane = lds0 + V0 + v_at<D>(0, lane);

  // As in prompt.hip: at `step` the keys of `step` + 1 and the values of `step` have landed.
  auto advance = [&](int step) __attribute__((always_inline)) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (step + 2 < n_steps) issue(step + 2, false);
    if (step + 1 < n_steps) issue(step + 1, true);
  };
  f16v_t s0[NKB], s1[NKB];
  float mt = -kInf;
  const int tail = (k_end - k_begin) % KEYS;
  auto body = [&](int step, f16v_t* cur, f16v_t* nxt) __attribute__((always_inline)) {
    advance(step);
    w.rescale(mt);
    u4_t p[w.PW];
    w.template weights<true, SIDE>(cur, p, k_lane + (uint32_t)(((step + 1) & 1) * 2 * SIDE), nxt);
    mt = w.template values<true, SIDE>(p, v_lane + (uint32_t)((step & 1) * VSIDE), nxt);
    if (tail && step + 2 == n_steps) {
      mask_tail<NKB>(nxt, tail, hh);
      mt = w.top(nxt);
    }
  };
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (active && n_steps > 0) {
    w.template scores<SIDE>(k_lane, s0);
    if (tail && n_steps == 1) mask_tail<NKB>(s0, tail, hh);
    mt = w.top(s0);
    int step = 0;
    for (; step + 2 < n_steps; step += 2) {
      body(step, s0, s1);
      body(step + 1, s1, s0);
    }
    if (step + 1 < n_steps) {
      body(step++, s0, s1);
      s0[0] = s1[0];
      s0[1] = s1[1];
    }
    advance(step);
    w.rescale(mt);
    u4_t p[w.PW];
    w.template weights<false, SIDE>(s0, p, 0, s0);
    w.template values<false, SIDE>(p, v_lane + (uint32_t)((step & 1) * VSIDE), s0);
  } else {
    for (int step = 0; step < n_steps; ++step) advance(step);
  }
  write_rows(w, a, h, r, z, hh);
}

template <int D, bool QLO, int WAVES, bool PLO, bool VLO>
static hipError_t launch_t(const PrefixArgs& a, hipStream_t s) {
  constexpr int lds = (WAVES == 8 ? 2 : 1) * Items<D, 8192 / D, VLO>::STEP;
  static std::atomic<uint64_t> attr_done{0};
  const hipError_t e = ensure_lds_limit((const void*)prefix_kernel<D, QLO, WAVES, PLO, VLO>, lds, &attr_done);
  if (e != hipSuccess) return e;
  constexpr int rows = 32 * WAVES;
  const dim3 grid((unsigned)((a.n * a.gqa + rows - 1) / rows * a.L.H), (unsigned)a.ranges);
  hipLaunchKernelGGL((prefix_kernel<D, QLO, WAVES, PLO, VLO>), grid, dim3(64 * WAVES), lds, s, a);
  return hipGetLastError();
}

template <int D, bool PLO, bool VLO>
static hipError_t launch_packed(const PrefixArgs& a, hipStream_t s) {
  constexpr int lds = (VLO ? 8 : 6) * kPackKeys * D * 2;
  static std::atomic<uint64_t> attr_done{0};
  hipError_t e = ensure_lds_limit((const void*)prefix_flash_kernel<D, PLO, VLO>, lds, &attr_done);
  if (e != hipSuccess) return e;
  const dim3 packs((unsigned)((long)(a.seg / kPackKeys) * a.L.H), (unsigned)a.ranges);
  const dim3 grid((unsigned)((a.n * a.gqa + 255) / 256 * a.L.H), (unsigned)a.ranges);
  PrefixArgs b = a;
  for (int from = 0; from < a.per; from += a.seg, ++b.slab) {
    hipLaunchKernelGGL((prefix_pack_kernel<D, VLO>), packs, dim3(256), 0, s, b);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    hipLaunchKernelGGL((prefix_flash_kernel<D, PLO, VLO>), grid, dim3(512), lds, s, b);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    b.suffix = nullptr;  // written by the first
  }
  return hipSuccess;
}

template <int D, bool PLO, bool VLO>
static hipError_t launch_16(const PrefixArgs& a, hipStream_t s) {
  if constexpr (D == 256) return launch_t<D, false, 4, PLO, VLO>(a, s);
  else if (a.pack) return launch_packed<D, PLO, VLO>(a, s);
  else if (prefix_rows(a.L.D, a.q_dtype, a.n * a.gqa, a.len) == 256) return launch_t<D, false, 8, PLO, VLO>(a, s);
  else return launch_t<D, false, 4, PLO, VLO>(a, s);
}

template <int D>
static hipError_t launch_d(const PrefixArgs& a, hipStream_t s) {
  if (a.q_dtype == ECHOKV_F32) {
    if constexpr (D == 256) return hipErrorInvalidValue;  // its registers do not fit: attend_any.hip
    else return a.exact ? launch_t<D, true, 4, true, true>(a, s) : launch_t<D, true, 4, true, false>(a, s);
  }
  if (a.exact) return launch_16<D, true, true>(a, s);
  return a.q_dtype == ECHOKV_F16 ? launch_16<D, true, false>(a, s) : launch_16<D, false, false>(a, s);
}

hipError_t launch_prefix(const PrefixArgs& a, hipStream_t s) {
  if (a.L.D == 64) return launch_d<64>(a, s);
  if (a.L.D == 128) return launch_d<128>(a, s);
  if (a.L.D == 256) return launch_d<256>(a, s);
  return hipErrorInvalidValue;
}

}  // namespace ek
