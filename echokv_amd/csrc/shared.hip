// Attention of many query rows over one cached block list on 16-bit matrix instructions (head
// sizes 64, 128 and 256, layouts whose items sit in one group; attend_any.hip takes the others).
//
// One workgroup per (128 query rows, KV head, range of keys): 32 rows per wave, rows are (entry, GQA
// head) pairs, whatever sequence they belong to, so a key is dequantized once for 128 of them. A
// step of 8192 / D keys is dequantized into LDS, keys as a float16 hi + lo pair (2^-22 of the
// value together) and values in float16 (one rounding, as prefill.hip), and each wave runs S^T,
// an online softmax and O^T over it (tiles.h). A thread dequantizes one item of a step (four keys
// x eight channels of K and of V), its loads a chain spread over the steps: step i + 1's codes,
// i + 2's page header and i + 3's block id are requested before step i's products.
#include "items.h"
#include "tiles.h"

namespace ek {
namespace {

constexpr int kWaves = 4;
constexpr float kInf = __builtin_inff();

// An item's words: each row's eight codes in the 8 bytes at or before them.
struct Raw {
  uint2 k[4], v[4];
  uint4 ks, km;  // float16 scale / min of the eight channels (the quad's K group)
  uint16_t vs[4], vm[4];
  int rg;   // K group of the block's residual slot (if it has one)
  bool ok;  // the item's keys can be read
};

}  // namespace

template <int D, bool QLO, int WAVES>
__global__ __launch_bounds__(64 * WAVES, D == 256 || (QLO && D == 128) ? 1 : 2) void prefix_kernel(PrefixArgs a) {
  static_assert(WAVES == 4 || WAVES == 8, "a thread takes its items' K and V, or one of them");
  constexpr bool BOTH = WAVES == 4;
  constexpr int BUFS = BOTH ? 1 : 2;        // steps in LDS
  constexpr int ROWS = 32 * WAVES;
  constexpr int KEYS = 8192 / D;            // keys per step: 256 items
  constexpr int NKB = KEYS >= 64 ? 2 : 1;   // 32-key blocks per softmax update
  constexpr int NS = D / 16, NDB = D / 32, OCTS = D / 8;
  constexpr int SIDE = KEYS * D * 2;        // bytes of K hi, then K lo, then V
  constexpr float kShift = 6.f;             // weights are 2^6 times the softmax's: small ones keep their bits
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];

  const Lay& L = a.L;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int tid = threadIdx.x, j = lane & 31, hh = lane >> 5;
  if (a.suffix)
    for (int t = (int)blockIdx.x * 64 * WAVES + tid; t < a.n; t += (int)gridDim.x * 64 * WAVES) {
      const long x = a.lens[t] - a.len;
      a.suffix[t] = x > 0 ? x : 0;
    }
  // Heads fastest, then row tiles: those of one head and range run together and on one XCD
  // (with 8 heads), which reads the range's pages once.
  const int h = (int)(blockIdx.x % (unsigned)L.H), tile = (int)(blockIdx.x / (unsigned)L.H), z = blockIdx.y;
  const int n_rows = (int)a.n * a.gqa;  // below 2^25, checked on the host
  const int k_begin = z * a.per, k_end = z == a.ranges - 1 ? a.len : min(a.len, k_begin + a.per);
  const int n_steps = k_end > k_begin ? (k_end - k_begin + KEYS - 1) / KEYS : 0;

  // ---- this thread's item of a step, and its chain of loads ----------------
  const int oct = tid % OCTS, quad = tid % 256 / OCTS;
  const bool keys = BOTH || wave < 4, values = BOTH || wave >= 4;  // wave-uniform: what of the item this thread takes
  const int ch = 8 * oct;
  const int G = D / L.VG, vg = ch / L.VG;
  // Nothing loaded is looked at before the step that needs it, and no load sits in a
  // branch (addresses are clamped instead): the wave would wait for it there.
  auto item_key = [&](int step) { return k_begin + step * KEYS + 4 * quad; };
  auto item_off = [&](int step) { return item_key(step) & (L.BS - 1); };
  auto load_blk = [&](int step) -> int {
    const int kp = item_key(step);
    return a.blocks[(kp < k_end - 1 ? kp : k_end - 1) >> a.bs_shift];
  };
  struct Head {
    uint4 h;
    int blk, rs;  // rs: the low word (slots are small, -1: none)
  };
  auto page_of = [&](int blk) { return (unsigned)blk < (unsigned long)L.nb ? (long)blk : 0l; };
  auto load_head = [&](int blk) {
    const long b = page_of(blk);
    return Head{*(const uint4*)(a.pages + b * L.stride), blk, *(const int32_t*)(a.block_res + b)};
  };
  auto load_raw = [&](int step, const Head& x, Raw& w) {
    const int rs = (unsigned)x.rs < (unsigned)a.res.rows ? x.rs : 0;
    w.rg = *(const int32_t*)(a.res_group + rs);  // the low word: groups are small
    const int off = item_off(step), bits = tier_of(x.h.x & 0xffu);
    const int tpc_shift = a.bs_shift + 1 - (bits == 8 ? 3 : bits == 4 ? 2 : 1);
    const int c = off >> tpc_shift;
    long cb = page_of(x.blk) * L.stride + L.o_data;
    bool ok = (unsigned)x.blk < (unsigned long)L.nb && item_key(step) < k_end;
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
    // A quad that cannot be read takes its page's first bytes instead (dequantized to zero).
    const uint8_t* kp = ok ? a.pages + cb + (long)(off & ((1 << tpc_shift) - 1)) * rowb + ((h * D + ch) * bits / 8 & ~7) : pg;
    const int step_b = ok ? rowb : 0;
    if (keys) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w.k[i] = *(const uint2*)(kp + i * step_b);
      const int se = ((off >> a.kg_shift) * L.H + h) * D + ch;
      w.ks = *(const uint4*)(pg + L.o_ks + 2 * se);
      w.km = *(const uint4*)(pg + L.o_km + 2 * se);
    }
    if (values) {
      const int ve = (off * L.H + h) * G + vg;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        (BOTH ? w.v : w.k)[i] = *(const uint2*)(kp + i * step_b + step_b / 2);
        w.vs[i] = *(const uint16_t*)(pg + L.o_vs + 2 * (ve + i * L.H * G));
        w.vm[i] = *(const uint16_t*)(pg + L.o_vm + 2 * (ve + i * L.H * G));
      }
    }
  };
  // The item dequantized into LDS (keys past the range and blocks that cannot be read: zeros).
  auto store_item = [&](int step, const Head& x, const Raw& w) {
    uint8_t* const buf = lds + (BOTH ? 0 : (step & 1) * 3 * SIDE);
    const int kp = item_key(step), off = item_off(step), bits = tier_of(x.h.x & 0xffu);
    const int key0 = 4 * quad;
    auto put_k = [&](int i, const float* x8) {
      u4_t hi, lo;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const h2_t p = {(_Float16)x8[2 * e], (_Float16)x8[2 * e + 1]};
        hi[e] = __builtin_bit_cast(uint32_t, p);
        lo[e] = pack2<false>(x8[2 * e] - (float)p[0], x8[2 * e + 1] - (float)p[1]);
      }
      const int at = (key0 + i) * (2 * D) + 16 * (oct ^ k_swz<D>(key0 + i));
      *(u4_t*)(buf + at) = hi;
      *(u4_t*)(buf + SIDE + at) = lo;
    };
    auto put_v = [&](int i, const u4_t x) {
      *(u4_t*)(buf + 2 * SIDE + (key0 + i) * (2 * D) + 16 * (oct ^ v_swz<D>(key0 + i))) = x;
    };
    const int sh = 8 * (((h * D + ch) * bits / 8) & 7);
    auto rows = [&](auto width) {
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
          put_k(i, x8);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      if (values) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          h2_t c[4];
          code_pairs<B>((BOTH ? w.v : w.k)[i], sh, c);
          const h2_t vs = u2h(w.vs[i] * 0x10001u), vm = u2h(w.vm[i] * 0x10001u);
          u4_t v;
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(c[e], vs, vm));
          put_v(i, v);
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
        if (keys) put_k(i, z8);
        if (values) put_v(i, u4_t{});
      }
    }
    if (keys && w.ok && (unsigned)x.rs < (unsigned)a.res.rows && w.rg == off >> a.kg_shift) {  // rare: an open K group
#pragma unroll 1
      for (int i = 0; i < 4 && kp + i < k_end; ++i) {
        float x8[8];
        ld_n<8>(a.res.ptr, a.res.dtype,
                x.rs * a.res.s0 + (long)((off + i) & (L.KG - 1)) * a.res.s1 + h * a.res.s2 + ch, x8);
        put_k(i, x8);
      }
    }
  };

  Raw raw;
  Head head{}, head1{};
  int blk2 = 0;
  if (n_steps > 0) {
    head = load_head(load_blk(0));
    head1 = load_head(load_blk(1));
    blk2 = load_blk(2);
    load_raw(0, head, raw);
  }

  // ---- this lane's query row: 16 bytes at a time, all requested together ------
  struct Row {
    int t, qh;
    long q_row;
    bool live;
  };
  auto row_of = [&](int jj) {
    const int r = tile * ROWS + 32 * wave + jj;
    const bool live = r < n_rows;
    const int t = live ? (int)((unsigned)r / (unsigned)a.gqa) : 0;
    return Row{t, h * a.gqa + (live ? r - t * a.gqa : 0), a.q_rows ? a.q_rows[t] : t, live};
  };
  const bool active = tile * ROWS + 32 * wave < n_rows;
  // As in prompt.hip: the scale positive.
  constexpr float kTiny = 7.8886090522101181e-31f;
  const float scale = fabsf(a.scale_log2) < kTiny ? kTiny : fabsf(a.scale_log2);
  h8_t q[NS], ql[QLO ? NS : 1];
  {
    const Row row = row_of(j);
    const uint8_t* src = (const uint8_t*)a.q + (row.q_row * a.q_s0 + (long)row.qh * a.q_s1 + 8 * hh) * (QLO ? 4 : 2);
    const uint32_t flip = a.scale_log2 < 0.f ? (QLO ? 0x80000000u : 0x80008000u) : 0u;
    u4_t w[NS][QLO ? 2 : 1];
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int i = 0; i < (QLO ? 2 : 1); ++i) w[s][i] = *(const u4_any_t*)(src + 32 * (QLO ? 2 : 1) * s + 16 * i) ^ flip;
    const bool bf = a.q_dtype == ECHOKV_BF16;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      if constexpr (QLO) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x = __uint_as_float(w[s][e >> 2][e & 3]);
          q[s][e] = (_Float16)x;
          ql[s][e] = (_Float16)(x - (float)q[s][e]);
        }
      } else {
        u4_t y;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          y[e] = pack2<false>(__uint_as_float(w[s][0][e] << 16), __uint_as_float(w[s][0][e] & 0xffff0000u));
        q[s] = __builtin_bit_cast(h8_t, bf ? y : w[s][0]);
      }
    }
  }

  f16v_t acc[NDB];
#pragma unroll
  for (int db = 0; db < NDB; ++db) acc[db] = f16v_t{};
  float m_run = -kInf, lsum = 0.f;
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)lds);
  // Slots are permuted by exclusive or, and LDS rows are whole multiples of their slots: a
  // fragment's address is the first one's with the slot's bits flipped.
  const uint32_t k_lane = lds0 + k_at<D>(0, j, hh), v_lane = lds0 + 2 * SIDE + v_at<D>(0, lane);

  // An item into LDS, then the words of the next one requested.
  auto put_step = [&](int step) {
    store_item(step, head, raw);
    if (step + 1 < n_steps) {
      head = head1;
      load_raw(step + 1, head, raw);
      head1 = load_head(blk2);
      blk2 = load_blk(step + 3);
    }
  };
  if (!BOTH && n_steps > 0) put_step(0);
  for (int step = 0; step < n_steps; ++step) {
    __syncthreads();  // every wave is done with the step before (eight waves: and this one is there)
    if constexpr (BOTH) {
      store_item(step, head, raw);
      __syncthreads();
      if (step + 1 < n_steps) {
        head = head1;
        load_raw(step + 1, head, raw);
        head1 = load_head(blk2);
        blk2 = load_blk(step + 3);
      }
    } else if (step + 1 < n_steps) {
      put_step(step + 1);
    }
    if (!active) continue;
    const uint32_t buf = BOTH ? 0u : (uint32_t)((step & 1) * 3 * SIDE);
#pragma unroll 1
    for (int sb = 0; sb < KEYS; sb += 32 * NKB) {
      const int left = k_end - (k_begin + step * KEYS + sb);  // keys of this block that there are
      if (left <= 0) break;
      f16v_t s[NKB];
#pragma unroll
      for (int kb = 0; kb < NKB; ++kb) s[kb] = f16v_t{};
      {
        h8_t f[2][NKB];
        auto load = [&](int u, h8_t* x) {  // channels 16 (u / 2) .. + 16 of K hi or lo
#pragma unroll
          for (int kb = 0; kb < NKB; ++kb)
            x[kb] = k_read<D>((k_lane ^ 32 * (u >> 1)) + (u & 1) * SIDE + buf + sb * 2 * D, kb);
        };
        load(0, f[0]);
#pragma unroll
        for (int u = 0; u < 2 * NS; ++u) {
          if (u + 1 < 2 * NS) load(u + 1, f[(u + 1) & 1]);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int kb = 0; kb < NKB; ++kb) s[kb] = mma<false>(f[u & 1][kb], q[u >> 1], s[kb]);
          if constexpr (QLO) {
            if (!(u & 1)) {
#pragma unroll
              for (int kb = 0; kb < NKB; ++kb) s[kb] = mma<false>(f[u & 1][kb], ql[u >> 1], s[kb]);
            }
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      if (left < 32 * NKB) {
        int mine = left - 4 * hh;
        asm volatile("" : "+v"(mine));  // keeps the 32 compares in this branch
#pragma unroll
        for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
          for (int i = 0; i < 16; ++i) s[kb][i] = 32 * kb + 8 * (i >> 2) + (i & 3) < mine ? s[kb][i] : -kInf;
      }
      float mx = -kInf;
#pragma unroll
      for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[kb][i]);
      const float mt = halves_max(mx) * scale;
      if (__builtin_amdgcn_ballot_w64(mt > m_run + 8.f)) {  // weights stay below 2^8 x 2^6
        const float m_new = fmaxf(m_run, mt);
        const float alpha = m_new == -kInf ? 1.f : __builtin_amdgcn_exp2f(m_run - m_new);
        lsum *= alpha;
#pragma unroll
        for (int db = 0; db < NDB; ++db) acc[db] *= alpha;
        m_run = m_new;
      }
      const float ms = m_run == -kInf ? 0.f : m_run - kShift;
      float sum[2] = {0.f, 0.f};
      u4_t p[2 * NKB];
#pragma unroll
      for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][i], scale, -ms));
          const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][i + 1], scale, -ms));
          sum[0] += x;
          sum[1] += y;
          p[2 * kb + (i >> 3)][(i & 7) >> 1] = pack2<false>(x, y);
        }
      lsum += sum[0] + sum[1];
      {
        constexpr int NG = NDB < 4 ? NDB : 4, NP = NDB / NG;
        h8_t f[2][NG];
        auto load = [&](int g, h8_t* x) {
#pragma unroll
          for (int i = 0; i < NG; ++i) x[i] = v_read<D>((v_lane ^ 64 * (g % NP * NG + i)) + buf + sb * 2 * D, g / NP);
        };
        load(0, f[0]);
#pragma unroll
        for (int g = 0; g < 2 * NKB * NP; ++g) {
          if (g + 1 < 2 * NKB * NP) load(g + 1, f[(g + 1) & 1]);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int i = 0; i < NG; ++i) {
            const int db = g % NP * NG + i;
            acc[db] = mma<false>(f[g & 1][i], __builtin_bit_cast(h8_t, p[g / NP]), acc[db]);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
  }

  const float l = halves_sum(lsum);
  int jj = j;
  asm volatile("" : "+v"(jj));  // the row's place is found again, not kept through the loop
  const auto [t, qh, q_row, live] = row_of(jj);
  if (!live) return;
  const bool direct = a.part != nullptr;
  const long pr = ((long)z * a.n + t) * a.hq + qh;
  if (hh == 0) {
    if (direct) a.lse[q_row * a.hq + qh] = l == 0.f ? -kInf : m_run - kShift + __log2f(l);
    else *(float2*)(a.ml + 2 * pr) = float2{m_run - kShift, l};
  }
  const float inv = !direct ? 1.f : l == 0.f ? 0.f : 1.f / l;
  float* dst = (direct ? a.part + q_row * a.p_s0 + (long)qh * a.p_s1 : a.acc + pr * D) + 4 * hh;
#pragma unroll
  for (int db = 0; db < NDB; ++db) {
    if (direct) acc[db] *= inv;
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *(f4_any_t*)(dst + 32 * db + 8 * g) = f4_t{acc[db][4 * g], acc[db][4 * g + 1], acc[db][4 * g + 2], acc[db][4 * g + 3]};
  }
}

template <int D, bool QLO, int WAVES>
static hipError_t launch_t(const PrefixArgs& a, hipStream_t s) {
  constexpr int lds = (WAVES == 8 ? 2 : 1) * 3 * 8192 * 2;
  static std::atomic<uint64_t> attr_done{0};
  const hipError_t e = ensure_lds_limit((const void*)prefix_kernel<D, QLO, WAVES>, lds, &attr_done);
  if (e != hipSuccess) return e;
  constexpr int rows = 32 * WAVES;
  const dim3 grid((unsigned)((a.n * a.gqa + rows - 1) / rows * a.L.H), (unsigned)a.ranges);
  hipLaunchKernelGGL((prefix_kernel<D, QLO, WAVES>), grid, dim3(64 * WAVES), lds, s, a);
  return hipGetLastError();
}

template <int D>
static hipError_t launch_d(const PrefixArgs& a, hipStream_t s) {
  if (a.q_dtype == ECHOKV_F32) {
    if constexpr (D == 256) return hipErrorInvalidValue;  // its registers do not fit: attend_any.hip
    else return launch_t<D, true, 4>(a, s);
  }
  if constexpr (D == 256) return launch_t<D, false, 4>(a, s);
  else return prefix_rows(a.L.D, a.q_dtype, a.n * a.gqa) == 256 ? launch_t<D, false, 8>(a, s) : launch_t<D, false, 4>(a, s);
}

hipError_t launch_prefix(const PrefixArgs& a, hipStream_t s) {
  if (a.L.D == 64) return launch_d<64>(a, s);
  if (a.L.D == 128) return launch_d<128>(a, s);
  if (a.L.D == 256) return launch_d<256>(a, s);
  return hipErrorInvalidValue;
}

}  // namespace ek
