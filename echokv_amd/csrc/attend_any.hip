// Attention over whole prompts and over a shared cached prefix in 32-bit arithmetic, for
// any head size that is a multiple of 4 (up to 256), any types, strides and alignment.
//
// A workgroup holds 64 query rows ((token, GQA head) pairs of one KV head), 16 per wave. The
// keys come in steps of 32 (16 at head sizes above 128), staged in LDS as float32 -- from the
// prompt's own rows, or dequantized from the cache's pages -- and each wave runs
//   S^T[key, row] = K Q^T         (v_mfma_f32_16x16x4_f32)
//   O^T[d, row]  += V^T P^T       (v_mfma_f32_16x16x4_f32)
// with an online softmax per row. A contraction index may be permuted as long as both
// operands are: lane group c takes channels 16 j + 4 c .. + 4 of the score products (one
// 16-byte read each), and keys 4 c + i of the value products, which is where the S^T
// accumulator holds them, so P^T needs no exchange.
#include "items.h"

namespace ek {
namespace {

constexpr int kRows = 64;  // query rows per workgroup
constexpr float kInf = __builtin_inff();

template <int DP>
struct Steps {
  static constexpr int KEYS = DP > 128 ? 16 : 32;
  static constexpr int PITCH = DP + 4;  // floats per LDS row: 16 rows' 16-byte reads spread over the banks
  static constexpr int NKH = KEYS / 16, NJ = DP / 16;
};

__device__ __forceinline__ float rows_max(float x) {
  x = fmaxf(x, __shfl_xor(x, 16, 64));
  return fmaxf(x, __shfl_xor(x, 32, 64));
}

__device__ __forceinline__ bool finite4(const float* x) {
  // An exponent of all ones somewhere.
  uint32_t bad = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) bad |= (__float_as_uint(x[e]) & 0x7f800000u) == 0x7f800000u;
  return !bad;
}

// One wave's 16 rows: accumulators O^T (lane (n, c): row n, channels 16 j + 4 c + i), the
// running max (log2 units) and this lane's share of the sum.
template <int DP>
struct State {
  f4_t acc[Steps<DP>::NJ];
  float m, l;
  __device__ __forceinline__ void init() {
#pragma unroll
    for (int j = 0; j < Steps<DP>::NJ; ++j) acc[j] = f4_t{0.f, 0.f, 0.f, 0.f};
    m = -kInf;
    l = 0.f;
  }
};

// A step of KEYS staged keys, the first at position kb: a row sees keys below its `lim`.
// `odd`: a value of the step is infinite or NaN, which a weight of zero must not reach.
template <int DP>
__device__ __forceinline__ void step_any(State<DP>& st, const f4_t* q, const float* kt, const float* vt, int kb,
                                         int lim, bool odd, int lane) {
  using S = Steps<DP>;
  const int n = lane & 15, c = lane >> 4;
  f4_t s[S::NKH];
#pragma unroll
  for (int kh = 0; kh < S::NKH; ++kh) s[kh] = f4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < S::NJ; ++j) {
#pragma unroll
    for (int kh = 0; kh < S::NKH; ++kh) {
      const f4_t k = *(const f4_t*)&kt[(16 * kh + n) * S::PITCH + 16 * j + 4 * c];
#pragma unroll
      for (int e = 0; e < 4; ++e) s[kh] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[e], q[j][e], s[kh], 0, 0, 0);
    }
  }
  float mt = -kInf;
#pragma unroll
  for (int kh = 0; kh < S::NKH; ++kh)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float x = kb + 16 * kh + 4 * c + i < lim ? s[kh][i] : -kInf;
      s[kh][i] = x;
      mt = fmaxf(mt, x);
    }
  mt = rows_max(mt);
  if (mt > st.m) {
    const float alpha = __builtin_amdgcn_exp2f(st.m - mt);
    st.l *= alpha;
#pragma unroll
    for (int j = 0; j < S::NJ; ++j) st.acc[j] *= alpha;
    st.m = mt;
  }
  const float ms = st.m == -kInf ? 0.f : st.m;
#pragma unroll
  for (int kh = 0; kh < S::NKH; ++kh)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s[kh][i] = __builtin_amdgcn_exp2f(s[kh][i] - ms);
      st.l += s[kh][i];
    }
  if (!odd) {
#pragma unroll
    for (int j = 0; j < S::NJ; ++j)
#pragma unroll
      for (int kh = 0; kh < S::NKH; ++kh)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          st.acc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(vt[(16 * kh + 4 * c + i) * S::PITCH + 16 * j + n], s[kh][i],
                                                           st.acc[j], 0, 0, 0);
    return;
  }
  // Rare: key by key, only where the row sees the key.
#pragma unroll
  for (int kh = 0; kh < S::NKH; ++kh)
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll 1
      for (int g = 0; g < 4; ++g) {
        const int key = 16 * kh + 4 * g + i;
        const float p = __shfl(s[kh][i], 16 * g + n, 64);
        if (kb + key >= lim) continue;
#pragma unroll
        for (int j = 0; j < S::NJ; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            st.acc[j][e] = __builtin_fmaf(p, vt[key * S::PITCH + 16 * j + 4 * c + e], st.acc[j][e]);
      }
}

// The row's query, times the softmax scale in log2 units (zeros past the head).
template <int DP>
__device__ __forceinline__ void load_q(const void* q, int dtype, long at, int D, float scale, int c, f4_t* x) {
#pragma unroll
  for (int j = 0; j < Steps<DP>::NJ; ++j) {
    const int ch = 16 * j + 4 * c;
    float y[4] = {0.f, 0.f, 0.f, 0.f};
    if (ch < D) ld4(q, dtype, at + ch, y);
    x[j] = f4_t{y[0] * scale, y[1] * scale, y[2] * scale, y[3] * scale};
  }
}

}  // namespace

// One workgroup per (tile, 64 / GROUPS of its rows, KV head); heads fastest, then tiles (longest
// first) or, with two groups, the tile's parts. GROUPS 2: waves 2 and 3 take the same rows as 0 and
// 1, over the odd steps of keys.
//
// A step is a chain (its rows stored, two barriers, products that wait for one another) of about
// 3 us whatever runs beside it, so with few workgroups a wave's number of steps is the time: two
// groups halve it, and stage each key for 32 rows instead of 64. They are taken up to three
// workgroups (of 64 rows) a CU, one above head size 128, whose registers leave room for one. us
// with one group / with two, 8 KV heads of GQA 4, float32: D 96, 300 tokens (160 workgroups)
// 36 / 26, 100 + 400 + 700 tokens (624) 97 / 76, 2000 (1008) 316 / 366, 4000 (2000) 1165 / 1338;
// D 128, 300 (160) 43 / 31, 1000 (512) 186 / 132, 2000 (1008) 390 / 462; D 64 (4 of GQA 8), 1500
// (752) 157 / 139, 3000 (1504) 425 / 467; D 256 (2 of GQA 4), 1000 (128) 271 / 171, 2000 (252)
// 532 / 350, 4000 (500) 1110 / 1309.
// Bound by the chain, then by the float32 matrix rate: 4000 tokens at D 96 run at 84 TFLOP/s of
// causal products, a library product of 4096^3 at 132.
template <int DP, int GROUPS>
__global__ __launch_bounds__(256, DP > 128 ? 1 : 2) void prompt_any_kernel(PromptArgs a) {
  using S = Steps<DP>;
  constexpr int ROWS = kRows / GROUPS, KEYS = GROUPS * S::KEYS;
  __shared__ __attribute__((aligned(16))) float kv[2 * KEYS * S::PITCH];
  float *const kt = kv, *const vt = kv + KEYS * S::PITCH;
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, c = lane >> 4;
  const int h = (int)(blockIdx.x % a.H);
  const int parts = (a.tile_m * a.gqa + ROWS - 1) / ROWS, at_tile = (int)(blockIdx.x / a.H);
  const int tile = GROUPS == 1 ? at_tile % a.n_tiles : at_tile / parts;
  const int32_t* td = a.tiles + 4 * (long)tile;
  const long row0 = td[0];
  const int seq = td[1], t0 = td[2], n_rows = td[3] * a.gqa;
  const int first = (GROUPS == 1 ? at_tile / a.n_tiles : at_tile % parts) * ROWS;
  if (first >= n_rows) return;
  const int last = min(first + ROWS, n_rows) - 1;
  const int kv_end = min(seq, t0 + last / a.gqa + 1);  // keys that any row sees
  const int r = first + (16 * (tid >> 6) & (ROWS - 1)) + n, group = tid >> 6 >= ROWS / 16;
  const bool live = r < n_rows;
  const int tok = t0 + (live ? r / a.gqa : 0), qh = h * a.gqa + (live ? r % a.gqa : 0);
  const int lim = live ? tok + 1 : 0;
  f4_t q[S::NJ];
  load_q<DP>(a.q, a.dtype, (row0 + tok) * a.q_s0 + (long)qh * a.q_s1, a.D, a.scale_log2, c, q);
  State<DP> st;
  st.init();
  // A step's rows are requested while the one before is computed.
  constexpr int ITEMS = KEYS * (DP / 4), NI = (ITEMS + 255) / 256;
  float x[NI][4], y[NI][4];
  auto fetch = [&](int kb) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < NI; ++u) {
      const int i = tid + 256 * u, key = kb + i / (DP / 4), ch = 4 * (i % (DP / 4));
      const long row = row0 + min(key, kv_end - 1);
      const int c4 = ch < a.D ? ch : 0;
      ld4(a.k, a.dtype, row * a.k_s0 + (long)h * a.k_s1 + c4, x[u]);
      ld4(a.v, a.dtype, row * a.v_s0 + (long)h * a.v_s1 + c4, y[u]);
    }
  };
  fetch(0);
  for (int kb = 0; kb < kv_end; kb += KEYS) {
    __syncthreads();
    bool odd = false;
#pragma unroll
    for (int u = 0; u < NI; ++u) {
      const int i = tid + 256 * u, key = i / (DP / 4), ch = 4 * (i % (DP / 4));
      if (i >= ITEMS) break;
      const bool there = kb + key < kv_end && ch < a.D;
      odd = odd || (there && !finite4(y[u]));
      *(f4_t*)&kt[key * S::PITCH + ch] = there ? f4_t{x[u][0], x[u][1], x[u][2], x[u][3]} : f4_t{0.f, 0.f, 0.f, 0.f};
      *(f4_t*)&vt[key * S::PITCH + ch] = there ? f4_t{y[u][0], y[u][1], y[u][2], y[u][3]} : f4_t{0.f, 0.f, 0.f, 0.f};
    }
    const int any_odd = __syncthreads_or(odd);
    if (kb + KEYS < kv_end) fetch(kb + KEYS);
    const int at = group * S::KEYS;
    if (GROUPS == 1 || kb + at < kv_end)
      step_any<DP>(st, q, kt + at * S::PITCH, vt + at * S::PITCH, kb + at, lim, any_odd != 0, lane);
  }
  if constexpr (GROUPS == 2) {  // the groups' rows added
    constexpr int N = 4 * S::NJ;
    float* const x = kv + (tid >> 6 & 1) * 64 * (N + 2) + lane;
    __syncthreads();
    if (group) {
#pragma unroll
      for (int e = 0; e < N; ++e) x[64 * e] = st.acc[e >> 2][e & 3];
      x[64 * N] = st.m;
      x[64 * (N + 1)] = st.l;
    }
    __syncthreads();
    if (group) return;
    const float m1 = x[64 * N], top = fmaxf(st.m, m1);
    const float w0 = top == -kInf ? 1.f : __builtin_amdgcn_exp2f(st.m - top);
    const float w1 = top == -kInf ? 1.f : __builtin_amdgcn_exp2f(m1 - top);
#pragma unroll
    for (int e = 0; e < N; ++e) st.acc[e >> 2][e & 3] = st.acc[e >> 2][e & 3] * w0 + x[64 * e] * w1;
    st.m = top;
    st.l = st.l * w0 + x[64 * (N + 1)] * w1;
  }
  float l = st.l + __shfl_xor(st.l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  if (!live) return;
  const long row = row0 + tok, lr = row * a.hq + qh;
  float inv = l == 0.f ? 0.f : 1.f / l, lse = l == 0.f ? -kInf : st.m + __log2f(l), wp = 0.f;
  if (a.part) {
    const float pl = a.part_lse[lr], top = fmaxf(pl, lse);
    if (top != -kInf) {
      const float ep = __builtin_amdgcn_exp2f(pl - top), eo = __builtin_amdgcn_exp2f(lse - top), sum = ep + eo;
      wp = ep / sum;
      inv *= eo / sum;
      lse = top + __log2f(sum);
    }
  }
  if (a.lse && c == 0) a.lse[lr] = lse;
#pragma unroll
  for (int j = 0; j < S::NJ; ++j) {
    const int ch = 16 * j + 4 * c;
    if (ch >= a.D) continue;
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = st.acc[j][e] * inv;
    if (wp != 0.f) {
      const float* p = a.part + row * a.p_s0 + (long)qh * a.p_s1 + ch;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] += wp * p[e];
    }
    st_n<4>(a.out, a.out_dtype, row * a.o_s0 + (long)qh * a.o_s1 + ch, y);
  }
}

// One workgroup per (64 rows, KV head, range); heads fastest, then ranges.
template <int DP>
__global__ __launch_bounds__(256) void prefix_any_kernel(PrefixArgs a) {
  using S = Steps<DP>;
  __shared__ __attribute__((aligned(16))) float kt[S::KEYS * S::PITCH], vt[S::KEYS * S::PITCH];
  const Lay& L = a.L;
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, c = lane >> 4;
  if (a.suffix)
    for (long t = (long)blockIdx.x * 256 + tid; t < a.n; t += (long)gridDim.x * 256) {
      const long x = a.lens[t] - a.len;
      a.suffix[t] = x > 0 ? x : 0;
    }
  const int h = (int)(blockIdx.x % L.H);
  const int z = (int)(blockIdx.x / L.H % a.ranges);
  const long r = blockIdx.x / L.H / a.ranges * kRows + 16 * (tid >> 6) + n;
  const bool live = r < a.n * a.gqa;
  const long t = live ? r / a.gqa : 0;
  const int qh = h * a.gqa + (live ? (int)(r % a.gqa) : 0);
  // A sequence shorter than the prefix (graph padding): its row index may be any.
  const long q_row = a.lens && a.lens[t] < a.len ? 0 : a.q_rows ? a.q_rows[t] : t;
  const int k_begin = z * a.per, k_end = z == a.ranges - 1 ? a.len : min(a.len, k_begin + a.per);
  f4_t q[S::NJ];
  load_q<DP>(a.q, a.q_dtype, q_row * a.q_s0 + (long)qh * a.q_s1, L.D, a.scale_log2, c, q);
  State<DP> st;
  st.init();
  constexpr int OCTS = DP / 8;
  for (int kb = k_begin; kb < k_end; kb += S::KEYS) {
    __syncthreads();
    for (int i = tid; i < S::KEYS / 4 * OCTS; i += 256) {
      const int quad = i / OCTS, ch = 8 * (i % OCTS), kp = kb + 4 * quad;
      float x[4][8] = {}, y[4][8] = {};
      if (kp < k_end && ch < L.D) {
        const long blk = a.blocks[kp / L.BS];
        if (blk >= 0 && blk < L.nb) {
          const int off = kp % L.BS, live_keys = k_end - kp;
          const Hdr hd = load_hdr(a.pages, L, blk);
          const int bits = tier_of(hd.tag);
          const long rs = a.block_res[blk];
          const int rg = (unsigned long)rs < (unsigned long)a.res.rows ? (int)a.res_group[rs] : -1;
          item_general<true>(L, a.pages, a.res, blk, hd, rs, rg, off, bits, live_keys, h, ch, x);
          item_general<false>(L, a.pages, a.res, blk, hd, rs, rg, off, bits, live_keys, h, ch, y);
        }
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int at = (4 * quad + k) * S::PITCH + ch;
        *(f4_t*)&kt[at] = f4_t{x[k][0], x[k][1], x[k][2], x[k][3]};
        *(f4_t*)&kt[at + 4] = f4_t{x[k][4], x[k][5], x[k][6], x[k][7]};
        *(f4_t*)&vt[at] = f4_t{y[k][0], y[k][1], y[k][2], y[k][3]};
        *(f4_t*)&vt[at + 4] = f4_t{y[k][4], y[k][5], y[k][6], y[k][7]};
      }
    }
    __syncthreads();
    step_any<DP>(st, q, kt, vt, kb, k_end, false, lane);
  }
  float l = st.l + __shfl_xor(st.l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  if (!live) return;
  const bool direct = a.part != nullptr;
  const long pr = ((long)z * a.n + t) * a.hq + qh;
  const float inv = !direct ? 1.f : (l == 0.f ? 0.f : 1.f / l);
  if (c == 0) {
    if (direct) a.lse[q_row * a.hq + qh] = l == 0.f ? -kInf : st.m + __log2f(l);
    else *(float2*)(a.ml + 2 * pr) = float2{st.m, l};
  }
  float* dst = direct ? a.part + q_row * a.p_s0 + (long)qh * a.p_s1 : a.acc + pr * L.D;
#pragma unroll
  for (int j = 0; j < S::NJ; ++j) {
    const int ch = 16 * j + 4 * c;
    if (ch >= L.D) continue;
#pragma unroll
    for (int e = 0; e < 4; ++e) dst[ch + e] = st.acc[j][e] * inv;
  }
}

// One wave per (entry, query head): its prefix ranges, then its suffix splits, 64 pieces at a
// time, a group of rows requested while the one before is added (the kernel is a chain of
// round trips to memory). 2048 rows of 16 ranges and up to 4 splits take 7.0 us (21 MB, 3.0 TB/s),
// 19008 of 3 ranges 11 (40 MB, 3.6 TB/s). Lane l holds channels [C l, C l + C) where the head is 64 C channels
// (ANY false: one vector load a piece), else l, l + 64, ...
template <int C, bool ANY, int GROUP>
__global__ __launch_bounds__(256) void join_kernel(JoinArgs a) {
  typedef float vec_t __attribute__((ext_vector_type(C)));
  const int lane = threadIdx.x & 63;
  const long row = (long)blockIdx.x * 4 + (threadIdx.x >> 6);  // entry * hq + head
  if (row >= a.n * a.hq) return;
  const int t = (int)((unsigned)row / (unsigned)a.hq), qh = (int)row - t * a.hq, D = a.D;
  const long len = a.lens ? a.lens[t] : 0;
  int count = a.ranges;
  if (a.acc) {
    const int nb = ((int)a.suffix[t] + a.BS - 1) / a.BS;
    const int bps = split_blocks(a.sp, nb);
    count += nb > 0 ? (nb + bps - 1) / bps : 0;
  }
  // Piece i's row of its workspace.
  const long stride = a.n * a.hq, split0 = row * a.num_splits - a.ranges;
  auto at = [&](int i) { return i < a.ranges ? row + i * stride : split0 + i; };
  auto load = [&](int i0, int last, float (*y)[C]) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < GROUP; ++u) {
      const int i = min(i0 + u, last);
      const float* src = (i < a.ranges ? a.p_acc : a.acc) + at(i) * D;
      if constexpr (ANY) {
#pragma unroll
        for (int e = 0; e < C; ++e) y[u][e] = src[min(lane + 64 * e, D - 1)];
      } else {
        const vec_t v = *(const vec_t*)(src + C * lane);
#pragma unroll
        for (int e = 0; e < C; ++e) y[u][e] = v[e];
      }
    }
  };
  float m = -kInf, den = 0.f, o[C] = {};
  for (int p0 = 0; p0 < count; p0 += 64) {
    const int n = min(64, count - p0);
    float y[2][GROUP][C];
    float2 x = float2{-kInf, 0.f};
    if (lane < n) x = *(const float2*)((p0 + lane < a.ranges ? a.p_ml : a.ml) + 2 * at(p0 + lane));
    load(p0, p0 + n - 1, y[0]);
    float mt = x.x;
#pragma unroll
    for (int k = 32; k > 0; k >>= 1) mt = fmaxf(mt, __shfl_xor(mt, k, 64));
    const float top = fmaxf(m, mt);
    const float alpha = top == -kInf ? 1.f : __builtin_amdgcn_exp2f(m - top);
    const float w = x.x == -kInf ? 0.f : __builtin_amdgcn_exp2f(x.x - top);
    float d = w * x.y;
#pragma unroll
    for (int k = 32; k > 0; k >>= 1) d += __shfl_xor(d, k, 64);
    den = den * alpha + d;
#pragma unroll
    for (int e = 0; e < C; ++e) o[e] *= alpha;
    m = top;
    auto add = [&](int i0, float (*z)[C]) __attribute__((always_inline)) {
#pragma unroll
      for (int u = 0; u < GROUP; ++u) {
        if (i0 + u >= n) continue;
        const float wu = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), i0 + u));
        if (wu == 0.f) continue;  // an empty piece, whatever its row holds
#pragma unroll
        for (int e = 0; e < C; ++e) o[e] = __builtin_fmaf(wu, z[u][e], o[e]);
      }
    };
    for (int i0 = 0; i0 < n; i0 += 2 * GROUP) {
      if (i0 + GROUP < n) load(p0 + i0 + GROUP, p0 + n - 1, y[1]);
      add(i0, y[0]);
      if (i0 + 2 * GROUP < n) load(p0 + i0 + 2 * GROUP, p0 + n - 1, y[0]);
      if (i0 + GROUP < n) add(i0 + GROUP, y[1]);
    }
  }
  if (a.lens && len < a.len) return;
  const long q_row = a.q_rows ? a.q_rows[t] : t;
  const float inv = den == 0.f ? 0.f : 1.f / den;
  if (a.lse && lane == 0) a.lse[q_row * a.hq + qh] = den == 0.f ? -kInf : m + __log2f(den);
  const long ob = q_row * a.o_s0 + (long)qh * a.o_s1;
  if constexpr (ANY) {
#pragma unroll
    for (int e = 0; e < C; ++e)
      if (lane + 64 * e < D) st(a.out, a.out_dtype, ob + lane + 64 * e, o[e] * inv);
  } else {
#pragma unroll
    for (int e = 0; e < C; ++e) o[e] *= inv;
    st_n<C>(a.out, a.out_dtype, ob + C * lane, o);
  }
}

template <int GROUPS>
static hipError_t launch_prompt_any_t(const PromptArgs& a, hipStream_t s) {
  constexpr int rows = kRows / GROUPS;
  const dim3 grid((unsigned)((long)a.n_tiles * a.H * (((long)a.tile_m * a.gqa + rows - 1) / rows)));
  if (a.D <= 64) hipLaunchKernelGGL((prompt_any_kernel<64, GROUPS>), grid, dim3(256), 0, s, a);
  else if (a.D <= 96) hipLaunchKernelGGL((prompt_any_kernel<96, GROUPS>), grid, dim3(256), 0, s, a);
  else if (a.D <= 128) hipLaunchKernelGGL((prompt_any_kernel<128, GROUPS>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((prompt_any_kernel<256, GROUPS>), grid, dim3(256), 0, s, a);
  return hipGetLastError();
}

hipError_t launch_prompt_any(const PromptArgs& a, hipStream_t s) {
  const long wgs = (long)a.n_tiles * a.H * (((long)a.tile_m * a.gqa + kRows - 1) / kRows);
  return wgs <= (a.D <= 128 ? 3 * 256 : 256) ? launch_prompt_any_t<2>(a, s) : launch_prompt_any_t<1>(a, s);
}

hipError_t launch_prefix_any(const PrefixArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)((a.n * a.gqa + kRows - 1) / kRows * a.L.H * a.ranges));
  if (a.L.D <= 64) hipLaunchKernelGGL(prefix_any_kernel<64>, grid, dim3(256), 0, s, a);
  else if (a.L.D <= 96) hipLaunchKernelGGL(prefix_any_kernel<96>, grid, dim3(256), 0, s, a);
  else if (a.L.D <= 128) hipLaunchKernelGGL(prefix_any_kernel<128>, grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL(prefix_any_kernel<256>, grid, dim3(256), 0, s, a);
  return hipGetLastError();
}

template <int GROUP>
static hipError_t launch_join_t(const JoinArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)((a.n * a.hq + 3) / 4));
  if (a.D == 64) hipLaunchKernelGGL((join_kernel<1, false, GROUP>), grid, dim3(256), 0, s, a);
  else if (a.D == 128) hipLaunchKernelGGL((join_kernel<2, false, GROUP>), grid, dim3(256), 0, s, a);
  else if (a.D == 256) hipLaunchKernelGGL((join_kernel<4, false, GROUP>), grid, dim3(256), 0, s, a);
  else if (a.D < 128) hipLaunchKernelGGL((join_kernel<2, true, GROUP>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((join_kernel<4, true, GROUP>), grid, dim3(256), 0, s, a);
  return hipGetLastError();
}

// A group's rows past the last piece are that one again: up to four pieces are one group of four.
// us of a prefix_attention in groups of eight / four: 594 rows of 3 ranges (behind 2048 keys) 60.2 /
// 57.1, 900 of 2 (1024) 57.3 / 52.3, 1000 of 2 (2048) 80.8 / 76.3.
hipError_t launch_join(const JoinArgs& a, hipStream_t s) {
  const int most = a.ranges + (a.acc ? a.num_splits : 0);
  return most <= 4 ? launch_join_t<4>(a, s) : launch_join_t<8>(a, s);
}

}  // namespace ek
