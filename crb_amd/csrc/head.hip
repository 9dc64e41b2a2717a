// Losses of a causal LM's output head over a large vocabulary, on MFMA, with
// their gradients and without keeping the logits.  (No counterpart in the
// reference, whose perplexity computes all logits and calls a cross
// entropy, eval_ppl_utils.py:626-636.)
//
// With z[t][v] = s sum_c h[t][c] W[v][c] and S_t the tokens listed for row t
// (cross entropy: its label, with probability 1; distillation: the teacher's
// k largest, with probabilities p and, optionally, a tail of probability
// p_T that stands for all other tokens together):
//   a_t    = log sum_{v not in S_t} exp z[t][v]
//   lse_t  = log(exp a_t + sum_{S_t} exp z[t][v])
//   loss_t = sum_{S_t} p_v (log p_v - z[t][v] + lse_t) + p_T (log p_T - a_t + lse_t)
// (a token listed twice: both entries' terms in the loss, its p_v in the
// gradient their sum),
// and with q_v = exp(z_v - lse), q_T = exp(a - lse):
//   dloss_t/dz_v = m q_v - p_v                   v in S_t (cross entropy: -q_T)
//                = (m q_T - p_T) exp(z_v - a)    otherwise
// where m = sum p + p_T: 1, unless the teacher's numbers do not add up.
// The sum a_t leaves the listed tokens out from the start, so that neither
// a confident row's loss nor its gradient is a difference of nearly equal
// numbers.
//
// Forward: one product over tiles of vocabulary x tokens whose epilogue
// keeps, per token, the running maximum and sum of exponentials of the tile
// (fp32) and the listed tokens' own z; a second kernel joins the tiles.
// Backward: per piece of the vocabulary, the product again with an epilogue
// that writes the piece's dz (16 bits, the operand of the two products that
// follow), then dh += dz W (fp32 sums) and dW = dz^T h.  dz is
// rounded to the inputs' type as the gradients themselves are: its error (at most 2^-8 or
// 2^-11 of it, independent from element to element) is that of the final rounding
// again.  Up to 64 tokens, where few elements of dz may make up a gradient and
// the products wait for memory anyway, a second 16-bit part holds what the rounding
// left (relative 2^-16).  dz is scaled by a power of two (fp16) and by the
// largest row coefficient so that it stays in range.
//
// The logits are computed twice, 4/3 of the operations that a step on kept logits
// has: keeping them (525 MB for 2047 x 128256 in 16 bits, 1 GB in 32) would save a product of
// 1.5 ms there, at the price of that memory from the forward pass to the
// backward pass and of 16-bit logits in the gradient.
//
// Measured (one MI355X, bf16 unless said otherwise; us, in brackets the TF of 2 T V C):
//   product, T x V x C                 forward       dz            dh            dW
//   2047 x 128256 x 4096               1550 (1390)   1670 (1290)   1530 (1400)   1815 (1185)
//   2047 x 50272 x 4096 fp16, 128 listed  760 (1110)   749 (1125)    645 (1310)    766 (1100)
//   2047 x 50272 x 768                 160           182           132           177
//   333 x 32007 x 1000                 32            36            37            36
//   250 x 50272 x 768, 20 listed       30            30            34            39
//   17 x 50272 x 2048 fp16, 64 listed  32            (206 MB of W at 6.3 TB/s, part of it cached)
//   1 x 128256 x 4096                  167 - 300     167 - 209     188           288
// The range of one token: W (1 GB) just read, or just pushed out of the caches by dW.
// The products of many tokens at 4096 channels: MFMAs busy 76, 72, 80 and 64 % of the
// time at 1.6 to 1.85 GHz; at 768, 55, 45, 71 and 61 %.
#include "gemm16.h"

namespace crbq {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;
constexpr int PAD_IDX = 0x7fffffff;     // an empty slot of a row's list

template <typename T8> struct Half;
template <> struct Half<h8_t> { typedef _Float16 t; };
template <> struct Half<b8_t> { typedef __bf16 t; };
template <typename T8>
__device__ __forceinline__ uint16_t to16(float x) {
  return __builtin_bit_cast(uint16_t, (typename Half<T8>::t)x);
}
// dz is kept times this: |dz| <= 1, below fp16's 65504 with room
template <typename T8>
constexpr float dz_scale() { return __is_same(T8, h8_t) ? 16384.f : 1.f; }

// lanes that differ in bits 4 and 5 (the four 16-lane groups): max and sum
__device__ __forceinline__ float gmax4(float v) {
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float gsum4(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

// (m, s): maximum and sum of 2^(x - m); joins two such pairs
__device__ __forceinline__ void ms_join(float& m, float& s, float m2, float s2) {
  const float mm = fmaxf(m, m2);
  const float x = m == mm ? s : s * __builtin_amdgcn_exp2f(m - mm);   // m = -inf = mm: s is 0
  const float y = m2 == mm ? s2 : s2 * __builtin_amdgcn_exp2f(m2 - mm);
  m = mm;
  s = x + y;
}
// log(exp a + exp b)
__device__ __forceinline__ float log_add(float a, float b) {
  const float m = fmaxf(a, b), d = -fabsf(a - b);
  return m == -INFINITY ? m : (d == d ? m + log1pf(expf(d)) : a + b);
}

// Where the listed tokens of the rows are (forward).
struct Listed {
  const int64_t* labels;   // cross entropy: one per row
  const uint32_t* mask;    // distillation: a bit per (row, token), 8 words a tile of 256,
  const int32_t* base;     //   and the row's listed tokens before each tile: a token's slot in
  int64_t ntile;           //   the row's ascending list is that plus the bits before its own
  int k;
};
// the bits of words before word w
__device__ __forceinline__ int bits_before(const uint32_t (&w)[8], int n) {
  int c = 0;
#pragma unroll
  for (int q = 0; q < 8; ++q) c += q < n ? __popc(w[q]) : 0;
  return c;
}

// ---------------------------------------------------------------------------
// forward product: partial (max, sum) of every (row, tile row of wavefronts)
// and the listed tokens' z
// ---------------------------------------------------------------------------
struct FwdArgs {
  const uint16_t *h, *W;
  int64_t ldh, ldw, T, V, C;
  float scale;
  Listed ls;
  int nm, nn;
  float2* part;
  int64_t npart;
  float* zt;
};

// Column t (n) of a wavefront's tile, MI times 16 tokens, the i-th 16 of them
// from v0 + off(i) on: listed tokens and what lies behind the vocabulary
// become -inf (the listed ones' z is written), then the maximum and the sum
// of exponentials.  lab: the label's place behind v0; words: each i's 16 mask
// bits; slots(s): s[q] = the slot of the first token of words[q].
// In units of log 2: exp z = 2^(acc * scale2), so an exponential is one
// multiply-add and one v_exp; the listed tokens and the end are looked for
// only where a wavefront has any.  Bound by the v_exp (16 cycles a wavefront)
// and the 2 to 3 vector operations beside each.
template <int MI, int NJ, bool XENT, int j, typename Off, typename Slots>
__device__ __forceinline__ void fwd_column(const FwdArgs& p, int64_t t, int64_t v0, Off off,
                                           int lab, const uint32_t (&words)[(MI + 1) / 2],
                                           const Slots& slots, f4_t (&acc)[MI][NJ], float2* out) {
  const int lane = g_lane(), g4 = (lane >> 4) * 4;
  const bool ok = t < p.T;
  bool any;
  if (XENT) {
    any = lab >= 0;
  } else {
    uint32_t w = 0;
#pragma unroll
    for (int q = 0; q < (MI + 1) / 2; ++q) w |= words[q];
    any = w != 0;
  }
  const float fin = p.scale < 0.f ? INFINITY : -INFINITY;        // scale * fin = -inf
  if (__any(any)) {
    int slot[(MI + 1) / 2] = {};
    if (!XENT) slots(slot);
    g_each<MI>([&](auto ii) __attribute__((always_inline)) {
      constexpr int i = decltype(ii)::value;
      const int o = off(i) + g4;
      const uint32_t nib = XENT ? (uint32_t)(lab >> 2 == o >> 2)
                                : (words[i / 2] >> (16 * (i & 1) + g4)) & 15u;
      if (nib)
        g_each<4>([&](auto rr) __attribute__((always_inline)) {
          constexpr int r = decltype(rr)::value;
          if (XENT ? o + r == lab : (nib >> r) & 1u) {
            const int bit = 16 * (i & 1) + g4 + r;     // of words[i / 2]
            p.zt[XENT ? t : t * p.ls.k + slot[i / 2] + __popc(words[i / 2] & ((1u << bit) - 1))] =
                acc[i][j][r] * p.scale;
            acc[i][j][r] = fin;
          }
        });
    });
  }
  if (v0 + off(MI - 1) + 16 > p.V) {
    const int end = (int)(p.V - v0);
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (off(i) + g4 + r >= end) acc[i][j][r] = fin;
  }
  const float scale2 = p.scale * LOG2E;
  float m = fin;
  if (p.scale < 0.f) {
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) m = fminf(m, acc[i][j][r]);
  } else {
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) m = fmaxf(m, acc[i][j][r]);
  }
  m = gmax4(m * scale2);
  const float mb = m == -INFINITY ? 0.f : m;           // nothing left: 2^-inf = 0
  float s[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      s[r & 1] += __builtin_amdgcn_exp2f(__builtin_fmaf(acc[i][j][r], scale2, -mb));
  const float sum = gsum4(s[0] + s[1]);
  if (ok && lane < 16) *out = make_float2(m, sum);
}

// Few tokens or few tiles: one tile of 256 tokens of the vocabulary a workgroup, 4 stages of
// the weight in LDS, 3 of them in flight: bound by reading W.
template <typename T8, typename G, bool XENT>
__global__ __launch_bounds__(G::THREADS) void k_head_fwd(const FwdArgs p) {
  __shared__ __attribute__((aligned(1024))) char smem[G::LDS];
  int tm, tn;
  g_band(g_xcd(blockIdx.x, gridDim.x), p.nm, p.nn, tm, tn);
  const int64_t v0 = (int64_t)tm * G::BM, t0 = (int64_t)tn * G::BN;
  const GOperand A{p.W + v0 * p.ldw, p.ldw, G_K, p.V - v0, p.C, nullptr};
  const GOperand B{p.h + t0 * p.ldh, p.ldh, G_K, p.T - t0, p.C, nullptr};
  f4_t acc[G::MI][G::NJ];
  g_tile<T8, G>(smem, A, B, 0, p.C, acc);
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int wr = wave / G::WGN;
  const int64_t vw = v0 + wr * G::WM;                  // the wavefront's first token
  g_each<G::NJ>([&](auto jj) __attribute__((always_inline)) {
    constexpr int j = decltype(jj)::value;
    const int64_t t = t0 + (wave % G::WGN) * G::WN + 16 * j + (lane & 15);
    const bool ok = t < p.T;
    int lab = -1;                                      // the label's place among the wavefront's
    uint32_t words[G::WM / 32] = {}, all[8] = {};
    if (XENT) {
      const int64_t y = ok ? p.ls.labels[t] : -1;
      lab = y >= vw && y < vw + G::WM ? (int)(y - vw) : -1;
    } else if (ok) {
      const uint4* w = (const uint4*)(p.ls.mask + (t * p.ls.ntile + tm) * 8);
      const uint4 a = w[0], b = w[1];
      all[0] = a.x; all[1] = a.y; all[2] = a.z; all[3] = a.w;
      all[4] = b.x; all[5] = b.y; all[6] = b.z; all[7] = b.w;
#pragma unroll
      for (int q = 0; q < 8; ++q)
#pragma unroll
        for (int e = 0; e < G::WM / 32; ++e)
          if (q == wr * (G::WM / 32) + e) words[e] = all[q];
    }
    auto slots = [&](int (&slot)[G::WM / 32]) __attribute__((always_inline)) {
      const int base = ok ? p.ls.base[t * p.ls.ntile + tm] : 0;
#pragma unroll
      for (int q = 0; q < G::WM / 32; ++q) slot[q] = base + bits_before(all, wr * (G::WM / 32) + q);
    };
    fwd_column<G::MI, G::NJ, XENT, j>(
        p, t, vw, [](int i) { return 16 * i; }, lab, words, slots, acc,
        p.part + t * p.npart + (int64_t)tm * G::WGM + wr);
  });
}

// Many tokens: persistent workgroups on 256 x 256 tiles (gemm16.h).  Bound by the MFMAs at
// the clock that their power leaves; the epilogue, 5 to 6 us of a tile's 100 at C = 4096
// and a quarter of the time at C = 768, runs while the next tile's first loads arrive.
template <bool XENT>
struct FwdJob {
  static constexpr bool MASKED = false;
  __device__ static int64_t lda() { return g_args<FwdArgs>().ldw; }
  __device__ static int64_t ldb() { return g_args<FwdArgs>().ldh; }
  __device__ static int64_t kstep_a() { return G_K; }
  __device__ static int64_t kstep_b() { return G_K; }
  __device__ static int64_t unit_a() { return G_K * lda(); }
  __device__ static int64_t unit_b() { return G_K * ldb(); }
  __device__ static int tiles() {
    const FwdArgs p = g_args<FwdArgs>();
    return p.nm * p.nn;
  }
  __device__ __forceinline__ static void place(const FwdArgs& p, int lin, int64_t& v0,
                                               int64_t& t0, int& tm) {
    int tn;
    g_band(lin, p.nm, p.nn, tm, tn);
    v0 = (int64_t)tm * 256;
    t0 = (int64_t)tn * 256;
  }
  __device__ static int stages(int) { return (int)((g_args<FwdArgs>().C + G_K - 1) / G_K); }
  __device__ __forceinline__ void tile(int lin, GOperand& A, GOperand& B, int64_t& k,
                                       int& nch) const {
    const FwdArgs p = g_args<FwdArgs>();
    int64_t v0, t0;
    int tm;
    place(p, lin, v0, t0, tm);
    A = GOperand{p.W + v0 * p.ldw, p.ldw, G_K, p.V - v0, p.C, nullptr};
    B = GOperand{p.h + t0 * p.ldh, p.ldh, G_K, p.T - t0, p.C, nullptr};
    k = 0;
    nch = stages(lin);
  }
  // the labels (or the tile's 8 mask words) of the wavefront's 2 x 32 rows
  __device__ __forceinline__ void side(int lin, char* priv) const {
    const FwdArgs p = g_args<FwdArgs>();
    int64_t v0, t0;
    int tm;
    place(p, lin, v0, t0, tm);
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int64_t t = t0 + 128 * b + 32 * (wave & 3), left = p.T - t;
      if (XENT) {
        g_load_lds_words(priv + 256 * b, p.ls.labels + t, left * 8, lane);
      } else {
        const int64_t rows = left < 32 ? left : 32;
        g_load_lds(priv + 1024 * b,
                   g_rsrc((const uint16_t*)(p.ls.mask + (t * p.ls.ntile + tm) * 8),
                          rows > 0 ? ((rows - 1) * p.ls.ntile + 1) * 32 : 0),
                   (unsigned)((lane >> 1) * p.ls.ntile * 32 + (lane & 1) * 16));
        g_load_lds_word(priv + 2048 + 256 * b,
                        g_rsrc((const uint16_t*)(p.ls.base + t * p.ls.ntile + tm),
                               rows > 0 ? ((rows - 1) * p.ls.ntile + 1) * 4 : 0),
                        (unsigned)(lane * p.ls.ntile * 4));      // (lanes behind the 32 rows: 0)
      }
    }
  }
  __device__ __forceinline__ void finish(int lin, char* priv, GAcc& acc) const {
    const FwdArgs p = g_args<FwdArgs>();
    int64_t v0, t0;
    int tm;
    place(p, lin, v0, t0, tm);
    const int lane = g_lane();
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int wr = wave >> 2;
    g_each<4>([&](auto jj) __attribute__((always_inline)) {
      constexpr int j = decltype(jj)::value;
      const int64_t t = t0 + g_n(j, wave, lane);
      const int row = 16 * (j & 1) + (lane & 15);      // of 32
      int lab = -1;
      uint32_t words[4] = {};
      if (XENT) {
        const int64_t y = ((const int64_t*)(priv + 256 * (j >> 1)))[row];
        lab = t < p.T && y >= v0 && y < v0 + 256 ? (int)(y - v0) : -1;
      } else {
        const uint32_t* w = (const uint32_t*)(priv + 1024 * (j >> 1)) + row * 8 + wr;
#pragma unroll
        for (int q = 0; q < 4; ++q) words[q] = w[2 * q];
      }
      // (the words between are the other wavefront's: all four read at once)
      auto slots = [&](int (&slot)[4]) __attribute__((always_inline)) {
        const uint32_t* w = (const uint32_t*)(priv + 1024 * (j >> 1)) + row * 8 + (wr ^ 1);
        int c = ((const int*)(priv + 2048 + 256 * (j >> 1)))[row];
        uint32_t o[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) o[q] = w[2 * q];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int between = __popc(o[q]);
          slot[q] = c + (wr ? between : 0);
          c += between + __popc(words[q]);
        }
      };
      fwd_column<8, 4, XENT, j>(
          p, t, v0, [&](int i) { return 64 * (i >> 1) + 32 * wr + 16 * (i & 1); }, lab, words,
          slots, acc.v, p.part + t * p.npart + (int64_t)tm * 2 + wr);
    });
  }
};

template <typename T8, bool XENT>
__global__ __launch_bounds__(G_THREADS) void k_head_fwd_p(const FwdArgs) {
  __shared__ __attribute__((aligned(1024))) char smem[G_LDS];
  g_run<T8, G_KC, G_KC>(smem, FwdJob<XENT>());
}

// The saved state of a forward: live rows (a bit each, 64-bit words), one
// factor (1, or 1 / the rows a mean is over) and one float unused; per row a,
// lse, the factor of exp(z - a) in dz and the row's weight there (both times
// dz_scale; 0 for a row left out); then cross entropy: z of the label;
// distillation: p_T, the sum of p log p over the listed entries, m, and of the
// lists' distinct tokens z [T][k], p [T][k] and, ascending, the tokens
// themselves (int32) [T][k].  live is written with a sum or mean only.
__host__ __device__ __forceinline__ int64_t live_words(int64_t T) {
  return T <= 64 ? 2 : (T + 63) / 64;
}
struct State {
  uint64_t* live;
  float *inv, *a, *lse, *rowb, *ratio, *pt, *ent, *mass, *zt, *p;
  int32_t* sidx;
  __host__ __device__ State(float* b, int64_t T, int64_t k) {
    live = (uint64_t*)b;
    inv = b + live_words(T) * 2;
    a = inv + 2;
    lse = a + T;
    rowb = lse + T;
    ratio = rowb + T;
    pt = ratio + T;
    ent = pt + T;
    mass = ent + T;
    zt = k ? mass + T : pt;
    p = zt + T * k;
    sidx = (int32_t*)(p + T * k);
  }
  static int64_t floats(int64_t T, int64_t k) {
    return live_words(T) * 2 + 2 + (k ? (3 * k + 7) * T : 5 * T);
  }
};

// Joins a row's partial sums and finishes its loss, a workgroup a row (with one
// wavefront a row, 26 us instead of 7 for one row of 128256 tokens, 4008 pairs; no faster
// at 4094 rows either).  Bound by the start of the launch and the pairs' way from
// memory: 2047 rows of 128256 tokens, 16 MB, in 8 us.  A row that is left out (ignored
// label, empty list) has loss 0 and live 0.
template <bool XENT>
__global__ __launch_bounds__(256) void k_head_join(const float2* __restrict__ part, int64_t npart,
                                                   int64_t V, int k,
                                                   const int64_t* __restrict__ labels,
                                                   int64_t ignore, State st, float zscale,
                                                   float* rows, uint8_t* live) {
  __shared__ float2 red[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t t = blockIdx.x;
  if (blockIdx.x == 0 && threadIdx.x == 0) st.inv[0] = 1.f;
  float m = -INFINITY, s = 0.f;
  const float2* pt = part + t * npart;
  int64_t i = threadIdx.x;
  for (; i + 3 * 256 < npart; i += 4 * 256) {
    float2 q[4];
#pragma unroll
    for (int d = 0; d < 4; ++d) q[d] = pt[i + d * 256];
#pragma unroll
    for (int d = 0; d < 4; ++d) ms_join(m, s, q[d].x, q[d].y);
  }
  for (; i < npart; i += 256) ms_join(m, s, pt[i].x, pt[i].y);
#pragma unroll
  for (int d = 32; d; d >>= 1) ms_join(m, s, __shfl_xor(m, d), __shfl_xor(s, d));
  if (lane == 0) red[wave] = make_float2(m, s);
  __syncthreads();
  if (wave) return;
  for (int w = 1; w < 4; ++w) ms_join(m, s, red[w].x, red[w].y);
  const float a = LN2 * (m + log2f(s));                // -inf where every token is listed
  float loss, lse, tail;                               // tail: the factor of exp(z - a)
  bool on;
  if (XENT) {
    const int64_t y = labels[t];
    on = y != ignore;
    const bool in = y >= 0 && y < V;
    const float z = in ? st.zt[t] : NAN;               // a label outside: NaN, loss and gradient
    const float d = a - z;
    loss = d > 0.f ? d + log1pf(expf(-d)) : log1pf(expf(d));
    lse = in ? z + loss : NAN;
    if (d != d) loss = d;
    tail = expf(a - lse);
  } else {
    float tm = -INFINITY, ts = 0.f, np = 0.f;
    for (int i = lane; i < k; i += 64)
      if (st.sidx[t * k + i] != PAD_IDX) {
        ms_join(tm, ts, st.zt[t * k + i] * LOG2E, 1.f);
        np += 1.f;
      }
#pragma unroll
    for (int d = 32; d; d >>= 1) ms_join(tm, ts, __shfl_xor(tm, d), __shfl_xor(ts, d));
    on = wave_sum_f(np) > 0.f;
    lse = log_add(a, LN2 * (tm + log2f(ts)));
    float l = 0.f;
    for (int i = lane; i < k; i += 64) {
      const float p = st.p[t * k + i];
      if (st.sidx[t * k + i] != PAD_IDX && !(p == 0.f)) l += p * (lse - st.zt[t * k + i]);
    }
    loss = wave_sum_f(l) + st.ent[t];
    float pt = st.pt[t], mass = st.mass[t];
    if (a == -INFINITY) {                              // no token is left for the tail
      mass -= pt;
      pt = 0.f;
      if (lane == 0) st.mass[t] = mass;
    }
    if (!(pt == 0.f)) loss += pt * (logf(pt) - a + lse);
    tail = mass * expf(a - lse) - pt;
  }
  if (lane == 0) {
    st.a[t] = a;
    st.lse[t] = lse;
    st.rowb[t] = on ? zscale * tail : 0.f;
    st.ratio[t] = on ? zscale : 0.f;
    rows[t] = on ? loss : 0.f;
    if (live) live[t] = on;
  }
}

// Sum or mean of the rows' losses, in a fixed order, and the live rows' bits,
// by one workgroup: the latency of a launch and of two trips to memory, 4 to 5 us.
// (Left to the workgroup that joins the last row instead, every workgroup has to release
// its row to the others, 25 ns one after the other: 250 rows no faster, 2047 rows 50 us
// slower.)
__global__ __launch_bounds__(1024) void k_head_reduce(const float* __restrict__ rows,
                                                      const uint8_t* __restrict__ live, int64_t T,
                                                      int mean, float* loss, State st) {
  __shared__ float ls[16], lc[16];
  float s = 0.f, c = 0.f;
  for (int64_t t0 = threadIdx.x & ~63; t0 < T; t0 += 1024) {
    const int64_t t = t0 + (threadIdx.x & 63);
    const bool on = t < T && live[t];
    const uint64_t bits = __ballot(on);
    if (t < T) s += rows[t];
    c += on ? 1.f : 0.f;
    if ((threadIdx.x & 63) == 0) {
      st.live[t0 / 64] = bits;
      if (T <= 64) st.live[1] = bits;                  // of the second parts
    }
  }
  s = wave_sum_f(s);
  c = wave_sum_f(c);
  if ((threadIdx.x & 63) == 0) {
    ls[threadIdx.x >> 6] = s;
    lc[threadIdx.x >> 6] = c;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    s = c = 0.f;
    for (int w = 0; w < 16; ++w) {
      s += ls[w];
      c += lc[w];
    }
    loss[0] = mean ? s / c : s;                        // a mean over no row: NaN
    st.inv[0] = mean ? (c > 0.f ? 1.f / c : 0.f) : 1.f;
  }
}

// The teacher's list of each row: tokens ascending, probabilities, the
// bits of the forward product (the row's words are cleared first).  One
// wavefront a row.  Tokens outside [0, V) are empty slots; of one listed twice
// the list holds one entry with the sum of its probabilities.  Repeats and ranks by
// comparing all pairs, 4 a read of LDS: k^2 / 256 reads a lane, no more than the clearing of
// the words takes: 2047 rows of 128 (50272 tokens) in 36 us, 250 of 20 in 7,
// 17 of 64 in 11 (the latency of its dependent steps).
constexpr int LIST_MAX = 256;
template <typename TV>
__global__ __launch_bounds__(64) void k_list(const TV* __restrict__ val, int64_t ldv,
                                             const int32_t* __restrict__ idx, int64_t ldi,
                                             const float* __restrict__ tlse, float itemp,
                                             int64_t V, int k, State st, uint32_t* mask,
                                             int32_t* base, int64_t ntile) {
  __shared__ __attribute__((aligned(16))) int ix[LIST_MAX];
  __shared__ __attribute__((aligned(16))) float pr[LIST_MAX];
  __shared__ int srt[LIST_MAX];
  const int lane = threadIdx.x;
  const int64_t t = blockIdx.x;
  uint32_t* words = mask + t * ntile * 8;
  for (int64_t i = lane; i < ntile * 2; i += 64) ((uint4*)words)[i] = make_uint4(0u, 0u, 0u, 0u);
  float m = -INFINITY;
  const int k4 = (k + 3) & ~3;
  if (lane < k4 - k) ix[k + lane] = -1;                // read by fours
  for (int i = lane; i < k; i += 64) {
    const int v = idx[t * ldi + i];
    const float x = (float)val[t * ldv + i] * itemp;
    ix[i] = v >= 0 && v < V ? v : -1;
    pr[i] = x;
    if (ix[i] >= 0) m = fmaxf(m, x);
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
  const float ref = tlse ? tlse[t] : m;
  float s = 0.f;
  for (int i = lane; i < k; i += 64) {
    pr[i] = ix[i] >= 0 ? expf(pr[i] - ref) : 0.f;
    s += pr[i];
  }
  s = wave_sum_f(s);
  // (the cleared words have arrived before their bits are set)
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  const float norm = tlse ? 1.f : 1.f / s;
  float ent = 0.f;
  for (int i = lane; i < k; i += 64) {
    const float p = pr[i] * norm;
    if (ix[i] >= 0 && !(p == 0.f)) ent += p * logf(p);
  }
  ent = wave_sum_f(ent);
  // first occurrences, and their probabilities with the repeats'
  int mine[LIST_MAX / 64];
  float prob[LIST_MAX / 64];
#pragma unroll
  for (int q = 0; q < LIST_MAX / 64; ++q) {
    const int i = lane + 64 * q;
    mine[q] = -1;
    prob[q] = 0.f;
    if (i < k && ix[i] >= 0) {
      bool first = true;
      const int me = ix[i];
      for (int j = 0; j < k4; j += 4) {
        const int4 o = *(const int4*)&ix[j];
        const int w[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (w[e] == me) {
            if (j + e < i) first = false;
            prob[q] += pr[j + e];
          }
      }
      mine[q] = first ? me : -1;
    }
  }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < LIST_MAX / 64; ++q)
    if (lane + 64 * q < k) {
      ix[lane + 64 * q] = mine[q];
      srt[lane + 64 * q] = PAD_IDX;
      st.sidx[t * k + lane + 64 * q] = PAD_IDX;
      st.p[t * k + lane + 64 * q] = 0.f;
      st.zt[t * k + lane + 64 * q] = 0.f;
    }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < LIST_MAX / 64; ++q)
    if (mine[q] >= 0) {
      int rank = 0;
      for (int j = 0; j < k4; j += 4) {
        const int4 o = *(const int4*)&ix[j];
        // (as unsigned numbers the empty slots, -1, are above all)
        rank += ((uint32_t)o.x < (uint32_t)mine[q]) + ((uint32_t)o.y < (uint32_t)mine[q]) +
                ((uint32_t)o.z < (uint32_t)mine[q]) + ((uint32_t)o.w < (uint32_t)mine[q]);
      }
      st.sidx[t * k + rank] = mine[q];
      st.p[t * k + rank] = prob[q] * norm;
      atomicOr(words + (mine[q] >> 5), 1u << (mine[q] & 31));
      srt[rank] = mine[q];
    }
  __syncthreads();
  // listed tokens before each tile of 256
  for (int64_t i = lane; i < ntile; i += 64) {
    int lo = 0, hi = k;
    while (lo < hi) {
      const int md = (lo + hi) >> 1;
      if (srt[md] < (int)(i * 256)) lo = md + 1;
      else hi = md;
    }
    base[t * ntile + i] = lo;
  }
  if (lane == 0) {
    st.ent[t] = ent;
    st.pt[t] = tlse && s < 1.f ? 1.f - s : 0.f;
    st.mass[t] = tlse && !(s < 1.f) ? s : 1.f;         // NaN stays NaN
  }
}

// ---------------------------------------------------------------------------
// backward
// ---------------------------------------------------------------------------
// max |g| over the rows, one workgroup (a gradient per row)
__global__ __launch_bounds__(1024) void k_absmax(const float* __restrict__ g, int64_t T,
                                                 float* out) {
  __shared__ float l[16];
  float m = 0.f;
  for (int64_t t = threadIdx.x; t < T; t += 1024) m = fmaxf(m, fabsf(g[t]));
#pragma unroll
  for (int d = 32; d; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
  if ((threadIdx.x & 63) == 0) l[threadIdx.x >> 6] = m;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 16; ++w) m = fmaxf(m, l[w]);
    out[0] = m;
  }
}

// A gradient for each row: the row's dz is stored relative to the largest one
// (undone where the sums are rounded).  live: bit t set where the row's gradient
// is not 0 (the other rows of h are read as zeros: a masked row's NaN stays out
// of dW).
__global__ __launch_bounds__(64) void k_grad_rows(State st, int64_t T,
                                                  const float* __restrict__ g,
                                                  const float* __restrict__ gmax, float* rowb,
                                                  float* ratio, uint64_t* live) {
  const int64_t t = (int64_t)blockIdx.x * 64 + threadIdx.x;
  float r = 0.f;
  if (t < T) {
    const float big = gmax[0];
    const float own = st.ratio[t];
    const float w = own == 0.f || big == 0.f ? 0.f : g[t] / big;
    r = own * w;
    ratio[t] = r;
    rowb[t] = r == 0.f ? 0.f : st.rowb[t] * w;
  }
  const uint64_t bits = __ballot(!(r == 0.f));
  if (threadIdx.x == 0) {
    live[blockIdx.x] = bits;
    if (T <= 64) live[1] = bits;                       // of the second parts
  }
}

// What undoes the scaling of dz: f0 f1 mul (the loss's gradient or the largest
// of the rows', 1 / the rows of a mean, scale / dz_scale).
struct Factor {
  const float *f0, *f1;
  float mul;
  __device__ float get() const { return f0[0] * f1[0] * mul; }
};

// dz of a piece of the vocabulary, the forward's product with another epilogue:
// dz[t][v - vbeg] = rowb exp(z - a), zeros in the columns past the vocabulary (and
// where rowb is 0, whatever z is).  A label's own dz is -rowb (cross entropy; in the
// persistent kernel put in place on the rows' way out: looked for at each 4 elements, 195 us
// instead of 182 at 2047 x 50272 x 768); the listed tokens' of a distillation follow
// (k_dz_listed).
struct DzArgs {
  const uint16_t *h, *W;
  int64_t ldh, ldw, T, nv, C;
  float scale;
  const float *a, *rowb;
  const int64_t* labels;   // may be null
  int64_t vbeg;
  int nm, nn;
  uint16_t* dz;
  int64_t zstep;
};

// A piece's dz in memory: blocks of 64 columns, each dz_rows(T) rows of 128
// bytes, so that a unit of either product that reads it is 8 KB in one
// piece (row by row, dW's loads went 64 KB from row to row: MFMAs busy 53 % of the
// time instead of 64).  The columns of whole tiles are
// written, zeros behind nv; the rows behind T are not, and dh's tiles, which
// read them, do not keep what comes of them.  Up to 64 tokens, rows 64 on hold the
// second parts.
__host__ __device__ __forceinline__ int64_t dz_cols(int64_t nv) { return (nv + 255) / 256 * 256; }
__host__ __device__ __forceinline__ int64_t dz_rows(int64_t T) {
  return T <= 64 ? 128 : (T + 255) / 256 * 256;
}
__device__ __forceinline__ uint16_t* dz_at(uint16_t* dz, int64_t zstep, int64_t t, int64_t v) {
  return dz + v / G_K * zstep + t * G_K + v % G_K;
}

// dz of 4 consecutive tokens of a row; rest: what the rounding leaves (TWO)
template <typename T8, bool TWO = false>
__device__ __forceinline__ uint2 dz_pack(const f4_t& acc, float scale2, float a2, float b,
                                         uint2* rest = nullptr) {
  typedef typename Half<T8>::t H;
  uint16_t o[4], l[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const float x = b * __builtin_amdgcn_exp2f(__builtin_fmaf(acc[r], scale2, -a2));
    o[r] = to16<T8>(x);
    if (TWO) l[r] = to16<T8>(x - (float)__builtin_bit_cast(H, o[r]));
  }
  if (TWO)
    *rest = b == 0.f ? make_uint2(0u, 0u)
                     : make_uint2(l[0] | (uint32_t)l[1] << 16, l[2] | (uint32_t)l[3] << 16);
  const uint2 u = make_uint2(o[0] | (uint32_t)o[1] << 16, o[2] | (uint32_t)o[3] << 16);
  return b == 0.f ? make_uint2(0u, 0u) : u;
}
// element r of 4 becomes x
__device__ __forceinline__ void set16(uint2& u, int r, uint32_t x) {
  uint32_t& w = r < 2 ? u.x : u.y;
  w = r & 1 ? (w & 0xffffu) | x << 16 : (w & 0xffff0000u) | x;
}
// the first `left` of 4 elements
__device__ __forceinline__ uint2 first16(const uint2& u, int64_t left) {
  return make_uint2(left >= 2 ? u.x : left == 1 ? u.x & 0xffffu : 0u,
                    left >= 4 ? u.y : left == 3 ? u.y & 0xffffu : 0u);
}

template <typename T8, typename G>
__global__ __launch_bounds__(G::THREADS) void k_head_dz(const DzArgs p) {
  __shared__ __attribute__((aligned(1024))) char smem[G::LDS];
  int tm, tn;
  g_band(g_xcd(blockIdx.x, gridDim.x), p.nm, p.nn, tm, tn);
  const int64_t v0 = (int64_t)tm * G::BM, t0 = (int64_t)tn * G::BN;
  const GOperand A{p.W + v0 * p.ldw, p.ldw, G_K, p.nv - v0, p.C, nullptr};
  const GOperand B{p.h + t0 * p.ldh, p.ldh, G_K, p.T - t0, p.C, nullptr};
  f4_t acc[G::MI][G::NJ];
  g_tile<T8, G>(smem, A, B, 0, p.C, acc);
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int64_t vw = v0 + (wave / G::WGN) * G::WM;
  const float scale2 = p.scale * LOG2E;
#pragma unroll
  for (int j = 0; j < G::NJ; ++j) {
    const int64_t t = t0 + (wave % G::WGN) * G::WN + 16 * j + (lane & 15);
    if (t >= p.T) continue;
    const float b = p.rowb[t], a2 = p.a[t] * LOG2E;
    const int64_t y = p.labels ? p.labels[t] - p.vbeg : -1;
#pragma unroll
    for (int i = 0; i < G::MI; ++i) {
      const int64_t v = vw + 16 * i + 4 * (lane >> 4);           // below dz_cols
      const int64_t o = y - v;
      uint2 rest, u = dz_pack<T8, true>(acc[i][j], scale2, a2, b, &rest);
      if (o >= 0 && o < 4) {
        const uint16_t x = to16<T8>(0.f - b);
        set16(u, (int)o, x);
        set16(rest, (int)o, to16<T8>(0.f - b - (float)__builtin_bit_cast(typename Half<T8>::t, x)));
      }
      *(uint2*)dz_at(p.dz, p.zstep, t, v) = first16(u, p.nv - v);
      if (p.T <= 64) *(uint2*)dz_at(p.dz, p.zstep, 64 + t, v) = first16(rest, p.nv - v);
    }
  }
}

template <typename T8>
struct DzJob {
  static constexpr bool MASKED = false;
  __device__ static int64_t lda() { return g_args<DzArgs>().ldw; }
  __device__ static int64_t ldb() { return g_args<DzArgs>().ldh; }
  __device__ static int64_t kstep_a() { return G_K; }
  __device__ static int64_t kstep_b() { return G_K; }
  __device__ static int64_t unit_a() { return G_K * lda(); }
  __device__ static int64_t unit_b() { return G_K * ldb(); }
  __device__ static int tiles() {
    const DzArgs p = g_args<DzArgs>();
    return p.nm * p.nn;
  }
  __device__ __forceinline__ static void place(const DzArgs& p, int lin, int64_t& v0,
                                               int64_t& t0) {
    int tm, tn;
    g_band(lin, p.nm, p.nn, tm, tn);
    v0 = (int64_t)tm * 256;
    t0 = (int64_t)tn * 256;
  }
  __device__ static int stages(int) { return (int)((g_args<DzArgs>().C + G_K - 1) / G_K); }
  __device__ __forceinline__ void tile(int lin, GOperand& A, GOperand& B, int64_t& k,
                                       int& nch) const {
    const DzArgs p = g_args<DzArgs>();
    int64_t v0, t0;
    place(p, lin, v0, t0);
    A = GOperand{p.W + v0 * p.ldw, p.ldw, G_K, p.nv - v0, p.C, nullptr};
    B = GOperand{p.h + t0 * p.ldh, p.ldh, G_K, p.T - t0, p.C, nullptr};
    k = 0;
    nch = stages(lin);
  }
  // a, rowb and label of the wavefront's 2 x 32 rows (64 words of each)
  __device__ __forceinline__ void side(int lin, char* priv) const {
    const DzArgs p = g_args<DzArgs>();
    int64_t v0, t0;
    place(p, lin, v0, t0);
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int64_t t = t0 + 128 * b + 32 * (wave & 3), left = (p.T - t) * 4;
      g_load_lds_words(priv + 768 * b, p.a + t, left, lane);
      g_load_lds_words(priv + 768 * b + 256, p.rowb + t, left, lane);
      if (p.labels) g_load_lds_words(priv + 768 * b + 512, p.labels + t, left * 2, lane);
    }
  }
  __device__ __forceinline__ void finish(int lin, char* priv, GAcc& acc) const {
    const DzArgs p = g_args<DzArgs>();
    int64_t v0, t0;
    place(p, lin, v0, t0);
    const int lane = g_lane();
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const float scale2 = p.scale * LOG2E;
    const int64_t vt = p.vbeg + v0;                    // the tile's first token
    float at[4], b[4];
    int lab[4];                                        // the label's place in the tile
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const char* q = priv + 768 * (j >> 1);
      const int row = 16 * (j & 1) + (lane & 15);
      at[j] = ((const float*)q)[row] * LOG2E;
      b[j] = ((const float*)q)[64 + row];
      const int64_t y = p.labels ? ((const int64_t*)(q + 512))[row] - vt : -1;
      // (a row's label is written by the first of its 4 lanes)
      const bool mine = y >= 0 && y < 256 && v0 + y < p.nv && (int)(y >> 5 & 1) == (wave >> 2);
      lab[j] = mine && lane < 16 ? (int)y : -1;
    }
    const bool whole = v0 + 256 <= p.nv;
    g_each<4>([&](auto jj) __attribute__((always_inline)) {
      constexpr int j = decltype(jj)::value;
      uint2 u[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        u[i] = dz_pack<T8>(acc.v[i][j], scale2, at[j], b[j]);
      if (!whole)
#pragma unroll
        for (int i = 0; i < 8; ++i) u[i] = first16(u[i], p.nv - (v0 + g_m(i, wave, lane)));
      g_rows_out(
          priv, u,
          [&]() __attribute__((always_inline)) {
            if (lab[j] >= 0) *g_rows_at(priv, lane, lab[j]) = to16<T8>(0.f - b[j]);
          },
          [&](int r, int m, const uint4& x) __attribute__((always_inline)) {
            const int64_t t = t0 + g_n(j, wave, 0) + r;
            if (t < p.T) *(uint4*)dz_at(p.dz, p.zstep, t, v0 + m) = x;
          });
    });
  }
};

template <typename T8>
__global__ __launch_bounds__(G_THREADS) void k_head_dz_p(const DzArgs) {
  __shared__ __attribute__((aligned(1024))) char smem[G_LDS];
  g_run<T8, G_KC, G_KC>(smem, DzJob<T8>());
}

// The listed tokens' dz within [vbeg, vbeg + nv) (distillation), a thread each: 5 to 7 us,
// in place of a search for listed tokens in the epilogue of the product.
template <typename T8>
__global__ __launch_bounds__(256) void k_dz_listed(State st, int64_t T, int k,
                                                   const float* __restrict__ ratio, int64_t vbeg,
                                                   int64_t nv, uint16_t* dz, int64_t zstep) {
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x, t = e / k;
  if (t >= T) return;
  const int64_t v = st.sidx[e];
  if (v == PAD_IDX || v < vbeg || v >= vbeg + nv) return;
  const float r = ratio[t], d = st.mass[t] * expf(st.zt[e] - st.lse[t]) - st.p[e];
  const float x = r == 0.f ? 0.f : r * d;
  const uint16_t o = to16<T8>(x);
  *dz_at(dz, zstep, t, v - vbeg) = o;
  if (T <= 64)
    *dz_at(dz, zstep, 64 + t, v - vbeg) =
        to16<T8>(x - (float)__builtin_bit_cast(typename Half<T8>::t, o));
}

// dh partial sums (fp32): P[split][t][c] (+)= sum of dz[t][v] W[v][c] over the
// split's v (span of them, a multiple of 64).  No atomics: a split's sums are its own,
// and the pieces of the vocabulary follow each other, so the result is the same each time.
struct DhArgs {
  const uint16_t *W, *dz;
  int64_t ldw, zstep, T, nv, C, span;
  int nm, nn, ns;
  float* P;
  int add;
};

// 4 channels c.. of row t
__device__ __forceinline__ void dh_add(const DhArgs& p, int split, int64_t t, int64_t c,
                                       const f4_t& a) {
  if (t >= p.T || c >= p.C) return;
  float4* q = (float4*)(p.P + ((int64_t)split * p.T + t) * p.C + c);
  float4 v = make_float4(a[0], a[1], a[2], a[3]);
  if (p.add) {
    const float4 u = *q;
    v.x += u.x; v.y += u.y; v.z += u.z; v.w += u.w;
  }
  *q = v;
}

template <typename T8, typename G>
__global__ __launch_bounds__(G::THREADS) void k_head_dh(const DhArgs p) {
  __shared__ __attribute__((aligned(1024))) char smem[G::LDS];
  int tm, tn;
  const int lin = g_xcd(blockIdx.x, gridDim.x), split = lin / (p.nm * p.nn);
  g_band(lin - split * p.nm * p.nn, p.nm, p.nn, tm, tn);
  // n tile 0: the tokens, 1: their second parts (the same rows of W, from L2)
  const int64_t c0 = (int64_t)tm * G::BM, t0 = (int64_t)tn * 64;
  const int64_t kb = split * p.span, ke = kb + p.span < p.nv ? kb + p.span : p.nv;
  const GOperand A{p.W + c0, p.ldw, G_K * p.ldw, p.C - c0, p.nv, nullptr};
  const GOperand B{p.dz + t0 * G_K, G_K, p.zstep, p.T, dz_cols(p.nv), nullptr};
  f4_t acc[G::MI][G::NJ];
  g_tile<T8, G>(smem, A, B, kb, ke, acc);
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
#pragma unroll
  for (int j = 0; j < G::NJ; ++j)
#pragma unroll
    for (int i = 0; i < G::MI; ++i)
      dh_add(p, 2 * split + tn, (wave % G::WGN) * G::WN + 16 * j + (lane & 15),
             c0 + (wave / G::WGN) * G::WM + 16 * i + 4 * (lane >> 4), acc[i][j]);
}

struct DhJob {
  static constexpr bool MASKED = false;
  __device__ static int64_t lda() { return g_args<DhArgs>().ldw; }
  __device__ static int64_t ldb() { return G_K; }
  __device__ static int64_t kstep_a() { return G_K * lda(); }
  __device__ static int64_t kstep_b() { return g_args<DhArgs>().zstep; }
  __device__ static int64_t unit_a() { return G_K; }
  __device__ static int64_t unit_b() { return G_K * G_K; }
  __device__ static int tiles() {
    const DhArgs p = g_args<DhArgs>();
    return p.nm * p.nn * p.ns;
  }
  __device__ __forceinline__ static void place(const DhArgs& p, int lin, int64_t& c0,
                                               int64_t& t0, int& split) {
    int tm, tn;
    split = lin / (p.nm * p.nn);
    g_band(lin - split * p.nm * p.nn, p.nm, p.nn, tm, tn);
    c0 = (int64_t)tm * 256;
    t0 = (int64_t)tn * 256;
  }
  __device__ static int stages(int lin) {
    const DhArgs p = g_args<DhArgs>();
    const int64_t k = lin / (p.nm * p.nn) * p.span, n = p.nv - k < p.span ? p.nv - k : p.span;
    return (int)((n + G_K - 1) / G_K);                 // n > 0 for every split of a launch
  }
  __device__ __forceinline__ void tile(int lin, GOperand& A, GOperand& B, int64_t& k,
                                       int& nch) const {
    const DhArgs p = g_args<DhArgs>();
    int64_t c0, t0;
    int split;
    place(p, lin, c0, t0, split);
    k = split * p.span;
    A = GOperand{p.W + c0, p.ldw, G_K * p.ldw, p.C - c0, p.nv, nullptr};
    B = GOperand{p.dz + t0 * G_K, G_K, p.zstep, p.T - t0, dz_cols(p.nv), nullptr};
    nch = stages(lin);
  }
  __device__ __forceinline__ void side(int, char*) const {}
  __device__ __forceinline__ void finish(int lin, char*, GAcc& acc) const {
    const DhArgs p = g_args<DhArgs>();
    int64_t c0, t0;
    int split;
    place(p, lin, c0, t0, split);
    const int lane = g_lane();
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        dh_add(p, split, t0 + g_n(j, wave, lane), c0 + g_m(i, wave, lane), acc.v[i][j]);
  }
};

template <typename T8>
__global__ __launch_bounds__(G_THREADS) void k_head_dh_p(const DhArgs) {
  __shared__ __attribute__((aligned(1024))) char smem[G_LDS];
  g_run<T8, G_KS, G_KC_BLOCKED>(smem, DhJob());
}

// dh = factor * (P[0] + P[1] + ...), rounded once; 4 channels a thread.  Bound by reading
// P: 2047 x 4096 in 22 us with 2 splits, 333 x 1000 in 8.
template <typename T8>
__global__ __launch_bounds__(256) void k_dh_out(const float* __restrict__ P, int ns, int64_t T,
                                                int64_t C, Factor fac, uint16_t* dh,
                                                int64_t ldd) {
  const int64_t n4 = T * (C / 4);
  const float f = fac.get();
  for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < n4; e += (int64_t)gridDim.x * 256) {
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    int s = 0;
    for (; s + 8 <= ns; s += 8) {
      float4 u[8];
#pragma unroll
      for (int d = 0; d < 8; ++d) u[d] = *(const float4*)(P + (int64_t)(s + d) * T * C + e * 4);
#pragma unroll
      for (int d = 0; d < 8; ++d) {
        v.x += u[d].x; v.y += u[d].y; v.z += u[d].z; v.w += u[d].w;
      }
    }
    for (; s < ns; ++s) {
      const float4 u = *(const float4*)(P + (int64_t)s * T * C + e * 4);
      v.x += u.x; v.y += u.y; v.z += u.z; v.w += u.w;
    }
    const int64_t t = e / (C / 4), c = (e - t * (C / 4)) * 4;
    *(uint2*)(dh + t * ldd + c) =
        make_uint2(to16<T8>(f * v.x) | (uint32_t)to16<T8>(f * v.y) << 16,
                   to16<T8>(f * v.z) | (uint32_t)to16<T8>(f * v.w) << 16);
  }
}

// dW[v][c] = factor * sum_t dz[t][v] h[t][c] of a piece's rows v.  From about 500 tokens on
// bound by the MFMAs, fed by transpose reads of both operands; with few tokens by
// writing dW: one token, 1 GB in 288 us (3.65 TB/s; a workgroup a CU waits for its own stores).
struct DwArgs {
  const uint16_t *h, *dz;
  int64_t ldh, zstep, T, nv, C;
  const uint64_t* live;
  int nm, nn;
  Factor fac;
  uint16_t* dW;
  int64_t ldo;
};

template <typename T8>
struct DwJob {
  static constexpr bool MASKED = true;
  __device__ static int64_t lda() { return g_args<DwArgs>().ldh; }
  __device__ static int64_t ldb() { return G_K; }
  __device__ static int64_t kstep_a() {
    const DwArgs p = g_args<DwArgs>();
    return p.T <= 64 ? 0 : G_K * p.ldh;
  }
  __device__ static int64_t kstep_b() { return G_K * G_K; }
  __device__ static int64_t unit_a() { return G_K; }
  __device__ static int64_t unit_b() { return g_args<DwArgs>().zstep; }
  __device__ static int tiles() {
    const DwArgs p = g_args<DwArgs>();
    return p.nm * p.nn;
  }
  __device__ __forceinline__ static void place(const DwArgs& p, int lin, int64_t& c0,
                                               int64_t& v0) {
    int tm, tn;
    g_band(lin, p.nm, p.nn, tm, tn);
    c0 = (int64_t)tm * 256;
    v0 = (int64_t)tn * 256;
  }
  // up to 64 tokens: a second stage, the same tokens times the second parts
  __device__ static int64_t K() {
    const int64_t T = g_args<DwArgs>().T;
    return T <= 64 ? 128 : T;
  }
  __device__ static int stages(int) { return (int)((K() + G_K - 1) / G_K); }
  __device__ __forceinline__ void tile(int lin, GOperand& A, GOperand& B, int64_t& k,
                                       int& nch) const {
    const DwArgs p = g_args<DwArgs>();
    int64_t c0, v0;
    place(p, lin, c0, v0);
    A = GOperand{p.h + c0, p.ldh, kstep_a(), p.C - c0, K(), p.live};
    B = GOperand{p.dz + v0 / G_K * p.zstep, G_K, G_K * G_K, 256, K(), nullptr};
    k = 0;
    nch = stages(lin);
  }
  __device__ __forceinline__ void side(int, char*) const {}
  __device__ __forceinline__ void finish(int lin, char* priv, GAcc& acc) const {
    const DwArgs p = g_args<DwArgs>();
    int64_t c0, v0;
    place(p, lin, c0, v0);
    const float f = p.fac.get();
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    g_each<4>([&](auto jj) __attribute__((always_inline)) {
      constexpr int j = decltype(jj)::value;
      uint2 u[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const f4_t& a = acc.v[i][j];
        u[i] = make_uint2(to16<T8>(f * a[0]) | (uint32_t)to16<T8>(f * a[1]) << 16,
                          to16<T8>(f * a[2]) | (uint32_t)to16<T8>(f * a[3]) << 16);
      }
      g_rows_out(priv, u, [] {}, [&](int r, int m, const uint4& x) __attribute__((always_inline)) {
        const int64_t v = v0 + g_n(j, wave, 0) + r;
        if (v < p.nv && c0 + m < p.C)                            // C: a multiple of 8
          *(uint4*)(p.dW + v * p.ldo + c0 + m) = x;
      });
    });
  }
};

template <typename T8>
__global__ __launch_bounds__(G_THREADS) void k_head_dw(const DwArgs) {
  __shared__ __attribute__((aligned(1024))) char smem[G_LDS];
  g_run<T8, G_KS, G_KS_BLOCKED>(smem, DwJob<T8>());
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
// Tiles of the products (m x n): vocabulary x tokens for z, channels x tokens
// for dh, channels x vocabulary for dW.
using ZM = GTile<256, 64, 4, 2, 4, true, true>;
using ZS = GTile<256, 16, 8, 1, 4, true, true>;
using HM = GTile<256, 64, 4, 2, 4, false, true>;
using HS = GTile<256, 16, 8, 1, 4, false, true>;
struct Big {               // the persistent 256 x 256 tiles
  static constexpr int BM = 256, BN = 256, WGM = 2;
};

static int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Tokens per tile of the logits: 0 = 16, 1 = 64, 2 = 256.  Forward over V = 128256, C =
// 4096: 16 tokens in 189 us with tiles of 16 and of 64, 17 in 211 and 188; 64 in 192 us
// with tiles of 64, 240 with 256; 65 in 225 and 238, 160 in 317 and 247.  The gradients
// of 16 tokens (50272 x 768, 32007 x 1000) take 76 and 66 us with tiles of 16, 81 and 70
// with 64.  Tiles of 64 also while there is at most one of them a CU: forward of 2047 x 2000 x
// 4096 in 56 us instead of 91, gradients 154 instead of 189; 250 x 16000 x 768, 25 and
// 30, 63 and 74 (a CU that has one tile takes 0.6 of the time of one of 256).
static int token_tile(int64_t T, int64_t V) {
  return T <= 16 ? 0 : T <= 64 || cdiv(T, 64) * cdiv(V, 256) <= 256 ? 1 : 2;
}
static int64_t n_part(int64_t T, int64_t V) {
  static const int wgm[3] = {ZS::WGM, ZM::WGM, Big::WGM};
  return cdiv(V, 256) * wgm[token_tile(T, V)];
}

// Vocabulary of a backward piece: dz of a piece in about 256 MB, at least 8192
// tokens of the vocabulary.  Larger pieces end fewer rounds of tiles half empty and
// add to dh's sums less often: gradients of 2047 x 50272 x 4096 in 2230, 2015
// and 2010 us with pieces of 128, 256 and 512 MB, of 4094 x 50272 x 768 in 1050, 980 and
// 930, of 4094 x 128256 x 4096 in 9850, 9750 and 9630.  256 MB is taken, for the
// memory it leaves; that the last-level cache holds a piece does not show.
static int64_t piece_of(int64_t T, int64_t V) {
  int64_t p = ((int64_t)128 << 20) / T / 256 * 256;
  if (p < 8192) p = 8192;
  const int64_t all = cdiv(V, 256) * 256;
  return p < all ? p : all;
}
// Parts that dh's sums over a piece are split into: the fewest rounds of 256
// workgroups times the 64-k stages of a part (1.2 us each, 6 more a tile), and
// the fp32 partial sums, written and read back at about 4 TB/s.
static int dh_splits(int64_t T, int64_t C, int64_t piece) {
  const int64_t tiles = cdiv(C, 256) * cdiv(T, T <= 16 ? 16 : T <= 64 ? 64 : 256);
  const int64_t stages = cdiv(piece, G_K);
  int64_t best = 1;
  double least = 0.;
  for (int64_t s = 1; s <= 256 && s * 4 <= stages; ++s) {
    const double t = (double)cdiv(tiles * s, 256) * ((double)cdiv(stages, s) * 1.2 + 6.) +
                     2e-6 * (double)(T * C) * (double)s;
    if (s == 1 || t < least) {
      least = t;
      best = s;
    }
  }
  return (int)best;
}

struct FwdWs {
  float2* part;
  float* rows;
  uint8_t* live;
  uint32_t* mask;
  int32_t* base;
  size_t bytes;
  FwdWs(void* ws, size_t cap, int64_t T, int64_t V, int64_t k, bool& ok) {
    WsCarver w(ws, cap);
    part = w.take<float2>((size_t)(T * n_part(T, V)));
    rows = w.take<float>((size_t)T);
    live = w.take<uint8_t>((size_t)T);
    mask = k ? w.take<uint32_t>((size_t)(T * cdiv(V, 256)) * 8) : nullptr;
    base = k ? w.take<int32_t>((size_t)(T * cdiv(V, 256))) : nullptr;
    bytes = w.off;
    ok = w.ok();
  }
};

struct GradWs {
  int64_t piece, span;
  int ns;                  // splits of dh's sums over the first (largest) piece
  uint16_t* dz;
  float *P, *rowb, *ratio, *gmax;
  uint64_t* live;
  size_t bytes;
  GradWs(void* ws, size_t cap, int64_t T, int64_t V, int64_t C, bool& ok) {
    WsCarver w(ws, cap);
    piece = piece_of(T, V);
    span = cdiv(cdiv(piece < V ? piece : V, dh_splits(T, C, piece)), G_K) * G_K;
    ns = (int)cdiv(piece < V ? piece : V, span);
    dz = w.take<uint16_t>((size_t)(dz_rows(T) * piece));
    P = w.take<float>((size_t)(T * C) * ns * (T <= 64 ? 2 : 1));
    rowb = w.take<float>((size_t)T);
    ratio = w.take<float>((size_t)T);
    gmax = w.take<float>(1);
    live = w.take<uint64_t>((size_t)live_words(T));
    bytes = w.off;
    ok = w.ok();
  }
};

static bool bad_matrix(const void* p, int64_t ld, int64_t C) {
  return !p || ld < C || ld >= G_MAX_LD || (ld & 7) || (((uintptr_t)p) & 15);
}
static int check_head(const void* h, int64_t ldh, const void* W, int64_t ldw, int dtype,
                      int64_t T, int64_t V, int64_t C) {
  if (dtype != CRBQ_F16 && dtype != CRBQ_BF16) return CRBQ_ERR_ARG;
  if (T < 1 || V < 1 || C < 8 || (C & 7) || V >= ((int64_t)1 << 28) ||
      T >= ((int64_t)1 << 22))
    return CRBQ_ERR_ARG;
  if (bad_matrix(h, ldh, C) || bad_matrix(W, ldw, C)) return CRBQ_ERR_ARG;
  if (cdiv(V, 256) * cdiv(T, 16) >= ((int64_t)1 << 31)) return CRBQ_ERR_ARG;
  return CRBQ_OK;
}

// Workgroups of a persistent launch: one per CU (160 KB of LDS each).
static unsigned persistent(int64_t tiles) {
  constexpr int CUS = 256;
  return (unsigned)(tiles < CUS ? tiles : CUS);
}

template <typename T8, typename G, bool XENT>
static void launch_fwd(FwdArgs p, hipStream_t s) {
  p.nm = (int)cdiv(p.V, G::BM);
  p.nn = (int)cdiv(p.T, G::BN);
  const int64_t tiles = (int64_t)p.nm * p.nn;
  if constexpr (std::is_same<G, Big>::value)
    k_head_fwd_p<T8, XENT><<<persistent(tiles), G_THREADS, 0, s>>>(p);
  else
    k_head_fwd<T8, G, XENT><<<(unsigned)tiles, G::THREADS, 0, s>>>(p);
}

template <typename T8, bool XENT>
static int head_fwd(const void* h, int64_t ldh, const void* W, int64_t ldw, int64_t T, int64_t V,
                    int64_t C, float scale, const Listed& ls, int64_t ignore, int reduction,
                    float* loss, const State& st, const FwdWs& w, hipStream_t s) {
  const FwdArgs p{(const uint16_t*)h, (const uint16_t*)W, ldh, ldw, T, V, C, scale, ls, 0, 0,
                  w.part, n_part(T, V), st.zt};
  switch (token_tile(T, V)) {
    case 0: launch_fwd<T8, ZS, XENT>(p, s); break;
    case 1: launch_fwd<T8, ZM, XENT>(p, s); break;
    default: launch_fwd<T8, Big, XENT>(p, s);
  }
  CRBQ_LAUNCH_CHECK();
  float* rows = reduction ? w.rows : loss;
  uint8_t* live = reduction ? w.live : nullptr;
  k_head_join<XENT><<<(unsigned)T, 256, 0, s>>>(w.part, n_part(T, V), V, ls.k, ls.labels, ignore,
                                                st, dz_scale<T8>(), rows, live);
  CRBQ_LAUNCH_CHECK();
  if (reduction) {
    k_head_reduce<<<1, 1024, 0, s>>>(w.rows, w.live, T, reduction == CRBQ_MEAN, loss, st);
    CRBQ_LAUNCH_CHECK();
  }
  return CRBQ_OK;
}

struct GradCall {
  const uint16_t *h, *W;
  int64_t ldh, ldw, T, V, C;
  const int64_t* labels;   // cross entropy; else null
  int k;
  float scale;
  const float* g;
  bool per_row;
  uint16_t *dh, *dW;
  int64_t ldd, ldo;
};

template <typename T8, typename GZ, typename GH>
static int head_grad(const GradCall& c, const State& st, const GradWs& w, hipStream_t s) {
  const int64_t T = c.T, V = c.V, C = c.C;
  const float *rowb = st.rowb, *ratio = st.ratio;
  const uint64_t* live = st.live;
  if (c.per_row) {
    k_absmax<<<1, 1024, 0, s>>>(c.g, T, w.gmax);
    CRBQ_LAUNCH_CHECK();
    k_grad_rows<<<(unsigned)cdiv(T, 64), 64, 0, s>>>(st, T, c.g, w.gmax, w.rowb, w.ratio, w.live);
    CRBQ_LAUNCH_CHECK();
    rowb = w.rowb;
    ratio = w.ratio;
    live = w.live;
  }
  const Factor fac{c.per_row ? w.gmax : c.g, st.inv, c.scale / dz_scale<T8>()};
  const int nt = (int)cdiv(T, GZ::BN);
  const int64_t zstep = dz_rows(T) * G_K;
  for (int64_t v = 0; v < V; v += w.piece) {
    const int64_t nv = V - v < w.piece ? V - v : w.piece;
    const uint16_t* Wv = c.W + v * c.ldw;
    const int nm = (int)cdiv(nv, GZ::BM);
    const DzArgs z{c.h, Wv, c.ldh, c.ldw, T, nv, C, c.scale, st.a, rowb, c.labels, v, nm, nt, w.dz,
                   zstep};
    if constexpr (std::is_same<GZ, Big>::value)
      k_head_dz_p<T8><<<persistent((int64_t)nm * nt), G_THREADS, 0, s>>>(z);
    else
      k_head_dz<T8, GZ><<<(unsigned)((int64_t)nm * nt), GZ::THREADS, 0, s>>>(z);
    CRBQ_LAUNCH_CHECK();
    if (!c.labels) {
      k_dz_listed<T8><<<(unsigned)cdiv(T * c.k, 256), 256, 0, s>>>(st, T, c.k, ratio, v, nv, w.dz,
                                                                   zstep);
      CRBQ_LAUNCH_CHECK();
    }
    if (c.dh) {
      const int mh = (int)cdiv(C, GH::BM);
      const int nn = T <= 64 ? 2 : (int)cdiv(T, 256);
      const DhArgs q{Wv, w.dz, c.ldw, zstep, T, nv, C, w.span, mh, nn, (int)cdiv(nv, w.span), w.P,
                     v > 0};
      const int64_t tiles = (int64_t)mh * nn * q.ns;
      if constexpr (std::is_same<GH, Big>::value)
        k_head_dh_p<T8><<<persistent(tiles), G_THREADS, 0, s>>>(q);
      else
        k_head_dh<T8, GH><<<(unsigned)tiles, GH::THREADS, 0, s>>>(q);
      CRBQ_LAUNCH_CHECK();
    }
    if (c.dW) {
      const int mw = (int)cdiv(C, 256), nw = (int)cdiv(nv, 256);
      k_head_dw<T8><<<persistent((int64_t)mw * nw), G_THREADS, 0, s>>>(
          DwArgs{c.h, w.dz, c.ldh, zstep, T, nv, C, live, mw, nw, fac, c.dW + v * c.ldo, c.ldo});
      CRBQ_LAUNCH_CHECK();
    }
  }
  if (c.dh) {
    const int64_t nb = cdiv(T * (C / 4), 256);
    k_dh_out<T8><<<(unsigned)(nb < 4096 ? nb : 4096), 256, 0, s>>>(
        w.P, w.ns * (T <= 64 ? 2 : 1), T, C, fac, c.dh, c.ldd);
    CRBQ_LAUNCH_CHECK();
  }
  return CRBQ_OK;
}

template <typename T8>
static int head_grad_t(const GradCall& c, const State& st, const GradWs& w, hipStream_t s) {
  switch (token_tile(c.T, w.piece)) {
    case 0: return head_grad<T8, ZS, HS>(c, st, w, s);
    case 1: return c.T <= 64 ? head_grad<T8, ZM, HM>(c, st, w, s)
                             : head_grad<T8, ZM, Big>(c, st, w, s);
    default: return head_grad<T8, Big, Big>(c, st, w, s);
  }
}

// (a scale of 0 would make the -inf of what is left out a NaN)
static bool bad_scale(float s) { return !(fabsf(s) > 0.f) || !(fabsf(s) < INFINITY); }
static bool bad_state(const void* p) { return !p || (((uintptr_t)p) & 7); }
static bool bad_ws(const void* p) { return (((uintptr_t)p) & 15) != 0; }
static bool bad_reduction(int r) { return r != CRBQ_NONE && r != CRBQ_MEAN && r != CRBQ_SUM; }

}  // namespace crbq

using namespace crbq;

extern "C" size_t crbq_head_state_floats(int64_t T, int64_t k) {
  if (T < 1 || k < 0 || k > CRBQ_HEAD_MAX_K) return 0;
  return (size_t)State::floats(T, k);
}

extern "C" size_t crbq_head_workspace_size(int64_t T, int64_t V, int64_t C, int64_t k, int grad) {
  if (T < 1 || V < 1 || C < 1 || k < 0 || k > CRBQ_HEAD_MAX_K) return 0;
  bool ok;
  return grad ? GradWs(nullptr, 0, T, V, C, ok).bytes : FwdWs(nullptr, 0, T, V, k, ok).bytes;
}

extern "C" int crbq_head_xent(const void* h, int64_t ldh, const void* W, int64_t ldw, int dtype,
                              int64_t T, int64_t V, int64_t C, const int64_t* labels,
                              int64_t ignore_index, float scale, int reduction, float* loss,
                              float* state, void* ws, size_t ws_bytes, void* stream) {
  if (int e = check_head(h, ldh, W, ldw, dtype, T, V, C)) return e;
  if (!labels || !loss || bad_state(state) || bad_reduction(reduction) || bad_scale(scale) ||
      bad_ws(ws))
    return CRBQ_ERR_ARG;
  bool ok;
  const FwdWs w(ws, ws_bytes, T, V, 0, ok);
  if (!ok) return CRBQ_ERR_WORKSPACE;
  const Listed ls{labels, nullptr, nullptr, 0, 0};
  const State st(state, T, 0);
  hipStream_t s = (hipStream_t)stream;
  return dtype == CRBQ_F16
             ? head_fwd<h8_t, true>(h, ldh, W, ldw, T, V, C, scale, ls, ignore_index, reduction,
                                    loss, st, w, s)
             : head_fwd<b8_t, true>(h, ldh, W, ldw, T, V, C, scale, ls, ignore_index, reduction,
                                    loss, st, w, s);
}

extern "C" int crbq_head_xent_grad(const void* h, int64_t ldh, const void* W, int64_t ldw,
                                   int dtype, int64_t T, int64_t V, int64_t C,
                                   const int64_t* labels, float scale, int reduction,
                                   const float* state, const float* g, void* dh, int64_t ldd,
                                   void* dW, int64_t ldo, void* ws, size_t ws_bytes,
                                   void* stream) {
  if (int e = check_head(h, ldh, W, ldw, dtype, T, V, C)) return e;
  if (!labels || bad_state(state) || !g || (!dh && !dW) || bad_reduction(reduction) ||
      bad_scale(scale) || bad_ws(ws))
    return CRBQ_ERR_ARG;
  if ((dh && bad_matrix(dh, ldd, C)) || (dW && bad_matrix(dW, ldo, C))) return CRBQ_ERR_ARG;
  bool ok;
  const GradWs w(ws, ws_bytes, T, V, C, ok);
  if (!ok) return CRBQ_ERR_WORKSPACE;
  const State st((float*)state, T, 0);
  const GradCall c{(const uint16_t*)h, (const uint16_t*)W, ldh, ldw, T, V, C, labels, 0, scale, g,
                   reduction == CRBQ_NONE, (uint16_t*)dh, (uint16_t*)dW, ldd, ldo};
  hipStream_t s = (hipStream_t)stream;
  return dtype == CRBQ_F16 ? head_grad_t<h8_t>(c, st, w, s) : head_grad_t<b8_t>(c, st, w, s);
}

extern "C" int crbq_head_distill(const void* h, int64_t ldh, const void* W, int64_t ldw,
                                 int dtype, int64_t T, int64_t V, int64_t C, const void* top_val,
                                 int val_dtype, int64_t ldv, const int32_t* top_idx, int64_t ldi,
                                 int k, const float* top_lse, float scale, float temperature,
                                 int reduction, float* loss, float* state, void* ws,
                                 size_t ws_bytes, void* stream) {
  if (int e = check_head(h, ldh, W, ldw, dtype, T, V, C)) return e;
  if (!top_val || !top_idx || !loss || bad_state(state) || bad_reduction(reduction) || k < 1 ||
      k > CRBQ_HEAD_MAX_K || ldv < k || ldi < k || !(temperature > 0.f) ||
      bad_scale(scale * (1.f / temperature)) || bad_ws(ws))
    return CRBQ_ERR_ARG;
  if (val_dtype != CRBQ_F32 && val_dtype != CRBQ_F16 && val_dtype != CRBQ_BF16)
    return CRBQ_ERR_ARG;
  bool ok;
  const FwdWs w(ws, ws_bytes, T, V, k, ok);
  if (!ok) return CRBQ_ERR_WORKSPACE;
  const State st(state, T, k);
  hipStream_t s = (hipStream_t)stream;
  const int64_t ntile = cdiv(V, 256);
  const float it = 1.f / temperature;
  if (val_dtype == CRBQ_F32)
    k_list<float><<<(unsigned)T, 64, 0, s>>>((const float*)top_val, ldv, top_idx, ldi, top_lse, it,
                                             V, k, st, w.mask, w.base, ntile);
  else if (val_dtype == CRBQ_F16)
    k_list<_Float16><<<(unsigned)T, 64, 0, s>>>((const _Float16*)top_val, ldv, top_idx, ldi,
                                                top_lse, it, V, k, st, w.mask, w.base, ntile);
  else
    k_list<__bf16><<<(unsigned)T, 64, 0, s>>>((const __bf16*)top_val, ldv, top_idx, ldi, top_lse,
                                              it, V, k, st, w.mask, w.base, ntile);
  CRBQ_LAUNCH_CHECK();
  const Listed ls{nullptr, w.mask, w.base, ntile, k};
  return dtype == CRBQ_F16 ? head_fwd<h8_t, false>(h, ldh, W, ldw, T, V, C, scale * it, ls, 0,
                                                   reduction, loss, st, w, s)
                           : head_fwd<b8_t, false>(h, ldh, W, ldw, T, V, C, scale * it, ls, 0,
                                                   reduction, loss, st, w, s);
}

extern "C" int crbq_head_distill_grad(const void* h, int64_t ldh, const void* W, int64_t ldw,
                                      int dtype, int64_t T, int64_t V, int64_t C, int k,
                                      float scale, float temperature, int reduction,
                                      const float* state, const float* g, void* dh, int64_t ldd,
                                      void* dW, int64_t ldo, void* ws, size_t ws_bytes,
                                      void* stream) {
  if (int e = check_head(h, ldh, W, ldw, dtype, T, V, C)) return e;
  if (bad_state(state) || !g || (!dh && !dW) || k < 1 || k > CRBQ_HEAD_MAX_K ||
      !(temperature > 0.f) || bad_reduction(reduction) ||
      bad_scale(scale * (1.f / temperature)) || bad_ws(ws))
    return CRBQ_ERR_ARG;
  if ((dh && bad_matrix(dh, ldd, C)) || (dW && bad_matrix(dW, ldo, C))) return CRBQ_ERR_ARG;
  bool ok;
  const GradWs w(ws, ws_bytes, T, V, C, ok);
  if (!ok) return CRBQ_ERR_WORKSPACE;
  const State st((float*)state, T, k);
  const GradCall c{(const uint16_t*)h, (const uint16_t*)W, ldh, ldw, T, V, C, nullptr, k,
                   scale * (1.f / temperature), g, reduction == CRBQ_NONE, (uint16_t*)dh,
                   (uint16_t*)dW, ldd, ldo};
  hipStream_t s = (hipStream_t)stream;
  return dtype == CRBQ_F16 ? head_grad_t<h8_t>(c, st, w, s) : head_grad_t<b8_t>(c, st, w, s);
}
