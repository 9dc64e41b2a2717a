// 16-bit matrix-product tiles of the output-head kernels (head.hip).
//
// A workgroup sums D[m][n] = sum_k A[m][k] B[n][k] over a
// BM x BN tile on v_mfma_f32_16x16x32_{f16,bf16} (fp32 accumulate).  Each
// operand comes in one of two layouts:
//   K-contiguous (KC): element (row, k) at P[row * ld + k];
//   K-strided:         element (row, k) at P[k * ld + row],
// and is staged through LDS 64 k at a time by direct-to-LDS buffer loads
// (16 bytes per lane, no register round trip).  A K-contiguous stage keeps
// its rows as 128 bytes with the 16-byte chunks XOR-permuted by the row, a
// K-strided stage keeps its 64 k rows as they are, chunks permuted by bits
// 0, 1 and 3 of the row, and the lanes read their 8 consecutive k with LDS
// transpose reads (ds_read_b64_tr_b16): either way half a wavefront's reads
// fall on distinct banks.  What lies outside an operand (rows past its end, k past its
// end) is turned into zeros by the buffer loads' range check, or, for the k
// tail inside a K-contiguous row, by an offset beyond any range.
//
// The accumulators: element r of acc[i][j] of a lane is
//   m = wm + 16 i + 4 (lane >> 4) + r,  n = wn + 16 j + (lane & 15),
// so a lane holds 4 consecutive m of one n: the kernels take the output's
// contiguous (or reduced) dimension as m.
#pragma once
#include <type_traits>

#include "common.h"

namespace crbq {

typedef int i4_t __attribute__((ext_vector_type(4)));
typedef __fp16 tr4_t __attribute__((__vector_size__(4 * sizeof(__fp16))));
typedef __attribute__((address_space(3))) tr4_t lds_tr4_t;

constexpr int G_K = 64;                 // k per stage
constexpr int64_t G_MAX_LD = (int64_t)1 << 22;   // 256 rows * ld * 2 bytes < 2^31

template <typename T8>
__device__ __forceinline__ f4_t g_mfma(T8 a, T8 b, f4_t c);
template <>
__device__ __forceinline__ f4_t g_mfma<h8_t>(h8_t a, h8_t b, f4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f4_t g_mfma<b8_t>(b8_t a, b8_t b, f4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// LDS-only barrier: this wavefront's LDS operations, not its global loads.
__device__ __forceinline__ void g_sync_lds() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}
template <int N>
__device__ __forceinline__ void g_wait_vm() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// One operand of a tile: `rows` x K elements from row0 on (`rows` = the rows
// that exist from row0 to the operand's end; more than the tile's are fine).
// The range check goes by whole 4-byte words: hence the even ends.
struct GOperand {
  const uint16_t* p;       // KC: &P[row0 * ld]; K-strided: &P[row0]
  int64_t ld;
  int64_t rows;            // rows (outputs) from row0 to the end; K-strided: even
  int64_t K;               // k's that exist; KC: a multiple of 8
  const uint64_t* live;    // K-strided only, may be null: bit k % 64 of word k / 64 clear =
                           // row k reads as zeros, whatever it holds
};

__device__ __forceinline__ i4_t g_rsrc(const uint16_t* base, int64_t nrec) {
  const uint64_t a = (uint64_t)base;
  return i4_t{__builtin_amdgcn_readfirstlane((int)(uint32_t)a),
              __builtin_amdgcn_readfirstlane((int)((a >> 32) & 0xffff)),
              __builtin_amdgcn_readfirstlane((int)nrec), 0x00020000};
}

// Row permutation of a K-strided stage (of 16-byte chunks, within 16).
__device__ __forceinline__ int g_swz(int t) { return ((t & 3) | ((t >> 1) & 4)) << 1; }

template <int R, bool KC, int NW>
struct GStage {
  static constexpr int BYTES = R * G_K * 2;
  static constexpr int LOADS = BYTES / 1024;                     // 1 KB each
  static constexpr int PER_WAVE = LOADS >= NW ? LOADS / NW : 1;  // fewer: some are issued twice
  static constexpr int ROWS_PER_LOAD = KC ? 8 : 512 / R;
  static_assert(KC ? R % 16 == 0 : (R == 128 || R == 256), "stage shape");

  __device__ static int group(int wave, int kk) { return (wave * PER_WAVE + kk) % LOADS; }
  // lane's row and 16-byte chunk (of the source) in load group g
  __device__ static int row(int g, int lane) {
    return KC ? 8 * g + (lane >> 3) : ROWS_PER_LOAD * g + lane / (R / 8);
  }
  __device__ static int chunk(int g, int lane) {
    const int r = row(g, lane);
    return KC ? (lane & 7) ^ (r & 7) : (lane % (R / 8)) ^ g_swz(r);
  }
  __device__ static unsigned voff(int g, int lane, int64_t ld) {
    return (unsigned)((row(g, lane) * ld + chunk(g, lane) * 8) * 2);
  }
  // descriptor of the stage that starts at k0 of K
  __device__ static i4_t rsrc(const GOperand& o, int64_t k0, int64_t K) {
    const int64_t kl = K - k0;
    int64_t n = 0;
    if (KC) {
      const int64_t rows = o.rows < R ? o.rows : R;
      if (kl > 0) n = ((rows - 1) * o.ld + kl) * 2;
      return g_rsrc(o.p + (kl > 0 ? k0 : 0), n);
    }
    const int64_t rows = kl < G_K ? kl : G_K;
    if (kl > 0) n = ((rows - 1) * o.ld + o.rows) * 2;
    return g_rsrc(o.p + (kl > 0 ? k0 * o.ld : 0), n);
  }
};

__device__ __forceinline__ void g_load_lds(const void* dst, i4_t rs, unsigned voff) {
  const unsigned d = __builtin_amdgcn_readfirstlane(
      (unsigned)(uintptr_t)(const __attribute__((address_space(3))) void*)dst);
  asm volatile("buffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(voff), "s"(rs), "{m0}"(d));
}

template <typename T8, int PITCH>
__device__ __forceinline__ T8 g_tr_frag(const char* p) {
  typedef __attribute__((address_space(3))) const char lchar;
  lchar* q = (lchar*)(const void*)p;
  const tr4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_tr4_t*)(q));
  const tr4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_tr4_t*)(q + 4 * PITCH));
  struct P { tr4_t a, b; } v{lo, hi};
  return __builtin_bit_cast(T8, v);
}

// Tile geometry: WGM x WGN wavefronts, NS stages in LDS.
template <int BM_, int BN_, int WGM_, int WGN_, int NS_, bool AKC_, bool BKC_>
struct GTile {
  static constexpr int BM = BM_, BN = BN_, WGM = WGM_, WGN = WGN_, NS = NS_;
  static constexpr int NW = WGM * WGN, THREADS = 64 * NW;
  static constexpr bool AKC = AKC_, BKC = BKC_;
  static constexpr int WM = BM / WGM, WN = BN / WGN, MI = WM / 16, NJ = WN / 16;
  using SA = GStage<BM, AKC, NW>;
  using SB = GStage<BN, BKC, NW>;
  static constexpr int STAGE = SA::BYTES + SB::BYTES;
  static constexpr int LDS = NS * STAGE;
  static constexpr int LW = SA::PER_WAVE + SB::PER_WAVE;         // loads of a wavefront, a stage
  static_assert(LDS <= 160 * 1024 && MI >= 1 && NJ >= 1 && (NS - 2) * LW <= 63, "tile shape");
};

// Workgroup id -> linear index such that the workgroups one XCD receives
// (every 8th id) take consecutive indices.
__device__ __forceinline__ int g_xcd(int id, int nwg) {
  const int q = nwg / 8, r = nwg % 8, x = id % 8, k = id / 8;
  return (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + k;
}
// Linear index -> (m tile, n tile) in bands of 8 n tiles: 32 consecutive
// indices (an XCD's CUs) form a 4 x 8 block of tiles that shares 12 panels.
__device__ __forceinline__ void g_band(int lin, int nm, int nn, int& tm, int& tn) {
  const int per = nm * 8, band = lin / per, n0 = band * 8;
  const int w = nn - n0 < 8 ? nn - n0 : 8, in = lin - band * per;
  tm = in / w;
  tn = n0 + in % w;
}

// What a lane needs to load stages and to read fragments of them.
template <typename T8, typename G>
struct GLane {
  using SA = typename G::SA;
  using SB = typename G::SB;
  static constexpr unsigned OUT = 0x80000000u;         // beyond any range
  unsigned va[SA::PER_WAVE], vb[SB::PER_WAVE];         // offsets of its loads
  int lane, wave, kc8, fa, fb, kx;

  __device__ GLane(int64_t lda, int64_t ldb) {
    lane = threadIdx.x & 63;
    wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
#pragma unroll
    for (int q = 0; q < SA::PER_WAVE; ++q) va[q] = SA::voff(SA::group(wave, q), lane, lda);
#pragma unroll
    for (int q = 0; q < SB::PER_WAVE; ++q) vb[q] = SB::voff(SB::group(wave, q), lane, ldb);
    kc8 = ((lane & 7) ^ ((lane >> 3) & 7)) * 8;        // a KC lane's first k of a stage
    const int wm = (wave / G::WGN) * G::WM, wn = (wave % G::WGN) * G::WN;
    fa = base<G::AKC, G::BM>(wm);
    fb = base<G::BKC, G::BN>(wn);
    kx = (lane >> 4) ^ (lane & 7);
  }
  // First fragment's address in a stage of R rows, at row w of it.  KC: rows
  // are 128 bytes, the chunk comes with the half stage; K-strided: lane (group gq, s)
  // addresses k row 8 gq + s / 4 at row w + 4 (s % 4).
  template <bool KC, int R>
  __device__ int base(int w) const {
    const int r16 = lane & 15, trow = 8 * (lane >> 4) + (r16 >> 2), ch = w + 4 * (r16 & 3);
    return KC ? (w + r16) * (G_K * 2)
              : trow * R * 2 + (((ch >> 3) ^ g_swz(trow)) << 4) + (ch & 7) * 2;
  }
  // Fragment i (16 rows on) of half h of the operand whose stage starts at
  // LDS address `at` (a multiple of 1024).  K-strided: 16 rows are two chunks,
  // address bits 5 to 7, which the permutation exclusive-ors.
  template <bool KC, int R>
  __device__ T8 frag(const char* smem, int at, int f, int h, int i) const {
    if constexpr (KC)
      return *(const T8*)(smem + (at + f + ((kx ^ (4 * h)) << 4)) + i * 16 * G_K * 2);
    else
      return g_tr_frag<T8, R * 2>(smem + ((at + f) ^ (i << 5)) + h * 32 * R * 2);
  }
  __device__ T8 fragA(const char* smem, int at, int h, int i) const {
    return frag<G::AKC, G::BM>(smem, at, fa, h, i);
  }
  __device__ T8 fragB(const char* smem, int at, int h, int j) const {
    return frag<G::BKC, G::BN>(smem, at + SA::BYTES, fb, h, j);
  }
  // a stage's descriptors and masks
  struct Src {
    i4_t ra, rb;
    bool kin;              // KC lanes: this lane's chunk lies before K
    uint64_t live;
  };
  __device__ Src source(const GOperand& A, const GOperand& B, int64_t k0, bool any) const {
    Src s;
    s.ra = SA::rsrc(A, k0, any ? A.K : 0);
    s.rb = SB::rsrc(B, k0, any ? B.K : 0);
    s.kin = k0 + kc8 < (G::BKC ? B.K : A.K);
    s.live = ~0ull;
    if (!G::AKC && A.live) s.live = any ? A.live[k0 / G_K] : 0;
    return s;
  }
  // load q (of G::LW) of a stage into the LDS at buf
  __device__ void load(char* buf, int q, const Src& s) const {
    if (q < SA::PER_WAVE) {
      const int g = SA::group(wave, q);
      unsigned v = va[q < SA::PER_WAVE ? q : 0];
      if (G::AKC) v = s.kin ? v : OUT;
      else v = ((s.live >> SA::row(g, lane)) & 1) ? v : OUT;
      g_load_lds(buf + g * 1024, s.ra, v);
    } else {
      const int qb = q - SA::PER_WAVE, g = SB::group(wave, qb);
      unsigned v = vb[qb >= 0 && qb < SB::PER_WAVE ? qb : 0];
      if (G::BKC) v = s.kin ? v : OUT;
      g_load_lds(buf + SA::BYTES + g * 1024, s.rb, v);
    }
  }
};

// f(integral constant 0), ..., f(N - 1): accumulators are indexed by constants only
template <int N, typename F>
__device__ __forceinline__ void g_each(const F& f) {
  if constexpr (N > 0) {
    g_each<N - 1>(f);
    f(std::integral_constant<int, N - 1>{});
  }
}

constexpr int G_PRIV = 32 * 1024;       // LDS beside the stages of g_run, in equal shares

// The lane, for an epilogue: opaque, so that what an epilogue computes from it
// is computed there and not kept in registers over the products.
__device__ __forceinline__ int g_lane() {
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));
  return lane;
}

template <typename G>
__device__ __forceinline__ void g_zero(f4_t (&acc)[G::MI][G::NJ]) {
#pragma unroll
  for (int i = 0; i < G::MI; ++i)
#pragma unroll
    for (int j = 0; j < G::NJ; ++j) acc[i][j] = f4_t{0.f, 0.f, 0.f, 0.f};
}

// One tile, NS - 1 stages of loads in flight (few rows of B: the loads of A
// are all that counts).  acc = its sums over k in [k_beg, k_end): both multiples
// of 64, or k_end the operands' end (where theirs differ, the shorter
// one's; what the longer one holds behind it meets zeros and has to be
// finite).  On return every wavefront has left the stages.
template <typename T8, typename G>
__device__ __forceinline__ void g_tile(char* smem, const GOperand& A, const GOperand& B,
                                       int64_t k_beg, int64_t k_end,
                                       f4_t (&acc)[G::MI][G::NJ]) {
  const GLane<T8, G> L(A.ld, B.ld);
  const int nch = k_end > k_beg ? (int)((k_end - k_beg + G_K - 1) / G_K) : 0;
  g_zero<G>(acc);
#pragma unroll
  for (int c = 0; c < G::NS - 1; ++c) {
    const auto s = L.source(A, B, k_beg + (int64_t)c * G_K, c < nch);
#pragma unroll
    for (int q = 0; q < G::LW; ++q) L.load(smem + c * G::STAGE, q, s);
  }
  g_wait_vm<(G::NS - 2) * G::LW>();
  g_sync_lds();
  for (int c = 0; c < nch; ++c) {
    const int n = c + G::NS - 1;
    const auto s = L.source(A, B, k_beg + (int64_t)n * G_K, n < nch);
    char* nbuf = smem + (n % G::NS) * G::STAGE;
    const int at = (c % G::NS) * G::STAGE;
#pragma unroll
    for (int h = 0; h < G_K / 32; ++h) {
      T8 bb[G::NJ];
#pragma unroll
      for (int j = 0; j < G::NJ; ++j) bb[j] = L.fragB(smem, at, h, j);
      T8 an = L.fragA(smem, at, h, 0);
#pragma unroll
      for (int i = 0; i < G::MI; ++i) {
        const T8 a = an;
        if (i + 1 < G::MI) an = L.fragA(smem, at, h, i + 1);
#pragma unroll
        for (int j = 0; j < G::NJ; ++j) acc[i][j] = g_mfma<T8>(a, bb[j], acc[i][j]);
        if (h == 0) {
          // the stage's loads between the MFMAs of its first half
#pragma unroll
          for (int q = 0; q < G::LW; ++q)
            if (q * G::MI / G::LW == i) L.load(nbuf, q, s);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
    g_wait_vm<(G::NS - 2) * G::LW>();
    g_sync_lds();
  }
  g_wait_vm<0>();
  g_sync_lds();
}

// A workgroup's share of a launch's tiles, one after the other without a
// gap: tiles lin, lin + gridDim, ... of job.tiles.
//   job.tile(lin, A, B, k_beg, nch)  a tile's operands, first k and stages (>= 1)
//   job.side(lin, priv)              loads what the tile's epilogue needs into the
//                                    wavefront's own share of G_PRIV (g_load_lds*)
//   job.finish(lin, priv, acc)       the epilogue
// Two stages in LDS.  While the MFMAs of one half stage run, the fragments of
// the next half are read into the other register set.  One barrier a stage,
// between its halves: there every wavefront has read all of the stage (so the
// stage after the next may be loaded over it), and the loads of the next
// stage, issued a whole stage before, have arrived (so its fragments may be
// read): no MFMA waits for an LDS read that could only start behind a
// barrier.  The next tile's first stages are loaded under this tile's last, so
// its loads run under the epilogue too.
template <typename T8, typename G, typename Job>
__device__ __forceinline__ void g_run(char* smem, const Job& job) {
  static_assert(G::NS == 2 && G::NJ <= G::MI, "two stages");
  const GLane<T8, G> L(job.lda, job.ldb);
  char* priv = smem + G::LDS + L.wave * (G_PRIV / G::NW);
  const int nwg = gridDim.x, first = g_xcd(blockIdx.x, nwg);
  // the stage to be loaded next: c of tile ll
  int ll = first, lc = 0, ln = 0;
  int64_t lk = 0;
  GOperand A, B;
  auto open = [&]() {
    if (ll < job.tiles) job.tile(ll, A, B, lk, ln);
  };
  auto source = [&]() {
    const auto s = L.source(A, B, lk + (int64_t)lc * G_K, ll < job.tiles);
    if (++lc == ln) {
      lc = 0;
      ll += nwg;
      open();
    }
    return s;
  };
  open();
  if (ll >= job.tiles) return;                         // no tile at all
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const auto s = source();
#pragma unroll
    for (int q = 0; q < G::LW; ++q) L.load(smem + c * G::STAGE, q, s);
  }
  g_wait_vm<G::LW>();
  g_sync_lds();
  int par = 0;                                         // the stage's buffer
  for (int lin = first; lin < job.tiles; lin += nwg) {
    // read again behind an epilogue, which needs the registers
    T8 a0[G::MI], b0[G::NJ], a1[G::MI], b1[G::NJ];
#pragma unroll
    for (int j = 0; j < G::NJ; ++j) b0[j] = L.fragB(smem, par * G::STAGE, 0, j);
#pragma unroll
    for (int i = 0; i < G::MI; ++i) a0[i] = L.fragA(smem, par * G::STAGE, 0, i);
    f4_t acc[G::MI][G::NJ];
    g_zero<G>(acc);
    int nch;
    {
      GOperand ta, tb;
      int64_t tk;
      job.tile(lin, ta, tb, tk, nch);
    }
    job.side(lin, priv);
    for (int c = 0; c < nch; ++c) {
      const int at = par * G::STAGE, nx = G::STAGE - at;
      const auto s = source();
#pragma unroll
      for (int i = 0; i < G::MI; ++i) {
        if (i < G::NJ) b1[i] = L.fragB(smem, at, 1, i);
        a1[i] = L.fragA(smem, at, 1, i);
#pragma unroll
        for (int j = 0; j < G::NJ; ++j) acc[i][j] = g_mfma<T8>(a0[i], b0[j], acc[i][j]);
        __builtin_amdgcn_sched_barrier(0);
      }
      g_wait_vm<0>();
      g_sync_lds();
#pragma unroll
      for (int i = 0; i < G::MI; ++i) {
        if (i < G::NJ) b0[i] = L.fragB(smem, nx, 0, i);
        a0[i] = L.fragA(smem, nx, 0, i);
#pragma unroll
        for (int q = 0; q < G::LW; ++q)
          if (q * G::MI / G::LW == i) L.load(smem + at, q, s);
#pragma unroll
        for (int j = 0; j < G::NJ; ++j) acc[i][j] = g_mfma<T8>(a1[i], b1[j], acc[i][j]);
        __builtin_amdgcn_sched_barrier(0);
      }
      par ^= 1;
    }
    job.finish(lin, priv, acc);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); // priv is free for the next side()
  }
  g_wait_vm<0>();
}

// 64 words (lane l: word l of p) and 64 rows of 16 bytes (lane l: p + l * ld) into
// the wavefront's own LDS; what lies behind nbytes reads as zeros.
__device__ __forceinline__ void g_load_lds_words(const void* dst, const void* p, int64_t nbytes,
                                                 int lane) {
  const unsigned d = __builtin_amdgcn_readfirstlane(
      (unsigned)(uintptr_t)(const __attribute__((address_space(3))) void*)dst);
  const i4_t rs = g_rsrc((const uint16_t*)p, nbytes > 0 ? (nbytes < 256 ? nbytes : 256) : 0);
  asm volatile("buffer_load_dword %0, %1, 0 offen lds" ::"v"(lane * 4), "s"(rs), "{m0}"(d));
}

// 16 rows (n) of a tile's 16-bit output, MI * 16 elements each, through the wavefront's
// own LDS: in as each lane's 4 consecutive elements of one row, out as
// 16-byte stores of whole rows.  put(row, m, 8 elements) stores.
template <typename G, typename F>
__device__ __forceinline__ void g_rows_out(char* priv, const uint2 (&v)[G::MI], F&& put) {
  static_assert(G::MI == 8, "rows of 256 bytes");
  const int lane = g_lane(), n = lane & 15, g = lane >> 4;
#pragma unroll
  for (int i = 0; i < G::MI; ++i)
    *(uint2*)(priv + n * 256 + (((2 * i + (g >> 1)) ^ n) << 4) + (g & 1) * 8) = v[i];
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int r = 4 * q + g;
    put(r, n * 8, *(const uint4*)(priv + r * 256 + ((n ^ r) << 4)));
  }
  asm volatile("" ::: "memory");
}

}  // namespace crbq
