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
  int64_t kstep;           // elements from one 64 k to the next: 64 (KC), 64 ld (K-strided)
  int64_t rows;            // rows (outputs) from row0 to the end; K-strided: even
  int64_t K;               // k's that exist; KC: a multiple of 8
  const uint64_t* live;    // K-strided A, may be null: bit k % 64 of word k / 64 clear = row k
                           // is not read but zeros (of a K-strided B too)
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
    const int64_t ks = kl < G_K ? kl : G_K;
    if (kl > 0) n = KC ? (((o.rows < R ? o.rows : R) - 1) * o.ld + ks) * 2
                       : ((ks - 1) * o.ld + o.rows) * 2;
    return g_rsrc(o.p + (kl > 0 ? k0 / G_K * o.kstep : 0), n);
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

// ---------------------------------------------------------------------------
// 256 x 256 tiles, persistent workgroups of 8 wavefronts (2 along m, 4 along n).
//
// A stage (64 k of both operands, 64 KB; two in LDS) consists of 4 + 4 units of 64
// rows, each 8 KB: 64 rows of 128 bytes (KC) or 64 k rows of 128 bytes (K-strided),
// whole lines of memory either way, one 1 KB load of each wavefront.  The output of
// wavefront (wr, wc) is interleaved so that a unit serves all wavefronts at one time:
//   m = 64 (i >> 1) + 32 wr + 16 (i & 1) + 4 (lane >> 4) + r,   i = 0..7
//   n = 128 (j >> 1) + 32 wc + 16 (j & 1) + (lane & 15),        j = 0..3
// A stage runs in four quarters, quarter u on A's unit u (16 MFMAs) and on B's
// fragments of the stage, which are held in registers.  Fragments are read
// from LDS a quarter ahead (A) or a stage ahead (B: units 0 and 1 in quarter
// 1, units 2 and 3 in quarter 3).  After each half stage, a barrier: the units
// read in it are free, and the loads of the half before the last have
// arrived.  So every half issues 4 loads of each wavefront, evenly spaced, and
// each has between 2 and 3 halves (of 1024 cycles of MFMAs) to arrive:
//   first half of stage c:   A(c + 2) unit 0, A(c + 1) unit 3, B(c + 2) units 2, 3
//   second half:             A(c + 2) units 1, 2,              B(c + 3) units 0, 1
// With one barrier a stage and each stage loaded as a whole in the half
// after it, the MFMAs were busy 64 % of the time, the loads being waited
// for; issued earlier within that half they stood in each other's way.  Now 77 %
// (2047 x 65536 x 4096, both K-contiguous), where the clock falls to 1.6 - 1.85 GHz.
// Measured and not kept: 4 wavefronts of 128 x 128 (accumulators copied between register
// files), wave priorities around the MFMAs (0 to 4 % slower), free instruction order
// within a quarter (2 to 5 % slower), loads ahead into L2 (10 to 17 % slower), tiles of a
// last, partly filled round cut into quarters (2 % at best).
// The stages of consecutive tiles follow on each other without a gap, so a tile's
// first loads run under the last stages and the epilogue of the one before.
//
// A workgroup takes the tiles lin, lin + gridDim, ... of a Job:
//   tiles(), stages(lin) >= 1         how many, and the 64-k stages of one
//   lda(), kstep_a(), unit_a(), ..b   row strides; elements from one 64 k, one unit to the next
//   tile(lin, A, B, k, nch)           a tile's operands, first k (a multiple of 64) and stages
//   side(lin, priv)                   loads what finish needs into the wavefront's own G_PRIV
//                                     bytes of LDS (g_load_lds*), a tile's products ahead
//   finish(lin, priv, acc)            the epilogue
//   MASKED                            A (and a K-strided B) have live rows
// ---------------------------------------------------------------------------
constexpr int G_UNIT = 8192, G_STAGE = 8 * G_UNIT, G_RING = 2 * G_STAGE;
constexpr int G_THREADS = 512;
constexpr int G_PRIV = 4096;            // LDS of each wavefront beside the stages
constexpr int G_LDS = G_RING + 8 * G_PRIV;
struct GAcc {
  f4_t v[8][4];
};
__device__ __forceinline__ int g_m(int i, int wave, int lane) {
  return 64 * (i >> 1) + 32 * (wave >> 2) + 16 * (i & 1) + 4 * (lane >> 4);
}
__device__ __forceinline__ int g_n(int j, int wave, int lane) {
  return 128 * (j >> 1) + 32 * (wave & 3) + 16 * (j & 1) + (lane & 15);
}

// bits 1 and 3 of a K-strided unit's k row permute its 32-byte groups
__device__ __forceinline__ int g_grp(int t) { return ((t >> 1) & 1) | ((t >> 2) & 2); }

template <bool KC>
struct GUnits {
  unsigned voff;           // this lane's offset in a unit's load
  int kc8, row;            // KC: its first k; K-strided: its k row
  int f0, f1;              // fragment addresses (KC: of half 0, 1 of k; K-strided: of 16 rows 0, 1)
  // w: this wavefront's 32-row block in a unit
  __device__ GUnits(int64_t ld, int wave, int lane, int w) {
    const int r = 8 * wave + (lane >> 3), c = lane & 7, r16 = lane & 15, gq = lane >> 4;
    if (KC) {
      kc8 = (c ^ (r & 7)) * 8;
      voff = (unsigned)((r * ld + kc8) * 2);
      f0 = (32 * w + r16) * 128 + ((gq ^ (r16 & 7)) << 4);
      f1 = f0 ^ 64;
    } else {
      kc8 = 0;
      voff = (unsigned)((r * ld + ((((c >> 1) ^ g_grp(r)) << 1) | (c & 1)) * 8) * 2);
      const int t = 8 * gq + (r16 >> 2);
      f0 = t * 128 + (((2 * w) ^ g_grp(t)) << 5) + (r16 & 3) * 8;
      f1 = f0 ^ 32;
    }
    row = r;
  }
  // fragment of half h of k, 16 rows e (0, 1) of the wavefront's block, from the unit at `at`
  template <typename T8>
  __device__ T8 frag(const char* smem, int at, int h, int e) const {
    if constexpr (KC) return *(const T8*)(smem + at + (h ? f1 : f0) + e * 16 * 128);
    else return g_tr_frag<T8, 128>(smem + at + (e ? f1 : f0) + h * 32 * 128);
  }
};

// A value the compiler takes for unknown from here on: what depends on it is
// not computed earlier and kept (scalar registers are as short as vector
// registers during the products).
template <typename T>
__device__ __forceinline__ T g_fresh(T v) {
  asm volatile("" : "+s"(v));
  return v;
}
// The kernel's only argument, a struct Args, read where it is needed.
template <typename Args>
__device__ __forceinline__ Args g_args() {
  typedef __attribute__((address_space(4))) const uint32_t cword;
  static_assert(sizeof(Args) % 4 == 0, "whole words");
  struct Words {
    uint32_t w[sizeof(Args) / 4];
  } a;
  cword* q = (cword*)g_fresh(__builtin_amdgcn_kernarg_segment_ptr());
#pragma unroll
  for (unsigned i = 0; i < sizeof(Args) / 4; ++i) a.w[i] = q[i];
  return __builtin_bit_cast(Args, a);
}

__device__ __forceinline__ int g_uni(int v) { return __builtin_amdgcn_readfirstlane(v); }
template <typename T>
__device__ __forceinline__ T* g_uni(T* q) {
  const uint64_t v = (uint64_t)q;
  return (T*)((uint64_t)(uint32_t)g_uni((int)(uint32_t)v) |
              (uint64_t)(uint32_t)g_uni((int)(v >> 32)) << 32);
}

// How g_run takes an operand: K-contiguous, K-strided, and both of a matrix
// [k or row blocks of 64][rows or k][64] in blocks, whose units of 64 x 64 are 8 KB in
// one piece.  Blocked operands are not range-checked: they have to hold
// every element of the tiles and stages asked for.
enum GLayout { G_KC, G_KS, G_KC_BLOCKED, G_KS_BLOCKED };
constexpr bool g_is_kc(GLayout l) { return l == G_KC || l == G_KC_BLOCKED; }
constexpr bool g_is_blocked(GLayout l) { return l == G_KC_BLOCKED || l == G_KS_BLOCKED; }

// Where the loads of one operand stand within a tile.
template <GLayout L>
struct GCursor {
  static constexpr bool KC = g_is_kc(L);
  const uint16_t* p;       // the stage's first element
  int rows, k;             // rows (at most 256) and k's left from there; k <= 0: none
  __device__ void open(const GOperand& o, int64_t k0) {
    const int64_t kl = o.K - k0;
    p = g_uni(o.p + k0 / G_K * o.kstep);
    rows = g_uni((int)(o.rows < 256 ? o.rows : 256));
    k = g_uni((int)(kl < (1 << 30) ? kl : (1 << 30)));
  }
  __device__ void advance(int kstep) {
    p += kstep;
    k -= G_K;
  }
  // descriptor of the whole stage (rows < 256 x 2^22 elements: below 2^31 bytes)
  __device__ i4_t rsrc(int ld) const {
    int n;
    if (KC) n = (rows - 1) * ld + (k < G_K ? k : G_K);
    else n = ((k < G_K ? k : G_K) - 1) * ld + rows;
    if (g_is_blocked(L)) n = 0x3fffffff;
    return g_rsrc(p, k > 0 ? n * 2 : 0);
  }
};

template <typename T8, GLayout LA, GLayout LB, typename Job>
__device__ __forceinline__ void g_run(char* smem, const Job& job) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  constexpr bool AKC = g_is_kc(LA), BKC = g_is_kc(LB);
  // row strides, and the elements from one 64 k to the next, from one unit to the next
  const int lda = g_uni((int)job.lda()), ldb = g_uni((int)job.ldb());
  const int ka = g_uni((int)job.kstep_a()), kb = g_uni((int)job.kstep_b());
  const int ua = g_uni((int)job.unit_a()) * 2, ub = g_uni((int)job.unit_b()) * 2;
  const int tiles = g_uni(job.tiles());
  const GUnits<AKC> UA(lda, wave, lane, wave >> 2);
  const GUnits<BKC> UB(ldb, wave, lane, wave & 1);
  const int bw = ((wave >> 1) & 1) * G_UNIT;           // n: 32 wc = 64 (wc >> 1) + 32 (wc & 1)
  char* priv = smem + G_RING + wave * G_PRIV;
  char* mine = smem + wave * 1024;                     // this wavefront's kilobyte of a unit
  const int nwg = gridDim.x, first = g_xcd(blockIdx.x, nwg);
  if (first >= tiles) return;                          // no tile at all

  // The stages in load order: stage lc of the ln of tile ll.
  GCursor<LA> ca;
  GCursor<LB> cb;
  const uint64_t* cl = nullptr;
  int ll = first, lc = 0, ln = 0;
  auto open = [&]() __attribute__((always_inline)) {
    ca.k = cb.k = 0;
    ln = 1 << 30;                                      // behind the last tile: no data, no end
    if (ll < tiles) {
      GOperand A, B;
      int64_t k;
      job.tile(ll, A, B, k, ln);
      ln = g_uni(ln);
      ca.open(A, k);
      cb.open(B, k);
      if (!AKC && A.live) cl = g_uni(A.live + k / G_K);
    }
    lc = 0;
  };
  struct Stage {
    i4_t ra, rb;
    int k;                 // KC operands: k's left
    uint64_t live;
  };
  auto next = [&]() __attribute__((always_inline)) {
    Stage s{ca.rsrc(lda), cb.rsrc(ldb), BKC ? cb.k : ca.k, ~0ull};
    // (a scalar load: a vector load's wait would be for all stages in flight)
    if (!AKC && cl)
      s.live = ca.k > 0 ? ((const __attribute__((address_space(4))) uint64_t*)cl)[lc] : 0;
    ca.advance(ka);
    cb.advance(kb);
    if (++lc == ln) {
      ll += nwg;
      open();
    }
    return s;
  };
  constexpr unsigned OUT = 0x80000000u;
  auto loadA = [&](auto uu, const Stage& s, int buf) __attribute__((always_inline)) {
    constexpr int u = decltype(uu)::value;
    char* d = mine + buf * G_STAGE + u * G_UNIT;
    const bool in = AKC ? UA.kc8 < s.k : !Job::MASKED || ((s.live >> UA.row) & 1);
    g_load_lds(d, s.ra, (in ? UA.voff : OUT) + (unsigned)(u * ua));
  };
  auto loadB = [&](auto uu, const Stage& s, int buf) __attribute__((always_inline)) {
    constexpr int u = decltype(uu)::value;
    char* d = mine + buf * G_STAGE + (4 + u) * G_UNIT;
    const bool in = BKC ? LB == G_KC_BLOCKED || UB.kc8 < s.k
                        : !Job::MASKED || ((s.live >> UB.row) & 1);
    g_load_lds(d, s.rb, (in ? UB.voff : OUT) + (unsigned)(u * ub));
  };
  // A fragment (h, e) of unit u; B fragment (h, j)
  auto fragA = [&](int buf, int u, int h, int e) __attribute__((always_inline)) -> T8 {
    return UA.template frag<T8>(smem, buf * G_STAGE + u * G_UNIT, h, e);
  };
  auto fragB = [&](int buf, int h, int j) __attribute__((always_inline)) -> T8 {
    return UB.template frag<T8>(smem, buf * G_STAGE + (4 + 2 * (j >> 1)) * G_UNIT + bw, h, j & 1);
  };
  constexpr std::integral_constant<int, 0> _0{};
  constexpr std::integral_constant<int, 1> _1{};
  constexpr std::integral_constant<int, 2> _2{};
  constexpr std::integral_constant<int, 3> _3{};

  open();
  // stage 0, what stage 1 needs early, then B's units 0 and 1 of stage 2 over stage 0's
  Stage s1, s2;
  {
    const Stage s0 = next();
    s1 = next();
    s2 = next();
    g_each<4>([&](auto uu) __attribute__((always_inline)) {
      loadA(uu, s0, 0);
      loadB(uu, s0, 0);
      loadB(uu, s1, 1);
      if constexpr (decltype(uu)::value < 3) loadA(uu, s1, 1);
    });
  }
  g_wait_vm<0>();
  g_sync_lds();
  T8 a0[4], a1[4], b0[8], b1[8];                       // [2 h + e], [4 h + j]
#pragma unroll
  for (int q = 0; q < 8; ++q) b0[q] = fragB(0, q >> 2, q & 3);
#pragma unroll
  for (int q = 0; q < 4; ++q) a0[q] = fragA(0, 0, q >> 1, q & 1);
  g_sync_lds();
  loadB(_0, s2, 0);
  loadB(_1, s2, 0);

  GAcc acc;
  // quarter u: 16 MFMAs on a; side(q) between them
  auto quarter = [&](auto uu, const T8(&a)[4], const T8(&b)[8], auto&& side)
      __attribute__((always_inline)) {
    constexpr int u = decltype(uu)::value;
    g_each<4>([&](auto qq) __attribute__((always_inline)) {
      constexpr int q = decltype(qq)::value, h = q >> 1, i = 2 * u + (q & 1);
      side(q);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        acc.v[i][j] = g_mfma<T8>(a[q], b[4 * h + j], acc.v[i][j]);
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  // a stage from buffer p; s1, s2: stages c + 1, c + 2
  auto stage = [&](int p, T8(&b)[8], T8(&bn)[8]) __attribute__((always_inline)) {
    const int o = p ^ 1;
    quarter(_0, a0, b, [&](int q) __attribute__((always_inline)) {
      a1[q] = fragA(p, 1, q >> 1, q & 1);
      if (q == 0) loadA(_3, s1, o);
      if (q == 2) loadA(_0, s2, p);
    });
    const Stage s3 = next();
    quarter(_1, a1, b, [&](int q) __attribute__((always_inline)) {
      a0[q] = fragA(p, 2, q >> 1, q & 1);
      bn[4 * (q >> 1) + (q & 1)] = fragB(o, q >> 1, q & 1);
      if (q == 0) loadB(_2, s2, p);
      if (q == 2) loadB(_3, s2, p);
    });
    g_wait_vm<8>();
    g_sync_lds();
    quarter(_2, a0, b, [&](int q) __attribute__((always_inline)) {
      a1[q] = fragA(p, 3, q >> 1, q & 1);
      if (q == 0) loadA(_1, s2, p);
      if (q == 2) loadA(_2, s2, p);
    });
    quarter(_3, a1, b, [&](int q) __attribute__((always_inline)) {
      a0[q] = fragA(o, 0, q >> 1, q & 1);
      bn[4 * (q >> 1) + 2 + (q & 1)] = fragB(o, q >> 1, 2 + (q & 1));
      if (q == 0) loadB(_0, s3, o);
      if (q == 2) loadB(_1, s3, o);
    });
    g_wait_vm<8>();
    g_sync_lds();
    s1 = s2;
    s2 = s3;
  };
  int par = 0;                                         // the stage's buffer
  for (int lin = first; lin < tiles; lin += nwg) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc.v[i][j] = f4_t{0.f, 0.f, 0.f, 0.f};
    job.side(lin, priv);
    const int nch = g_uni(job.stages(lin));
    int c = 0;
    for (; c + 2 <= nch; c += 2) {
      stage(par, b0, b1);
      stage(par ^ 1, b1, b0);
    }
    if (c < nch) {
      stage(par, b0, b1);
      par ^= 1;
#pragma unroll
      for (int q = 0; q < 8; ++q) b0[q] = b1[q];
    }
    job.finish(lin, priv, acc);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); // priv is free for the next side()
  }
  g_wait_vm<0>();
}

__device__ __forceinline__ void g_load_lds_word(const void* dst, i4_t rs, unsigned voff) {
  const unsigned d = __builtin_amdgcn_readfirstlane(
      (unsigned)(uintptr_t)(const __attribute__((address_space(3))) void*)dst);
  asm volatile("buffer_load_dword %0, %1, 0 offen lds" ::"v"(voff), "s"(rs), "{m0}"(d));
}

// 64 words (lane l: word l of p) into the wavefront's own LDS; what lies behind
// nbytes reads as zeros.
__device__ __forceinline__ void g_load_lds_words(const void* dst, const void* p, int64_t nbytes,
                                                 int lane) {
  g_load_lds_word(dst, g_rsrc((const uint16_t*)p, nbytes > 0 ? (nbytes < 256 ? nbytes : 256) : 0),
                  lane * 4);
}

// 16 rows (n) of a wavefront's 16-bit output of a 256 x 256 tile (128 elements each, m
// as above) through its own LDS: in as each lane's 4 consecutive
// elements of one row, out as 16-byte stores, 64 bytes of a row side by
// side.  put(row, m, 8 elements) stores.  g_rows_at(priv, n, m) is where element
// m of row n lies meanwhile: patch() may change some there.
__device__ __forceinline__ uint16_t* g_rows_at(char* priv, int n, int m) {
  const int i = 2 * (m >> 6) + ((m >> 4) & 1), g = (m >> 2) & 3;
  return (uint16_t*)(priv + n * 256 + (((2 * i + (g >> 1)) ^ n) << 4) + (g & 1) * 8) + (m & 3);
}
template <typename P, typename F>
__device__ __forceinline__ void g_rows_out(char* priv, const uint2 (&v)[8], P&& patch, F&& put) {
  const int lane = g_lane(), n = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
#pragma unroll
  for (int i = 0; i < 8; ++i)
    *(uint2*)(priv + n * 256 + (((2 * i + (g >> 1)) ^ n) << 4) + (g & 1) * 8) = v[i];
  asm volatile("" ::: "memory");                      // (other types at the same place)
  patch();
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int r = 4 * q + g;
    put(r, 64 * (n >> 2) + 32 * (wave >> 2) + 8 * (n & 3),
        *(const uint4*)(priv + r * 256 + ((n ^ r) << 4)));
  }
  asm volatile("" ::: "memory");
}

}  // namespace crbq
