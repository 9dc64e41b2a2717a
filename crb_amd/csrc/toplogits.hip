// The k largest logits of each row with their indices (ties to the lowest
// index) and the row's log-sum-exp: what a teacher leaves behind for
// distillation instead of its logits.
//
// One workgroup a row.  One pass over the row takes each thread's largest logit
// and its sum of exponentials against that (rescaled the few times the largest
// one rises): 8.5 vector instructions' time an element, below the time its bytes
// take.  The k-th largest of the threads' maxima is a lower bound of the row's k-th
// largest logit that only about k elements reach (with k of 1024 threads hit, -1024
// log(1 - k / 1024) elements: 137 for k = 128).  Each thread keeps the largest logit of
// each of its 16-byte groups (every 16th of them where it has more than 16) and
// reads those groups again that reach the bound: about k of them, where all groups of
// all threads whose maximum reaches it cost as much as the row over again (2047 rows of
// 128256: 85 us of 200).  What they hold above the bound is ranked by counting.  Rows whose
// ties leave more candidates than the list holds (a constant row, a row masked to one
// value) and rows with a NaN are selected exactly, by digits of the key.
// Measured, 16 bits: 2047 x 128256, k = 128, in 123 us (4.3 TB/s), 2047 x 50272 in 63;
// 301 x 32007 in fp32, 19; one row of 50272, 12 us: the latency of its steps.
// Logits are compared as whole numbers in the order of the values (-0 as
// +0, NaN above everything); the values written are the logits themselves.
#include "common.h"

namespace crbq {

constexpr int TL_SCALAR = 2560;         // rows up to this: one element a thread and step
constexpr int TL_GROUPS = 16;           // group maxima a thread keeps

template <typename E> struct TL;
template <> struct TL<float> {
  typedef uint32_t bits;
  static constexpr int DIGITS = 4;
  __device__ static float f(uint32_t b) { return __builtin_bit_cast(float, b); }
  __device__ static uint32_t bits_of(float x) { return __builtin_bit_cast(uint32_t, x); }
  __device__ static uint32_t key(uint32_t b) {
    if ((b & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
    if (b == 0x80000000u) b = 0;
    return b & 0x80000000u ? ~b : b | 0x80000000u;
  }
};
template <uint16_t INF>
struct TL16 {
  typedef uint16_t bits;
  static constexpr int DIGITS = 2;
  __device__ static uint32_t key(uint32_t b) {
    if ((b & 0x7fffu) > INF) return 0xffffu;
    if (b == 0x8000u) b = 0;
    return (b & 0x8000u ? ~b : b | 0x8000u) & 0xffffu;
  }
};
template <> struct TL<_Float16> : TL16<0x7c00> {
  __device__ static float f(uint32_t b) { return (float)__builtin_bit_cast(_Float16, (uint16_t)b); }
  __device__ static uint32_t bits_of(float x) {       // x is one of the logits
    return __builtin_bit_cast(uint16_t, (_Float16)x);
  }
};
template <> struct TL<__bf16> : TL16<0x7f80> {
  __device__ static float f(uint32_t b) { return __builtin_bit_cast(float, b << 16); }
  __device__ static uint32_t bits_of(float x) { return __builtin_bit_cast(uint32_t, x) >> 16; }
};

// A row as the threads share it: 16-byte groups from the first 16-byte boundary
// on (long rows), elements one by one before and behind.
template <typename E, int NT>
struct TLRow {
  typedef typename TL<E>::bits B;
  static constexpr int N = 16 / sizeof(B);
  const B* x;
  int64_t V, nv;
  int head;
  const uint4* q;
  __device__ TLRow(const B* row, int64_t V_) : x(row), V(V_) {
    head = V <= TL_SCALAR ? (int)V : (int)(((16 - ((uintptr_t)x & 15)) & 15) / sizeof(B));
    nv = (V - head) / N;
    q = (const uint4*)(x + head);
  }
  __device__ static uint32_t bits(const uint4& u, int e) {
    const uint32_t w = e * sizeof(B) / 4 == 0 ? u.x : e * sizeof(B) / 4 == 1 ? u.y
                     : e * sizeof(B) / 4 == 2 ? u.z : u.w;
    return N == 4 ? w : (w >> (16 * (e & 1))) & 0xffffu;
  }
  // f(index, bits) for this thread's elements
  template <typename F>
  __device__ __forceinline__ void each(F&& f) const {
    const int tid = threadIdx.x;
    for (int64_t i = tid; i < nv; i += NT) {
      const uint4 u = q[i];
#pragma unroll
      for (int e = 0; e < N; ++e) f((int)(head + i * N + e), bits(u, e));
    }
    for (int64_t i = tid; i < head; i += NT) f((int)i, (uint32_t)x[i]);
    for (int64_t i = head + nv * N + tid; i < V; i += NT) f((int)i, (uint32_t)x[i]);
  }
};

// A thread's largest logit m and s = sum of 2^(c (x - m)) (against 0 where m is
// infinite; a NaN makes s one).
struct TLSum {
  float m = -INFINITY, s = 0.f, ref = 0.f;
  __device__ __forceinline__ void rise(float top, float c) {
    if (top > m) {
      const float r = fabsf(top) < INFINITY ? top : 0.f;
      s = m == -INFINITY ? s : s * __builtin_amdgcn_exp2f((ref - r) * c);
      m = top;
      ref = r;
    }
  }
  __device__ __forceinline__ void add(float x, float c) {
    s += __builtin_amdgcn_exp2f((x - ref) * c);        // (x * c may be beyond fp32)
  }
};

template <typename E, int NT>
__global__ __launch_bounds__(NT) void k_top_logits(const void* logits, int64_t V,
                                                           int64_t ld, int k, float itemp,
                                                           void* val, int32_t* __restrict__ idx,
                                                           float* __restrict__ lse) {
  constexpr int TL_WAVES = NT / 64;
  constexpr int TL_LOG = NT == 1024 ? 4 : NT == 512 ? 3 : 2;     // log2 of the wavefronts
  constexpr int TL_CAP = NT == 256 ? 1024 : 2048;                // candidates
  typedef TL<E> L;
  typedef typename L::bits B;
  __shared__ uint32_t tmax[NT];
  __shared__ uint64_t cand[TL_CAP];     // key << 32 | ~index: larger is earlier
  __shared__ float wred[TL_WAVES], wsum[TL_WAVES];
  __shared__ int hist[256];
  __shared__ uint32_t sh[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t t = blockIdx.x;
  const B* x = (const B*)logits + t * ld;

  const TLRow<E, NT> row(x, V);
  constexpr int N = TLRow<E, NT>::N;
  const float c = itemp * 1.4426950408889634f;
  TLSum acc;
  auto group = [&](const uint4& u) __attribute__((always_inline)) {
    float v[N];
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = L::f(TLRow<E, NT>::bits(u, e));
    float top = v[0];
#pragma unroll
    for (int e = 1; e < N; ++e) top = fmaxf(top, v[e]);
    acc.rise(top, c);
#pragma unroll
    for (int e = 0; e < N; ++e) acc.add(v[e], c);
    return top;
  };
  float gm[TL_GROUPS];                                 // maximum of groups i, i + 16, ...
#pragma unroll
  for (int i = 0; i < TL_GROUPS; ++i) gm[i] = -INFINITY;
  for (int64_t g0 = tid; g0 - tid < row.nv; g0 += (int64_t)TL_GROUPS * NT) {
#pragma unroll
    for (int i0 = 0; i0 < TL_GROUPS; i0 += 4) {
      const int64_t g = g0 + (int64_t)i0 * NT;
      if (g - tid >= row.nv) break;
      uint4 u[4];
#pragma unroll
      for (int d = 0; d < 4; ++d)
        u[d] = row.q[g + d * NT < row.nv ? g + d * NT : row.nv - 1];
#pragma unroll
      for (int d = 0; d < 4; ++d)
        if (g + d * NT < row.nv) gm[i0 + d] = fmaxf(gm[i0 + d], group(u[d]));
    }
  }
  auto one = [&](int64_t i) __attribute__((always_inline)) {
    const float v = L::f((uint32_t)x[i]);
    acc.rise(v, c);
    acc.add(v, c);
  };
  for (int64_t i = tid; i < row.head; i += NT) one(i);
  for (int64_t i = row.head + row.nv * N + tid; i < V; i += NT) one(i);
  const bool some = V >= NT || tid < V;        // threads without an element: key 0
  const uint32_t best = some ? L::key(L::bits_of(acc.m)) : 0;
  tmax[tid] = best;
  if (tid == 0) sh[1] = 0;
  // the row's maximum, and its sum of exponentials against it
  float top = acc.m;
#pragma unroll
  for (int d = 32; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
  if (lane == 0) wred[wave] = top;
  __syncthreads();
  for (int w = 0; w < TL_WAVES; ++w) top = fmaxf(top, wred[w]);
  const float ref = fabsf(top) < INFINITY ? top : 0.f;
  // (-inf: s is 0 or NaN; below an infinite maximum only NaN matters)
  const float part = acc.m == -INFINITY || !(fabsf(top) < INFINITY)
                         ? acc.s : acc.s * __builtin_amdgcn_exp2f((acc.ref - ref) * c);
  const float sum = wave_sum_f(part);
  if (lane == 0) wsum[wave] = sum;
  // the k-th largest of the maxima, TL_LOG bits at a time from the top:
  // wavefront w counts the maxima that reach w as the next bits (one wavefront
  // bit by bit waits for a count as often as there are bits)
  uint32_t mine[TL_WAVES], thr = 0;
#pragma unroll
  for (int w = 0; w < TL_WAVES; ++w) mine[w] = tmax[w * 64 + lane];
  constexpr int STEPS = (L::DIGITS * 8 + TL_LOG - 1) / TL_LOG;
#pragma unroll 1
  for (int d = STEPS - 1; d >= 0; --d) {
    // (the top step may have bits that no key has)
    const uint64_t want = thr | (uint64_t)wave << (TL_LOG * d);
    int n = 0;
#pragma unroll
    for (int w = 0; w < TL_WAVES; ++w) n += __popcll(__ballot(mine[w] >= want));
    int* cnt = hist + (d & 1) * TL_WAVES;
    if (lane == 0) cnt[wave] = n;
    __syncthreads();
    const uint64_t ok = __ballot(lane < TL_WAVES && cnt[lane & (TL_WAVES - 1)] >= k);
    thr |= (uint32_t)(63 - __clzll((long long)(ok | 1))) << (TL_LOG * d);
  }
  float s = 0.f;
  for (int w = 0; w < TL_WAVES; ++w) s += wsum[w];
  const bool nan = !(s == s);
  if (tid == 0) lse[t] = nan || fabsf(top) < INFINITY ? ref * itemp + logf(s) : top;
  // candidates among n elements from i0 on
  auto take = [&](const uint32_t (&key)[N], int i0, int n) __attribute__((always_inline)) {
    uint32_t hit = 0;
#pragma unroll
    for (int e = 0; e < N; ++e) hit |= (uint32_t)(e < n && key[e] >= thr) << e;
    if (!hit) return;
    uint32_t at = atomicAdd(&sh[1], (uint32_t)__popc(hit));
#pragma unroll
    for (int e = 0; e < N; ++e)
      if ((hit >> e) & 1) {
        if (at < TL_CAP) cand[at] = (uint64_t)key[e] << 32 | (uint32_t)~(i0 + e);
        ++at;
      }
  };
  auto take_one = [&](int64_t i) __attribute__((always_inline)) {
    uint32_t key[N] = {};
    key[0] = L::key((uint32_t)x[i]);
    take(key, (int)i, 1);
  };
  if (best >= thr && !nan) {
    uint32_t todo = 0;
#pragma unroll
    for (int i = 0; i < TL_GROUPS; ++i)
      todo |= (uint32_t)(row.nv > tid && L::key(L::bits_of(gm[i])) >= thr) << i;
    // (a lane's next group whatever the others': their loads run at one time)
    while (todo) {
      const int i = __ffs((int)todo) - 1;
      todo &= todo - 1;
      for (int64_t g = tid + (int64_t)i * NT; g < row.nv;
           g += (int64_t)TL_GROUPS * NT) {
        const uint4 u = row.q[g];
        uint32_t key[N];
#pragma unroll
        for (int e = 0; e < N; ++e) key[e] = L::key(TLRow<E, NT>::bits(u, e));
        take(key, (int)(row.head + g * N), N);
      }
    }
    for (int64_t i = tid; i < row.head; i += NT) take_one(i);
    for (int64_t i = row.head + row.nv * N + tid; i < V; i += NT) take_one(i);
  }
  __syncthreads();
  int n = (int)sh[1];
  if (n > TL_CAP || nan) {
    // too many candidates, or NaN: the k-th key digit by digit, then the elements
    // above it and the first of its equals
    uint32_t pre = 0;
    int need = k;                       // of the elements whose upper digits are pre
    for (int d = L::DIGITS - 1; d >= 0; --d) {
      __syncthreads();
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      row.each([&](int, uint32_t b) {
        const uint32_t q = L::key(b);
        const bool in = d == L::DIGITS - 1 || (q >> (8 * d + 8)) == pre;
        const int dig = (int)((q >> (8 * d)) & 255);
        // one add for a wavefront whose elements agree
        const uint64_t act = __ballot(in);
        if (!in) return;
        const int first = __shfl(dig, __ffsll((unsigned long long)act) - 1);
        const uint64_t same = __ballot(dig == first);
        if (dig != first) atomicAdd(&hist[dig], 1);
        else if (lane == __ffsll((unsigned long long)same) - 1)
          atomicAdd(&hist[dig], __popcll(same));
      });
      __syncthreads();
      if (tid == 0) {
        int c = 0, dig = 255;
        while (dig > 0 && c + hist[dig] < need) c += hist[dig--];
        sh[2] = (uint32_t)dig;
        sh[3] = (uint32_t)c;
      }
      __syncthreads();
      pre = pre << 8 | sh[2];
      need -= (int)sh[3];
    }
    __syncthreads();
    if (tid == 0) sh[1] = 0;
    __syncthreads();
    row.each([&](int i, uint32_t b) {
      const uint32_t q = L::key(b);
      if (q > pre) cand[atomicAdd(&sh[1], 1u)] = (uint64_t)q << 32 | (uint32_t)~i;   // below k
    });
    __syncthreads();
    int have = (int)sh[1];              // k - need
    for (int64_t i0 = 0; i0 < V && have < k; i0 += NT) {
      const int64_t i = i0 + tid;
      const bool eq = i < V && L::key((uint32_t)x[i]) == pre;
      const uint64_t bits = __ballot(eq);
      __syncthreads();
      if (lane == 0) hist[wave] = __popcll(bits);
      __syncthreads();
      int at = have + __popcll(bits & ((1ull << lane) - 1)), all = 0;
      for (int w = 0; w < TL_WAVES; ++w) {
        if (w < wave) at += hist[w];
        all += hist[w];
      }
      if (eq && at < k) cand[at] = (uint64_t)pre << 32 | (uint32_t)~(int)i;
      have += all;
    }
    __syncthreads();
    n = k;
  }
  for (int c = tid; c < n; c += NT) {
    const uint64_t q = cand[c];
    int rank = 0, j = 0;
    for (; j + 4 <= n; j += 4)
      rank += (cand[j] > q) + (cand[j + 1] > q) + (cand[j + 2] > q) + (cand[j + 3] > q);
    for (; j < n; ++j) rank += cand[j] > q;
    if (rank < k) {
      const int i = ~(int)(uint32_t)q;
      idx[t * k + rank] = i;
      ((B*)val)[t * k + rank] = x[i];
    }
  }
}

// Threads a row.  After its pass over the row a workgroup mostly waits, so that with many
// rows what counts is the rows at work on a CU (2, 4 or 8), with few the row's own
// latency, and for k above 128 a bound from 256 maxima is loose.  Measured with k = 100, us
// with 256, 512 and 1024 threads: 256 rows of 32007 in 16 bits 16.9, 13.9, 14.2; of
// 128256 40.8, 26.5, 22.6; 301 rows of 32007 in 32 bits 23.5, 19.3, 27.2; 2047 rows of 8000
// 28.6, 36.5, 67; of 32007 45, 50, 84; of 50272 61, 58, 96; of 128256 133, 118, 151.
template <typename E>
static void top_logits(const void* logits, int64_t T, int64_t V, int64_t ld, int k, float it,
                       void* val, int32_t* idx, float* lse, hipStream_t s) {
  const int64_t bytes = V * (int64_t)sizeof(E);
  if (T <= 256 && bytes > 160 * 1024)
    k_top_logits<E, 1024><<<(unsigned)T, 1024, 0, s>>>(logits, V, ld, k, it, val, idx, lse);
  else if (T <= 512 || k > 128 || bytes > 96 * 1024)
    k_top_logits<E, 512><<<(unsigned)T, 512, 0, s>>>(logits, V, ld, k, it, val, idx, lse);
  else
    k_top_logits<E, 256><<<(unsigned)T, 256, 0, s>>>(logits, V, ld, k, it, val, idx, lse);
}

}  // namespace crbq

using namespace crbq;

extern "C" int crbq_top_logits(const void* logits, int dtype, int64_t T, int64_t V, int64_t ld,
                               int k, float temperature, void* val, int32_t* idx, float* lse,
                               void* stream) {
  if (!logits || !val || !idx || !lse || T < 1 || T >= ((int64_t)1 << 31) || V < 1 ||
      V >= ((int64_t)1 << 31) - 2048 || ld < V || k < 1 || k > CRBQ_HEAD_MAX_K || k > V ||
      !(temperature > 0.f))
    return CRBQ_ERR_ARG;
  hipStream_t s = (hipStream_t)stream;
  const float it = 1.f / temperature;
  switch (dtype) {
    case CRBQ_F32: top_logits<float>(logits, T, V, ld, k, it, val, idx, lse, s); break;
    case CRBQ_F16: top_logits<_Float16>(logits, T, V, ld, k, it, val, idx, lse, s); break;
    case CRBQ_BF16: top_logits<__bf16>(logits, T, V, ld, k, it, val, idx, lse, s); break;
    default: return CRBQ_ERR_ARG;
  }
  CRBQ_LAUNCH_CHECK();
  return CRBQ_OK;
}
