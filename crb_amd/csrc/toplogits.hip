// The k largest logits of each row with their indices (ties to the lowest
// index) and the row's log-sum-exp: what a teacher leaves behind for
// distillation instead of its logits.
//
// One workgroup of 1024 threads a row.  A first pass takes each thread's
// largest logit; the k-th largest of these 1024 is a lower bound of the
// row's k-th largest logit that only about k elements reach (with k of 1024
// threads hit, -1024 log(1 - k / 1024) elements: 137 for k = 128).  A second
// pass sums the exponentials against the row's maximum and collects the
// elements at or above the bound, which are then ranked by counting.  Rows
// whose ties leave more candidates than the list holds (a constant row, a
// row masked to one value) are selected exactly, by digits of the key.
// Logits are compared as whole numbers in the order of the values (-0 as
// +0, NaN above everything); the values written are the logits themselves.
#include "common.h"

namespace crbq {

constexpr int TL_THREADS = 1024;
constexpr int TL_WAVES = TL_THREADS / 64;
constexpr int TL_CAP = 2048;            // candidates
constexpr int TL_SCALAR = 8192;         // rows up to this: one element a thread and step

template <typename E> struct TL;
template <> struct TL<float> {
  typedef uint32_t bits;
  static constexpr int DIGITS = 4;
  __device__ static float f(uint32_t b) { return __builtin_bit_cast(float, b); }
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
};
template <> struct TL<__bf16> : TL16<0x7f80> {
  __device__ static float f(uint32_t b) { return __builtin_bit_cast(float, b << 16); }
};

// f(index, bits) for every element of the row: 16-byte loads from the first
// 16-byte boundary on (long rows), elements one by one before and behind.
template <typename E, typename F>
__device__ __forceinline__ void tl_each(const typename TL<E>::bits* __restrict__ x, int64_t V,
                                        F&& f) {
  typedef typename TL<E>::bits B;
  constexpr int N = 16 / sizeof(B);
  const int tid = threadIdx.x;
  if (V <= TL_SCALAR) {
    for (int64_t i = tid; i < V; i += TL_THREADS) f((int)i, (uint32_t)x[i]);
    return;
  }
  const int head = (int)(((16 - ((uintptr_t)x & 15)) & 15) / sizeof(B));
  const int64_t nv = (V - head) / N;
  const uint4* __restrict__ q = (const uint4*)(x + head);
  for (int64_t i = tid; i < nv; i += TL_THREADS) {
    const uint4 u = q[i];
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const uint32_t b = N == 4 ? w[e] : (w[e / 2] >> (16 * (e & 1))) & 0xffffu;
      f((int)(head + i * N + e), b);
    }
  }
  if (tid < head) f(tid, (uint32_t)x[tid]);
  for (int64_t i = head + nv * N + tid; i < V; i += TL_THREADS) f((int)i, (uint32_t)x[i]);
}

template <typename E>
__global__ __launch_bounds__(TL_THREADS) void k_top_logits(const void* logits, int64_t V,
                                                           int64_t ld, int k, float itemp,
                                                           void* val, int32_t* __restrict__ idx,
                                                           float* __restrict__ lse) {
  typedef TL<E> L;
  typedef typename L::bits B;
  __shared__ uint32_t tmax[TL_THREADS];
  __shared__ uint64_t cand[TL_CAP];     // key << 32 | ~index: larger is earlier
  __shared__ float wred[TL_WAVES];
  __shared__ int hist[256];
  __shared__ uint32_t sh[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t t = blockIdx.x;
  const B* x = (const B*)logits + t * ld;

  uint32_t best = 0;
  tl_each<E>(x, V, [&](int, uint32_t b) {
    const uint32_t q = L::key(b);
    best = q > best ? q : best;
  });
  tmax[tid] = best;
  if (tid == 0) sh[1] = 0;
  __syncthreads();
  // k-th largest of the 1024, by its bits from the top; every wavefront for itself
  uint32_t mine[TL_WAVES], top = 0;
#pragma unroll
  for (int w = 0; w < TL_WAVES; ++w) {
    mine[w] = tmax[w * 64 + lane];
    top = mine[w] > top ? mine[w] : top;
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    const uint32_t o = __shfl_xor(top, d);
    top = o > top ? o : top;
  }
  if (wave == 0) {
    uint32_t thr = 0;
#pragma unroll 1
    for (int bit = L::DIGITS * 8 - 1; bit >= 0; --bit) {
      const uint32_t c = thr | (1u << bit);
      int n = 0;
#pragma unroll
      for (int w = 0; w < TL_WAVES; ++w) n += __popcll(__ballot(mine[w] >= c));
      if (n >= k) thr = c;
    }
    if (lane == 0) sh[0] = thr;
  }
  __syncthreads();
  const uint32_t thr = sh[0];
  // the row's maximum as a float (NaN and infinities: reference 0)
  const uint32_t tb = top >> (L::DIGITS * 8 - 1) ? top & ~(1u << (L::DIGITS * 8 - 1))
                                                 : ~top & (L::DIGITS == 4 ? 0xffffffffu : 0xffffu);
  float m = L::f(tb) * itemp;
  if (!(fabsf(m) < INFINITY)) m = 0.f;

  float s = 0.f;
  tl_each<E>(x, V, [&](int i, uint32_t b) {
    s += __expf(L::f(b) * itemp - m);
    const uint32_t q = L::key(b);
    if (q >= thr) {
      const uint32_t at = atomicAdd(&sh[1], 1u);
      if (at < TL_CAP) cand[at] = (uint64_t)q << 32 | (uint32_t)~i;
    }
  });
  s = wave_sum_f(s);
  if (lane == 0) wred[wave] = s;
  __syncthreads();
  if (tid == 0) {
    s = 0.f;
    for (int w = 0; w < TL_WAVES; ++w) s += wred[w];
    lse[t] = m + logf(s);
  }
  int n = (int)sh[1];
  if (n > TL_CAP) {
    // too many candidates: the k-th key digit by digit, then the elements
    // above it and the first of its equals
    uint32_t pre = 0;
    int need = k;                       // of the elements whose upper digits are pre
    for (int d = L::DIGITS - 1; d >= 0; --d) {
      __syncthreads();
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      tl_each<E>(x, V, [&](int, uint32_t b) {
        const uint32_t q = L::key(b);
        const bool in = d == L::DIGITS - 1 || (q >> (8 * d + 8)) == pre;
        const int dig = (int)((q >> (8 * d)) & 255);
        // one add for a wavefront whose elements agree
        const uint64_t act = __ballot(in);
        if (!in) return;
        const int first = __shfl(dig, __ffsll((unsigned long long)act) - 1);
        const uint64_t same = __ballot(dig == first);
        if (dig != first) atomicAdd(&hist[dig], 1);
        else if (lane == __ffsll((unsigned long long)same) - 1) atomicAdd(&hist[dig], __popcll(same));
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
    tl_each<E>(x, V, [&](int i, uint32_t b) {
      const uint32_t q = L::key(b);
      if (q > pre) cand[atomicAdd(&sh[1], 1u)] = (uint64_t)q << 32 | (uint32_t)~i;   // below k
    });
    __syncthreads();
    int have = (int)sh[1];              // k - need
    for (int64_t i0 = 0; i0 < V && have < k; i0 += TL_THREADS) {
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
  for (int c = tid; c < n; c += TL_THREADS) {
    const uint64_t q = cand[c];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += cand[j] > q;
    if (rank < k) {
      const int i = ~(int)(uint32_t)q;
      idx[t * k + rank] = i;
      ((B*)val)[t * k + rank] = x[i];
    }
  }
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
    case CRBQ_F32:
      k_top_logits<float><<<(unsigned)T, TL_THREADS, 0, s>>>(logits, V, ld, k, it, val, idx, lse);
      break;
    case CRBQ_F16:
      k_top_logits<_Float16><<<(unsigned)T, TL_THREADS, 0, s>>>(logits, V, ld, k, it, val, idx, lse);
      break;
    case CRBQ_BF16:
      k_top_logits<__bf16><<<(unsigned)T, TL_THREADS, 0, s>>>(logits, V, ld, k, it, val, idx, lse);
      break;
    default: return CRBQ_ERR_ARG;
  }
  CRBQ_LAUNCH_CHECK();
  return CRBQ_OK;
}
