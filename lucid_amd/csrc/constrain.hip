// Constraints on the next token on CDNA4 (gfx950): logit rows with the penalties of tokens that have occurred, a bias and
// a bit mask of allowed tokens (no counterpart in the reference; stands beside token_logprobs.hip).  For row r and token v, with
// N_rv the times that v occurs in the row's history from its prompt's end on:
//   x = logit;  if v occurs in the history: x = x > 0 ? x / rho : x rho;  x = x - pi [N_rv > 0] - phi N_rv;
//   x = x + bias_v;  -inf where v is not allowed
// Its gradient is 1, 1 / rho or rho (by the logit's sign), 0 where v is not allowed.
#include "logit_rows.h"

namespace lucid {

constexpr int kConstrainSeg = 8192;  // values of a workgroup, a counter in LDS for each
constexpr unsigned kConstrainSeen = 0x80000000u;  // of a counter: the token occurs in the prompt

struct ConstrainRows {
  const int64_t* history;  // [R][N] at hstride, negative: none
  int64_t hstride;
  int N;
  const int32_t* prompt;  // [R] or null: none of it is a prompt
  const float *rep, *pres, *freq;  // [R] or null: the value beside
  float rep0, pres0, freq0;
  const float* bias;  // [R][V] at bstride, or null
  int64_t bstride;
  const uint32_t* allowed;  // [R][ceil(V / 32)] at astride, or null
  int64_t astride;
};

// Bits j .. j+7 of a row's mask of V (beyond them 0)
__device__ __forceinline__ unsigned allowed_bits(const uint32_t* m, int j, int V) {
  const int word = j >> 5, last = (V - 1) >> 5;
  const unsigned lo = word >= 0 && word <= last ? m[word] : 0u, hi = word + 1 <= last && word + 1 >= 0 ? m[word + 1] : 0u;
  return (unsigned)((((uint64_t)hi << 32) | lo) >> (j & 31));
}

// Grid R x segments, 512 threads.  BWD: x is the incoming gradient and raw the logits' row, whose sign is asked for where a
// token has occurred.
template <typename T, bool HIST, bool BWD>
__global__ __launch_bounds__(512) void lucid_constrain_kernel(const T* __restrict__ x, int64_t sb, int64_t st,
                                                              const T* __restrict__ raw, int64_t rb, int64_t rt, int Tn, int V,
                                                              int segs, ConstrainRows a, T* __restrict__ out) {
  constexpr int NT = 512, N = LpRow<T>::N, C = kConstrainSeg / NT / N;
  __shared__ unsigned count[HIST ? kConstrainSeg : 1];
  const int r = blockIdx.x / segs, seg = blockIdx.x - r * segs, tid = threadIdx.x;
  const LpRow<T> row(lp_row(x, sb, st, Tn, r), V);
  const int q0 = seg * NT * C + tid, lo = row.first(seg * NT * C);  // (may be negative: the first chunk)
  typename LpRow<T>::V xv[C];
#pragma unroll
  for (int c = 0; c < C; ++c)
    if (row.first(q0 + c * NT) < V) xv[c] = row.load(q0 + c * NT);
  if constexpr (HIST) {
#pragma unroll
    for (int i = tid; i < kConstrainSeg; i += NT) count[i] = 0;
    __syncthreads();
    const int64_t* h = a.history + r * a.hstride;
    const int from = a.prompt ? a.prompt[r] : 0;
#pragma unroll 8
    for (int i = tid; i < a.N; i += NT) {
      const int64_t v = h[i];
      const int64_t at = v - lo;
      if (v >= 0 && v < V && at >= 0 && at < kConstrainSeg) {
        if (i >= from)
          atomicAdd(&count[at], 1u);
        else
          atomicOr(&count[at], kConstrainSeen);
      }
    }
    __syncthreads();
  }
  const float rho = a.rep ? a.rep[r] : a.rep0, pi = a.pres ? a.pres[r] : a.pres0, phi = a.freq ? a.freq[r] : a.freq0;
  const uint32_t* mask = a.allowed ? a.allowed + r * a.astride : nullptr;
  const float* bias = a.bias ? a.bias + r * a.bstride : nullptr;
  const T* rr = BWD ? lp_row(raw, rb, rt, Tn, r) : nullptr;
  T* orow = out + (int64_t)r * V;
  const bool same = (reinterpret_cast<uintptr_t>(orow) & 15) / sizeof(T) == (unsigned)row.shift;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int q = q0 + c * NT, j = row.first(q);
    if (j >= V) break;
    const unsigned ok = mask ? allowed_bits(mask, j, V) : ~0u;
    typename LpRow<T>::V o;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      float y = (float)xv[c][e];
      if constexpr (HIST) {
        const unsigned n = count[j + e - lo];
        if (n) {
          if constexpr (BWD) {
            const float z = j + e >= 0 && j + e < V ? (float)rr[j + e] : 0.f;
            y = z > 0.f ? y / rho : y * rho;
          } else {
            y = y > 0.f ? y / rho : y * rho;
            const unsigned k = n & ~kConstrainSeen;
            if (k) y = (y - pi) - phi * (float)k;
          }
        }
      }
      if (!BWD && bias && j + e >= 0 && j + e < V) y += bias[j + e];
      if (!(ok >> e & 1)) y = BWD ? 0.f : -INFINITY;
      o[e] = (T)y;
    }
    if (same && row.whole(q)) {
      *reinterpret_cast<typename LpRow<T>::V*>(orow + j) = o;
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (j + e >= 0 && j + e < V) orow[j + e] = o[e];
    }
  }
}

}  // namespace lucid
