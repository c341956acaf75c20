// Constraints on the next token on CDNA4 (gfx950): logit rows with the penalties of tokens that have occurred, a bias and
// a bit mask of allowed tokens (no counterpart in the reference; stands beside token_logprobs.hip).  For row r and token v, with
// N_rv the times that v occurs in the row's history from its prompt's end on:
//   x = logit;  if v occurs in the history: x = x > 0 ? x / rho : x rho;  x = x - pi [N_rv > 0] - phi N_rv;
//   x = x + bias_v;  -inf where v is not allowed
// Its gradient is 1, 1 / rho or rho (by the logit's sign), 0 where v is not allowed.  One read and one write of the rows, a
// segment of 8192 values to a workgroup; each reads the row's whole history, which the caches hold.  HBM bounds large calls: 8192 rows
// of 32000 bf16 values behind 500 tokens, 1.05 GB, 236 us, 4.4 TB/s, and their gradient, 1.05 GB, 250 us; 64 of 131072 behind
// 4000, 35 MB, 15 us; 4 of 32003 fp32 values behind 100000 tokens 24 us: 16 workgroups, each over its row's whole history.
#include "logit_rows.h"

namespace lucid {

typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));  // four values at any address

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

// Whether a history's token names a value of the segment from lo on, and which
__device__ __forceinline__ bool constrain_names(int64_t v, int lo, int V, unsigned& at) {
  at = (unsigned)((int)v - lo);
  return (uint64_t)v < (unsigned)V && at < (unsigned)kConstrainSeg;
}

constexpr int kConstrainThreads = 512;
constexpr int kConstrainHeld = 8;  // tokens of a history that a lane holds

// How a workgroup finds the tokens of its segment that have occurred
enum class History {
  None,
  Counted,  // a counter of each value in LDS (clearing only those of tokens held in registers, with a bit a value for the rest,
            // was a tenth slower: 64 rows of 131072 behind 4000 tokens, 256 of 32000 fp32 behind 2000)
  Held,     // the gradient of up to 512 kConstrainHeld tokens: a bit of each value for an occurrence and for a logit above 0, both
            // from the tokens themselves, held in registers (8192 rows of 32000 behind 500 tokens, with the forward: 472 us; with
            // counters, and the logits looked up value by value, 582)
};

// Grid R x segments.  BWD: x is the incoming gradient and raw the logits' row, whose sign is asked for where a
// token has occurred.
// PAST: the results pass the caches by (the launcher's rule).
template <typename T, History H, bool BWD, bool PAST>
__global__ __launch_bounds__(kConstrainThreads) void lucid_constrain_kernel(const T* __restrict__ x, int64_t sb, int64_t st,
                                                                            const T* __restrict__ raw, int64_t rb, int64_t rt,
                                                                            int Tn, int V, int segs, ConstrainRows a,
                                                                            T* __restrict__ out) {
  constexpr int NT = kConstrainThreads, N = LpRow<T>::N, C = kConstrainSeg / NT / N;
  static_assert(BWD || H != History::Held, "a forward counts");
  __shared__ __attribute__((aligned(16))) unsigned count[H == History::Counted ? kConstrainSeg : 4];
  __shared__ unsigned bits[H == History::Held ? kConstrainSeg / 32 : 1];
  __shared__ unsigned plus[H == History::Held ? kConstrainSeg / 32 : 1];  // of tokens whose logit is positive
  const int r = blockIdx.x / segs, seg = blockIdx.x - r * segs, tid = threadIdx.x;
  const LpRow<T> row(lp_row(x, sb, st, Tn, r), V);
  const int q0 = seg * NT * C + tid, lo = row.first(seg * NT * C);  // (lo may be negative: the first chunk)
  const int64_t* h = H == History::None ? nullptr : a.history + r * a.hstride;
  const int from = H == History::None || BWD || !a.prompt ? 0 : a.prompt[r];
  const T* rr = BWD ? lp_row(raw, rb, rt, Tn, r) : nullptr;
  int64_t held[H == History::Held ? kConstrainHeld : 1];
  if constexpr (H == History::Held) {
#pragma unroll
    for (int k = 0; k < kConstrainHeld; ++k)
      if (k * NT < a.N) held[k] = k * NT + tid < a.N ? h[k * NT + tid] : -1;
  }
  typename LpRow<T>::V xv[C];
#pragma unroll
  for (int c = 0; c < C; ++c)
    if (row.first(q0 + c * NT) < V) xv[c] = row.load(q0 + c * NT);
  // what else a value takes is asked for here too, before anything waits
  const float rho = a.rep ? a.rep[r] : a.rep0, pi = a.pres ? a.pres[r] : a.pres0, phi = a.freq ? a.freq[r] : a.freq0;
  const uint32_t* mask = a.allowed ? a.allowed + r * a.astride : nullptr;
  const float* bias = a.bias ? a.bias + r * a.bstride : nullptr;
  unsigned ok[C];
  float bv[BWD ? 1 : C][N];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int q = q0 + c * NT, j = row.first(q);
    ok[c] = mask && j < V ? allowed_bits(mask, j, V) : ~0u;
    if constexpr (!BWD) {
#pragma unroll
      for (int e = 0; e < N; ++e) bv[c][e] = 0.f;
      if (bias && row.whole(q)) {
#pragma unroll
        for (int e = 0; e < N; e += 4) {
          const f32x4_any z = *reinterpret_cast<const f32x4_any*>(bias + j + e);
#pragma unroll
          for (int k = 0; k < 4; ++k) bv[c][e + k] = z[k];
        }
      } else if (bias) {
#pragma unroll
        for (int e = 0; e < N; ++e)
          if (j + e >= 0 && j + e < V) bv[c][e] = bias[j + e];
      }
    }
  }
  if constexpr (H == History::Held) {
    unsigned at;
    if (tid < kConstrainSeg / 32) {
      bits[tid] = 0;
      plus[tid] = 0;
    }
    bool up[kConstrainHeld];
#pragma unroll
    for (int k = 0; k < kConstrainHeld; ++k)
      up[k] = k * NT < a.N && constrain_names(held[k], lo, V, at) && (float)rr[held[k]] > 0.f;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kConstrainHeld; ++k)
      if (k * NT < a.N && constrain_names(held[k], lo, V, at)) {
        atomicOr(&bits[at >> 5], 1u << (at & 31));
        if (up[k]) atomicOr(&plus[at >> 5], 1u << (at & 31));
      }
    __syncthreads();
  } else if constexpr (H == History::Counted) {
    for (int i = tid; i < kConstrainSeg / 4; i += NT) *reinterpret_cast<u32x4*>(&count[4 * i]) = u32x4{0, 0, 0, 0};
    __syncthreads();
    for (int i0 = tid; i0 < a.N; i0 += kConstrainHeld * NT) {
      int64_t v[kConstrainHeld];
#pragma unroll
      for (int k = 0; k < kConstrainHeld; ++k) v[k] = i0 + k * NT < a.N ? h[i0 + k * NT] : -1;
#pragma unroll
      for (int k = 0; k < kConstrainHeld; ++k) {
        unsigned at;
        if (constrain_names(v[k], lo, V, at)) {
          if (i0 + k * NT >= from)
            atomicAdd(&count[at], 1u);
          else
            atomicOr(&count[at], kConstrainSeen);
        }
      }
    }
    __syncthreads();
  }
  T* orow = out + (int64_t)r * V;
  const bool same = (reinterpret_cast<uintptr_t>(orow) & 15) / sizeof(T) == (unsigned)row.shift;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int q = q0 + c * NT, j = row.first(q);
    if (j >= V) break;
    float y[N];
#pragma unroll
    for (int e = 0; e < N; ++e) y[e] = (float)xv[c][e];
    if constexpr (H != History::None) {
      const int at = (q - seg * NT * C) * N;  // j - lo
      unsigned n[N], positive = 0;
      bool any = false;
      if constexpr (H == History::Held) {
        const unsigned b = bits[at >> 5] >> (at & 31);
        any = (b & ((1u << N) - 1)) != 0;
        positive = plus[at >> 5] >> (at & 31);
        if (any) {
#pragma unroll
          for (int e = 0; e < N; ++e) n[e] = b >> e & 1 ? kConstrainSeen : 0u;
        }
      } else {
#pragma unroll
        for (int e = 0; e < N; e += 4) {
          const u32x4 z = *reinterpret_cast<const u32x4*>(&count[at + e]);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            n[e + k] = z[k];
            any |= z[k] != 0;
          }
        }
      }
      if (any) {
#pragma unroll
        for (int e = 0; e < N; ++e)
          if (n[e]) {
            const bool up = !BWD                      ? y[e] > 0.f
                            : H == History::Held ? (positive >> e & 1)
                                                 : j + e >= 0 && j + e < V && (float)rr[j + e] > 0.f;
            y[e] = up ? y[e] / rho : y[e] * rho;
            const unsigned k = n[e] & ~kConstrainSeen;
            if (!BWD && k) y[e] = (y[e] - pi) - phi * (float)k;
          }
      }
    }
    typename LpRow<T>::V o;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      if (!BWD) y[e] += bv[BWD ? 0 : c][e];
      if (!(ok[c] >> e & 1)) y[e] = BWD ? 0.f : -INFINITY;
      o[e] = (T)y[e];
    }
    if (same && row.whole(q)) {
      auto* to = reinterpret_cast<typename LpRow<T>::V*>(orow + j);
      if constexpr (PAST)
        __builtin_nontemporal_store(o, to);
      else
        *to = o;
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (j + e >= 0 && j + e < V) orow[j + e] = o[e];
    }
  }
}

}  // namespace lucid
