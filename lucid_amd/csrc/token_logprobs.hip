// Log probabilities of given tokens, entropy and the top alternatives of logit rows, and their
// gradient, on CDNA4 (gfx950); stands beside the causal-LM loss of model_ops.hip
// (modeling_lucid.py:847-967 has the logits; the reference reads nothing but the mean loss from
// them).  With x = logits / temperature, a row of V values:
//   lse = log sum_j exp x_j,  p_j = exp(x_j - lse)
//   logprob = x_tok - lse,  entropy H = -sum_j p_j log p_j = log s - t / s,
//     s = sum_j exp(x_j - m), t = sum_j exp(x_j - m) (x_j - m), m = max_j x_j
//   alternatives: the `top` largest logits, ties by the lowest index, with x_i - lse
//   dx_j = [j = tok] g_lp + sum_i [j = top_i] g_i - p_j (g_lp + sum_i g_i + g_H (log p_j + H))
//
//   lucid_token_logprobs_kernel        a workgroup per row (or per 32768-value segment of it) keeps
//                                      its values in registers: one read of the logits serves the
//                                      maximum, the sums and the alternatives
//   lucid_token_logprobs_merge_kernel  rows of several segments: the segments' sums and sorted
//                                      alternatives joined
//   lucid_token_logprobs_bwd_kernel    one read of the logits and one write of their gradient
#include "lucid_common.h"

namespace lucid {

constexpr int kLpLane = 32;     // logits a lane holds, in chunks of 16 bytes
constexpr int kLpMaxTop = 64;   // alternatives of a row
constexpr int kLpCand = 1024;   // values considered for the alternatives of a segment
constexpr int kLpMaxSegs = 64;  // segments of a row
constexpr float kLpNone = -1000.f;  // a log2 probability whose exp2 is 0: stands for every lower one
// Largest |m c| whose wave takes a = x c - m c in one fma: the product's rounding, by which every a is then off, is
// at most 2^-5 below it and leaves exactly.  Beyond it (a wave of values all masked with -1e9, say) the rounding grows
// to whole powers of two, from 2^31 on past exp2's range.
constexpr float kLpOneStep = 1048576.f;

// What a forward row leaves for the backward: p_j = exp2(a_j - l2), a_j = (logit_j - m) c with c = log2 e /
// temperature (the difference first: one of two logits of the type's lowest value is 0, where their products
// with c overflow)
struct LpStats {
  float m, l2, ent;
};

// A row of logits as aligned chunks of N = 16 bytes: chunk q holds the values N q - shift + e, e < N, so that
// every whole chunk starts at a 16-byte boundary (rows of odd V do not); the first and the last chunk may lie
// partly outside the row and are read value by value.
template <typename T>
struct LpRow {
  static constexpr int N = 16 / sizeof(T), C = kLpLane / N;  // values of a chunk, chunks of a lane
  typedef T V __attribute__((ext_vector_type(N)));
  const T* row;
  int len, shift;
  __device__ __forceinline__ LpRow(const T* r, int v)
      : row(r), len(v), shift((int)((reinterpret_cast<uintptr_t>(r) & 15) / sizeof(T))) {}
  __device__ __forceinline__ int first(int q) const { return q * N - shift; }
  __device__ __forceinline__ bool whole(int q) const { return first(q) >= 0 && first(q) + N <= len; }
  __device__ __forceinline__ V load(int q) const {  // outside the row: -inf
    const int j = first(q);
    if (whole(q)) return *reinterpret_cast<const V*>(row + j);
    V x;
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = j + e >= 0 && j + e < len ? row[j + e] : (T)(-INFINITY);
    return x;
  }
};

// Row r of [R / Tn][Tn] rows at element strides sb, st
template <typename T>
__device__ __forceinline__ const T* lp_row(const T* logits, int64_t sb, int64_t st, int Tn, int r) {
  return logits + (int64_t)(r / Tn) * sb + (int64_t)(r % Tn) * st;
}

// Order of the alternatives as one unsigned number: by value (NaN above everything, as torch sorts;
// -0 as 0), then the lowest index.  0 is below every value's key.
__device__ __forceinline__ unsigned long long lp_key(float x, int j) {
  unsigned u = __builtin_bit_cast(unsigned, x + 0.f);
  u = (u >> 31) ? ~u : u | 0x80000000u;
  if (x != x) u = 0xffffffffu;
  return ((unsigned long long)u << 32) | (0xffffffffu - (unsigned)j);
}
__device__ __forceinline__ int lp_index(unsigned long long key) { return (int)(0xffffffffu - (unsigned)key); }
// the value of a key (any NaN for a NaN's)
__device__ __forceinline__ float lp_value(unsigned long long key) {
  const unsigned u = (unsigned)(key >> 32);
  return __builtin_bit_cast(float, u == 0xffffffffu ? 0x7fc00000u : (u >> 31) ? u & 0x7fffffffu : ~u);
}

__device__ __forceinline__ unsigned long long lp_wave_max(unsigned long long v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    const unsigned long long w = __shfl_xor(v, o, 64);
    v = w > v ? w : v;
  }
  return v;
}

struct LpOut {
  float* logprob;    // [R]
  float* entropy;    // [R]
  LpStats* stats;    // [R] or null
  float* top_lp;     // [R][top]
  int64_t* top_idx;  // [R][top]
  // partials of rows of several segments
  float* pm;                 // [R][segs] maximum
  float* ps;                 // [R][segs] sum
  float* pt;                 // [R][segs] entropy sum, log2 units
  unsigned long long* pkey;  // [R][segs][top], descending
};

constexpr int64_t kLpIgnore = -100;  // the loss's ignore index

// The row's results from its maximum m, s = sum exp2(a_j) and t = sum exp2(a_j) a_j; returns log2 s
__device__ __forceinline__ float lp_finish(const LpOut& out, int r, float m, float s, float t, float inv_temp, int64_t tok,
                                           int V, float xtok) {
  constexpr float kLn2 = 0.69314718055994531f;
  const float l2 = log2f(s), ent = kLn2 * (l2 - t / s);
  float lp = 0.f;
  if (tok != kLpIgnore)
    lp = tok < 0 || tok >= V ? __builtin_nanf("") : (xtok - m) * inv_temp - kLn2 * l2;
  out.logprob[r] = lp;
  out.entropy[r] = ent;
  if (out.stats) out.stats[r] = LpStats{m, l2, ent};
  return l2;
}

// The parts (m, s, t) of a row that K adjacent lanes hold, joined in each of them: with M the largest m_i and
// d_i = (m_i - M) c, s = sum s_i exp2(d_i), t = sum exp2(d_i) (t_i + s_i d_i).  A part of -inf alone has
// m = -inf and adds its sums as they are: 0, or NaN where there was one.
template <int K>
__device__ __forceinline__ void lp_join(float& m, float& s, float& t, float c2) {
  const float M = lanes_max<K>(m);
  const bool has = m != -INFINITY;
  const float d = (m - M) * c2, f = __builtin_amdgcn_exp2f(d);
  t = lanes_sum<K>(has ? f * fmaf(s, fmaxf(d, kLpNone), t) : t);
  s = lanes_sum<K>(has ? s * f : s);
  m = M;
}

// Grid R x segs; NT threads.  top <= kLpMaxTop.  Each wave takes its own maximum for the reference of its
// sums, so that nothing waits for the row's; one wave joins the waves.
// Alternatives: the lanes form 64 groups, and the top-th largest of the groups' maxima is a bound that
// at least `top` values reach and, over values in no order, few more than that (20 alternatives: 24).  Those
// are collected and each counts the ones before it.  Rows with more than kLpCand values at or above the
// bound (masks of one finite value, few allowed tokens, ordered logits) are tried again with the equal ones
// limited to low indices, which is enough wherever such values are dense, and else taken one a round.
// 4000 rows of 32000 bf16 values (256 MB): 49 us without alternatives, 5.2 TB/s; 73 with 8, 91 with 50, where
// the workgroup's four barriers and the lists in LDS bound it (the bf16 instances also spill 16 registers, 36 bytes a
// lane, under the cap of 64 that two workgroups of 1024 on a CU set).  8 rows with 20 alternatives: 8.2 us.  TOP = false
// leaves the lists out (368 -> 317 us forward and backward of 8192 rows, when they still cost the second workgroup
// on a CU).
template <typename T, int NT, bool TOP>
__global__ __launch_bounds__(NT) __attribute__((amdgpu_waves_per_eu(8))) void lucid_token_logprobs_kernel(
    const T* __restrict__ logits, int64_t sb, int64_t st, int Tn, const int64_t* __restrict__ tokens, int V,
    float inv_temp, int top, int segs, LpOut out) {
  constexpr int NW = NT / 64;
  constexpr int GL = NT / 64;  // lanes of one of 64 groups
  __shared__ float red[3][NW], gmax[TOP ? 64 : 1];
  __shared__ unsigned long long kred[TOP ? NW : 1], best[TOP ? kLpMaxTop : 1], cand[TOP ? kLpCand : 1];
  __shared__ float bound_, stat[2];
  __shared__ int found[2];
  const int r = blockIdx.x / segs, seg = blockIdx.x - r * segs;
  const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63;
  const LpRow<T> row(lp_row(logits, sb, st, Tn, r), V);
  constexpr int N = LpRow<T>::N, C = LpRow<T>::C;
  const int q0 = seg * NT * C + tid;
  typename LpRow<T>::V x[C];
#pragma unroll
  for (int c = 0; c < C; ++c) x[c] = row.load(q0 + c * NT);

  constexpr int JW = TOP ? 1 : 0;  // the joining wave (the first one finds the alternatives' bound)
  int64_t tok = kLpIgnore;
  float xtok = 0.f;
  if (segs == 1 && w == JW) {  // wanted at the end
    tok = tokens[r];
    if (tok >= 0 && tok < V) xtok = (float)row.row[tok];
  }
  float m = -INFINITY;
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int e = 0; e < N; ++e) m = fmaxf(m, (float)x[c][e]);
  m = lanes_max<GL>(m);
  if (TOP && tid % GL == 0) gmax[tid / GL] = m;
  m = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, lanes_max<64>(m))));
  const float c2 = LOG2E_F * inv_temp, mref = m == -INFINITY ? 0.f : m, mc = mref * c2;
  float s = 0.f, t = 0.f;  // p = 0 where a = -inf
  const bool one_step = fabsf(mc) < kLpOneStep;
  if (one_step) {  // a = x c - m c
#pragma unroll
    for (int c = 0; c < C; ++c) {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float a = fmaf((float)x[c][e], c2, -mc), p = __builtin_amdgcn_exp2f(a);
        s += p;
        t = fmaf(p, fmaxf(a, kLpNone), t);
      }
    }
  } else {  // the difference first: a finite mask's value, or inf
#pragma unroll
    for (int c = 0; c < C; ++c) {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float a = ((float)x[c][e] - mref) * c2, p = __builtin_amdgcn_exp2f(a);
        s += p;
        t = fmaf(p, fmaxf(a, kLpNone), t);
      }
    }
  }
  s = lanes_sum<64>(s);
  t = lanes_sum<64>(t);
  if (lane == 0) {
    // m c was rounded: every a is larger by the difference (exact in one fma), which leaves here
    const float off = one_step ? fmaf(mref, c2, -mc) : 0.f, f = __builtin_amdgcn_exp2f(-off);
    red[0][w] = m;
    red[1][w] = s * f;
    red[2][w] = fmaf(-off, s, t) * f;
  }
  if (TOP && tid < 2) found[tid] = 0;
  __syncthreads();
  if (TOP && w == 0) {  // the top-th largest group maximum: its order key (lp_key's upper half) bit by bit
    const unsigned mine = (unsigned)(lp_key(gmax[lane], 0) >> 32);
    unsigned bits = 0;
#pragma unroll
    for (int i = 31; i >= (sizeof(T) == 2 ? 16 : 0); --i)
      bits = __popcll(__ballot(mine >= (bits | 1u << i))) >= top ? bits | 1u << i : bits;
    if (sizeof(T) == 2 && !(bits >> 31)) bits |= 0xffff;  // (a negative bf16's key ends in ones)
    if (lane == 0) bound_ = lp_value((unsigned long long)bits << 32);
  }
  if (w == JW) {
    const bool on = lane < NW;
    m = on ? red[0][lane % NW] : -INFINITY;
    s = on ? red[1][lane % NW] : 0.f;
    t = on ? red[2][lane % NW] : 0.f;
    lp_join<NW>(m, s, t, c2);
    if (lane == 0) {
      if (segs == 1) {
        stat[0] = m;
        stat[1] = lp_finish(out, r, m, s, t, inv_temp, tok, V, xtok);
      } else {
        const int64_t at = (int64_t)r * segs + seg;
        out.pm[at] = m;
        out.ps[at] = s;
        out.pt[at] = t;
      }
    }
  }
  if constexpr (TOP) {
    __syncthreads();
    const float bound = bound_;
    const int lo = max(row.first(seg * NT * C), 0);  // the segment's first index
    // Offers what passes: everything from the bound up (and NaN), or, the second time, the values above it and
    // those equal to it among the segment's first kLpCand / 2.
    auto offer = [&](int pass, typename LpRow<T>::V xv, int j) {
      bool any = false;
#pragma unroll
      for (int e = 0; e < N; ++e) any |= !((float)xv[e] < bound);
      if (any) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float v = (float)xv[e];
          if (v < bound || j + e < 0 || j + e >= V) continue;
          if (pass == 1 && v == bound && j + e - lo >= kLpCand / 2) continue;
          const int at = atomicAdd(&found[pass], 1);
          if (at < kLpCand) cand[at] = lp_key(v, j + e);
        }
      }
    };
    int qa = q0;
    asm volatile("" : "+v"(qa));  // the indices are worked out here, not kept from the loads
#pragma unroll
    for (int c = 0; c < C; ++c) offer(0, x[c], row.first(qa + c * NT));
    __syncthreads();
    int n = found[0];
    if (n > kLpCand) {
      // (from here on the row is read again: its registers would cost the rows that never get here)
#pragma unroll 1
      for (int c = 0; c < C; ++c) offer(1, row.load(qa + c * NT), row.first(qa + c * NT));
      __syncthreads();
      n = found[1];
    }
    if (n <= kLpCand && (n >= top || found[0] <= kLpCand)) {
      if (tid < top && tid >= n) best[tid] = 0;  // a short last segment
      // a wave counts what is above a value; the first 128 stay in its registers
      const unsigned long long c0 = lane < n ? cand[lane] : 0, c1 = lane + 64 < n ? cand[lane + 64] : 0;
#pragma unroll 4
      for (int i = w; i < n; i += NW) {
        const unsigned long long key = cand[i];
        int above = __popcll(__ballot(c0 > key)) + __popcll(__ballot(c1 > key));
        for (int k = lane + 128; k - lane < n; k += 64) above += __popcll(__ballot(k < n && cand[k] > key));
        if (lane == 0 && above < top) best[above] = key;
      }
    } else {
      // one a round: each lane offers its largest key below the last one taken
      unsigned long long mine = 0, last = ~0ull;
      bool scan = true;
#pragma unroll 1
      for (int k = 0; k < top; ++k) {
        if (scan) {
          mine = 0;
#pragma unroll 1
          for (int c = 0; c < C; ++c) {
            const int j = row.first(qa + c * NT);
            const typename LpRow<T>::V xv = row.load(qa + c * NT);
#pragma unroll
            for (int e = 0; e < N; ++e) {
              const unsigned long long key = lp_key((float)xv[e], j + e);
              if (j + e >= 0 && j + e < V && key < last && key > mine) mine = key;
            }
          }
        }
        unsigned long long b = lp_wave_max(mine);
        if (lane == 0) kred[w] = b;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NW; ++i) b = kred[i] > b ? kred[i] : b;
        if (tid == 0) best[k] = b;
        scan = mine == b;
        last = b;
        __syncthreads();
      }
    }
  }
  if constexpr (TOP) {
    __syncthreads();
    if (tid < top) {
      const unsigned long long key = best[tid];
      if (segs == 1) {
        out.top_idx[(int64_t)r * top + tid] = lp_index(key);
        out.top_lp[(int64_t)r * top + tid] = (lp_value(key) - stat[0]) * inv_temp - 0.69314718055994531f * stat[1];
      } else {
        out.pkey[((int64_t)r * segs + seg) * top + tid] = key;
      }
    }
  }
}

// Rows of several segments, one workgroup each.  A key's place among the row's alternatives is
// the number above it: its place in its own segment's list and those that it would have in the others' (by
// bisection: 4.4 us for 64 rows of four segments with 50 alternatives, 5.5 with all keys compared).
template <typename T>
__global__ __launch_bounds__(256) void lucid_token_logprobs_merge_kernel(const T* __restrict__ logits, int64_t sb,
                                                                         int64_t st, int Tn,
                                                                         const int64_t* __restrict__ tokens, int V,
                                                                         float inv_temp, int top, int segs, LpOut out) {
  __shared__ unsigned long long keys[kLpMaxSegs * kLpMaxTop];
  __shared__ float stat[2];
  const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  const float c2 = LOG2E_F * inv_temp;
  const int64_t at = (int64_t)r * segs;
  const int n = segs * top;
  for (int i = tid; i < n; i += 256) keys[i] = out.pkey[at * top + i];
  if (tid < 64) {
    const bool on = lane < segs;
    float m = on ? out.pm[at + lane] : -INFINITY, s = on ? out.ps[at + lane] : 0.f, t = on ? out.pt[at + lane] : 0.f;
    const int64_t tok = tokens[r];
    const float xtok = tok >= 0 && tok < V ? (float)lp_row(logits, sb, st, Tn, r)[tok] : 0.f;
    lp_join<64>(m, s, t, c2);
    if (lane == 0) {
      stat[0] = m;
      stat[1] = lp_finish(out, r, m, s, t, inv_temp, tok, V, xtok);
    }
  }
  __syncthreads();
  for (int i = tid; i < n; i += 256) {
    const unsigned long long key = keys[i];
    if (!key) continue;
    // every segment's keys are in descending order
    const int own = i / top;
    int above = i - own * top;
    for (int g = 0; g < segs; ++g) {
      if (g == own) continue;
      int lo = 0, hi = top;
      while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (keys[g * top + mid] > key)
          lo = mid + 1;
        else
          hi = mid;
      }
      above += lo;
    }
    if (above >= top) continue;
    out.top_idx[(int64_t)r * top + above] = lp_index(key);
    out.top_lp[(int64_t)r * top + above] = (lp_value(key) - stat[0]) * inv_temp - 0.69314718055994531f * stat[1];
  }
}

struct LpGrads {
  const float* lp;   // [R] or null: gradients of the log probability,
  const float* ent;  // [R] or null: of the entropy,
  const float* top;  // [R][top] or null: of the alternatives' log probabilities
};

// Grid R x blocks (column blocks of a row).  Every value gets the softmax part; then the values that a token or an
// alternative names are written once more with their whole gradient (rounded once).  Memory bounds it: 8192 rows of
// 32000 bf16 values in 165 to 180 us (1.05 GB, 5.8 to 6.3 TB/s), 1021 of 32003 fp32 values in 44.  PAST: the gradient passes the caches by (the launcher's rule).
template <typename T, bool PAST>
__global__ __launch_bounds__(256) void lucid_token_logprobs_bwd_kernel(const T* __restrict__ logits, int64_t sb,
                                                                       int64_t st, int Tn,
                                                                       const int64_t* __restrict__ tokens, int V,
                                                                       float inv_temp, int top,
                                                                       const LpStats* __restrict__ stats,
                                                                       const int64_t* __restrict__ top_idx, LpGrads g,
                                                                       T* __restrict__ dlogits, int blocks) {
  constexpr int NT = 256, N = LpRow<T>::N, C = LpRow<T>::C;
  __shared__ int name[kLpMaxTop + 1];
  __shared__ float gain[kLpMaxTop + 1];
  const int r = blockIdx.x / blocks, col = blockIdx.x - r * blocks, tid = threadIdx.x;
  const LpRow<T> row(lp_row(logits, sb, st, Tn, r), V);
  T* drow = dlogits + (int64_t)r * V;
  const LpStats z = stats[r];
  const float c2 = LOG2E_F * inv_temp;
  const int64_t tok = tokens[r];
  float glp = g.lp && tok != kLpIgnore ? g.lp[r] : 0.f;
  if (g.lp && tok != kLpIgnore && (tok < 0 || tok >= V)) glp = __builtin_nanf("");
  if (tid == 0) {
    name[0] = tok >= 0 && tok < V ? (int)tok : -1;
    gain[0] = glp;
  }
  if (tid < top) {
    name[tid + 1] = (int)top_idx[(int64_t)r * top + tid];
    gain[tid + 1] = g.top ? g.top[(int64_t)r * top + tid] : 0.f;
  }
  __syncthreads();
  float all = glp;
  const float gh = g.ent ? g.ent[r] : 0.f;
  bool wanted = glp != 0.f || gh != 0.f;  // no gradient comes in: none goes out, whatever the row holds
  for (int k = 1; k <= top; ++k) {
    all += gain[k];
    wanted |= gain[k] != 0.f;
  }
  // dx of the softmax part: -p (all + gh (ln p + H)), ln p = ln2 a
  const float ka = all + gh * z.ent, kb = gh * 0.69314718055994531f;
  auto soft = [&](float x) {
    const float a = fmaf(x - z.m, c2, -z.l2);
    const float p = __builtin_amdgcn_exp2f(a);
    return wanted ? -p * fmaf(kb, fmaxf(a, kLpNone), ka) : 0.f;
  };
  const bool same = (reinterpret_cast<uintptr_t>(drow) & 15) / sizeof(T) == (unsigned)row.shift;
  const int q0 = col * NT * C + tid;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int q = q0 + c * NT, j = row.first(q);
    if (j >= V) break;
    const typename LpRow<T>::V x = row.load(q);
    typename LpRow<T>::V o;
#pragma unroll
    for (int e = 0; e < N; ++e) o[e] = (T)(soft((float)x[e]) * inv_temp);
    if (same && row.whole(q)) {
      auto* at = reinterpret_cast<typename LpRow<T>::V*>(drow + j);
      if constexpr (PAST)
        __builtin_nontemporal_store(o, at);
      else
        *at = o;
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (j + e >= 0 && j + e < V) drow[j + e] = o[e];
    }
  }
  __syncthreads();
  if (tid <= top) {
    const int j = name[tid];
    const int lo = row.first(col * NT * C), hi = lo + NT * kLpLane;
    if (j >= 0 && j >= lo && j < hi) {
      bool firstly = true;
      float add = 0.f;
      for (int k = 0; k <= top; ++k) {
        if (name[k] != j) continue;
        if (k < tid) firstly = false;
        add += gain[k];
      }
      if (firstly) drow[j] = (T)((add + soft((float)row.row[j])) * inv_temp);
    }
  }
}

}  // namespace lucid
