// Rotary positions on CDNA4 (gfx950): queries and keys turned by their positions (modeling_lucid.py:78-145 is the
// reference's: tables of cos and sin in the activations' type, the whole head in halves).  With f_i the i-th frequency and p a
// token's position, the pair (a_i, b_i) of every head becomes
//   (a_i cos(p f_i) - b_i sin(p f_i), b_i cos(p f_i) + a_i sin(p f_i)) scale,  i < part / 2
// pairs (i, i + part / 2) in the half layout, (2 i, 2 i + 1) in the interleaved one; columns from part on stay as they
// are.  The gradient is the turn by -p f_i.  One pass over q and k: a workgroup works the angles of its tokens out
// once, for all heads, in 64 bits: at position 131072 a product in 32 bits is off by up to 2^-8 of a radian.  HBM bounds long
// calls: 131072 tokens of 40 heads of 128 bf16 columns (2.7 GB read and written) 503 us, 5.3 TB/s; 8 x 2048 of 36 heads of 68
// fp32 columns (321 MB) 70 us, 4.6 TB/s; 32 tokens are 4 us of latency (position, angle, rows).
#include "lucid_common.h"

namespace lucid {

constexpr int kRotaryPairs = 128;  // of a head, at most
constexpr int kRotaryTokens = 2;   // of a workgroup, at most

struct RotaryTensor {
  const void* x;
  Strides xs;
  void* y;
  Strides ys;
  int heads;
};
struct RotaryCall {
  RotaryTensor q, k;
  const void* pos;  // int32 or int64 at element strides pb, pt
  int64_t pb, pt;
  int pos64;
  const void* freq;  // fp64 or fp32 [part / 2]
  int freq64;
  int B, T, d, part;
  int tokens;      // of a workgroup
  float scale, dir;  // dir -1: the gradient
  int turning, units;        // units of a head: those of pairs, and with those of columns that stay
  int stay;                  // columns of a unit that stay: V or 2 V
  float per_unit, per_head;  // 1 / units, 1 / (units (Hq + Hkv))
};

template <bool PAST, typename V>
__device__ __forceinline__ void rotary_put(void* to, const V& x) {
  if constexpr (PAST)
    __builtin_nontemporal_store(x, static_cast<V*>(to));
  else
    *static_cast<V*>(to) = x;
}

// i / n by the reciprocal r of n: exact for i < 2^22
__device__ __forceinline__ int div_by(int i, float r) { return (int)(((float)i + 0.5f) * r); }

// V pairs a unit: V columns of either half, or 2 V adjacent ones.  A run that is no whole number of units
// ends in one that overlaps the one before (the same values twice), so that any head dim goes in 16-byte accesses, which
// need no alignment.  256 threads.
// PAST: results pass the caches by (the launcher's rule).
template <typename T, int V, bool INTER, bool PAST>
__global__ __launch_bounds__(256) void lucid_rotary_kernel(const RotaryCall c) {
  typedef T TV __attribute__((ext_vector_type(V), aligned(sizeof(T))));
  typedef T T2 __attribute__((ext_vector_type(2 * V), aligned(sizeof(T))));
  __shared__ __attribute__((aligned(16))) float2 turn[kRotaryTokens][kRotaryPairs];
  const int half = c.part / 2;
  const int64_t all = (int64_t)c.B * c.T, t0 = (int64_t)blockIdx.x * c.tokens;
  const int n = (int)min((int64_t)c.tokens, all - t0);
  for (int i = threadIdx.x; i < n * half; i += 256) {
    const int tk = i / half, p = i - tk * half;
    const int64_t tok = t0 + tk, b = tok / c.T, at = b * c.pb + (tok - b * c.T) * c.pt;
    const double pos = c.pos64 ? (double)static_cast<const int64_t*>(c.pos)[at] : (double)static_cast<const int32_t*>(c.pos)[at];
    const double f = c.freq64 ? static_cast<const double*>(c.freq)[p] : (double)static_cast<const float*>(c.freq)[p];
    // in half turns, less whole turns; a quarter of a turn at most is left to 32 bits
    const double u = pos * f * 0.31830988618379067154, whole = 2.0 * rint(0.5 * u);
    double r = u - whole;  // -1 .. 1
    const double q = rint(2.0 * r);
    const float x = (float)(r - 0.5 * q);  // -1/4 .. 1/4
    float s, co;
    sincospif(x, &s, &co);
    const int quad = (int)q & 3;
    const float sn = quad == 0 ? s : quad == 1 ? co : quad == 2 ? -s : -co;
    const float cs = quad == 0 ? co : quad == 1 ? -s : quad == 2 ? -co : s;
    turn[tk][p] = make_float2(cs * c.scale, sn * c.scale * c.dir);
  }
  __syncthreads();
  const int heads = c.q.heads + c.k.heads, work = n * heads * c.units;
#pragma unroll 2
  for (int i = threadIdx.x; i < work; i += 256) {
    const int tk = div_by(i, c.per_head), rest = i - tk * heads * c.units;
    int h = div_by(rest, c.per_unit);
    const int u = rest - h * c.units;
    const bool isk = h >= c.q.heads;
    if (isk) h -= c.q.heads;
    const int64_t tok = t0 + tk, bt = tok / c.T, t = tok - bt * c.T;
    const Strides xs = isk ? c.k.xs : c.q.xs, ys = isk ? c.k.ys : c.q.ys;
    const T* x = static_cast<const T*>(isk ? c.k.x : c.q.x) + bt * xs.b + h * xs.h + t * xs.t;
    T* y = static_cast<T*>(isk ? c.k.y : c.q.y) + bt * ys.b + h * ys.h + t * ys.t;
    if (u >= c.turning) {
      const int col = min(c.part + (u - c.turning) * c.stay, c.d - c.stay);
      if (INTER && c.stay == 2 * V)
        rotary_put<PAST>(y + col, *reinterpret_cast<const T2*>(x + col));
      else
        rotary_put<PAST>(y + col, *reinterpret_cast<const TV*>(x + col));
      continue;
    }
    const int p0 = min(u * V, half - V);  // first pair
    const float2* tn = &turn[tk][p0];
    if constexpr (INTER) {
      const T2 z = *reinterpret_cast<const T2*>(x + 2 * p0);
      T2 o;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float a = (float)z[2 * e], b = (float)z[2 * e + 1];
        o[2 * e] = (T)fmaf(a, tn[e].x, -(b * tn[e].y));
        o[2 * e + 1] = (T)fmaf(b, tn[e].x, a * tn[e].y);
      }
      rotary_put<PAST>(y + 2 * p0, o);
    } else {
      const TV a = *reinterpret_cast<const TV*>(x + p0), b = *reinterpret_cast<const TV*>(x + half + p0);
      TV o, p;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        o[e] = (T)fmaf((float)a[e], tn[e].x, -((float)b[e] * tn[e].y));
        p[e] = (T)fmaf((float)b[e], tn[e].x, (float)a[e] * tn[e].y);
      }
      rotary_put<PAST>(y + p0, o);
      rotary_put<PAST>(y + half + p0, p);
    }
  }
}

}  // namespace lucid
