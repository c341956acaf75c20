// Rows of logits as the kernels on them read them.
#pragma once
#include "lucid_common.h"

namespace lucid {

constexpr int kLpLane = 32;  // logits a lane holds, in chunks of 16 bytes

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

}  // namespace lucid
