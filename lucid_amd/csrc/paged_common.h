// What the kernels on paged (K, V') caches share: sequences and their tables, pools, rows read from callers' tensors
// and tiles of rows in LDS.
#pragma once
#include "lucid_common.h"

namespace lucid {

struct PagedBatch {
  const int32_t* table;  // [B][M] page ids, rows tstride apart
  int64_t tstride;
  const int32_t* lens;  // [B] rows cached before the call
  int B, M, P, page;
  int shift;  // log2 of page, -1 where it is no power of two
  int L;      // new tokens of the call
  int done;   // of earlier passes
};
__device__ __forceinline__ int page_of(const PagedBatch& s, int j) { return s.shift >= 0 ? j >> s.shift : j / s.page; }

// A pool by its strides in units of 16 bytes (8 elements); the host checks that every row's offset
// fits 32 bits, a pool of 64 GB.
struct PagedPool {
  bf16* base;
  unsigned page, head, row;
};
__device__ __forceinline__ bf16* paged_at(const PagedPool& p, unsigned off) { return p.base + (size_t)off * 8; }

// The scale s, and s log2 e and log2 e / s as the exponents take them
struct PagedScale {
  double s;
  float sl2, c0;
};

// Four consecutive columns c .. c+3 of a row of d, zeros beyond d; vec: the row starts at an 8-byte
// boundary
__device__ __forceinline__ bf16x4 ld4_cols(const bf16* row, int c, int d, bool vec) {
  if (vec && c + 4 <= d) return *reinterpret_cast<const bf16x4*>(row + c);
  bf16x4 x;
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = c + e < d ? row[c + e] : (bf16)0.f;
  return x;
}

// A tile of rows in LDS as the direct loads write it: W / 8 chunks of 16 bytes a row, chunk c of
// row r at c ^ (r & 7) for rows of 128 and 256 bytes; rows of 160 and 192 bytes fall on different
// banks by themselves.
constexpr bool paged_swizzled(int W) { return W == 64 || W == 128; }

// MFMA A operand of 16 rows from row0 and columns col0 + lane % 32 of a V' tile (lds_tr_a of
// lucid_common.h for the row widths of a page)
template <int W>
__device__ __forceinline__ bf16x8 paged_tr_a(const bf16* tile, int row0, int col0) {
  typedef __attribute__((address_space(3))) bf16x4 lds_bf16x4;
  if constexpr (paged_swizzled(W)) {
    return lds_tr_a<W / 8>(tile, row0, col0);
  } else {
    const int lane = threadIdx.x & 63, s = lane & 15;
    const int col = col0 + 16 * ((lane >> 4) & 1) + 4 * (s & 3);
    const int r1 = row0 + 4 * (lane >> 5) + (s >> 2);
    const bf16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)(tile + r1 * W + col));
    const bf16x4 v2 = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)(tile + (r1 + 8) * W + col));
    return bf16x8{v1[0], v1[1], v1[2], v1[3], v2[0], v2[1], v2[2], v2[3]};
  }
}

}  // namespace lucid
