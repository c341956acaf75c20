// Host helpers of the entry points on paged (K, V') caches.
#pragma once
#include "capi_common.h"
#include "paged_common.h"

namespace {

// Row width of a page for a head dim (0: unsupported)
inline int page_width(int D) { return D < 1 ? 0 : D <= 64 ? 64 : D <= 80 ? 80 : D <= 96 ? 96 : D <= 128 ? 128 : 0; }

// log2 of a page size that is a power of two, whose rows are found by a shift (-1: by a division, 20.7 against
// 20.2 us at 32 sequences of up to 3500 rows, nothing at one of 131072)
inline int page_shift(int page) { return page & (page - 1) ? -1 : __builtin_ctz((unsigned)page); }

inline int check_pool(const char* name, void* p, const int64_t* s, int pages, int Hkv, int page, int W, lucid::PagedPool* out) {
  if (!p || !s) return fail(std::string(name) + " or its strides are null");
  if (misaligned16(p)) return fail(std::string(name) + " must be 16-byte aligned");
  for (int i = 0; i < 3; ++i)
    if (s[i] < 0 || s[i] % 8) return fail(std::string(name) + " strides must be non-negative multiples of 8 elements");
  // offsets in units of 16 bytes have to fit 32 bits; each factor first, so that the sum cannot wrap
  const int64_t most = (int64_t)1 << 32;
  const int64_t n[3] = {pages, Hkv, page};
  int64_t end = W / 8;
  for (int i = 0; i < 3; ++i) {
    if (s[i] / 8 >= most || (n[i] > 1 && s[i] / 8 > most / (n[i] - 1)))
      return fail(std::string(name) + " spans more than 64 GB");
    end += (n[i] - 1) * (s[i] / 8);
  }
  if (end > most) return fail(std::string(name) + " spans more than 64 GB");
  *out = lucid::PagedPool{(bf16*)p, (unsigned)(s[0] / 8), (unsigned)(s[1] / 8), (unsigned)(s[2] / 8)};
  return LUCID_OK;
}

// Whether rows of these tensors start at boundaries of 4 elements
inline bool rows_of_4(const void* p, const int64_t* s, size_t size) {
  return reinterpret_cast<uintptr_t>(p) % (4 * size) == 0 && s[0] % 4 == 0 && s[1] % 4 == 0 && s[2] % 4 == 0;
}

}  // namespace
