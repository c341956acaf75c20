// Host helpers of the library's C ABI, shared by its translation units (lucid_capi.hip, which holds the error
// text, and prompt_capi.hip).
#pragma once
#include <string>

#include "../../include/lucid_amd.h"
#include "lucid_common.h"
#include "profiling.h"

extern thread_local std::string g_last_error;

namespace {

inline int fail(const std::string& msg) {
  g_last_error = msg;
  return LUCID_EINVAL;
}

inline int hip_status(const char* where) {
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) {
    g_last_error = std::string(where) + ": " + hipGetErrorString(e);
    return LUCID_EHIP + (int)e;
  }
  return LUCID_OK;
}

inline size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

// Workspaces hold operands whose blocks of rows must fill whole cache lines.
inline int check_ws(const char* name, const void* p) {
  if (reinterpret_cast<uintptr_t>(p) % 256) return fail(std::string(name) + " must be 256-byte aligned");
  return LUCID_OK;
}

inline bool misaligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 != 0; }

inline lucid::Strides S(const int64_t* s) { return lucid::Strides{s[0], s[1], s[2]}; }

}  // namespace

#define LUCID_LAUNCH(NAME, KERNEL, GRID, ST, ...) LUCID_TIMED_LAUNCH(hip_status, NAME, KERNEL, GRID, ST, __VA_ARGS__)
#define LUCID_LAUNCH_B(NAME, KERNEL, GRID, BLOCK, ST, ...) \
  LUCID_TIMED_LAUNCH_B(hip_status, NAME, KERNEL, GRID, BLOCK, ST, __VA_ARGS__)
