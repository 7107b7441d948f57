// What the C entries of libajq_serve.so and libajq_draft.so share: error reporting, argument checks, choice of a kernel's types.
#pragma once
#include <algorithm>
#include <math.h>
#include <stdarg.h>
#include <stdio.h>
#include <stdlib.h>

#include "../../include/ajq_serve.h"
#include "host_math.h"
#include "lane_rows.h"

using namespace ajq;

namespace {

thread_local char g_error[512] = "";

int fail(int status, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_error, sizeof(g_error), fmt, ap);
  va_end(ap);
  return status;
}
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }
bool known(int dtype) { return dtype == AJQS_BF16 || dtype == AJQS_F32; }
int check_launch(const char* what) {
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(AJQ_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
  return AJQ_OK;
}
const long long* int64s(const int64_t* p) { return reinterpret_cast<const long long*>(p); }

// Calls fn(T{}) for the element type of a dtype flag.
template <typename F>
void with_type(int dtype, F&& fn) {
  if (dtype == AJQS_BF16) fn(uint16_t{});
  else fn(float{});
}
template <int N> struct Size {
  static constexpr int value = N;
};
template <typename F>
void with_dim(int dim, F&& fn) {
  if (dim == 128) fn(Size<128>{});
  else if (dim == 64) fn(Size<64>{});
  else fn(Size<32>{});
}
bool built_dim(int dim) { return dim == 128 || dim == 64 || dim == 32; }

int check_caches(const char* what, const void* keys, const void* values, long long outer, long long head) {
  if (!aligned16(keys) || !aligned16(values) || outer % 8 != 0 || head % 8 != 0)
    return fail(AJQ_ERR_ALIGN, "%s: caches must be 16-byte aligned, their strides multiples of 8 elements", what);
  if (outer < 0 || head < 0) return fail(AJQ_ERR_SHAPE, "%s: negative cache stride", what);
  return AJQ_OK;
}

// Whether one of the blocks of `size` numbers at i * outer + j * inner (i < n, j < m) meets one of the same blocks moved by d numbers (d 0: another one).
bool blocks_meet(long long d, long long outer, long long n, long long inner, long long m, long long size) {
  const bool nested = (m == 1 || inner >= size) && (n == 1 || outer >= (m - 1) * inner + size);
  const bool crossed = (n == 1 || outer >= size) && (m == 1 || inner >= (n - 1) * outer + size);
  if ((nested || crossed) && (d == 0 || std::abs(d) >= (n - 1) * outer + (m - 1) * inner + size)) return false;
  for (long long j = 1 - m; j < m; ++j) {
    const long long x = d + j * inner, near = outer ? -x / outer : 0;
    for (long long i = near - 1; i <= near + 1; ++i) {
      const long long k = std::max(1 - n, std::min(i, n - 1));
      if (std::abs(x + k * outer) < size && (d != 0 || j != 0 || k != 0)) return true;
    }
  }
  return false;
}
// The same of one row-major matrix and another.
bool rows_meet(const void* a, long long a_pitch, long long a_bytes, const void* b, long long b_pitch, long long b_bytes, long long rows) {
  const long long d = (long long)(reinterpret_cast<uintptr_t>(b) - reinterpret_cast<uintptr_t>(a));   // (bytes)
  if (d >= (rows - 1) * a_pitch + a_bytes || -d >= (rows - 1) * b_pitch + b_bytes) return false;
  if (rows == 1 || a_pitch != b_pitch) return true;   // (pitches that differ: taken to meet)
  const long long r = (d % a_pitch + a_pitch) % a_pitch;
  return r < a_bytes || a_pitch - r < b_bytes;
}

constexpr int kLdsLimit = 160 * 1024;
template <typename K>
int allow_lds(K kernel, int bytes, const char* what) {
  if (bytes > kLdsLimit) return fail(AJQ_ERR_UNSUPPORTED, "%s: %d bytes of LDS needed", what, bytes);
  if (bytes > 64 * 1024) {
    hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != hipSuccess) return fail(AJQ_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
  }
  return AJQ_OK;
}

constexpr long long kMostLanes = 0xFFFFFFFFLL;   // of a grid in a dimension: HIP launches no more

}  // namespace
