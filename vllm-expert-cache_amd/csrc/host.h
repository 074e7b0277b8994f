// Argument checks that the entry points of both translation units share.
#pragma once
#include <stdint.h>

namespace ec {
namespace {

// [p, p + pn) and [q, q + qn) share a byte
inline bool ranges_meet(const void* p, long long pn, const void* q, long long qn) {
  const long long a = (long long)reinterpret_cast<uintptr_t>(p);
  const long long b = (long long)reinterpret_cast<uintptr_t>(q);
  return pn > 0 && qn > 0 && a < b + qn && b < a + pn;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace ec
