// A launcher's arguments as one packed record: pointers, 32- and 64-bit integers and floats in the launcher's order, each at its natural
// alignment, which is what Python's `struct` makes of them.  Handing over one pointer costs the caller a fifth of what ctypes takes to
// convert 28 arguments (1.0 us against 4.8).
#pragma once
#include <stdint.h>
#include <string.h>
#include <tuple>

namespace ilb {

template <typename T>
inline T take_packed(const char*& at, const char* base) {
  at = base + ((at - base) + alignof(T) - 1) / alignof(T) * alignof(T);
  T v;
  memcpy(&v, at, sizeof(T));
  at += sizeof(T);
  return v;
}

template <typename... A>
inline int call_packed(int (*f)(A...), const char* record) {
  const char* at = record;
  std::tuple<A...> args{take_packed<A>(at, record)...};      // (in a braced list: from left to right)
  return std::apply(f, args);
}

}  // namespace ilb

#define ILB_PACKED(launcher) \
  ILB_EXPORT int launcher##_packed(const char* record) { return ilb::call_packed(launcher, record); }
