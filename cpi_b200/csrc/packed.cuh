// Calls with their arguments in one block of memory, eight bytes each: addresses and integers as 64-bit integers, floats as
// doubles.  A foreign-function layer that converts arguments one by one takes longer for thirty of them (0.1 us each from Python)
// than the launch itself; one block takes it less than 1 us.
#pragma once
#include <cstdint>
#include <cstring>
#include <type_traits>
#include <utility>

namespace cpi {

template <typename T> inline T unpacked(const uint64_t* a, size_t i) {
  if constexpr (std::is_floating_point_v<T>) {
    double d;
    std::memcpy(&d, a + i, 8);
    return static_cast<T>(d);
  } else if constexpr (std::is_pointer_v<T>) {
    return reinterpret_cast<T>(static_cast<uintptr_t>(a[i]));
  } else {
    return static_cast<T>(static_cast<int64_t>(a[i]));
  }
}
template <typename... A, size_t... I>
inline int call_unpacked(int (*f)(A...), const uint64_t* a, std::index_sequence<I...>) { return f(unpacked<A>(a, I)...); }
template <typename... A> inline int call_packed(int (*f)(A...), const uint64_t* a) {
  return call_unpacked(f, a, std::index_sequence_for<A...>{});
}

}  // namespace cpi

// name_packed(a): name with its arguments taken from a[0], a[1], ...
#define CPI_PACKED(name) \
  extern "C" int name##_packed(const uint64_t* a) { return cpi::call_packed(&name, a); }
