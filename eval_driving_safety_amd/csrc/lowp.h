// shared by dropout.hip and mx4.hip: the three floating-point types their entry points take, and accesses to a few consecutive elements
#ifndef ADV_LOWP_H
#define ADV_LOWP_H
#include <hip/hip_runtime.h>

#include <cstdint>

#include "advengine.h"

namespace lowp {

// 16 bytes = V consecutive elements, at any address that suits the element: rows of odd length are ordinary here, and the hardware takes
// 16-byte accesses there.  As four dwords, so that the compiler keeps it one instruction.
// STREAM: non-temporal, for what is read or written once - without its lines in the L2 a 411 MB matrix is rounded to MXFP4 and back in 163 instead of
// 219 us; what several workgroups or the next launch read again goes through the caches.
typedef uint32_t Bits16 __attribute__((ext_vector_type(4), aligned(2)));
template <class T>
struct Elems {
  T v[16 / sizeof(T)];
};

template <class T, int V, bool STREAM = true>
__device__ __forceinline__ void load(const T* p, float (&out)[V]) {
  static_assert(V * sizeof(T) == 16, "one 16-byte access");
  const Bits16* at = reinterpret_cast<const Bits16*>(p);
  const Elems<T> q = __builtin_bit_cast(Elems<T>, STREAM ? __builtin_nontemporal_load(at) : *at);
#pragma unroll
  for (int i = 0; i < V; ++i) out[i] = static_cast<float>(q.v[i]);
}
// the first n of V, zeros behind
template <class T, int V>
__device__ __forceinline__ void load_some(const T* p, float (&out)[V], int n) {
#pragma unroll
  for (int i = 0; i < V; ++i) out[i] = i < n ? static_cast<float>(p[i]) : 0.0f;
}
// eight elements, the first n of them real
template <class T>
__device__ __forceinline__ void load_eight(const T* p, float (&out)[8], int n) {
  if (n < 8) {
    load_some<T, 8>(p, out, n);
  } else if constexpr (sizeof(T) == 2) {
    load<T, 8>(p, out);
  } else {
    float a[4], b[4];
    load<T, 4>(p, a);
    load<T, 4>(p + 4, b);
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = a[i], out[4 + i] = b[i];
  }
}
template <class T, int V>
__device__ __forceinline__ void store(T* p, const float (&in)[V]) {
  static_assert(V * sizeof(T) == 16, "one 16-byte access");
  Elems<T> q;
#pragma unroll
  for (int i = 0; i < V; ++i) q.v[i] = static_cast<T>(in[i]);      // to nearest, ties to even
  __builtin_nontemporal_store(__builtin_bit_cast(Bits16, q), reinterpret_cast<Bits16*>(p));
}
template <class T, int V>
__device__ __forceinline__ void store_some(T* p, const float (&in)[V], int n) {
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (i < n) p[i] = static_cast<T>(in[i]);
}

inline int size_of(int dtype) { return dtype == ADV_F32 ? 4 : 2; }
inline bool known(int dtype) { return dtype == ADV_F32 || dtype == ADV_BF16 || dtype == ADV_F16; }
inline bool aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & static_cast<uintptr_t>(bytes - 1)) == 0; }
// [a, a + an) and [b, b + bn) share a byte
inline bool overlap(const void* a, int64_t an, const void* b, int64_t bn) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return x < y + static_cast<uintptr_t>(bn) && y < x + static_cast<uintptr_t>(an);
}

}  // namespace lowp
#endif
