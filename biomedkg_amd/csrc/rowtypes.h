// The element types a table of rows may have (fp32 / bf16 / fp16) and the widest aligned access its layout allows.
#pragma once
#include "common.h"

namespace bkg {

constexpr int BKG_T_F32 = 0, BKG_T_BF16 = 1, BKG_T_F16 = 2;
static inline int type_bytes(int t) { return t == BKG_T_F32 ? 4 : 2; }

__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(__bf16 v) { return (float)v; }
__device__ __forceinline__ float widen(_Float16 v) { return (float)v; }

// N consecutive elements as one access (N * sizeof(T) = 2 .. 16 bytes, aligned to their size)
template <typename T, int N> struct alignas(sizeof(T) * N) Pack { T v[N]; };

// A 16-byte pack written as ONE store.  (As a plain struct copy hipcc splits it into element stores where another branch
// writes the same elements one by one: a request per lane instead of one per 64 bytes.)
typedef int rt_i32x4 __attribute__((ext_vector_type(4)));
template <typename T> __device__ __forceinline__ void store16(T* p, const Pack<T, 16 / sizeof(T)>& v) {
  *reinterpret_cast<rt_i32x4*>(p) = __builtin_bit_cast(rt_i32x4, v);
}

// The same past the caches (non-temporal): for results beyond STREAM_BYTES, the Infinity Cache's size, which no later call finds
// there anyway and which would push out what this one still reads.
constexpr int64_t STREAM_BYTES = 256 << 20;
template <typename T> __device__ __forceinline__ void stream16(T* p, const Pack<T, 16 / sizeof(T)>& v) {
  __builtin_nontemporal_store(__builtin_bit_cast(rt_i32x4, v), reinterpret_cast<rt_i32x4*>(p));
}

// the largest access in bytes (<= 16) that `bytes`, a row of it and its start are all multiples of
static inline int access_bytes(const void* p, int64_t row_bytes, int64_t ld_bytes) {
  const uint64_t all = (uint64_t)(uintptr_t)p | (uint64_t)row_bytes | (uint64_t)ld_bytes | 16u;
  return (int)(all & (~all + 1));
}

}  // namespace bkg
