// select_rows.hpp — pieces of the kernels that move rows by a selection matrix
// (embedding.hip, expert_rows.hip): 16-byte slices of rows in any value type.
#pragma once

#include "fs_common.hpp"

namespace fs {

// Arithmetic type of a value type: 32 bits for 16- and 32-bit values.
template <class V>
struct Elem {
  using acc = float;
};
template <>
struct Elem<double> {
  using acc = double;
};
template <class V>
__device__ inline typename Elem<V>::acc widen(V v) {
  return (typename Elem<V>::acc)v;
}

// A lane's slice: 16 bytes of a row, at any element: the 16-byte load and store
// instructions take addresses that only elements are aligned to (compiled alike
// either way, so there is no variant for rows at multiples of 16 bytes).
template <class V>
struct Slice {
  static constexpr int n = 16 / (int)sizeof(V);
  V v[n];
};
template <class V>
__device__ inline Slice<V> load_slice(const V* p) {
  Slice<V> s;
  __builtin_memcpy(&s, p, 16);
  return s;
}
template <class V>
__device__ inline void store_slice(V* p, const Slice<V>& s) {
  __builtin_memcpy(p, &s, 16);
}
// Slices of a row: the last one ends with the row and overlaps the one before
// (its elements are computed twice, alike).  Rows shorter than a slice have
// none; their elements are taken one by one.
template <class V>
__host__ __device__ inline int64_t slices_of(int64_t width) {
  return width >= Slice<V>::n ? (width + Slice<V>::n - 1) / Slice<V>::n : 0;
}
template <class V>
__device__ inline int64_t slice_start(int64_t c, int64_t width) {
  const int64_t h = c * Slice<V>::n, last = width - Slice<V>::n;
  return h < last ? h : last;
}

template <class A>
__device__ inline A wave_sum(A v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
  return v;
}

// Whether rows `ld_bytes` apart all start at multiples of 16 bytes.
inline bool aligned16(const void* p, int64_t ld_bytes) {
  return ((uintptr_t)p & 15) == 0 && (ld_bytes & 15) == 0;
}

inline size_t value_bytes(int val_t) {
  switch (val_t) {
    case FS_F16:
    case FS_BF16: return 2;
    case FS_F32: return 4;
    case FS_F64: return 8;
  }
  return 0;
}

// Threads of a workgroup of 256 that share a row of `slices` slices.
inline int lanes_per_row(int64_t slices) {
  int l = 8;
  while (l < 256 && l < slices) l <<= 1;
  return l;
}

// Runs f with a value of the value type: real types only.
template <class F>
int with_value_type(int val_t, const char* who, F&& f) {
  switch (val_t) {
    case FS_F16: return f((_Float16)0);
    case FS_BF16: return f((__bf16)0);
    case FS_F32: return f(0.0f);
    case FS_F64: return f(0.0);
  }
  return fail(FS_E_INVALID, std::string(who) + ": bad value type");
}

// select_sort.hip
size_t select_sort_bytes(int64_t n, int64_t n_keys);
int select_sort(const void* ids, int id_t, int64_t n, int64_t n_keys, uint32_t* keys_out, int32_t* order,
                int32_t* inverse, int32_t* offsets, uint8_t* ws, hipStream_t s);

}  // namespace fs
