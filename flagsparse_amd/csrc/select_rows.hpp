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
// PAST: past the caches (of their own kind, a choice at run time is compiled
// into plain stores).
template <bool PAST = false, class V>
__device__ inline void store_slice(V* p, const Slice<V>& s) {
  if constexpr (PAST) {
    typedef uint32_t words4 __attribute__((ext_vector_type(4)));
    typedef words4 words __attribute__((aligned(2)));
    words u;
    __builtin_memcpy(&u, &s, 16);
    __builtin_nontemporal_store(u, reinterpret_cast<words*>(p));
  } else {
    __builtin_memcpy(p, &s, 16);
  }
}
// Whether a call that reads and writes `bytes` in all stores past the caches:
// where that is more than the Infinity Cache holds, keeping results there only
// drives out what is still to be read.  us with and without, inputs not in cache:
// dispatch 16384 x 8 of 2048 bf16 103 and 110, its 4096 tokens 26 and 23; combine 108
// and 117; embedding gradient 65536 tokens x 2048, 131072 rows bf16 214 and 228, 512 x
// 1024, 50000 rows f32 42 and 43.  combine_grad gains where the call before left its
// inputs in cache and loses where not: 4096 x 4 of 2048 f32 44 and 50, 60 and 51, 8191 x
// 8 of 2560 f16 134 and 140, 137 and 135, 32768 x 8 of 4096 bf16 869 and 875.
// (Rows of whole words: dispatch 2047 wide took 148 and 133.)
inline bool store_past_caches(int64_t bytes, int64_t row_bytes) {
  return bytes >= (int64_t)256 << 20 && row_bytes % 4 == 0;
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

// Inclusive sum over the lanes up to this one (row shifts, then row broadcasts;
// lanes without a source read 0).
template <int CTRL, int ROWS>
__device__ inline uint32_t lane_shifted(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false);
}
__device__ inline uint32_t wave_sum_scan(uint32_t v) {
  v += lane_shifted<0x111, 0xF>(v);  // row_shr:1
  v += lane_shifted<0x112, 0xF>(v);  // row_shr:2
  v += lane_shifted<0x114, 0xF>(v);  // row_shr:4
  v += lane_shifted<0x118, 0xF>(v);  // row_shr:8
  v += lane_shifted<0x142, 0xA>(v);  // row_bcast:15 -> rows 1, 3
  v += lane_shifted<0x143, 0xC>(v);  // row_bcast:31 -> rows 2, 3
  return v;
}

// Threads of a workgroup of 256 that share a row of `slices` slices.
inline int lanes_per_row(int64_t slices) {
  int l = 8;
  while (l < 256 && l < slices) l <<= 1;
  return l;
}

// Workgroups in two dimensions: a dimension of a grid holds below 2^32 threads.
inline dim3 row_grid(int64_t blocks) {
  const int64_t x = std::min<int64_t>(blocks, 1 << 22);
  return dim3((uint32_t)x, (uint32_t)ceil_div(blocks, x));
}
__device__ inline int64_t row_block() { return (int64_t)blockIdx.y * gridDim.x + blockIdx.x; }

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
int64_t select_sort_fill_bytes(int64_t n);
int select_sort(const void* ids, int id_t, int64_t n, int64_t n_keys, uint32_t* keys_out, int32_t* order,
                int32_t* inverse, int32_t* offsets, uint8_t* ws, hipStream_t s, void* zeros, int64_t zero_bytes);

}  // namespace fs
