// matrix_core.hpp — 16x16 matrix instructions of the value types, loads straight to
// LDS, waits and barriers: what the kernels on matrix cores share
// (expert_product.hip, block_*.hip).
#pragma once

#include "fs_common.hpp"

namespace fs {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) uint8_t lds_byte;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) u32x2 lds_u32x2;
typedef __attribute__((address_space(3))) float lds_float;

template <class T>
struct Mma;
template <>
struct Mma<_Float16> {
  using frag = f16x8;
  __device__ static f32x4 run(frag a, frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Mma<__bf16> {
  using frag = bf16x8;
  __device__ static f32x4 run(frag a, frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Mma<float> {
  using frag = f32x4;  // four steps of one k a lane
  __device__ static f32x4 run(frag a, frag b, f32x4 c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
    return c;
  }
};

// Offsets of buffer loads that count from their base.
constexpr uint32_t kInBuffer = 1u << 30;

// (No register is written, so none is taken too early; M0 has no other use here.)
template <int WIDTH>
__device__ inline void lds_dma(uint32_t lds, uint32_t offset, u32x4 rsrc) {
  if constexpr (WIDTH == 16)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(offset),
                 "s"(rsrc)
                 : "memory");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(lds), "v"(offset),
                 "s"(rsrc)
                 : "memory");
}
// 16 bytes a lane, from base + offset + shift (a scalar, in bytes, not part of what is
// compared with the buffer's end).
__device__ inline void lds_dma_shifted(uint32_t lds, uint32_t offset, u32x4 rsrc, uint32_t shift) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(lds), "v"(offset),
               "s"(rsrc), "s"(shift)
               : "memory");
}
// The same from an address a lane.
__device__ inline void lds_dma_at(uint32_t lds, const void* p) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(p) : "memory");
}
__device__ inline u32x4 buffer_at(const void* p) {
  const uint64_t a = (uint64_t)(uintptr_t)p;
  return u32x4{(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)a),
               (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(a >> 32)) & 0xffffu, kInBuffer, 0x00020000u};
}

// Waits and the barrier, which nothing is moved across.
template <int LEFT>
__device__ inline void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LEFT) : "memory");
}
__device__ inline void wait_reads() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
}
__device__ inline void barrier() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_barrier" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

}  // namespace
}  // namespace fs
