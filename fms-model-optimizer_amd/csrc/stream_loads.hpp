// 16-byte loads and stores through a buffer descriptor: a lane that has nothing to load asks for an offset past its end and gets zeros (a store
// there is dropped), without a branch around the access.  Branches around loads cost their order: where loads may or may not have been issued,
// the compiler waits for more of them than are needed, and what was asked for steps ahead is waited for at once, and 64-bit addresses cost registers
// (an expert block's gate and up products, 16 tokens 160 us so, 154 without branches; 64 tokens of e4m3 73 and 67; 128 registers and 78).
#pragma once
#include "common.hpp"

namespace fmsmo {

constexpr uint32_t BUF_END = 0x7fffff00u, BUF_NONE = 0x7fffff80u;  // offsets in use are below the first

typedef __amdgpu_buffer_rsrc_t Buf;
// base: the same in all lanes of a wave
__device__ __forceinline__ Buf buf_of(const void* base) { return __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, (int)BUF_END, 0x00020000); }
__device__ __forceinline__ v4i buf_load(Buf b, uint32_t off, uint32_t uniform_off = 0) {
  return __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(b, off, uniform_off, 0));
}
// read once: not kept in the caches
__device__ __forceinline__ v4i buf_stream(Buf b, uint32_t off, uint32_t uniform_off = 0) {
  return __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(b, off, uniform_off, 2));
}
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
// The whole offset in the lane's register: behind a 16-byte store with an offset in a scalar register the compiler puts no wait states before the
// data's registers are written again, and gfx950 has then now and then stored what they were written with (seen in the lowest four bytes).
__device__ __forceinline__ void buf_store(Buf b, v4i v, uint32_t off) {
  __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(v4u, v), b, off, 0, 0);
}

}  // namespace fmsmo
