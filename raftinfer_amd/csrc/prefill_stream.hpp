// Device pieces of the prefill kernels that stream K and V tiles through LDS with the
// O^T accumulators in the accumulation registers by number.
#pragma once

#include "prefill_tile.hpp"

#include <type_traits>
#include <utility>

namespace raftinfer::amd {
namespace prefill {

__device__ __forceinline__ bf16x8 lds_read_b128(unsigned addr) {
  return __builtin_bit_cast(bf16x8, *(const __attribute__((address_space(3))) u32x4 *)(std::uintptr_t)(addr));
}
__device__ __forceinline__ u32x2 lds_read_tr16(unsigned addr) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4v *)(std::uintptr_t)(addr)));
}
template <typename T> __device__ __forceinline__ T *lds_ptr(unsigned addr) {
  return (T *)(__attribute__((address_space(3))) T *)(std::uintptr_t)(addr);
}
// off ^ x and off + a, as asm so that the results are formed where they are used:
// hoisted out of the tile loop, the offsets of all loads took registers from the
// Q operands.
template <unsigned kXor, unsigned kAdd> __device__ __forceinline__ std::uint32_t load_offset(std::uint32_t off) {
  std::uint32_t x = off;
  if constexpr (kXor != 0) asm volatile("v_xor_b32 %0, %2, %1" : "=v"(x) : "v"(off), "n"(kXor));
  if constexpr (kAdd != 0) asm volatile("v_add_u32 %0, %2, %1" : "=v"(x) : "v"(x), "n"(kAdd));
  return x;
}
// load_lds_b128 with an instruction offset, which the hardware adds to both the
// memory and the LDS address.  Between the write of M0 and the load the hardware
// needs a wait state; the five in front of it for a base that a vector instruction
// writes are for the compiler's scalar arithmetic to give (the build checks both).
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
template <int kOffset>
__device__ __forceinline__ void load_lds_b128_at(const void *base, std::uint32_t voff, unsigned lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 offset:%3"
               :
               : "s"(lds), "v"(voff), "s"(base), "n"(kOffset)
               : "memory", "m0");
}

// 16 bytes from an address of each lane's own into LDS at lds + 16 * lane.
__device__ __forceinline__ void load_lds_b128_lane(const void *from, unsigned lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(lds), "v"(from) : "memory", "m0");
}
#pragma clang diagnostic pop

// The O^T accumulators (2 column blocks x 8 dim blocks x 16 registers) fill the
// 256 accumulation registers, and are addressed by number from asm: block
// `kAcc` (8 b + nb) is a[16 kAcc : 16 kAcc + 15].  Left to the register
// allocator, values of this size were copied and spilled around every tile.
// acc_fence clobbers the whole file around every tile, so the compiler keeps
// nothing of its own there (the statements in between carry no clobber list,
// which took minutes to compile); the build checks that no instruction outside
// asm uses an accumulation register (raftinfer_amd/asm_check.py).
#define RAFT_AGPR10(n) \
  "a" #n "0", "a" #n "1", "a" #n "2", "a" #n "3", "a" #n "4", "a" #n "5", "a" #n "6", "a" #n "7", "a" #n "8", "a" #n "9"
#define RAFT_ALL_AGPRS \
  "a0", "a1", "a2", "a3", "a4", "a5", "a6", "a7", "a8", "a9", \
      RAFT_AGPR10(1), RAFT_AGPR10(2), RAFT_AGPR10(3), RAFT_AGPR10(4), \
      RAFT_AGPR10(5), RAFT_AGPR10(6), RAFT_AGPR10(7), RAFT_AGPR10(8), \
      RAFT_AGPR10(9), RAFT_AGPR10(10), RAFT_AGPR10(11), RAFT_AGPR10(12), \
      RAFT_AGPR10(13), RAFT_AGPR10(14), RAFT_AGPR10(15), RAFT_AGPR10(16), \
      RAFT_AGPR10(17), RAFT_AGPR10(18), RAFT_AGPR10(19), RAFT_AGPR10(20), \
      RAFT_AGPR10(21), RAFT_AGPR10(22), RAFT_AGPR10(23), RAFT_AGPR10(24), \
      "a250", "a251", "a252", "a253", "a254", "a255"

__device__ __forceinline__ void acc_fence() { asm volatile("" : : : RAFT_ALL_AGPRS); }
template <int kAcc> __device__ __forceinline__ void acc_mfma(bf16x8 a, bf16x8 b) {
  asm volatile("v_mfma_f32_32x32x16_bf16 a[%0:%1], %2, %3, a[%0:%1]"
               :
               : "n"(16 * kAcc), "n"(16 * kAcc + 15), "v"(a), "v"(b));
}
// s = a b and s += a b with s in vector registers.  A statement writes no
// result for another 19 wait states: new_max reads S(t + 4) only after PV(t),
// and after the first tile's chain the kernel drains.
__device__ __forceinline__ void s_mfma_zero(floatx16 &s, bf16x8 a, bf16x8 b) {
  asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, 0" : "=&v"(s) : "v"(a), "v"(b));
}
__device__ __forceinline__ void s_mfma(floatx16 &s, bf16x8 a, bf16x8 b) {
  asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+v"(s) : "v"(a), "v"(b));
}
template <int kReg> __device__ __forceinline__ void acc_set(float x) {
  asm volatile("v_accvgpr_write_b32 a[%0], %1" : : "n"(kReg), "v"(x));
}
template <int kReg> __device__ __forceinline__ float acc_get() {
  float x;
  asm volatile("v_accvgpr_read_b32 %0, a[%1]" : "=v"(x) : "n"(kReg));
  return x;
}
// max(a, b, c).  As asm: on results of the asm MFMAs fmaxf adds a canonicalising
// instruction per operand.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float x;
  asm volatile("v_max3_f32 %0, %1, %2, %3" : "=v"(x) : "v"(a), "v"(b), "v"(c));
  return x;
}
// The wait states between the last s_mfma of a chain and the first use of s.
template <int NB> __device__ __forceinline__ void s_drain(floatx16 (&s)[NB]) {
  if constexpr (NB == 2)
    asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 3" : "+v"(s[0]), "+v"(s[1]));
  else
    asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 3" : "+v"(s[0]));
}
// f(integral_constant<int, 0>) .. f(integral_constant<int, N - 1>)
template <int N, typename F> __device__ __forceinline__ void static_for(F &&f) {
  [&]<int... I>(std::integer_sequence<int, I...>) __attribute__((always_inline)) { (f(std::integral_constant<int, I>{}), ...); }
  (std::make_integer_sequence<int, N>{});
}

} // namespace prefill
} // namespace raftinfer::amd
