// Direct-to-LDS loads, LDS barriers and transposed LDS reads shared by the
// attention kernels (gfx950).
#pragma once

#include "kvc_internal.h"

namespace kvc {

constexpr int kBufWord3 = 0x00020000;  // gfx9 raw buffer: 32-bit data format

// One 16-byte-per-lane load straight into LDS: lane i's 16 bytes from
// rsrc + voff land at LDS address lds + 16 i.  Issued through inline asm so
// the compiler's wait-count pass does not treat it as a pending LDS write
// (it would then drain every load in flight before each barrier and LDS read,
// serialising the prefetch); the caller waits with explicit vmcnt counts.
// M0 carries the LDS address and is restored afterwards; a load may not read
// it in the cycle after a scalar write (one wait state, which the compiler
// does not insert inside inline asm).
typedef int i32x4_t __attribute__((ext_vector_type(4)));
__device__ __forceinline__ i32x4_t raw_rsrc(const void* base, int bytes) {
  const uint64_t a = reinterpret_cast<uint64_t>(base);
  return i32x4_t{int(__builtin_amdgcn_readfirstlane(uint32_t(a))),
                 int(__builtin_amdgcn_readfirstlane(uint32_t(a >> 32) & 0xffffu)),
                 int(__builtin_amdgcn_readfirstlane(uint32_t(bytes))), kBufWord3};
}

__device__ __forceinline__ void dma_to_lds(const i32x4_t& rsrc, int voff, uint32_t lds) {
  uint32_t saved;
  asm volatile(
      "s_mov_b32 %0, m0\n\t"
      "s_mov_b32 m0, %2\n\t"
      "s_nop 0\n\t"
      "buffer_load_dwordx4 %1, %3, 0 offen nt lds\n\t"
      "s_mov_b32 m0, %0"
      : "=&s"(saved)
      : "v"(voff), "s"(lds), "s"(rsrc)
      : "memory");
}

// The same load with the default cache policy, for data that other
// workgroups read again soon (prefill keys and queries).
__device__ __forceinline__ void dma_to_lds_cached(const i32x4_t& rsrc, int voff, uint32_t lds) {
  uint32_t saved;
  asm volatile(
      "s_mov_b32 %0, m0\n\t"
      "s_mov_b32 m0, %2\n\t"
      "s_nop 0\n\t"
      "buffer_load_dwordx4 %1, %3, 0 offen lds\n\t"
      "s_mov_b32 m0, %0"
      : "=&s"(saved)
      : "v"(voff), "s"(lds), "s"(rsrc)
      : "memory");
}

__device__ __forceinline__ uint32_t lds_addr(const void* p) {
  return __builtin_amdgcn_readfirstlane(
      uint32_t(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const char*)p)));
}

// s_waitcnt immediate for lgkmcnt(0) alone (vmcnt 63 and expcnt 7 do not wait).
constexpr int kWaitLgkm0 = 0xC07F;

// Workgroup barrier over LDS only: this wave's LDS accesses are complete and
// every wave has arrived.  (__syncthreads would also wait for the epilogue's
// global stores, and with them for every direct-to-LDS load in flight.)  The
// wait and the barrier are builtins, so the compiler's wait-count model knows
// the LDS queue is empty after it; the empty asm statements keep memory
// accesses from moving across it.
__device__ __forceinline__ void pf_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(kWaitLgkm0);
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Scalar loads (block-table entries, chunk bounds) are waited for right where
// they are issued: while one is pending the compiler's wait-count model must
// treat the LDS counter as out of order and waits for every LDS read before
// the first use of any, which serialises the K and V operand reads with the
// MFMAs.  With the queue drained here its LDS waits stay partial.
__device__ __forceinline__ void smem_drain() { __builtin_amdgcn_s_waitcnt(kWaitLgkm0); }

typedef short s16x4v_t __attribute__((ext_vector_type(4)));
__device__ __forceinline__ u32x2_t lds_read_tr16(const char* p) {
  const s16x4v_t r = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (__attribute__((address_space(3))) s16x4v_t*)(
          (__attribute__((address_space(3))) char*)(p)));
  return __builtin_bit_cast(u32x2_t, r);
}

}  // namespace kvc
