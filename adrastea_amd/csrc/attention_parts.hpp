// Pieces that the attention kernels share: the layouts of key and value tiles in LDS, exchanges between
// lanes, and transfers from global memory to LDS.
#pragma once

#include "adr_common.hpp"

#define ADR_LDS_PTR(p) ((__attribute__((address_space(3))) void*)(p))

namespace adr {
namespace {

typedef float float2_t __attribute__((ext_vector_type(2)));

// K tile: [64 rows][CPR 16-byte chunks]; chunk kc of row r sits at position kc ^ (line & 15)
// of its 256-byte line (16 lanes reading the same chunk of 16 consecutive rows hit 16
// different bank groups).
template <int CPR>
__device__ __forceinline__ int k_chunk_off(int row, int kc) {
  const int idx = row * CPR + kc, line = idx >> 4, pos = idx & 15;
  return ((line << 4) | (pos ^ (line & (CPR - 1)))) << 4;
}
template <int CPR>
__device__ __forceinline__ void k_chunk_inv(int phys, int& row, int& kc) {
  const int line = phys >> 4, pos = (phys & 15) ^ (line & (CPR - 1));
  const int idx = (line << 4) | pos;
  row = idx / CPR;
  kc = idx % CPR;
}
// V tile: [64 rows][CPR chunks], chunk c of row r at position c ^ v_swz(r): a transposing read
// touches 4 consecutive rows x 4 consecutive chunks per 32 lanes, and the XOR spreads those 16
// chunks over the 16 bank groups (rows of 128 bytes share a 256-byte line in pairs).
template <int CPR>
__device__ __forceinline__ int v_swz(int row) {
  return CPR == 16 ? ((row & 3) << 2) : (((row >> 1) & 1) << 2);
}

// The same for transposing reads of 8 consecutive rows x 2 consecutive chunks per 32 lanes.
template <int CPR>
__device__ __forceinline__ int v_swz8(int row) {
  return CPR == 16 ? ((row & 7) << 1) : (((row >> 1) & 3) << 1);
}

// v_permlane32_swap exchanges the upper half of the first register with the lower half of the second,
// v_permlane16_swap the odd rows of 16 lanes of the first with the even rows of the second: with one
// value in both, a lane then holds its own and its partner's (lane ^ 32, lane ^ 16), without a trip
// through LDS.  The second result passes through an empty asm statement: without it the compiler
// folds a floating-point operation on the two results as if they were the same register.
__device__ __forceinline__ void swap_halves(float& x, float& y) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, y), false, false);
  uint32_t r0 = r[0], r1 = r[1];
  asm volatile("" : "+v"(r1));
  x = __builtin_bit_cast(float, r0);
  y = __builtin_bit_cast(float, r1);
}
__device__ __forceinline__ void swap_rows(float& x, float& y) {
  const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, y), false, false);
  uint32_t r0 = r[0], r1 = r[1];
  asm volatile("" : "+v"(r1));
  x = __builtin_bit_cast(float, r0);
  y = __builtin_bit_cast(float, r1);
}
__device__ __forceinline__ float pair_max(float v) {
  float x = v, y = v;
  swap_halves(x, y);
  return fmaxf(x, y);
}
__device__ __forceinline__ float pair_sum(float v) {
  float x = v, y = v;
  swap_halves(x, y);
  return x + y;
}

// Global -> LDS transfers of 1 KiB (16 bytes per lane, lane l to lds + 16 l).  Assembly, so that the
// compiler does not make every LDS read of the other buffers wait for the transfers in flight;
// the waits are written out below.  The buffer form reads zeros past the end of its descriptor: rows
// beyond the last key need no clamp, and a descriptor of 0 bytes is no transfer at all.  It makes two
// transfers, the second one's offset of 1024 bytes counting on both sides.  (The s_nop: m0, and
// scalars that a vector instruction wrote, need wait states before a memory instruction reads them.)
template <int FIRST>
__device__ __forceinline__ void dma_buffer_pair(uint32_t lds, uint32_t voff0, uint32_t voff1, u32x4_t desc) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %3, 0 offen offset:%4 lds\n\t"
               "buffer_load_dwordx4 %2, %3, 0 offen offset:%5 lds"
               :: "s"(lds), "v"(voff0), "v"(voff1), "s"(desc), "n"(FIRST * 1024), "n"(FIRST * 1024 + 1024) : "memory");
}
// N transfers in a row of what is read once (its lines are the first to leave the caches); the j-th one's offset of j KiB
// counts on both sides.
template <int N>
__device__ __forceinline__ void dma_buffer_once(uint32_t lds, const uint32_t (&voff)[N], u32x4_t desc) {
  static_assert(N == 2 || N == 4, "16 rows of 64 or 128 values");
  if constexpr (N == 4)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %5, 0 offen nt lds\n\t"
                 "buffer_load_dwordx4 %2, %5, 0 offen offset:0x400 nt lds\n\t"
                 "buffer_load_dwordx4 %3, %5, 0 offen offset:0x800 nt lds\n\t"
                 "buffer_load_dwordx4 %4, %5, 0 offen offset:0xc00 nt lds"
                 :: "s"(lds), "v"(voff[0]), "v"(voff[1]), "v"(voff[2]), "v"(voff[3]), "s"(desc) : "memory");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %3, 0 offen nt lds\n\t"
                 "buffer_load_dwordx4 %2, %3, 0 offen offset:0x400 nt lds"
                 :: "s"(lds), "v"(voff[0]), "v"(voff[1]), "s"(desc) : "memory");
}
__device__ __forceinline__ void dma_global(uint32_t lds, const void* p) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, off"
               :: "s"(lds), "v"(p) : "memory");
}
// One transfer of 1 KiB, of what may be read again; one of 256 bytes, a word from each lane.
__device__ __forceinline__ void dma_buffer(uint32_t lds, uint32_t voff, u32x4_t desc) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" :: "s"(lds), "v"(voff), "s"(desc) : "memory");
}
__device__ __forceinline__ void dma_global_word(uint32_t lds, const void* p) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dword %1, off" :: "s"(lds), "v"(p) : "memory");
}
template <int N>
__device__ __forceinline__ void wait_vm() {
  asm volatile("s_waitcnt vmcnt(%0)" :: "n"(N) : "memory");
}
// (A barrier alone: it does not wait for LDS reads in flight.  Whoever reads what another wavefront may
// overwrite behind the next barrier waits for the reads first.  Those issued ahead at the end of a half
// tile, read_v(cV, 0) and read_k(cK, 0) below, need not: they are used, hence waited for, before the
// next barrier, and their buffers are refilled behind that one.)
__device__ __forceinline__ void barrier() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_barrier" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

}  // namespace
}  // namespace adr
