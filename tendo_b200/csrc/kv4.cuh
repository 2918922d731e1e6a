// kv4.cuh — the paged 4-bit KV cache: layout and row format shared by its
// kernels (kv4.cu, kv4_attention.cu).
//
// A cache is pages[num_blocks][Hkv][block_size / 16] of tiles.  A tile holds
// 16 consecutive positions of one kv head as one contiguous run of whole
// 128-byte lines with everything a warp needs about them:
//   K codes [16][D / 2], V codes [16][D / 2], K words [16], V words [16].
// A code byte j of a row holds channels 2j (low nibble) and 2j + 1, each as
// code + 8 with codes -8 .. 7.  A word is (bf16 scale) | (bf16 zero) << 16,
// and value = zero + scale * code: one rounding, since scale * code has at
// most 12 significant bits.
#pragma once

#include <stdint.h>

#include <atomic>

#include "common.cuh"

namespace tb {

constexpr int kKv4Tile = 16;  // positions per tile

__host__ __device__ constexpr int kv4_tile_bytes(int D) { return 16 * D + 128; }
__host__ __device__ constexpr int kv4_codes_off(int D, int part) { return part * 8 * D; }
__host__ __device__ constexpr int kv4_words_off(int D, int part) { return 16 * D + 64 * part; }

__device__ __forceinline__ float kv4_scale(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float kv4_zero(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// Of a row that cannot be held, one with an infinity or a NaN among them: it
// reads back as NaN.
constexpr uint32_t kKv4NanWord = 0x7fc07fc0u;

// Scale and zero of a row with minimum mn and maximum mx (finite).  The zero
// is rounded to bf16 first and the scale is then the smallest bf16 that still
// covers the row from that zero, so neither rounding can push a value off the
// grid: every value lies within half a scale of its code.  A row for which fp32
// or bf16 has no such zero and scale (values near their ends) cannot be held.
__device__ __forceinline__ uint32_t kv4_word(float mn, float mx) {
  const float z32 = __fadd_rn(__fmul_rn(mn, (float)(7.0 / 15.0)), __fmul_rn(mx, (float)(8.0 / 15.0)));
  const uint32_t zb = (uint32_t)__bfloat16_as_ushort(__float2bfloat16_rn(z32)) << 16;
  const float z = __uint_as_float(zb);
  const float s32 = fmaxf(__fmul_rn(__fsub_rn(z, mn), 0.125f), __fmul_rn(__fsub_rn(mx, z), (float)(1.0 / 7.0)));
  const uint32_t sb = (__float_as_uint(s32) + 0xffffu) >> 16;
  return s32 < INFINITY ? zb | sb : kKv4NanWord;
}

// Code + 8 of x in a row with this scale and zero.
__device__ __forceinline__ uint32_t kv4_code(float x, float scale, float zero) {
  if (!(scale > 0.f)) return 8u;
  const float c = fminf(fmaxf(rintf(__fdiv_rn(__fsub_rn(x, zero), scale)), -8.f), 7.f);
  return (uint32_t)((int)c + 8);
}

__device__ __forceinline__ float kv4_value(uint32_t u, float scale, float zero) {
  return __fadd_rn(zero, __fmul_rn(scale, (float)((int)u - 8)));
}

// Lets `kernel` have `bytes` of dynamic shared memory on the current device,
// once per device (`ready` has a bit for each): always the most that a call may
// ask for, since host threads may launch it side by side.
inline tb_status_t allow_smem(const void* kernel, size_t bytes, std::atomic<uint64_t>& ready) {
  int dev = 0;
  TB_CUDA(cudaGetDevice(&dev));
  const uint64_t bit = dev >= 0 && dev < 64 ? 1ull << dev : 0;
  if (bit && (ready.load(std::memory_order_acquire) & bit)) return TB_SUCCESS;
  TB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
  ready.fetch_or(bit, std::memory_order_release);
  return TB_SUCCESS;
}

}  // namespace tb
