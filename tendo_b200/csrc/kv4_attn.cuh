// kv4_attn.cuh — what the two attention kernels over the 4-bit cache share:
// kv4_attention.cu (a few query rows per kv head) and kv4_prefill.cu (more).
#pragma once

#include <limits.h>

#include <cuda_fp16.h>

#include "common.cuh"
#include "kv4.cuh"

namespace tb {

constexpr int kKv4MaxB = 1024;        // 20 bytes per request in shared memory
// Query rows per kv head up to which kv4_attention.cu is the faster kernel.  It
// and kv4_prefill.cu, 8 kv heads of 128 with 8 heads each: 16 requests of 2100
// positions, 64 rows 101 and 99 us, 80 rows 110 and 96, 96 rows 144 and 103; 4 of 8000:
// 48 rows 67 and 73, 80 rows 86 and 70; 64 of 600: 64 rows 133 and 163, 80 rows 161
// and 177, 96 rows 188 and 177.  Heads of 32, 16 of 2100: 48 rows 45 and 54, 80 rows
// 60 and 52.  So the crossing lies between 48 and 96 rows by the number of units,
// and the rule, which looks at the rows alone, is up to 10% off on either side.
constexpr int kKv4FewRows = 64;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNoMax = -1e30f;      // running maximum of a row that has seen no key

// One launch: the requests whose query rows per kv head (new tokens times the
// group) lie in min_rows .. max_rows.
struct Kv4AttnArgs {
  float* out;
  const float* q;
  const uint8_t* pages;
  const int32_t *table, *lens, *starts;
  float* part;   // [2 * CTAs + workers][rows][D + 4]: CTAs' chains, warps' first segments
  int4* desc;    // [CTAs] units that a CTA begins and others go on with
  int32_t* bad;
  int64_t q_stride;
  int B, T, H, Hkv, G, block, max_blocks, num_blocks;
  float scale;
  int tpb, rpb;            // tokens and query rows of a unit (kv4_prefill.cu)
  int bpt_shift;           // log2 of a page's tiles, or -1
  int min_rows, max_rows;
  bool vec, fill;          // fill: this launch zeroes the rows of no request
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two fp32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n .reg .b64 a, b, c, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n mov.b64 c, {%6, %7};\n"
      " fma.rn.f32x2 d, a, b, c;\n mov.b64 {%0, %1}, d;\n}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n .reg .b64 a, b, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n add.rn.f32x2 d, a, b;\n"
      " mov.b64 {%0, %1}, d;\n}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n .reg .b64 a, b, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n mul.rn.f32x2 d, a, b;\n"
      " mov.b64 {%0, %1}, d;\n}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
// fp16 values code + bias of nibbles, minus the bias: `magic` puts the nibble
// into the mantissa of 1024 (bits 0-3) or 64 (bits 4-7).
__device__ __forceinline__ uint32_t nibble_f16(uint32_t w, uint32_t mask, uint32_t magic, uint32_t bias) {
  uint32_t x;  // (w & mask) | magic in one instruction
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(x) : "r"(w), "r"(mask), "r"(magic));
  __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&bias));
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Requests of the launch as the kernel uses them: counts that a caller got
// wrong are cut to what the buffers hold.
__device__ __forceinline__ int req_start(const Kv4AttnArgs& a, int b) { return min(max(a.starts[b], 0), a.T); }
__device__ __forceinline__ int req_new(const Kv4AttnArgs& a, int b) {  // 0: not this launch's
  const int n = max(req_start(a, b + 1) - req_start(a, b), 0), rows = n * a.G;
  return rows >= a.min_rows && rows <= a.max_rows ? n : 0;
}
__device__ __forceinline__ int req_len(const Kv4AttnArgs& a, int b) {
  // a length rounded up to whole chunks or tiles, and a position past it, are ints
  const int64_t most = min((int64_t)a.max_blocks * a.block, (int64_t)(INT_MAX - 127));
  const int len = max(a.lens[b], 0);
  return len < most ? len : (int)most;
}

// Zeroes the rows of no request, before the first one's and after the last
// one's (offsets may be those of a part of a batch); threads of the whole grid.
// Out of line, where it takes no registers from the kernels' loops.
static __device__ __noinline__ void zero_but(float* out, int begin, int end, int T, int row) {
  const int64_t before = (int64_t)begin * row, skip = (int64_t)end * row - before;
  const int64_t n = (int64_t)T * row - skip;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x)
    out[i < before ? i : i + skip] = 0.f;
}
__device__ __forceinline__ void zero_rows_of_none(const Kv4AttnArgs& a, int D) {
  const int end = a.B > 0 ? req_start(a, a.B) : 0, begin = a.B > 0 ? min(req_start(a, 0), end) : 0;
  if (begin > 0 || end < a.T) zero_but(a.out, begin, end, a.T, a.H * D);
}

// kv4_prefill.cu: G at most 128.  Parts and descriptors of a launch in `ws`.
size_t kv4_prefill_workspace(int64_t G, int64_t max_q, int64_t D);
tb_status_t kv4_prefill(Kv4AttnArgs a, int64_t max_q, int D, void* ws, cudaStream_t st);

}  // namespace tb
