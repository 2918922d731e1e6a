// kv4_attention.cu — attention over the paged 4-bit KV cache (kv4.cuh).
//
//   out[i, h] = sum_j softmax_j(scale q_i . k_j) v_j,  j <= len - n + i
//
// for the n new tokens i of each request, whose keys are already in the cache.
//
// The codes are integers -8 .. 7, so both products run on fp16 tensor cores
// without rounding the cache: q . k_j = s_j (q . u_j - 8 sum q) + z_j sum q
// with u_j = code + 8, and p_j v_j = (p_j s_j) c_j + p_j z_j.  The fp32
// operands q and p_j s_j are split into two fp16 terms (22 bits), which sit in
// neighbouring columns of the MMA's 8-column side; positions (or channels)
// are its 16-row side.  So 4 query rows of one kv head share every unpacked
// code, and a lane holds both terms of a score and adds them.
#include <limits.h>
#include <math.h>

#include <cuda_fp16.h>

#include "common.cuh"
#include "kernels.h"
#include "kv4.cuh"
#include "tma_common.cuh"

namespace tb {
namespace {

constexpr int kChunk = 32;      // positions a warp takes at a time: two tiles
constexpr int kMaxB = 2048;     // prefix of 8 bytes per request in shared memory
constexpr float kLog2e = 1.4426950408889634f;

struct Kv4AttnArgs {
  float* out;
  const float* q;
  const uint8_t* pages;
  const int32_t *table, *lens, *starts;
  float* part;   // [2 * workers][rows][D + 2]
  int4* desc;    // [workers] units that a worker begins and others go on with
  int32_t* bad;
  int* err;
  int64_t q_stride;
  int B, T, H, Hkv, G, block, max_blocks, num_blocks, workers;
  float scale;
  bool vec;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// D += A[16 x 16] . B[16 x 8], fp16 in, fp32 accumulate.
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Transposes an 8 x 8 matrix of 16-bit elements held two to a lane.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// (lo, hi) of two floats as fp16.
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
// x = high + low with the high term's 11 leading bits exact in fp16 (truncated,
// so that the difference is exact), packed high first.
__device__ __forceinline__ uint32_t split_f16(float x) {
  const float hi = __uint_as_float(__float_as_uint(x) & 0xffffe000u);
  return pack_f16(hi, x - hi);
}
// fp16 values code + bias of nibbles, minus the bias: `magic` puts the nibble
// into the mantissa of 1024 (bits 0-3) or 64 (bits 4-7).
__device__ __forceinline__ uint32_t nibble_f16(uint32_t w, uint32_t mask, uint32_t magic, uint32_t bias) {
  const uint32_t x = (w & mask) | magic;
  __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&bias));
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <int N>
struct Words {
  uint32_t w[N];
};
template <int N>
__device__ __forceinline__ Words<N> lds_words(const uint8_t* p) {
  Words<N> r;
  if constexpr (N == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    r.w[0] = v.x, r.w[1] = v.y, r.w[2] = v.z, r.w[3] = v.w;
  } else if constexpr (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    r.w[0] = v.x, r.w[1] = v.y;
  } else {
    r.w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
  return r;
}

// Where a worker stands in the flat list of chunks.
struct Cursor {
  int b, head, rb;     // request, kv head, row block
  int chunk, chunks;   // position within the unit and its length
};

// Requests of the launch as the kernel uses them: counts that a caller got
// wrong are cut to what the buffers hold.
__device__ __forceinline__ int req_start(const Kv4AttnArgs& a, int b) { return min(max(a.starts[b], 0), a.T); }
__device__ __forceinline__ int req_new(const Kv4AttnArgs& a, int b) {
  return max(req_start(a, b + 1) - req_start(a, b), 0);
}
__device__ __forceinline__ int req_len(const Kv4AttnArgs& a, int b) {
  const int64_t most = (int64_t)a.max_blocks * a.block;
  const int len = max(a.lens[b], 0);
  return len < most ? len : (int)most;
}

template <int D, int NT>
struct Smem {
  static constexpr int kTile = kv4_tile_bytes(D);
  static constexpr int kStage = 2 * kTile;
  static constexpr int kQFrags = NT > 2 ? NT * (D / 16) * 2 * 32 * 4 : 0;  // bytes per warp
  static constexpr int kPerWarpFixed = kQFrags + 128;                      // + barriers and tile flags
};

template <int D, int NT, int WARPS, int STAGES>
__global__ void __launch_bounds__(WARPS * 32, 1) kv4_attn_kernel(Kv4AttnArgs a) {
  constexpr int KW = D / 32;        // K words of a lane per row
  constexpr int MT = D / 16;        // 16-channel tiles of the output
  constexpr int VC = D / 8;         // channels of a lane in V rows and in the output
  constexpr int RPB = 4 * NT;       // query rows per unit
  constexpr bool kQS = NT > 2;      // q fragments in shared memory
  using S = Smem<D, NT>;
  extern __shared__ __align__(128) uint8_t smem[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
  uint8_t* ring = smem + warp * (STAGES * S::kStage);
  uint8_t* fixed = smem + WARPS * (STAGES * S::kStage) + warp * S::kPerWarpFixed;
  uint32_t* qfs = reinterpret_cast<uint32_t*>(fixed);
  uint64_t* bar = reinterpret_cast<uint64_t*>(fixed + S::kQFrags);
  volatile int* flags = reinterpret_cast<volatile int*>(fixed + S::kQFrags + 8 * STAGES);
  static_assert(12 * STAGES <= 128, "barriers and flags of a warp");
  int64_t* pre = reinterpret_cast<int64_t*>(smem + WARPS * (STAGES * S::kStage + S::kPerWarpFixed));
  __shared__ int64_t wsum[WARPS];

  if (lane == 0)
    for (int s = 0; s < STAGES; s++) mbarrier_init(&bar[s], 1);
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");

  // chunks of each request over its kv heads and row blocks, as a running sum
  {
    const int per = (a.B + WARPS * 32 - 1) / (WARPS * 32);
    const int b0 = min(tid * per, a.B), b1 = min(b0 + per, a.B);
    auto chunks_of = [&](int b) {
      const int rows = req_new(a, b) * a.G, len = req_len(a, b);
      return (int64_t)((rows + RPB - 1) / RPB) * a.Hkv * ((len + kChunk - 1) / kChunk);
    };
    int64_t mine = 0;
    for (int b = b0; b < b1; b++) mine += chunks_of(b);
    int64_t inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t v = __shfl_up_sync(~0u, inc, o);
      if (lane >= o) inc += v;
    }
    if (lane == 31) wsum[warp] = inc;
    __syncthreads();
    int64_t run = inc - mine;
    for (int w = 0; w < warp; w++) run += wsum[w];
    for (int b = b0; b < b1; b++) {
      pre[b] = run;
      run += chunks_of(b);
    }
    if (b1 == a.B && (b0 < a.B || tid == 0)) pre[a.B] = run;
    __syncthreads();
  }
  // rows of no request, and of requests without a key, are zero
  {
    const int used = a.B > 0 ? req_start(a, a.B) : 0;
    const int64_t n = (int64_t)(a.T - used) * a.H * D;
    for (int64_t i = (int64_t)blockIdx.x * (WARPS * 32) + tid; i < n; i += (int64_t)gridDim.x * (WARPS * 32))
      a.out[(int64_t)used * a.H * D + i] = 0.f;
    for (int b = blockIdx.x; b < a.B; b += gridDim.x)
      if (pre[b] == pre[b + 1]) {
        const int64_t m = (int64_t)req_new(a, b) * a.H * D;
        for (int64_t i = tid; i < m; i += WARPS * 32) a.out[(int64_t)req_start(a, b) * a.H * D + i] = 0.f;
      }
  }
  const int64_t total = pre[a.B];
  const int64_t per = max((total + a.workers - 1) / a.workers, (int64_t)1);
  const int worker = blockIdx.x * WARPS + warp;
  const int64_t beg = min(worker * per, total), end = min(beg + per, total);
  if (lane == 0) a.desc[worker] = make_int4(-1, 0, 0, 0);
  pdl_launch_dependents();
  if (beg >= end) return;

  auto seek = [&](int64_t x) {
    int lo = 0, hi = a.B;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (pre[mid] <= x)
        lo = mid;
      else
        hi = mid;
    }
    // lo is the last request with pre <= x, and so one that has chunks
    Cursor c;
    c.b = lo;
    c.chunks = (req_len(a, lo) + kChunk - 1) / kChunk;
    const int64_t rel = x - pre[lo];
    const int unit = (int)(rel / c.chunks);
    c.chunk = (int)(rel - (int64_t)unit * c.chunks);
    const int rbs = (req_new(a, lo) * a.G + RPB - 1) / RPB;
    c.head = unit / rbs;
    c.rb = unit - c.head * rbs;
    return c;
  };
  // the chunk after c (x is its place in the flat list)
  auto step = [&](Cursor& c, int64_t x) {
    if (++c.chunk == c.chunks && x < end) c = seek(x);
  };

  // --- producer side of the warp: lanes 0 and 1 bring one tile each ---------
  Cursor pc = seek(beg);
  int64_t px = beg;
  int next_blk = -1;
  auto look = [&]() {  // the table entry of the chunk at the producer's cursor
    next_blk = -1;
    if (lane < 2 && px < end) {
      const int pos = pc.chunk * kChunk + lane * kKv4Tile;
      if (pos < req_len(a, pc.b)) next_blk = a.table[(int64_t)pc.b * a.max_blocks + pos / a.block];
      else next_blk = -2;
    }
  };
  int issue_stage = 0;
  auto issue = [&]() {
    if (px >= end) return;
    const bool wanted = lane < 2 && next_blk != -2;
    const bool good = wanted && next_blk >= 0 && next_blk < a.num_blocks;
    const unsigned m = __ballot_sync(~0u, good);
    if (wanted && !good && a.bad) atomicAdd(a.bad, 1);
    if (lane == 0) {
      flags[issue_stage] = (int)m;
      mbarrier_expect_tx(&bar[issue_stage], __popc(m) * S::kTile);
    }
    __syncwarp();
    if (good) {
      const int pos = pc.chunk * kChunk + lane * kKv4Tile;
      const int sub = pos % a.block / kKv4Tile;
      const uint8_t* src = a.pages + (((int64_t)next_blk * a.Hkv + pc.head) * (a.block / kKv4Tile) + sub) *
                                         (int64_t)S::kTile;
      bulk_copy_g2s(ring + issue_stage * S::kStage + lane * S::kTile, src, S::kTile, &bar[issue_stage]);
    }
    issue_stage = issue_stage + 1 == STAGES ? 0 : issue_stage + 1;
    px++;
    step(pc, px);
    look();
  };
  look();
#pragma unroll 1
  for (int s = 0; s < STAGES; s++) issue();

  // --- consumer --------------------------------------------------------------
  float o[MT][NT][4];
  uint32_t qf[kQS ? 1 : NT][kQS ? 1 : D / 16][2];
  float A1[NT], A2[NT], m[NT], l[NT], za[NT];
  int vis[NT];
  int vexp = 0;  // accumulators hold 2^vexp times the sums
  int min_vis = 0;
  Cursor c = seek(beg);
  int64_t x = beg, unit_first = beg - c.chunk;
  bool fresh = true;
  int stage = 0;
  uint32_t phase = 0;

#pragma unroll 1
  while (x < end) {
    if (fresh) {
      fresh = false;
      const int nq = req_new(a, c.b), len = req_len(a, c.b), rows = nq * a.G, r0 = c.rb * RPB;
      const int64_t first = req_start(a, c.b);
      // q rows as fp16 pairs: column g of tile nt is term g & 1 of row 4 nt + g / 2
      float st_a1[NT], st_a2[NT];
#pragma unroll
      for (int nt = 0; nt < NT; nt++) {
        const int r = r0 + 4 * nt + (g >> 1);
        float v[D / 4];
        if (r < rows) {
          const float* src = a.q + (first + r / a.G) * a.q_stride + (c.head * a.G + r % a.G) * D + t4 * (D / 4);
          if (a.vec) {
#pragma unroll
            for (int i = 0; i < D / 16; i++) {
              const float4 f = reinterpret_cast<const float4*>(src)[i];
              v[4 * i] = f.x, v[4 * i + 1] = f.y, v[4 * i + 2] = f.z, v[4 * i + 3] = f.w;
            }
          } else {
#pragma unroll
            for (int i = 0; i < D / 4; i++) v[i] = src[i];
          }
        } else {
#pragma unroll
          for (int i = 0; i < D / 4; i++) v[i] = 0.f;
        }
        float mx = 0.f, sum = 0.f;
#pragma unroll
        for (int i = 0; i < D / 4; i++) {
          mx = fmaxf(mx, fabsf(v[i]));
          sum += v[i];
        }
        mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, 2));
        sum += __shfl_xor_sync(~0u, sum, 1);
        sum += __shfl_xor_sync(~0u, sum, 2);
        // a power of two that brings the row's largest element to 2^13 .. 2^14
        int e = mx > 0.f ? 13 - ((int)(__float_as_uint(mx) >> 23) - 127) : 0;
        e = max(min(e, 100), -114);
        const float up = __int_as_float((e + 127) << 23);
        st_a1[nt] = a.scale * kLog2e * __int_as_float((127 - e) << 23) * 16777216.f;
        st_a2[nt] = a.scale * kLog2e * sum;
#pragma unroll
        for (int i = 0; i < D / 32; i++)
#pragma unroll
          for (int s = 0; s < 2; s++) {
            const float* w = v + 8 * i + 2 * s;
            const float f[4] = {w[0] * up, w[4] * up, w[1] * up * 0.0625f, w[5] * up * 0.0625f};
            float h[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
              const float hi = __half2float(__float2half_rn(f[j]));
              h[j] = (g & 1) ? f[j] - hi : hi;
            }
            const uint32_t b0 = pack_f16(h[0], h[1]), b1 = pack_f16(h[2], h[3]);
            if (kQS) {
              reinterpret_cast<uint2*>(qfs)[(nt * (D / 16) + 2 * i + s) * 32 + lane] = make_uint2(b0, b1);
            } else {
              qf[nt][2 * i + s][0] = b0;
              qf[nt][2 * i + s][1] = b1;
            }
          }
      }
      min_vis = INT_MAX;
#pragma unroll
      for (int nt = 0; nt < NT; nt++) {  // a lane's scores are of row 4 nt + t4: column 2 t4
        A1[nt] = __shfl_sync(~0u, st_a1[nt], 8 * t4);
        A2[nt] = __shfl_sync(~0u, st_a2[nt], 8 * t4);
        const int r = r0 + 4 * nt + t4;
        vis[nt] = r < rows ? len - nq + r / a.G + 1 : 0;
        min_vis = min(min_vis, len - nq + min(r, rows - 1) / a.G + 1);
        m[nt] = -INFINITY;
        l[nt] = za[nt] = 0.f;
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
          for (int j = 0; j < 4; j++) o[i][nt][j] = 0.f;
      }
      min_vis = __reduce_min_sync(~0u, min_vis);
      vexp = 1000;  // no scale chosen yet
      if (kQS) __syncwarp();
    }

    mbarrier_wait(&bar[stage], phase, a.err);
    const uint8_t* buf = ring + stage * S::kStage;
    const int tiles = flags[stage];
    const int p0 = c.chunk * kChunk;

    // scores: two tiles of 16 positions x 4 NT rows (two columns a row)
    float s[2][NT][4];
#pragma unroll
    for (int j = 0; j < 2; j++) {
      const Words<KW> ka = lds_words<KW>(buf + j * S::kTile + g * (D / 2) + t4 * (D / 8));
      const Words<KW> kb = lds_words<KW>(buf + j * S::kTile + (g + 8) * (D / 2) + t4 * (D / 8));
#pragma unroll
      for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int i = 0; i < 4; i++) s[j][nt][i] = 0.f;
#pragma unroll
      for (int i = 0; i < KW; i++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
          // a nibble in the low bits of an fp16 is the subnormal u 2^-24, one
          // place up u 2^-20: q's matching half carries the 1/16
          const uint32_t wa = ka.w[i] >> (8 * h), wb = kb.w[i] >> (8 * h);
          const uint32_t a0 = wa & 0x000f000fu, a1 = wb & 0x000f000fu, a2 = wa & 0x00f000f0u, a3 = wb & 0x00f000f0u;
#pragma unroll
          for (int nt = 0; nt < NT; nt++) {
            uint32_t b0, b1;
            if (kQS) {
              const uint2 b = reinterpret_cast<const uint2*>(qfs)[(nt * (D / 16) + 2 * i + h) * 32 + lane];
              b0 = b.x, b1 = b.y;
            } else {
              b0 = qf[kQS ? 0 : nt][kQS ? 0 : 2 * i + h][0];
              b1 = qf[kQS ? 0 : nt][kQS ? 0 : 2 * i + h][1];
            }
            mma_f16(s[j][nt], a0, a1, a2, a3, b0, b1);
          }
        }
    }
    // this lane's positions: p0 + 16 j + g (+ 8)
    float ks[4], kz[4], vs[4], vz[4];
    float smax = 0.f;
#pragma unroll
    for (int j = 0; j < 2; j++)
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const uint32_t* words = reinterpret_cast<const uint32_t*>(buf + j * S::kTile + kv4_words_off(D, 0));
        const uint32_t kw = words[g + 8 * h], vw = words[16 + g + 8 * h];
        ks[2 * j + h] = kv4_scale(kw);
        kz[2 * j + h] = kv4_zero(kw);
        vs[2 * j + h] = kv4_scale(vw);
        vz[2 * j + h] = kv4_zero(vw);
      }
    const bool whole = tiles == 3 && p0 + kChunk <= min_vis;
    float tsc[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float sum = s[i >> 1][nt][2 * (i & 1)] + s[i >> 1][nt][2 * (i & 1) + 1];
        tsc[nt][i] = fmaf(ks[i], fmaf(sum, A1[nt], -8.f * A2[nt]), kz[i] * A2[nt]);
      }
    if (!whole) {
      // positions that no row of the block sees may hold anything
      int last = 0;
#pragma unroll
      for (int nt = 0; nt < NT; nt++) last = max(last, vis[nt]);
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int p = p0 + 16 * (i >> 1) + g + 8 * (i & 1);
        const bool there = tiles >> (i >> 1) & 1;
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
          if (p >= vis[nt] || !there) tsc[nt][i] = -INFINITY;
        if (p >= last || !there) vs[i] = vz[i] = 0.f;
      }
    }
#pragma unroll
    for (int i = 0; i < 4; i++) smax = fmaxf(smax, vs[i]);

    // running maxima; rescale what is summed so far when one moves
    float mnew[NT];
    bool moved = false;
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      float v = fmaxf(fmaxf(tsc[nt][0], tsc[nt][1]), fmaxf(tsc[nt][2], tsc[nt][3]));
      v = fmaxf(v, __shfl_xor_sync(~0u, v, 4));
      v = fmaxf(v, __shfl_xor_sync(~0u, v, 8));
      v = fmaxf(v, __shfl_xor_sync(~0u, v, 16));
      mnew[nt] = fmaxf(m[nt], v);
      moved |= mnew[nt] > m[nt];
    }
    // V's scales: 2^vexp s stays at or below 2^15 (fp16 holds 40 binades of it)
    int vnew = vexp;
    const float cap = vexp == 1000 ? 0.f : __int_as_float((15 - vexp + 127) << 23);
    if (__any_sync(~0u, smax > cap && smax < INFINITY)) {
      float v = smax < INFINITY ? smax : 0.f;
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) v = fmaxf(v, __shfl_xor_sync(~0u, v, off));
      vnew = min(vexp, max(min(13 - ((int)(__float_as_uint(v) >> 23) - 127), 100), -100));
      moved = true;
    }
    if (__any_sync(~0u, moved)) {
      const float dv = vexp == 1000 ? 1.f : vnew - vexp < -126 ? 0.f : __int_as_float((vnew - vexp + 127) << 23);
#pragma unroll
      for (int nt = 0; nt < NT; nt++) {
        const float f = m[nt] == -INFINITY ? 0.f : ex2(m[nt] - mnew[nt]);
        m[nt] = mnew[nt];
        l[nt] *= f;
        za[nt] *= f;
        const float fo = f * dv;
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
          for (int j = 0; j < 4; j++) o[i][nt][j] *= fo;
      }
      vexp = vnew;
    }
    const float vup = vexp == 1000 ? 0.f : __int_as_float((vexp + 127) << 23);
    uint32_t pb[2][NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      const float base = m[nt] == -INFINITY ? 0.f : m[nt];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float p = ex2(tsc[nt][i] - base);
        l[nt] += p;
        float w = p * (vs[i] * vup), z = p * vz[i];
        if (!whole && tsc[nt][i] == -INFINITY) w = z = 0.f;  // an unseen row's words may be NaN
        za[nt] += z;
        pb[i >> 1][nt][i & 1] = transpose8(split_f16(w));
      }
    }
    // O^T += V^T P^T: lane g has channels g VC .. g VC + VC - 1
#pragma unroll
    for (int j = 0; j < 2; j++) {
      const uint8_t* vb = buf + j * S::kTile + kv4_codes_off(D, 1) + g * (D / 16);
#pragma unroll
      for (int i = 0; i < (VC + 7) / 8; i++) {
        uint32_t r[4];
#pragma unroll
        for (int h = 0; h < 4; h++) {
          const uint8_t* row = vb + (2 * t4 + (h & 1) + 8 * (h >> 1)) * (D / 2);
          if (VC == 4)
            r[h] = *reinterpret_cast<const uint16_t*>(row);
          else
            r[h] = reinterpret_cast<const uint32_t*>(row)[i];
        }
        // channels 8 i + 4 half + n: nibble n of both positions' halves
#pragma unroll
        for (int half = 0; half < (VC >= 8 ? 2 : 1); half++) {
          const uint32_t sel = half ? 0x7632u : 0x5410u;
          const uint32_t lo = __byte_perm(r[0], r[1], sel), hi = __byte_perm(r[2], r[3], sel);
#pragma unroll
          for (int n = 0; n < 2; n++) {
            const uint32_t x0 = lo >> (8 * n), x1 = hi >> (8 * n);
            const uint32_t a0 = nibble_f16(x0, 0x000f000fu, 0x64006400u, 0x64086408u);
            const uint32_t a1 = nibble_f16(x0, 0x00f000f0u, 0x54005400u, 0x54805480u);
            const uint32_t a2 = nibble_f16(x1, 0x000f000fu, 0x64006400u, 0x64086408u);
            const uint32_t a3 = nibble_f16(x1, 0x00f000f0u, 0x54005400u, 0x54805480u);
            const int mt = 4 * i + 2 * half + n;
#pragma unroll
            for (int nt = 0; nt < NT; nt++) mma_f16(o[mt][nt], a0, a1, a2, a3, pb[j][nt][0], pb[j][nt][1]);
          }
        }
      }
    }
    __syncwarp();
    issue();
    if (++stage == STAGES) {
      stage = 0;
      phase ^= 1;
    }

    // --- end of the unit, or of this worker's share of it ---------------------
    x++;
    const bool unit_done = c.chunk + 1 == c.chunks;
    if (unit_done || x == end) {
      const int nq = req_new(a, c.b), rows = nq * a.G, r0 = c.rb * RPB;
      const int64_t first = req_start(a, c.b);
      const float down = vexp == 1000 ? 0.f : __int_as_float((127 - vexp) << 23);
      const bool mine = unit_first >= beg;  // this worker began the unit
      const bool direct = mine && unit_done;
      const int slot = 2 * worker + (mine ? 1 : 0);
#pragma unroll
      for (int nt = 0; nt < NT; nt++) {
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) {
          l[nt] += __shfl_xor_sync(~0u, l[nt], off);
          za[nt] += __shfl_xor_sync(~0u, za[nt], off);
        }
        const int r = r0 + 4 * nt + t4;
        if (r < rows) {
          const float norm = !direct ? 1.f : l[nt] == 0.f ? 0.f : 1.f / l[nt];
          float* dst;
          if (direct) {
            dst = a.out + ((first + r / a.G) * a.H + c.head * a.G + r % a.G) * D + g * VC;
          } else {
            float* base = a.part + ((int64_t)slot * RPB + 4 * nt + t4) * (D + 4);
            if (g == 0) *reinterpret_cast<float2*>(base + D) = make_float2(m[nt], l[nt]);
            dst = base + g * VC;
          }
#pragma unroll
          for (int i = 0; i < VC / 4; i++) {
            float4 f;
            f.x = (fmaf(o[2 * i][nt][0] + o[2 * i][nt][1], down, za[nt])) * norm;
            f.y = (fmaf(o[2 * i][nt][2] + o[2 * i][nt][3], down, za[nt])) * norm;
            f.z = (fmaf(o[2 * i + 1][nt][0] + o[2 * i + 1][nt][1], down, za[nt])) * norm;
            f.w = (fmaf(o[2 * i + 1][nt][2] + o[2 * i + 1][nt][3], down, za[nt])) * norm;
            reinterpret_cast<float4*>(dst)[i] = f;
          }
        }
      }
      if (mine && !unit_done && lane == 0) {
        const int last = (int)((unit_first + c.chunks - 1) / per);
        a.desc[worker] = make_int4(c.b, c.head, c.rb, last);
      }
      fresh = true;
    }
    step(c, x);
    if (fresh) unit_first = x;
  }
}

// Joins the parts of units that more than one worker took: one warp per
// (worker that began a unit, row).
template <int D, int RPB>
__global__ void __launch_bounds__(256) kv4_combine_kernel(Kv4AttnArgs a) {
  constexpr int V = D / 32;  // channels per lane
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int id = blockIdx.x * 8 + (threadIdx.x >> 5), w = id / RPB, row = id % RPB;
  if (w >= a.workers) return;
  const int4 d = a.desc[w];
  if (d.x < 0) return;
  const int rows = req_new(a, d.x) * a.G, r = d.z * RPB + row;
  if (r >= rows) return;
  auto base = [&](int i) {
    return a.part + ((int64_t)(i == w ? 2 * w + 1 : 2 * i) * RPB + row) * (D + 4);
  };
  float m = -INFINITY;
  for (int i = w + lane; i <= d.w; i += 32) m = fmaxf(m, base(i)[D]);
  m = warp_max(m);
  float l = 0.f, o[V];
#pragma unroll
  for (int j = 0; j < V; j++) o[j] = 0.f;
#pragma unroll 4
  for (int i = w; i <= d.w; i++) {
    const float* p = base(i);
    const float2 ml = *reinterpret_cast<const float2*>(p + D);
    const float f = ml.x == -INFINITY ? 0.f : ex2(ml.x - m);
    l = fmaf(ml.y, f, l);
#pragma unroll
    for (int j = 0; j < V; j++) o[j] = fmaf(p[lane + 32 * j], f, o[j]);
  }
  const float norm = l == 0.f ? 0.f : 1.f / l;
  float* dst = a.out + (((int64_t)req_start(a, d.x) + r / a.G) * a.H + d.y * a.G + r % a.G) * D;
#pragma unroll
  for (int j = 0; j < V; j++) dst[lane + 32 * j] = o[j] * norm;
}

// Warps and ring stages of a variant: as many warps as registers allow, the
// ring as deep as shared memory allows beside the request prefix.
template <int D, int NT>
struct Shape {
  static constexpr int kWarps = NT == 1 ? 16 : NT == 2 ? 12 : 8;
  static constexpr int kStages = D == 128 ? (NT == 1 ? 3 : NT == 2 ? 4 : 4) : 4;
};

template <int D, int NT>
tb_status_t launch(Kv4AttnArgs a, cudaStream_t st) {
  constexpr int W = Shape<D, NT>::kWarps, ST = Shape<D, NT>::kStages;
  using S = Smem<D, NT>;
  const size_t smem = W * (size_t)(ST * S::kStage + S::kPerWarpFixed) + 8 * (size_t)(a.B + 1);
  auto kernel = kv4_attn_kernel<D, NT, W, ST>;
  TB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  const unsigned grid = (unsigned)(a.workers / W);
  kernel<<<grid, W * 32, smem, st>>>(a);
  TB_TRY(check_launch("kv4_attn_kernel"));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((a.workers * 4 * NT + 7) / 8));
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  TB_CUDA(cudaLaunchKernelEx(&cfg, kv4_combine_kernel<D, 4 * NT>, a));
  return check_launch("kv4_combine_kernel");
}

// Query rows of a unit: one MMA column pair each, 4 to a column tile.
int row_tiles(int64_t G, int64_t max_q) { return G * max_q <= 4 ? 1 : G * max_q <= 8 ? 2 : 4; }
int warps_of(int nt) { return nt == 1 ? 16 : nt == 2 ? 12 : 8; }

size_t attn_workspace(int64_t G, int64_t max_q, int64_t D) {
  const int nt = row_tiles(G, max_q);
  const size_t workers = (size_t)sm_count() * warps_of(nt);
  return workers * sizeof(int4) + 2 * workers * 4 * nt * (size_t)(D + 4) * sizeof(float);
}

template <int D>
tb_status_t launch_nt(const Kv4AttnArgs& a, int nt, cudaStream_t st) {
  if (nt == 1) return launch<D, 1>(a, st);
  if (nt == 2) return launch<D, 2>(a, st);
  return launch<D, 4>(a, st);
}

}  // namespace
}  // namespace tb

extern "C" size_t tb_kv4_attention_workspace_size(int64_t T, int64_t H, int64_t Hkv, int64_t D, int64_t max_q) {
  if (T <= 0 || H <= 0 || Hkv <= 0 || H % Hkv != 0 || D <= 0 || max_q <= 0) return 0;
  return tb::attn_workspace(H / Hkv, max_q, D);
}

extern "C" tb_status_t tb_kv4_attention_f32(float* out, const float* q, int64_t q_stride, const uint8_t* pages,
                                            const int32_t* block_table, const int32_t* seq_lens,
                                            const int32_t* q_start, int32_t* bad_count, int64_t B, int64_t T,
                                            int64_t max_q, int64_t H, int64_t Hkv, int64_t D, int64_t block_size,
                                            int64_t max_blocks, int64_t num_blocks, float scale, void* workspace,
                                            size_t workspace_bytes, tb_stream_t stream) {
  TB_INJECT("tb_kv4_attention_f32");
  TB_REQUIRE(B >= 0 && T >= 0 && T <= INT_MAX && H > 0 && Hkv > 0 && H % Hkv == 0 && H <= 65535 && D > 0);
  TB_REQUIRE(block_size > 0 && block_size % tb::kKv4Tile == 0 && max_blocks >= 0 && max_blocks <= INT_MAX);
  TB_REQUIRE(num_blocks > 0 && num_blocks <= INT_MAX && block_size <= INT_MAX && num_blocks * block_size <= INT_MAX);
  TB_REQUIRE(max_q >= 0 && max_q <= T);
  if (D != 32 && D != 64 && D != 128) return TB_ERROR_NOT_SUPPORTED;
  if (B > tb::kMaxB || T * (H / Hkv) > INT_MAX) return TB_ERROR_NOT_SUPPORTED;
  if (T == 0) return TB_SUCCESS;
  TB_REQUIRE(max_q >= 1);
  TB_REQUIRE(out && q && q_stride >= H * D && pages && (B == 0 || (seq_lens && q_start && (max_blocks == 0 || block_table))));
  TB_REQUIRE(tb::aligned(out, 16) && tb::aligned(pages, 16));
  TB_REQUIRE(workspace && tb::aligned(workspace, 16) &&
             workspace_bytes >= tb::attn_workspace(H / Hkv, max_q, D));
  const int nt = tb::row_tiles(H / Hkv, max_q);
  tb::Kv4AttnArgs a{};
  a.out = out;
  a.q = q;
  a.pages = pages;
  a.table = block_table;
  a.lens = seq_lens;
  a.starts = q_start;
  a.workers = tb::sm_count() * tb::warps_of(nt);
  a.desc = static_cast<int4*>(workspace);
  a.part = reinterpret_cast<float*>(a.desc + a.workers);
  a.bad = bad_count;
  a.err = tb::wait_timeout_word();
  a.q_stride = q_stride;
  a.B = (int)B;
  a.T = (int)T;
  a.H = (int)H;
  a.Hkv = (int)Hkv;
  a.G = (int)(H / Hkv);
  a.block = (int)block_size;
  a.max_blocks = (int)max_blocks;
  a.num_blocks = (int)num_blocks;
  a.scale = scale;
  a.vec = tb::aligned(q, 16) && q_stride % 4 == 0;
  cudaStream_t st = (cudaStream_t)stream;
  if (D == 128) return tb::launch_nt<128>(a, nt, st);
  if (D == 64) return tb::launch_nt<64>(a, nt, st);
  return tb::launch_nt<32>(a, nt, st);
}
