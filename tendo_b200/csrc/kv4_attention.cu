// kv4_attention.cu — attention over the paged 4-bit KV cache (kv4.cuh).
//
//   out[i, h] = sum_j softmax_j(scale q_i . k_j) v_j,  j <= len - n + i
//
// for the n new tokens i of each request, whose keys are already in the cache.
//
// The codes c are integers -8 .. 7, so both products run on fp16 tensor cores
// without rounding the cache: q . k_j = s_j (q . c_j) + z_j sum q, and
// p_j v_j = (p_j s_j) c_j + p_j z_j.  The fp32
// operands q and p_j s_j are split into two fp16 terms (22 bits), which sit in
// neighbouring columns of the MMA's 8-column side; positions (or channels)
// are its 16-row side.  So 4 query rows of one kv head share every unpacked
// code, and a lane holds both terms of a score and adds them.  Units of up to 4
// rows take q as an integer of four signed bytes instead (30 bits), against the
// codes as bytes: exact sums, a third of the unpacking, half the MMAs' depth (64
// sequences of 1500 positions and 32 heads: 107 us, as fp16 terms 112; for 16
// rows a unit the digits' sums would spill, 93 against 81).
//
// The chunks of 32 positions of all units are one list, cut into equal shares
// for the CTAs (one per SM) and again for their warps: lengths may differ as they
// will.  A warp copies its chunks through a ring of its own, two ahead, and
// shares nothing until its part is summed.  What bounds it is the work on the
// codes, some 670 instructions of a warp per chunk of one row tile (860 of two):
// 64 sequences of 1500 positions, 32 heads of 128 each with a kv head: 107 us, 4.1
// TB/s or 63% of a copy's rate, issue slots 63% busy.  One of 131072 positions, 64
// heads on 8: 59 us, 2.4 TB/s.  16 of 2100: 30 us, where a warp has 5 chunks and
// start, joins and a second launch are half; with five tokens each 80 us, as
// three units of 16 rows unpack every code.
#include <limits.h>
#include <math.h>

#include <type_traits>

#include "kv4_attn.cuh"

namespace tb {
namespace {

constexpr int kChunk = 32;      // positions a warp takes at a time: two tiles

// D += A[16 x 16] . B[16 x 8], fp16 in, fp32 accumulate.
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same from zero.
__device__ __forceinline__ void mma_f16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
// D = A[16 x 32] . B[32 x 8] (+ C) of signed bytes, exact.  The first of a sum
// starts from kMagic: as long as |sum| < 2^22 the result's bits are those of
// the float 2^23 + 2^22 + sum.
constexpr int kMagic = 0x4b400000;
__device__ __forceinline__ void mma_s8_first(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint2 b) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b.x), "r"(b.y), "r"(kMagic));
}
__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint2 b) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b.x), "r"(b.y));
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
template <int N>
struct Words {
  uint32_t w[N];
};
// N words of 4 bytes (0: two bytes).
template <int N>
__device__ __forceinline__ Words<(N ? N : 1)> ld_words(const uint8_t* p) {
  Words<(N ? N : 1)> r;
  if constexpr (N == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    r.w[0] = v.x, r.w[1] = v.y, r.w[2] = v.z, r.w[3] = v.w;
  } else if constexpr (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    r.w[0] = v.x, r.w[1] = v.y;
  } else if constexpr (N == 1) {
    r.w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else {
    r.w[0] = *reinterpret_cast<const uint16_t*>(p);
  }
  return r;
}
__device__ __forceinline__ void copy16(uint32_t dst, const uint8_t* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// Where a worker stands in the flat list of chunks.
struct Cursor {
  int b, head, rb;     // request, kv head, row block
  int chunk, chunks;   // position within the unit and its length
};

// Quotients of the list by a CTA count or a unit's length, nearly always of 32
// bits.  The rest is out of line: the kernel's code has to stay small enough
// for the instruction caches.
__device__ __noinline__ int64_t quotient64(int64_t x, int64_t y) { return x / y; }
__device__ __forceinline__ int64_t quotient(int64_t x, int64_t y) {
  if (((uint64_t)x | (uint64_t)y) >> 32) return quotient64(x, y);
  return (int64_t)((uint32_t)x / (uint32_t)y);
}

// The x-th chunk of the list (pre: running sum of the requests' chunks).
__device__ __noinline__ Cursor seek_chunk(const int64_t* pre, const int32_t* nq_of, const int32_t* len_of, int B, int G,
                                          int rpb, int64_t x) {
  int lo = 0, hi = B;
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
  c.chunks = (len_of[lo] + kChunk - 1) / kChunk;
  const int64_t rel = x - pre[lo];
  const int unit = (int)quotient(rel, c.chunks);
  c.chunk = (int)(rel - (int64_t)unit * c.chunks);
  const int rbs = (nq_of[lo] * G + rpb - 1) / rpb;
  c.head = rbs == 1 ? unit : unit / rbs;
  c.rb = unit - c.head * rbs;
  return c;
}

// A segment is what one warp sums of one unit.  Those that are not whole units
// meet in the CTA when its work is done: a warp's first one, if it ends before
// the warp's share does, waits in the workspace, its last one in shared memory.
struct Segs {
  int64_t first, last;  // where the segments' units begin in the list, -1: none
  int4 unit[2];         // of them: request, kv head, row block, chunks
};

// What a warp needs only where a unit begins or ends, out of its registers.
struct Place {
  Cursor sum, load;  // units in hand on the summing and on the loading side
  int64_t beg;       // the warp's share of the list
};

template <int D, int NT>
struct Smem {
  static constexpr int kTile = kv4_tile_bytes(D);
  static constexpr int kStage = 2 * kTile;
  static constexpr int kStages = 3;
  static constexpr int kRing = kStages * kStage;
  static constexpr int kSeg = 4 * NT * (D + 4) * 4;                        // a segment's rows: sums, maximum, sum of p
  static constexpr int kQFrags = NT > 1 ? NT * 16 * D + 32 * NT : 0;  // q's rows, or fragments; sums and factors of them
  static constexpr int kPerWarp = kRing + kQFrags + 96;                    // + Segs, Place
  static_assert(kSeg <= kRing, "a segment waits in the ring");
};

template <int D, int NT, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, 1) kv4_attn_kernel(Kv4AttnArgs a) {
  constexpr int KW = D / 32;        // K words of a lane per row
  constexpr int MT = D / 16;        // 16-channel tiles of the output
  constexpr int VC = D / 8;         // channels of a lane in V rows and in the output
  constexpr int VW = D / 64;        // V words of a lane per row (0: half a word)
  constexpr int RPB = 4 * NT;       // query rows per unit
  constexpr bool kQS = NT > 1;      // q as fp16 pairs in shared memory, else as digits in registers
  using S = Smem<D, NT>;
  extern __shared__ __align__(128) uint8_t smem[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
  auto seg_of = [&](int w) { return reinterpret_cast<float*>(smem + w * S::kPerWarp); };
  auto segs_of = [&](int w) { return reinterpret_cast<Segs*>(smem + w * S::kPerWarp + S::kRing + S::kQFrags); };
  volatile Place* here = reinterpret_cast<volatile Place*>(smem + warp * S::kPerWarp + S::kRing + S::kQFrags + 48);
  static_assert(sizeof(Segs) == 48 && sizeof(Place) <= 48, "kPerWarp");
  uint32_t* qfs = reinterpret_cast<uint32_t*>(smem + warp * S::kPerWarp + S::kRing);
  int64_t* pre = reinterpret_cast<int64_t*>(smem + WARPS * S::kPerWarp);
  // the requests' first rows, rows and lengths: every warp asks for them again
  // and again, and 148 SMs asking L2 for the same line wait for one another
  int32_t* start_of = reinterpret_cast<int32_t*>(pre + a.B + 1);
  int32_t *nq_of = start_of + a.B, *len_of = nq_of + a.B;
  __shared__ int64_t wsum[WARPS];
  __shared__ volatile int64_t share[3];  // the CTA's part of the list: from, to, chunks of a CTA

  // chunks of each request over its kv heads and row blocks, as a running sum
  {
    const int per = (a.B + WARPS * 32 - 1) / (WARPS * 32);
    const int b0 = min(tid * per, a.B), b1 = min(b0 + per, a.B);
    auto chunks_of = [&](int b) {
      const int rows = nq_of[b] * a.G, len = len_of[b];
      return (int64_t)((rows + RPB - 1) / RPB) * a.Hkv * ((len + kChunk - 1) / kChunk);
    };
    int64_t mine = 0;
    for (int b = b0; b < b1; b++) {
      start_of[b] = req_start(a, b);
      nq_of[b] = req_new(a, b);
      len_of[b] = req_len(a, b);
      mine += chunks_of(b);
    }
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
  pdl_launch_dependents();
  auto get = [](const volatile Cursor& v) { return Cursor{v.b, v.head, v.rb, v.chunk, v.chunks}; };
  auto set = [](volatile Cursor& v, const Cursor& c) {  // by every lane: each reads what it wrote
    v.b = c.b, v.head = c.head, v.rb = c.rb, v.chunk = c.chunk, v.chunks = c.chunks;
  };
  const int64_t total = pre[a.B];
  int todo;  // chunks of this warp
  {
    const int64_t cta_per = max(quotient(total + gridDim.x - 1, gridDim.x), (int64_t)1);
    const int64_t cta_beg = min(blockIdx.x * cta_per, total), cta_end = min(cta_beg + cta_per, total);
    const int64_t n = cta_end - cta_beg, beg = cta_beg + quotient(n * warp, WARPS);
    here->beg = beg;
    todo = (int)(cta_beg + quotient(n * (warp + 1), WARPS) - beg);
    if (tid == 0) share[0] = cta_beg, share[1] = cta_end, share[2] = cta_per;
  }
  if (tid == 0) a.desc[blockIdx.x] = make_int4(-1, 0, 0, 0);
  if (lane == 0) segs_of(warp)->first = segs_of(warp)->last = -1;

  auto seek = [&](int64_t x) { return seek_chunk(pre, nq_of, len_of, a.B, a.G, RPB, x); };
  // the unit after c's, which begins at this warp's i-th chunk
  auto next_unit = [&](Cursor c, int i) {
    const int rbs = (nq_of[c.b] * a.G + RPB - 1) / RPB;
    c.chunk = 0;
    if (c.rb + 1 < rbs) {
      c.rb++;
    } else if (c.head + 1 < a.Hkv) {
      c.rb = 0;
      c.head++;
    } else {
      c = seek(here->beg + i);
    }
    return c;
  };

  // --- loads: a chunk's tiles kStages - 1 chunks ahead of their use, the table
  // entries of them one more --------------------------------------------------
  const int bpt = a.block / kKv4Tile;
  const uint32_t page_bytes = (uint32_t)(a.Hkv * bpt * S::kTile);
  int px = 0;  // of the chunk whose entries come next
  int col = 0, sub = 0, tiles_left = 0;  // its first tile: table column, place in the page, tiles from there on
  const int32_t* row = nullptr;
  int head0 = 0;  // the unit's tiles within a page
  int e0 = -1, e1 = -1, sub0 = 0, sub1 = 0;  // entries in flight and their tiles' places
  int asked = 0;  // how many of them were looked up: what is in the table says nothing about that
  auto place = [&](const Cursor& pc) {
    set(here->load, pc);
    const int tile = pc.chunk * 2;
    col = tile / bpt;
    sub = tile - col * bpt;
    tiles_left = (len_of[pc.b] + kKv4Tile - 1) / kKv4Tile - tile;
    row = a.table + (int64_t)pc.b * a.max_blocks;
    head0 = pc.head * bpt;
  };
  auto look = [&]() {
    asked = 0;
    if (px >= todo) return;
    const bool turn = sub + 1 == bpt;
    sub0 = head0 + sub;
    sub1 = turn ? head0 : sub0 + 1;
    e0 = row[col];
    asked = 1;
    e1 = -1;
    if (tiles_left > 1) e1 = row[col + turn], asked = 2;
    px++;
    if (tiles_left > 2) {
      tiles_left -= 2;
      col += turn;
      sub = sub1 - head0 + 1;
      if (sub == bpt) sub = 0, col++;
    } else if (px < todo) {
      place(next_unit(get(here->load), px));
    }
  };
  uint8_t* ring = smem + warp * S::kPerWarp;
  const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring) + 16 * lane;
  int there = 0;  // two bits per stage: which tiles it holds
  // Query row k of the unit in hand: its token and head within the kv head's
  // group.  u0 and h0 are those of row 0; k + h0 is small, so one product with
  // the reciprocal divides it exactly.
  const float inv_g = 1.f / a.G;
  auto token_of = [&](int u0, int h0, int k, int& h) {
    const int up = (int)((h0 + k + 0.5f) * inv_g);
    h = h0 + k - up * a.G;
    return u0 + up;
  };
  // A row's token, and its head in h0.
  auto first_token = [&](int r, int& h0) {
    int u = (int)(r * inv_g);
    while (u * a.G > r) u--;
    while (u * a.G + a.G <= r) u++;
    h0 = r - u * a.G;
    return u;
  };
  // Asks for q's rows of a unit, into the place of their fragments: 16-byte
  // pieces, those of a lane's share swizzled so that 8 lanes read 8 banks' worth.
  constexpr int PL = D / 16;  // pieces of a lane's share of a row
  auto ask_q = [&](const Cursor& c) {
    const int r0 = c.rb * RPB, rows = nq_of[c.b] * a.G;
    int h0;
    const int u0 = first_token(r0, h0);
    const uint32_t to = (uint32_t)__cvta_generic_to_shared(qfs);
#pragma unroll 1
    for (int i = lane; i < RPB * (D / 4); i += 32) {
      const int k = i / (D / 4), piece = i % (D / 4);
      if (r0 + k >= rows) break;
      int h;
      const int u = token_of(u0, h0, k, h);
      copy16(to + k * (4 * D) + ((piece ^ ((piece / PL + 4 * (k & 1)) & (PL - 1))) << 4),
             reinterpret_cast<const uint8_t*>(a.q + (start_of[c.b] + u) * a.q_stride + (c.head * a.G + h) * D + 4 * piece));
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  // Copies the tiles whose entries have come into a stage.
  auto fetch = [&](int stage) {
    const bool ok0 = (unsigned)e0 < (unsigned)a.num_blocks, ok1 = (unsigned)e1 < (unsigned)a.num_blocks;
    there = (there & ~(3 << (2 * stage))) | (ok0 + 2 * ok1) << (2 * stage);
    if (lane == 0 && a.bad && ok0 + ok1 < asked) atomicAdd(a.bad, asked - ok0 - ok1);
    if (asked) {  // a tile that is not there is hidden, and its copy is of page 0
      const uint8_t* n0 = a.pages + ((uint64_t)(ok0 ? e0 : 0) * page_bytes + (uint32_t)(sub0 * S::kTile + 16 * lane));
      const uint8_t* n1 = a.pages + ((uint64_t)(ok1 ? e1 : 0) * page_bytes + (uint32_t)(sub1 * S::kTile + 16 * lane));
      const uint32_t to = ring_at + stage * S::kStage;
#pragma unroll
      for (int i = 0; i < D / 32; i++) {
        copy16(to + 512 * i, n0 + 512 * i);
        copy16(to + S::kTile + 512 * i, n1 + 512 * i);
      }
      // the 128 bytes left of each: lanes 0 - 7 and 8 - 15
      const uint8_t* tail = (lane < 8 ? n0 : n1 - 128) + 16 * D;
      if (lane < 16) copy16(to + 16 * D + (lane < 8 ? 0 : S::kTile - 128), tail);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  const int koff = g * (D / 2) + t4 * (D / 8), voff = 8 * D + 2 * t4 * (D / 2) + g * (D / 16), woff = 16 * D + 4 * g;

  float o[MT][NT][4];
  uint2 qf[2][KW];  // (!kQS) two high digits, two low ones
  float A2[NT], m[NT];
  float2 l2[NT], za2[NT];  // in two halves
  int vis[NT];
  int vexp = 0;     // accumulators hold 2^vexp times the sums
  float kup[NT];    // 2^-(the exponent of q's row)
  float vup = 0.f, vcap = 0.f;
  int min_vis = 0;

  // Rows of the segment in hand: unnormalised sums, maximum and sum of p into
  // dst (rows of D + 4 floats), or the output itself.
  auto put = [&](const Cursor& c, float* dst, bool direct) {
    const int rows = nq_of[c.b] * a.G, r0 = c.rb * RPB;
    int h0;
    const int u0 = first_token(r0, h0);
    const int64_t first = start_of[c.b];
    const float down = vup == 0.f ? 0.f : __int_as_float((127 - vexp) << 23);
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      float l = l2[nt].x + l2[nt].y, za = za2[nt].x + za2[nt].y;
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) {
        l += __shfl_xor_sync(~0u, l, off);
        za += __shfl_xor_sync(~0u, za, off);
      }
      const int r = r0 + 4 * nt + t4;
      if (r < rows) {
        const float norm = !direct ? 1.f : l == 0.f ? 0.f : 1.f / l;
        float* to;
        if (direct) {
          int h;
          const int u = token_of(u0, h0, 4 * nt + t4, h);
          to = a.out + ((first + u) * a.H + c.head * a.G + h) * D + g * VC;
        } else {
          to = dst + (4 * nt + t4) * (D + 4);
          if (g == 0) *reinterpret_cast<float2*>(to + D) = make_float2(m[nt], l);
          to += g * VC;
        }
#pragma unroll
        for (int i = 0; i < VC / 4; i++) {
          float4 f;
          f.x = (fmaf(o[2 * i][nt][0] + o[2 * i][nt][1], down, za)) * norm;
          f.y = (fmaf(o[2 * i][nt][2] + o[2 * i][nt][3], down, za)) * norm;
          f.z = (fmaf(o[2 * i + 1][nt][0] + o[2 * i + 1][nt][1], down, za)) * norm;
          f.w = (fmaf(o[2 * i + 1][nt][2] + o[2 * i + 1][nt][3], down, za)) * norm;
          reinterpret_cast<float4*>(to)[i] = f;
        }
      }
    }
  };

  int p0 = 0, left = 0;  // the chunk's first position, and the unit's chunks from here on
  if (todo > 0) {
    const Cursor c = seek(here->beg);
    set(here->sum, c);
    if (kQS && a.vec) ask_q(c);  // before the cache's tiles: behind them it would wait for them all
    place(c);
    p0 = c.chunk * kChunk;
    left = c.chunks - c.chunk;
  }
  static_assert(S::kStages == 3, "two chunks ahead");
  int x = todo > 0 ? -3 : 0, stage = 0;
  bool fresh = true;

  // Three turns before the first chunk only look up and fetch.
#pragma unroll 1
  while (x < todo) {
    if (x >= 0) asm volatile("cp.async.wait_group %0;" ::"n"(S::kStages - 2) : "memory");
    __syncwarp();  // every lane's part of the chunk is there, and the last chunk's stage is read
    if (x > -3) fetch(stage == 0 ? S::kStages - 1 : stage - 1);
    look();
    if (x < 0) {
      x++;
      stage = x == 0 ? 0 : x + 3;  // chunk 0 goes to stage 0, chunk 1 to stage 1
      continue;
    }
    if (fresh) {
      fresh = false;
      const Cursor c = get(here->sum);
      const int nq = nq_of[c.b], len = len_of[c.b], rows = nq * a.G, r0 = c.rb * RPB;
      int h0;
      const int u0 = first_token(r0, h0);
      const int64_t first = start_of[c.b];
      // q rows, with the score's factors in them: scores come out in log2 units
      float v[D / 4];
      if (kQS && a.vec) {
        if (x > 0) {
          ask_q(c);
          asm volatile("cp.async.wait_all;" ::: "memory");
          __syncwarp();
        }  // a warp's first unit asked ahead of chunk 0, which is there
      }
      auto load = [&](int nt) {
        int h;
        if (kQS && a.vec) {
          const int k = 4 * nt + (g >> 1), turn = (t4 + 4 * (k & 1)) & (PL - 1);
          const uint8_t* from = reinterpret_cast<const uint8_t*>(qfs) + k * (4 * D) + t4 * D;
#pragma unroll
          for (int i = 0; i < PL; i++) {
            const float4 f = *reinterpret_cast<const float4*>(from + ((i ^ turn) << 4));
            const bool in = r0 + k < rows;
            v[4 * i] = in ? f.x : 0.f, v[4 * i + 1] = in ? f.y : 0.f;
            v[4 * i + 2] = in ? f.z : 0.f, v[4 * i + 3] = in ? f.w : 0.f;
          }
          return;
        }
        const int r = r0 + 4 * nt + (g >> 1), u = token_of(u0, h0, 4 * nt + (g >> 1), h);
        const float* src = a.q + (first + u) * a.q_stride + (c.head * a.G + h) * D + t4 * (D / 4);
        if (r >= rows) {
#pragma unroll
          for (int i = 0; i < D / 4; i++) v[i] = 0.f;
        } else if (a.vec) {
#pragma unroll
          for (int i = 0; i < D / 16; i++) {
            const float4 f = reinterpret_cast<const float4*>(src)[i];
            v[4 * i] = f.x, v[4 * i + 1] = f.y, v[4 * i + 2] = f.z, v[4 * i + 3] = f.w;
          }
        } else {
#pragma unroll
          for (int i = 0; i < D / 4; i++) v[i] = src[i];
        }
      };
      const float unit = a.scale * kLog2e;
      float* sums = reinterpret_cast<float*>(qfs) + S::kQFrags / 4 - 8 * NT;  // of the rows, and their factors (kQS)
      float sum = 0.f, back = 0.f;
#pragma unroll 1
      for (int nt = 0; nt < NT; nt++) {
        load(nt);
        float mx = 0.f;
        sum = 0.f;
#pragma unroll
        for (int i = 0; i < D / 4; i++) {
          mx = fmaxf(mx, fabsf(v[i]));
          sum += v[i];
        }
#pragma unroll
        for (int off = 1; off < 4; off <<= 1) {
          sum += __shfl_xor_sync(~0u, sum, off);
          mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, off));
        }
        sum *= unit;
        mx *= fabsf(unit);
        // a power of two that brings the row's largest element to 2^13 .. 2^14
        // as fp16 pairs, to 2^29 .. 2^30 as integers; a row with an infinity or
        // a NaN (its sum has it) has no scores
        constexpr int kTop = kQS ? 13 : 29;
        int e = mx > 0.f ? kTop - ((int)(__float_as_uint(mx) >> 23) - 127) : 0;
        e = max(min(e, 100), -120 + kTop / 2);
        const float up = __int_as_float((e + 127) << 23);
        back = mx < INFINITY ? __int_as_float((127 - (kQS ? 0 : 4) - e) << 23) : NAN;  // codes times 16 meet the integers
        if constexpr (kQS) {
          if ((lane & 7) == 0) sums[4 * nt + (g >> 1)] = sum, sums[4 * (NT + nt) + (g >> 1)] = back;
          __syncwarp();  // the pairs take the place of rows that are read
          // column g of the tile is term g & 1 of row g / 2
#pragma unroll
          for (int i = 0; i < D / 32; i++)
#pragma unroll
            for (int s = 0; s < 2; s++) {
              const float* w = v + 8 * i + 2 * s;
              float h[4] = {w[0], w[4], w[1], w[5]};
#pragma unroll
              for (int j = 0; j < 4; j++) {
                const float x = h[j] * unit * up, hi = __uint_as_float(__float_as_uint(x) & 0xffffe000u);
                h[j] = (g & 1) ? x - hi : hi;
              }
              reinterpret_cast<uint2*>(qfs)[(nt * (D / 16) + 2 * i + s) * 32 + lane] =
                  make_uint2(pack_f16(h[0], h[1]), pack_f16(h[2], h[3]));
            }
        } else {
          // columns 2 r and 2 r + 1 are digits of row r
#pragma unroll
          for (int i = 0; i < KW; i++) {
            uint32_t z[8];  // its bytes are the signed digits
#pragma unroll
            for (int j = 0; j < 8; j++)
              z[j] = ((uint32_t)__float2int_rn(v[8 * i + j] * unit * up) + 0x80808080u) ^ 0x80808080u;
            // digit n of channels j, j + 2, j + 4, j + 6 of the lane's word i
            auto digits = [&](int n, int j) {
              const uint32_t sel = n + 16 * (n + 4);
              return __byte_perm(__byte_perm(z[j], z[j + 2], sel), __byte_perm(z[j + 4], z[j + 6], sel), 0x5410);
            };
#pragma unroll
            for (int k = 0; k < 2; k++) {
              const int n = 3 - 2 * k - (g & 1);
              qf[k][i] = make_uint2(digits(n, 0), digits(n, 1));
            }
          }
        }
      }
      if (kQS) __syncwarp();
#pragma unroll
      for (int nt = 0; nt < NT; nt++) {  // a lane's scores are of row 4 nt + t4: columns 2 t4 and 2 t4 + 1
        A2[nt] = kQS ? sums[4 * nt + t4] : __shfl_sync(~0u, sum, 8 * t4);
        kup[nt] = kQS ? sums[4 * (NT + nt) + t4] : __shfl_sync(~0u, back, 8 * t4);
        const int r = r0 + 4 * nt + t4;
        int h;
        vis[nt] = r < rows ? len - nq + token_of(u0, h0, 4 * nt + t4, h) + 1 : 0;
        m[nt] = kNoMax;
        l2[nt] = za2[nt] = make_float2(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
          for (int j = 0; j < 4; j++) o[i][nt][j] = 0.f;
      }
      min_vis = len - nq + u0 + 1;  // the unit's first row sees least
      vexp = 127, vup = vcap = 0.f;  // no scale chosen yet
      if (kQS) __syncwarp();
    }

    const uint8_t* buf = ring + stage * S::kStage;
    const int tiles = there >> (2 * stage) & 3;
    if (++stage == S::kStages) stage = 0;

    // scores: two tiles of 16 positions x 4 NT rows (two columns a row)
    float2 s[2][NT];  // of a lane's positions 16 j + g and + 8
    {
      Words<KW> k[2][2];
#pragma unroll
      for (int j = 0; j < 2; j++)
#pragma unroll
        for (int h = 0; h < 2; h++) k[j][h] = ld_words<KW>(buf + j * S::kTile + h * 4 * D + koff);
      if constexpr (kQS) {
        float d[2][NT][4];
#pragma unroll
        for (int i = 0; i < KW; i++)
#pragma unroll
          for (int h = 0; h < 2; h++) {
            uint32_t b[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
              const uint2 v = reinterpret_cast<const uint2*>(qfs)[(nt * (D / 16) + 2 * i + h) * 32 + lane];
              b[nt][0] = v.x, b[nt][1] = v.y;
            }
#pragma unroll
            for (int j = 0; j < 2; j++) {
              const uint32_t wa = k[j][0].w[i] >> (8 * h), wb = k[j][1].w[i] >> (8 * h);
              const uint32_t a0 = nibble_f16(wa, 0x000f000fu, 0x64006400u, 0x64086408u);
              const uint32_t a1 = nibble_f16(wb, 0x000f000fu, 0x64006400u, 0x64086408u);
              const uint32_t a2 = nibble_f16(wa, 0x00f000f0u, 0x54005400u, 0x54805480u);
              const uint32_t a3 = nibble_f16(wb, 0x00f000f0u, 0x54005400u, 0x54805480u);
#pragma unroll
              for (int nt = 0; nt < NT; nt++) {
                if (i + h == 0)
                  mma_f16_first(d[j][nt], a0, a1, a2, a3, b[nt][0], b[nt][1]);
                else
                  mma_f16(d[j][nt], a0, a1, a2, a3, b[nt][0], b[nt][1]);
              }
            }
          }
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
          for (int nt = 0; nt < NT; nt++)
            s[j][nt] = mul2(make_float2(d[j][nt][0] + d[j][nt][1], d[j][nt][2] + d[j][nt][3]),
                            make_float2(kup[nt], kup[nt]));
      } else {
        int d[2][2][4];
#pragma unroll
        for (int i = 0; i < KW; i++) {
#pragma unroll
          for (int j = 0; j < 2; j++) {
            // stored codes are c + 8: with the top bit turned over, 16 c as a byte
            const uint32_t a0 = ((k[j][0].w[i] << 4) & 0xf0f0f0f0u) ^ 0x80808080u;
            const uint32_t a1 = ((k[j][1].w[i] << 4) & 0xf0f0f0f0u) ^ 0x80808080u;
            const uint32_t a2 = (k[j][0].w[i] & 0xf0f0f0f0u) ^ 0x80808080u;
            const uint32_t a3 = (k[j][1].w[i] & 0xf0f0f0f0u) ^ 0x80808080u;
#pragma unroll
            for (int n = 0; n < 2; n++) {
              if (i == 0)
                mma_s8_first(d[j][n], a0, a1, a2, a3, qf[n][i]);
              else
                mma_s8(d[j][n], a0, a1, a2, a3, qf[n][i]);
            }
          }
        }
        // each digit's sum is exact as a float, being at most 2^21
        const float2 off = make_float2(-12582912.f, -12582912.f), by = make_float2(256.f, 256.f);
#pragma unroll
        for (int j = 0; j < 2; j++) {
          auto digit = [&](int k, int c) {
            return add2(make_float2(__int_as_float(d[j][k][c]), __int_as_float(d[j][k][c + 2])), off);
          };
          const float2 high = fma2(digit(0, 0), by, digit(0, 1)), low = fma2(digit(1, 0), by, digit(1, 1));
          s[j][0] = mul2(fma2(high, make_float2(65536.f, 65536.f), low), make_float2(kup[0], kup[0]));
        }
      }
    }
    // this lane's positions: p0 + 16 j + g (+ 8)
    float ks[4], kz[4], vs[4], vz[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const uint8_t* w = buf + (i >> 1) * S::kTile + 32 * (i & 1) + woff;
      const uint32_t kw = ld_words<1>(w).w[0], vw = ld_words<1>(w + 64).w[0];
      ks[i] = kv4_scale(kw);
      kz[i] = kv4_zero(kw);
      vs[i] = kv4_scale(vw);
      vz[i] = kv4_zero(vw);
    }
    const bool edge = tiles != 3 || p0 + kChunk > min_vis;  // some row does not see all of the chunk
    auto hidden = [&](int nt, int i) {
      const int p = p0 + 16 * (i >> 1) + g + 8 * (i & 1);
      return p >= vis[nt] || !(tiles >> (i >> 1) & 1);
    };
    // scores less the row's maximum so far
    float t[NT][4], top = -INFINITY, smax = 0.f;
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        const float2 y = fma2(make_float2(ks[i], ks[i + 1]), s[i >> 1][nt],
                              fma2(make_float2(kz[i], kz[i + 1]), make_float2(A2[nt], A2[nt]),
                                   make_float2(-m[nt], -m[nt])));
        t[nt][i] = y.x, t[nt][i + 1] = y.y;
      }
    if (edge) {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        bool seen = false;
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
          if (hidden(nt, i))
            t[nt][i] = -INFINITY;
          else
            seen = true;
        }
        if (!seen) vs[i] = vz[i] = 0.f;  // a position that no row of this lane sees may hold anything
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
      for (int i = 0; i < 4; i++) top = fmaxf(top, t[nt][i]);
#pragma unroll
    for (int i = 0; i < 4; i++) smax = fmaxf(smax, vs[i]);
    // The reference maximum moves only when a score passes it by 2^8, and V's
    // scale when 2^vexp s passes 2^7: p s 2^vexp stays below 2^15 either way,
    // and fp16 reaches 40 binades below that.
    if (__any_sync(~0u, top > 8.f || smax > vcap)) {
      float v = smax < INFINITY ? smax : 0.f;
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) v = fmaxf(v, __shfl_xor_sync(~0u, v, off));
      float dv = 1.f;
      if (v > vcap) {
        const int vnew = max(min(6 - ((int)(__float_as_uint(v) >> 23) - 127), 100), -100);
        dv = vup == 0.f || vnew - vexp < -126 ? 0.f : __int_as_float((min(vnew - vexp, 0) + 127) << 23);
        vexp = vnew;
        vup = __int_as_float((vexp + 127) << 23);
        vcap = __int_as_float((7 - vexp + 127) << 23);
      }
#pragma unroll
      for (int nt = 0; nt < NT; nt++) {
        float raw[4];
        v = m[nt];
#pragma unroll
        for (int i = 0; i < 4; i++) {
          raw[i] = fmaf(ks[i], i & 1 ? s[i >> 1][nt].y : s[i >> 1][nt].x, kz[i] * A2[nt]);
          if (t[nt][i] != -INFINITY) v = fmaxf(v, raw[i]);
        }
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) v = fmaxf(v, __shfl_xor_sync(~0u, v, off));
        const float f = ex2(m[nt] - v);
        m[nt] = v;
        l2[nt] = mul2(l2[nt], make_float2(f, f));
        za2[nt] = mul2(za2[nt], make_float2(f, f));
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
          for (int j = 0; j < 4; j += 2) {
            const float2 y = mul2(make_float2(o[i][nt][j], o[i][nt][j + 1]), make_float2(f * dv, f * dv));
            o[i][nt][j] = y.x, o[i][nt][j + 1] = y.y;
          }
#pragma unroll
        for (int i = 0; i < 4; i++)
          if (t[nt][i] != -INFINITY) t[nt][i] = raw[i] - v;
      }
    }
    uint32_t pb[2][NT][2];
#pragma unroll
    for (int i = 0; i < 4; i++) vs[i] *= vup;
    auto weigh = [&](auto edge_c) {
#pragma unroll
      for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
          const float2 p = make_float2(ex2(t[nt][i]), ex2(t[nt][i + 1]));
          l2[nt] = add2(l2[nt], p);
          float2 w = mul2(p, make_float2(vs[i], vs[i + 1])), z = make_float2(vz[i], vz[i + 1]);
          // a position that others see but this row does not may be NaN
          if (decltype(edge_c)::value && t[nt][i] == -INFINITY) w.x = z.x = 0.f;
          if (decltype(edge_c)::value && t[nt][i + 1] == -INFINITY) w.y = z.y = 0.f;
          za2[nt] = fma2(p, z, za2[nt]);
          pb[i >> 1][nt][0] = transpose8(split_f16(w.x));
          pb[i >> 1][nt][1] = transpose8(split_f16(w.y));
        }
    };
    if (edge)
      weigh(std::true_type{});
    else
      weigh(std::false_type{});

    // O^T += V^T P^T: lane g has channels g VC .. g VC + VC - 1
#pragma unroll
    for (int i = 0; i < (VC + 7) / 8; i++) {
      uint32_t r[2][4];  // V rows 2 t4, + 1, + 8, + 9
#pragma unroll
      for (int j = 0; j < 2; j++)
#pragma unroll
        for (int h = 0; h < 4; h++)
          r[j][h] = ld_words<VW ? 1 : 0>(buf + j * S::kTile + voff + 4 * i + ((h & 1) + 8 * (h >> 1)) * (D / 2)).w[0];
      // channels 8 i + 4 half + n: nibble n of both positions' halves
#pragma unroll
      for (int half = 0; half < (VC >= 8 ? 2 : 1); half++) {
        const uint32_t sel = half ? 0x7632u : 0x5410u;
#pragma unroll
        for (int n = 0; n < 2; n++) {
          const int mt = 4 * i + 2 * half + n;
          // The chunk's sums start from zero: over many chunks the MMA's
          // truncating accumulation would lose bits that these additions keep.
          float d[NT][4];
#pragma unroll
          for (int j = 0; j < 2; j++) {
            const uint32_t x0 = __byte_perm(r[j][0], r[j][1], sel) >> (8 * n);
            const uint32_t x1 = __byte_perm(r[j][2], r[j][3], sel) >> (8 * n);
            const uint32_t a0 = nibble_f16(x0, 0x000f000fu, 0x64006400u, 0x64086408u);
            const uint32_t a1 = nibble_f16(x0, 0x00f000f0u, 0x54005400u, 0x54805480u);
            const uint32_t a2 = nibble_f16(x1, 0x000f000fu, 0x64006400u, 0x64086408u);
            const uint32_t a3 = nibble_f16(x1, 0x00f000f0u, 0x54005400u, 0x54805480u);
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
              if (j == 0)
                mma_f16_first(d[nt], a0, a1, a2, a3, pb[j][nt][0], pb[j][nt][1]);
              else
                mma_f16(d[nt], a0, a1, a2, a3, pb[j][nt][0], pb[j][nt][1]);
            }
          }
#pragma unroll
          for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int k = 0; k < 4; k += 2) {
              const float2 y = add2(make_float2(o[mt][nt][k], o[mt][nt][k + 1]), make_float2(d[nt][k], d[nt][k + 1]));
              o[mt][nt][k] = y.x, o[mt][nt][k + 1] = y.y;
            }
        }
      }
    }

    // --- end of the unit, or of this worker's share of it ---------------------
    x++;
    left--;
    p0 += kChunk;
    if (left == 0 || x == todo) {
      const Cursor c = get(here->sum);
      const int64_t at = here->beg + x - (c.chunks - left);  // where the unit begins
      const bool direct = left == 0 && c.chunks - left <= x, last = x == todo;
      if (last) {
        asm volatile("cp.async.wait_all;" ::: "memory");  // the last groups are empty
        __syncwarp();
      }
      put(c,
          last ? seg_of(warp) : a.part + (int64_t)(2 * gridDim.x + blockIdx.x * WARPS + warp) * RPB * (D + 4), direct);
      if (!direct && lane == 0) {
        (last ? segs_of(warp)->last : segs_of(warp)->first) = at;
        segs_of(warp)->unit[last] = make_int4(c.b, c.head, c.rb, c.chunks);
      }
      fresh = true;
      if (x < todo) {
        const Cursor n = next_unit(c, x);
        set(here->sum, n);
        p0 = 0;
        left = n.chunks;
      }
    }
  }

  // --- the CTA's open segments ----------------------------------------------
  // In list order they are warp 0's first and last, warp 1's, and so on; those
  // of one unit are neighbours.  A chain of them is a whole unit, or a part
  // for kv4_combine_kernel if the unit reaches into another CTA.
  __syncthreads();
  const int64_t cta_beg = share[0], cta_end = share[1], cta_per = share[2];
  static_assert(2 * WARPS <= 32, "a lane per segment");
  const int64_t my_unit = lane >= 2 * WARPS ? -1 : lane & 1 ? segs_of(lane >> 1)->last : segs_of(lane >> 1)->first;
  const float* my_data = lane >= 2 * WARPS ? nullptr
                         : lane & 1  ? seg_of(lane >> 1)
                                  : a.part + (int64_t)(2 * gridDim.x + blockIdx.x * WARPS + (lane >> 1)) * RPB * (D + 4);
  const unsigned same = __match_any_sync(~0u, my_unit);
  unsigned chains = __ballot_sync(~0u, my_unit >= 0 && lane == __ffs(same) - 1);  // by first segment
  int item = 0;
#pragma unroll 1
  while (chains) {
    const int lead = __ffs(chains) - 1;
    chains &= chains - 1;
    const unsigned mine = __shfl_sync(~0u, same, lead);
    const int64_t unit = __shfl_sync(~0u, my_unit, lead);
    const int4 c = segs_of(lead >> 1)->unit[lead & 1];  // request, kv head, row block, chunks
    const bool begins = unit >= cta_beg, ends = unit + c.w <= cta_end;
    const int r0 = c.z * RPB, rows = min(nq_of[c.x] * a.G - r0, RPB);
    int h0;
    const int u0 = first_token(r0, h0);
    // rows in turn to the warps, from one chain to the next
    int r = warp - item;
    if (r < 0) r += WARPS;
    item = (item + rows) % WARPS;
#pragma unroll 1
    for (; r < rows; r += WARPS) {
      constexpr int V = D / 32;
      const bool in = mine >> lane & 1;
      const float2 ml = in ? *reinterpret_cast<const float2*>(my_data + r * (D + 4) + D) : make_float2(kNoMax, 0.f);
      const float mx = warp_max(ml.x), f = ex2(ml.x - mx), sum = warp_sum(ml.y * f);
      float v[V];
#pragma unroll
      for (int k = 0; k < V; k++) v[k] = 0.f;
#pragma unroll 4
      for (unsigned left = mine; left; left &= left - 1) {
        const int n = __ffs(left) - 1;
        const float* from = reinterpret_cast<const float*>(__shfl_sync(~0u, (uint64_t)my_data, n)) + r * (D + 4);
        const float fn = __shfl_sync(~0u, f, n);
#pragma unroll
        for (int k = 0; k < V; k++) v[k] = fmaf(from[lane + 32 * k], fn, v[k]);
      }
      if (begins && ends) {
        const float norm = sum == 0.f ? 0.f : 1.f / sum;
        int h;
        const int u = token_of(u0, h0, r, h);
        float* to = a.out + (((int64_t)start_of[c.x] + u) * a.H + c.y * a.G + h) * D;
#pragma unroll
        for (int k = 0; k < V; k++) to[lane + 32 * k] = v[k] * norm;
      } else {
        float* to = a.part + ((int64_t)(2 * blockIdx.x + begins) * RPB + r) * (D + 4);
#pragma unroll
        for (int k = 0; k < V; k++) to[lane + 32 * k] = v[k];
        if (lane == 0) to[D] = mx, to[D + 1] = sum;
      }
    }
    if (tid == 0 && begins && !ends)
      a.desc[blockIdx.x] = make_int4(c.x, c.y, c.z, (int)quotient(unit + c.w - 1, cta_per));
  }
  // rows of no request, and of requests without a key, are zero
  if (a.fill) zero_rows_of_none(a, D);
  for (int b = blockIdx.x; b < a.B; b += gridDim.x)
    if (pre[b] == pre[b + 1]) {
      const int64_t m = (int64_t)nq_of[b] * a.H * D;
      for (int64_t i = tid; i < m; i += WARPS * 32) a.out[(int64_t)start_of[b] * a.H * D + i] = 0.f;
    }
}

// Joins the parts of units that more than one CTA took: a block per (CTA that
// began a unit, row), its warps over the parts.  Nothing but latency, 2 to 3 us;
// it is launched early and waits on the device.
template <int D, int RPB>
__global__ void __launch_bounds__(128) kv4_combine_kernel(Kv4AttnArgs a) {
  constexpr int V = D / 32;  // channels per lane
  __shared__ float sm[4][D + 2];
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int first = blockIdx.x / RPB, row = blockIdx.x % RPB;
  const int4 d = a.desc[first];
  if (d.x < 0) return;
  const int r = d.z * RPB + row;
  if (r >= req_new(a, d.x) * a.G) return;
  float m = -1e30f, l = 0.f, o[V];
#pragma unroll
  for (int j = 0; j < V; j++) o[j] = 0.f;
#pragma unroll 4
  for (int i = first + warp; i <= d.w; i += 4) {
    const float* p = a.part + ((int64_t)(2 * i + (i == first)) * RPB + row) * (D + 4);
    const float m1 = p[D], l1 = p[D + 1], mn = fmaxf(m, m1);
    const float f0 = ex2(m - mn), f1 = ex2(m1 - mn);
    m = mn;
    l = l * f0 + l1 * f1;
#pragma unroll
    for (int j = 0; j < V; j++) o[j] = o[j] * f0 + p[lane + 32 * j] * f1;
  }
#pragma unroll
  for (int j = 0; j < V; j++) sm[warp][lane + 32 * j] = o[j];
  if (lane == 0) sm[warp][D] = m, sm[warp][D + 1] = l;
  __syncthreads();
  const float mx = fmaxf(fmaxf(sm[0][D], sm[1][D]), fmaxf(sm[2][D], sm[3][D]));
  float f[4], sum = 0.f;
#pragma unroll
  for (int w = 0; w < 4; w++) {
    f[w] = ex2(sm[w][D] - mx);
    sum = fmaf(sm[w][D + 1], f[w], sum);
  }
  const float norm = sum == 0.f ? 0.f : 1.f / sum;
  float* dst = a.out + (((int64_t)req_start(a, d.x) + r / a.G) * a.H + d.y * a.G + r % a.G) * D;
  for (int k = threadIdx.x; k < D; k += 128)
    dst[k] = (sm[0][k] * f[0] + sm[1][k] * f[1] + sm[2][k] * f[2] + sm[3][k] * f[3]) * norm;
}

// Warps of a CTA, one CTA per SM: as many as their registers allow (128, 168 and
// 255 a thread).
constexpr int warps_of(int nt) { return nt == 1 ? 16 : nt == 2 ? 12 : 8; }

template <int D, int NT>
tb_status_t launch(Kv4AttnArgs a, cudaStream_t st) {
  constexpr int W = warps_of(NT);
  const size_t smem = W * (size_t)Smem<D, NT>::kPerWarp + 8 * (size_t)(a.B + 1) + 12 * (size_t)a.B;
  auto kernel = kv4_attn_kernel<D, NT, W>;
  static std::atomic<uint64_t> ready{0};  // devices on which the kernel may have its shared memory
  TB_TRY(allow_smem(reinterpret_cast<const void*>(kernel),
                    W * (size_t)Smem<D, NT>::kPerWarp + 8 * (kKv4MaxB + 1) + 12 * (size_t)kKv4MaxB, ready));
  const unsigned grid = (unsigned)sm_count();
  kernel<<<grid, W * 32, smem, st>>>(a);
  TB_TRY(check_launch("kv4_attn_kernel"));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid * 4 * NT);
  cfg.blockDim = dim3(128);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  TB_CUDA(cudaLaunchKernelEx(&cfg, kv4_combine_kernel<D, 4 * NT>, a));
  return check_launch("kv4_combine_kernel");
}

// Query rows of a unit: one MMA column pair each, 4 to a column tile.  The least
// that holds the longest request's: 64 sequences with 1 row take 107, 145 and 229 us
// with 1, 2 and 4 tiles; 16 with 8 rows 30 and 38 us with 2 and 4.  The other requests
// of a call run in the same tiles: 63 single tokens beside one chunk of 500 take 298
// us together, 108 and 65 by themselves.
int row_tiles(int64_t G, int64_t max_q) { return G * max_q <= 4 ? 1 : G * max_q <= 8 ? 2 : 4; }
size_t few_workspace(int64_t G, int64_t max_q, int64_t D) {
  const int nt = row_tiles(G, max_q);
  const size_t ctas = (size_t)sm_count();
  return ctas * sizeof(int4) + ctas * (2 + warps_of(nt)) * 4 * nt * (size_t)(D + 4) * sizeof(float);
}
// More query rows per kv head than this kernel is made for.
bool many_rows(int64_t G, int64_t max_q) { return G * max_q > kKv4FewRows && G <= 128; }

size_t attn_workspace(int64_t G, int64_t max_q, int64_t D) {
  return few_workspace(G, max_q, D) + (many_rows(G, max_q) ? kv4_prefill_workspace(G, max_q, D) : 0);
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
  const int64_t page = Hkv * (block_size / tb::kKv4Tile) * tb::kv4_tile_bytes((int)D);
  if (page > INT_MAX) return TB_ERROR_NOT_SUPPORTED;
  if (B > tb::kKv4MaxB || T * (H / Hkv) > INT_MAX) return TB_ERROR_NOT_SUPPORTED;
  if (T == 0) return TB_SUCCESS;
  TB_REQUIRE(max_q >= 1);
  TB_REQUIRE(out && q && q_stride >= H * D && pages);
  TB_REQUIRE(B == 0 || (seq_lens && q_start && (max_blocks == 0 || block_table)));
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
  a.desc = static_cast<int4*>(workspace);
  a.part = reinterpret_cast<float*>(a.desc + tb::sm_count());
  a.bad = bad_count;
  a.q_stride = q_stride;
  a.B = (int)B;
  a.T = (int)T;
  a.H = (int)H;
  a.Hkv = (int)Hkv;
  a.G = (int)(H / Hkv);
  a.block = (int)block_size;
  const int bpt = (int)block_size / tb::kKv4Tile;
  a.bpt_shift = -1;
  for (int i = 0; i < 31; i++)
    if (bpt == 1 << i) a.bpt_shift = i;
  a.max_blocks = (int)max_blocks;
  a.num_blocks = (int)num_blocks;
  a.scale = scale;
  a.vec = tb::aligned(q, 16) && q_stride % 4 == 0;
  cudaStream_t st = (cudaStream_t)stream;
  a.min_rows = 1;
  a.max_rows = INT_MAX;
  a.fill = true;
  if (tb::many_rows(a.G, max_q)) {
    // where every request has max_q rows no one is left for this file's kernel
    const bool all = T == B * max_q;
    tb::Kv4AttnArgs more = a;
    if (!all) more.min_rows = tb::kKv4FewRows + 1;
    TB_TRY(tb::kv4_prefill(more, max_q, (int)D, static_cast<uint8_t*>(workspace) + tb::few_workspace(a.G, max_q, D),
                           st));
    if (all) return TB_SUCCESS;
    a.max_rows = tb::kKv4FewRows;
    a.fill = false;
  }
  if (D == 128) return tb::launch_nt<128>(a, nt, st);
  if (D == 64) return tb::launch_nt<64>(a, nt, st);
  return tb::launch_nt<32>(a, nt, st);
}
