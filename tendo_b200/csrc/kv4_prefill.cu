// kv4_prefill.cu — attention over the paged 4-bit cache for prompt chunks and
// drafted tokens: more than a few query rows per kv head (kv4_attention.cu has
// the rest).
//
// A unit is up to 256 query rows (tokens times the group) of one request and
// kv head, as two halves of 128, the rows of a tcgen05.mma; a tile is 64
// positions.  For each half and tile
//   S = [Q_hi Q_lo] [C_k; C_k]^T     Q as two fp16 terms in shared memory, the
//                                    K codes as fp16 (exact), S in TMEM;
//   softmax in registers, one thread per row, scales and zeros applied there;
//   O = [P_hi P_lo] [C_v; C_v]       p times V's scale as two fp16 terms in
//                                    TMEM over S, the V codes as fp16.
// Each tile's O starts from zero in TMEM and is added to fp32 registers: a
// chain of MMAs over a whole context would lose bits in their truncating
// accumulation.  One CTA of 16 warps per SM: 4 softmax warps for each half
// (192 registers), one warp that issues the MMAs, one that looks tiles up and
// reads their scales and zeros, three that unpack K and three that unpack V.
// The halves share the unpacked tiles, and one's softmax runs beside the
// other's MMAs.  The list of (unit, tile) pairs is cut into equal runs, one per
// CTA; units that more than one CTA took are joined by a second kernel.
//
// Two CTAs of 128 rows per SM took 662 us for what one of 256 took 581 for: the
// codes are unpacked once for all rows.  Now 4 requests with 523 to 923 new
// tokens behind 1169 to 1783 others, 64 heads on 8 of 128: 489 us, 329 TFLOP/s (the
// two terms make the MMAs' own rate twice that), 5 times the time that the
// products alone would need.  A tile takes a half 5300 cycles, of which its
// MMAs are 1750: the softmax's 700 instructions a warp take 3300, since the
// row's 128 sums leave 64 registers to work in and little can be in flight, and
// adding a tile's O another 550.  A unit's begin and end take 20000 cycles per
// 28 tiles.  Units of 128 rows or fewer go to both halves, which take turns at the
// tiles and add their sums up at the end (4 requests of 8000 positions with 16 new
// tokens: 110 us with one half at work, 91 with both; 16 of 2100: 120 and 106).
#include <limits.h>
#include <math.h>
#include <stdlib.h>

#include <type_traits>

#include "kv4_attn.cuh"
#include "tc_common.cuh"

namespace tb {
namespace {

constexpr int kPos = 64;       // positions per tile
constexpr int kRows = 128;     // rows of the MMA
constexpr int kThreads = 512;
constexpr int kExpired = -2;   // Kv4AttnArgs::desc[..].x of a CTA of which a wait ran out (-1: no unit to join)
constexpr int kSmRegs = 192, kUnRegs = 64;
static_assert((2 * kSmRegs + 2 * kUnRegs) * 128 == kThreads * 128, "register shares add up to the launch's");

struct Unit {
  int b, head, rb;
  int tile, tiles;  // first tile of this CTA's part, tiles of the unit
};

// Barriers, the CTA's scalars.
struct Ctl {
  // Barriers in a ring of two or eight tiles: an entry's next phase cannot end
  // before every waiter has seen this one.  (A tile's K may be replaced when
  // its scores are done, but a softmax may then still be two tiles of its half
  // behind, four where the halves take turns, and V's loads too: those waits
  // have the longer ring.)
  uint64_t u_full, q_ready[2], at_full[8], par_full[8], k_full[2], v_full[2], k_free[2], v_free[2];
  uint64_t qk_done[2][2], p_ready[2][2], pv_done[2], o_free[2];
  uint64_t given[2];  // where the halves took turns: the second's sums are there, and are read
  uint64_t drained;   // every product and arrival that the issuing thread asked for has happened
  uint32_t tmem;
  int dead;  // a wait ran out: no one waits any more, and no unit is begun
  float kup;  // 2^-(q's exponent)
  int64_t at[8][4];  // where a tile's four parts of 16 positions lie, -1: nowhere
  Unit unit[4];      // the CTA's units in turn, found by the issuing warp
  float4 head[8];    // per tile: V's scale, its inverse, absent parts, unused
};

template <int D>
struct Lay {
  // 128-byte columns of a row.  Of 32 channels half of one is used: the scores
  // take no more steps, and what V's other half holds ends in columns of O
  // that no one reads.
  static constexpr int kAtoms = D < 64 ? 1 : D / 64;
  static constexpr int kQ = kAtoms * kRows * 128;   // one term of a half's Q
  static constexpr int kKv = kAtoms * kPos * 128;   // a tile's K or V as fp16
  static constexpr int kK = 4 * kQ, kV = kK + 2 * kKv, kPar = kV + 2 * kKv, kCtl = kPar + 8 * 4 * kPos * 4;
  static constexpr int kPre = kCtl + 1024;
  static constexpr int kTileBytes = kv4_tile_bytes(D);
  static_assert(sizeof(Ctl) <= 1024, "Ctl");
};

__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
__device__ __forceinline__ float top11(float x) { return __uint_as_float(__float_as_uint(x) & 0xffffe000u); }

// 32 aligned bytes in one load: in two, whole sectors would be asked for twice.
__device__ __forceinline__ void ld32(const float* p, float (&v)[8]) {
  asm volatile("ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
               : "l"(p));
}

// D[tmem] (+)= A . B^T, one K = 16 step of fp16: A in shared memory or in TMEM.
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(
          d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// True in one lane of a converged warp.  With a branch on elect.sync the
// compiler keeps the MMAs' operands in uniform registers; behind a branch on
// the lane number it moves them there one MMA at a time (95 cycles each).
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(p));
  return p != 0;
}
// Instruction descriptor: fp16 operands, fp32 accumulator, M 128; b_mn: B's
// rows along N (its N index contiguous in shared memory).
constexpr uint32_t idesc_f16(int N, bool b_mn) {
  return (1u << 4) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
}
// Descriptor of an operand whose MN index is contiguous, 128-byte swizzle:
// blocks of 64 elements `lbo` bytes apart, groups of 8 K rows 1024 apart.
__device__ __forceinline__ uint64_t sw128_mn_desc(uint32_t saddr, int lbo) {
  return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)(lbo >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// CTAs of which a wait ran out since tb_kv4_attention_status last asked.
__device__ int g_expired;

__device__ __noinline__ void expire(Ctl* ctl) {
  if (atomicExch(&ctl->dead, 1) == 0) atomicAdd(&g_expired, 1);
}
// Waits for a phase of a barrier; false if that ran out.  Every wait is bounded
// (a poll of a barrier that does not move takes 1.5 us, 2^22 of them 6 s) and
// ends at once where another of the CTA has run out: the roles then go on with
// whatever lies in their buffers, inside their bounds, to the end of the unit in
// hand, begin no other, and the call's output is NaN.
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t phase, Ctl* ctl, uint32_t polls) {
  const uint32_t at = smem_addr(bar);
  for (uint32_t it = 0; it < polls; it++) {
    uint32_t done;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
        : "=r"(done)
        : "r"(at), "r"(phase & 1)
        : "memory");
    if (done) return true;
    if (*reinterpret_cast<volatile int*>(&ctl->dead)) return false;
  }
  expire(ctl);
  return false;
}

__device__ __forceinline__ bool ready(uint64_t* bar, uint32_t phase) {
  uint32_t done;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
      : "=r"(done)
      : "r"(smem_addr(bar)), "r"(phase & 1)
      : "memory");
  return done;
}

// A unit holds whole tokens: tpb of them, all of a kv head's group.
__device__ __forceinline__ int req_units(const Kv4AttnArgs& a, int nq) { return (nq + a.tpb - 1) / a.tpb; }
// Positions of the request that the unit's last row sees.
__device__ __forceinline__ int unit_vis(const Kv4AttnArgs& a, int nq, int len, int rb) {
  return max(len - nq + min((rb + 1) * a.tpb, nq), 0);
}
__device__ __forceinline__ int unit_tiles(const Kv4AttnArgs& a, int nq, int len, int rb) {
  return (unit_vis(a, nq, len, rb) + kPos - 1) / kPos;
}
__device__ __forceinline__ int64_t quotient(int64_t x, int64_t y) {  // nearly always of 32 bits
  return ((uint64_t)x | (uint64_t)y) >> 32 ? x / y : (int64_t)((uint32_t)x / (uint32_t)y);
}
// Sum of floor((p i + q) / m) over i < n, by Euclid's steps (p, q >= 0, m > 0).
__device__ __forceinline__ int64_t floor_sum(int64_t n, int64_t m, int64_t p, int64_t q) {
  int64_t sum = 0;
  while (n > 0) {
    const int64_t pm = quotient(p, m), qm = quotient(q, m);
    sum += (n - 1) * n / 2 * pm + n * qm;
    p -= pm * m;
    q -= qm * m;
    const int64_t y = p * n + q;
    if (y < m) break;
    n = quotient(y, m);
    q = y - n * m;
    const int64_t t = m;
    m = p;
    p = t;
  }
  return sum;
}
// Tiles of the request's units (of one kv head).
__device__ __forceinline__ int64_t tiles_of(const Kv4AttnArgs& a, int nq, int len) {
  if (nq <= 0) return 0;
  const int whole = req_units(a, nq) - 1;  // the last unit may hold fewer tokens
  const int64_t c = len - nq;
  const int64_t blind = c < 0 ? min((int64_t)whole, -c / a.tpb) : 0;  // units that see nothing
  return floor_sum(whole - blind, kPos, a.tpb, c + (blind + 1) * a.tpb + kPos - 1) + unit_tiles(a, nq, len, whole);
}

// The x-th tile of the list, by a whole warp: every lane has the answer.
__device__ __forceinline__ Unit seek_unit(const Kv4AttnArgs& a, const int64_t* pre, int64_t x, int lane) {
  int lo = 0, hi = a.B;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (pre[mid] <= x)
      lo = mid;
    else
      hi = mid;
  }
  const int nq = req_new(a, lo), len = req_len(a, lo);
  const int64_t rel = x - pre[lo], of_head = quotient(pre[lo + 1] - pre[lo], a.Hkv);
  Unit u;
  u.b = lo;
  u.head = (int)quotient(rel, of_head);
  int64_t left = rel - u.head * of_head;
  // 32 units at a time until their tiles reach past `left`
  for (int rb0 = 0;; rb0 += 32) {
    const int mine = rb0 + lane < req_units(a, nq) ? unit_tiles(a, nq, len, rb0 + lane) : 0;
    int inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(~0u, inc, o);
      if (lane >= o) inc += v;
    }
    const unsigned past = __ballot_sync(~0u, inc > left);
    if (past || rb0 + 32 >= req_units(a, nq)) {
      const int at = past ? __ffs(past) - 1 : 0;
      u.rb = rb0 + at;
      u.tiles = __shfl_sync(~0u, mine, at);
      u.tile = (int)(left - __shfl_sync(~0u, inc - mine, at));
      return u;
    }
    left -= __shfl_sync(~0u, inc, 31);
  }
}
// The next unit that sees a position.  Requests without tiles may be many (a
// batch's single tokens are another kernel's), and one thread looks while the
// CTA waits: 1000 of them between two prompts of 128 heads took 14.4 ms head by
// head, 0.5 ms in all now that `pre` says which they are.
__device__ __forceinline__ void next_unit(const Kv4AttnArgs& a, const int64_t* pre, Unit* u) {
  do {
    u->rb++;
    while (u->rb >= req_units(a, req_new(a, u->b))) {
      u->rb = 0;
      if (++u->head < a.Hkv) continue;
      u->head = 0;
#pragma unroll 1
      do {
        if (++u->b >= a.B) return;
      } while (pre[u->b] == pre[u->b + 1]);
    }
    u->tile = 0;
    u->tiles = unit_tiles(a, req_new(a, u->b), req_len(a, u->b), u->rb);
  } while (u->tiles == 0);
}

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
    kv4_prefill_kernel(const __grid_constant__ Kv4AttnArgs a, uint32_t polls) {
  using L = Lay<D>;
  extern __shared__ __align__(1024) uint8_t raw_smem[];
  uint8_t* sm = raw_smem + (1024 - (smem_addr(raw_smem) & 1023)) % 1024;
  Ctl* ctl = reinterpret_cast<Ctl*>(sm + L::kCtl);
  float* par = reinterpret_cast<float*>(sm + L::kPar);  // [8][ks, kz, vs, vz][64]
  int64_t* pre = reinterpret_cast<int64_t*>(sm + L::kPre);
  __shared__ int64_t wsum[kThreads / 32];
  __shared__ float sum_of[2 * kRows], own_of[2 * kRows];  // of q's rows: sum, what the scores lack beyond the unit's scale
  __shared__ float2 ml_of[kRows];  // of the second half's rows: maximum and sum of p
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(~0u, tid >> 5, 0);

  if (tid == 0) {
    mbarrier_init(&ctl->u_full, 1);
    mbarrier_init(&ctl->drained, 1);
    for (int i = 0; i < 2; i++) {
      mbarrier_init(&ctl->given[i], 4);
      mbarrier_init(&ctl->q_ready[i], 4);
      mbarrier_init(&ctl->k_full[i], 3);
      mbarrier_init(&ctl->v_full[i], 3);
      mbarrier_init(&ctl->k_free[i], 1);
      mbarrier_init(&ctl->v_free[i], 1);
      mbarrier_init(&ctl->pv_done[i], 1);
      mbarrier_init(&ctl->o_free[i], 4);
      for (int j = 0; j < 2; j++) {
        mbarrier_init(&ctl->qk_done[i][j], 1);
        mbarrier_init(&ctl->p_ready[i][j], 4);
      }
    }
    for (int i = 0; i < 8; i++) {
      mbarrier_init(&ctl->at_full[i], 1);
      mbarrier_init(&ctl->par_full[i], 1);
    }
    ctl->dead = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 8) tmem_alloc(&ctl->tmem, 512);
  if (warp == 9) ctl->at[lane >> 2][lane & 3] = -1;
  // tiles of each request over its kv heads and row blocks, as a running sum
  {
    const int per = (a.B + kThreads - 1) / kThreads;
    const int b0 = min(tid * per, a.B), b1 = min(b0 + per, a.B);
    int64_t mine = 0;
    for (int b = b0; b < b1; b++) mine += pre[b] = tiles_of(a, req_new(a, b), req_len(a, b)) * a.Hkv;
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
      const int64_t n = pre[b];
      pre[b] = run;
      run += n;
    }
    if (b1 == a.B && (b0 < a.B || tid == 0)) pre[a.B] = run;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
  }
  const uint32_t tmem = ctl->tmem;
  pdl_launch_dependents();
  // rows of no request, and rows that see no key, are zero
  if (a.fill) zero_rows_of_none(a, D);
  for (int b = blockIdx.x; b < a.B; b += gridDim.x) {
    const int64_t m = (int64_t)max(req_new(a, b) - req_len(a, b), 0) * a.H * D;
    for (int64_t i = tid; i < m; i += kThreads) a.out[(int64_t)req_start(a, b) * a.H * D + i] = 0.f;
  }
  const int64_t total = pre[a.B];
  const int64_t share = max((total + gridDim.x - 1) / gridDim.x, (int64_t)1);
  const int64_t beg = min(blockIdx.x * share, total), end = min(beg + share, total);
  if (tid == 0) a.desc[blockIdx.x] = make_int4(-1, 0, 0, 0);

  const int bpt = a.block / kKv4Tile;
  const int64_t page_bytes = (int64_t)a.Hkv * bpt * L::kTileBytes;

  if (warp < 8) {
    // ----- softmax: a warpgroup per half, a thread per row ----------------------
    const int half = warp >> 2, hrow = tid & 127;
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSmRegs));
    const uint32_t at = tmem + 256 * half + ((uint32_t)((warp & 3) * 32) << 16);  // S and P twice, O
    // tiles, this half's tiles, units so far (the top bit is the parity of those
    // that the halves took turns at)
    uint32_t j = 0, jh = 0, seg = 0;
    const int todo = (int)(end - beg);
    // What outlives a unit's first lines is kept small: 128 registers hold the
    // row's sums.  The rest is read again from ctl where the unit ends.
    for (int done = 0; done < todo; seg++) {
      if (!__all_sync(~0u, wait(&ctl->u_full, seg, ctl, polls))) break;
      float A2;
      int n, p0, vis, min_vis, step;  // step 2: few rows, which both halves take, and turns at the tiles
      bool busy;
      {
        const Unit u = ctl->unit[seg & 3];
        n = min(u.tiles - u.tile, todo - done);
        const int nq = req_new(a, u.b), len = req_len(a, u.b), rows = min(nq * a.G - u.rb * a.rpb, a.rpb);
        done += n;
        step = rows <= kRows ? 2 : 1;
        p0 = (u.tile + (step - 1) * half) * kPos;
        const int skip = (step - 1) * half * kRows;  // from this thread's number to its row
        busy = (tid & ~31) - skip < rows;
        vis = len - nq + (u.rb * a.rpb + min(tid - skip, rows - 1)) / a.G + 1;
        min_vis = __reduce_min_sync(~0u, vis);
        // q's rows, 8 channels a lane and RPP rows at a time: 9000 cycles for 128
        // of them; with a thread to a row, 25000
        const float unit = a.scale * kLog2e;  // scores come out in log2 units
        if (busy) {
          constexpr int LPR = D / 8, RPP = 32 / LPR, TURNS = LPR < 8 ? LPR / 2 : 4;
          static_assert(LPR % (2 * TURNS) == 0, "two sets of turns in flight");
          const int c = lane % LPR, w0 = (tid & ~31) + lane / LPR;
          const float inv_g = 1.f / a.G;
          const float* first = a.q + ((int64_t)req_start(a, u.b) + u.rb * a.tpb) * a.q_stride + u.head * a.G * D + 8 * c;
          const bool vec = ((uint64_t)a.q & 31) == 0 && (a.q_stride & 7) == 0;
          auto load8 = [&](int row, float (&v)[8]) {
            const int r = min(row - skip, rows - 1);  // rows past the last repeat it and are not kept
            const int tok = (int)((r + 0.5f) * inv_g);
            const float* src = first + tok * a.q_stride + (r - tok * a.G) * D;
            if (vec) {
              ld32(src, v);
            } else {
#pragma unroll
              for (int i = 0; i < 8; i++) v[i] = src[i];
            }
          };
          // max and sum of N rows over their lanes; a NaN as maximum says that
          // the row has an infinity or a NaN
          auto measure = [&](const auto& v, auto& big, auto& sum) {
            constexpr int N = sizeof(v) / 32;
#pragma unroll
            for (int k = 0; k < N; k++) {
              big[k] = fmaxf(fmaxf(fmaxf(fabsf(v[k][0]), fabsf(v[k][1])), fmaxf(fabsf(v[k][2]), fabsf(v[k][3]))),
                             fmaxf(fmaxf(fabsf(v[k][4]), fabsf(v[k][5])), fmaxf(fabsf(v[k][6]), fabsf(v[k][7]))));
              sum[k] = ((v[k][0] + v[k][1]) + (v[k][2] + v[k][3])) + ((v[k][4] + v[k][5]) + (v[k][6] + v[k][7]));
            }
#pragma unroll
            for (int off = 1; off < LPR; off <<= 1)
#pragma unroll
              for (int k = 0; k < N; k++) {
                big[k] = fmaxf(big[k], __shfl_xor_sync(~0u, big[k], off));
                sum[k] += __shfl_xor_sync(~0u, sum[k], off);
              }
#pragma unroll
            for (int k = 0; k < N; k++) big[k] = fabsf(sum[k]) < INFINITY ? big[k] * fabsf(unit) : NAN;
          };
          // the power of two that brings x to 2^11 .. 2^12
          auto top12 = [](float x) { return x > 0.f ? max(min(11 - ((int)(__float_as_uint(x) >> 23) - 127), 100), -116) : 0; };
          float v[2][TURNS][8], ref[1][8], big[TURNS], sum[TURNS];
          load8(skip, ref[0]);
#pragma unroll
          for (int k = 0; k < TURNS; k++) load8(w0 + k * RPP, v[0][k]);
          // The unit's power of two is its first row's.  Rows up to 8 times as
          // large fit fp16 beside it, rows down to 2^-12 of it lose nothing that
          // counts; others have their own.
          measure(ref, big, sum);
          const int e = top12(big[0]);
          if (tid == 0) ctl->kup = __int_as_float((127 - e) << 23);
          bool odd = false;
#pragma unroll
          for (int b = 0; b < LPR; b += TURNS) {
            float(&now)[TURNS][8] = v[b / TURNS & 1];
            if (b + TURNS < LPR) {
#pragma unroll
              for (int k = 0; k < TURNS; k++) load8(w0 + (b + TURNS + k) * RPP, v[(b / TURNS & 1) ^ 1][k]);
            }
            measure(now, big, sum);
#pragma unroll
            for (int k = 0; k < TURNS; k++) {
              const int row = w0 + (b + k) * RPP, hr = row & 127;
              int more = big[k] > 0.f ? top12(big[k]) - e : 0;
              more = more > 12 || more < -3 ? max(min(more, 126), -126) : 0;
              const float own = big[k] < INFINITY ? __int_as_float((127 - more) << 23) : NAN;
              const float up = __int_as_float((e + more + 127) << 23);
              odd |= own != 1.f;
              if (c == 0) own_of[row] = own, sum_of[row] = sum[k];
              // a chunk is 8 channels, in the order that unpacking a word gives
              // (0 4 1 5 2 6 3 7); rows of 128 bytes, chunks swizzled by row
              float lo[8];
#pragma unroll
              for (int i = 0; i < 8; i++) {
                const float x = now[k][i] * unit * up;
                now[k][i] = top11(x);
                lo[i] = x - now[k][i];
              }
              uint8_t* to = sm + half * 2 * L::kQ + (c >> 3) * (kRows * 128) + hr * 128 + (((c & 7) ^ (hr & 7)) << 4);
              *reinterpret_cast<uint4*>(to) = make_uint4(pack2(now[k][0], now[k][4]), pack2(now[k][1], now[k][5]),
                                                         pack2(now[k][2], now[k][6]), pack2(now[k][3], now[k][7]));
              *reinterpret_cast<uint4*>(to + L::kQ) =
                  make_uint4(pack2(lo[0], lo[4]), pack2(lo[1], lo[5]), pack2(lo[2], lo[6]), pack2(lo[3], lo[7]));
            }
          }
          if (__any_sync(~0u, odd)) min_vis = INT_MIN;  // none of the warp's tiles goes without a look at its rows
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        A2 = busy ? sum_of[tid] * unit : 0.f;
        if (lane == 0) mbarrier_arrive(&ctl->q_ready[half]);
      }

      float o[D];
#pragma unroll
      for (int i = 0; i < D; i++) o[i] = 0.f;
      float m = kNoMax, vdown = 0.f;
      float2 l = make_float2(0.f, 0.f), za = l;
      // adds the tile's O in TMEM, then applies f
      auto take = [&](uint32_t of, float f) {
        wait(&ctl->pv_done[half], of, ctl, polls);
        tc_fence_after();
        if (busy) {
#pragma unroll
          for (int c = 0; c < D / 16; c++) {
            uint32_t t[16];
            tmem_ld16(at + 128 + 16 * c, t);
            tmem_wait_ld();
            pin16(t);
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
              const float2 s = add2(make_float2(o[16 * c + i], o[16 * c + i + 1]),
                                    make_float2(__uint_as_float(t[i]), __uint_as_float(t[i + 1])));
              o[16 * c + i] = s.x, o[16 * c + i + 1] = s.y;
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbarrier_arrive(&ctl->o_free[half]);
        if (__any_sync(~0u, f != 1.f)) {
#pragma unroll
          for (int i = 0; i < D; i += 2) {
            const float2 s = mul2(make_float2(o[i], o[i + 1]), make_float2(f, f));
            o[i] = s.x, o[i + 1] = s.y;
          }
        }
      };

      const int own = step == 2 ? (n + 1 - half) >> 1 : n;  // tiles of this half
      const uint32_t j_end = j + n;
      if (step == 2) j += half;
#pragma unroll 1
      for (int k = 0; k <= own; k++) {
        float f = 1.f;
        if (k < own) {
          wait(&ctl->par_full[j & 7], j >> 3, ctl, polls);  // the tile's parameters
          wait(&ctl->qk_done[half][jh & 1], jh >> 1, ctl, polls);
          tc_fence_after();
          const float* pk = par + (j & 7) * (4 * kPos);
          const float4 hd = ctl->head[j & 7];
          const uint32_t sbuf = at + (jh & 1) * 64;
          const int absent = __float_as_int(hd.z);
          if (vdown != hd.y) {  // V's scale has changed since the half's last tile (or O is 0 yet)
            f = vdown * hd.x;
            vdown = hd.y;
          }
          auto soft = [&](auto edge_c) {
            constexpr bool edge = decltype(edge_c)::value;
            const float2 aa = make_float2(A2, A2);
#pragma unroll 1
            for (int c = 0; c < 4; c++) {
              uint32_t t[16], w[16];
              tmem_ld16(sbuf + 16 * c, t);
              tmem_wait_ld();
              pin16(t);
              if (edge) {
                const float own = own_of[tid];
#pragma unroll
                for (int i = 0; i < 16; i++) t[i] = __float_as_uint(__uint_as_float(t[i]) * own);
              }
              const int seen = absent >> c & 1 ? 0 : vis - p0 - 16 * c;  // positions from 16 c on that the row sees
              float2 x[8];
              float top = -INFINITY;
#pragma unroll
              for (int i = 0; i < 8; i++) {
                const float4 s4 = reinterpret_cast<const float4*>(pk + 16 * c)[i >> 1];
                const float4 z4 = reinterpret_cast<const float4*>(pk + kPos + 16 * c)[i >> 1];
                const float2 s2 = i & 1 ? make_float2(s4.z, s4.w) : make_float2(s4.x, s4.y);
                const float2 z2 = i & 1 ? make_float2(z4.z, z4.w) : make_float2(z4.x, z4.y);
                x[i] = fma2(s2, make_float2(__uint_as_float(t[2 * i]), __uint_as_float(t[2 * i + 1])), mul2(z2, aa));
                if (edge && 2 * i >= seen) x[i].x = -INFINITY;
                if (edge && 2 * i + 1 >= seen) x[i].y = -INFINITY;
                top = fmaxf(top, fmaxf(x[i].x, x[i].y));
              }
              // the reference maximum moves only when a score passes it by 2^8
              if (__any_sync(~0u, top > m + 8.f)) {
                const float f1 = top > m + 8.f ? ex2(m - top) : 1.f;
                m = top > m + 8.f ? top : m;
                f *= f1;
                l = mul2(l, make_float2(f1, f1));
                za = mul2(za, make_float2(f1, f1));
                // what this tile has stored already is of the old one
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
#pragma unroll 1
                for (int d = 0; d < c; d++) {
                  tmem_ld16(sbuf + 16 * d, w);
                  tmem_wait_ld();
                  pin16(w);
#pragma unroll
                  for (int i = 0; i < 8; i++) {
                    const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
                    const float2 g = __half22float2(*reinterpret_cast<const __half2*>(&w[8 + i]));
                    const float2 y = mul2(add2(h, g), make_float2(f1, f1));
                    const float2 hi = make_float2(top11(y.x), top11(y.y));
                    w[i] = pack2(hi.x, hi.y);
                    w[8 + i] = pack2(y.x - hi.x, y.y - hi.y);
                  }
                  tmem_st16(sbuf + 16 * d, w);
                }
              }
              const float2 mm = make_float2(-m, -m);
              // the 16 positions' sums from zero: added one by one over a context of
              // 131072, equal terms lose up to 1e-3, and random ones 3.4e-6 (1.3e-6 so)
              float2 lc = make_float2(0.f, 0.f), zc = lc;
#pragma unroll
              for (int i = 0; i < 8; i++) {
                const float4 s4 = reinterpret_cast<const float4*>(pk + 2 * kPos + 16 * c)[i >> 1];
                const float4 z4 = reinterpret_cast<const float4*>(pk + 3 * kPos + 16 * c)[i >> 1];
                float2 vs = i & 1 ? make_float2(s4.z, s4.w) : make_float2(s4.x, s4.y);
                float2 vz = i & 1 ? make_float2(z4.z, z4.w) : make_float2(z4.x, z4.y);
                if (edge) {  // a position that others see but this row does not may be NaN
                  if (2 * i >= seen) vs.x = vz.x = 0.f;
                  if (2 * i + 1 >= seen) vs.y = vz.y = 0.f;
                }
                const float2 d = add2(x[i], mm), pr = make_float2(ex2(d.x), ex2(d.y));
                lc = add2(lc, pr);
                zc = fma2(pr, vz, zc);
                const float2 y = mul2(pr, vs), hi = make_float2(top11(y.x), top11(y.y));
                w[i] = pack2(hi.x, hi.y);
                w[8 + i] = pack2(y.x - hi.x, y.y - hi.y);
              }
              tmem_st16(sbuf + 16 * c, w);
              l = add2(l, lc);
              za = add2(za, zc);
            }
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
          };
          if (busy) {
            if (absent != 0 || p0 + kPos > min_vis)  // some row does not see all of it, or is not of the unit's scale
              soft(std::true_type{});
            else
              soft(std::false_type{});
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbarrier_arrive(&ctl->p_ready[half][jh & 1]);
          j += step;
          jh++;
          p0 += step * kPos;
        }
        if (k > 0) take(jh - (k < own ? 2 : 1), f);
      }
      j = j_end;

      // The rows, or their part for kv4_join_kernel, by way of the place of
      // their q, which no product reads any more: whole rows to a warp's store.
      const Unit u = ctl->unit[seg & 3];
      const int rows = min(req_new(a, u.b) * a.G - u.rb * a.rpb, a.rpb);
      const bool begins = u.tile == 0, ends = u.tile + n == u.tiles, whole = begins && ends;
      // Where the halves took turns the second hands its sums to the first.
      const bool turns = rows <= kRows, gives = turns && half == 1;
      if (turns && half == 0) wait(&ctl->given[0], seg >> 31, ctl, polls);
      if (busy) {
        float sum = l.x + l.y, f0 = 1.f, f1 = 0.f;
        if (turns && half == 0) {
          const float2 other = ml_of[hrow];
          const float mx = fmaxf(m, other.x);
          f0 = ex2(m - mx), f1 = ex2(other.x - mx);
          sum = sum * f0 + other.y * f1;
          m = mx;
        }
        const float norm = !whole || gives ? 1.f : sum == 0.f ? 0.f : 1.f / sum;
        const float down = vdown * f0 * norm, z = (za.x + za.y) * f0 * norm;
        f1 *= norm;
        float* part = a.part + ((int64_t)(2 * blockIdx.x + begins) * a.rpb + (tid & ~31)) * (D + 4);
        if (gives)
          ml_of[hrow] = make_float2(m, sum);
        else if (!whole && tid < rows)
          *reinterpret_cast<float2*>(part + lane * (D + 4) + D) = make_float2(m, sum);
        uint8_t* mine = sm + half * 2 * L::kQ + (hrow & ~31) * 128;
        // the i-th 16 bytes of the warp's row r
        auto at16 = [&](int r, int i) { return mine + (i >> 3) * (kRows * 128) + r * 128 + (((i & 7) ^ (r & 7)) << 4); };
#pragma unroll
        for (int c = 0; c < D; c += 8) {
          float v[8];
#pragma unroll
          for (int i = 0; i < 8; i++) v[i] = fmaf(o[c + 2 * (i & 3) + (i >> 2)], down, z);
          if (turns && half == 0) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
              const float4 f = *reinterpret_cast<const float4*>(at16(lane, c / 4 + i) + 2 * L::kQ);
              v[4 * i] = fmaf(f.x, f1, v[4 * i]), v[4 * i + 1] = fmaf(f.y, f1, v[4 * i + 1]);
              v[4 * i + 2] = fmaf(f.z, f1, v[4 * i + 2]), v[4 * i + 3] = fmaf(f.w, f1, v[4 * i + 3]);
            }
          }
          *reinterpret_cast<float4*>(at16(lane, c / 4)) = make_float4(v[0], v[1], v[2], v[3]);
          *reinterpret_cast<float4*>(at16(lane, c / 4 + 1)) = make_float4(v[4], v[5], v[6], v[7]);
        }
        __syncwarp();
        constexpr int LPR = D / 4, RPP = 32 / LPR;  // lanes of a row, rows at a time
        const float inv_g = 1.f / a.G;
        const int most = gives ? 0 : min(rows - (tid & ~31), 32);
        float* first = a.out + (((int64_t)req_start(a, u.b) + u.rb * a.tpb) * a.H + u.head * a.G) * D;
#pragma unroll 8
        for (int k = 0; k < 32; k += RPP) {
          const int r = k + lane / LPR;
          if (r >= most) break;
          const int row = (tid & ~31) + r, tok = (int)((row + 0.5f) * inv_g);
          float* to = whole ? first + ((int64_t)tok * a.H + row - tok * a.G) * D : part + r * (D + 4);
          reinterpret_cast<float4*>(to)[lane % LPR] = *reinterpret_cast<const float4*>(at16(r, lane % LPR));
        }
        __syncwarp();
      }
      if (turns) {
        if (lane == 0) mbarrier_arrive(&ctl->given[1 - half]);  // its sums are there, or are read
        if (half == 1) wait(&ctl->given[1], seg >> 31, ctl, polls);
        seg ^= 1u << 31;
      }
      if (tid == 0 && begins && !ends)
        a.desc[blockIdx.x] = make_int4(u.b, u.head, u.rb, (int)((beg + done - n + u.tiles - 1) / share));
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kUnRegs));
    if (warp == 8) {
      // ----- MMA issue ---------------------------------------------------------
      Unit u = {};
      if (beg < end) u = seek_unit(a, pre, beg, lane);
      if (beg < end && elect_one()) {
        // descriptors of the buffers' first steps; a step's is a sum, made anew
        // each time (hoisted out of the loops they would spill)
        uint64_t dq = sw128_desc(smem_addr(sm)), dk = sw128_desc(smem_addr(sm + L::kK)),
                 dv = sw128_mn_desc(smem_addr(sm + L::kV), kPos * 128);
        uint32_t jh[2] = {0, 0};  // the halves' tiles so far
        const uint32_t id_qk = idesc_f16(kPos, false), id_pv = idesc_f16(64 * L::kAtoms, true);
        uint32_t j = 0, seg = 0;
        for (int64_t x = beg; x < end; seg++) {
          if (x > beg) next_unit(a, pre, &u);
          ctl->unit[seg & 3] = u;
          mbarrier_arrive(&ctl->u_full);
          const int n = (int)min((int64_t)(u.tiles - u.tile), end - x);
          x += n;
          // 1: the halves, of the same rows, take turns at the tiles
          const int turns = min(req_new(a, u.b) * a.G - u.rb * a.rpb, a.rpb) <= kRows;
          bool alive = true;
          for (int h = 0; h < 2; h++) alive &= wait(&ctl->q_ready[h], seg, ctl, polls);
          // A half's scores run at most one tile ahead of its products with V;
          // whatever is ready goes next (one copy of each product: the
          // instruction cache holds the roles' loops).
          const uint32_t last = j + n;
          uint32_t tq0 = j, tp0 = j, tq1 = j + turns, tp1 = tq1;
          uint32_t spins = 0;
#pragma unroll 1
          for (int h = 0; alive && (tp0 < last || tp1 < last); h ^= 1) {
            const uint32_t tq = h ? tq1 : tq0, tp = h ? tp1 : tp0;
            // the half's own numbers of these tiles
            const uint32_t nq = (h ? jh[1] : jh[0]) + ((tq - j) >> turns), np = (h ? jh[1] : jh[0]) + ((tp - j) >> turns);
            const uint32_t base = tmem + 256 * h;
            if (tq < last && nq <= np + 1 && ready(&ctl->k_full[tq & 1], tq >> 1)) {
              tc_fence_after();
              asm volatile("" : "+l"(dq), "+l"(dk));
              const uint64_t qd = dq + (uint64_t)(h * 2 * L::kQ >> 4), kd = dk + (uint64_t)((tq & 1) * L::kKv >> 4);
              const uint32_t to = base + (nq & 1) * 64;
#pragma unroll
              for (int term = 1; term >= 0; term--)  // the small terms first: each MMA truncates its sum
#pragma unroll
                for (int s = 0; s < D / 16; s++)
                  mma_ss(to, qd + ((term * L::kQ + (s >> 2) * (kRows * 128) + (s & 3) * 32) >> 4),
                         kd + (((s >> 2) * (kPos * 128) + (s & 3) * 32) >> 4), id_qk, term == 0 || s > 0);
              tc_commit(&ctl->qk_done[h][nq & 1]);
              if (turns || tq < (h ? tq0 : tq1)) tc_commit(&ctl->k_free[tq & 1]);  // the other half is past it
              (h ? tq1 : tq0) += 1 + turns;
              spins = 0;
            } else if (tp < tq && ready(&ctl->p_ready[h][np & 1], np >> 1) &&
                       ready(&ctl->v_full[tp & 1], tp >> 1)) {
              // (no waiting for V here: its buffer may want the other half's product first)
              if (np > 0) wait(&ctl->o_free[h], np - 1, ctl, polls);
              tc_fence_after();
              asm volatile("" : "+l"(dv));
              const uint64_t vd = dv + (uint64_t)((tp & 1) * L::kKv >> 4);
              const uint32_t from = base + (np & 1) * 64;
#pragma unroll
              for (int term = 1; term >= 0; term--)
#pragma unroll
                for (int s = 0; s < kPos / 16; s++)
                  mma_ts(base + 128, from + 16 * s + 8 * term, vd + (2048 * s >> 4), id_pv, term == 0 || s > 0);
              tc_commit(&ctl->pv_done[h]);
              if (turns || tp < (h ? tp0 : tp1)) tc_commit(&ctl->v_free[tp & 1]);
              (h ? tp1 : tp0) += 1 + turns;
              spins = 0;
            } else if (++spins > 4 * polls) {
              expire(ctl);
            }
            if (*reinterpret_cast<volatile int*>(&ctl->dead)) alive = false;
          }
          if (!alive) break;
          jh[0] += (n + turns) >> turns;
          jh[1] += n >> turns;
          j = last;
        }
        // no arrival may come after the CTA's end, nor a product after its TMEM's
        tc_commit(&ctl->drained);
        for (uint32_t it = 0; it < (1u << 22) && !ready(&ctl->drained, 0); it++) {
        }
      }
      __syncwarp();
    } else {
      // ----- warp 9: where tiles lie, and their scales and zeros; warps 10 to 12
      // and 13 to 15: K and V codes to fp16 tiles ----------------------------------
      uint32_t j = 0, seg = 0;
      const int todo = (int)(end - beg);
      for (int done = 0; done < todo; seg++) {
        if (!__all_sync(~0u, wait(&ctl->u_full, seg, ctl, polls))) break;
        const Unit u = ctl->unit[seg & 3];
        const int n = min(u.tiles - u.tile, todo - done);
        done += n;
        if (warp == 9) {
          const int len = req_len(a, u.b), seen = min(unit_vis(a, req_new(a, u.b), len, u.rb), len);
          const int head0 = u.head * bpt;
          const int32_t* row = a.table + (int64_t)u.b * a.max_blocks;
          // lane p < 4 looks the tile's p-th 16 positions up, a tile ahead
          int part = u.tile * 4 + (lane & 3), entry = -1, place = 0;
          auto look = [&]() {
            const int col = a.bpt_shift >= 0 ? part >> a.bpt_shift : part / bpt;
            place = head0 + part - col * bpt;
            entry = -1;
            if (lane < 4 && part * kKv4Tile < seen) entry = row[col];
            part += 4;
          };
          look();
          float kup = 0.f, vup = 0.f;
#pragma unroll 1
          for (int k = 0; k < n; k++, j++) {
            // whose places and parameters these replace are read by then
            if (j > 1) wait(&ctl->k_free[j & 1], (j - 2) >> 1, ctl, polls);
            const bool ok = (unsigned)entry < (unsigned)a.num_blocks;
            const int64_t at = ok ? entry * page_bytes + (int64_t)place * L::kTileBytes : -1;  // -1: nowhere
            const bool asked = lane < 4 && (part - 4) * kKv4Tile < seen;  // else nothing was there to look up
            if (!ok && asked && a.bad) atomicAdd(a.bad, 1);
            if (lane < 4) ctl->at[j & 7][lane] = at;
            __syncwarp();
            if (lane == 0) mbarrier_arrive(&ctl->at_full[j & 7]);
            const int absent = (int)__ballot_sync(~0u, asked && !ok);
            const int left = seen - (part - 4 - (lane & 3)) * kKv4Tile;  // positions from the tile's first on
            float* pk = par + (j & 7) * (4 * kPos);
            uint32_t kw[2], vw[2];
#pragma unroll
            for (int i = 0; i < 2; i++) {
              const int64_t t = __shfl_sync(~0u, at, 2 * i + (lane >> 4));
              kw[i] = vw[i] = 0;
              if (t >= 0 && 32 * i + lane < left) {
                const uint32_t* words = reinterpret_cast<const uint32_t*>(a.pages + t + 16 * D) + (lane & 15);
                kw[i] = __ldg(words);
                vw[i] = __ldg(words + 16);
              }
            }
            if (k + 1 < n) look();
            if (k == 0) {  // the unpacking of the unit's first tiles is under way
              for (int h = 0; h < 2; h++) wait(&ctl->q_ready[h], seg, ctl, polls);
              kup = *reinterpret_cast<volatile float*>(&ctl->kup);
            }
            float vs[2], top = 0.f;
#pragma unroll
            for (int i = 0; i < 2; i++) {
              pk[32 * i + lane] = kv4_scale(kw[i]) * kup;
              pk[kPos + 32 * i + lane] = kv4_zero(kw[i]);
              pk[3 * kPos + 32 * i + lane] = kv4_zero(vw[i]);
              vs[i] = kv4_scale(vw[i]);
              if (vs[i] < INFINITY) top = fmaxf(top, vs[i]);
            }
            top = warp_max(top);
            // vup V's scale stays below 2^7, p at or below 2^8: fp16 holds 40
            // binades below their product
            if (top * vup >= 128.f || (vup == 0.f && top > 0.f)) {
              const int vexp = max(min(6 - ((int)(__float_as_uint(top) >> 23) - 127), 100), -100);
              vup = __int_as_float((vexp + 127) << 23);
            }
#pragma unroll
            for (int i = 0; i < 2; i++) pk[2 * kPos + 32 * i + lane] = vs[i] * vup;
            if (lane == 0)
              ctl->head[j & 7] = make_float4(vup, vup == 0.f ? 0.f : 1.f / vup, __int_as_float(absent), 0.f);
            __syncwarp();
            if (lane == 0) mbarrier_arrive(&ctl->par_full[j & 7]);
          }
          continue;
        }
        constexpr int Q = D / 32;              // 16-byte pieces of a code row
        constexpr int PI = 32 / Q;             // positions a warp takes at a time
        constexpr int NI = kPos / PI;          // such pieces of work of a tile, for three warps
        constexpr int MI = (NI + 2) / 3;
        const int v = warp > 12, i0 = (warp - 10 - 3 * v) * MI;
        const int pl = (lane & 7) + 8 * (lane / (8 * Q)), q = (lane >> 3) % Q;  // this lane's position and piece
        // where the piece's first 16 bytes of fp16 go: rows of 128 bytes, chunks
        // swizzled by row; its k-th 16 bytes are at this address ^ 16 k
        const uint32_t spot = smem_addr(sm + (v ? L::kV : L::kK)) + (q >> 1) * (kPos * 128) + (i0 * PI + pl) * 128 +
                              (((4 * (q & 1)) ^ (pl & 7)) << 4);
        uint64_t* full = v ? ctl->v_full : ctl->k_full;
        uint64_t* free = v ? ctl->v_free : ctl->k_free;
#pragma unroll 1
        for (int k = 0; k < n; k++, j++) {
          wait(&ctl->at_full[j & 7], j >> 3, ctl, polls);
          uint4 raw[MI];
#pragma unroll
          for (int i = 0; i < MI; i++) {
            const int pos = (i0 + i) * PI + pl;
            raw[i] = make_uint4(0, 0, 0, 0);
            if (pos < kPos) {
              const int64_t t = *reinterpret_cast<volatile int64_t*>(&ctl->at[j & 7][pos / kKv4Tile]);
              if (t >= 0)
                raw[i] = __ldg(reinterpret_cast<const uint4*>(a.pages + t +
                                                              (v * 8 * D + (pos % kKv4Tile) * (D / 2) + 16 * q)));
            }
          }
          if (j > 1) wait(&free[j & 1], (j - 2) >> 1, ctl, polls);
#pragma unroll
          for (int i = 0; i < MI; i++) {
            if ((i0 + i) * PI >= kPos) continue;
            const uint32_t wd[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
            for (int c = 0; c < 4; c++) {
              const uint32_t x0 = wd[c], x1 = wd[c] >> 8;
              asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"((spot ^ (16 * c)) + (j & 1) * L::kKv +
                                                                             i * (PI * 128)),
                           "r"(nibble_f16(x0, 0x000f000fu, 0x64006400u, 0x64086408u)),
                           "r"(nibble_f16(x0, 0x00f000f0u, 0x54005400u, 0x54805480u)),
                           "r"(nibble_f16(x1, 0x000f000fu, 0x64006400u, 0x64086408u)),
                           "r"(nibble_f16(x1, 0x00f000f0u, 0x54005400u, 0x54805480u))
                           : "memory");
            }
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) mbarrier_arrive(&full[j & 1]);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) tmem_dealloc(tmem, 512);
  if (tid == 0 && ctl->dead) a.desc[blockIdx.x].x = kExpired;
}

// Joins the parts of units that more than one CTA took: a warp per (CTA that
// began a unit, row).  A CTA has two parts at most.
template <int D>
__global__ void __launch_bounds__(256, 8) kv4_join_kernel(Kv4AttnArgs a, int groups) {
  constexpr int V = D / 32;
  pdl_wait();
  const int lane = threadIdx.x & 31, first = blockIdx.x / groups;
  const int row = blockIdx.x % groups * 8 + (threadIdx.x >> 5);
  const int4 d = a.desc[first];
  if (d.x == kExpired) {  // what this CTA should have written is anywhere
    const int64_t n = (int64_t)a.T * a.H * D;
    for (int64_t i = (int64_t)(blockIdx.x % groups) * blockDim.x + threadIdx.x; i < n; i += groups * blockDim.x)
      a.out[i] = NAN;
    return;
  }
  if (d.x < 0 || row >= a.rpb) return;
  const int r = d.z * a.rpb + row;
  if (r >= req_new(a, d.x) * a.G) return;
  float m = kNoMax, l = 0.f, o[V];
#pragma unroll
  for (int k = 0; k < V; k++) o[k] = 0.f;
#pragma unroll 4
  for (int i = first; i <= d.w; i++) {
    const float* p = a.part + ((int64_t)(2 * i + (i == first)) * a.rpb + row) * (D + 4);
    const float m1 = p[D], l1 = p[D + 1], mn = fmaxf(m, m1);
    const float f0 = ex2(m - mn), f1 = a.desc[i].x == kExpired ? NAN : ex2(m1 - mn);
    m = mn;
    l = l * f0 + l1 * f1;
#pragma unroll
    for (int k = 0; k < V; k++) o[k] = o[k] * f0 + p[lane + 32 * k] * f1;
  }
  const float norm = l == 0.f ? 0.f : 1.f / l;
  const int tok = r / a.G;
  float* to = a.out + (((int64_t)req_start(a, d.x) + tok) * a.H + d.y * a.G + r - tok * a.G) * D;
#pragma unroll
  for (int k = 0; k < V; k++) to[lane + 32 * k] = o[k] * norm;
}

// Polls of a device wait before it counts as run out.  TENDO_B200_KV4_POLLS sets
// another number, so that tests can let waits of a sound pipeline run out.
uint32_t wait_polls() {
  static const uint32_t n = [] {
    const char* e = getenv("TENDO_B200_KV4_POLLS");
    const long v = e ? atol(e) : 0;
    return v > 0 && v < (1 << 22) ? (uint32_t)v : 1u << 22;
  }();
  return n;
}
int ctas() { return sm_count(); }
// Tokens of a unit: as many as two halves hold, or as there are.
int tokens_of(int64_t G, int64_t max_q) { return (int)(max_q < 2 * kRows / G ? max_q : 2 * kRows / G); }

template <int D>
tb_status_t launch(const Kv4AttnArgs& a, cudaStream_t st) {
  const size_t smem = 1024 + Lay<D>::kPre + 8 * (size_t)(a.B + 1);
  static std::atomic<uint64_t> ready{0};
  TB_TRY(allow_smem(reinterpret_cast<const void*>(kv4_prefill_kernel<D>),
                    1024 + Lay<D>::kPre + 8 * (size_t)(kKv4MaxB + 1), ready));
  kv4_prefill_kernel<D><<<ctas(), kThreads, smem, st>>>(a, wait_polls());
  TB_TRY(check_launch("kv4_prefill_kernel"));
  cudaLaunchConfig_t cfg = {};
  const int groups = (a.rpb + 7) / 8;
  cfg.gridDim = dim3((unsigned)(ctas() * groups));
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  TB_CUDA(cudaLaunchKernelEx(&cfg, kv4_join_kernel<D>, a, groups));
  return check_launch("kv4_join_kernel");
}

}  // namespace

size_t kv4_prefill_workspace(int64_t G, int64_t max_q, int64_t D) {
  return ctas() * sizeof(int4) + 2 * (size_t)ctas() * tokens_of(G, max_q) * G * (size_t)(D + 4) * sizeof(float);
}

tb_status_t kv4_prefill(Kv4AttnArgs a, int64_t max_q, int D, void* ws, cudaStream_t st) {
  a.desc = static_cast<int4*>(ws);
  a.part = reinterpret_cast<float*>(a.desc + ctas());
  a.tpb = tokens_of(a.G, max_q);
  a.rpb = a.tpb * a.G;
  if (D == 128) return launch<128>(a, st);
  return D == 64 ? launch<64>(a, st) : launch<32>(a, st);
}

}  // namespace tb

extern "C" tb_status_t tb_kv4_attention_status(tb_stream_t stream) {
  TB_INJECT("tb_kv4_attention_status");
  cudaStream_t st = (cudaStream_t)stream;
  void* word = nullptr;
  int expired = 0;
  TB_CUDA(cudaGetSymbolAddress(&word, tb::g_expired));
  TB_CUDA(cudaMemcpyAsync(&expired, word, sizeof(int), cudaMemcpyDeviceToHost, st));
  TB_CUDA(cudaStreamSynchronize(st));
  if (expired == 0) return TB_SUCCESS;
  TB_CUDA(cudaMemsetAsync(word, 0, sizeof(int), st));
  TB_CUDA(cudaStreamSynchronize(st));
  return TB_ERROR_TIMEOUT;
}
