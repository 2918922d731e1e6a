// kv4.cu — the paged 4-bit KV cache: planning (block tables and slot maps
// from request lengths), append with RoPE, and reads by slot.
#include <limits.h>

#include "common.cuh"
#include "kv4.cuh"

namespace tb {
namespace {

// ---------------------------------------------------------------------------
// Plan
//
// Every CTA scans the requests' three counts (pages given back, pages taken,
// new tokens) into shared memory for itself: B is at most a few thousand, the
// scan is a few microseconds at most, and no CTA then waits for another.  The
// free list is a stack.  Surplus pages are pushed and missing ones popped, but
// no pop reads what a push of this launch wrote: the k-th popped page is
// element count + R - 1 - k of the stack after the pushes, and an element past
// `count` is looked up where it came from, in the table row that gives it
// back.  Reads are of entries that no CTA writes (table columns below what a
// request holds, stack entries below `count`), so the launch needs no order
// among its CTAs and repeating it with the same inputs changes nothing.
// Latency bounds it: 64 requests of one token 5.4 us, 1024 requests with
// prompt chunks (some 30000 tokens) 8.9 us, of which an empty launch is 2.5.
// ---------------------------------------------------------------------------
constexpr int kPlanThreads = 512;
constexpr int kPlanMaxB = 16384;  // three int32 prefix arrays: 192 KB of shared memory

struct PlanArgs {
  int32_t *q_start, *seq_lens, *positions, *slots, *count_out, *bad, *table, *free_list;
  const int32_t *count, *held, *ctx, *add;
  int B, T, max_blocks, num_blocks, block;
};

struct Sum3 {
  long long give, take, add;
};
__device__ __forceinline__ Sum3 plus(Sum3 a, Sum3 b) { return {a.give + b.give, a.take + b.take, a.add + b.add}; }

// Pages of n positions (n + block - 1 may pass INT_MAX).
__device__ __forceinline__ int pages_of(const PlanArgs& a, int n) {
  return (int)(((unsigned)n + (unsigned)a.block - 1u) / (unsigned)a.block);
}

// One request's counts; false when its lengths are not ones a plan can serve:
// no request holds more pages than there are.
__device__ __forceinline__ bool plan_request(const PlanArgs& a, int b, int& have, int& need, Sum3& s) {
  const long long h = a.held[b], c = a.ctx[b], n = a.add[b];
  const long long hb = (h + a.block - 1) / a.block, nb = (c + n + a.block - 1) / a.block;
  s = {0, 0, 0};
  have = need = 0;
  const int most = min(a.max_blocks, a.num_blocks);
  if (h < 0 || c < 0 || n < 0 || hb > most || nb > most || c + n > INT_MAX) return false;
  have = (int)hb;
  need = (int)nb;
  s.give = hb > nb ? hb - nb : 0;
  s.take = nb > hb ? nb - hb : 0;
  s.add = n;
  return true;
}

// Largest b with pre[b] <= x (pre[0] = 0, non-decreasing, x < pre[B]).
__device__ __forceinline__ int find(const int32_t* pre, int B, int x) {
  int lo = 0, hi = B;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (pre[mid] <= x)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(kPlanThreads) kv4_plan_kernel(PlanArgs a) {
  extern __shared__ int32_t sm[];
  int32_t* give = sm;                // [B + 1] exclusive prefix sums
  int32_t* take = give + a.B + 1;
  int32_t* add = take + a.B + 1;
  __shared__ Sum3 wsum[kPlanThreads / 32];
  __shared__ int sbad;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) sbad = 0;
  __syncthreads();
  const int per = (a.B + kPlanThreads - 1) / kPlanThreads;
  const int b0 = min(tid * per, a.B), b1 = min(b0 + per, a.B);
  Sum3 mine = {0, 0, 0};
  bool ok = true;
  for (int b = b0; b < b1; b++) {
    int have, need;
    Sum3 s;
    ok &= plan_request(a, b, have, need, s);
    mine = plus(mine, s);
  }
  if (!ok) sbad = 1;
  Sum3 inc = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const Sum3 v = {__shfl_up_sync(~0u, inc.give, o), __shfl_up_sync(~0u, inc.take, o),
                    __shfl_up_sync(~0u, inc.add, o)};
    if (lane >= o) inc = plus(inc, v);
  }
  if (lane == 31) wsum[warp] = inc;
  __syncthreads();
  Sum3 run = {inc.give - mine.give, inc.take - mine.take, inc.add - mine.add}, all = {0, 0, 0};
#pragma unroll
  for (int w = 0; w < kPlanThreads / 32; w++) {
    if (w < warp) run = plus(run, wsum[w]);
    all = plus(all, wsum[w]);
  }
  for (int b = b0; b < b1; b++) {
    int have, need;
    Sum3 s;
    plan_request(a, b, have, need, s);
    give[b] = (int32_t)run.give;
    take[b] = (int32_t)run.take;
    add[b] = (int32_t)run.add;
    run = plus(run, s);
  }
  if (tid == 0) {
    give[a.B] = (int32_t)all.give;
    take[a.B] = (int32_t)all.take;
    add[a.B] = (int32_t)all.add;
  }
  __syncthreads();
  const long long count = a.count[0];
  const bool bad = sbad || count < 0 || count + all.give > a.num_blocks || all.take > count + all.give ||
                   all.add > a.T;
  const int step = gridDim.x * kPlanThreads, first = blockIdx.x * kPlanThreads + tid;
  if (blockIdx.x == 0) {
    if (tid == 0) {
      *a.count_out = (int32_t)(bad ? count : count + all.give - all.take);
      if (a.bad) *a.bad = bad;
    }
    for (int b = tid; b <= a.B; b += kPlanThreads) a.q_start[b] = bad ? 0 : add[b];
    for (int b = tid; b < a.B; b += kPlanThreads) a.seq_lens[b] = a.ctx[b] + (bad ? 0 : a.add[b]);
  }
  if (bad) {  // nothing moves; no token has a slot
    for (int t = first; t < a.T; t += step) {
      a.positions[t] = 0;
      a.slots[t] = -1;
    }
    return;
  }
  const int n_take = (int)all.take, n_give = (int)all.give, n_add = (int)all.add, top = (int)count + n_give;
  // the r-th page given back, and the k-th page taken
  auto given = [&](int r) {
    const int b = find(give, a.B, r);
    const int need = pages_of(a, a.ctx[b] + a.add[b]);
    return a.table[(int64_t)b * a.max_blocks + need + (r - give[b])];
  };
  auto taken = [&](int k) {
    const int v = top - 1 - k;
    return v < (int)count ? a.free_list[v] : given(v - (int)count);
  };
  for (int t = first; t < a.T; t += step) {
    int pos = 0, slot = -1;
    if (t < n_add) {
      const int b = find(add, a.B, t);
      pos = a.ctx[b] + t - add[b];
      const int have = pages_of(a, a.held[b]), col = pos / a.block;
      const int blk = col < have ? a.table[(int64_t)b * a.max_blocks + col] : taken(take[b] + col - have);
      slot = blk < 0 || blk >= a.num_blocks ? -1 : blk * a.block + (pos - col * a.block);
    }
    a.positions[t] = pos;
    a.slots[t] = slot;
  }
  for (int r = first; r < n_give; r += step) a.free_list[(int)count + r] = given(r);
  for (int k = first; k < n_take; k += step) {
    const int b = find(take, a.B, k);
    const int have = pages_of(a, a.held[b]);
    a.table[(int64_t)b * a.max_blocks + have + (k - take[b])] = taken(k);
  }
}

// ---------------------------------------------------------------------------
// Append and read
//
//   y = RoPE(x);  zero = bf16(7/15 min y + 8/15 max y), scale the smallest bf16
//   that covers y from there;  code = round((y - zero) / scale) in -8 .. 7.
//
// D / 8 lanes hold a row: lane l has channels 4l .. 4l + 3 and D/2 + 4l ..
// D/2 + 4l + 3, so rotate-half pairs stay in a lane, loads are 16 bytes and
// a lane's codes are two 16-bit stores.  Memory bounds both: 8192 tokens of 64
// heads and 8 kv heads of 128 appended and read back take 128 us, 5.4 TB/s, 82%
// of a copy's rate; 64 tokens of 32 heads 5.5 us, launches in the main.
// ---------------------------------------------------------------------------
struct AppendArgs {
  uint8_t* pages;
  float* q_out;  // [T, H, D], null without q
  const float *q, *k, *v, *cos_t, *sin_t;
  const int32_t *positions, *slots;
  int32_t* bad;
  int64_t q_stride, k_stride, v_stride, slots_max;
  int T, H, Hkv, block, max_pos;
};

template <bool VEC>
__device__ __forceinline__ float4 load4(const float* p) {
  if (VEC) return *reinterpret_cast<const float4*>(p);
  return make_float4(p[0], p[1], p[2], p[3]);
}

// A block of 256 threads takes 256 / L neighbouring rows (heads of q, k and v in
// turn) of one token at a time, and `turns` such groups: RoPE's factors stay in
// registers, and a thread's next rows are on their way while it works on one.
template <int D, bool VEC>
__global__ void __launch_bounds__(256) kv4_append_kernel(AppendArgs a, int turns) {
  constexpr int L = D / 8;       // lanes per row
  constexpr int R = 256 / L;     // rows of a block at a time
  constexpr int U = 4;           // rows of a thread in flight
  const int heads = a.H + 2 * a.Hkv;
  const int l = threadIdx.x % L, t = blockIdx.x;
  const unsigned mask = L == 32 ? ~0u : (((1u << L) - 1u) << ((threadIdx.x & 31) / L * L));
  const int slot = a.slots[t], pos = a.positions ? a.positions[t] : 0;
  const bool rope = a.cos_t != nullptr;
  const bool fits = slot < a.slots_max && (!rope || (pos >= 0 && pos < a.max_pos));
  if (!fits && blockIdx.y == 0 && threadIdx.x == 0 && a.bad) atomicAdd(a.bad, 1);
  const bool keep = fits && slot >= 0;
  float4 c = make_float4(1.f, 1.f, 1.f, 1.f), s = make_float4(0.f, 0.f, 0.f, 0.f);
  if (rope && fits) {
    c = *reinterpret_cast<const float4*>(a.cos_t + (int64_t)pos * (D / 2) + 4 * l);
    s = *reinterpret_cast<const float4*>(a.sin_t + (int64_t)pos * (D / 2) + 4 * l);
  }
  const int blk = keep ? slot / a.block : 0, in = keep ? slot - blk * a.block : 0;
  const int h0 = blockIdx.y * (R * turns) + threadIdx.x / L, h1 = min(heads, (int)(blockIdx.y + 1) * (R * turns));
#pragma unroll 1
  for (int hb = h0; hb < h1; hb += R * U) {
    float4 xs[U], ys[U];
#pragma unroll
    for (int k = 0; k < U; k++) {
      const int hh = hb + R * k;
      xs[k] = ys[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (hh >= h1 || (hh >= a.H ? !keep : !fits)) continue;
      const float* src = hh < a.H ? a.q + t * a.q_stride + hh * D
                         : hh < a.H + a.Hkv ? a.k + t * a.k_stride + (hh - a.H) * D
                                            : a.v + t * a.v_stride + (hh - a.H - a.Hkv) * D;
      xs[k] = load4<VEC>(src + 4 * l);
      ys[k] = load4<VEC>(src + D / 2 + 4 * l);
    }
#pragma unroll
    for (int k = 0; k < U; k++) {
      const int hh = hb + R * k;
      if (hh >= h1) continue;
      const bool is_q = hh < a.H, is_v = hh >= a.H + a.Hkv;
      if (!is_q && !keep) continue;
      float4 x = xs[k], y = ys[k];
      if (!is_v && rope) {
        const float4 x0 = x, y0 = y;
#define TB_TURN(e)                                             \
  x.e = __fsub_rn(__fmul_rn(x0.e, c.e), __fmul_rn(y0.e, s.e)); \
  y.e = __fadd_rn(__fmul_rn(x0.e, s.e), __fmul_rn(y0.e, c.e));
        TB_TURN(x) TB_TURN(y) TB_TURN(z) TB_TURN(w)
#undef TB_TURN
      }
      if (is_q) {
        float* o = a.q_out + ((int64_t)t * a.H + hh) * D + 4 * l;
        *reinterpret_cast<float4*>(o) = x;
        *reinterpret_cast<float4*>(o + D / 2) = y;
        continue;
      }
      const int head = is_v ? hh - a.H - a.Hkv : hh - a.H;
      float mn = fminf(fminf(fminf(x.x, x.y), fminf(x.z, x.w)), fminf(fminf(y.x, y.y), fminf(y.z, y.w)));
      float mx = fmaxf(fmaxf(fmaxf(x.x, x.y), fmaxf(x.z, x.w)), fmaxf(fmaxf(y.x, y.y), fmaxf(y.z, y.w)));
      // fminf and fmaxf drop NaNs: a product with 0 keeps them, and infinities
      const float odd =
          0.f * x.x + 0.f * x.y + 0.f * x.z + 0.f * x.w + 0.f * y.x + 0.f * y.y + 0.f * y.z + 0.f * y.w;
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) {
        mn = fminf(mn, __shfl_xor_sync(mask, mn, o));
        mx = fmaxf(mx, __shfl_xor_sync(mask, mx, o));
      }
      const bool finite = (__ballot_sync(mask, odd == 0.f) & mask) == mask;
      const uint32_t word = finite ? kv4_word(mn, mx) : kKv4NanWord;
      const float scale = kv4_scale(word), zero = kv4_zero(word);
      const uint32_t cx = kv4_code(x.x, scale, zero) | kv4_code(x.y, scale, zero) << 4 |
                          kv4_code(x.z, scale, zero) << 8 | kv4_code(x.w, scale, zero) << 12;
      const uint32_t cy = kv4_code(y.x, scale, zero) | kv4_code(y.y, scale, zero) << 4 |
                          kv4_code(y.z, scale, zero) << 8 | kv4_code(y.w, scale, zero) << 12;
      uint8_t* tile = a.pages + (((int64_t)blk * a.Hkv + head) * (a.block / kKv4Tile) + in / kKv4Tile) *
                                    (int64_t)kv4_tile_bytes(D);
      const int r = in % kKv4Tile, part = is_v;
      uint16_t* codes = reinterpret_cast<uint16_t*>(tile + kv4_codes_off(D, part) + r * (D / 2));
      codes[l] = (uint16_t)cx;
      codes[D / 8 + l] = (uint16_t)cy;
      if (l == 0) reinterpret_cast<uint32_t*>(tile + kv4_words_off(D, part))[r] = word;
    }
  }
}

// Rows by slot back as fp32: a row of a slot outside the cache (padding is
// -1) reads as zero.
template <int D>
__global__ void __launch_bounds__(256) kv4_read_kernel(float* k, float* v, const uint8_t* pages, const int32_t* slots,
                                                       int T, int Hkv, int block, int64_t slots_max) {
  constexpr int L = D / 8;
  const int l = threadIdx.x % L;
  const int64_t rows = (int64_t)T * Hkv * 2;
  for (int64_t row = (blockIdx.x * (int64_t)blockDim.x + threadIdx.x) / L; row < rows;
       row += (int64_t)gridDim.x * blockDim.x / L) {
    const int part = (int)(row & 1);
    const int64_t th = row >> 1;
    const int t = (int)(th / Hkv), head = (int)(th - (int64_t)t * Hkv);
    const int slot = slots[t];
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f), y = x;
    if (slot >= 0 && slot < slots_max) {
      const int blk = slot / block, in = slot - blk * block;
      const uint8_t* tile = pages + (((int64_t)blk * Hkv + head) * (block / kKv4Tile) + in / kKv4Tile) *
                                        (int64_t)kv4_tile_bytes(D);
      const int r = in % kKv4Tile;
      const uint16_t* codes = reinterpret_cast<const uint16_t*>(tile + kv4_codes_off(D, part) + r * (D / 2));
      const uint32_t w = reinterpret_cast<const uint32_t*>(tile + kv4_words_off(D, part))[r];
      const float s = kv4_scale(w), z = kv4_zero(w);
      const uint32_t cx = codes[l], cy = codes[D / 8 + l];
      x = make_float4(kv4_value(cx & 15, s, z), kv4_value(cx >> 4 & 15, s, z), kv4_value(cx >> 8 & 15, s, z),
                      kv4_value(cx >> 12, s, z));
      y = make_float4(kv4_value(cy & 15, s, z), kv4_value(cy >> 4 & 15, s, z), kv4_value(cy >> 8 & 15, s, z),
                      kv4_value(cy >> 12, s, z));
    }
    float* o = (part ? v : k) + th * D + 4 * l;
    *reinterpret_cast<float4*>(o) = x;
    *reinterpret_cast<float4*>(o + D / 2) = y;
  }
}

template <int D>
void append_launch(const AppendArgs& a, bool vec, cudaStream_t st) {
  const int rows = 256 / (D / 8), heads = a.H + 2 * a.Hkv, groups = (heads + rows - 1) / rows;
  // Few tokens: a block per group of rows, for the most loads in flight; many: a
  // block per token, which reads RoPE's factors once.  80 rows a token, the one
  // and the other: 64 tokens 5.4 and 5.7 us, 128 6.5 and 5.9, 8192 226 and 129.
  const int turns = (int64_t)a.T * groups <= 3 * sm_count() ? 1 : groups;
  const dim3 grid((unsigned)a.T, (unsigned)((groups + turns - 1) / turns));
  if (vec)
    kv4_append_kernel<D, true><<<grid, 256, 0, st>>>(a, turns);
  else
    kv4_append_kernel<D, false><<<grid, 256, 0, st>>>(a, turns);
}

// CTAs of 256 threads for `rows` rows of D / 8 lanes.
unsigned row_grid(int64_t rows, int64_t D) {
  const int64_t n = (rows * (D / 8) + 255) / 256;
  return (unsigned)(n < 65536 ? n : 65536);
}

bool kv4_shape_ok(int64_t Hkv, int64_t D, int64_t block_size, int64_t num_blocks) {
  return Hkv > 0 && Hkv <= 65535 && D > 0 && block_size > 0 && block_size % kKv4Tile == 0 && num_blocks > 0 &&
         block_size <= INT_MAX && num_blocks <= INT_MAX && num_blocks * block_size <= INT_MAX;
}
bool kv4_dim_ok(int64_t D) { return D == 32 || D == 64 || D == 128; }

}  // namespace
}  // namespace tb

extern "C" size_t tb_kv4_tile_bytes(int64_t D) { return tb::kv4_dim_ok(D) ? (size_t)tb::kv4_tile_bytes((int)D) : 0; }

extern "C" tb_status_t tb_kv4_plan(int32_t* q_start, int32_t* seq_lens, int32_t* positions, int32_t* slots,
                                   int32_t* free_count_out, int32_t* bad_count, int32_t* block_table,
                                   int32_t* free_list, const int32_t* free_count, const int32_t* held_lens,
                                   const int32_t* ctx_lens, const int32_t* new_lens, int64_t B, int64_t T,
                                   int64_t max_blocks, int64_t num_blocks, int64_t block_size, tb_stream_t stream) {
  TB_INJECT("tb_kv4_plan");
  TB_REQUIRE(B >= 0 && T >= 0 && max_blocks >= 0 && num_blocks > 0 && block_size > 0);
  TB_REQUIRE(block_size % tb::kKv4Tile == 0 && T <= INT_MAX - (1 << 20) && max_blocks <= INT_MAX);
  TB_REQUIRE(num_blocks <= INT_MAX && block_size <= INT_MAX && num_blocks * block_size <= INT_MAX);
  TB_REQUIRE(q_start && free_count_out && free_list && free_count && free_count != free_count_out);
  TB_REQUIRE(B == 0 || (seq_lens && held_lens && ctx_lens && new_lens && (max_blocks == 0 || block_table)));
  TB_REQUIRE(T == 0 || (positions && slots));
  if (B > tb::kPlanMaxB) return TB_ERROR_NOT_SUPPORTED;
  const tb::PlanArgs a{q_start,    seq_lens,  positions,  slots,    free_count_out, bad_count,       block_table,
                       free_list,  free_count, held_lens, ctx_lens, new_lens,       (int)B,          (int)T,
                       (int)max_blocks, (int)num_blocks, (int)block_size};
  const size_t smem = 3 * (size_t)(B + 1) * sizeof(int32_t);
  static std::atomic<uint64_t> ready{0};
  if (smem > 40 * 1024)
    TB_TRY(tb::allow_smem(reinterpret_cast<const void*>(tb::kv4_plan_kernel),
                          3 * (size_t)(tb::kPlanMaxB + 1) * sizeof(int32_t), ready));
  // one token (or moved page) per thread up to a CTA on every SM
  int64_t grid = (T + tb::kPlanThreads - 1) / tb::kPlanThreads;
  if (grid < 1) grid = 1;
  if (grid > tb::sm_count()) grid = tb::sm_count();
  tb::kv4_plan_kernel<<<(unsigned)grid, tb::kPlanThreads, smem, (cudaStream_t)stream>>>(a);
  return tb::check_launch("kv4_plan_kernel");
}

extern "C" tb_status_t tb_kv4_append_rope_f32(uint8_t* pages, float* q_out, const float* q, const float* k,
                                              const float* v, int64_t q_stride, int64_t k_stride, int64_t v_stride,
                                              const float* cos_t, const float* sin_t, const int32_t* positions,
                                              const int32_t* slots, int32_t* bad_count, int64_t T, int64_t H,
                                              int64_t Hkv, int64_t D, int64_t block_size, int64_t num_blocks,
                                              int64_t max_seq, tb_stream_t stream) {
  TB_INJECT("tb_kv4_append_rope_f32");
  TB_REQUIRE(T >= 0 && T <= INT_MAX && H >= 0 && H <= 65535 && tb::kv4_shape_ok(Hkv, D, block_size, num_blocks));
  if (!tb::kv4_dim_ok(D)) return TB_ERROR_NOT_SUPPORTED;
  TB_REQUIRE((q == nullptr) == (q_out == nullptr) && (cos_t == nullptr) == (sin_t == nullptr));
  if (T == 0) return TB_SUCCESS;
  TB_REQUIRE(pages && k && v && slots && (!cos_t || (positions && max_seq > 0)));
  TB_REQUIRE(k_stride >= Hkv * D && v_stride >= Hkv * D && (!q || (H > 0 && q_stride >= H * D)));
  TB_REQUIRE(tb::aligned(pages, 16) && tb::aligned(q_out, 16) && tb::aligned(cos_t, 16) && tb::aligned(sin_t, 16));
  const int Hq = q ? (int)H : 0;
  const bool vec = tb::aligned(q, 16) && tb::aligned(k, 16) && tb::aligned(v, 16) && k_stride % 4 == 0 &&
                   v_stride % 4 == 0 && (!q || q_stride % 4 == 0);
  const tb::AppendArgs a{pages,     q_out,    q,        k,        v,
                         cos_t,     sin_t,    positions, slots,   bad_count,
                         q_stride,  k_stride, v_stride, num_blocks * block_size,
                         (int)T,    Hq,       (int)Hkv, (int)block_size, (int)(max_seq < INT_MAX ? max_seq : INT_MAX)};
  cudaStream_t st = (cudaStream_t)stream;
  if (D == 128)
    tb::append_launch<128>(a, vec, st);
  else if (D == 64)
    tb::append_launch<64>(a, vec, st);
  else
    tb::append_launch<32>(a, vec, st);
  return tb::check_launch("kv4_append_kernel");
}

extern "C" tb_status_t tb_kv4_read_f32(float* k, float* v, const uint8_t* pages, const int32_t* slots, int64_t T,
                                       int64_t Hkv, int64_t D, int64_t block_size, int64_t num_blocks,
                                       tb_stream_t stream) {
  TB_INJECT("tb_kv4_read_f32");
  TB_REQUIRE(T >= 0 && T <= INT_MAX && tb::kv4_shape_ok(Hkv, D, block_size, num_blocks));
  if (!tb::kv4_dim_ok(D)) return TB_ERROR_NOT_SUPPORTED;
  if (T == 0) return TB_SUCCESS;
  TB_REQUIRE(k && v && pages && slots);
  TB_REQUIRE(tb::aligned(pages, 16) && tb::aligned(k, 16) && tb::aligned(v, 16));
  const unsigned grid = tb::row_grid(T * Hkv * 2, D);
  const int64_t most = num_blocks * block_size;
  cudaStream_t st = (cudaStream_t)stream;
  if (D == 128)
    tb::kv4_read_kernel<128><<<grid, 256, 0, st>>>(k, v, pages, slots, (int)T, (int)Hkv, (int)block_size, most);
  else if (D == 64)
    tb::kv4_read_kernel<64><<<grid, 256, 0, st>>>(k, v, pages, slots, (int)T, (int)Hkv, (int)block_size, most);
  else
    tb::kv4_read_kernel<32><<<grid, 256, 0, st>>>(k, v, pages, slots, (int)T, (int)Hkv, (int)block_size, most);
  return tb::check_launch("kv4_read_kernel");
}
