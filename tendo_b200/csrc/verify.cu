// verify.cu — verification of drafted tokens against the target model's
// probabilities (speculative sampling), from uniforms that the caller gives.
//
// Draft i of a request is accepted while u_i q_i(x_i) < p_i(x_i); at the first
// refusal r the replacement is drawn from max(0, p_r - q_r), and with every
// draft accepted the next token is drawn from p_n.  The draw is an inverse CDF
// over fixed-point weights floor(w 2^36) whose sums are 64-bit integers: exact
// in any order, so the token does not depend on how the row is split.
//
// One cluster of CTAs per request: each sums its slice of the row, the sums
// meet in distributed shared memory, and the CTA whose slice holds the target
// narrows it down: its warps take the owning warp's span in pieces, and the
// owner of the piece walks it.  The row is read from memory once (what is read
// again is in L1 or L2): 64 requests with a vocabulary of 128000 take 20 us, 3.3
// TB/s of both rows, bound by memory latency (a CTA reads two slices of 128 KB
// and then waits for its cluster); one request 5 to 7 us.
#include <limits.h>

#include <cooperative_groups.h>

#include "common.cuh"

namespace cg = cooperative_groups;

namespace tb {
namespace {

constexpr int kMaxCluster = 8;
constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
typedef unsigned long long u64;

struct VerifyArgs {
  int64_t* tokens;
  int32_t* accepted;
  const float *p, *q, *u;
  const int64_t* draft;
  const int32_t* lens;
  int32_t* bad;
  int64_t p_req, p_row, q_req, q_row;  // strides in elements
  int K, V;
};

__device__ __forceinline__ u64 fixed(float w) {
  return (u64)(long long)(fminf(fmaxf(w, 0.f), 1.f) * 68719476736.f);  // NaN counts as 0
}

// Weights of up to four neighbours from v on (v < end).
template <bool VEC>
__device__ __forceinline__ void weights(const float* p, const float* q, int64_t removed, int v, int end, u64 (&w)[4]) {
  float x[4] = {0.f, 0.f, 0.f, 0.f}, y[4] = {0.f, 0.f, 0.f, 0.f};
  if (VEC) {
    const float4 f = *reinterpret_cast<const float4*>(p + v);
    x[0] = f.x, x[1] = f.y, x[2] = f.z, x[3] = f.w;
    if (q) {
      const float4 h = *reinterpret_cast<const float4*>(q + v);
      y[0] = h.x, y[1] = h.y, y[2] = h.z, y[3] = h.w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; j++)
      if (v + j < end) {
        x[j] = p[v + j];
        if (q) y[j] = q[v + j];
      }
  }
#pragma unroll
  for (int j = 0; j < 4; j++) w[j] = v + j >= end || v + j == removed ? 0 : fixed(x[j] - y[j]);
}

__device__ __forceinline__ u64 warp_sum64(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}

template <bool VEC>
__global__ void __launch_bounds__(kThreads, 2) verify_kernel(VerifyArgs a) {
  cg::cluster_group cl = cg::this_cluster();
  const int cluster = (int)cl.num_blocks(), b = blockIdx.x / cluster, rank = (int)cl.block_rank();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  __shared__ u64 wsum[kWarps], psum[kWarps];
  __shared__ u64 csum[2];  // one per pass: a peer may still read the first
  __shared__ int first_no;
  const int n = a.lens ? min(max(a.lens[b], 0), a.K) : a.K;
  if (tid == 0) first_no = n;
  __syncthreads();
  const float* P = a.p + b * a.p_req;
  const float* Q = a.q ? a.q + b * a.q_req : nullptr;
  const float* U = a.u + (int64_t)b * (a.K + 1);
  const int64_t* X = a.draft + (int64_t)b * a.K;
  for (int i = tid; i < n; i += kThreads) {
    const int64_t x = X[i];
    const bool in = x >= 0 && x < a.V;
    if (!in && rank == 0 && a.bad) atomicAdd(a.bad, 1);
    const bool yes = in && __fmul_rn(U[i], Q ? Q[i * a.q_row + x] : 1.f) < P[i * a.p_row + x];
    if (!yes) atomicMin(&first_no, i);
  }
  __syncthreads();
  const int r = first_no;
  if (rank == 0) {
    for (int j = tid; j <= a.K; j += kThreads)
      if (j != r) a.tokens[(int64_t)b * (a.K + 1) + j] = j < r ? X[j] : -1;
    if (tid == 0) a.accepted[b] = r;
  }
  const float* pr = P + r * a.p_row;
  const float* qr = Q && r < n ? Q + r * a.q_row : nullptr;
  // without draft probabilities a draft was certain: the rest is p without it
  int64_t removed = !Q && r < n ? X[r] : -1;
  const float u = U[a.K];
  const u64 m = (u64)(long long)(fminf(fmaxf(u, 0.f), 1.f) * 16777216.f);
  // spans in vocabulary order: CTA rank, then warp
  const int slice = ((a.V + cluster - 1) / cluster + 3) / 4 * 4;
  const int span = ((slice + kWarps - 1) / kWarps + 3) / 4 * 4;
  const int c0 = rank * slice, c1 = min(a.V, c0 + slice);
  const int v0 = min(c0 + warp * span, c1), v1 = min(v0 + span, c1);
#pragma unroll 1
  for (int pass = 0; pass < 2; pass++) {
    auto sum_of = [&](int from, int to) {
      u64 mine = 0;
#pragma unroll 4
      for (int v = from + 4 * lane; v < to; v += 128) {
        u64 w[4];
        weights<VEC>(pr, qr, removed, v, to, w);
        mine += (w[0] + w[1]) + (w[2] + w[3]);
      }
      return warp_sum64(mine);
    };
    const u64 mine = sum_of(v0, v1);
    if (lane == 0) wsum[warp] = mine;
    __syncthreads();
    if (tid == 0) {
      u64 s = 0;
      for (int w = 0; w < kWarps; w++) s += wsum[w];
      csum[pass] = s;
    }
    cl.sync();
    u64 before = 0, total = 0;
    for (int c = 0; c < cluster; c++) {
      const u64 s = *cl.map_shared_rank(&csum[pass], c);
      if (c < rank) before += s;
      total += s;
    }
    if (total == 0 && pass == 0) {
      // nothing left of p - q (they are equal up to rounding): draw from p
      qr = nullptr;
      removed = -1;
      __syncthreads();
      continue;
    }
    if (total == 0) {  // p is empty too
      if (rank == 0 && tid == 0) {
        a.tokens[(int64_t)b * (a.K + 1) + r] = 0;
        if (a.bad) atomicAdd(a.bad, 1);
      }
      break;
    }
    // floor(u total) without a 128-bit product; u = m / 2^24, below total
    u64 target = (total >> 24) * m + (((total & 0xffffffu) * m) >> 24);
    if (target >= total) target = total - 1;
    if (target < before || target - before >= csum[pass]) break;  // another CTA's
    int owner = 0;
    while (target - before >= wsum[owner]) before += wsum[owner++];
    // the owner's span in pieces for the CTA's warps
    const int s0 = min(c0 + owner * span, c1), s1 = min(s0 + span, c1);
    const int piece = ((s1 - s0 + kWarps - 1) / kWarps + 3) / 4 * 4;
    const u64 part = sum_of(min(s0 + warp * piece, s1), min(s0 + (warp + 1) * piece, s1));
    if (lane == 0) psum[warp] = part;
    __syncthreads();
    owner = 0;
    while (target - before >= psum[owner]) before += psum[owner++];
    if (warp == owner) {
      const int p0 = min(s0 + owner * piece, s1), p1 = min(p0 + piece, s1);
      u64 run = before;
      for (int v = p0; v < p1; v += 128) {
        const int at = v + 4 * lane;
        u64 w[4] = {0, 0, 0, 0};
        if (at < p1) weights<VEC>(pr, qr, removed, at, p1, w);
        const u64 sum = (w[0] + w[1]) + (w[2] + w[3]);
        u64 inc = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const u64 t = __shfl_up_sync(~0u, inc, o);
          if (lane >= o) inc += t;
        }
        const unsigned past = __ballot_sync(~0u, run + inc > target);
        if (past) {
          if (lane == __ffs(past) - 1) {
            u64 e = run + inc - sum;
            int j = 0;
            while (j < 3 && e + w[j] <= target) e += w[j++];
            a.tokens[(int64_t)b * (a.K + 1) + r] = at + j;
          }
          break;
        }
        run += __shfl_sync(~0u, inc, 31);
      }
    }
    break;
  }
  cl.sync();  // no CTA leaves while a peer reads its sum
}

}  // namespace
}  // namespace tb

extern "C" tb_status_t tb_verify_draft_f32(int64_t* tokens, int32_t* accepted, const float* target_probs,
                                           int64_t target_req_stride, int64_t target_row_stride,
                                           const int64_t* draft_tokens, const float* draft_probs,
                                           int64_t draft_req_stride, int64_t draft_row_stride,
                                           const int32_t* draft_lens, const float* uniforms, int32_t* bad_count,
                                           int64_t B, int64_t K, int64_t V, tb_stream_t stream) {
  TB_INJECT("tb_verify_draft_f32");
  TB_REQUIRE(B >= 0 && K >= 0 && V > 0 && K <= INT_MAX - 1024 && V <= INT_MAX - 1024);
  TB_REQUIRE(B <= INT_MAX / tb::kMaxCluster);
  // 64-bit sums of weights below 2^36 + 1
  if (V > (1 << 26)) return TB_ERROR_NOT_SUPPORTED;
  if (B == 0) return TB_SUCCESS;
  TB_REQUIRE(tokens && accepted && target_probs && uniforms && (K == 0 || draft_tokens));
  TB_REQUIRE(target_row_stride >= V && target_req_stride >= 0);
  TB_REQUIRE(!draft_probs || (draft_row_stride >= V && draft_req_stride >= 0));
  if (K == 0) draft_probs = nullptr;
  const tb::VerifyArgs a{tokens,       accepted,  target_probs,      draft_probs,       uniforms,
                         draft_tokens, draft_lens, bad_count,        target_req_stride, target_row_stride,
                         draft_req_stride, draft_row_stride, (int)K, (int)V};
  const bool vec = V % 4 == 0 && tb::aligned(target_probs, 16) && target_req_stride % 4 == 0 &&
                   target_row_stride % 4 == 0 &&
                   (!draft_probs || (tb::aligned(draft_probs, 16) && draft_req_stride % 4 == 0 &&
                                     draft_row_stride % 4 == 0));
  // The largest cluster that keeps every CTA resident.  Two fit an SM, but parts
  // of the chip have no place for a whole cluster: of 7/4 an SM all were.  8, 4, 2
  // and 1 CTAs: 16 requests of 128000 10.6, 11.6, 15.3, 22.2 us; 36 of 32000 12.0,
  // 8.8, 8.1, 9.4; 64 of 128000 25.9, 19.8, 23.2, 32.9.
  int cluster = tb::kMaxCluster;
  while (cluster > 1 && B * cluster > 7 * tb::sm_count() / 4) cluster /= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(B * cluster));
  cfg.blockDim = dim3(tb::kThreads);
  cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (vec)
    TB_CUDA(cudaLaunchKernelEx(&cfg, tb::verify_kernel<true>, a));
  else
    TB_CUDA(cudaLaunchKernelEx(&cfg, tb::verify_kernel<false>, a));
  return tb::check_launch("verify_kernel");
}
