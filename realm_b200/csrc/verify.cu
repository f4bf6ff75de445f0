// Verification of drafted tokens. Request r has the rows [a, b): row i < b - 1 is the target's
// distribution p_i before draft d_i, which was drawn from q_i (or not drawn: q_i(d_i) = 1).
//   accepted while u_i q_i(d_i) < p_i(d_i)
//   the first other row j draws from max(p_j - q_j, 0); after all, row b - 1 from p
// so that the tokens are distributed as the target's own. Both tests and differences are
// exact: products of fp32 values in 64 bits, and p - q as F = floor((p - q) 2^44) in a 64-bit
// integer (2^18 of them fit), whose sums depend on no order. The draw is the first index whose
// running sum exceeds floor(u sum F).
//
// One cluster a request. Each CTA finds row j by itself (a few gathered values), each warp sums
// its contiguous share of the row and remembers the sum of each batch of 512 elements, the cluster adds up, and the one
// warp in whose share the target falls goes over its batch once more: the row is read once.
//
// Rows of device memory may be those of two requests (offsets that fell between them), and tokens may be drafts: then one
// request writes drafts that another reads. What is drawn there is left open, but CTAs that meet different drafts take
// the same turns: a CTA's threads share one reading of the refused draft, and whether there is a second turn goes with the sums.
//
// Bound by latency: offsets, drafts, their probabilities, the row, the exchange, the share again, one after the other.
// 64 requests of 1 to 9 rows of 151937 22.5 us (63 MB read: 2.8 TB/s; 30 us when the share was gone over vector by vector,
// 37 when the sums were too); one request of 7 rows of 32000 the call itself, 9 us. Rows of which a looked-up draft is
// taken out, and p and q that lie unlike, go vector by vector, one on its way a lane: the same requests looked up 35 us.
#include <cooperative_groups.h>

#include <algorithm>

#include "common.cuh"
#include "filter.cuh"
#include "verify.cuh"

namespace cg = cooperative_groups;

namespace rb {

namespace {

constexpr int kVT = 256, kVW = kVT / 32;
constexpr int kVMaxCluster = 8;
constexpr int kDeep = 4, kBatch = 32 * kDeep;                     // vectors of 4 elements a lane, a warp takes at a time
constexpr int kBatches = (kFilterMaxVocab / 4 / kVW + kBatch) / kBatch + 1;  // of a warp's share, at most
constexpr uint32_t kNone = 0xffffffffu;
using u64 = unsigned long long;

__device__ __forceinline__ float unit(float p) { return fminf(fmaxf(p, 0.f), 1.f); }  // fmaxf: 0 for a NaN

__device__ __forceinline__ u64 weight(float p, float q) {
  const double r = (double)unit(p) - (double)unit(q);
  return r > 0.0 ? (u64)(r * 0x1p44) : 0;
}
__device__ __forceinline__ u64 warp_total(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ u64 warp_incl(u64 v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  return v;
}

// One row of the draw. Vectors of 4 elements, the first one up to 3 elements before the row;
// p and q lie alike in them where VQ holds, else q is read by elements.
struct DrawRow {
  const float *p, *q;  // q null: 0 everywhere but at skip, where the weight is 0
  int vocab, mis;
  uint32_t skip;
  bool same;
  __device__ __forceinline__ void weights(int v, u64 (&w)[4]) const {
    const int i = v * 4 - mis;
    float x[4], z[4] = {0.f, 0.f, 0.f, 0.f};
    if (i >= 0 && i + 4 <= vocab) {
      const float4 t = __ldg(reinterpret_cast<const float4*>(p + i));
      x[0] = t.x, x[1] = t.y, x[2] = t.z, x[3] = t.w;
      if (q) {
        if (same) {
          const float4 y = __ldg(reinterpret_cast<const float4*>(q + i));
          z[0] = y.x, z[1] = y.y, z[2] = y.z, z[3] = y.w;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) z[e] = __ldg(q + i + e);
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool in = i + e >= 0 && i + e < vocab;
        x[e] = in ? __ldg(p + i + e) : 0.f;
        if (q && in) z[e] = __ldg(q + i + e);
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = (uint32_t)(i + e) == skip ? 0 : weight(x[e], z[e]);
  }
};

__device__ __forceinline__ u64 vector(const DrawRow& row, int v) {
  u64 w[4];
  row.weights(v, w);
  return (w[0] + w[1]) + (w[2] + w[3]);
}

template <int N>
__global__ void __launch_bounds__(kVT) verify_kernel(const __grid_constant__ VerifyArgs a) {
  __shared__ u64 part[kVW];
  __shared__ u64 batch[kVW][kBatches];
  __shared__ u64 sums[2][kVMaxCluster];
  __shared__ uint32_t first, refused_draft;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = N > 1 ? (int)cg::this_cluster().block_rank() : 0, req = blockIdx.x / N;
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t r0 = a.offsets[req], r1 = a.offsets[req + 1];
  if (r0 >= r1 || r1 > (uint32_t)a.n_rows) {  // the whole cluster
    if (rank == 0 && tid == 0) a.accepted[req] = r0 == r1 && r1 <= (uint32_t)a.n_rows ? 0 : -1;
    return;
  }
  if (tid == 0) first = r1 - 1;
  if (N > 1) cg::this_cluster().barrier_arrive();
  __syncthreads();
  for (uint32_t b = r0; b < r1 - 1; b += kVT) {
    const uint32_t i = b + tid;
    bool refused = false;
    if (i < r1 - 1) {
      const uint32_t d = a.drafts[i];
      float p = 0.f, q = 1.f;
      if (d < (uint32_t)a.vocab) {
        p = unit(a.probs[(int64_t)i * a.ldp + d]);
        if (a.draft_probs) q = unit(a.draft_probs[(int64_t)i * a.ldq + d]);
      }
      refused = !((double)a.uniforms[i] * (double)q < (double)p);
      if (refused) atomicMin(&first, i);
    }
    if (__syncthreads_or(refused)) break;
  }
  const uint32_t at = first;
  const bool inner = at < r1 - 1;
  if (!a.draft_probs) {
    if (tid == 0) refused_draft = inner ? a.drafts[at] : kNone;
    __syncthreads();
  }
  DrawRow row;
  row.p = a.probs + (int64_t)at * a.ldp;
  row.q = inner && a.draft_probs ? a.draft_probs + (int64_t)at * a.ldq : nullptr;
  row.skip = a.draft_probs ? kNone : refused_draft;
  row.vocab = a.vocab;
  row.mis = (int)((reinterpret_cast<uintptr_t>(row.p) & 15) / 4);
  row.same = ((reinterpret_cast<uintptr_t>(row.p) ^ reinterpret_cast<uintptr_t>(row.q)) & 15) == 0;
  const int vecs = (a.vocab + row.mis + 3) / 4, share = (vecs + N - 1) / N, ours = (share + kVW - 1) / kVW;
  const int end = min(vecs, (rank + 1) * share), v0 = min(end, rank * share + warp * ours), v1 = min(end, v0 + ours);
  if (N > 1) cg::this_cluster().barrier_wait();  // every CTA of the cluster runs before its shared memory is written
  u64 total = 0, before = 0;
#pragma unroll 1
  for (int turn = 0; turn < 2; ++turn) {
    // whole vectors, a batch of kDeep of each row a lane on their way; what lies at the row's ends, or unlike in
    // p and q, by elements
    const bool alike = row.skip == kNone && (!row.q || row.same);
    const int f0 = row.mis > 0, f1 = (a.vocab + row.mis) / 4;
    u64 s = 0;
#pragma unroll 1
    for (int k = 0; v0 + k * kBatch < v1; ++k) {
      const int b = v0 + k * kBatch + lane;
      u64 here = 0;
      float4 x[kDeep], z[kDeep];
#pragma unroll
      for (int j = 0; j < kDeep; ++j) {
        const int v = b + 32 * j, i = v * 4 - row.mis;
        const bool whole = alike && v < v1 && v >= f0 && v < f1;
        x[j] = whole ? __ldg(reinterpret_cast<const float4*>(row.p + i)) : make_float4(0.f, 0.f, 0.f, 0.f);
        z[j] = whole && row.q ? __ldg(reinterpret_cast<const float4*>(row.q + i)) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
#pragma unroll
      for (int j = 0; j < kDeep; ++j)
        here += (weight(x[j].x, z[j].x) + weight(x[j].y, z[j].y)) + (weight(x[j].z, z[j].z) + weight(x[j].w, z[j].w));
#pragma unroll 1
      for (int v = b; v < v1 && v < b + kBatch; v += 32)
        if (!(alike && v >= f0 && v < f1)) here += vector(row, v);
      here = warp_total(here);
      if (lane == 0) batch[warp][k] = here;
      s += here;
    }
    if (lane == 0) part[warp] = s;
    __syncthreads();
    u64 mine = 0;
    before = 0;
#pragma unroll
    for (int w = 0; w < kVW; ++w) {
      if (w < warp) before += part[w];
      mine += part[w];
    }
    bool less = row.q || row.skip != kNone;  // something was taken off p
    if (N > 1) {
      constexpr u64 kLess = 1ull << 63;  // above all sums
      if (tid < N) *cg::this_cluster().map_shared_rank(&sums[turn][rank], tid) = mine | (less ? kLess : 0);
      cg::this_cluster().sync();
      total = 0;
      less = false;
#pragma unroll
      for (int c = 0; c < N; ++c) {
        const u64 s = sums[turn][c];
        if (c < rank) before += s & ~kLess;
        total += s & ~kLess;
        less |= s >= kLess;
      }
    } else {
      __syncthreads();  // part has been read
      total = mine;
    }
    // p nowhere above q (the same in every thread of the cluster): from p
    if (total || !less) break;
    row.q = nullptr;
    row.skip = kNone;
  }
  const u64 target = total ? [&] {
    const double x = (double)a.uniforms[r1 - 1] * (double)total;
    if (!(x > 0.0)) return (u64)0;
    return x < (double)total ? min((u64)x, total - 1) : total - 1;
  }() : 0;
  // the share that holds the target: exactly one warp's, as target < total
  if (total && before <= target && target < before + part[warp]) {
    u64 sum = before;
    int k = 0;  // the batch of the share that holds it
    for (int n = (v1 - v0 + kBatch - 1) / kBatch; k < n; k += 32) {
      const u64 here = k + lane < n ? batch[warp][k + lane] : 0, incl = warp_incl(here);
      const uint32_t past = __ballot_sync(0xffffffffu, target < sum + incl);
      if (past) {
        const int l = __ffs(past) - 1;
        sum += __shfl_sync(0xffffffffu, incl - here, l);
        k += l;
        break;
      }
      sum += __shfl_sync(0xffffffffu, incl, 31);
    }
    u64 here[kDeep];
#pragma unroll
    for (int j = 0; j < kDeep; ++j) {
      const int v = v0 + k * kBatch + 32 * j + lane;
      here[j] = v < v1 ? vector(row, v) : 0;
    }
#pragma unroll
    for (int j = 0; j < kDeep; ++j) {
      const u64 incl = warp_incl(here[j]);
      u64 run = sum + incl - here[j];
      if (run <= target && target < run + here[j]) {
        const int v = v0 + k * kBatch + 32 * j + lane;
        u64 w[4];
        row.weights(v, w);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (run <= target && target < run + w[e]) a.tokens[at] = (uint32_t)(v * 4 - row.mis + e);
          run += w[e];
        }
      }
      sum += __shfl_sync(0xffffffffu, incl, 31);
    }
  }
  if (rank) return;
  // drafts may be tokens: every CTA has read its own by now
  for (uint32_t i = r0 + tid; i < r1; i += kVT)
    if (i != at || !total) a.tokens[i] = i < at ? a.drafts[i] : kNone;
  if (tid == 0) a.accepted[req] = (int32_t)(at - r0);
}

template <int N>
cudaError_t launch(const VerifyArgs& a, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.n_requests * N));
  cfg.blockDim = dim3(kVT);
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = N;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, verify_kernel<N>, a);
}

}  // namespace

cudaError_t verify_launch(const VerifyArgs& a, int num_sms, cudaStream_t s) {
  const int n = std::min(4 * num_sms / a.n_requests, a.vocab / (4 * kVT));
  if (n >= 8) return launch<8>(a, s);
  if (n >= 4) return launch<4>(a, s);
  if (n >= 2) return launch<2>(a, s);
  return launch<1>(a, s);
}

}  // namespace rb
