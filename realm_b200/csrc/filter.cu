// Filtered sampling of logits rows of any vocabulary up to kFilterMaxVocab.
//
// With x the row after its repetition penalty, m = max x and t the temperature,
// a token's weight is w = exp(x/t - m/t) in fp32, held as W = floor(w 2^40) in a
// 64-bit integer: every sum of weights is exact, so neither the thresholds nor
// the draw depend on the order of the sums. Tokens rank by weight descending,
// then index ascending. Kept are
//   top-k   the first k ranks (0 < k < vocab),
//   min-p   those with w >= min_p (the first rank's w is 1),
//   top-p   of these, the ranks with less than floor(p sum W) before them,
// and the draw takes the first index whose running sum of kept W exceeds
// floor(u sum W). t < 1e-7 takes the first rank.
//
// A cluster of CTAs holds one row in shared memory, each CTA a contiguous share
// cut into one chunk per thread. Thresholds come from a radix walk over the bits
// of w in three digits of ten bits, each one histogram (counts and sums) that the
// cluster adds up through distributed shared memory.
#include <cooperative_groups.h>

#include "common.cuh"
#include "filter.cuh"

namespace cg = cooperative_groups;

namespace rb {

namespace {

constexpr int kFT = 1024, kFW = kFT / 32;
constexpr int kBins = 1024;       // ten bits of w a pass: w <= 1 has 30 significant bits
constexpr int kMaxCluster = 8;
constexpr double kFix = 1099511627776.0;  // 2^40
using u64 = unsigned long long;

struct FilterShared {
  uint32_t cnt[2][kBins];
  u64 sum[2][kBins];
  u64 xch[2][kMaxCluster];  // one value of every CTA of the cluster
  u64 red[kFW];
  uint32_t redc[kFW];
  u64 out_a, out_b;
  uint32_t out_bin, out_cnt;
};

__device__ __forceinline__ u64 fix(float w) { return (u64)((double)w * kFix); }

__device__ __forceinline__ u64 warp_sum(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ u64 warp_max(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const u64 x = __shfl_xor_sync(0xffffffffu, v, o);
    v = x > v ? x : v;
  }
  return v;
}

template <bool MAX>
__device__ u64 block_reduce(u64 v, FilterShared& s) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  v = MAX ? warp_max(v) : warp_sum(v);
  __syncthreads();
  if (lane == 0) s.red[w] = v;
  __syncthreads();
  v = s.red[lane];
  return MAX ? warp_max(v) : warp_sum(v);
}

// exclusive prefix in thread order, and the block's total
__device__ u64 block_scan(u64 v, FilterShared& s, u64& total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  u64 x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) s.red[w] = x;
  __syncthreads();
  const u64 t = s.red[lane];
  u64 incl = t;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  total = __shfl_sync(0xffffffffu, incl, 31);
  return __shfl_sync(0xffffffffu, incl - t, w) + x - v;
}

// Every CTA's value to every CTA; slot alternates, so that one barrier a call does.
struct Cluster {
  cg::cluster_group g;
  FilterShared& s;
  int n, rank, turn = 0;
  __device__ Cluster(FilterShared& sh) : g(cg::this_cluster()), s(sh), n(g.num_blocks()), rank(g.block_rank()) {}
  __device__ const u64* share(u64 v) {
    u64* mine = s.xch[turn & 1];
    if ((int)threadIdx.x < n) g.map_shared_rank(mine, threadIdx.x)[rank] = v;
    ++turn;
    g.sync();
    return mine;
  }
};

__host__ __device__ inline int share_len(int V, int n) { return (V + n - 1) / n; }
__host__ __device__ inline int chunk_len(int S) { return (S + kFT - 1) / kFT; }
// an odd stride between the threads' chunks: a warp that walks its chunks in step meets 32 banks
__host__ __device__ inline int chunk_stride(int C) { return C | 1; }

// The walk over the digits. Among elements with bits <= cap (cap_eq of those equal
// to it, by index; only their number matters here) finds the largest threshold T
//   by count: so that `want` elements rank at or before T's last kept tie,
//   by sum:   so that the sum ranked before a kept element is below `want`.
// Returns T, the ties to keep, and the count and sum strictly above T.
struct Cut {
  uint32_t bits, ties;
  u64 above;  // sum of W above bits
};

template <bool COUNT>
__device__ Cut radix_cut(const float* sc, int n, const Cut& top, u64 want, Cluster& cl) {
  FilterShared& s = cl.s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint32_t pre = 0;
  u64 acc_s = 0, acc_c = 0;
  for (int pass = 2; pass >= 0; --pass) {
    const int turn = cl.turn & 1;
    s.cnt[turn][tid] = 0;
    s.sum[turn][tid] = 0;
    __syncthreads();
    const int sh = 10 * pass;
    const uint32_t hmask = pass == 2 ? 0u : 0xffffffffu << (sh + 10);
    for (int i = 0; i < n; ++i) {
      const uint32_t b = __float_as_uint(sc[i]);
      if (b && (b & hmask) == pre) {
        atomicAdd(&s.cnt[turn][(b >> sh) & 1023u], 1u);
        atomicAdd(&s.sum[turn][(b >> sh) & 1023u], fix(sc[i]));
      }
    }
    cl.g.sync();
    uint32_t c = 0;
    u64 w = 0;
    // thread t owns bin 1023 - t: prefixes in thread order run from the largest weight down
    const int bin = kBins - 1 - tid;
    for (int r = 0; r < cl.n; ++r) {
      c += cl.g.map_shared_rank(&s.cnt[turn][0], r)[bin];
      w += cl.g.map_shared_rank(&s.sum[turn][0], r)[bin];
    }
    u64 tot_s, tot_c;
    const u64 above_c = block_scan(c, s, tot_c) + acc_c;
    const u64 above_s = block_scan(w, s, tot_s) + acc_s;
    // the last bin, going down, that still holds a kept element
    const bool has = c > 0 && (COUNT ? above_c < want : above_s < want);
    const unsigned any = __ballot_sync(0xffffffffu, has);
    __syncthreads();
    if (lane == 0) s.redc[warp] = any;
    __syncthreads();
    int pick = 0;
    for (int q = 0; q < kFW; ++q)
      if (s.redc[q]) pick = q * 32 + 31 - __clz(s.redc[q]);
    if (tid == pick) {
      s.out_bin = (uint32_t)bin;
      s.out_a = above_c;
      s.out_b = above_s;
      s.out_cnt = c;
    }
    __syncthreads();
    pre |= s.out_bin << sh;
    acc_c = s.out_a;
    acc_s = s.out_b;
    ++cl.turn;
  }
  Cut r;
  r.bits = pre;
  r.above = acc_s;
  const uint32_t eq = s.out_cnt;
  if (COUNT) {
    const u64 left = want > acc_c ? want - acc_c : 0;
    r.ties = left < eq ? (uint32_t)left : eq;
  } else {
    const u64 tq = fix(__uint_as_float(pre));
    u64 ties = eq;
    if (tq) {
      const u64 k = want > acc_s ? (want - acc_s + tq - 1) / tq : 0;  // j-th tie kept while above + j tq < want
      ties = k < eq ? k : eq;
    }
    r.ties = (uint32_t)ties;
  }
  if (r.bits == top.bits && r.ties > top.ties) r.ties = top.ties;
  return r;
}

template <class T>
__global__ void __launch_bounds__(kFT) filter_kernel(const __grid_constant__ FilterArgs a) {
  extern __shared__ float sv[];
  __shared__ FilterShared s;
  Cluster cl(s);
  const int tid = threadIdx.x;
  cl.g.sync();  // every CTA of the cluster runs before its shared memory is written
  const int row = blockIdx.x / cl.n;
  rb_sampling_filter p = a.params[row];
  p.min_p = fminf(p.min_p, 1.f);  // the first rank always stays
  const int V = a.vocab, S = share_len(V, cl.n), C = chunk_len(S), CS = chunk_stride(C);
  const int base = cl.rank * S, len = max(0, min(S, V - base));
  const T* lg = reinterpret_cast<const T*>(a.logits) + (size_t)row * a.ld + base;
  for (int i = tid; i < len; i += kFT) {
    float x;
    if constexpr (sizeof(T) == 2) x = __half2float(lg[i]);
    else x = lg[i];
    sv[(i / C) * CS + i % C] = x != x ? -INFINITY : x;
  }
  __syncthreads();
  if (a.prev_off && p.repetition_penalty != 1.0f) {
    // one thread applies all occurrences of a token, in order
    const uint32_t j1 = a.prev_off[row + 1];
    for (uint32_t j = a.prev_off[row]; j < j1; ++j) {
      const long long t = (long long)a.prev[j] - base;
      if (t >= 0 && t < len && (int)(t % kFT) == tid) {
        float& x = sv[(t / C) * CS + t % C];
        x = x > 0.f ? __fdiv_rn(x, p.repetition_penalty) : __fmul_rn(x, p.repetition_penalty);
      }
    }
    __syncthreads();
  }
  const int i0 = min(tid * C, len), n = min(C, len - i0);
  float* sc = sv + tid * CS;
  const float t = p.temperature;
  const bool greedy = !(t >= 1e-7f);
  u64 best = 0;  // order key of the value, then the lowest index
  for (int i = 0; i < n; ++i) {
    const float x = greedy ? sc[i] : __fdiv_rn(sc[i], t);
    sc[i] = x;
    const u64 k = ((u64)float_order_key(x) << 32) | (0xffffffffu - (uint32_t)(base + i0 + i));
    best = k > best ? k : best;
  }
  best = block_reduce<true>(best, s);
  {
    const u64* all = cl.share(best);
    for (int r = 0; r < cl.n; ++r) best = all[r] > best ? all[r] : best;
  }
  const uint32_t mk = (uint32_t)(best >> 32);
  const float m = __uint_as_float((mk & 0x80000000u) ? mk & 0x7fffffffu : ~mk);
  if (m == -INFINITY || greedy) {  // the same in every thread of the cluster
    if (cl.rank == 0 && tid == 0) {
      const bool none = m == -INFINITY;
      a.tokens[row] = none ? 0xffffffffu : 0xffffffffu - (uint32_t)best;
      if (a.probs) a.probs[row] = none ? 0.f : 1.f;
    }
    cl.g.sync();
    return;
  }
  u64 mass = 0;
  for (int i = 0; i < n; ++i) {
    float w = sc[i] == m ? 1.f : expf(sc[i] - m);
    if (!(w >= p.min_p)) w = 0.f;
    sc[i] = w;
    mass += fix(w);
  }
  mass = block_reduce<false>(mass, s);
  u64 total = 0;
  {
    const u64* all = cl.share(mass);
    for (int r = 0; r < cl.n; ++r) total += all[r];
  }
  Cut cut{0u, 0xffffffffu, 0};  // keeps everything
  if (p.top_k > 0 && p.top_k < (uint32_t)V) {
    cut = radix_cut<true>(sc, n, cut, p.top_k, cl);
    total = cut.above + (u64)cut.ties * fix(__uint_as_float(cut.bits));
  }
  if (p.top_p > 0.f && p.top_p < 1.f) {
    u64 want = (u64)((double)total * (double)p.top_p);
    if (want < 1) want = 1;
    Cut c = radix_cut<false>(sc, n, cut, want, cl);
    if (c.bits >= cut.bits) cut = c;
    total = cut.above + (u64)cut.ties * fix(__uint_as_float(cut.bits));
  }
  // kept weights: bits above the cut, and its ties with the lowest indices
  u64 eq = 0;
  for (int i = 0; i < n; ++i) eq += __float_as_uint(sc[i]) == cut.bits;
  u64 cta_eq;
  u64 tie = block_scan(eq, s, cta_eq);
  {
    const u64* all = cl.share(cta_eq);
    for (int r = 0; r < cl.rank; ++r) tie += all[r];
  }
  u64 mine = 0;
  {
    u64 k = tie;
    for (int i = 0; i < n; ++i) {
      const uint32_t b = __float_as_uint(sc[i]);
      if (b < cut.bits || (b == cut.bits && k++ >= cut.ties)) sc[i] = 0.f;
      else mine += fix(sc[i]);
    }
  }
  u64 cta_mass;
  u64 run = block_scan(mine, s, cta_mass);
  {
    const u64* all = cl.share(cta_mass);
    total = 0;
    for (int r = 0; r < cl.n; ++r) {
      if (r < cl.rank) run += all[r];
      total += all[r];
    }
  }
  const u64 target = (u64)((double)a.uniforms[row] * (double)total);
  // exactly one thread's kept weights reach past the target (target < total)
  if (run <= target && target < run + mine) {
    for (int i = 0; i < n; ++i) {
      const u64 w = fix(sc[i]);
      if (run + w > target) {
        a.tokens[row] = (uint32_t)(base + i0 + i);
        if (a.probs) a.probs[row] = (float)((double)w / (double)total);
        break;
      }
      run += w;
    }
  }
  cl.g.sync();  // no CTA leaves while another reads its shared memory
}

template <class T>
cudaError_t launch_t(const FilterArgs& a, int n, cudaStream_t s) {
  const size_t smem = (size_t)kFT * chunk_stride(chunk_len(share_len(a.vocab, n))) * 4;
  int dev = 0;
  cudaGetDevice(&dev);
  const int most = kFT * chunk_stride(chunk_len(share_len(kFilterMaxVocab, kMaxCluster))) * 4;
  if (cudaError_t e = ensure_smem_attr(filter_kernel<T>, most, dev)) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.n_rows * n));
  cfg.blockDim = dim3(kFT);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = n;
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, filter_kernel<T>, a);
}

}  // namespace

cudaError_t filter_launch(const FilterArgs& a, int num_sms, cudaStream_t s) {
  (void)num_sms;
  return a.x16 ? launch_t<__half>(a, kMaxCluster, s) : launch_t<float>(a, kMaxCluster, s);
}

}  // namespace rb
