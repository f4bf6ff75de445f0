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
// floor(u sum W) (draw_target). t < 1e-7 takes the first rank.
//
// Two kernels. The one for short lists (below) settles the rows that keep few tokens; the
// other takes every row: a cluster of CTAs holds the row in shared memory, each CTA a
// contiguous share of its 16-byte vectors, thread t the vectors t, t + 1024, ... of the
// share. Thresholds come from a radix walk over the bits of w: first its binade (W has 40
// bits, so 41 of them), then the 23 bits of its mantissa in digits of 8, 8 and 7, until a
// bin is kept whole; each step is a histogram of counts and sums that the cluster adds up
// through distributed shared memory. Within a binade W is v << s with a v of 24 bits, so a
// sum is that of v's low 10 and high 14 bits, in 32-bit words: 64-bit shared-memory atomics
// are loops. The binades of a row are few, so their histogram has a copy per lane (no two
// lanes of a warp meet); mantissas are spread, and there only the elements of the chosen
// binade count.
//
// Bound by the chain of barriers (about ten) and by instructions: 96 rows of 151937 take
// 101 us with the elements in shared memory and two CTAs an SM, took 129 us with them in
// registers (one CTA an SM), 208 us with chunks of consecutive elements a thread, 315 us
// with 64-bit atomics. With short lists 50 us with nothing of the row in L2, 42 to 45 us in a loop
// over other inputs (58 MB, 1.2 to 1.4 TB/s, on two thirds of the SMs: reading for the
// maximum, from L2 for the list, 7 us for thresholds and draw, 3 for the second kernel,
// which finds nothing left). One row of 32000: 13-14 us. Without a min-p or top-k 128 us.
// A history costs 0.6 us a token (96 rows with 500 each 425 us): every thread goes over it.
#include <cooperative_groups.h>

#include <algorithm>

#include "common.cuh"
#include "filter.cuh"

namespace cg = cooperative_groups;

namespace rb {

namespace {

constexpr int kFT = 1024, kFW = kFT / 32;
constexpr int kBinades = 48;      // 41 in use: binade b holds exponents 127 - b
constexpr int kBins = 256;
constexpr int kMaxCluster = 8;
constexpr uint32_t kLeft = 0xfffffffeu;  // in place of a token: a row left to the second kernel
constexpr int kShortWarp = 384;   // candidates a warp may find
constexpr int kShortBins = 512;
constexpr int kShortMax = 8192;   // candidates of a row
constexpr int kShortSums = 4095;  // of a bin: 4095 (2^20 + 2^20) fits the 32-bit sums of W's halves
constexpr float kShortFloor = 0x1p-13f, kShortFloor2 = 0x1p-8f;
constexpr int kMaxElems = 40;     // of a thread: one vector more than 262144 / 8 / 1024, for rows off 16 bytes
using u64 = unsigned long long;

struct FilterShared {
  // per lane: count << 21 | sum of low parts; sum of high parts. In short lists: two histograms.
  uint32_t ba[2 * kBinades * 32];
  __device__ uint32_t* bb() { return ba + kBinades * 32; }
  uint32_t cnt[2][kBins], lo[2][kBins], hi[2][kBins];
  u64 xch[2][kMaxCluster];  // one value of every CTA of the cluster
  u64 red[kFW], red2[kFW];
  u64 part[kMaxElems / 4][kFW];  // kept weight by vector round and warp
  u64 above_c, above_s, in_s, base;
  uint32_t bin, in_bin, round, warp;
};
static_assert(2 * 3 * kShortBins <= 2 * kBinades * 32 && kFilterMaxVocab / kFW + 2 * 8 * 32 < 65536, "");
// one lane's copy takes at most kMaxElems elements of each warp: 11 bits of count, 21 of low parts
static_assert(kFW * kMaxElems < 2048 && kFilterMaxVocab + 8 <= kMaxCluster * kFT * kMaxElems, "");

// W and its parts: W = v << s
__device__ __forceinline__ uint32_t part_of(float w, int& binade) {
  const uint32_t b = __float_as_uint(w), m = (b & 0x7fffffu) | 0x800000u;
  binade = 127 - (int)(b >> 23);
  return binade > 40 ? 0u : binade > 17 ? m >> (binade - 17) : m;
}
__device__ __forceinline__ int shift_of(int binade) { return binade > 17 ? 0 : 17 - binade; }
__device__ __forceinline__ u64 fix(float w) {
  int b;
  const uint32_t v = part_of(w, b);
  return (u64)v << shift_of(b);
}

__device__ __forceinline__ u64 warp_max(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const u64 x = __shfl_xor_sync(0xffffffffu, v, o);
    v = x > v ? x : v;
  }
  return v;
}
__device__ __forceinline__ u64 warp_scan(u64 v) {  // inclusive
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  return v;
}

// exclusive prefix in thread order, and the block's total
__device__ u64 block_scan(u64 v, u64* red, u64& total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const u64 x = warp_scan(v);
  __syncthreads();
  if (lane == 31) red[w] = x;
  __syncthreads();
  const u64 t = red[lane], incl = warp_scan(t);
  total = __shfl_sync(0xffffffffu, incl, 31);
  return __shfl_sync(0xffffffffu, incl - t, w) + x - v;
}
// sum over the warp of values below 2^43
__device__ __forceinline__ u64 warp_sum43(u64 v) {
  const uint32_t lo = __reduce_add_sync(0xffffffffu, (uint32_t)v & 0x3fffffu),
                 hi = __reduce_add_sync(0xffffffffu, (uint32_t)(v >> 22));
  return ((u64)hi << 22) + lo;
}

// Buffers alternate with `turn`, which every barrier of the cluster raises: one
// barrier per exchange does.
template <int N>
struct Cluster {
  cg::cluster_group g;
  FilterShared& s;
  int rank, turn = 0;
  __device__ Cluster(FilterShared& sh) : g(cg::this_cluster()), s(sh), rank(N > 1 ? (int)g.block_rank() : 0) {}
  __device__ void sync() {
    if (N > 1) g.sync();
    else __syncthreads();
    ++turn;
  }
  // every CTA's value (the same in all its threads) to every CTA
  __device__ const u64* share(u64 v) {
    u64* mine = s.xch[turn & 1];
    if (threadIdx.x < N) *g.map_shared_rank(&mine[rank], threadIdx.x) = v;
    sync();
    return mine;
  }
  // the sum of everybody's copies of a histogram word
  __device__ u64 gather(const uint32_t* p) {
    if (N == 1) return *p;
    uint32_t x[N];
#pragma unroll
    for (int r = 0; r < N; ++r) x[r] = *g.map_shared_rank(p, r);
    u64 t = 0;
#pragma unroll
    for (int r = 0; r < N; ++r) t += x[r];
    return t;
  }
};

// A thread's elements: NQ quads, kFT apart in shared memory, which no other thread touches.
template <int NQ, class F>
__device__ __forceinline__ void each(const float4* mine, F f) {
#pragma unroll 2
  for (int q = 0; q < NQ; ++q) {
    const float4 v = mine[q * kFT];
    f(v.x);
    f(v.y);
    f(v.z);
    f(v.w);
  }
}
template <int NQ, class F>
__device__ __forceinline__ void change(float4* mine, F f) {
#pragma unroll 2
  for (int q = 0; q < NQ; ++q) {
    float4 v = mine[q * kFT];
    v.x = f(v.x);
    v.y = f(v.y);
    v.z = f(v.z);
    v.w = f(v.w);
    mine[q * kFT] = v;
  }
}

// The running sum that the draw has to pass, below `total` (at least 1) for every u, so that each
// row gets a token: u >= 1 draws the last kept one, u <= 0 or not a number the first.
__device__ __forceinline__ u64 draw_target(float u, u64 total) {
  const double x = (double)u * (double)total;
  if (!(x > 0.0)) return 0;
  return x < (double)total ? min((u64)x, total - 1) : total - 1;
}

// What is kept: weights with more than `bits`, and the first `ties` of those with
// just these bits, of which there are `equal`.
struct Cut {
  uint32_t bits, ties, equal;
};

// One step's choice: thread t < n holds the count c and sum w of a bin, the bins in
// falling order of weight. The last bin that holds an element ranked before `want`
// (by count, or by the sum before it) is taken; acc_*: what lies above its range.
template <bool COUNT>
__device__ void choose(uint32_t c, u64 w, int n, u64 want, u64& acc_c, u64& acc_s, FilterShared& s) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nw = n >> 5;
  u64 ic = 0, is = 0;
  if (warp < nw) {
    ic = warp_scan(c);
    is = warp_scan(w);
    if (lane == 31) {
      s.red[warp] = ic;
      s.red2[warp] = is;
    }
  }
  __syncthreads();
  if (warp < nw) {
    u64 bc = acc_c, bs = acc_s;
    for (int q = 0; q < warp; ++q) {
      bc += s.red[q];
      bs += s.red2[q];
    }
    const u64 ac = bc + ic - c, as = bs + is - w;
    const bool has = c > 0 && (COUNT ? ac < want : as < want);
    const unsigned any = __ballot_sync(0xffffffffu, has);
    const u64 ec = bc + __shfl_sync(0xffffffffu, ic, 31), es = bs + __shfl_sync(0xffffffffu, is, 31);
    bool last = any != 0;
    if (last && (COUNT ? ec < want : es < want)) {  // a later warp with a bin of its own has the say
      u64 rest = 0;
      for (int q = warp + 1; q < nw; ++q) rest += s.red[q];
      last = rest == 0;
    }
    if (last && lane == 31 - __clz(any)) {
      s.bin = tid;
      s.in_bin = c;
      s.in_s = w;
      s.above_c = ac;
      s.above_s = as;
    }
  }
  __syncthreads();
  acc_c = s.above_c;
  acc_s = s.above_s;
}

// The cut of one rule. bc, bw: this thread's binade (thread t < kBinades holds binade
// t). total: the sum of what it keeps.
template <bool COUNT, int NQ, int N>
__device__ Cut radix_cut(const float4* mine, uint32_t bc, u64 bw, u64 want, Cluster<N>& cl, u64& total) {
  FilterShared& s = cl.s;
  const int tid = threadIdx.x;
  u64 acc_c = 0, acc_s = 0;
  choose<COUNT>(bc, bw, 64, want, acc_c, acc_s, s);
  const int binade = (int)s.bin, shift = shift_of(binade);
  uint32_t pre = (uint32_t)(127 - binade) << 23;
  int sh = 23;
  // a bin with one element, or (by count) without one too many, is kept whole
  auto whole = [&]() { return s.in_bin == 1 || (COUNT && acc_c + s.in_bin <= want); };
  while (sh > 0 && !whole()) {
    const int width = sh == 7 ? 7 : 8;
    const uint32_t hmask = 0xffffffffu << sh;
    sh -= width;
    const int turn = cl.turn & 1;
    uint32_t *cnt = s.cnt[turn], *lo = s.lo[turn], *hi = s.hi[turn];
    if (tid < kBins) cnt[tid] = lo[tid] = hi[tid] = 0;
    __syncthreads();
    each<NQ>(mine, [&](float x) {
      const uint32_t b = __float_as_uint(x);
      if ((b & hmask) == pre) {
        int e;
        const uint32_t v = part_of(x, e), bin = (b >> sh) & ((1u << width) - 1);
        atomicAdd(&cnt[bin], 1u);
        atomicAdd(&lo[bin], v & 1023u);
        atomicAdd(&hi[bin], v >> 10);
      }
    });
    cl.sync();
    // thread t owns bin 2^width - 1 - t
    uint32_t c = 0;
    u64 w = 0;
    const int bin = (1 << width) - 1 - tid;
    if (bin >= 0) {
      c = (uint32_t)cl.gather(&cnt[bin]);
      w = cl.gather(&lo[bin]) + (cl.gather(&hi[bin]) << 10);
    }
    choose<COUNT>(c, w << shift, 1 << width, want, acc_c, acc_s, s);
    pre |= ((1u << width) - 1 - s.bin) << sh;
  }
  if (whole()) {
    total = acc_s + s.in_s;
    return Cut{pre, 0xffffffffu, 0xffffffffu};
  }
  const u64 tq = fix(__uint_as_float(pre));
  // by sum: the j-th tie is kept while above + j tq < want
  const u64 ties = COUNT ? want - acc_c : (want - acc_s + tq - 1) / tq;
  Cut r{pre, ties < s.in_bin ? (uint32_t)ties : s.in_bin, s.in_bin};
  total = acc_s + r.ties * tq;
  return r;
}

// Rows with a short list. Most rows keep only tokens within a few binades of the first rank: a
// min-p of at least kShortFloor keeps no others, nor does a top-k for which there are k above
// that weight. They are some thousandth of the vocabulary, so a first kernel reads the row
// twice (once for the maximum, once, from L2, for the list), and the first CTA of its
// cluster does the rest by itself on the list, which is in the order of the indices. The
// rows whose list does not fit, that need the whole vocabulary or have repetitions to
// penalise are left to the other kernel, which holds all their elements.

// A thread's candidates of the short list: K consecutive ones.
struct ShortList {
  uint2* mine;  // weight's bits, index
  int K;
  template <class F>
  __device__ __forceinline__ void each(F f) const {
    for (int e = 0; e < K; ++e) f(mine[e]);
  }
};
__device__ __forceinline__ uint32_t short_key(uint32_t bits) { return 0x3f800000u - bits; }  // below 2^27

// Histogram of the digit at `sh` of the candidates whose key continues `pre`; thread t < kShortBins
// gets bin t's count and sum. `turn` alternates; the other buffer is cleared for the next one.
__device__ void short_hist(const ShortList& l, uint32_t pre, int sh, int& turn, uint32_t& c, u64& w, FilterShared& s) {
  const int tid = threadIdx.x;
  uint32_t* h = s.ba + (turn & 1) * 3 * kShortBins;
  uint32_t* other = s.ba + (~turn & 1) * 3 * kShortBins;
  ++turn;
  l.each([&](uint2 v) {
    const uint32_t key = short_key(v.x);
    if (v.x && key >> (sh + 9) == pre) {
      const uint32_t b = (key >> sh) & (kShortBins - 1);
      const u64 f = fix(__uint_as_float(v.x));
      atomicAdd(&h[b], 1u);
      atomicAdd(&h[kShortBins + b], (uint32_t)f & 0xfffffu);
      atomicAdd(&h[2 * kShortBins + b], (uint32_t)(f >> 20));
    }
  });
  for (int i = tid; i < 3 * kShortBins; i += kFT) other[i] = 0;
  __syncthreads();
  c = 0;
  w = 0;
  if (tid < kShortBins) {
    c = h[tid];
    w = h[kShortBins + tid] + ((u64)h[2 * kShortBins + tid] << 20);
  }
}

// The cut of one rule over the short list; (c, w): the first digit's bin of this thread.
template <bool COUNT>
__device__ Cut short_cut(const ShortList& l, uint32_t c, u64 w, u64 want, int& turn, u64& total, FilterShared& s) {
  u64 acc_c = 0, acc_s = 0;
  uint32_t pre = 0;
  int sh = 27;
  auto whole = [&]() { return s.in_bin == 1 || (COUNT && acc_c + s.in_bin <= want); };
  do {
    sh -= 9;
    if (sh < 18) short_hist(l, pre, sh, turn, c, w, s);
    choose<COUNT>(c, w, kShortBins, want, acc_c, acc_s, s);
    pre = pre << 9 | s.bin;
  } while (sh > 0 && !whole());
  const uint32_t bits = 0x3f800000u - (((pre + 1) << sh) - 1);  // the least of the bin
  if (whole()) {
    total = acc_s + s.in_s;
    return Cut{bits, 0xffffffffu, 0xffffffffu};
  }
  const u64 tq = fix(__uint_as_float(bits));
  const u64 ties = COUNT ? want - acc_c : (want - acc_s + tq - 1) / tq;
  Cut r{bits, ties < s.in_bin ? (uint32_t)ties : s.in_bin, s.in_bin};
  total = acc_s + r.ties * tq;
  return r;
}

// Thresholds and draw over the n candidates of `list`, by one CTA. False: more of one bin than its sums hold.
__device__ bool short_finish(uint2* list, int n, const rb_sampling_filter& p, bool use_k, bool use_p, const FilterArgs& a,
                             int row, FilterShared& s) {
  const int tid = threadIdx.x;
  const int K = (n + kFT - 1) / kFT;
  for (int i = tid; i < 6 * kShortBins; i += kFT) s.ba[i] = 0;
  for (int i = n + tid; i < K * kFT; i += kFT) list[i] = make_uint2(0, 0);
  __syncthreads();
  const ShortList l{list + tid * K, K};
  int turn = 0;
  Cut cut{0u, 0xffffffffu, 0xffffffffu};
  u64 total = 0;
  if (use_k || use_p) {
    uint32_t c;
    u64 w;
    short_hist(l, 0, 18, turn, c, w, s);
    if (n > kShortSums && __syncthreads_or(c > kShortSums)) return false;
    if (use_k) {
      cut = short_cut<true>(l, c, w, p.top_k, turn, total, s);
    } else {
      block_scan(w, s.red, total);
    }
    if (use_p) {
      u64 want = (u64)((double)total * (double)p.top_p);
      if (want < 1) want = 1;
      __syncthreads();  // s.in_bin and the like have been read
      const Cut q = short_cut<false>(l, c, w, want, turn, total, s);
      if (q.bits > cut.bits || (q.bits == cut.bits && q.ties < cut.ties)) cut = q;
    }
    if (cut.ties < cut.equal) {  // the same in every thread
      u64 eq = 0, all;
      l.each([&](uint2 v) { eq += v.x == cut.bits; });
      u64 rank = block_scan(eq, s.red, all);
      for (int e = 0; e < K; ++e)
        if (l.mine[e].x == cut.bits && rank++ >= cut.ties) l.mine[e].x = 0;
    }
  }
  u64 sum = 0;
  l.each([&](uint2 v) {
    if (v.x >= cut.bits) sum += fix(__uint_as_float(v.x));
  });
  u64 at = block_scan(sum, s.red, total);
  const u64 target = draw_target(a.uniforms[row], total);
  if (target < at || target >= at + sum) return true;
  for (int e = 0; e < K; ++e) {
    const uint2 v = l.mine[e];
    const u64 f = v.x >= cut.bits ? fix(__uint_as_float(v.x)) : 0;
    if (at + f > target) {
      a.tokens[row] = v.y;
      if (a.probs) a.probs[row] = (float)((double)f / (double)total);
      return true;
    }
    at += f;
  }
  return true;
}

// One CTA an SM, for the registers of four vectors in flight a thread: 96 rows of 151937
// 50 us, with two vectors and two CTAs 65 us; 200 rows 93 and 114 (nothing in L2).
template <class T, int N>
__global__ void __launch_bounds__(kFT, 1) filter_short_kernel(const __grid_constant__ FilterArgs a) {
  constexpr int E = 16 / sizeof(T), U = 4;
  extern __shared__ uint2 list[];            // of the first CTA: all candidates
  __shared__ uint16_t own[kFW][kShortWarp];  // each warp's, as places in its part of the row
  __shared__ FilterShared s;
  __shared__ uint32_t kept;  // of the first CTA
  Cluster<N> cl(s);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_launch_dependents();
  const int row = blockIdx.x / N;
  rb_sampling_filter p = a.params[row];
  p.min_p = fminf(p.min_p, 1.f);  // the first rank always stays
  const int V = a.vocab;
  const float t = p.temperature;
  const bool greedy = !(t >= 1e-7f);
  const bool use_k = p.top_k > 0 && p.top_k < (uint32_t)V, use_p = p.top_p > 0.f && p.top_p < 1.f;
  bool all_of = p.min_p >= kShortFloor;  // the list has all that is kept
  if (!(greedy || use_k || all_of) ||
      (a.prev_off && p.repetition_penalty != 1.0f && a.prev_off[row + 1] > a.prev_off[row])) {
    if (cl.rank == 0 && tid == 0) a.tokens[row] = kLeft;
    return;  // the whole cluster
  }
  if (tid == 0) kept = 0;
  if (N > 1) cg::this_cluster().barrier_arrive();
  const T* lg = reinterpret_cast<const T*>(a.logits) + (size_t)row * a.ld;
  // the row's 16-byte vectors, the first one up to E - 1 elements before the row; each CTA has a
  // contiguous share of them, and each of its warps of those
  const int mis = (int)((reinterpret_cast<uintptr_t>(lg) & 15) / sizeof(T));
  const int vecs = (V + mis + E - 1) / E, share = (vecs + N - 1) / N, ours = (share + kFW - 1) / kFW;
  const int v0 = cl.rank * share + warp * ours, v1 = min(min(vecs, (cl.rank + 1) * share), v0 + ours);
  // f(elements, vector) for U vectors a lane; -inf where there is none
  auto scan = [&](auto f) {
#pragma unroll 1
    for (int b = v0; b < v1; b += 32 * U) {
      constexpr uint32_t none = sizeof(T) == 2 ? 0xfc00fc00u : 0xff800000u;
      uint4 q[U];
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int v = b + 32 * j + lane, i = v * E - mis;
        q[j] = make_uint4(none, none, none, none);
        if (v < v1 && i >= 0 && i + E <= V) q[j] = __ldg(reinterpret_cast<const uint4*>(lg + i));
      }
      if (b == 0 || b + 32 * U >= vecs) {  // the row's ends may be within a vector
#pragma unroll
        for (int j = 0; j < U; ++j) {
          const int v = b + 32 * j + lane, i = v * E - mis;
          if (v < v1 && (i < 0 || i + E > V)) {
            T y[E];
            *reinterpret_cast<uint4*>(y) = q[j];
#pragma unroll
            for (int e = 0; e < E; ++e)
              if (i + e >= 0 && i + e < V) y[e] = lg[i + e];
            q[j] = *reinterpret_cast<uint4*>(y);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const T* y = reinterpret_cast<const T*>(&q[j]);
        float x[E];
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = (float)y[e];
        f(x, b + 32 * j + lane);
      }
    }
  };
  float top = -INFINITY;
  scan([&](const float (&x)[E], int) {
#pragma unroll
    for (int e = 0; e < E; ++e) top = fmaxf(top, x[e]);  // not of what is not a number
  });
  uint32_t key = __reduce_max_sync(0xffffffffu, float_order_key(top));
  if (lane == 0) s.red[warp] = key;
  __syncthreads();
  key = __reduce_max_sync(0xffffffffu, (uint32_t)s.red[lane]);
  if (N > 1) {
    cg::this_cluster().barrier_wait();  // every CTA of the cluster runs before its shared memory is written
    const u64* all = cl.share(key);
#pragma unroll
    for (int r = 0; r < N; ++r) key = max(key, (uint32_t)all[r]);
  }
  top = __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key);
  if (top == -INFINITY) {
    if (cl.rank == 0 && tid == 0) {
      a.tokens[row] = 0xffffffffu;
      if (a.probs) a.probs[row] = 0.f;
    }
    return;
  }
  if (greedy) {  // the lowest index that has it
    uint32_t at = 0xffffffffu;
    scan([&](const float (&x)[E], int v) {
#pragma unroll
      for (int e = E - 1; e >= 0; --e)
        if (x[e] == top) at = min(at, (uint32_t)(v * E + e - mis));
    });
    at = __reduce_min_sync(0xffffffffu, at);
    if (lane == 0) s.red2[warp] = at;
    __syncthreads();
    at = __reduce_min_sync(0xffffffffu, (uint32_t)s.red2[lane]);
    if (N > 1) {
      const u64* all = cl.share(at);
#pragma unroll
      for (int r = 0; r < N; ++r) at = min(at, (uint32_t)all[r]);
    }
    if (cl.rank == 0 && tid == 0) {
      a.tokens[row] = at;
      if (a.probs) a.probs[row] = 1.f;
    }
    return;
  }
  const float m = t == 1.f ? top : __fdiv_rn(top, t);  // the largest quotient: division keeps the order
  float least = all_of ? p.min_p : kShortFloor;
  uint32_t count, before;
  int n;
#pragma unroll 1
  while (true) {
    // below `far` no quotient's weight reaches `least` (where this overflows or is not a number, all are listed)
    const float ln = logf(least) - 1e-3f, far = (m + ln) * t - (fabsf(m) - ln) * t * 1e-6f;
    n = 0;
    scan([&](const float (&x)[E], int v) {
      bool some = false;
#pragma unroll
      for (int e = 0; e < E; ++e) some |= !(x[e] < far);
      if (!__any_sync(0xffffffffu, some)) return;
      int at = n;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const unsigned b = __ballot_sync(0xffffffffu, !(x[e] < far));
        at += __popc(b & ((1u << lane) - 1));
        n += __popc(b);
      }
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (!(x[e] < far)) {
          if (at < kShortWarp) own[warp][at] = (uint16_t)((v - v0) * E + e);
          ++at;
        }
    });
    if (lane == 0) s.red2[warp] = (u64)n;
    __syncthreads();
    const uint32_t warps_n = (uint32_t)s.red2[lane], scanned = (uint32_t)warp_scan(warps_n);
    before = __shfl_sync(0xffffffffu, scanned - warps_n, warp);
    count = __shfl_sync(0xffffffffu, scanned, 31);
    if (__any_sync(0xffffffffu, warps_n > kShortWarp)) count = 1u << 24;
    if (N > 1) {
      const u64* all = cl.share(count);
      count = 0;
#pragma unroll
      for (int r = 0; r < N; ++r) {
        if (r < cl.rank) before += (uint32_t)all[r];
        count += (uint32_t)all[r];
      }
    }
    // too many: fewer do for a top-k
    if (count <= kShortMax || !use_k || least >= kShortFloor2) break;
    least = kShortFloor2;
    all_of = false;
    __syncthreads();  // s.red2 has been read
  }
  if (count > kShortMax) {  // the same in every thread of the cluster
    if (cl.rank == 0 && tid == 0) a.tokens[row] = kLeft;
    return;
  }
  {
    uint2* first = N > 1 ? cl.g.map_shared_rank(list, 0) : list;
    uint32_t found = 0;
    for (int b = 0; b < n; b += 32) {
      bool in = false;
      if (b + lane < n) {
        const int place = own[warp][b + lane], i = v0 * E + place - mis;
        float x = -INFINITY;  // where all are listed, places past the warp's part are too
        if (v0 + place / E < v1 && i >= 0 && i < V) x = (float)lg[i];
        if (t != 1.f) x = __fdiv_rn(x, t);
        const float w = x == m ? 1.f : expf(x - m);
        in = w >= least;
        first[before + b + lane] = make_uint2(in ? __float_as_uint(w) : 0u, (uint32_t)i);
      }
      found += __popc(__ballot_sync(0xffffffffu, in));
    }
    if (lane == 0 && found) atomicAdd(N > 1 ? cl.g.map_shared_rank(&kept, 0) : &kept, found);
  }
  cl.sync();
  if (cl.rank) return;
  if ((!all_of && kept < p.top_k) || !short_finish(list, (int)count, p, use_k, use_p, a, row, s))
    if (tid == 0) a.tokens[row] = kLeft;
}

// Two CTAs an SM (32 registers a thread) where their elements fit and keep a CTA busy
// for long enough: one works while the other waits at a barrier (96 rows of 151937: 101 us
// against 129 with one).
template <class T, int NV>
constexpr int two_ctas() {
  return NV >= 3 && NV * (16 / (int)sizeof(T)) <= 24 ? 2 : 1;
}

template <class T, int NV, int N>
__global__ void __launch_bounds__(kFT, two_ctas<T, NV>()) filter_kernel(const __grid_constant__ FilterArgs a) {
  constexpr int E = 16 / sizeof(T), Q = E / 4, NQ = NV * Q;  // quads of a vector, of a thread
  extern __shared__ float4 quads[];
  __shared__ FilterShared s;
  Cluster<N> cl(s);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x / N;
  pdl_wait();
  if (!a.all && a.tokens[row] != kLeft) return;  // the whole cluster
  if (N > 1) cg::this_cluster().barrier_arrive();
  rb_sampling_filter p = a.params[row];
  p.min_p = fminf(p.min_p, 1.f);  // the first rank always stays
  const int V = a.vocab;
  const T* lg = reinterpret_cast<const T*>(a.logits) + (size_t)row * a.ld;
  // the row's 16-byte vectors, the first one up to E - 1 elements before the row
  const int mis = (int)((reinterpret_cast<uintptr_t>(lg) & 15) / sizeof(T));
  const int vecs = (V + mis + E - 1) / E, share = (vecs + N - 1) / N;
  const int v0 = cl.rank * share, v1 = min(vecs, v0 + share);
  auto index = [&](int r) { return (v0 + r * kFT + tid) * E - mis; };  // of vector round r's first element
  float4* mine = quads + tid;
#pragma unroll
  for (int r = 0; r < NV; ++r) {
    const int i = index(r);
    const bool in = v0 + r * kFT + tid < v1;
    float x[E];
    if (in && i >= 0 && i + E <= V) {
      const uint4 q = __ldcs(reinterpret_cast<const uint4*>(lg + i));
      const T* y = reinterpret_cast<const T*>(&q);
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] = (float)y[e];
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] = in && i + e >= 0 && i + e < V ? (float)lg[i + e] : -INFINITY;
    }
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (x[e] != x[e]) x[e] = -INFINITY;
#pragma unroll
    for (int h = 0; h < Q; ++h) mine[(r * Q + h) * kFT] = make_float4(x[4 * h], x[4 * h + 1], x[4 * h + 2], x[4 * h + 3]);
  }
  for (int i = tid; i < 2 * kBinades * 32; i += kFT) s.ba[i] = 0;
  const float t = p.temperature;
  const bool greedy = !(t >= 1e-7f);
  float top = -INFINITY;
  if (a.prev_off && p.repetition_penalty != 1.0f) {
    // one thread applies all occurrences of a token, in order
    const uint32_t j1 = a.prev_off[row + 1];
    for (uint32_t j = a.prev_off[row]; j < j1; ++j) {
      const uint32_t tok = a.prev[j];
      const int at = tok < (uint32_t)V ? (int)tok + mis : -1, local = at / E - v0;
      if (at >= 0 && local >= 0 && at / E < v1 && local % kFT == tid) {
        float& x = reinterpret_cast<float*>(mine + (local / kFT * Q + at % E / 4) * kFT)[at % 4];
        x = x > 0.f ? __fdiv_rn(x, p.repetition_penalty) : __fmul_rn(x, p.repetition_penalty);
      }
    }
  }
  if (!greedy && t != 1.f) change<NQ>(mine, [&](float x) { return __fdiv_rn(x, t); });
  each<NQ>(mine, [&](float x) { top = fmaxf(top, x); });
  u64 best = (u64)float_order_key(top) << 32;
  if (greedy) {  // and the lowest index that has it
    uint32_t at = 0xffffffffu;
    for (int q = NQ - 1; q >= 0; --q)
      for (int e = 3; e >= 0; --e)
        if (reinterpret_cast<float*>(mine + q * kFT)[e] == top && top != -INFINITY)
          at = (uint32_t)(index(q / Q) + q % Q * 4 + e);
    best |= 0xffffffffu - at;
  }
  best = warp_max(best);
  if (lane == 0) s.red[warp] = best;
  __syncthreads();
  best = warp_max(s.red[lane]);
  if (N > 1) {
    cg::this_cluster().barrier_wait();  // every CTA of the cluster runs before its shared memory is written
    const u64* all = cl.share(best);
#pragma unroll
    for (int r = 0; r < N; ++r) best = all[r] > best ? all[r] : best;
  }
  const uint32_t mk = (uint32_t)(best >> 32);
  const float m = __uint_as_float((mk & 0x80000000u) ? mk & 0x7fffffffu : ~mk);
  if (m == -INFINITY || greedy) {  // the same in every thread of the cluster
    if (cl.rank == 0 && tid == 0) {
      const bool none = m == -INFINITY;
      a.tokens[row] = none ? 0xffffffffu : 0xffffffffu - (uint32_t)best;
      if (a.probs) a.probs[row] = none ? 0.f : 1.f;
    }
    return;
  }
  const bool use_k = p.top_k > 0 && p.top_k < (uint32_t)V, use_p = p.top_p > 0.f && p.top_p < 1.f;
  const bool hist = use_k || use_p;
  change<NQ>(mine, [&](float x) {
    const float w = x == m ? 1.f : expf(x - m);
    int b;
    const uint32_t v = part_of(w, b);
    const bool in = w >= p.min_p && v != 0;  // v 0: below the fixed point, never drawn
    if (hist && in) {
      atomicAdd(&s.ba[b * 32 + lane], 1u << 21 | (v & 1023u));
      atomicAdd(&s.bb()[b * 32 + lane], v >> 10);
    }
    return in ? w : 0.f;
  });
  if (hist) {
    Cut cut{0u, 0xffffffffu, 0xffffffffu};
    // the row's binades: sums over the lanes' copies, then over the cluster
    const int turn = cl.turn & 1;
    __syncthreads();
    for (int b = warp; b < kBinades; b += kFW) {
      const uint32_t y = s.ba[b * 32 + lane], z = s.bb()[b * 32 + lane];
      const uint32_t c = __reduce_add_sync(0xffffffffu, y >> 21), l = __reduce_add_sync(0xffffffffu, y & 0x1fffffu),
                     h = __reduce_add_sync(0xffffffffu, z);
      if (lane == 0) {
        s.cnt[turn][b] = c;
        s.lo[turn][b] = l;
        s.hi[turn][b] = h;
      }
    }
    cl.sync();
    uint32_t bc = 0;
    u64 bw = 0;
    if (tid < kBinades) {
      bc = (uint32_t)cl.gather(&s.cnt[turn][tid]);
      bw = (cl.gather(&s.lo[turn][tid]) + (cl.gather(&s.hi[turn][tid]) << 10)) << shift_of(tid);
    }
    u64 total = 0;
    if (use_k) {
      cut = radix_cut<true, NQ, N>(mine, bc, bw, p.top_k, cl, total);
    } else {
      if (tid < 64) {  // two warps hold the binades
        const u64 y = warp_scan(bw);
        if (lane == 31) s.red[warp] = y;
      }
      __syncthreads();
      total = s.red[0] + s.red[1];
      __syncthreads();
    }
    if (use_p) {
      u64 want = (u64)((double)total * (double)p.top_p);
      if (want < 1) want = 1;
      const Cut c = radix_cut<false, NQ, N>(mine, bc, bw, want, cl, total);
      // never below the first cut; at the same weight, the fewer ties
      if (c.bits > cut.bits || (c.bits == cut.bits && c.ties < cut.ties)) cut = c;
    }
    // kept: bits above the cut, and its ties with the lowest indices
    change<NQ>(mine, [&](float x) { return __float_as_uint(x) < cut.bits ? 0.f : x; });
    if (cut.ties < cut.equal) {  // the same in every thread of the cluster
      u64 count = 0, cta;
      each<NQ>(mine, [&](float x) { count += __float_as_uint(x) == cut.bits; });
      block_scan(count, s.red, cta);
      u64 before = 0;
      if (N > 1) {
        const u64* all = cl.share(cta);
        for (int r = 0; r < cl.rank; ++r) before += all[r];
      }
      for (int r = 0; r < NV; ++r) {
        u64 eq = 0;
        each<Q>(mine + r * Q * kFT, [&](float x) { eq += __float_as_uint(x) == cut.bits; });
        u64 round;
        u64 rank = before + block_scan(eq, s.red, round);
        before += round;
        change<Q>(mine + r * Q * kFT, [&](float x) { return __float_as_uint(x) == cut.bits && rank++ >= cut.ties ? 0.f : x; });
      }
    }
  }
  // the draw: rounds of vectors, then warps, then lanes are in the order of the indices
  for (int r = 0; r < NV; ++r) {
    u64 w = 0;
    each<Q>(mine + r * Q * kFT, [&](float x) {
      if (x != 0.f) w += fix(x);
    });
    w = warp_sum43(w);
    if (lane == 0) s.part[r][warp] = w;
  }
  __syncthreads();
  u64 mass = 0;
#pragma unroll
  for (int r = 0; r < NV; ++r) mass += s.part[r][lane];
  u64 total = __shfl_sync(0xffffffffu, warp_scan(mass), 31), run = 0;
  mass = total;
  if (N > 1) {
    const u64* all = cl.share(total);
    total = 0;
#pragma unroll
    for (int r = 0; r < N; ++r) {
      if (r < cl.rank) run += all[r];
      total += all[r];
    }
  }
  const u64 target = draw_target(a.uniforms[row], total);
  if (target < run || target >= run + mass) return;  // the whole CTA
  // exactly one CTA's, warp's and lane's kept weights reach past the target (target < total)
  if (warp == 0) {
    u64 at = run;
#pragma unroll 1
    for (int r = 0; r < NV; ++r) {
      const u64 w = s.part[r][lane], incl = at + warp_scan(w);
      if (incl - w <= target && target < incl) {
        s.round = r;
        s.warp = lane;
        s.base = incl - w;
      }
      at = __shfl_sync(0xffffffffu, incl, 31);
    }
  }
  __syncthreads();
  if (warp != (int)s.warp) return;
  const int round = (int)s.round;
  u64 w = 0;
  each<Q>(mine + round * Q * kFT, [&](float x) { w += fix(x); });
  u64 at = s.base + warp_scan(w) - w;
  if (at <= target && target < at + w) {
    int i = index(round);
    bool found = false;
    each<Q>(mine + round * Q * kFT, [&](float x) {
      const u64 f = fix(x);
      if (!found && at + f > target) {
        a.tokens[row] = (uint32_t)i;
        if (a.probs) a.probs[row] = (float)((double)f / (double)total);
        found = true;
      }
      at += f;
      ++i;
    });
  }
}

template <class T, int NV, int N>
cudaError_t launch(const FilterArgs& a, cudaStream_t s) {
  constexpr int smem = NV * kFT * (16 / (int)sizeof(T)) * 4;
  int dev = 0;
  cudaGetDevice(&dev);
  if (cudaError_t e = ensure_smem_attr(filter_kernel<T, NV, N>, smem, dev)) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.n_rows * N));
  cfg.blockDim = dim3(kFT);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = N;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, filter_kernel<T, NV, N>, a);
}

template <class T, int N>
cudaError_t launch_short(const FilterArgs& a, cudaStream_t s) {
  constexpr int smem = kShortMax * 8;
  int dev = 0;
  cudaGetDevice(&dev);
  if (cudaError_t e = ensure_smem_attr(filter_short_kernel<T, N>, smem, dev)) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.n_rows * N));
  cfg.blockDim = dim3(kFT);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = N;
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, filter_short_kernel<T, N>, a);
}

// CTAs a row: one for each SM, with a vector a thread at least. 1, 2, 3, 4, 6 and 8 CTAs a row,
// us: 200 rows of 151937 93, 93, 101, 109, 136, 154; 96 rows 50, 58, 60, 62, 73, 81; 48 rows 46,
// 38, 43, 42, 44, 52; 16 rows 40, 32, 30, 28, 26, 30; one row 30, 26, 24, 21, 21, 19; 96 rows of
// 32000 24, 36, 36, 41, 52, 60; 32 rows 24, 24, 22, 21, 28, 34.
template <class T>
cudaError_t launch_shorts(const FilterArgs& a, int num_sms, cudaStream_t s) {
  const int vecs = a.vocab / (16 / (int)sizeof(T)), n = std::min(num_sms / a.n_rows, vecs / kFT);
  if (n >= 8) return launch_short<T, 8>(a, s);
  if (n >= 6) return launch_short<T, 6>(a, s);
  if (n >= 4) return launch_short<T, 4>(a, s);
  if (n >= 3) return launch_short<T, 3>(a, s);
  if (n >= 2) return launch_short<T, 2>(a, s);
  return launch_short<T, 1>(a, s);
}

template <class T, int N>
cudaError_t launch_rounds(const FilterArgs& a, int rounds, cudaStream_t s) {
  constexpr int E = 16 / sizeof(T);
  if (rounds <= 1) return launch<T, 1, N>(a, s);
  if (rounds <= 2) return launch<T, 2, N>(a, s);
  if (rounds <= 3) return launch<T, 3, N>(a, s);
  if constexpr (E == 4) {
    if (rounds <= 5) return launch<T, 5, N>(a, s);
    if constexpr (N == 8) return launch<T, 9, N>(a, s);
  } else {
    if constexpr (N == 8) return launch<T, 5, N>(a, s);
  }
  return cudaErrorInvalidValue;
}

// CTAs a row: as few as hold it with two CTAs an SM, and then more while all rows'
// CTAs stay resident at once and a thread has more than one vector. 96 rows of 32000
// (2 CTAs a row, one wave): 39 us, with 4 45 and with 8 84 us; one row of 32000: 22, 16 and 14.
template <class T>
cudaError_t launch_type(const FilterArgs& a, int num_sms, cudaStream_t s) {
  constexpr int E = 16 / sizeof(T);
  const int vecs = (a.vocab + E - 1 + E - 1) / E;  // of a row, wherever it starts
  auto rounds = [&](int n) { return ((vecs + n - 1) / n + kFT - 1) / kFT; };
  int n = 1;
  while (n < kMaxCluster && rounds(n) > (E == 4 ? 5 : 3)) n *= 2;
  while (n < kMaxCluster && rounds(n) > 1 && (long long)a.n_rows * n * 2 <= 2ll * num_sms) n *= 2;
  // Short lists first, unless a thread would have one vector and a CTA an SM of its own: one and
  // eight rows of 32000 take 14 and 18.5 us without them, 17 and 21 with; 32 rows 39 and 21.5, one
  // row of 151937 29 and 19.5, 96 rows 107 and 50.
  FilterArgs b = a;
  b.all = rounds(n) <= 1 && (long long)a.n_rows * n <= num_sms;
  if (!b.all)
    if (cudaError_t e = launch_shorts<T>(a, num_sms, s)) return e;
  switch (n) {
    case 1: return launch_rounds<T, 1>(b, rounds(1), s);
    case 2: return launch_rounds<T, 2>(b, rounds(2), s);
    case 4: return launch_rounds<T, 4>(b, rounds(4), s);
    default: return launch_rounds<T, 8>(b, rounds(8), s);
  }
}

}  // namespace

cudaError_t filter_launch(const FilterArgs& a, int num_sms, cudaStream_t s) {
  return a.x16 ? launch_type<__half>(a, num_sms, s) : launch_type<float>(a, num_sms, s);
}

}  // namespace rb
