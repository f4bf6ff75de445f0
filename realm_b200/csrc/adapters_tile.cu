// Low-rank adapters for many rows (prompts): the function of adapters.cu, tile by tile on
// the tensor cores. A tile is up to `tile_rows` <= 128 rows of one adapter; a cluster of CTAs has it,
// splits k for v = down x and n for up v, and exchanges its parts of v through distributed
// shared memory in between, so that one kernel reads x once and writes out once.
//
//   v = down x: D[128 rows][rank] += X[128][chunk] down[rank][chunk]^T, chunks of 128 bytes a
//     row. Four warps fetch 32 rows each (wherever they lie) into a ring of their own, and put them into
//     tensor memory, the A operand, a thread a row; the fifth issues tcgen05.mma. fp16
//     rows are multiplied as they are (kind::f16). An fp32 x is two tf32 parts, x = hi + lo
//     (22 bits), the low one first, and the fp16 weights are exact in tf32.
//   out = y + scale up v: v is brought to a power of two near 2^13 row by row and split into fp16
//     hi + lo (22 bits of the row's largest), the A operand in tensor memory again; D[128 rows]
//     [64 columns] = v up^T, with up's tiles copied in bulk. y comes through the rings, each
//     row's thread adds its part there, and whole lines go out.
//
// The tensor core cuts a running sum off (towards 0) after every instruction, so fp32 rows sum at
// most 128 elements of k there; the sums of these chains are added in registers, with rounding.
//
// x and y are read and out is written once, which is most of the bytes. 8192 rows, rank 64, k = n = 4096, fp16 72 us
// (2.9 TB/s, floor 32 us), fp32 111 us (floor 62); 1024 rows 39 and 55 us. Bound by the workers' instructions
// and their latency: with four warps a CTA (168 registers a thread) two are there for each scheduler, which issue in
// 27 % of the slots; tensor cores 9 % busy, DRAM 26 %. Ranks above 64 leave one CTA an SM: 202 us (fp32).
// Tried and not kept: eight warps a CTA (96 registers spill: 103 us, 217 fp32), x and the low parts as
// operands in shared memory (152, 195), rows by bulk copies of 128 bytes (115, 192: 17 clocks a copy and SM), y as
// registers (115, 176).
//
// Tiles are found in the kernel: every CTA counts the rows of each slot, and a tile's rows are
// the next ones of its slot in the order of the rows. Clusters take tiles in turn.
#include <cooperative_groups.h>

#include <algorithm>

#include "adapters.cuh"
#include "common.cuh"

namespace cg = cooperative_groups;

namespace rb {

namespace {

constexpr int kWarps = 4, kWorkers = kWarps * 32, kTT = kWorkers + 32;  // fetch and finish; a warp for the products
constexpr uint32_t kNoSlot = 0xffff;
static_assert(kAdapterMaxSlots < (int)kNoSlot, "");
constexpr int kSpanRows = 8192;                     // rows of a launch
constexpr int kCols = 64;                           // columns of out a product covers
constexpr int kUps = 3;                             // bulk copies of weights in flight or use

// K-major operand in blocks of 8 rows x 16 bytes, `lbo` apart along K
__device__ __forceinline__ uint64_t desc_blocks(uint32_t saddr, uint32_t lbo) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)((lbo >> 4) & 0x3FFFu) << 16) | (8ull << 32) | (1ull << 46);
}
__device__ __forceinline__ uint32_t idesc_of(int tf32, int n) {
  return (1u << 4) | (tf32 ? (2u << 7) | (2u << 10) : 0u) | ((uint32_t)(n >> 3) << 17) | (8u << 24);
}
template <int TF32>
__device__ __forceinline__ void mma(uint32_t on, uint32_t d, uint32_t at, uint64_t bd, uint32_t id, uint32_t acc) {
  if constexpr (TF32)
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::tf32 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(at), "l"(bd), "r"(id), "r"(acc), "r"(on)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(at), "l"(bd), "r"(id), "r"(acc), "r"(on)
        : "memory");
}
__device__ __forceinline__ void commit(uint32_t on, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)),
      "r"(on)
      : "memory");
}
__device__ __forceinline__ uint32_t elect_lane() {
  uint32_t on;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(on));
  return on;
}
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void st4(uint32_t ta, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(ta), "r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3])
               : "memory");
}
__device__ __forceinline__ void st16(uint32_t ta, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16};" ::"r"(ta),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// 8 columns of this thread's TMEM lane; valid after wait_ld()
__device__ __forceinline__ void ld8(uint32_t ta, float* r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7])
               : "r"(ta)
               : "memory");
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// 16 bytes of which the first `left` elements exist (zeros behind them), one by one
template <class T>
__device__ __forceinline__ void copy_tail(uint8_t* dst, const T* src, int left) {
  T t[16 / sizeof(T)];
#pragma unroll
  for (int e = 0; e < (int)(16 / sizeof(T)); ++e) t[e] = e < left ? src[e] : T(0.f);
  *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<uint4*>(t);
}
// the same from rows off 16 bytes: fp32 as copies of 4 bytes
template <class T>
__device__ __forceinline__ void copy_single(uint8_t* dst, const T* src, int left) {
  if constexpr (sizeof(T) == 4) {
    const uint32_t at = smem_u32(dst);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (e < left) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(at + 4 * e), "l"(src + e) : "memory");
      else reinterpret_cast<float*>(dst)[e] = 0.f;
    }
  } else {
    copy_tail(dst, src, left);
  }
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void workers_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }

// mbar_wait without unrolling, which keeps these kernels' code small: a short call waits for it, a line at a time
__device__ __forceinline__ bool wait_rolled(uint64_t* bar, uint32_t parity, uint32_t* err, uint32_t code) {
#pragma unroll 1
  for (uint32_t i = 0; i < kSpinLimit; ++i)
    if (mbar_try_wait(bar, parity)) return true;
  report_error(err, code);
  return false;
}

// T: type of the rows. RP: ranks up to 64 (two CTAs an SM), or from 65 to 128.
template <class T, int RP>
struct Cfg {
  static constexpr int F32 = sizeof(T) == 4;
  static constexpr int E = 16 / (int)sizeof(T);     // elements of 16 bytes
  static constexpr int CE = 8 * E;                  // of a chunk: 128 bytes a row
  static constexpr int NS = RP == 64 ? 5 : 8;       // blocks of a warp's ring: 32 rows x 128 bytes
  static constexpr int RING = NS * 4096;
  static constexpr int B = RP * 128;                // bytes of a chunk's weights, and of a tile of up
  // weights: places for bulk copies, before them (fp32 rows) two chunks of weights in fp32, in whose place up goes later
  static constexpr int RAW = F32 ? B / 2 : B, RAW_AT = F32 ? 2 * B : 0;
  static constexpr int W_AT = kWarps * RING, W = RAW_AT + kUps * RAW > kUps * B ? RAW_AT + kUps * RAW : kUps * B;
  static constexpr int MAIN = W_AT + W;
  static constexpr int PARTS = RP * 128 * 4;        // of v in fp32, in place of the rings: the CTA's part, then the sum
  static constexpr int CHAIN = F32 ? 128 / CE : 1024 / CE;  // chunks summed on the tensor core
  static constexpr int CTAS = RP == 64 ? 2 : 1, ABOVE = RP == 64 ? 0 : 64;  // this kernel's ranks
  static int smem(int n_slots) { return MAIN + 4 * n_slots; }
  // TMEM columns: two accumulators (of kCols later), then two chunks of x (v later)
  static constexpr int D = RP, A0 = 2 * RP, AW = F32 ? 64 : 32, COLS = RP == 64 ? 256 : 512;
  // never more CTAs an SM than have columns
  static_assert(CTAS * MAIN <= 226 * 1024 && (CTAS + 1) * MAIN > 228 * 1024 && 2 * PARTS <= W_AT && 2 * kSpanRows <= W_AT, "");
  static_assert(A0 + 2 * AW <= COLS && A0 + RP <= COLS && 2 * kCols <= A0 && 2 * kCols == 128, "");
};

struct TileShared {
  uint64_t full[2], empty[2];    // chunks of x in tensor memory
  uint64_t dfull[2], dfree[2];   // accumulators of v
  uint64_t ofull[2], ofree[2];   // and of out
  uint64_t wfull[kUps], vready;
  uint32_t tmem;
  int n_tiles, scan[kWarps], counts[kWarps];
  int rows[128];
};

// Slots of rows 4 i .. 4 i + 3; -1 past the last row.
__device__ __forceinline__ int4 slots4(const AdapterArgs& a, int i, bool vec) {
  const int r = 4 * i;
  if (vec && r + 4 <= a.n_rows) return __ldg(reinterpret_cast<const int4*>(a.slots) + i);
  int4 v = make_int4(-1, -1, -1, -1);
  if (r < a.n_rows) v.x = a.slots[r];
  if (r + 1 < a.n_rows) v.y = a.slots[r + 1];
  if (r + 2 < a.n_rows) v.z = a.slots[r + 2];
  if (r + 3 < a.n_rows) v.w = a.slots[r + 3];
  return v;
}

// The rows' slots into shared memory, kNoSlot where there is none, by `threads` threads; f(slot of four rows) for each four.
template <class F>
__device__ __forceinline__ void load_slots(const AdapterArgs& a, uint16_t* to, int threads, F f) {
  const bool vec = (reinterpret_cast<uintptr_t>(a.slots) & 15) == 0;
  const int quads = (a.n_rows + 127) / 128 * 32;  // whole warps
#pragma unroll 1
  for (int b = threadIdx.x & ~31; b < quads; b += 4 * threads) {
    int4 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) v[u] = slots4(a, b + u * threads + (threadIdx.x & 31), vec);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (b + u * threads >= quads) break;
      auto in = [&](int x) { return x >= 0 && x < a.w.n_slots ? (uint32_t)x : kNoSlot; };
      const uint32_t lo = in(v[u].x) | in(v[u].y) << 16, hi = in(v[u].z) | in(v[u].w) << 16;
      reinterpret_cast<uint2*>(to)[b + u * threads + (threadIdx.x & 31)] = make_uint2(lo, hi);
      f(lo, hi);
    }
  }
}

// The rows of a tile: those of `slot` with ranks [r0, r0 + tile_rows) among its rows. Warp w looks through a
// share of the rows, a lane through four at a time. Rank i of the tile goes to row i / 4 of warp i % 4, so
// that a small tile keeps all warps busy.
__device__ __forceinline__ int find_rows(const AdapterArgs& a, const uint16_t* slots, int slot, int r0, int tile_rows,
                                         TileShared& s) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int all = (a.n_rows + 127) / 128, rounds = (all + kWarps - 1) / kWarps, first = warp * rounds;
  static_assert(kSpanRows <= kWarps * 128 * 16, "");
  unsigned long long mine = 0;  // bits 4 i .. 4 i + 3: the lane's rows of round i
  const uint32_t both = (uint32_t)slot * 0x10001u;
  for (int i = 0; i < rounds && first + i < all; ++i) {
    const uint2 v = reinterpret_cast<const uint2*>(slots)[(first + i) * 32 + lane];
    const uint32_t x = v.x ^ both, y = v.y ^ both;
    const uint32_t m = (uint32_t)!(x & 0xffff) | (uint32_t)!(x >> 16) << 1 | (uint32_t)!(y & 0xffff) << 2 | (uint32_t)!(y >> 16) << 3;
    mine |= (unsigned long long)m << (4 * i);
  }
  const int count = __reduce_add_sync(0xffffffffu, __popcll(mine));
  if (lane == 0) s.counts[warp] = count;
  workers_sync();
  int at = -r0, total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) at += s.counts[w];
    total += s.counts[w];
  }
  if (count && at < tile_rows && at + count > 0) {
    for (int i = 0; i < rounds && at < tile_rows; ++i) {
      const uint32_t m = (uint32_t)(mine >> (4 * i)) & 15;
      const uint32_t b0 = __ballot_sync(0xffffffffu, m & 1), b1 = __ballot_sync(0xffffffffu, m & 2),
                     b2 = __ballot_sync(0xffffffffu, m & 4), b3 = __ballot_sync(0xffffffffu, m & 8);
      const uint32_t below = (1u << lane) - 1;
      int rank = at + __popc(b0 & below) + __popc(b1 & below) + __popc(b2 & below) + __popc(b3 & below);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (m >> e & 1) {
          if (rank >= 0 && rank < tile_rows) s.rows[(rank & 3) * 32 + (rank >> 2)] = 4 * ((first + i) * 32 + lane) + e;
          ++rank;
        }
      at += __popc(b0) + __popc(b1) + __popc(b2) + __popc(b3);
    }
  }
  workers_sync();
  return min(tile_rows, total - r0);
}

template <class T, int RP, bool VX, bool VY>
__global__ void __launch_bounds__(kTT, Cfg<T, RP>::CTAS) adapters_tile_kernel(const __grid_constant__ AdapterArgs a,
                                                                             const int tile_rows) {
  using G = Cfg<T, RP>;
  constexpr int F32 = G::F32, E = G::E, NS = G::NS;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ TileShared s;
  int* start = reinterpret_cast<int*>(smem + G::MAIN);  // [n_slots]: first a slot's rows, then its first tile
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int C = (int)cg::this_cluster().num_blocks(), rank_c = (int)cg::this_cluster().block_rank();
  const int cluster = blockIdx.x / C, n_clusters = gridDim.x / C;
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.full[i], kWarps);
      mbar_init(&s.empty[i], 1);
      mbar_init(&s.dfull[i], 1);
      mbar_init(&s.dfree[i], kWarps);
      mbar_init(&s.ofull[i], 1);
      mbar_init(&s.ofree[i], kWarps);
    }
    for (int i = 0; i < kUps; ++i) mbar_init(&s.wfull[i], 1);
    mbar_init(&s.vready, kWarps);
    fence_barrier_init();
  }
  for (int i = tid; i < a.w.n_slots; i += kTT) start[i] = 0;
  pdl_wait();
  // The kernels before this one have left the tensor memory, and the next one does not start before this
  // one has its own: neither waits for columns while the other waits for it to end.
  if (warp == kWarps) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s.tmem)), "r"(G::COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_before();
  __syncthreads();
  tc_after();
  pdl_launch_dependents();
  const uint32_t tmem = s.tmem;

  // ---- tiles: rows of every slot, then the first tile of each ----
  uint16_t* slots = reinterpret_cast<uint16_t*>(smem);  // while the rings are empty
  load_slots(a, slots, kTT, [&](uint32_t x, uint32_t y) {
    auto count = [&](uint32_t v, int n) {
      if (v != kNoSlot) atomicAdd(&start[v], n);
    };
    const bool same = x == y && x >> 16 == (x & 0xffff);
    const uint32_t lead = __shfl_sync(0xffffffffu, x, 0);
    // mostly rows of one slot follow one another
    if (__all_sync(0xffffffffu, same && x == lead)) {
      if (lane == 0) count(x & 0xffff, 128);
    } else if (same) {
      count(x & 0xffff, 4);
    } else {
      count(x & 0xffff, 1);
      count(x >> 16, 1);
      count(y & 0xffff, 1);
      count(y >> 16, 1);
    }
  });
  __syncthreads();
  if (warp < kWarps) {
    int base = 0;
    for (int b = 0; b < a.w.n_slots; b += kWorkers) {
      const int i = b + tid;
      int n = 0;
      const int rank = i < a.w.n_slots ? a.w.meta[i].rank : 0;
      if (rank > G::ABOVE && rank <= RP) n = (start[i] + tile_rows - 1) / tile_rows;
      int incl = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
      }
      if (lane == 31) s.scan[warp] = incl;
      workers_sync();
      int before = base, all = 0;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        if (w < warp) before += s.scan[w];
        all += s.scan[w];
      }
      if (i < a.w.n_slots) start[i] = before + incl - n;
      base += all;
      workers_sync();
    }
    if (tid == 0) s.n_tiles = base;
  }
  __syncthreads();
  const int n_tiles = s.n_tiles;

  bool ok = true;
  auto wait = [&](uint64_t* bar, uint32_t n, uint32_t code) {  // for the bar's n-th completion
    if (ok) ok = wait_rolled(bar, n & 1, a.err, code);
    __syncwarp();
  };
  uint32_t nc = 0, nd = 0, no = 0, nv = 0, nw = 0;  // chunks, accumulators of v and out, tiles, copies of weights so far
  const uint32_t sbase = smem_u32(smem);
  // this CTA's chunks of k and its columns of out
  const int ct = (a.w.k + G::CE - 1) / G::CE, q0 = ct * rank_c / C, q1 = ct * (rank_c + 1) / C, nq = q1 - q0;
  const int nu8 = (a.w.n + 7) / 8, n0 = (int)((int64_t)nu8 * rank_c / C) * 8,
            n1 = min(a.w.n, (int)((int64_t)nu8 * (rank_c + 1) / C) * 8), nt = (max(0, n1 - n0) + kCols - 1) / kCols;

  const uint32_t on = warp == kWarps ? elect_lane() : 0;
  for (int tile = cluster; tile < n_tiles; tile += n_clusters) {
    int lo = 0, hi = a.w.n_slots - 1;  // the last slot that starts at or before the tile
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (start[mid] <= tile) lo = mid;
      else hi = mid - 1;
    }
    const int slot = lo, r16 = (a.w.meta[slot].rank + 15) / 16 * 16;
    const uint16_t* down = a.w.down + (int64_t)slot * a.w.rp * a.w.kp;
    const uint16_t* up = a.w.up + (int64_t)slot * a.w.rp * a.w.n;

    if (warp < kWarps) {
      if (tile != cluster) {  // the rings have been in use
        load_slots(a, slots, kWorkers, [](uint32_t, uint32_t) {});
        workers_sync();
      }
      const int cnt = find_rows(a, slots, slot, (tile - start[slot]) * tile_rows, tile_rows, s);
      const int row = warp * 32 + lane;
      const uint32_t tlane = tmem + ((uint32_t)(warp * 32) << 16);
      // Blocks of the ring are 32 rows x 128 bytes, piece p of row r at r * 128 + (p ^ r & 7) * 16. A lane
      // fetches piece lane % 8 of the rows lane / 8 + 4 j.
      uint8_t* ring = smem + warp * G::RING;
      const uint32_t ring_at = sbase + warp * G::RING;
      const int piece = lane & 7, top = lane >> 3;
      const uint32_t put0 = top * 128 + ((piece ^ top) << 4), put1 = top * 128 + ((piece ^ top ^ 4) << 4);  // even, odd j
      // ---- fetch x and down ----
      const int first = q0 * G::CE + piece * E;
      // the lane's rows that there are, the first ones of eight
      const int mine = min(8, max(0, (cnt - warp + kWarps - 1) / kWarps - top + 3) / 4);
      const T* xp[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        xp[j] = reinterpret_cast<const T*>(a.x) + (j < mine ? s.rows[warp * 32 + 4 * j + top] : 0) * a.ldx + first;
      uint32_t to = 0;  // the place in the ring that is filled next
      auto fetch = [&](int q) {
        const int left = a.w.k - first - q * G::CE;  // elements up to the row's end
        if (VX && left >= E) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (j < mine) copy16(ring_at + to + (j & 1 ? put1 : put0) + j * 512, xp[j] + q * G::CE);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (j < mine) copy_single(ring + to + (j & 1 ? put1 : put0) + j * 512, xp[j] + q * G::CE, left);
        }
      };
      // where the pieces of weights that a thread has of a chunk go
      constexpr int NB = F32 ? RP * 4 / kWorkers : 1;
      uint32_t bat[NB];
#pragma unroll
      for (int i = 0; i < NB; ++i) bat[i] = ((tid + i * kWorkers) / r16 * 2 * r16 + (tid + i * kWorkers) % r16) * 16;
      // chunk q is here: into the operands of the products
      uint32_t at = 0;  // the place that is read next
      auto ready = [&](int q) {
        const uint32_t b = nc & 1, to = tlane + G::A0 + b * G::AW;
        const uint8_t* from = ring + at + lane * 128;
        if (nc >= 2) wait(&s.empty[b], nc / 2 - 1, DEV_TIMEOUT_EMPTY);
        tc_after();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t x[16];
#pragma unroll
          for (int p = 0; p < 4; ++p) {
            const uint4 v = *reinterpret_cast<const uint4*>(from + ((h * 4 + p) ^ (lane & 7)) * 16);
            x[4 * p] = v.x, x[4 * p + 1] = v.y, x[4 * p + 2] = v.z, x[4 * p + 3] = v.w;
          }
          st16(to + h * 16, x);  // fp32: the tensor core reads the upper 19 bits
          if constexpr (F32) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const float f = __uint_as_float(x[e]) - __uint_as_float(x[e] & 0xffffe000u);
              x[e] = __float_as_uint(f) + 0x1000u;  // to the nearest
            }
            st16(to + 32 + h * 16, x);
          }
        }
        if constexpr (F32) {  // 16-byte pieces of weights, each of which becomes two of fp32
          wait(&s.wfull[(nw + q) % kUps], (nw + q) / kUps, DEV_TIMEOUT_FULL);
          const uint4* raw = reinterpret_cast<const uint4*>(smem + G::W_AT + G::RAW_AT + (nw + q) % kUps * G::RAW);
          uint8_t* wbase = smem + G::W_AT + b * G::B;
          const int items = r16 * 4;
#pragma unroll
          for (int i = 0; i < NB; ++i) {
            const int it = tid + i * kWorkers;
            if (it >= items) continue;
            const uint4 t = raw[it];
            uint8_t* w = wbase + bat[i];
            const float2 f0 = __half22float2(u32_as_h2(t.x)), f1 = __half22float2(u32_as_h2(t.y)),
                         f2 = __half22float2(u32_as_h2(t.z)), f3 = __half22float2(u32_as_h2(t.w));
            *reinterpret_cast<float4*>(w) = make_float4(f0.x, f0.y, f1.x, f1.y);
            *reinterpret_cast<float4*>(w + r16 * 16) = make_float4(f2.x, f2.y, f3.x, f3.y);
          }
          proxy_fence();
        }
        wait_st();
        tc_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.full[b]);
        ++nc;
      };
      float v[RP];  // this thread's row
#pragma unroll
      for (int j = 0; j < RP; ++j) v[j] = 0.f;
      auto drain = [&] {
        const uint32_t from = tlane + (nd & 1) * G::D;
        wait(&s.dfull[nd & 1], nd >> 1, DEV_TIMEOUT_DRAIN);
        tc_after();
#pragma unroll
        for (int h = 0; h < RP; h += 16) {
          if (h >= r16) continue;
          float t[16];
          ld8(from + h, t);
          ld8(from + h + 8, t + 8);
          wait_ld();
#pragma unroll
          for (int e = 0; e < 16; ++e) v[h + e] += t[e];
        }
        tc_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.dfree[nd & 1]);
        ++nd;
      };
      // one place for all fetches: the chunks NS - 1 ahead, before the first only those
      int drained = 0;
#pragma unroll 1
      for (int q = 1 - NS; q < nq; ++q) {
        if (q >= 0) {
          copies_wait<NS - 2>();
          __syncwarp();  // the lanes' copies, and what they have read of the block that is next
        }
        if (q + NS - 1 < nq) fetch(q + NS - 1);
        copies_commit();
        to = to == (NS - 1) * 4096 ? 0 : to + 4096;
        if (q < 0) continue;
        ready(q);
        at = at == (NS - 1) * 4096 ? 0 : at + 4096;
        if (q == (drained + 1) * G::CHAIN && q + 1 < nq) {  // the next chain is under way
          drain();
          ++drained;
        }
      }
#pragma unroll 1
      while (drained * G::CHAIN < nq) {
        drain();
        ++drained;
      }
      copies_wait<0>();
      workers_sync();  // the parts take the rings' place
      // ---- v from the cluster's parts ----
      float* parts = reinterpret_cast<float*>(smem);  // [column][row]
#pragma unroll
      for (int j = 0; j < RP; ++j)
        if (j < r16) parts[j * 128 + row] = v[j];
      cluster_arrive();
      cluster_wait();
      // each CTA adds up some columns, and all get the sums
      float* sums = reinterpret_cast<float*>(smem + G::PARTS);
      for (int i = r16 * rank_c / C * 32 + tid; i < r16 * (rank_c + 1) / C * 32; i += kWorkers) {
        float4 p[8], t = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int d = 0; d < 8; ++d)
          if (d < C) p[d] = *cg::this_cluster().map_shared_rank(reinterpret_cast<float4*>(parts) + i, d);
#pragma unroll
        for (int d = 0; d < 8; ++d)
          if (d < C) t = make_float4(t.x + p[d].x, t.y + p[d].y, t.z + p[d].z, t.w + p[d].w);
#pragma unroll
        for (int d = 0; d < 8; ++d)
          if (d < C) *cg::this_cluster().map_shared_rank(reinterpret_cast<float4*>(sums) + i, d) = t;
      }
      cluster_arrive();
      cluster_wait();
      float most = 0.f;
#pragma unroll
      for (int j = 0; j < RP; ++j) {
        v[j] = j < r16 ? sums[j * 128 + row] : 0.f;
        most = fmaxf(most, fabsf(v[j]));
      }
      workers_sync();  // y takes the sums' place
      // 2^(13 - exponent of the row's largest), and its inverse; no row is lifted by more than 2^110
      const int ex = max(30, (int)(__float_as_uint(most) >> 23));
      const float lift = __uint_as_float((uint32_t)(127 + 13 - min(ex - 127, 126)) << 23);
      const AdapterMeta meta = a.w.meta[slot];
      const float factor = meta.scale * __uint_as_float((uint32_t)(127 - 13 + min(ex - 127, 126)) << 23) * meta.f1 * meta.f2;
      // ---- y, a block at a time ----
      constexpr int BC = 8 * E, PER = kCols / BC;  // columns of a block, blocks of a tile
      const T* y = reinterpret_cast<const T*>(a.y);
      T* out = reinterpret_cast<T*>(a.out);
      const int blocks = nt * PER;
      auto multiply_v = [&] {
#pragma unroll
        for (int u = 0; u < RP / 8; ++u) {
          if (u * 8 >= r16) continue;
          uint32_t h[4], l[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x0 = v[u * 8 + 2 * e] * lift, x1 = v[u * 8 + 2 * e + 1] * lift;
            const __half2 hh = __floats2half2_rn(x0, x1);
            const float2 hf = __half22float2(hh);
            h[e] = h2_as_u32(hh);
            l[e] = h2_as_u32(__floats2half2_rn(x0 - hf.x, x1 - hf.y));
          }
          st4(tlane + G::A0 + u * 4, h);
          st4(tlane + G::A0 + RP / 2 + u * 4, l);
        }
        wait_st();
        tc_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.vready);
      };
      multiply_v();
      const T* yp[8];
      T* op[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int r = j < mine ? s.rows[warp * 32 + 4 * j + top] : 0;
        yp[j] = y + r * a.ldy + n0 + piece * E;
        op[j] = out + r * a.ldo + n0 + piece * E;
      }
      to = at = 0;
      auto fetch_y = [&](int i) {
        const int left = n1 - n0 - i * BC - piece * E;
        if (VY && left >= E) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (j < mine) copy16(ring_at + to + (j & 1 ? put1 : put0) + j * 512, yp[j] + i * BC);
        } else if (left > 0) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (j < mine) copy_single(ring + to + (j & 1 ? put1 : put0) + j * 512, yp[j] + i * BC, left);
        }
      };
      // ---- out = y + factor * D ----
#pragma unroll 1
      for (int i = 1 - NS; i < blocks; ++i) {
        if (i + NS - 1 < blocks) fetch_y(i + NS - 1);
        copies_commit();
        to = to == (NS - 1) * 4096 ? 0 : to + 4096;
        if (i < 0) continue;
        const uint32_t tile_o = no + i / PER;
        if (i % PER == 0) {
          wait(&s.ofull[tile_o & 1], tile_o >> 1, DEV_TIMEOUT_DRAIN);
          tc_after();
        }
        copies_wait<NS - 1>();
        __syncwarp();
        uint8_t* block = ring + at;
        at = at == (NS - 1) * 4096 ? 0 : at + 4096;
        const uint32_t from = tlane + (tile_o & 1) * kCols + i % PER * BC;
#pragma unroll
        for (int c = 0; c < BC; c += 16) {
          float d[16];
          ld8(from + c, d);
          ld8(from + c + 8, d + 8);
          wait_ld();
          if (i % PER == PER - 1 && c + 16 == BC) {
            tc_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&s.ofree[tile_o & 1]);
          }
#pragma unroll
          for (int p = 0; p < 16 / E; ++p) {
            uint4* w = reinterpret_cast<uint4*>(block + lane * 128 + ((c / E + p) ^ (lane & 7)) * 16);
            uint4 t = *w;
            if constexpr (F32) {
              t.x = __float_as_uint(fmaf(factor, d[4 * p], __uint_as_float(t.x)));
              t.y = __float_as_uint(fmaf(factor, d[4 * p + 1], __uint_as_float(t.y)));
              t.z = __float_as_uint(fmaf(factor, d[4 * p + 2], __uint_as_float(t.z)));
              t.w = __float_as_uint(fmaf(factor, d[4 * p + 3], __uint_as_float(t.w)));
            } else {
              auto add = [&](uint32_t z, int e) {
                const float2 f = __half22float2(u32_as_h2(z));
                return h2_as_u32(__floats2half2_rn(fmaf(factor, d[8 * p + e], f.x), fmaf(factor, d[8 * p + e + 1], f.y)));
              };
              t = make_uint4(add(t.x, 0), add(t.y, 2), add(t.z, 4), add(t.w, 6));
            }
            *w = t;
          }
        }
        __syncwarp();
        const int left = n1 - n0 - i * BC - piece * E;
        if (VY && left >= E) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (j < mine) *reinterpret_cast<uint4*>(op[j] + i * BC) = *reinterpret_cast<const uint4*>(block + (j & 1 ? put1 : put0) + j * 512);
        } else if (left > 0) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            if (j >= mine) continue;
            const T* t = reinterpret_cast<const T*>(block + (j & 1 ? put1 : put0) + j * 512);
#pragma unroll
            for (int e = 0; e < E; ++e)
              if (e < left) op[j][i * BC + e] = t[e];
          }
        }
        __syncwarp();  // before the block's place is filled again
      }
      no += nt;
      nw += nq + nt;  // as the products' warp counts
      copies_wait<0>();
      workers_sync();  // before the next tile's rows
    } else {
      // ---- products ----
      const uint32_t lbo = (uint32_t)r16 * 16;
      const uint32_t id1 = idesc_of(F32, r16), id2 = idesc_of(0, kCols);
      // copies of weights take the places in turn
      auto expect = [&](uint32_t i, int bytes) {
        if (lane == 0) mbar_arrive_expect_tx(&s.wfull[i % kUps], (uint32_t)bytes);
        __syncwarp();
      };
      auto fetch_down = [&](int q) {  // a chunk's weights as they lie
        const uint32_t i = nw + q;
        if (!ok) return;
        expect(i, r16 * G::CE * 2);
        if (lane == 0)
          bulk_g2s(smem + G::W_AT + G::RAW_AT + i % kUps * G::RAW, down + (int64_t)(q0 + q) * G::CE * r16,
                   (uint32_t)(r16 * G::CE * 2), &s.wfull[i % kUps]);
      };
      auto fetch_up = [&](int t) {  // columns n0 + 64 t ...
        const uint32_t i = nw + t;
        const int c0 = n0 + t * kCols, rows = min(kCols, n1 - c0), ch = r16 / 8;
        if (!ok) return;
        expect(i, ch * rows * 16);
        if (lane < ch)
          bulk_g2s(smem + G::W_AT + i % kUps * G::B + lane * kCols * 16, up + ((int64_t)lane * a.w.n + c0) * 8,
                   (uint32_t)(rows * 16), &s.wfull[i % kUps]);
      };
      int fetched = 0;
      for (; fetched < min(kUps, nq); ++fetched) fetch_down(fetched);
#pragma unroll 1
      for (int q = 0; q < nq; ++q, ++nc) {
        const uint32_t b = nc & 1;
        if (q % G::CHAIN == 0 && nd >= 2) wait(&s.dfree[nd & 1], (nd >> 1) - 1, DEV_TIMEOUT_DRAIN);
        if (!F32) wait(&s.wfull[(nw + q) % kUps], (nw + q) / kUps, DEV_TIMEOUT_FULL);
        wait(&s.full[b], nc / 2, DEV_TIMEOUT_FULL);
        ok = __all_sync(0xffffffffu, ok);
        tc_after();
        if (ok) {
          const uint64_t bd = desc_blocks(sbase + G::W_AT + (F32 ? b : (nw + q) % kUps) * G::B, lbo);
#pragma unroll
          for (int part = F32; part >= 0; --part)  // the low part first
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
              mma<F32>(on, tmem + (nd & 1) * G::D, tmem + G::A0 + b * G::AW + part * 32 + ks * 8, bd + (uint64_t)(ks * 2 * lbo >> 4),
                       id1, q % G::CHAIN || part < F32 || ks);
          commit(on, &s.empty[b]);
        }
        if ((q + 1) % G::CHAIN == 0 || q + 1 == nq) {
          if (ok) commit(on, &s.dfull[nd & 1]);
          ++nd;
        }
        // into the place that the threads have read, for the chunk at hand (fp32), or the product before this one
        if ((F32 || q > 0) && fetched < nq) {
          if (!F32) wait(&s.empty[b ^ 1], (nc - 1) / 2, DEV_TIMEOUT_EMPTY);
          ok = __all_sync(0xffffffffu, ok);
          fetch_down(fetched++);
        }
      }
      auto land = [&] {  // copies in flight land before the CTA's shared memory goes away
        if (!ok)
          for (int t = max(0, fetched - kUps); t < fetched; ++t)
            mbar_wait(&s.wfull[(nw + t) % kUps], (nw + t) / kUps & 1, nullptr, 0);
      };
      land();
      nw += nq;
      // the weights' places are free once the last accumulator is there
      if (nq > 0) wait(&s.dfull[(nd - 1) & 1], (nd - 1) >> 1, DEV_TIMEOUT_DRAIN);
      ok = __all_sync(0xffffffffu, ok);
      for (fetched = 0; fetched < min(kUps, nt); ++fetched) fetch_up(fetched);
      for (int i = 0; i < 2; ++i) {  // as above
        cluster_arrive();
        cluster_wait();
      }
      wait(&s.vready, nv, DEV_TIMEOUT_SMEM);
#pragma unroll 1
      for (int t = 0; t < nt; ++t, ++no) {
        const uint32_t b = no & 1;
        if (no >= 2) wait(&s.ofree[b], (no >> 1) - 1, DEV_TIMEOUT_DRAIN);
        wait(&s.wfull[(nw + t) % kUps], (nw + t) / kUps, DEV_TIMEOUT_FULL);
        ok = __all_sync(0xffffffffu, ok);
        tc_after();
        if (ok) {
          const uint64_t bd = desc_blocks(sbase + G::W_AT + (nw + t) % kUps * G::B, kCols * 16);
#pragma unroll 1
          for (int part = 1; part >= 0; --part)
#pragma unroll 1
            for (int ks = 0; ks < r16 / 16; ++ks)
              mma<0>(on, tmem + b * kCols, tmem + G::A0 + part * (RP / 2) + ks * 8, bd + (uint64_t)(ks * 2 * kCols), id2,
                     part < 1 || ks);
          commit(on, &s.ofull[b]);
        }
        if (t > 0 && fetched < nt) {
          wait(&s.ofull[b ^ 1], (no - 1) >> 1, DEV_TIMEOUT_DRAIN);
          ok = __all_sync(0xffffffffu, ok);
          fetch_up(fetched++);
        }
      }
      land();
      nw += nt;
      if (nt > 0) wait(&s.ofull[(no - 1) & 1], (no - 1) >> 1, DEV_TIMEOUT_DRAIN);  // the places are free again
    }
    ++nv;
  }
  if (RP == 64 && a.out != a.y && warp < kWarps)
    for (int r = blockIdx.x; r < a.n_rows; r += gridDim.x) {
      const int v = a.slots[r];
      if (v >= 0 && v < a.w.n_slots && a.w.meta[v].rank > 0) continue;
      const T* y = reinterpret_cast<const T*>(a.y) + r * a.ldy;
      T* o = reinterpret_cast<T*>(a.out) + r * a.ldo;
      for (int j = tid; j < a.w.n; j += kWorkers) o[j] = y[j];
    }
  tc_before();
  __syncthreads();
  tc_after();
  if (warp == kWarps)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(G::COLS) : "memory");
}

template <class T, int RP, bool VX, bool VY>
cudaError_t launch(const AdapterArgs& a, int num_sms, cudaStream_t s) {
  using G = Cfg<T, RP>;
  int dev = 0;
  cudaGetDevice(&dev);
  const int smem = G::smem(a.w.n_slots);
  if (cudaError_t e = ensure_smem_attr(adapters_tile_kernel<T, RP, VX, VY>, G::smem(kAdapterMaxSlots), dev)) return e;
  const int ctas = num_sms * (2 * (smem + 3072) <= 228 * 1024 ? G::CTAS : 1);
  // Clusters of eight, and the smallest tiles whose CTAs all run at once: a CTA's steps over k and n, more than its
  // rows, are what a call of few rows takes. Where even tiles of 128 rows are too many, smaller clusters.
  auto tiles = [&](int rows) { return (a.n_rows + rows - 1) / rows; };
  int tile_rows = 128, cluster = 8;
  while (tile_rows > 16 && tiles(tile_rows / 2) * cluster <= ctas) tile_rows /= 2;
  while (cluster > 4 && tiles(tile_rows) * cluster > ctas) cluster /= 2;
  const int most = a.n_rows / tile_rows + std::min(a.w.n_slots, a.n_rows);  // tiles
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(std::min(std::max(1, ctas / cluster), most) * cluster));
  cfg.blockDim = dim3(kTT);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)cluster;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, adapters_tile_kernel<T, RP, VX, VY>, a, tile_rows);
}

template <class T, int RP>
cudaError_t launch_rank(const AdapterArgs& a, int num_sms, cudaStream_t s) {
  auto on = [](const void* p, int64_t ld, int bytes) {
    return (uintptr_t)p % bytes == 0 && ld * (int)sizeof(T) % bytes == 0;
  };
  const bool vx = on(a.x, a.ldx, 16), vy = on(a.y, a.ldy, 16) && on(a.out, a.ldo, 16);
  if (vx) return vy ? launch<T, RP, true, true>(a, num_sms, s) : launch<T, RP, true, false>(a, num_sms, s);
  return vy ? launch<T, RP, false, true>(a, num_sms, s) : launch<T, RP, false, false>(a, num_sms, s);
}

}  // namespace

cudaError_t adapters_tile_launch(const AdapterArgs& a, int num_sms, cudaStream_t s) {
  for (int64_t r = 0; r < a.n_rows; r += kSpanRows) {
    AdapterArgs b = a;
    const int esz = a.x16 ? 2 : 4;
    b.n_rows = (int)std::min<int64_t>(kSpanRows, a.n_rows - r);
    b.slots = a.slots + r;
    b.x = (const uint8_t*)a.x + r * a.ldx * esz;
    b.y = (const uint8_t*)a.y + r * a.ldy * esz;
    b.out = (uint8_t*)a.out + r * a.ldo * esz;
    cudaError_t e;
    // Which ranks the rows' slots have is not known here (a captured call is replayed with others). Two launches where
    // a set may have large ones: 4096 rows of ranks 8 to 128 (k = 11008) 233 us, in one launch for all ranks 278.
    e = a.x16 ? launch_rank<__half, 64>(b, num_sms, s) : launch_rank<float, 64>(b, num_sms, s);
    if (!e && a.w.rp > 64) e = a.x16 ? launch_rank<__half, 128>(b, num_sms, s) : launch_rank<float, 128>(b, num_sms, s);
    if (e) return e;
  }
  return cudaSuccess;
}

}  // namespace rb
