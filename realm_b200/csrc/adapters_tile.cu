// Low-rank adapters for many rows (prompts): the function of adapters.cu, tile by tile on
// the tensor cores. A tile is up to `tile_rows` <= 128 rows of one adapter; a cluster of CTAs has it,
// splits k for v = down x and n for up v, and exchanges its parts of v through distributed
// shared memory in between, so that one kernel reads x once and writes out once.
//
//   v = down x: D[128 rows][rank] += X[128][chunk] down[rank][chunk]^T, chunks of 128 bytes a
//     row. Eight warps fetch rows (wherever they lie) and weights, the ninth issues
//     tcgen05.mma. fp16 rows are multiplied as they are (kind::f16). An fp32 x is two tf32
//     parts, x = hi + lo (22 bits), the low one first, and the fp16 weights are exact in tf32.
//   out = y + scale up v: v is brought to a power of two near 2^13 row by row and split into fp16
//     hi + lo (22 bits of the row's largest); D[128 rows][128 columns] = v up^T, with up's
//     tiles copied in bulk. A warp turns 32 x 32 results around in shared memory, so that y
//     and out are read and written in whole lines.
//
// The tensor core cuts a running sum off (towards 0) after every instruction, so fp32 rows sum at
// most 256 elements of k there; the sums of these chains are added in registers, with rounding.
//
// Bound by memory: x and y are read and out is written once, which is most of the bytes.
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

constexpr int kWorkers = 256, kTT = kWorkers + 32;  // threads that fetch and finish; a warp for the products
constexpr int kSpanRows = 8192;                     // rows of a launch
constexpr int kCols = 128;                          // columns of out a product covers
constexpr int kStagePitch = 36;                     // floats between rows of a turned block

__device__ __forceinline__ uint64_t desc_of(uint32_t saddr, uint32_t lbo, uint32_t sbo, uint64_t layout) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)((lbo >> 4) & 0x3FFFu) << 16) |
         ((uint64_t)((sbo >> 4) & 0x3FFFu) << 32) | (1ull << 46) | (layout << 61);
}
// K-major operands: rows of 128 bytes with the 128-byte swizzle; or 8 x 16-byte blocks, `lbo` apart along K
__device__ __forceinline__ uint64_t desc_rows(uint32_t saddr) { return desc_of(saddr, 16, 1024, 2); }
__device__ __forceinline__ uint64_t desc_blocks(uint32_t saddr, uint32_t lbo) { return desc_of(saddr, lbo, 128, 0); }
__device__ __forceinline__ uint32_t idesc_of(int tf32, int n) {
  return (1u << 4) | (tf32 ? (2u << 7) | (2u << 10) : 0u) | ((uint32_t)(n >> 3) << 17) | (8u << 24);
}
template <int TF32>
__device__ __forceinline__ void mma(uint32_t on, uint32_t d, uint64_t ad, uint64_t bd, uint32_t id, uint32_t acc) {
  if constexpr (TF32)
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::tf32 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(ad), "l"(bd), "r"(id), "r"(acc), "r"(on)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(ad), "l"(bd), "r"(id), "r"(acc), "r"(on)
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
// 8 and 32 columns of this thread's TMEM lane; valid after wait_ld()
__device__ __forceinline__ void ld8(uint32_t ta, float* r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7])
               : "r"(ta)
               : "memory");
}
// 16 (or 4) bytes to shared memory, the last 16 - n of them zero
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, int n) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src, int n) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void workers_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }

// T: type of the rows. RP: ranks up to 64 (two CTAs an SM) or 128.
template <class T, int RP>
struct Cfg {
  static constexpr int F32 = sizeof(T) == 4;
  static constexpr int E = 16 / (int)sizeof(T);     // elements of 16 bytes
  static constexpr int CE = 8 * E;                  // of a chunk: 128 bytes a row
  static constexpr int A = 128 * 128;               // bytes of a chunk's rows (one part)
  static constexpr int B = RP * 128;                // and of its weights
  // fp32: the rows as they are (the tensor core reads their upper 19 bits), then the low parts and weights
  // of two chunks, which threads make; fp16: rows and weights
  static constexpr int STAGE = F32 ? A : A + B;
  static constexpr int NS = F32 ? (RP == 64 ? 3 : 5) : (RP == 64 ? 4 : 6);
  static constexpr int AHEAD = F32 && RP == 64 ? 2 : NS - 2;  // chunks on their way
  static constexpr int LOW = F32 ? A + B : 0;
  static constexpr int RING = NS * STAGE + 2 * LOW;
  static constexpr int CHAIN = F32 ? 256 / CE : 1024 / CE;  // chunks summed on the tensor core
  // after the chunks: v (hi, lo), two tiles of up, and the parts of v or the turned blocks
  static constexpr int V = RP * 256;                // bytes of v, one part: [RP / 8][128 rows][16]
  static constexpr int UP = RP * 2 * kCols;
  static constexpr int P_AT = 2 * V + 2 * UP;
  static constexpr int TURN = 8 * 32 * kStagePitch * 4;
  static constexpr int PARTS = RP * 128 * 4;
  static constexpr int MAIN0 = P_AT + (TURN > PARTS ? TURN : PARTS);
  static constexpr int MAIN = MAIN0 > RING ? MAIN0 : RING;
  static constexpr int CTAS = RP == 64 ? 2 : 1;
  static int smem(int n_slots) { return MAIN + 4 * n_slots; }
  // TMEM: 256 columns for each of up to two CTAs an SM, never a third
  static_assert(CTAS * MAIN <= 226 * 1024 && 3 * MAIN > 228 * 1024 && 2 * V == PARTS, "");
};

struct TileShared {
  uint64_t full[6], empty[6], dfull[2], dfree[2], upfull[2], vready;
  uint32_t tmem;
  int n_tiles, scan[8], counts[8];
  int rows[128];
  float most[2][128];
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

// The rows of a tile: those of `slot` with ranks [r0, r0 + tile_rows) among its rows. Warp w has
// the rows [w seg, (w + 1) seg), a lane four at a time.
__device__ __noinline__ int find_rows(const AdapterArgs& a, int slot, int r0, int tile_rows, TileShared& s) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rounds = (a.n_rows + 8 * 128 - 1) / (8 * 128), i0 = warp * rounds * 32 + lane;
  const bool vec = (reinterpret_cast<uintptr_t>(a.slots) & 15) == 0;
  uint32_t mine = 0;  // bits 4 i .. 4 i + 3: the lane's rows of round i
#pragma unroll 4
  for (int i = 0; i < rounds; ++i) {
    const int4 v = slots4(a, i0 + 32 * i, vec);
    mine |= ((uint32_t)(v.x == slot) | (uint32_t)(v.y == slot) << 1 | (uint32_t)(v.z == slot) << 2 |
             (uint32_t)(v.w == slot) << 3)
            << (4 * i);
  }
  const int count = __reduce_add_sync(0xffffffffu, __popc(mine));
  if (lane == 0) s.counts[warp] = count;
  workers_sync();
  int at = -r0, total = 0;
#pragma unroll
  for (int w = 0; w < 8; ++w) {
    if (w < warp) at += s.counts[w];
    total += s.counts[w];
  }
  if (count && at < tile_rows && at + count > 0) {
    for (int i = 0; i < rounds; ++i) {
      const uint32_t m = mine >> (4 * i) & 15;
      int incl = __popc(m);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
      }
      int rank = at + incl - __popc(m);
      for (int e = 0; e < 4; ++e)
        if (m >> e & 1) {
          if (rank >= 0 && rank < tile_rows) s.rows[rank] = 4 * (i0 + 32 * i) + e;
          ++rank;
        }
      at += __shfl_sync(0xffffffffu, incl, 31);
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
  extern __shared__ __align__(1024) uint8_t smem[];  // the swizzle follows the address bits
  __shared__ TileShared s;
  int* start = reinterpret_cast<int*>(smem + G::MAIN);  // [n_slots]: first a slot's rows, then its first tile
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int C = (int)cg::this_cluster().num_blocks(), rank_c = (int)cg::this_cluster().block_rank();
  const int cluster = blockIdx.x / C, n_clusters = gridDim.x / C;
  if (smem_u32(smem) & 1023) {  // the same in every CTA
    report_error(a.err, DEV_TIMEOUT_SMEM);
    return;
  }
  if (tid == 0) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(&s.full[i], 8);  // warps
      mbar_init(&s.empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.dfull[i], 1);
      mbar_init(&s.dfree[i], 8);
      mbar_init(&s.upfull[i], 1);
    }
    mbar_init(&s.vready, 8);
    fence_barrier_init();
  }
  for (int i = tid; i < a.w.n_slots; i += kTT) start[i] = 0;
  pdl_wait();
  // The kernels before this one have left the tensor memory, and the next one does not start before this
  // one has its own: neither waits for columns while the other waits for it to end.
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s.tmem)), "r"(256)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_before();
  __syncthreads();
  tc_after();
  pdl_launch_dependents();
  const uint32_t tmem = s.tmem;

  // ---- tiles: rows of every slot, then the first tile of each ----
  {
    const bool vec = (reinterpret_cast<uintptr_t>(a.slots) & 15) == 0;
    auto count = [&](int v, int n) {
      if (v >= 0 && v < a.w.n_slots) atomicAdd(&start[v], n);
    };
    const int quads = (a.n_rows + 3) / 4;
#pragma unroll 4
    for (int b = warp * 32; b < quads; b += kTT) {
      const int4 v = b + lane < quads ? slots4(a, b + lane, vec) : make_int4(-1, -1, -1, -1);
      const bool same = v.x == v.y && v.x == v.z && v.x == v.w;
      const int lead = __shfl_sync(0xffffffffu, v.x, 0);
      // mostly rows of one slot follow one another
      if (__all_sync(0xffffffffu, same && v.x == lead)) {
        if (lane == 0) count(v.x, 128);
      } else if (same) {
        count(v.x, 4);
      } else {
        count(v.x, 1);
        count(v.y, 1);
        count(v.z, 1);
        count(v.w, 1);
      }
    }
  }
  __syncthreads();
  if (warp < 8) {
    int base = 0;
    for (int b = 0; b < a.w.n_slots; b += kWorkers) {
      const int i = b + tid;
      int n = 0;
      if (i < a.w.n_slots && a.w.meta[i].rank > 0) n = (start[i] + tile_rows - 1) / tile_rows;
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
      for (int w = 0; w < 8; ++w) {
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
    if (ok) ok = mbar_wait(bar, n & 1, a.err, code);
    __syncwarp();
  };
  uint32_t nc = 0, nd = 0, nv = 0, nu = 0;  // chunks, accumulators, tiles and tiles of up so far
  const uint32_t sbase = smem_u32(smem);
  // this CTA's chunks of k and its columns of out
  const int ct = (a.w.k + G::CE - 1) / G::CE, q0 = ct * rank_c / C, q1 = ct * (rank_c + 1) / C, nq = q1 - q0;
  const int nu8 = (a.w.n + 7) / 8, n0 = (int)((int64_t)nu8 * rank_c / C) * 8,
            n1 = min(a.w.n, (int)((int64_t)nu8 * (rank_c + 1) / C) * 8), nt = (max(0, n1 - n0) + kCols - 1) / kCols;

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

    if (warp < 8) {
      const int cnt = find_rows(a, slot, (tile - start[slot]) * tile_rows, tile_rows, s);
      // ---- fetch x and down ----
      const int piece = tid & 7, rg = tid >> 3;  // rows rg + 32 j
      const T* xp[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        xp[j] = rg + 32 * j < cnt
                    ? reinterpret_cast<const T*>(a.x) + s.rows[rg + 32 * j] * a.ldx + q0 * G::CE + piece * E
                    : nullptr;
      // where the piece goes; row & 7 is the same for all four, whose places are 4096 bytes apart
      const uint32_t at = (uint32_t)rg * 128 + ((piece ^ (rg & 7)) << 4);
      constexpr int NB = RP * (F32 ? 4 : 8) / kWorkers;  // 16-byte pieces of weights a thread has of a chunk
      const int items = r16 * (F32 ? 4 : 8);
      const uint4* wp = reinterpret_cast<const uint4*>(down) + (int64_t)q0 * items + tid;
      uint4 wb[NB];  // fp32: the next chunk's
      uint32_t bat[NB];
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const int it = tid + i * kWorkers;
        bat[i] = F32 ? (uint32_t)(it / r16 * 2 * r16 + it % r16) * 16 : (uint32_t)it * 16;
      }
      // chunk q of this CTA, the ch-th of all, is on its way
      auto fetch = [&](int q, uint32_t ch) {
        const uint32_t st = ch % NS;
        if (ch >= NS) wait(&s.empty[st], ch / NS - 1, DEV_TIMEOUT_EMPTY);
        const uint32_t base = sbase + st * G::STAGE + at;
        const int left = a.w.k - (q0 + q) * G::CE - piece * E;  // elements up to the row's end
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (!xp[j]) continue;  // rows of the products stay apart
          const T* p = xp[j] + (int64_t)q * G::CE;
          if constexpr (VX) {
            const int n = min(max(left, 0), E) * (int)sizeof(T);
            copy16(base + j * 4096, n ? p : xp[j], n);
          } else if constexpr (F32) {
#pragma unroll
            for (int e = 0; e < E; ++e) copy4(base + j * 4096 + e * 4, e < left ? p + e : xp[j], e < left ? 4 : 0);
          } else {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t lo = 2 * e < left ? __half_as_ushort(p[2 * e]) : 0u, hi = 2 * e + 1 < left ? __half_as_ushort(p[2 * e + 1]) : 0u;
              w[e] = lo | hi << 16;
            }
            *reinterpret_cast<uint4*>(smem + st * G::STAGE + at + j * 4096) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
        if constexpr (!F32)
#pragma unroll
          for (int i = 0; i < NB; ++i)
            if (tid + i * kWorkers < items) copy16(sbase + st * G::STAGE + G::A + bat[i], wp + (int64_t)q * items + i * kWorkers, 16);
      };
      auto weights = [&](int q) {
#pragma unroll
        for (int i = 0; i < NB; ++i)
          if (tid + i * kWorkers < items) wb[i] = __ldg(wp + (int64_t)q * items + i * kWorkers);
      };
      // the chunk is here: fp32 rows get their low part, and the products may begin
      auto ready = [&](uint32_t ch) {
        const uint32_t st = ch % NS;
        if constexpr (F32) {
          if (ch >= 2) wait(&s.empty[(ch - 2) % NS], (ch - 2) / NS, DEV_TIMEOUT_EMPTY);
          uint8_t* low = smem + NS * G::STAGE + (ch & 1) * G::LOW;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (!xp[j]) continue;
            const uint4 x = *reinterpret_cast<const uint4*>(smem + st * G::STAGE + at + j * 4096);
            const uint32_t v[4] = {x.x, x.y, x.z, x.w};
            uint32_t l[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float f = __uint_as_float(v[e]), g = __uint_as_float(v[e] & 0xffffe000u);
              l[e] = f == g ? 0u : __float_as_uint(f - g) + 0x1000u;  // to the nearest; 0 for infinities
            }
            *reinterpret_cast<uint4*>(low + at + j * 4096) = make_uint4(l[0], l[1], l[2], l[3]);
          }
#pragma unroll
          for (int i = 0; i < NB; ++i) {
            if (tid + i * kWorkers >= items) continue;
            const float2 f0 = __half22float2(u32_as_h2(wb[i].x)), f1 = __half22float2(u32_as_h2(wb[i].y)),
                         f2 = __half22float2(u32_as_h2(wb[i].z)), f3 = __half22float2(u32_as_h2(wb[i].w));
            *reinterpret_cast<float4*>(low + G::A + bat[i]) = make_float4(f0.x, f0.y, f1.x, f1.y);
            *reinterpret_cast<float4*>(low + G::A + bat[i] + r16 * 16) = make_float4(f2.x, f2.y, f3.x, f3.y);
          }
        }
        proxy_fence();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.full[st]);
      };
      const int quarter = warp & 3, half = warp >> 2, row = quarter * 32 + lane, hc = r16 / 2;
      const uint32_t tlane = tmem + ((uint32_t)(quarter * 32) << 16);
      float v[RP / 2];  // this thread's row, columns half * hc + j
#pragma unroll
      for (int j = 0; j < RP / 2; ++j) v[j] = 0.f;
      auto drain = [&] {
        wait(&s.dfull[nd & 1], nd >> 1, DEV_TIMEOUT_DRAIN);
        tc_after();
#pragma unroll
        for (int h = 0; h < RP / 2; h += 16) {
          float t[16];
          if (h < hc) ld8(tlane + (nd & 1) * 128 + half * hc + h, t);
          if (h + 8 < hc) ld8(tlane + (nd & 1) * 128 + half * hc + h + 8, t + 8);
          wait_ld();
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (h + (e & 8) < hc) v[h + e] += t[e];
        }
        tc_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.dfree[nd & 1]);
        ++nd;
      };
      if (F32 && nq > 0) weights(0);
#pragma unroll 1
      for (int q = 0; q < G::AHEAD; ++q) {
        if (q < nq) fetch(q, nc + q);
        copies_commit();
      }
      int drained = 0;
#pragma unroll 1
      for (int q = 0; q < nq; ++q) {
        if (q + G::AHEAD < nq) fetch(q + G::AHEAD, nc + q + G::AHEAD);
        copies_commit();
        copies_wait<G::AHEAD>();
        ready(nc + q);
        if (F32 && q + 1 < nq) weights(q + 1);
        if (q + 1 == (drained + 1) * G::CHAIN + 2 && q + 1 < nq) {  // the next chain is under way
          drain();
          ++drained;
        }
      }
      nc += nq;
      while (drained * G::CHAIN < nq) {
        drain();
        ++drained;
      }
      // ---- v from the cluster's parts ----
      float* parts = reinterpret_cast<float*>(smem + G::P_AT);  // [column][row]; all products have read their operands
#pragma unroll
      for (int j = 0; j < RP / 2; ++j)
        if (j < hc) parts[(half * hc + j) * 128 + row] = v[j];
      cluster_arrive();
      cluster_wait();
      // each CTA adds up some columns, and all get the sums, in place of the chunks
      float* sums = reinterpret_cast<float*>(smem);
      {
        const int j0 = r16 * rank_c / C, j1 = r16 * (rank_c + 1) / C;
#pragma unroll 2
        for (int i = j0 * 128 + tid; i < j1 * 128; i += kWorkers) {
          float t = 0.f;
#pragma unroll 8
          for (int d = 0; d < C; ++d) t += *cg::this_cluster().map_shared_rank(parts + i, d);
#pragma unroll 8
          for (int d = 0; d < C; ++d) *cg::this_cluster().map_shared_rank(sums + i, d) = t;
        }
      }
      cluster_arrive();
      cluster_wait();
#pragma unroll
      for (int j = 0; j < RP / 2; ++j) v[j] = j < hc ? sums[(half * hc + j) * 128 + row] : 0.f;
      float most = 0.f;
#pragma unroll
      for (int j = 0; j < RP / 2; ++j)
        if (j < hc) most = fmaxf(most, fabsf(v[j]));
      s.most[half][row] = most;
      workers_sync();
      most = fmaxf(s.most[0][row], s.most[1][row]);
      // 2^(13 - exponent of the row's largest), and its inverse; no row is lifted by more than 2^110
      const int ex = max(30, (int)(__float_as_uint(most) >> 23));
      const float lift = __uint_as_float((uint32_t)(127 + 13 - min(ex - 127, 126)) << 23);
      const float factor = a.w.meta[slot].scale * __uint_as_float((uint32_t)(127 - 13 + min(ex - 127, 126)) << 23);
#pragma unroll
      for (int u = 0; u < RP / 16; ++u) {
        if (u * 8 >= hc) continue;
        uint32_t h[4], l[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x0 = v[u * 8 + 2 * e] * lift, x1 = v[u * 8 + 2 * e + 1] * lift;
          const __half2 hh = __floats2half2_rn(x0, x1);
          const float2 hf = __half22float2(hh);
          h[e] = h2_as_u32(hh);
          l[e] = h2_as_u32(__floats2half2_rn(x0 == hf.x ? 0.f : x0 - hf.x, x1 == hf.y ? 0.f : x1 - hf.y));
        }
        const int at = ((half * hc / 8 + u) * 128 + row) * 16;
        *reinterpret_cast<uint4*>(smem + at) = make_uint4(h[0], h[1], h[2], h[3]);
        *reinterpret_cast<uint4*>(smem + G::V + at) = make_uint4(l[0], l[1], l[2], l[3]);
      }
      proxy_fence();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.vready);
      // ---- out = y + factor * D ----
      float* turn = reinterpret_cast<float*>(smem + G::P_AT) + warp * 32 * kStagePitch;
      const T* y = reinterpret_cast<const T*>(a.y);
      T* out = reinterpret_cast<T*>(a.out);
      for (int t = 0; t < nt; ++t, ++nd) {
#pragma unroll 1
        for (int b = 0; b < 2; ++b) {
          const int c0 = n0 + t * kCols + half * 64 + b * 32;
          const int col = c0 + (VY ? (lane & 7) * 4 : lane);
          constexpr int NR = VY ? 8 : 32;  // rows a lane has of the turned block
          float4 yv[8];
          if constexpr (VY) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int r = quarter * 32 + i * 4 + (lane >> 3);
              yv[i] = make_float4(0.f, 0.f, 0.f, 0.f);
              if (r < cnt && col < n1) {
                const T* p = y + s.rows[r] * a.ldy + col;
                if (col + 4 <= n1) {
                  if constexpr (F32) {
                    yv[i] = *reinterpret_cast<const float4*>(p);
                  } else {
                    const uint2 w = *reinterpret_cast<const uint2*>(p);
                    const float2 f0 = __half22float2(u32_as_h2(w.x)), f1 = __half22float2(u32_as_h2(w.y));
                    yv[i] = make_float4(f0.x, f0.y, f1.x, f1.y);
                  }
                } else {
                  yv[i].x = (float)p[0];
                  if (col + 1 < n1) yv[i].y = (float)p[1];
                  if (col + 2 < n1) yv[i].z = (float)p[2];
                }
              }
            }
          }
          if (b == 0) {
            wait(&s.dfull[nd & 1], nd >> 1, DEV_TIMEOUT_DRAIN);
            tc_after();
          }
          float d[32];
#pragma unroll
          for (int u = 0; u < 4; ++u) ld8(tlane + (nd & 1) * 128 + half * 64 + b * 32 + u * 8, d + u * 8);
          wait_ld();
          if (b == 1) {
            tc_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&s.dfree[nd & 1]);
          }
          __syncwarp();
#pragma unroll
          for (int u = 0; u < 8; ++u)
            *reinterpret_cast<float4*>(turn + lane * kStagePitch + u * 4) =
                make_float4(d[4 * u] * factor, d[4 * u + 1] * factor, d[4 * u + 2] * factor, d[4 * u + 3] * factor);
          __syncwarp();
#pragma unroll
          for (int i = 0; i < NR; ++i) {
            const int rr = VY ? i * 4 + (lane >> 3) : i, r = quarter * 32 + rr;
            if (r >= cnt || col >= n1) continue;
            const int64_t row_g = s.rows[r];
            T* o = out + row_g * a.ldo + col;
            if constexpr (VY) {
              const float4 z = *reinterpret_cast<const float4*>(turn + rr * kStagePitch + (lane & 7) * 4);
              const float4 w = make_float4(yv[i].x + z.x, yv[i].y + z.y, yv[i].z + z.z, yv[i].w + z.w);
              if (col + 4 <= n1) {
                if constexpr (F32) {
                  *reinterpret_cast<float4*>(o) = w;
                } else {
                  *reinterpret_cast<uint2*>(o) = make_uint2(h2_as_u32(__floats2half2_rn(w.x, w.y)),
                                                            h2_as_u32(__floats2half2_rn(w.z, w.w)));
                }
              } else {
                o[0] = (T)w.x;
                if (col + 1 < n1) o[1] = (T)w.y;
                if (col + 2 < n1) o[2] = (T)w.z;
              }
            } else {
              *o = (T)((float)y[row_g * a.ldy + col] + turn[rr * kStagePitch + lane]);
            }
          }
        }
      }
      workers_sync();  // before the next tile's chunks: every warp is done with its turned blocks and rows
    } else {
      // ---- products ----
      const uint32_t on = elect_lane();
      const uint32_t lbo = (uint32_t)r16 * 16;
      const uint32_t id1 = idesc_of(F32, r16), id2 = idesc_of(0, kCols);
      for (int q = 0; q < nq; ++q, ++nc) {
        const int st = nc % NS;
        if (q % G::CHAIN == 0) {
          if (nd >= 2) wait(&s.dfree[nd & 1], (nd >> 1) - 1, DEV_TIMEOUT_DRAIN);
        }
        wait(&s.full[st], nc / NS, DEV_TIMEOUT_FULL);
        ok = __all_sync(0xffffffffu, ok);
        tc_after();
        if (ok) {
          const uint32_t base = sbase + st * G::STAGE, low = sbase + NS * G::STAGE + (nc & 1) * G::LOW;
          const uint64_t bd = desc_blocks((F32 ? low : base) + G::A, lbo);
#pragma unroll
          for (int part = F32; part >= 0; --part) {  // the low part first
            const uint64_t ad = desc_rows(part ? low : base);
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
              mma<F32>(on, tmem + (nd & 1) * 128, ad + ks * 2, bd + (uint64_t)(ks * 2 * lbo >> 4), id1,
                       q % G::CHAIN || part < F32 || ks);
          }
          commit(on, &s.empty[st]);
        }
        if ((q + 1) % G::CHAIN == 0 || q + 1 == nq) {
          if (ok) commit(on, &s.dfull[nd & 1]);
          ++nd;
        }
      }
      // the chunks' memory is free once the last accumulator is there
      if (nq > 0) wait(&s.dfull[(nd - 1) & 1], (nd - 1) >> 1, DEV_TIMEOUT_DRAIN);
      ok = __all_sync(0xffffffffu, ok);
      auto fetch = [&](int t) {  // columns n0 + 128 t ... of up
        const int b = (nu + t) & 1, c0 = n0 + t * kCols, rows = min(kCols, n1 - c0), ch = r16 / 8;
        if (!ok) return;
        if (lane == 0) mbar_arrive_expect_tx(&s.upfull[b], (uint32_t)(ch * rows * 16));
        __syncwarp();
        if (lane < ch)
          bulk_g2s(smem + 2 * G::V + b * G::UP + lane * kCols * 16, up + ((int64_t)lane * a.w.n + c0) * 8,
                   (uint32_t)(rows * 16), &s.upfull[b]);
      };
      int fetched = 0;
      for (; fetched < min(2, nt); ++fetched) fetch(fetched);
      for (int i = 0; i < 2; ++i) {  // as above
        cluster_arrive();
        cluster_wait();
      }
      wait(&s.vready, nv, DEV_TIMEOUT_SMEM);
      for (int t = 0; t < nt; ++t, ++nd) {
        const int b = (nu + t) & 1;
        if (nd >= 2) wait(&s.dfree[nd & 1], (nd >> 1) - 1, DEV_TIMEOUT_DRAIN);
        wait(&s.upfull[b], (nu + t) >> 1, DEV_TIMEOUT_FULL);
        ok = __all_sync(0xffffffffu, ok);
        tc_after();
        if (ok) {
          const uint64_t bd = desc_blocks(sbase + 2 * G::V + b * G::UP, kCols * 16);
#pragma unroll 1
          for (int part = 1; part >= 0; --part) {
            const uint64_t ad = desc_blocks(sbase + part * G::V, 128 * 16);
#pragma unroll 1
            for (int ks = 0; ks < r16 / 16; ++ks)
              mma<0>(on, tmem + (nd & 1) * 128, ad + (uint64_t)(ks * 2 * 2048 >> 4), bd + (uint64_t)(ks * 2 * kCols * 16 >> 4),
                     id2, part < 1 || ks);
          }
          commit(on, &s.dfull[nd & 1]);
        }
        if (fetched < nt) {  // into the buffer that this product reads
          wait(&s.dfull[nd & 1], nd >> 1, DEV_TIMEOUT_DRAIN);
          ok = __all_sync(0xffffffffu, ok);
          fetch(fetched++);
        }
      }
      // copies in flight land before the CTA's shared memory goes away
      if (!ok)
        for (int b = 0; b < 2; ++b)
          if (fetched > 0) mbar_wait(&s.upfull[b], (nu + fetched - 1) >> 1 & 1, nullptr, 0);
      nu += nt;
    }
    ++nv;
  }
  if (a.out != a.y && warp < 8)
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
  if (warp == 8)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(256) : "memory");
}

template <class T, int RP, bool VX, bool VY>
cudaError_t launch(const AdapterArgs& a, int num_sms, cudaStream_t s) {
  using G = Cfg<T, RP>;
  int dev = 0;
  cudaGetDevice(&dev);
  const int smem = G::smem(a.w.n_slots);
  if (cudaError_t e = ensure_smem_attr(adapters_tile_kernel<T, RP, VX, VY>, G::smem(kAdapterMaxSlots), dev)) return e;
  const int ctas = num_sms * (smem <= 113 * 1024 ? G::CTAS : 1);
  // Small tiles while there are too few rows for all CTAs, then smaller clusters.
  int tile_rows = 128;
  while (tile_rows > 16 && (a.n_rows + tile_rows - 1) / tile_rows * 8 < ctas) tile_rows /= 2;
  int cluster = 8;
  while (cluster > 2 && (a.n_rows + tile_rows - 1) / tile_rows * cluster > ctas) cluster /= 2;
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
  const int four = 4 * sizeof(T);
  const bool vx = on(a.x, a.ldx, 16), vy = on(a.y, a.ldy, four) && on(a.out, a.ldo, four);
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
    if (a.w.rp <= 64) e = a.x16 ? launch_rank<__half, 64>(b, num_sms, s) : launch_rank<float, 64>(b, num_sms, s);
    else e = a.x16 ? launch_rank<__half, 128>(b, num_sms, s) : launch_rank<float, 128>(b, num_sms, s);
    if (e) return e;
  }
  return cudaSuccess;
}

}  // namespace rb
