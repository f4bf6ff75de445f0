// Masked attention of long runs of rows (prompts, chunks) over fp16 caches on
// tcgen05: the function of rows_attn.cu for up to 256 query vectors of one kv head
// and tenant, as two tiles of 128 that share every block of 128 keys.
//
// Per tile and block: S = Q K^T (tcgen05.mma, both operands in shared memory, S in
// TMEM), softmax in registers with two threads a row (tcgen05.ld, 64 keys each: four
// warps a scheduler hide one another's latencies), P back to TMEM over S, O += P V with P as the TMEM operand and V as it lies in the page
// ([key][element]: the MN-major operand). The tiles take turns: while one's scores
// are in the softmax warps the tensor core works on the other's.
//
// fp32 rows: q and p as fp16 hi + lo parts, two products each (22 bits); q is
// brought to a power of two near 2^8 first. p counts from 2^kBias and the running
// maximum is raised only when a score passes it by 2^kSlack, so p stays below
// 2^15, fp16's range, and O is rarely rescaled.
//
// Warps: 0-7 softmax of tile 0 (0-3 the first 64 keys of a block, 4-7 the others), 8-15
// of tile 1, 16 issues the products, 17 the loads (18 and 19 fill the last warpgroup,
// which gives registers to the others).
#include "common.cuh"
#include "rows.cuh"

namespace rb {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kBias = 6.f, kSlack = 8.f;
#ifndef TPR_
#define TPR_ 1
#endif
constexpr int kTpr = TPR_;                    // softmax threads a row
constexpr int kSoftWarps = 8 * kTpr;
constexpr int kTileThreads = (kSoftWarps + 4) * 32;
// registers a thread at launch, of a softmax warp and of the others: the split uses what the launch gave
constexpr int kRegSoft = kTpr == 1 ? 224 : 104, kRegRest = kTpr == 1 ? 56 : 64;

// ---- tcgen05 ----
// shared-memory operand with 128-byte swizzle; sbo: bytes between groups of 8 rows,
// lbo: between panels of 64 columns (MN-major only)
__device__ __forceinline__ uint64_t desc128(uint32_t saddr, uint32_t lbo, uint32_t sbo) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)((lbo >> 4) & 0x3FFFu) << 16) |
         ((uint64_t)((sbo >> 4) & 0x3FFFu) << 32) | (1ull << 46) | (2ull << 61);
}
__host__ __device__ constexpr uint32_t idesc16(int m, int n, int b_mn_major) {
  return (1u << 4) | ((uint32_t)b_mn_major << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// The whole warp runs these converged, so that the operands stay in uniform registers;
// the lane with `on` issues.
__device__ __forceinline__ void mma_ss(uint32_t on, uint32_t d, uint64_t ad, uint64_t bd, uint32_t id, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(ad), "l"(bd), "r"(id), "r"(acc), "r"(on)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t on, uint32_t d, uint32_t at, uint64_t bd, uint32_t id, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(at), "l"(bd), "r"(id), "r"(acc), "r"(on)
      : "memory");
}
__device__ __forceinline__ void tc_commit(uint32_t on, uint64_t* bar) {
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
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// 32 columns of this thread's TMEM lane; the registers are valid after wait_ld()
__device__ __forceinline__ void ld32(uint32_t ta, float* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]),
        "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]), "=f"(r[16]),
        "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]), "=f"(r[24]),
        "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31])
      : "r"(ta)
      : "memory");
}
__device__ __forceinline__ void st32(uint32_t ta, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(ta),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
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
__device__ __forceinline__ float ld1(uint32_t ta) {
  float r;
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=f"(r) : "r"(ta) : "memory");
  wait_ld();
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm volatile("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack2(float a, float b) { return h2_as_u32(__floats2half2_rn(a, b)); }
__device__ __forceinline__ uint32_t pack2_lo(float a, float b, uint32_t hi) {
  const float2 f = __half22float2(u32_as_h2(hi));
  return pack2(a - f.x, b - f.y);
}
__device__ __forceinline__ float min3(float a, float b, float c) {
  float y;
  asm("min.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
// two fp32 values in one register pair, and the packed operations on them
using f2 = unsigned long long;
__device__ __forceinline__ f2 pair(float a, float b) {
  f2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpair(f2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
  f2 r;
  asm volatile("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
  f2 r;
  asm volatile("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f2 add2(f2 a, f2 b) {
  f2 r;
  asm volatile("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// tanh(y) = y P(y^2) for |y| <= limit, fitted for the least largest relative
// error: 6e-7 with four terms (fp16 rows, whose probabilities are rounded to 2^-12),
// 4e-9 with six.
template <int HL>
struct Tanh;
template <>
struct Tanh<0> {
  static constexpr int N = 4;
  static constexpr float limit = 0.5f;
  static __device__ __forceinline__ float c(int i) {
    constexpr float k[4] = {0.999999456f, -0.333263179f, 0.131902966f, -0.0444022264f};
    return k[i];
  }
};
template <>
struct Tanh<1> {
  static constexpr int N = 6;
  static constexpr float limit = 0.625f;
  static __device__ __forceinline__ float c(int i) {
    constexpr float k[6] = {0.999999996f, -0.333332605f, 0.133311275f, -0.053721068f, 0.0205909884f, -0.00565998907f};
    return k[i];
  }
};
// barrier of the n softmax threads in use, with the "or" of their values
__device__ __forceinline__ bool any_softmax(int n, bool v) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, 1, %2, p;\n\tselp.u32 %0, 1, 0, "
      "q;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)v), "r"(n)
      : "memory");
  return r != 0;
}
// the sign bits of the two halves of w that are infinite or not a number
__device__ __forceinline__ uint32_t not_finite(uint32_t w) { return ((w & 0x7c007c00u) + 0x04000400u) & 0x80008000u; }

template <bool V>
struct Flag {
  static constexpr bool value = V;
};

template <int HD, int HL>
struct TileCfg {
  static constexpr int PANEL = 128 * 128;             // 128 rows x 64 fp16
  static constexpr int QT = HD / 64 * PANEL;          // one tile of q (one part)
  static constexpr int SLOT = HD / 64 * PANEL;        // a block of K or V
  static constexpr int NS = HD == 128 ? (HL ? 3 : 4) : 6;
  static constexpr int SMEM = 2 * (1 + HL) * QT + NS * SLOT;
  // TMEM columns. Where they fit, p has its own (PW a tile) and one S serves both tiles
  // in turn, since the softmax threads take it into registers at once: the next scores
  // are then computed while the softmax runs. fp32 rows at head size 128 need all 512
  // columns otherwise: there p lies over its tile's scores.
  static constexpr bool SEP = HD == 64 || !HL;
  static constexpr int PW = SEP ? 64 * (1 + HL) : kTileKeys;
  static constexpr int P0 = 2 * HD, S0 = SEP ? 512 - kTileKeys : P0, SW = SEP ? 0 : kTileKeys;
  static_assert(P0 + 2 * PW + (SEP ? kTileKeys : 0) <= 512, "");
  // column, within a tile's P, of the 16 keys of k-step ks; lo: their low parts
  static constexpr __host__ __device__ int pcol(int ks, int lo) {
    return SEP ? lo * 64 + ks * 8 : (ks >> 1) * 32 + lo * 16 + (ks & 1) * 8;
  }
};

template <int HD, int HL, int CAP, int BIAS>
__global__ void __launch_bounds__(kTileThreads, 1) rows_tile_kernel(const __grid_constant__ RowAttnArgs a) {
  using C = TileCfg<HD, HL>;
  constexpr int NS = C::NS, B = kTileKeys, H = B / kTpr, NSOFT = 128 * kTpr;  // softmax threads a tile
  extern __shared__ __align__(1024) uint8_t smem[];  // the swizzle follows the address bits
  if (smem_u32(smem) & 1023) {
    report_error(a.err, DEV_TIMEOUT_SMEM);
    return;
  }
  uint8_t* ring = smem + 2 * (1 + HL) * C::QT;
  __shared__ uint64_t q_bar[2], s_bar[2], p_bar[2], o_bar[2], s_free, full[NS], freeb[NS], drain;
  __shared__ uint32_t tmem_slot;
  __shared__ int primed[2];    // O holds something before the first product
  __shared__ int span[2][2];  // keys that every row of a tile sees
  __shared__ int seen[2];     // keys that some row of the unit sees
  // Between the two threads of a row, by block parity: one may be a block ahead of the
  // other, except where S waits for both (p over S).
  __shared__ float xch[C::SEP ? 2 : 1][2][kTpr][128];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const AttnUnit u = a.units[blockIdx.x];
  const int nt = u.nv > 128 ? 2 : 1, nb = (u.k1 - u.k0 + B - 1) / B;

  if (warp == kSoftWarps) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (tid == 0) {
    for (int t = 0; t < 2; ++t) {
      mbar_init(&q_bar[t], NSOFT);
      mbar_init(&s_bar[t], 1);
      mbar_init(&p_bar[t], NSOFT);
      mbar_init(&o_bar[t], 1);
      primed[t] = 0;
      span[t][0] = 0;
      span[t][1] = 0x7fffffff;
    }
    for (int i = 0; i < NS; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&freeb[i], 1);
    }
    mbar_init(&drain, 1);
    mbar_init(&s_free, NSOFT);
    seen[0] = 0x7fffffff;
    seen[1] = 0;
    fence_barrier_init();
  }
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tmem = tmem_slot;
  // softmax warps: this thread has row tr of its tile and half of a block's keys
  const int tile = warp / (4 * kTpr), half = kTpr == 1 ? 0 : (warp >> 2) & 1, tr = (warp & 3) * 32 + lane, vec_id = tile * 128 + tr;
  RowInfo r{0, 0, 0x7fffffff, 0};
  int head = 0, row = 0;
  const bool active = warp < kSoftWarps && vec_id < u.nv;
  if (active) {
    const int v = u.v0 + vec_id;
    row = u.row0 + v / a.n_rep;
    head = u.kvh * a.n_rep + v % a.n_rep;
    r = a.rows[row];
    atomicMax(&span[tile][0], r.lo);
    atomicMin(&span[tile][1], r.hi);
    if (r.hi > r.lo) {
      atomicMin(&seen[0], r.lo);
      atomicMax(&seen[1], r.hi);
    }
  }
  __syncthreads();

  if (warp >= kSoftWarps + 2) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegRest));
  } else if (warp == kSoftWarps + 1) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegRest));
    // ---- loads: blocks K0, V0, K1, V1, ... through the ring ----
    bool ok = true;
    int it = 0;
    const int page_end = (u.k1 + 15) >> 4;
    const int32_t* pt = a.kv.ptab + (size_t)u.tenant * a.kv.ptab_stride;
    for (int j = 0; j < nb && ok; ++j) {
      const int p0 = (u.k0 >> 4) + j * (B / 16), np = min(B / 16, page_end - p0);
      const int mine = lane & 7, page = mine < np ? pt[p0 + mine] : 0;
      for (int w = 0; w < 2; ++w, ++it) {
        const int s = it % NS;
        if (it >= NS) {
          if (lane == 0) ok = mbar_wait(&freeb[s], (uint32_t)((it / NS - 1) & 1), a.err, DEV_TIMEOUT_EMPTY);
          ok = __shfl_sync(0xffffffffu, ok, 0);
        }
        if (!ok) break;  // the whole warp
        if (lane == 0) mbar_arrive_expect_tx(&full[s], (uint32_t)(np * 16 * HD * 2));
        __syncwarp();
        if (mine < np && (lane >> 3) < HD / 64) {
          const int y = (((page * a.kv.n_layers + a.layer) * 2 + w) * a.kv.n_kv + u.kvh) * 16;
          asm volatile(
              "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], "
              "[%4];" ::"r"(smem_u32(ring + s * C::SLOT + (lane >> 3) * C::PANEL + mine * 2048)),
              "l"(reinterpret_cast<uint64_t>(&a.tmap)), "r"((lane >> 3) * 64), "r"(y), "r"(smem_u32(&full[s]))
              : "memory");
        }
      }
    }
    // copies in flight land before the CTA's shared memory goes away
    for (int i = max(0, it - NS); i < it; ++i) mbar_wait(&full[i % NS], (uint32_t)((i / NS) & 1), nullptr, 0);
  } else if (warp == kSoftWarps) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegRest));
    // ---- products ----
    if (nb > 0) {
      bool ok = true;
      const uint32_t on = elect_lane();
      constexpr uint32_t ids = idesc16(128, B, 0), ido = idesc16(128, HD, 1);
      const uint32_t qa = smem_u32(smem), ra = smem_u32(ring);
      auto scores = [&](int t, int slot) {
        const uint64_t kd = (desc128(ra + slot * C::SLOT, 16, 1024));
#pragma unroll
        for (int part = 0; part < 1 + HL; ++part) {
          const uint64_t qd = (desc128(qa + (t * (1 + HL) + part) * C::QT, 16, 1024));
#pragma unroll
          for (int ks = 0; ks < HD / 16; ++ks) {
            const uint32_t off = ((ks >> 2) * C::PANEL + (ks & 3) * 32) >> 4;
            mma_ss(on, tmem + C::S0 + t * C::SW, qd + off, kd + off, ids, part || ks);
          }
        }
      };
      auto wait = [&](uint64_t* bar, int phase, uint32_t code) {
        ok = __all_sync(0xffffffffu, ok && mbar_wait(bar, (uint32_t)(phase & 1), a.err, code));
        tc_after();
      };
      int n_s = 0;  // scores issued
      auto issue_scores = [&](int t, int j) {
        const int slot = 2 * j % NS;
        if (t == 0) wait(&full[slot], 2 * j / NS, DEV_TIMEOUT_FULL);
        if (j == 0) wait(&q_bar[t], 0, DEV_TIMEOUT_SMEM);
        // S is free when its last tile has it in registers
        if (C::SEP && n_s > 0) wait(&s_free, n_s - 1, DEV_TIMEOUT_EMPTY);
        if (!ok) return;
        scores(t, slot);
        tc_commit(on, &s_bar[t]);
        if (t == nt - 1) tc_commit(on, &freeb[slot]);
        ++n_s;
      };
      auto issue_pv = [&](int t, int j) {
        const int slot = (2 * j + 1) % NS;
        if (t == 0) wait(&full[slot], (2 * j + 1) / NS, DEV_TIMEOUT_FULL);
        wait(&p_bar[t], j, DEV_TIMEOUT_DRAIN);
        if (!ok) return;
        const uint32_t more = j || *(volatile int*)&primed[t];
        const uint64_t vd = (desc128(ra + slot * C::SLOT, C::PANEL, 1024));
#pragma unroll
        for (int part = 0; part < 1 + HL; ++part)
#pragma unroll
          for (int ks = 0; ks < B / 16; ++ks)
            mma_ts(on, tmem + t * HD, tmem + C::P0 + t * C::PW + C::pcol(ks, part), vd + ks * (2048 >> 4), ido,
                   more || part || ks);
        tc_commit(on, &o_bar[t]);
        if (t == nt - 1) tc_commit(on, &freeb[slot]);
      };
      for (int t = 0; t < nt && ok; ++t) issue_scores(t, 0);
      for (int j = 0; j < nb && ok; ++j)
        for (int t = 0; t < nt && ok; ++t) {
          if (C::SEP && j + 1 < nb) issue_scores(t, j + 1);
          if (ok) issue_pv(t, j);
          if (ok && !C::SEP && j + 1 < nb) issue_scores(t, j + 1);
        }
      tc_commit(on, &drain);  // own products complete before the accumulators are freed
      mbar_wait(&drain, 0, a.err, DEV_TIMEOUT_DRAIN);
    }
    __syncwarp();
  } else if (tile < nt) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegSoft));
    // ---- softmax ----
    const int d_begin = half * (HD / kTpr), d_end = d_begin + HD / kTpr;  // this thread's part of O
    const uint32_t lane_base = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t ts = lane_base + C::S0 + tile * C::SW + half * H, to = lane_base + tile * HD,
                   tp = lane_base + C::P0 + tile * C::PW;
    bool alive = true;
    float sv = fabsf(a.scale);
    {  // q into shared memory, K-major with 128-byte swizzle; a negative scale turns q
      const float sign = a.scale < 0.f ? -1.f : 1.f;
      uint8_t* qd = smem + tile * (1 + HL) * C::QT + tr * 128;
      const size_t at = (size_t)row * a.ldq + (size_t)head * HD;
      const int rx = tr & 7;
      if (HL) {
        const float* q = reinterpret_cast<const float*>(a.q) + at;
        const bool vec = ((reinterpret_cast<uintptr_t>(a.q) | (size_t)a.ldq * 4) & 15) == 0;
        float top = 0.f;
        if (active)
          for (int d = 0; d < HD; d += 4) {
            if (vec) {
              const float4 x = *reinterpret_cast<const float4*>(q + d);
              top = fmaxf(fmaxf(top, fmaxf(fabsf(x.x), fabsf(x.y))), fmaxf(fabsf(x.z), fabsf(x.w)));
            } else {
              for (int e = 0; e < 4; ++e) top = fmaxf(top, fabsf(q[d + e]));
            }
          }
        float mul = 1.f;
        const int e = (int)(__float_as_uint(top) >> 23);
        if (e > 8 && e < 255) mul = __uint_as_float((uint32_t)min(254, 127 + 8 + 127 - e) << 23);
        sv = sv / mul;
        mul *= sign;
        for (int ch = d_begin / 8; ch < d_end / 8; ++ch) {
          float x[8];
          if (active && vec) {
            *reinterpret_cast<float4*>(x) = *reinterpret_cast<const float4*>(q + ch * 8);
            *reinterpret_cast<float4*>(x + 4) = *reinterpret_cast<const float4*>(q + ch * 8 + 4);
          } else {
            for (int i = 0; i < 8; ++i) x[i] = active ? q[ch * 8 + i] : 0.f;
          }
          uint4 hi, lo;
          uint32_t* h = &hi.x;
          uint32_t* l = &lo.x;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            x[2 * i] *= mul;
            x[2 * i + 1] *= mul;
            h[i] = pack2(x[2 * i], x[2 * i + 1]);
            l[i] = pack2_lo(x[2 * i], x[2 * i + 1], h[i]);
          }
          uint8_t* dst = qd + (ch >> 3) * C::PANEL + (((ch & 7) ^ rx) << 4);
          *reinterpret_cast<uint4*>(dst) = hi;
          *reinterpret_cast<uint4*>(dst + HL * C::QT) = lo;
        }
      } else {
        const __half* q = reinterpret_cast<const __half*>(a.q) + at;
        const bool vec = ((reinterpret_cast<uintptr_t>(a.q) | (size_t)a.ldq * 2) & 15) == 0;
        const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;
        for (int ch = d_begin / 8; ch < d_end / 8; ++ch) {
          uint4 x = make_uint4(0, 0, 0, 0);
          if (active) {
            if (vec) {
              x = *reinterpret_cast<const uint4*>(q + ch * 8);
            } else {
              uint16_t* h = reinterpret_cast<uint16_t*>(&x);
              for (int i = 0; i < 8; ++i) h[i] = __half_as_ushort(q[ch * 8 + i]);
            }
          }
          x.x ^= flip;
          x.y ^= flip;
          x.z ^= flip;
          x.w ^= flip;
          *reinterpret_cast<uint4*>(qd + (ch >> 3) * C::PANEL + (((ch & 7) ^ rx) << 4)) = x;
        }
      }
      proxy_fence();
      mbar_arrive(&q_bar[tile]);
    }
    const int all0 = span[tile][0], all1 = span[tile][1], in0 = seen[0], in1 = seen[1];
    const int both0 = max(span[0][0], span[1][0]), both1 = min(span[0][1], span[1][1]);
    const float slope = BIAS && active ? a.slopes[head] * kLog2e : 0.f;
    const float cap2 = a.cap * kLog2e, kcap = CAP ? sv / a.cap : 0.f;
    const float mult = (CAP || BIAS) ? 1.f : fmaxf(sv * kLog2e, 1e-30f);  // scores to base-2 units (-inf stays)
    const float sv2 = sv * kLog2e;
    float m = -INFINITY, l = 0.f;
    for (int j = 0; j < nb; ++j) {
      const int kb = u.k0 + j * B, kh = kb + half * H;  // the block's first key, and this thread's
      if (alive) alive = mbar_wait(&s_bar[tile], (uint32_t)(j & 1), a.err, DEV_TIMEOUT_FULL);
      tc_after();
      float x[H];
#pragma unroll
      for (int i = 0; i < H / 32; ++i) ld32(ts + 32 * i, x + 32 * i);
      wait_ld();
      if (C::SEP) {
        tc_before();
        mbar_arrive(&s_free);
      }
      const bool partial = kb < all0 || kb + B > all1;  // the same for the whole tile
      bool fused = false;  // the cap is applied together with the exponential
      float raw_top = 0.f;
      if (CAP) {
        // the largest magnitude, from both ends: the maximum is wanted anyway
        float lo4[4] = {0.f, 0.f, 0.f, 0.f}, hi4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < H; i += 8)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            lo4[q] = min3(lo4[q], x[i + 2 * q], x[i + 2 * q + 1]);
            hi4[q] = max3(hi4[q], x[i + 2 * q], x[i + 2 * q + 1]);
          }
        const float lo = min3(fminf(lo4[0], lo4[1]), lo4[2], lo4[3]);
        raw_top = max3(fmaxf(hi4[0], hi4[1]), hi4[2], hi4[3]);
        fused = !BIAS && !partial && __all_sync(0xffffffffu, fmaxf(raw_top, -lo) * kcap <= Tanh<HL>::limit);
        if (!fused) {
          // cap tanh(y) = cap - 2 cap / (1 + e^(2 y))
          const float k = 2.f * kLog2e * kcap;
#pragma unroll
          for (int i = 0; i < H; ++i) x[i] = fmaf(-2.f * cap2, rcp(1.f + ex2(x[i] * k)), cap2);
        }
      }
      if (BIAS) {
        if (__all_sync(0xffffffffu, kh + H - 1 <= r.pos)) {  // no key after its row: the distance is linear
          const f2 sl = pair(slope, slope), s2 = pair(CAP ? 1.f : sv2, CAP ? 1.f : sv2);
          const float b0 = slope * (float)(kh - r.pos);
          const f2 b2 = pair(b0, b0);
#pragma unroll
          for (int i = 0; i < H; i += 2)
            unpair(fma2(pair(x[i], x[i + 1]), s2, fma2(pair((float)i, (float)(i + 1)), sl, b2)), x[i], x[i + 1]);
        } else {
#pragma unroll
          for (int i = 0; i < H; ++i)
            x[i] = fmaf(-slope, fabsf((float)(r.pos - kh - i)), CAP ? x[i] : x[i] * sv2);
        }
      }
      if (partial) {
        const uint32_t base = (uint32_t)(kh - r.lo), n = (uint32_t)max(0, r.hi - r.lo);
#pragma unroll
        for (int i = 0; i < H; ++i) x[i] = base + i < n ? x[i] : -INFINITY;
      }
      float mx;
      if (CAP && fused) {
        // the cap keeps the order: it is applied to the maximum alone
        mx = fmaf(-2.f * cap2, rcp(1.f + ex2(raw_top * (2.f * kLog2e * kcap))), cap2);
      } else {
        float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < H; i += 8)
#pragma unroll
          for (int q = 0; q < 4; ++q) mx4[q] = max3(mx4[q], x[i + 2 * q], x[i + 2 * q + 1]);
        mx = max3(fmaxf(mx4[0], mx4[1]), mx4[2], mx4[3]) * mult;
      }
      if (kTpr == 2) {  // the row's other thread
        float(*xb)[128] = xch[C::SEP ? j & 1 : 0][tile];
        xb[half][tr] = mx;
        asm volatile("bar.sync %0, 64;" ::"r"(2 + tile * 4 + (warp & 3)) : "memory");
        mx = fmaxf(mx, xb[half ^ 1][tr]);
      }
      // each row raises its maximum by its own scores alone
      const bool up = mx > (m == -INFINITY ? m : m + kSlack);
      float alpha = 1.f;
      if (up) {
        alpha = ex2(m - mx);
        l *= alpha;
        m = mx;
      }
      if (j > 0) {  // the last block's P V has read P, and O is at rest
        if (alive) alive = mbar_wait(&o_bar[tile], (uint32_t)((j - 1) & 1), a.err, DEV_TIMEOUT_DRAIN);
        tc_after();
      }
      if (__any_sync(0xffffffffu, up) && j > 0) {
#pragma unroll 1
        for (int d = d_begin; d < d_end; d += 32) {
          float o[32];
          ld32(to + d, o);
          wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] *= alpha;
          st32(to + d, reinterpret_cast<uint32_t*>(o));
        }
      }
      const float off = kBias - (m == -INFINITY ? 0.f : m);
      const f2 mult2 = pair(mult, mult), off2 = pair(off, off);
      f2 s2[2] = {0ull, 0ull};
      // Groups of 2 G keys, every step for the whole group before the next one: the
      // steps of a key wait for one another, the keys do not.
      auto exps = [&](auto capped) {
        constexpr bool FUSED = decltype(capped)::value;
        using P = Tanh<HL>;
        f2 pc[P::N];
#pragma unroll
        for (int q = 0; q < P::N; ++q) pc[q] = pair(cap2 * P::c(q), cap2 * P::c(q));
        constexpr int G = kTpr == 1 ? 8 : 4;  // pairs
#pragma unroll
        for (int i = 0; i < H / 32; ++i) {
          uint32_t hi[16], lo[16];
#pragma unroll
          for (int h = 0; h < 16 / G; ++h) {
            f2 y[G];
            float e[2 * G];
#pragma unroll
            for (int g = 0; g < G; ++g) y[g] = pair(x[32 * i + 2 * G * h + 2 * g], x[32 * i + 2 * G * h + 2 * g + 1]);
            if (FUSED) {
              const f2 k2 = pair(kcap, kcap);
              f2 z[G], t[G];
#pragma unroll
              for (int g = 0; g < G; ++g) y[g] = mul2(y[g], k2);
#pragma unroll
              for (int g = 0; g < G; ++g) z[g] = mul2(y[g], y[g]);
#pragma unroll
              for (int g = 0; g < G; ++g) t[g] = pc[P::N - 1];
#pragma unroll
              for (int q = P::N - 2; q >= 0; --q)
#pragma unroll
                for (int g = 0; g < G; ++g) t[g] = fma2(t[g], z[g], pc[q]);
#pragma unroll
              for (int g = 0; g < G; ++g) y[g] = fma2(t[g], y[g], off2);
            } else {
#pragma unroll
              for (int g = 0; g < G; ++g) y[g] = fma2(y[g], mult2, off2);
            }
#pragma unroll
            for (int g = 0; g < G; ++g) {
              float a0, a1;
              unpair(y[g], a0, a1);
              e[2 * g] = ex2(a0);
              e[2 * g + 1] = ex2(a1);
            }
#pragma unroll
            for (int g = 0; g < G; ++g) s2[g & 1] = add2(s2[g & 1], pair(e[2 * g], e[2 * g + 1]));
#pragma unroll
            for (int g = 0; g < G; ++g) hi[G * h + g] = pack2(e[2 * g], e[2 * g + 1]);
            if (HL)
#pragma unroll
              for (int g = 0; g < G; ++g) lo[G * h + g] = pack2_lo(e[2 * g], e[2 * g + 1], hi[G * h + g]);
          }
          st16(tp + C::pcol(half * (H / 16) + 2 * i, 0), hi);
          if (HL) st16(tp + C::pcol(half * (H / 16) + 2 * i, 1), lo);
        }
      };
      if (CAP && fused) exps(Flag<true>());
      else exps(Flag<false>());
      {
        float p0, p1;
        unpair(add2(s2[0], s2[1]), p0, p1);
        l += p0 + p1;
      }
      if (kb < both0 || kb + B > both1) {
        // A block that some row of the unit does not see whole. Values of keys that no
        // row sees become 0, and so do those of pages that were not loaded. Values that
        // are not finite enter O here, each row adding those of its own keys, and are 0
        // for the product: 0 times one of them would reach the rows that do not see it.
        const int vs = (2 * j + 1) % NS;
        if (alive) alive = mbar_wait(&full[vs], (uint32_t)(((2 * j + 1) / NS) & 1), a.err, DEV_TIMEOUT_FULL);
        uint8_t* vrow = ring + vs * C::SLOT + tr * 128;
        const bool in = kb + tr >= in0 && kb + tr < in1;
        const int nc = HD / 8 / kTpr / nt, c0 = (tile * kTpr + half) * nc, c1 = c0 + nc;  // the threads of a key share its chunks
        uint32_t bad = 0;
        for (int ch = c0; ch < c1; ++ch) {
          uint4* p = reinterpret_cast<uint4*>(vrow + (ch >> 3) * C::PANEL + ((ch & 7) << 4));
          if (in) {
            const uint4 q = *p;
            bad |= not_finite(q.x) | not_finite(q.y) | not_finite(q.z) | not_finite(q.w);
          } else {
            *p = make_uint4(0, 0, 0, 0);
          }
        }
        proxy_fence();
        wait_st();
        tc_before();
        if (any_softmax(NSOFT * nt, bad != 0)) {
          tc_after();
#pragma unroll 1
          for (int d = d_begin; d < d_end; d += 32) {
            float o[32];
            ld32(to + d, o);
            wait_ld();
            if (j == 0)
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = 0.f;
#pragma unroll 1
            for (int k = 0; k < B; ++k) {
              float p = 0.f;
#pragma unroll
              for (int part = 0; part < 1 + HL; ++part) {
                const uint32_t w = __float_as_uint(ld1(tp + C::pcol(k >> 4, part) + ((k & 15) >> 1)));
                p += half_bits_to_float((k & 1) ? w >> 16 : w);
              }
              const uint8_t* vk = ring + vs * C::SLOT + k * 128 + (d >> 6) * C::PANEL;
              if (p != 0.f)
#pragma unroll
                for (int ch = 0; ch < 4; ++ch) {
                  const uint4 q = *reinterpret_cast<const uint4*>(vk + (((((d >> 3) + ch) & 7) ^ (k & 7)) << 4));
                  const uint32_t* w = &q.x;
#pragma unroll
                  for (int e = 0; e < 4; ++e) {
                    const uint32_t nf = not_finite(w[e]);
                    const float2 f = __half22float2(u32_as_h2(w[e]));
                    if (nf & 0x8000u) o[ch * 8 + 2 * e] = fmaf(p, f.x, o[ch * 8 + 2 * e]);
                    if (nf & 0x80000000u) o[ch * 8 + 2 * e + 1] = fmaf(p, f.y, o[ch * 8 + 2 * e + 1]);
                  }
                }
              __syncwarp();
            }
            st32(to + d, reinterpret_cast<uint32_t*>(o));
          }
          any_softmax(NSOFT * nt, false);  // all rows have taken theirs
          for (int ch = c0; ch < c1; ++ch) {
            uint4* p = reinterpret_cast<uint4*>(vrow + (ch >> 3) * C::PANEL + ((ch & 7) << 4));
            uint32_t* w = reinterpret_cast<uint32_t*>(p);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t nf = not_finite(w[e]);
              w[e] &= ((nf & 0x8000u) ? 0u : 0xffffu) | ((nf & 0x80000000u) ? 0u : 0xffff0000u);
            }
          }
          proxy_fence();
          any_softmax(NSOFT * nt, false);
          if (tr == 0 && half == 0 && j == 0) *(volatile int*)&primed[tile] = 1;
        }
      }
      wait_st();
      tc_before();
      mbar_arrive(&p_bar[tile]);
    }
    if (nb > 0) {
      if (alive) alive = mbar_wait(&o_bar[tile], (uint32_t)((nb - 1) & 1), a.err, DEV_TIMEOUT_DRAIN);
      tc_after();
    }
    if (kTpr == 2) {
      xch[0][tile][half][tr] = l;  // all maxima are read: the last P V had both threads' p
      asm volatile("bar.sync %0, 64;" ::"r"(2 + tile * 4 + (warp & 3)) : "memory");
      l = xch[0][tile][0][tr] + xch[0][tile][kTpr - 1][tr];
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int slot = u.slot + vec_id;
    if (u.slot >= 0 && active && half == 0) a.part_ml[slot] = make_float2(m, l);
    const size_t at = (size_t)row * a.ldo + (size_t)head * HD;
    const bool vec = ((reinterpret_cast<uintptr_t>(a.out) | (size_t)a.ldo * (HL ? 4 : 2)) & 15) == 0;
#pragma unroll 1
    for (int d = d_begin; d < d_end; d += 32) {
      float o[32];
      ld32(to + d, o);
      wait_ld();
      if (nb == 0 || l == 0.f)
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = 0.f;
      if (!active) continue;
      if (u.slot >= 0) {
        float4* dst = reinterpret_cast<float4*>(a.part_o + (size_t)slot * HD + d);
#pragma unroll
        for (int i = 0; i < 8; ++i) dst[i] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
      } else if (HL) {
        float* dst = reinterpret_cast<float*>(a.out) + at + d;
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] *= inv;
        if (vec) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            reinterpret_cast<float4*>(dst)[i] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) dst[i] = o[i];
        }
      } else {
        __half* dst = reinterpret_cast<__half*>(a.out) + at + d;
        uint32_t h[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) h[i] = pack2(o[2 * i] * inv, o[2 * i + 1] * inv);
        if (vec) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            reinterpret_cast<uint4*>(dst)[i] = make_uint4(h[4 * i], h[4 * i + 1], h[4 * i + 2], h[4 * i + 3]);
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i)
            dst[i] = __ushort_as_half((unsigned short)((i & 1) ? h[i >> 1] >> 16 : h[i >> 1]));
        }
      }
    }
  }
  tc_before();
  __syncthreads();
  tc_after();
  if (warp == kSoftWarps)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

template <int HD, int HL, int CAP, int BIAS>
cudaError_t launch(const RowAttnArgs& a, cudaStream_t s) {
  int dev = 0;
  cudaGetDevice(&dev);
  constexpr int smem = TileCfg<HD, HL>::SMEM;
  if (cudaError_t e = ensure_smem_attr(rows_tile_kernel<HD, HL, CAP, BIAS>, smem, dev)) return e;
  rows_tile_kernel<HD, HL, CAP, BIAS><<<a.n_units, kTileThreads, smem, s>>>(a);
  return cudaGetLastError();
}
template <int HD, int HL>
cudaError_t launch_score(const RowAttnArgs& a, cudaStream_t s) {
  if (a.cap > 0.f) return a.slopes ? launch<HD, HL, 1, 1>(a, s) : launch<HD, HL, 1, 0>(a, s);
  return a.slopes ? launch<HD, HL, 0, 1>(a, s) : launch<HD, HL, 0, 0>(a, s);
}

}  // namespace

cudaError_t rows_tile_launch(const RowAttnArgs& a, cudaStream_t s) {
  if (a.n_units < 1) return cudaSuccess;
  if (!a.kv.f16) return cudaErrorInvalidValue;
  if (a.kv.hd == 128) return a.q16 ? launch_score<128, 0>(a, s) : launch_score<128, 1>(a, s);
  return a.q16 ? launch_score<64, 0>(a, s) : launch_score<64, 1>(a, s);
}

}  // namespace rb
