// Masked attention of long runs of rows (prompts, chunks) over fp16 caches on
// tcgen05: the function of rows_attn.cu for up to 256 query vectors of one kv head
// and tenant, as two tiles of 128 that share every block of 128 keys.
//
// Per tile and block: S = Q K^T (tcgen05.mma, both operands in shared memory, S in
// TMEM), softmax in registers with one thread a row (tcgen05.ld), P back to TMEM,
// O += P V with P as the TMEM operand and V as it lies in the page ([key][element]: the
// MN-major operand). The tiles take turns: while one's scores are in the softmax warps
// the tensor core works on the other's.
//
// Bound by the softmax warps' instructions: one prompt of 8192, 32 heads of 128 on 8, cap
// 50, fp16: 661 us, 832 TFLOP/s (issue slots 47 % used, tensor cores 44 %; without the cap
// 0.91 of it). A unit's start and end (q, the first scores, O) cost 10 K clocks (fp16 rows,
// head size 64) to 25 K (fp32 rows, 128), as much as two or three pairs of blocks: short
// documents are bound by those (6 prompts of 200-1500 in documents of 300: 129 us).
//
// fp32 rows: q and p as fp16 hi + lo parts, two products each (22 bits); q is
// brought to a power of two near 2^8 first. The tensor core cuts a sum off (towards 0)
// after every 16 products, so the low part comes first, while the sum is small: error
// against 64 bits of 6 prompts in documents of 300 1.14e-6 with the high part first, 0.56e-6 so.
// What is cut off a long sum still adds up, so O is taken out every CHAIN = 2 blocks and
// added to what its row holds in memory (in L2: 128 KB an SM), with rounding, which takes
// about the 2000 clocks that 128 KB take to L2. Rows over 4000 keys, random and positive
// values: 0.8e-6 and 1.4e-6 (plain fp32 0.8e-6, 0.2e-6); in chains of 3 1.1e-6 and 2.2e-6,
// of 4 1.4e-6 and 3.1e-6, without 9e-6 and 27e-6. One prompt of 8192, cap 50: 1203, 1178, 1133
// and 1040 us. fp16 rows: 2e-5 at 8192 keys, a tenth of their own rounding; units end
// after 32768.
//
// p counts from 2^bias and the running maximum is raised only when a score passes it by
// 2^slack, so p stays below 2^16, fp16's range, and O is rarely rescaled. What the bias
// leaves is the steps of light keys, 2^-24 of p: 2^-37 of the heaviest weight for fp32
// rows, 2^-34 for fp16 ones (Scale). More slack saves rescaling: a prompt of 8192, cap 50,
// fp16 rows with bias and slack 6 and 8 653 us, 10 and 5.9 664, 11 and 4.9 676, 13 and 2.9
// 688; but with 6 and 8 weights from 2^-20 of the heaviest on lost bits and were 0 below
// 2^-31, which shows in the output of thousands of such keys beside a heavy one whose
// value is small.
//
// Warps: 0-3 softmax of tile 0, 4-7 of tile 1, 8 issues the products, 9 the loads (10
// and 11 fill the last warpgroup, which gives registers to the others).
#include <type_traits>

#include "common.cuh"
#include "rows.cuh"

namespace rb {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
template <int HL>
struct Scale {
  static constexpr float bias = HL ? 13.f : 10.f, slack = HL ? 2.9f : 5.9f;
};
constexpr int kSoftWarps = 8;
constexpr int kTileThreads = (kSoftWarps + 4) * 32;
// registers a thread at launch, of a softmax warp and of the others: the split uses what the launch gave
constexpr int kRegSoft = 224, kRegRest = 56;  // 256 x 224 + 128 x 56 = 384 x 168

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
// p[0..3] += v in memory, each sum rounded
__device__ __forceinline__ void add4(float* p, float4 v) {
  asm volatile("red.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(p), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
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
// tanh(y) = y P(y^2) for |y| <= limit, fitted for the least largest relative error. In
// the fused form (together with the exponential): 1e-06 with three terms (fp16 rows, whose
// probabilities are rounded to 2^-12), 1e-08 with five. An odd number of terms has a
// positive last one, so that a masked score, -inf, stays -inf.
template <int HL>
struct Fused {
  static constexpr int N = HL ? 5 : 3;
  static constexpr float limit = HL ? 0.5f : 0.3f;
  static __device__ __forceinline__ float c(int i) {
    constexpr float k[5] = {0.999999987f, -0.333330694f, 0.133247793f, -0.0529860753f, 0.0171350067f}, k3[3] = {0.999998839f, -0.333100216f, 0.12633946f};
    return HL ? k[i] : k3[i < 3 ? i : 0];
  }
};
// For larger scores: 3e-07 and 5e-09.
template <int HL>
struct Wide {
  static constexpr int N = HL ? 9 : 7;
  static constexpr float limit = 1.2f;
  static __device__ __forceinline__ float c(int i) {
    constexpr float k[9] = {1.f,           -0.333332747f,  0.133322015f,   -0.0538841411f, 0.0215497930f,
                            -0.00815800484f, 0.00262519997f, -0.000594539568f, 6.65760599e-05f},
                    k7[7] = {0.999999583f,    -0.333305687f,  0.133013666f,  -0.0525437407f,
                             0.0187073722f, -0.00493616611f, 0.000659012294f};
    return HL ? k[i] : k7[i < 7 ? i : 0];
  }
};
// named barrier `id` of n threads, with the "or" of their values
__device__ __forceinline__ bool any_softmax(int id, int n, bool v) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, %3, %2, p;\n\tselp.u32 %0, 1, 0, "
      "q;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)v), "r"(n), "r"(id)
      : "memory");
  return r != 0;
}
// the sign bits of the two halves of w that are infinite or not a number
__device__ __forceinline__ uint32_t not_finite(uint32_t w) { return ((w & 0x7c007c00u) + 0x04000400u) & 0x80008000u; }

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
  // columns otherwise: there p lies over its tile's scores. (fp16 rows with p over the
  // scores: a prompt of 8192 at head size 128 649 us against 585, chunks at 64 281 against 243.)
  static constexpr bool SEP = HD == 64 || !HL;
  static constexpr int PW = SEP ? 64 * (1 + HL) : kTileKeys;
  static constexpr int P0 = 2 * HD, S0 = SEP ? 512 - kTileKeys : P0, SW = SEP ? 0 : kTileKeys;
  // fp32 rows: blocks that O sums up on the tensor core before it is added, with rounding, to
  // what the row holds in memory.
  static constexpr int CHAIN = 2;
  static_assert(P0 + 2 * PW + (SEP ? kTileKeys : 0) <= 512, "");
  // column, within a tile's P, of the 16 keys of k-step ks; lo: their low parts
  static constexpr __host__ __device__ int pcol(int ks, int lo) {
    return SEP ? lo * 64 + ks * 8 : (ks >> 1) * 32 + lo * 16 + (ks & 1) * 8;
  }
};

template <int HD, int HL, int CAP, int BIAS>
__global__ void __launch_bounds__(kTileThreads, 1) rows_tile_kernel(const __grid_constant__ RowAttnArgs a) {
  using C = TileCfg<HD, HL>;
  constexpr int NS = C::NS, B = kTileKeys;
  extern __shared__ __align__(1024) uint8_t smem[];  // the swizzle follows the address bits
  if (smem_u32(smem) & 1023) {
    report_error(a.err, DEV_TIMEOUT_SMEM);
    return;
  }
  uint8_t* ring = smem + 2 * (1 + HL) * C::QT;
  __shared__ uint64_t q_bar[2], s_bar[2], p_bar[2], o_bar[2], s_free, full[NS], freeb[NS], drain, mend_bar;
  __shared__ uint32_t tmem_slot;
  __shared__ int primed[2];    // 1 + the block before whose product O holds something already
  __shared__ int hold_slot;    // this CTA's place in a.hold, or -1
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_launch_dependents();
  const AttnUnit u = a.units[blockIdx.x];
  const TileSpan sp = a.spans[blockIdx.x];
  const int nt = u.nv > 128 ? 2 : 1, nb = (u.k1 - u.k0 + B - 1) / B;

  if (warp == kSoftWarps) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (tid == 0) {
    int slot = -1;
    if (HL && nb > C::CHAIN) {  // one of as many places as there are SMs, each of which runs one CTA
      uint32_t at;
      asm volatile("mov.u32 %0, %%smid;" : "=r"(at));
      for (int i = 0; i < 4 * a.n_hold && slot < 0; ++i) {
        const int p = (int)((at + i) % (uint32_t)a.n_hold);
        if (atomicCAS(a.hold_busy + p, 0, 1) == 0) slot = p;
      }
      if (slot < 0) report_error(a.err, DEV_TIMEOUT_SMEM);
    }
    hold_slot = slot;
    for (int t = 0; t < 2; ++t) {
      mbar_init(&q_bar[t], 128);
      mbar_init(&s_bar[t], 1);
      mbar_init(&p_bar[t], 128);
      mbar_init(&o_bar[t], 1);
      primed[t] = 0;
    }
    for (int i = 0; i < NS; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&freeb[i], 1);
    }
    mbar_init(&drain, 1);
    mbar_init(&s_free, 128);
    mbar_init(&mend_bar, 128 * nt);
    fence_barrier_init();
  }
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tmem = tmem_slot;
  const bool hold = HL && hold_slot >= 0;
  // whether O starts anew with block j
  auto anew = [&](int j) { return j == 0 || (hold && j % C::CHAIN == 0); };
  // softmax warps: this thread has row tr of its tile
  const int tile = warp >> 2, tr = (warp & 3) * 32 + lane, vec_id = tile * 128 + tr;
  RowInfo r{0, 0, 0x7fffffff, 0};
  int head = 0, row = 0;
  const bool active = warp < kSoftWarps && vec_id < u.nv;
  if (active) {
    const int v = u.v0 + vec_id;
    row = u.row0 + v / a.n_rep;
    head = u.kvh * a.n_rep + v % a.n_rep;
    r = a.rows[row];
  }

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
        for (int part = HL; part >= 0; --part) {  // the low part first (below)
          const uint64_t qd = (desc128(qa + (t * (1 + HL) + part) * C::QT, 16, 1024));
#pragma unroll
          for (int ks = 0; ks < HD / 16; ++ks) {
            const uint32_t off = ((ks >> 2) * C::PANEL + (ks & 3) * 32) >> 4;
            mma_ss(on, tmem + C::S0 + t * C::SW, qd + off, kd + off, ids, part < HL || ks);
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
        const uint32_t more = !anew(j) || *(volatile int*)&primed[t] == j + 1;
        const uint64_t vd = (desc128(ra + slot * C::SLOT, C::PANEL, 1024));
#pragma unroll
        for (int part = HL; part >= 0; --part)
#pragma unroll
          for (int ks = 0; ks < B / 16; ++ks)
            mma_ts(on, tmem + t * HD, tmem + C::P0 + t * C::PW + C::pcol(ks, part), vd + ks * (2048 >> 4), ido,
                   more || part < HL || ks);
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
    const uint32_t lane_base = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t ts = lane_base + C::S0 + tile * C::SW, to = lane_base + tile * HD,
                   tp = lane_base + C::P0 + tile * C::PW;
    bool alive = true;
    float sv = fabsf(a.scale);
    // This warp's 32 rows move between global memory and shared memory 16 bytes a lane,
    // whole rows at a time: a lane per row would touch 32 lines with every access.
    // Chunk ch (16 bytes) of row tr in part `part` of the tile's q, K-major with swizzle:
    uint8_t* const q_tile = smem + tile * (1 + HL) * C::QT;
    auto chunk_at = [&](int row_, int part, int ch) {
      return reinterpret_cast<uint4*>(q_tile + part * C::QT + (ch >> 3) * C::PANEL + row_ * 128 +
                                      (((ch & 7) ^ (row_ & 7)) << 4));
    };
    const int w0 = (warp & 3) * 32;  // the warp's first row
    constexpr int ESZ = HL ? 4 : 2, NCH = HD * ESZ / 16, LPR = NCH, RPI = 32 / LPR;  // lanes a row, rows an access
    const int sub = lane / LPR, ch = lane % LPR;
    {  // q; a negative scale turns it
      const unsigned long long mine =
          active ? (unsigned long long)a.q + ((size_t)row * a.ldq + (size_t)head * HD) * ESZ : 0ull;
      const bool vec = ((reinterpret_cast<uintptr_t>(a.q) | (size_t)a.ldq * ESZ) & 15) == 0;
      // All of the warp's rows at once, asynchronously: fp16 to their place, an fp32 row to those of
      // its two parts, which then replace it. (Loops stay rolled: this code runs once a unit, and
      // fetching it unrolled took 16 K clocks of the 51 K of a short unit.)
      if (vec) {
#pragma unroll 4
        for (int i = 0; i < 32; i += RPI) {
          const unsigned long long p = __shfl_sync(0xffffffffu, mine, i + sub);
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                           smem_u32(chunk_at(w0 + i + sub, ch / (HD / 8), ch % (HD / 8)))),
                       "l"(p ? p + 16 * ch : (unsigned long long)a.q), "r"(p ? 16 : 0)
                       : "memory");
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
      } else {
#pragma unroll 1
        for (int i = 0; i < 32; i += RPI) {
          const unsigned long long p = __shfl_sync(0xffffffffu, mine, i + sub);
          uint4 v = make_uint4(0, 0, 0, 0);
          if (p && HL) {
            const uint32_t* q = reinterpret_cast<const uint32_t*>(p) + 4 * ch;
            v = make_uint4(q[0], q[1], q[2], q[3]);
          } else if (p) {
            const uint16_t* q = reinterpret_cast<const uint16_t*>(p) + 8 * ch;
            v = make_uint4(q[0] | (uint32_t)q[1] << 16, q[2] | (uint32_t)q[3] << 16, q[4] | (uint32_t)q[5] << 16,
                           q[6] | (uint32_t)q[7] << 16);
          }
          *chunk_at(w0 + i + sub, ch / (HD / 8), ch % (HD / 8)) = v;
        }
      }
      __syncwarp();
      float my_mul = 1.f;
      if (HL) {
        const float sign = a.scale < 0.f ? -1.f : 1.f;
#pragma unroll 4
        for (int i = 0; i < 32; i += RPI) {
          const int rr = w0 + i + sub;
          const uint4 raw = *chunk_at(rr, ch / (HD / 8), ch % (HD / 8));
          const float x[4] = {__uint_as_float(raw.x), __uint_as_float(raw.y), __uint_as_float(raw.z),
                              __uint_as_float(raw.w)};
          const float big = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
          uint32_t top = __float_as_uint(big);  // magnitudes in the order of their bits
          if (LPR == 32) {
            top = __reduce_max_sync(0xffffffffu, top);
          } else {
#pragma unroll
            for (int o = LPR / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
          }
          float mul = 1.f;  // 2^(8 - exponent of top), for normal finite tops
          const int e = (int)(top >> 23);
          if (e > 8 && e < 255) mul = __uint_as_float((uint32_t)min(254, 127 + 8 + 127 - e) << 23);
#pragma unroll
          for (int q = 0; q < RPI; ++q) {
            const float m = __shfl_sync(0xffffffffu, mul, q * LPR);
            if (lane == i + q) my_mul = m;
          }
          mul *= sign;
          uint2 hi, lo;
          hi.x = pack2(x[0] * mul, x[1] * mul);
          hi.y = pack2(x[2] * mul, x[3] * mul);
          lo.x = pack2_lo(x[0] * mul, x[1] * mul, hi.x);
          lo.y = pack2_lo(x[2] * mul, x[3] * mul, hi.y);
          __syncwarp();  // the whole row has been read
          reinterpret_cast<uint2*>(chunk_at(rr, 0, ch >> 1))[ch & 1] = hi;
          reinterpret_cast<uint2*>(chunk_at(rr, HL, ch >> 1))[ch & 1] = lo;
        }
      } else if (a.scale < 0.f) {
#pragma unroll 1
        for (int i = 0; i < 32; i += RPI) {
          uint4* v = chunk_at(w0 + i + sub, 0, ch);
          *v = make_uint4(v->x ^ 0x80008000u, v->y ^ 0x80008000u, v->z ^ 0x80008000u, v->w ^ 0x80008000u);
        }
      }
      if (HL) sv /= my_mul;
      proxy_fence();
      mbar_arrive(&q_bar[tile]);
    }
    const int all0 = sp.all0[tile], all1 = sp.all1[tile], in0 = sp.in0, in1 = sp.in1;
    const int both0 = max(sp.all0[0], sp.all0[1]), both1 = min(sp.all1[0], sp.all1[1]);
    const float slope = BIAS && active ? a.slopes[head] * kLog2e : 0.f;
    const float cap2 = a.cap * kLog2e, kcap = CAP ? fmaxf(sv / a.cap, 1.2e-38f) : 0.f;  // above 0: -inf stays -inf
    const float mult = (CAP || BIAS) ? 1.f : fmaxf(sv * kLog2e, 1e-30f);  // scores to base-2 units (-inf stays)
    const float sv2 = sv * kLog2e;
    // coefficients of the fused form, for fp16 rows in powers of the raw score (kept normal)
    float coef[Fused<HL>::N];
    float kp = HL ? cap2 : cap2 * kcap;
#pragma unroll
    for (int q = 0; q < Fused<HL>::N; ++q) {
      coef[q] = kp * Fused<HL>::c(q);
      if (!HL) kp *= kcap * kcap;
    }
    const bool fuse_ok = HL || (kcap > 1e-6f && kcap < 1e4f && cap2 < 1e6f);
    // How the warp applies the cap: 1 Fused and 2 Wide, together with the exponential; 3 on its
    // own, with no bound on the scores. One prompt of 8192, 32 heads of 128: fp16 rows 575,
    // 711 and 970 us, fp32 rows 1203, 1405 and 1708. A larger score raises the form for
    // good: with one chosen for each block, warps that went back and forth between two of
    // them took longer than with either (fp16 rows, 1 and 2: 993 us).
    int form = BIAS || !__all_sync(0xffffffffu, fuse_ok) ? 2 : 1;
    float m = -INFINITY, l = 0.f;
    // elements d .. d + 3 of what this row holds, in units of 2^held: held_at[d * 128 .. + 3]
    float* const held_at = a.hold + (size_t)((hold ? hold_slot : 0) * 2 + tile) * (HD * 128) + tr * 4;
    float held = -INFINITY;
    // Both tiles meet. Not a named barrier, which has no limit: after a wait that ran out
    // one of them may have read other values and not come.
    int met = 0;
    auto meet = [&]() {
      mbar_arrive(&mend_bar);
      if (alive) alive = mbar_wait(&mend_bar, (uint32_t)(met & 1), a.err, DEV_TIMEOUT_DRAIN);
      ++met;
    };
    for (int j = 0; j < nb; ++j) {
      const int kb = u.k0 + j * B;
      if (alive) alive = mbar_wait(&s_bar[tile], (uint32_t)(j & 1), a.err, DEV_TIMEOUT_FULL);
      tc_after();
      float x[B];
#pragma unroll
      for (int i = 0; i < B / 32; ++i) ld32(ts + 32 * i, x + 32 * i);
      wait_ld();
      if (C::SEP) {
        tc_before();
        mbar_arrive(&s_free);
      }
      const bool partial = kb < all0 || kb + B > all1;  // the same for the whole tile
      if (CAP && kb + B > u.k1) {  // keys past the end may be anything and do not choose the form
        const int n = u.k1 - kb;
#pragma unroll
        for (int i = 0; i < B; ++i) x[i] = i < n ? x[i] : 0.f;
      }
      if (CAP && form < 3) {  // the largest magnitude of the warp's scores, unseen keys' included
        float lo4[4] = {0.f, 0.f, 0.f, 0.f}, hi4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < B; i += 8)
#pragma unroll
          for (int q = 0; q < 4; ++q) lo4[q] = min3(lo4[q], x[i + 2 * q], x[i + 2 * q + 1]);
#pragma unroll
        for (int i = 0; i < B; i += 8)
#pragma unroll
          for (int q = 0; q < 4; ++q) hi4[q] = max3(hi4[q], x[i + 2 * q], x[i + 2 * q + 1]);
        const float top = fmaxf(max3(fmaxf(hi4[0], hi4[1]), hi4[2], hi4[3]),
                                -min3(fminf(lo4[0], lo4[1]), lo4[2], lo4[3]));
        const float far = top * kcap;
        if (!__all_sync(0xffffffffu, far <= Wide<HL>::limit)) form = 3;
        else if (!__all_sync(0xffffffffu, far <= Fused<HL>::limit)) form = 2;
      }
      const bool fused = CAP && !BIAS && form < 3;
      if (CAP && !fused) {
        using P = Wide<HL>;
        if (form == 2) {
          const f2 k2 = pair(kcap, kcap);
#pragma unroll
          for (int i = 0; i < B; i += 2) {
            const f2 y = mul2(pair(x[i], x[i + 1]), k2), z = mul2(y, y);
            f2 t = pair(cap2 * P::c(P::N - 1), cap2 * P::c(P::N - 1));
#pragma unroll
            for (int q = P::N - 2; q >= 0; --q) t = fma2(t, z, pair(cap2 * P::c(q), cap2 * P::c(q)));
            unpair(mul2(t, y), x[i], x[i + 1]);
          }
        } else if constexpr (!HL) {
          // cap tanh(y) = cap - 2 cap / (1 + e^(2 y)), off by 2^-22 of the cap: for caps up to 128
          // a weight by 2^-15 of itself, an eighth of what fp16 rows round it by
          const float k = 2.f * kLog2e * kcap;
#pragma unroll
          for (int i = 0; i < B; ++i) x[i] = fmaf(-2.f * cap2, rcp(1.f + ex2(x[i] * k)), cap2);
        } else {
          // the same, but small scores, which other rows' large ones brought here, take the
          // polynomial (a prompt of 8192 with cap 4 takes a fifth longer for it)
          const f2 k2 = pair(kcap, kcap);
#pragma unroll
          for (int i = 0; i < B; i += 2) {
            const f2 y = mul2(pair(x[i], x[i + 1]), k2), z = mul2(y, y);
            f2 t = pair(cap2 * P::c(P::N - 1), cap2 * P::c(P::N - 1));
#pragma unroll
            for (int q = P::N - 2; q >= 0; --q) t = fma2(t, z, pair(cap2 * P::c(q), cap2 * P::c(q)));
            float s0, s1, y0, y1;
            unpair(mul2(t, y), s0, s1);
            unpair(y, y0, y1);
            const float b0 = fmaf(-2.f * cap2, rcp(1.f + ex2(y0 * (2.f * kLog2e))), cap2);
            const float b1 = fmaf(-2.f * cap2, rcp(1.f + ex2(y1 * (2.f * kLog2e))), cap2);
            x[i] = fabsf(y0) <= P::limit ? s0 : b0;
            x[i + 1] = fabsf(y1) <= P::limit ? s1 : b1;
          }
        }
      }
      if (BIAS) {
        if (__all_sync(0xffffffffu, kb + B - 1 <= r.pos)) {  // no key after its row: the distance is linear
          const f2 sl = pair(slope, slope), s2 = pair(CAP ? 1.f : sv2, CAP ? 1.f : sv2);
          const float b0 = slope * (float)(kb - r.pos);
          const f2 b2 = pair(b0, b0);
#pragma unroll
          for (int i = 0; i < B; i += 2)
            unpair(fma2(pair(x[i], x[i + 1]), s2, fma2(pair((float)i, (float)(i + 1)), sl, b2)), x[i], x[i + 1]);
        } else {
#pragma unroll
          for (int i = 0; i < B; ++i)
            x[i] = fmaf(-slope, fabsf((float)(r.pos - kb - i)), CAP ? x[i] : x[i] * sv2);
        }
      }
      if (partial) {
        const int lo = r.lo - kb, hi = max(r.hi, r.lo) - kb;
        if (__any_sync(0xffffffffu, hi < B)) {
#pragma unroll
          for (int i = 0; i < B; ++i) x[i] = i < hi ? x[i] : -INFINITY;
        }
        if (__any_sync(0xffffffffu, lo > 0)) {
#pragma unroll
          for (int i = 0; i < B; ++i) x[i] = i >= lo ? x[i] : -INFINITY;
        }
      }
      float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int i = 0; i < B; i += 8)
#pragma unroll
        for (int q = 0; q < 4; ++q) mx4[q] = max3(mx4[q], x[i + 2 * q], x[i + 2 * q + 1]);
      float mx = max3(fmaxf(mx4[0], mx4[1]), mx4[2], mx4[3]) * mult;
      // the cap keeps the order: where it is fused, it is applied to the maximum alone (by the polynomial
      // as well: an error in proportion to the cap would move all of p)
      if (CAP && fused && mx != -INFINITY) {
        using P = Wide<HL>;
        const float y = mx * kcap, z = y * y;
        float t = P::c(P::N - 1);
#pragma unroll
        for (int q = P::N - 2; q >= 0; --q) t = fmaf(t, z, P::c(q));
        mx = t * y * cap2;
      }
      // each row raises its maximum by its own scores alone
      const bool up = mx > (m == -INFINITY ? m : m + Scale<HL>::slack);
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
      if (HL && j > 0 && anew(j)) {
        if (held == -INFINITY) held = m;  // still so in a row that has seen no key: it holds zeros
        const bool far = m - held > 60.f;
        if (__any_sync(0xffffffffu, far)) {  // scores rose by much: other units
          const float f = far ? ex2(held - m) : 1.f;
#pragma unroll 1
          for (int d = 0; d < HD; d += 4) {
            float4 h = __ldcg(reinterpret_cast<const float4*>(held_at + d * 128));
            h.x *= f, h.y *= f, h.z *= f, h.w *= f;
            __stcg(reinterpret_cast<float4*>(held_at + d * 128), h);
          }
          if (far) held = m;
        }
        const float f = m == -INFINITY ? 1.f : alpha * ex2(m - held);
#pragma unroll 1
        for (int d = 0; d < HD; d += 32) {
          float o[32];
          ld32(to + d, o);
          wait_ld();
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            const float4 v = make_float4(o[i] * f, o[i + 1] * f, o[i + 2] * f, o[i + 3] * f);
            if (j > C::CHAIN) add4(held_at + (d + i) * 128, v);
            else __stcg(reinterpret_cast<float4*>(held_at + (d + i) * 128), v);
          }
        }
      } else if (__any_sync(0xffffffffu, up) && j > 0) {
#pragma unroll 1
        for (int d = 0; d < HD; d += 32) {
          float o[32];
          ld32(to + d, o);
          wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] *= alpha;
          st32(to + d, reinterpret_cast<uint32_t*>(o));
        }
      }
      const float off = Scale<HL>::bias - (m == -INFINITY ? 0.f : m);
      const f2 mult2 = pair(mult, mult), off2 = pair(off, off);
      f2 s2[2] = {0ull, 0ull};
      // Groups of 16 keys, every step for the whole group before the next one: the
      // steps of a key wait for one another, the keys do not.
      auto exps = [&](auto capped) {
        constexpr int FUSED = decltype(capped)::value;
        using P = std::conditional_t<FUSED == 2, Wide<HL>, Fused<HL>>;
        f2 pc[P::N];
#pragma unroll
        for (int q = 0; q < P::N; ++q) {
          const float c = FUSED == 2 ? cap2 * P::c(q) : coef[q < Fused<HL>::N ? q : 0];
          pc[q] = pair(c, c);
        }
        constexpr int G = 8;  // pairs
#pragma unroll
        for (int i = 0; i < B / 32; ++i) {
          uint32_t hi[16], lo[16];
#pragma unroll
          for (int h = 0; h < 16 / G; ++h) {
            f2 y[G];
            float e[2 * G];
#pragma unroll
            for (int g = 0; g < G; ++g) y[g] = pair(x[32 * i + 2 * G * h + 2 * g], x[32 * i + 2 * G * h + 2 * g + 1]);
            if (FUSED) {
              f2 z[G], t[G];
              if (HL || FUSED == 2) {  // fp32 rows have scales of their own, too far apart for powers of them
                const f2 k2 = pair(kcap, kcap);
#pragma unroll
                for (int g = 0; g < G; ++g) y[g] = mul2(y[g], k2);
              }
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
          st16(tp + C::pcol(2 * i, 0), hi);
          if (HL) st16(tp + C::pcol(2 * i, 1), lo);
        }
      };
      if (fused && form == 1) exps(std::integral_constant<int, 1>());
      else if (fused) exps(std::integral_constant<int, 2>());
      else exps(std::integral_constant<int, 0>());
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
        // Each tile looks at the whole block; both find the same, so that they meet below
        // only where something has to be mended.
        uint32_t bad = 0;
#pragma unroll
        for (int ch = 0; ch < HD / 8; ++ch) {
          uint4* p = reinterpret_cast<uint4*>(vrow + (ch >> 3) * C::PANEL + (((ch & 7) ^ (tr & 7)) << 4));
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
        if (any_softmax(2 + tile, 128, bad != 0)) {
          tc_after();
#pragma unroll 1
          for (int d = 0; d < HD; d += 32) {
            float o[32];
            ld32(to + d, o);
            wait_ld();
            if (anew(j))
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
          meet();  // all rows have taken theirs
          for (int ch = tile * (HD / 8 / nt); ch < (tile + 1) * (HD / 8 / nt); ++ch) {
            uint4* p = reinterpret_cast<uint4*>(vrow + (ch >> 3) * C::PANEL + (((ch & 7) ^ (tr & 7)) << 4));
            uint32_t* w = reinterpret_cast<uint32_t*>(p);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t nf = not_finite(w[e]);
              w[e] &= ((nf & 0x8000u) ? 0u : 0xffffu) | ((nf & 0x80000000u) ? 0u : 0xffff0000u);
            }
          }
          proxy_fence();
          meet();
          if (tr == 0) *(volatile int*)&primed[tile] = j + 1;
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
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const bool part = u.slot >= 0;
    if (part && active) a.part_ml[u.slot + vec_id] = make_float2(m, l);
    // O through the tile's place of q, which no product reads any more. Parts stay
    // unnormalised in fp32; fp16 rows have room for half of such a row at a time.
    const int out_esz = part || HL ? 4 : 2, passes = part && !HL ? 2 : 1, nd = HD / passes;
    const unsigned long long mine =
        !active ? 0ull
        : part  ? (unsigned long long)(a.part_o + (size_t)(u.slot + vec_id) * HD)
                : (unsigned long long)a.out + ((size_t)row * a.ldo + (size_t)head * HD) * ESZ;
    const bool vec = part || ((reinterpret_cast<uintptr_t>(a.out) | (size_t)a.ldo * ESZ) & 15) == 0;
#pragma unroll 1
    for (int pass = 0; pass < passes; ++pass) {
#pragma unroll 1
      for (int d = 0; d < nd; d += 32) {
        float o[32];
        ld32(to + pass * nd + d, o);
        wait_ld();
        if (hold) {
          const float f = ex2(held - m);
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            const float4 h = __ldcg(reinterpret_cast<const float4*>(held_at + (d + i) * 128));
            o[i] = fmaf(h.x, f, o[i]);
            o[i + 1] = fmaf(h.y, f, o[i + 1]);
            o[i + 2] = fmaf(h.z, f, o[i + 2]);
            o[i + 3] = fmaf(h.w, f, o[i + 3]);
          }
        }
        if (nb == 0 || l == 0.f)
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0.f;
        if (!part)
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] *= inv;
        if (out_esz == 4) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int c = d / 4 + i;
            *chunk_at(tr, c / (HD / 8), c % (HD / 8)) =
                make_uint4(__float_as_uint(o[4 * i]), __float_as_uint(o[4 * i + 1]), __float_as_uint(o[4 * i + 2]),
                           __float_as_uint(o[4 * i + 3]));
          }
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            *chunk_at(tr, 0, d / 8 + i) = make_uint4(pack2(o[8 * i], o[8 * i + 1]), pack2(o[8 * i + 2], o[8 * i + 3]),
                                                     pack2(o[8 * i + 4], o[8 * i + 5]), pack2(o[8 * i + 6], o[8 * i + 7]));
        }
      }
      __syncwarp();
      const int nch = nd * out_esz / 16, lg = 31 - __clz(nch);  // chunks a row: 8, 16 or 32
      if (vec) {
#pragma unroll 4
        for (int i = 0; i < nch; ++i) {
          const int at = i * 32 + lane, rr = at >> lg, c = at & (nch - 1);
          const unsigned long long p = __shfl_sync(0xffffffffu, mine, rr);
          const uint4 v = *chunk_at(w0 + rr, c / (HD / 8), c % (HD / 8));
          if (p) reinterpret_cast<uint4*>(p + (size_t)pass * nd * out_esz)[c] = v;
        }
      } else {  // rows off 16 bytes (never parts)
        constexpr int EO = HL ? 4 : 2;
#pragma unroll 1
        for (int i = 0; i < nch; ++i) {
          const int at = i * 32 + lane, rr = at >> lg, c = at & (nch - 1);
          const unsigned long long p = __shfl_sync(0xffffffffu, mine, rr);
          const uint4* v = chunk_at(w0 + rr, c / (HD / 8), c % (HD / 8));
          if (!p) continue;
          if (HL) {
#pragma unroll
            for (int e = 0; e < 4; ++e) reinterpret_cast<uint32_t*>(p)[4 * c + e] = (&v->x)[e];
          } else {
#pragma unroll
            for (int e = 0; e < 16 / EO; ++e) reinterpret_cast<uint16_t*>(p)[8 * c + e] = reinterpret_cast<const uint16_t*>(v)[e];
          }
        }
      }
      __syncwarp();
    }
  }
  tc_before();
  __syncthreads();
  tc_after();
  if (tid == 0 && hold) {
    __threadfence();
    atomicExch(a.hold_busy + hold_slot, 0);
  }
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
