// Masked attention of a plan's rows over the paged cache.
//
// Row r at position t sees the keys [lo, hi) of its tenant (causal, window,
// document and prefix masks are such intervals). With x_k = scale q.k,
//   s_k = cap tanh(x_k / cap)  (cap 0: s_k = x_k),  s_k -= slope |t - k|,
//   out = sum_k exp(s_k - m) v_k / sum_k exp(s_k - m),  m = max_k s_k,
// and 0 for a row that sees no key.
#include <type_traits>

#include "common.cuh"
#include "rows.cuh"

namespace rb {

namespace {

constexpr float kLog2e = 1.4426950408889634f;

template <class T>
__device__ __forceinline__ float ld_f32(const void* p, size_t i) {
  if constexpr (sizeof(T) == 2) return __half2float(reinterpret_cast<const __half*>(p)[i]);
  else return reinterpret_cast<const float*>(p)[i];
}

struct VecInfo {
  int lo, hi, pos;
  float slope;
};

// Vector v of a unit: the row of the call and the query head.
__device__ __forceinline__ int vec_row(const RowAttnArgs& a, int row0, int v0, int v) { return row0 + (v0 + v) / a.n_rep; }
__device__ __forceinline__ int vec_head(const RowAttnArgs& a, int kvh, int v0, int v) {
  return kvh * a.n_rep + (v0 + v) % a.n_rep;
}
__device__ __forceinline__ VecInfo vec_info(const RowAttnArgs& a, const AttnUnit& u, int v) {
  VecInfo w{0, 0, 0, 0.f};
  if (v < u.nv) {
    const RowInfo r = a.rows[vec_row(a, u.row0, u.v0, v)];
    w.lo = r.lo;
    w.hi = r.hi;
    w.pos = r.pos;
    if (a.slopes) w.slope = a.slopes[vec_head(a, u.kvh, u.v0, v)] * kLog2e;
  }
  return w;
}
template <class TO>
__device__ __forceinline__ void store_out(const RowAttnArgs& a, size_t at, float x) {
  if constexpr (sizeof(TO) == 2) reinterpret_cast<__half*>(a.out)[at] = __float2half_rn(x);
  else reinterpret_cast<float*>(a.out)[at] = x;
}

// This warp's loads run ahead of its math, over the ends of units: unit pu, key pk.
struct Ahead {
  int pu, end, pk, pk1, tenant, kvh;
  __device__ __forceinline__ void open(const RowAttnArgs& a) {  // the first unit from pu on that has keys
    for (; pu < end; ++pu) {
      const AttnUnit& u = a.units[pu];
      pk = u.k0;
      pk1 = u.k1;
      tenant = u.tenant;
      kvh = u.kvh;
      if (pk < pk1) return;
    }
  }
  __device__ __forceinline__ void next(const RowAttnArgs& a) {
    pk += kRowPage;
    if (pk >= pk1) {
      ++pu;
      open(a);
    }
  }
};
// The page of a tenant's token k; a warp keeps 32 entries of the table, one a lane.
struct PageCache {
  int tenant = -1, first = 0, val = 0;
  __device__ __forceinline__ int page(const RowAttnArgs& a, int t, int k) {
    const int p = k >> 4;
    if (t != tenant || p < first || p >= first + 32) {
      tenant = t;
      first = p;
      const int at = p + (threadIdx.x & 31);
      val = at < a.kv.ptab_stride ? a.kv.ptab[(size_t)t * a.kv.ptab_stride + at] : 0;
    }
    return __shfl_sync(0xffffffffu, val, p - first);
  }
};

// fp32 caches: K and V in fp32 on the CUDA cores. Each warp streams its share of the
// pages through a ring of its own (bulk copies, K and V blocks in turn). Scores: lane
// (j, hh) has key j and half of its elements, starting at chunk j, so that eight lanes
// meet all banks; P V: a lane owns HD / 32 elements. NV: the vectors an item of this
// launch may have, so that a query head without others on its kv head (1) does not
// pay for eight: 8 tenants of 100-3001 tokens, 16 kv heads of 64, one, two and four
// vectors 38, 40 and 44 us, with the form for eight 56, 56 and 58. Bound by memory:
// with a window of 1024 16 us for 55 MB (3.4 TB/s; 12 pages a warp are little to stream).
template <int HD, int NV>
struct F32Cfg {
  static constexpr int BLK = 16 * HD * 4;
  static constexpr int NST = HD == 128 ? 3 : 6;   // blocks a warp: 96 KB a CTA
  static constexpr int SMEM = 128 + kRowWarps * NST * (BLK + 8);
  // Two CTAs an SM, as the plan counts its warps: 228 KB, of which each takes 1 KB for the system.
  // The probabilities go through shared memory where that leaves room (PB), else by shuffles: eight
  // vectors at 128, 8 tenants x 64 rows after 2000 tokens, 32 heads on 8, 1115 us against 1510 with one
  // CTA; eight at 64, where both fit, 790 us by shuffles, 730 through shared memory.
  static constexpr int Q = kRowWarps * NV * (HD * 4 + (int)sizeof(VecInfo)), P = kRowWarps * NV * 16 * 4;
  static constexpr bool PB = 2 * (SMEM + Q + P + 1024) <= 228 * 1024;
  static_assert(2 * (SMEM + Q + 1024) <= 228 * 1024, "");
};

template <int HD, int NV, class TQ>
__global__ void __launch_bounds__(kRowWarps * 32, 2) rows_f32_kernel(const __grid_constant__ RowAttnArgs a) {
  using C = F32Cfg<HD, NV>;
  constexpr int DPL = HD / 32, NST = C::NST, NCH = HD / 8;  // 16-byte chunks in half a key
  extern __shared__ uint8_t raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 127) & ~uintptr_t(127));
  __shared__ __align__(16) float q_all[kRowWarps][NV][HD];
  __shared__ VecInfo vi_all[kRowWarps][NV];
  __shared__ float pb_all[C::PB ? kRowWarps : 1][C::PB ? NV : 1][16];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, j = lane & 15, hh = lane >> 4;
  const int me = blockIdx.x * kRowWarps + warp;
  pdl_launch_dependents();
  if (me >= a.n_warps) return;
  auto qs = q_all[warp];
  VecInfo* vi = vi_all[warp];
  auto pb = pb_all[C::PB ? warp : 0];
  const float* pool = reinterpret_cast<const float*>(a.kv.pool);
  uint8_t* ring = smem + warp * NST * C::BLK;
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + kRowWarps * NST * C::BLK) + warp * NST;
  if (lane == 0) {
    for (int i = 0; i < NST; ++i) mbar_init(&bar[i], 1);
    fence_barrier_init();
  }
  __syncwarp();
  const int u_begin = a.warps[me], u_end = a.warps[me + 1];
  Ahead ah{u_begin, u_end, 0, 0, 0, 0};
  PageCache pages;
  ah.open(a);
  int issued = 0, landed = 0, used = 0, which = 0;
  bool alive = true;  // the same in every lane; a wait that ran out ends the warp's work
  const float* block = nullptr;
  auto issue = [&](int limit) {
    while (alive && issued < limit && ah.pu < u_end) {
      if (which == 0) {
        const int page = pages.page(a, ah.tenant, ah.pk);
        block = pool + ((((size_t)page * a.kv.n_layers + a.layer) * 2) * a.kv.n_kv + ah.kvh) * 16 * HD;
      }
      if (lane == 0) {
        const int s = issued % NST;
        mbar_arrive_expect_tx(&bar[s], C::BLK);
        bulk_g2s(ring + s * C::BLK, block + (which ? (size_t)a.kv.n_kv * 16 * HD : 0), C::BLK, &bar[s]);
      }
      ++issued;
      which ^= 1;
      if (which == 0) ah.next(a);
    }
  };
  issue(NST);
  // the next block of the ring; done with it: release()
  auto take = [&]() {
    const int s = used % NST;
    if (alive) alive = __all_sync(0xffffffffu, mbar_wait(&bar[s], (used / NST) & 1, a.err, DEV_TIMEOUT_FULL));
    landed += alive;
    return reinterpret_cast<const float*>(ring + s * C::BLK);
  };
  auto release = [&]() {
    __syncwarp();
    ++used;
    issue(used + NST);
  };
  for (int ui = u_begin; ui < u_end && alive; ++ui) {
    const AttnUnit u = a.units[ui];
    __syncwarp();
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const size_t at = (size_t)vec_row(a, u.row0, u.v0, v) * a.ldq + (size_t)vec_head(a, u.kvh, u.v0, v) * HD + lane;
#pragma unroll
      for (int i = 0; i < DPL; ++i) qs[v][lane + 32 * i] = v < u.nv ? ld_f32<TQ>(a.q, at + 32 * i) : 0.f;
    }
    if (lane < NV) vi[lane] = vec_info(a, u, lane);
    __syncwarp();
    float m[NV], l[NV], o[NV][DPL];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      m[v] = -INFINITY;
      l[v] = 0.f;
#pragma unroll
      for (int d = 0; d < DPL; ++d) o[v][d] = 0.f;
    }
    for (int k = u.k0; k < u.k1 && alive; k += kRowPage) {
      const float* kb = take();
      float dot[NV];
#pragma unroll
      for (int v = 0; v < NV; ++v) dot[v] = 0.f;
#pragma unroll 8
      for (int ch = 0; ch < NCH; ++ch) {
        const int d = hh * (HD / 2) + ((ch + j) & (NCH - 1)) * 4;
        const float4 kf = *reinterpret_cast<const float4*>(kb + j * HD + d);
#pragma unroll
        for (int v = 0; v < NV; ++v) {
          const float4 q = *reinterpret_cast<const float4*>(&qs[v][d]);
          dot[v] = fmaf(q.x, kf.x, fmaf(q.y, kf.y, fmaf(q.z, kf.z, fmaf(q.w, kf.w, dot[v]))));
        }
      }
      release();
      const int key = k + j;
      float pk[NV];  // of key j, in both lanes that have it
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        float x = (dot[v] + __shfl_xor_sync(0xffffffffu, dot[v], 16)) * a.scale;
        if (a.cap > 0.f) x = a.cap * tanhf(x / a.cap);
        x = fmaf(x, kLog2e, -vi[v].slope * fabsf((float)(vi[v].pos - key)));
        const bool in = key >= vi[v].lo && key < vi[v].hi;
        // the maximum is raised only when some score passes it; the sums stay per lane
        if (__any_sync(0xffffffffu, in && x > m[v])) {
          float mx = in ? x : -INFINITY;
#pragma unroll
          for (int w = 8; w > 0; w >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
          mx = fmaxf(m[v], mx);
          const float alpha = mx == -INFINITY ? 1.f : exp2f(m[v] - mx);
          l[v] *= alpha;
          m[v] = mx;
#pragma unroll
          for (int d = 0; d < DPL; ++d) o[v][d] *= alpha;
        }
        const float p = in ? exp2f(x - (m[v] == -INFINITY ? 0.f : m[v])) : 0.f;
        if (hh == 0) l[v] += p;
        pk[v] = p;
        if (C::PB && hh == 0) pb[v][j] = p;
      }
      const float* vb = take();
      if (C::PB) __syncwarp();
      const int nk = min(16, u.k1 - k);
#pragma unroll 4
      for (int t = 0; t < nk; ++t) {
        float vf[DPL];
        if constexpr (DPL == 4) *reinterpret_cast<float4*>(vf) = *reinterpret_cast<const float4*>(vb + t * HD + lane * DPL);
        else *reinterpret_cast<float2*>(vf) = *reinterpret_cast<const float2*>(vb + t * HD + lane * DPL);
#pragma unroll
        for (int v = 0; v < NV; ++v) {
          const float p = C::PB ? pb[v][t] : __shfl_sync(0xffffffffu, pk[v], t);
          // a masked key adds nothing, whatever its value holds
#pragma unroll
          for (int d = 0; d < DPL; ++d) o[v][d] = p == 0.f ? o[v][d] : fmaf(p, vf[d], o[v][d]);
        }
      }
      release();
    }
    if (!alive) break;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
#pragma unroll
      for (int w = 16; w > 0; w >>= 1) l[v] += __shfl_xor_sync(0xffffffffu, l[v], w);
      if (v >= u.nv) continue;
      if (u.slot >= 0) {
#pragma unroll
        for (int d = 0; d < DPL; ++d) a.part_o[(size_t)(u.slot + v) * HD + lane * DPL + d] = o[v][d];
        if (lane == 0) a.part_ml[u.slot + v] = make_float2(m[v], l[v]);
      } else {
        const float r = l[v] == 0.f ? 0.f : 1.f / l[v];
        const size_t at = (size_t)vec_row(a, u.row0, u.v0, v) * a.ldo + (size_t)vec_head(a, u.kvh, u.v0, v) * HD;
#pragma unroll
        for (int d = 0; d < DPL; ++d) store_out<TQ>(a, at + lane * DPL + d, o[v][d] * r);
      }
    }
  }
  // after a wait that ran out: what is in flight lands before the shared memory goes away
  for (; landed < issued; ++landed) mbar_wait(&bar[landed % NST], (landed / NST) & 1, a.err, DEV_TIMEOUT_FULL);
}

// ---------------------------------------------------------------------------
// fp16 caches: the same items on the tensor cores (mma.sync m16n8k16).
//
// Per page of 16 keys and item of 8 query vectors: S^T = K Q^T (A = K by
// ldmatrix, B = the queries), the softmax of a vector in the lanes of its column,
// O^T += V^T P^T (A = V by ldmatrix.trans, B = P by movmatrix). fp32 rows split q
// and p into fp16 hi + lo (two products each, 22 bits); fp16 rows take q as it is
// and round p. q is brought to a power of two near 2^8 first and p counts from
// 2^12 down, so that neither part meets fp16's subnormals where it matters.
//
// Bound by memory: each warp streams its share of the pages through a ring of its own
// (TMA boxes of 16 rows x 128 bytes with 128-byte swizzle); the loads run ahead over
// the ends of units. Warps share nothing: with the four warps of a CTA on one unit,
// its start and end (barriers, merges) took 6 us a unit, 72 us for 16 tenants of
// 512-8192 tokens; so 62 us (285 MB, 4.6 TB/s). 4 tenants of 65537-131072 tokens with 64
// heads: 250 to 270 us, 6.0 to 6.4 TB/s.
// ---------------------------------------------------------------------------
template <int HD>
struct MmaCfg {
  static constexpr int BLK = 16 * HD * 2;                 // K or V of one page and kv head
  static constexpr int STAGE = 2 * BLK;
  static constexpr int NST = HD == 128 ? 3 : 6;           // 96 KB a CTA, two CTAs an SM
  static constexpr int RING = kRowWarps * NST * STAGE;
  static constexpr int SMEM = 1024 + RING + kRowWarps * NST * 8;
};
constexpr float kPBias = 12.f;  // p = 2^(s - m + 12)

__device__ __forceinline__ int swz16(int r, int k) {  // byte of (row r, 16-byte chunk k) in swizzled boxes of 64 columns
  return (k >> 3) * 2048 + r * 128 + (((k & 7) ^ (r & 7)) << 4);
}
__device__ __forceinline__ void tma_2d(void* dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void ldm4(uint32_t r[4], const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(smem_u32(p)));
}
__device__ __forceinline__ void ldm4t(uint32_t r[4], const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(smem_u32(p)));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack2(float a, float b) { return h2_as_u32(__floats2half2_rn(a, b)); }
__device__ __forceinline__ uint32_t pack2_lo(float a, float b, uint32_t hi) {
  const float2 f = __half22float2(u32_as_h2(hi));
  return pack2(a - f.x, b - f.y);
}

// Two consecutive elements of a query vector as the B operand wants them
template <int HL>
__device__ __forceinline__ float2 load_q2(const RowAttnArgs& a, size_t at, bool whole) {
  if (HL) {
    const float* p = reinterpret_cast<const float*>(a.q) + at;
    return whole ? *reinterpret_cast<const float2*>(p) : make_float2(p[0], p[1]);
  }
  const __half* p = reinterpret_cast<const __half*>(a.q) + at;
  return __half22float2(whole ? *reinterpret_cast<const __half2*>(p) : __halves2half2(p[0], p[1]));
}

template <int HD, int HL>
__global__ void __launch_bounds__(kRowWarps * 32, 2) rows_mma_kernel(const __grid_constant__ RowAttnArgs a) {
  using C = MmaCfg<HD>;
  using TO = typename std::conditional<HL != 0, float, __half>::type;
  constexpr int NV = kSmallVecs, KS = HD / 16, NST = C::NST;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  __shared__ float pt_all[kRowWarps][16][NV];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int me = blockIdx.x * kRowWarps + warp;
  pdl_launch_dependents();
  if (me >= a.n_warps) return;
  auto pt = pt_all[warp];
  uint8_t* ring = smem + warp * NST * C::STAGE;
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + C::RING) + warp * NST;
  if (lane == 0) {
    for (int i = 0; i < NST; ++i) mbar_init(&bar[i], 1);
    fence_barrier_init();
  }
  __syncwarp();
  const int u_begin = a.warps[me], u_end = a.warps[me + 1];
  Ahead ah{u_begin, u_end, 0, 0, 0, 0};
  PageCache pages;
  ah.open(a);
  int issued = 0, landed = 0, used = 0;
  bool alive = true;  // the same in every lane; a wait that ran out ends the warp's work
  auto issue = [&](int limit) {
    while (alive && issued < limit && ah.pu < u_end) {
      const int page = pages.page(a, ah.tenant, ah.pk);
      if (lane == 0) {
        const int s = issued % NST;
        mbar_arrive_expect_tx(&bar[s], C::STAGE);
        const int y = (((page * a.kv.n_layers + a.layer) * 2) * a.kv.n_kv + ah.kvh) * 16;
#pragma unroll
        for (int w = 0; w < 2; ++w)
#pragma unroll
          for (int b = 0; b < HD / 64; ++b)
            tma_2d(ring + s * C::STAGE + w * C::BLK + b * 2048, &a.tmap, b * 64, y + w * a.kv.n_kv * 16, &bar[s]);
      }
      ++issued;
      ah.next(a);
    }
  };
  issue(NST);
  int koff[KS], voff[KS];
  {
    const int mi = lane >> 3, rr = lane & 7;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      koff[ks] = swz16(rr + (mi & 1) * 8, ks * 2 + (mi >> 1));
      voff[ks] = swz16(rr + (mi >> 1) * 8, ks * 2 + (mi & 1));
    }
  }
  const bool whole = ((reinterpret_cast<uintptr_t>(a.q) | (size_t)a.ldq * (HL ? 4 : 2)) & (HL ? 7 : 3)) == 0;
  for (int ui = u_begin; ui < u_end && alive; ++ui) {
    const AttnUnit u = a.units[ui];
    uint32_t qb[KS][1 + HL][2];
    float mul = 1.f;
    {  // lane (g, c) holds elements 2c, 2c + 1 and 2c + 8, 2c + 9 of every 16 of vector g
      const size_t at = (size_t)vec_row(a, u.row0, u.v0, g) * a.ldq + (size_t)vec_head(a, u.kvh, u.v0, g) * HD + 2 * c;
      float2 x[KS][2];
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int b = 0; b < 2; ++b)
          x[ks][b] = g < u.nv ? load_q2<HL>(a, at + ks * 16 + 8 * b, whole) : make_float2(0.f, 0.f);
      if (HL) {
        float top = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int b = 0; b < 2; ++b) top = fmaxf(top, fmaxf(fabsf(x[ks][b].x), fabsf(x[ks][b].y)));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // 2^(8 - exponent of top), for normal finite tops
        const int e = (int)(__float_as_uint(top) >> 23);
        if (e > 8 && e < 255) mul = __uint_as_float((uint32_t)min(254, 127 + 8 + 127 - e) << 23);
      }
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          qb[ks][0][b] = pack2(x[ks][b].x * mul, x[ks][b].y * mul);
          if (HL) qb[ks][HL][b] = pack2_lo(x[ks][b].x * mul, x[ks][b].y * mul, qb[ks][0][b]);
        }
    }
    // this lane's two vectors in the scores (columns 2c, 2c + 1)
    VecInfo w[2];
    float sv[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      w[h] = vec_info(a, u, 2 * c + h);
      sv[h] = a.scale / __shfl_sync(0xffffffffu, mul, (2 * c + h) * 4);
      if (!(a.cap > 0.f)) sv[h] *= kLog2e;
    }
    const bool one_row = u.v0 + u.nv <= a.n_rep;
    const float icap = a.cap > 0.f ? 1.f / a.cap : 0.f, cap2 = a.cap * kLog2e;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, ot[KS][4];
#pragma unroll
    for (int i = 0; i < KS; ++i) ot[i][0] = ot[i][1] = ot[i][2] = ot[i][3] = 0.f;
    for (int k = u.k0; k < u.k1; k += kRowPage) {
      const int s = used % NST;
      alive = __all_sync(0xffffffffu, mbar_wait(&bar[s], (used / NST) & 1, a.err, DEV_TIMEOUT_FULL));
      if (!alive) break;
      ++landed;
      const uint8_t* kb = ring + s * C::STAGE;
      const uint8_t* vb = kb + C::BLK;
      float sa[4][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) sa[i][0] = sa[i][1] = sa[i][2] = sa[i][3] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        uint32_t af[4];
        ldm4(af, kb + koff[ks]);
        if (HL) {
          mma_16816(sa[(ks & 1) * 2], af, qb[ks][0][0], qb[ks][0][1]);
          mma_16816(sa[(ks & 1) * 2 + 1], af, qb[ks][HL][0], qb[ks][HL][1]);
        } else {
          mma_16816(sa[ks & 3], af, qb[ks][0][0], qb[ks][0][1]);
        }
      }
      const bool full = k >= u.all0 && k + 16 <= u.all1;  // the same in every lane
      float x[4];  // (key g, vector 2c), (g, 2c + 1), (g + 8, 2c), (g + 8, 2c + 1)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int h = i & 1, key = k + g + (i >> 1) * 8;
        float y = ((sa[0][i] + sa[2][i]) + (sa[1][i] + sa[3][i])) * sv[h];
        if (a.cap > 0.f) y = cap2 * tanhf(y * icap);
        if (a.slopes) y -= w[h].slope * fabsf((float)(w[h].pos - key));
        if (!full && !(key >= w[h].lo && key < w[h].hi)) y = -INFINITY;
        x[i] = y;
      }
      // the maximum is raised only when some score passes it
      if (__any_sync(0xffffffffu, fmaxf(x[0], x[2]) > m[0] || fmaxf(x[1], x[3]) > m[1])) {
        float al[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float mx = fmaxf(x[h], x[2 + h]);
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
          mx = fmaxf(m[h], mx);
          al[h] = mx == -INFINITY ? 1.f : ex2(m[h] - mx);
          l[h] *= al[h];
          m[h] = mx;
        }
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          ot[i][0] *= al[0];
          ot[i][1] *= al[1];
          ot[i][2] *= al[0];
          ot[i][3] *= al[1];
        }
      }
      float p[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float mm = m[i & 1];
        p[i] = ex2(x[i] - (mm == -INFINITY ? 0.f : mm) + kPBias);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) l[h] += p[h] + p[2 + h];
      if (full || one_row) {
        uint32_t h0 = pack2(p[0], p[1]), h1 = pack2(p[2], p[3]), l0 = 0, l1 = 0;
        if (HL) {
          l0 = transpose8(pack2_lo(p[0], p[1], h0));
          l1 = transpose8(pack2_lo(p[2], p[3], h1));
        }
        h0 = transpose8(h0);
        h1 = transpose8(h1);
        // values of keys that no vector sees do not enter the product
        uint32_t z0 = 0xffffffffu, z1 = 0xffffffffu;
        if (!full) {
          auto half_mask = [&](int key) { return key >= u.in0 && key < u.in1 ? 0xffffu : 0u; };
          z0 = half_mask(k + 2 * c) | half_mask(k + 2 * c + 1) << 16;
          z1 = half_mask(k + 2 * c + 8) | half_mask(k + 2 * c + 9) << 16;
        }
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          uint32_t af[4];
          ldm4t(af, vb + voff[i]);
          if (!full) {
            af[0] &= z0;
            af[1] &= z0;
            af[2] &= z1;
            af[3] &= z1;
          }
          float t[4] = {0.f, 0.f, 0.f, 0.f};  // a page by itself: the tensor core cuts sums off, the adds below round
          if (HL) mma_16816(t, af, l0, l1);
          mma_16816(t, af, h0, h1);
#pragma unroll
          for (int e = 0; e < 4; ++e) ot[i][e] += t[e];
        }
      } else {
        // rows that see different keys of this page: in fp32, each vector over its own keys
        pt[g][2 * c] = p[0];
        pt[g][2 * c + 1] = p[1];
        pt[g + 8][2 * c] = p[2];
        pt[g + 8][2 * c + 1] = p[3];
        __syncwarp();
        for (int t = 0; t < 16; ++t) {
          const float p0 = pt[t][2 * c], p1 = pt[t][2 * c + 1];
#pragma unroll
          for (int i = 0; i < KS; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int d = i * 16 + g + 8 * e;
              const float v = __half2float(*reinterpret_cast<const __half*>(vb + swz16(t, d >> 3) + 2 * (d & 7)));
              if (p0 != 0.f) ot[i][2 * e] = fmaf(p0, v, ot[i][2 * e]);
              if (p1 != 0.f) ot[i][2 * e + 1] = fmaf(p1, v, ot[i][2 * e + 1]);
            }
        }
      }
      __syncwarp();  // the stage is read before it is loaded again
      ++used;
      issue(used + NST);
    }
    if (!alive) break;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) l[h] += __shfl_xor_sync(0xffffffffu, l[h], o);
    // 32-byte runs of a vector in eight lanes
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int v = 2 * c + h;
      if (v >= u.nv) continue;
      if (u.slot >= 0) {
        float* dst = a.part_o + (size_t)(u.slot + v) * HD + g;
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          dst[i * 16] = ot[i][h];
          dst[i * 16 + 8] = ot[i][2 + h];
        }
        if (g == 0) a.part_ml[u.slot + v] = make_float2(m[h], l[h]);
      } else {
        const float r = l[h] == 0.f ? 0.f : 1.f / l[h];
        const size_t at = (size_t)vec_row(a, u.row0, u.v0, v) * a.ldo + (size_t)vec_head(a, u.kvh, u.v0, v) * HD + g;
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          store_out<TO>(a, at + i * 16, ot[i][h] * r);
          store_out<TO>(a, at + i * 16 + 8, ot[i][2 + h] * r);
        }
      }
    }
  }
  // after a wait that ran out: what is in flight lands before the shared memory goes away
  for (; landed < issued; ++landed) mbar_wait(&bar[landed % NST], (landed / NST) & 1, a.err, DEV_TIMEOUT_FULL);
}

// Joins the parts of the items that were cut, parts in the order of the keys: a thread
// has four elements of one vector, and sixteen parts' loads do not wait for one another.
// A kernel of its own, launched ahead of its start (its launch costs nothing then): the
// last warp of an item joining its parts took 40 us for 37 parts of 8 vectors.
template <int HD, class TO>
__global__ void __launch_bounds__(128) rows_join_kernel(const __grid_constant__ RowAttnArgs a) {
  constexpr int LPV = HD / 4, NP = 16;
  const JoinItem it = a.joins[blockIdx.x];
  const int v = blockIdx.y * (128 / LPV) + threadIdx.x / LPV, d = threadIdx.x % LPV * 4;
  if (v >= it.nv) return;
  pdl_wait();
  float M = -INFINITY, L = 0.f;
  float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int p0 = 0; p0 < it.n_parts; p0 += NP) {
    float2 ml[NP];
    float4 o[NP];
#pragma unroll
    for (int q = 0; q < NP; ++q) {
      const bool in = p0 + q < it.n_parts;
      const size_t s = (size_t)it.slot0 + (size_t)(p0 + q) * it.nv + v;
      ml[q] = in ? __ldcg(a.part_ml + s) : make_float2(-INFINITY, 0.f);
      o[q] = in ? __ldcg(reinterpret_cast<const float4*>(a.part_o + s * HD + d)) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    float mn = M;
#pragma unroll
    for (int q = 0; q < NP; ++q) mn = fmaxf(mn, ml[q].x);
    const float f0 = mn == -INFINITY ? 1.f : exp2f(M - mn);
    L *= f0;
    O.x *= f0;
    O.y *= f0;
    O.z *= f0;
    O.w *= f0;
#pragma unroll
    for (int q = 0; q < NP; ++q) {
      const float f = mn == -INFINITY ? 1.f : exp2f(ml[q].x - mn);
      L += ml[q].y * f;
      O.x += o[q].x * f;
      O.y += o[q].y * f;
      O.z += o[q].z * f;
      O.w += o[q].w * f;
    }
    M = mn;
  }
  const float r = L == 0.f ? 0.f : 1.f / L;
  const size_t at = (size_t)vec_row(a, it.row0, it.v0, v) * a.ldo + (size_t)vec_head(a, it.kvh, it.v0, v) * HD + d;
  store_out<TO>(a, at, O.x * r);
  store_out<TO>(a, at + 1, O.y * r);
  store_out<TO>(a, at + 2, O.z * r);
  store_out<TO>(a, at + 3, O.w * r);
}

}  // namespace

template <int HD, int HL>
static cudaError_t launch_mma(const RowAttnArgs& a, cudaStream_t s) {
  int dev = 0;
  cudaGetDevice(&dev);
  if (cudaError_t e = ensure_smem_attr(rows_mma_kernel<HD, HL>, MmaCfg<HD>::SMEM, dev)) return e;
  rows_mma_kernel<HD, HL><<<(a.n_warps + kRowWarps - 1) / kRowWarps, kRowWarps * 32, MmaCfg<HD>::SMEM, s>>>(a);
  return cudaGetLastError();
}

template <int HD, int NV>
static cudaError_t launch_f32(const RowAttnArgs& a, cudaStream_t s) {
  int dev = 0;
  cudaGetDevice(&dev);
  constexpr int smem = F32Cfg<HD, NV>::SMEM;
  if (a.q16) {
    if (cudaError_t e = ensure_smem_attr(rows_f32_kernel<HD, NV, __half>, smem, dev)) return e;
    rows_f32_kernel<HD, NV, __half><<<(a.n_warps + kRowWarps - 1) / kRowWarps, kRowWarps * 32, smem, s>>>(a);
  } else {
    if (cudaError_t e = ensure_smem_attr(rows_f32_kernel<HD, NV, float>, smem, dev)) return e;
    rows_f32_kernel<HD, NV, float><<<(a.n_warps + kRowWarps - 1) / kRowWarps, kRowWarps * 32, smem, s>>>(a);
  }
  return cudaGetLastError();
}
template <int HD>
static cudaError_t launch_f32_vecs(const RowAttnArgs& a, cudaStream_t s) {
  if (a.max_nv <= 1) return launch_f32<HD, 1>(a, s);
  if (a.max_nv <= 2) return launch_f32<HD, 2>(a, s);
  if (a.max_nv <= 4) return launch_f32<HD, 4>(a, s);
  return launch_f32<HD, 8>(a, s);
}

cudaError_t rows_small_launch(const RowAttnArgs& a, cudaStream_t s) {
  if (a.n_warps < 1) return cudaSuccess;
  if (a.kv.f16) {
    if (a.kv.hd == 128) return a.q16 ? launch_mma<128, 0>(a, s) : launch_mma<128, 1>(a, s);
    return a.q16 ? launch_mma<64, 0>(a, s) : launch_mma<64, 1>(a, s);
  }
  return a.kv.hd == 128 ? launch_f32_vecs<128>(a, s) : launch_f32_vecs<64>(a, s);
}

template <int HD, class TO>
static cudaError_t launch_join(const RowAttnArgs& a, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)a.n_joins, (unsigned)((a.join_nv * (HD / 4) + 127) / 128));
  cfg.blockDim = dim3(128);
  cfg.stream = s;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, rows_join_kernel<HD, TO>, a);
}

cudaError_t rows_join_launch(const RowAttnArgs& a, cudaStream_t s) {
  if (a.n_joins < 1) return cudaSuccess;
  if (a.kv.hd == 128) return a.q16 ? launch_join<128, __half>(a, s) : launch_join<128, float>(a, s);
  return a.q16 ? launch_join<64, __half>(a, s) : launch_join<64, float>(a, s);
}

}  // namespace rb
