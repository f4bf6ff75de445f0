// Masked attention of a plan's rows over the paged cache.
//
// Row r at position t sees the keys [lo, hi) of its tenant (causal, window,
// document and prefix masks are such intervals). With x_k = scale q.k,
//   s_k = cap tanh(x_k / cap)  (cap 0: s_k = x_k),  s_k -= slope |t - k|,
//   out = sum_k exp(s_k - m) v_k / sum_k exp(s_k - m),  m = max_k s_k,
// and 0 for a row that sees no key.
#include "common.cuh"
#include "rows.cuh"

namespace rb {

namespace {

constexpr int kRowWarps = 4;
constexpr float kLog2e = 1.4426950408889634f;

template <class T>
__device__ __forceinline__ float ld_f32(const void* p, size_t i) {
  if constexpr (sizeof(T) == 2) return __half2float(reinterpret_cast<const __half*>(p)[i]);
  else return reinterpret_cast<const float*>(p)[i];
}

struct VecInfo {
  int lo, hi, pos, head;
  float slope;
};

// Joins the parts of vector v of an item for the four elements at d, parts in the order
// of the keys; their loads do not wait for one another.
template <int HD, class TO>
__device__ __forceinline__ void join_vec(const RowAttnArgs& a, const JoinItem& it, int v, int d) {
  const float2* pml = a.part_ml + it.slot0 + v;
  const float4* po = reinterpret_cast<const float4*>(a.part_o + (size_t)(it.slot0 + v) * HD + d);
  float M = -INFINITY, L = 0.f;
  float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int p0 = 0; p0 < it.n_parts; p0 += 8) {
    float2 ml[8];
    float4 o[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const bool in = p0 + q < it.n_parts;
      ml[q] = in ? __ldcg(pml + (size_t)(p0 + q) * it.nv) : make_float2(-INFINITY, 0.f);
      o[q] = in ? __ldcg(po + (size_t)(p0 + q) * it.nv * (HD / 4)) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    float m8 = M;
#pragma unroll
    for (int q = 0; q < 8; ++q) m8 = fmaxf(m8, ml[q].x);
    const float f0 = m8 == -INFINITY ? 1.f : exp2f(M - m8);
    L *= f0;
    O.x *= f0;
    O.y *= f0;
    O.z *= f0;
    O.w *= f0;
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const float f = m8 == -INFINITY ? 1.f : exp2f(ml[q].x - m8);
      L += ml[q].y * f;
      O.x += o[q].x * f;
      O.y += o[q].y * f;
      O.z += o[q].z * f;
      O.w += o[q].w * f;
    }
    M = m8;
  }
  const float r = L == 0.f ? 0.f : 1.f / L;
  const float e[4] = {O.x * r, O.y * r, O.z * r, O.w * r};
  const size_t at = (size_t)(it.row0 + (it.v0 + v) / a.n_rep) * a.ldo +
                    (size_t)(it.kvh * a.n_rep + (it.v0 + v) % a.n_rep) * HD + d;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    if constexpr (sizeof(TO) == 2) reinterpret_cast<__half*>(a.out)[at + q] = __float2half_rn(e[q]);
    else reinterpret_cast<float*>(a.out)[at + q] = e[q];
  }
}

// The last CTA that deposits a part of unit u's item joins all of them, whichever CTA
// that is, so the result depends on no order of arrival. Every thread's parts are
// stored before. Ends with a barrier of the CTA.
template <int HD, class TO>
__device__ void join_last(const RowAttnArgs& a, const AttnUnit& u) {
  __shared__ int last;
  const JoinItem it = a.joins[u.join];
  __syncthreads();
  if (threadIdx.x == 0) {
    last = atom_add_acq_rel(&a.counters[u.join], 1) == it.n_parts - 1;
    if (last) a.counters[u.join] = 0;
  }
  __syncthreads();
  if (last)
    for (int i = threadIdx.x; i < it.nv * (HD / 4); i += blockDim.x)
      join_vec<HD, TO>(a, it, i / (HD / 4), i % (HD / 4) * 4);
  __syncthreads();
}

// fp32 caches: K and V in fp32 on the CUDA cores. Each warp streams every fourth page
// of its CTA's share through a ring of its own (bulk copies). Scores: lane (j, hh)
// has key j and half of its elements, starting at chunk j, so that eight lanes meet
// all banks; P V: a lane owns HD / 32 elements. NVT: the vectors an item of this
// launch may have, so that a query head without others on its kv head (1) does not
// pay for eight.
template <int HD>
struct F32Cfg {
  static constexpr int BLK = 16 * HD * 4;
  static constexpr int STAGE = 2 * BLK;
  static constexpr int NST = HD == 128 ? 1 : 3;   // 64 / 96 KB a CTA
  static constexpr int SMEM = 128 + kRowWarps * NST * STAGE + kRowWarps * NST * 8;
};

template <int HD, int NV, class TQ>
__global__ void __launch_bounds__(kRowWarps * 32) rows_f32_kernel(const __grid_constant__ RowAttnArgs a) {
  using C = F32Cfg<HD>;
  constexpr int DPL = HD / 32, NST = C::NST, NCH = HD / 8;  // 16-byte chunks in half a key
  extern __shared__ uint8_t raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 127) & ~uintptr_t(127));
  __shared__ __align__(16) float qs[NV][HD];
  __shared__ VecInfo vi[NV];
  __shared__ float pb[kRowWarps][NV][16];
  __shared__ float mo[kRowWarps][NV][HD];
  __shared__ float mm[kRowWarps][NV], ml[kRowWarps][NV];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, j = lane & 15, hh = lane >> 4;
  const float* pool = reinterpret_cast<const float*>(a.kv.pool);
  uint8_t* ring = smem + warp * NST * C::STAGE;
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + kRowWarps * NST * C::STAGE) + warp * NST;
  if (lane == 0) {
    for (int i = 0; i < NST; ++i) mbar_init(&bar[i], 1);
    fence_barrier_init();
  }
  __syncwarp();
  const int u_begin = a.cta[blockIdx.x], u_end = a.cta[blockIdx.x + 1];
  int pu = u_begin, pk = 0, pk1 = 0, pten = 0, pkvh = 0;
  auto open = [&]() {
    for (; pu < u_end; ++pu) {
      const AttnUnit u = a.units[pu];
      pk = u.k0 + 16 * warp;
      pk1 = u.k1;
      pten = u.tenant;
      pkvh = u.kvh;
      if (pk < pk1) return;
    }
  };
  open();
  int issued = 0, used = 0;
  auto issue = [&](int limit) {
    while (issued < limit && pu < u_end) {
      if (lane == 0) {
        const int page = a.kv.ptab[(size_t)pten * a.kv.ptab_stride + (pk >> 4)], s = issued % NST;
        const float* kb = pool + ((((size_t)page * a.kv.n_layers + a.layer) * 2) * a.kv.n_kv + pkvh) * 16 * HD;
        mbar_arrive_expect_tx(&bar[s], C::STAGE);
        bulk_g2s(ring + s * C::STAGE, kb, C::BLK, &bar[s]);
        bulk_g2s(ring + s * C::STAGE + C::BLK, kb + (size_t)a.kv.n_kv * 16 * HD, C::BLK, &bar[s]);
      }
      ++issued;
      pk += 16 * kRowWarps;
      if (pk >= pk1) {
        ++pu;
        open();
      }
    }
  };
  issue(NST);
  bool alive = true;
  for (int ui = u_begin; ui < u_end; ++ui) {
    const AttnUnit u = a.units[ui];
    __syncthreads();
    for (int i = threadIdx.x; i < NV * HD; i += blockDim.x) {
      const int v = i / HD, d = i % HD;
      float x = 0.f;
      if (v < u.nv) {
        const int row = u.row0 + (u.v0 + v) / a.n_rep, head = u.kvh * a.n_rep + (u.v0 + v) % a.n_rep;
        x = ld_f32<TQ>(a.q, (size_t)row * a.ldq + (size_t)head * HD + d);
      }
      qs[v][d] = x;
    }
    if (threadIdx.x < NV) {
      VecInfo w{0, 0, 0, 0, 0.f};
      if ((int)threadIdx.x < u.nv) {
        const int v = u.v0 + threadIdx.x;
        const RowInfo r = a.rows[u.row0 + v / a.n_rep];
        w.lo = r.lo;
        w.hi = r.hi;
        w.pos = r.pos;
        w.head = u.kvh * a.n_rep + v % a.n_rep;
        w.slope = a.slopes ? a.slopes[w.head] : 0.f;
      }
      vi[threadIdx.x] = w;
    }
    __syncthreads();
    float m[NV], l[NV], o[NV][DPL];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      m[v] = -INFINITY;
      l[v] = 0.f;
#pragma unroll
      for (int d = 0; d < DPL; ++d) o[v][d] = 0.f;
    }
    for (int k = u.k0 + 16 * warp; k < u.k1; k += 16 * kRowWarps) {
      issue(used + NST);
      const int s = used % NST;
      if (alive) alive = mbar_wait(&bar[s], (used / NST) & 1, a.err, DEV_TIMEOUT_FULL);
      const float* kb = reinterpret_cast<const float*>(ring + s * C::STAGE);
      const float* vb = kb + 16 * HD;
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
      const int key = k + j;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        float x = (dot[v] + __shfl_xor_sync(0xffffffffu, dot[v], 16)) * a.scale;
        if (a.cap > 0.f) x = a.cap * tanhf(x / a.cap);
        x = (x - vi[v].slope * fabsf((float)(vi[v].pos - key))) * kLog2e;
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
        if (hh == 0) {
          l[v] += p;
          pb[warp][v][j] = p;
        }
      }
      __syncwarp();
      const int nk = min(16, u.k1 - k);
#pragma unroll 4
      for (int t = 0; t < nk; ++t) {
        float vf[DPL];
        if constexpr (DPL == 4) *reinterpret_cast<float4*>(vf) = *reinterpret_cast<const float4*>(vb + t * HD + lane * DPL);
        else *reinterpret_cast<float2*>(vf) = *reinterpret_cast<const float2*>(vb + t * HD + lane * DPL);
#pragma unroll
        for (int v = 0; v < NV; ++v) {
          const float p = pb[warp][v][t];
          // a masked key adds nothing, whatever its value holds
#pragma unroll
          for (int d = 0; d < DPL; ++d) o[v][d] = p == 0.f ? o[v][d] : fmaf(p, vf[d], o[v][d]);
        }
      }
      __syncwarp();
      ++used;
    }
#pragma unroll
    for (int v = 0; v < NV; ++v) {
#pragma unroll
      for (int w = 8; w > 0; w >>= 1) l[v] += __shfl_xor_sync(0xffffffffu, l[v], w);
#pragma unroll
      for (int d = 0; d < DPL; ++d) mo[warp][v][lane * DPL + d] = o[v][d];
      if (lane == 0) {
        mm[warp][v] = m[v];
        ml[warp][v] = l[v];
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < u.nv * HD; i += blockDim.x) {
      const int v = i / HD, d = i % HD;
      float M = -INFINITY, L = 0.f, O = 0.f;
#pragma unroll
      for (int w = 0; w < kRowWarps; ++w) M = fmaxf(M, mm[w][v]);
#pragma unroll
      for (int w = 0; w < kRowWarps; ++w) {
        const float f = M == -INFINITY ? 1.f : exp2f(mm[w][v] - M);
        L += ml[w][v] * f;
        O += mo[w][v][d] * f;
      }
      if (u.slot >= 0) {
        a.part_o[(size_t)(u.slot + v) * HD + d] = O;
        if (d == 0) a.part_ml[u.slot + v] = make_float2(M, L);
      } else {
        const float r = L == 0.f ? 0.f : O / L;
        const size_t at = (size_t)(u.row0 + (u.v0 + v) / a.n_rep) * a.ldo + (size_t)vi[v].head * HD + d;
        if constexpr (sizeof(TQ) == 2) reinterpret_cast<__half*>(a.out)[at] = __float2half_rn(r);
        else reinterpret_cast<float*>(a.out)[at] = r;
      }
    }
    if (u.slot >= 0) join_last<HD, TQ>(a, u);
  }
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
// Bound by memory: each warp streams every fourth page of its CTA's share through
// a ring of its own (TMA boxes of 16 rows x 128 bytes with 128-byte swizzle);
// the loads run ahead over the ends of units.
// ---------------------------------------------------------------------------
template <int HD>
struct MmaCfg {
  static constexpr int BLK = 16 * HD * 2;                 // K or V of one page and kv head
  static constexpr int STAGE = 2 * BLK;
  static constexpr int NST = HD == 128 ? 3 : 6;           // 96 KB a CTA, two CTAs an SM
  static constexpr int RING = kRowWarps * NST * STAGE;
  static constexpr int SMEM = 1024 + RING + 2 * kSmallVecs * (HD + 2) * 4 + kRowWarps * NST * 8;
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

template <int HD, int HL>
__global__ void __launch_bounds__(kRowWarps * 32, 2) rows_mma_kernel(const __grid_constant__ RowAttnArgs a) {
  using C = MmaCfg<HD>;
  constexpr int NV = kSmallVecs, KS = HD / 16, NST = C::NST;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  float* qs = reinterpret_cast<float*>(smem + C::RING);
  uint64_t* bars = reinterpret_cast<uint64_t*>(qs + 2 * NV * (HD + 2));
  auto mrg = reinterpret_cast<float(*)[NV][HD + 2]>(qs);  // [2], over the queries
  __shared__ float pt[kRowWarps][16][NV];
  __shared__ VecInfo vi[NV];
  __shared__ float qmul[NV];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int u_begin = a.cta[blockIdx.x], u_end = a.cta[blockIdx.x + 1];
  uint8_t* ring = smem + warp * NST * C::STAGE;
  uint64_t* bar = bars + warp * NST;
  if (lane == 0) {
    for (int i = 0; i < NST; ++i) mbar_init(&bar[i], 1);
    fence_barrier_init();
  }
  __syncwarp();

  // this warp's loads: unit pu, key pk (its page), running ahead of the math
  int pu = u_begin, pk = 0, pk1 = 0, pten = 0, pkvh = 0;
  auto open = [&]() {  // the first unit at or after pu with a page for this warp
    for (; pu < u_end; ++pu) {
      const AttnUnit u = a.units[pu];
      pk = u.k0 + 16 * warp;
      pk1 = u.k1;
      pten = u.tenant;
      pkvh = u.kvh;
      if (pk < pk1) return;
    }
  };
  open();
  int cached_t = -1, cached_p = 0, cached = 0;  // lane i: the page of page index cached_p + 4 i
  int issued = 0, used = 0;
  auto issue = [&](int limit) {
    while (issued < limit && pu < u_end) {
      const int p = pk >> 4, off = p - cached_p;
      if (pten != cached_t || off < 0 || (off & 3) || off >= 128) {
        cached_t = pten;
        cached_p = p;
        const int at = p + 4 * lane;
        cached = at < a.kv.ptab_stride ? a.kv.ptab[(size_t)pten * a.kv.ptab_stride + at] : 0;
      }
      const int page = __shfl_sync(0xffffffffu, cached, (p - cached_p) >> 2);
      if (lane == 0) {
        const int s = issued % NST;
        mbar_arrive_expect_tx(&bar[s], C::STAGE);
        const int y = (((page * a.kv.n_layers + a.layer) * 2) * a.kv.n_kv + pkvh) * 16;
#pragma unroll
        for (int w = 0; w < 2; ++w)
#pragma unroll
          for (int b = 0; b < HD / 64; ++b)
            tma_2d(ring + s * C::STAGE + w * C::BLK + b * 2048, &a.tmap, b * 64, y + w * a.kv.n_kv * 16, &bar[s]);
      }
      ++issued;
      pk += 16 * kRowWarps;
      if (pk >= pk1) {
        ++pu;
        open();
      }
    }
  };
  issue(NST);
  bool alive = true;
  int koff[KS], voff[KS];
  {
    const int mi = lane >> 3, rr = lane & 7;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      koff[ks] = swz16(rr + (mi & 1) * 8, ks * 2 + (mi >> 1));
      voff[ks] = swz16(rr + (mi >> 1) * 8, ks * 2 + (mi & 1));
    }
  }
  for (int ui = u_begin; ui < u_end; ++ui) {
    const AttnUnit u = a.units[ui];
    __syncthreads();  // the last unit's queries and partial results are read
    for (int v = warp; v < NV; v += kRowWarps) {  // a warp per vector: load, largest magnitude
      float top = 0.f;
      const int at_v = u.v0 + v;
      const size_t at = (size_t)(u.row0 + at_v / a.n_rep) * a.ldq + (size_t)(u.kvh * a.n_rep + at_v % a.n_rep) * HD;
#pragma unroll
      for (int i = 0; i < HD / 32; ++i) {
        float x = 0.f;
        if (v < u.nv) x = HL ? ld_f32<float>(a.q, at + lane + 32 * i) : ld_f32<__half>(a.q, at + lane + 32 * i);
        qs[v * HD + lane + 32 * i] = x;
        top = fmaxf(top, fabsf(x));
      }
      float mul = 1.f;
      if (HL) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        // 2^(8 - exponent of top), for normal finite tops
        const int e = (int)(__float_as_uint(top) >> 23);
        if (e > 8 && e < 255) mul = __uint_as_float((uint32_t)min(254, 127 + 8 + 127 - e) << 23);
      }
      if (lane == 0) qmul[v] = mul;
      if (lane == 1) {
        VecInfo w{0, 0, 0, 0, 0.f};
        if (v < u.nv) {
          const RowInfo r = a.rows[u.row0 + at_v / a.n_rep];
          w.lo = r.lo;
          w.hi = r.hi;
          w.pos = r.pos;
          w.head = u.kvh * a.n_rep + at_v % a.n_rep;
          w.slope = a.slopes ? a.slopes[w.head] : 0.f;
        }
        vi[v] = w;
      }
    }
    __syncthreads();
    uint32_t qb[KS][1 + HL][2];
    {
      const float mul = HL ? qmul[g] : 1.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const float x0 = qs[g * HD + ks * 16 + 2 * c + 8 * b] * mul, x1 = qs[g * HD + ks * 16 + 2 * c + 8 * b + 1] * mul;
          qb[ks][0][b] = pack2(x0, x1);
          if (HL) qb[ks][HL][b] = pack2_lo(x0, x1, qb[ks][0][b]);
        }
    }
    __syncthreads();  // the queries' place takes the warps' results
    // this lane's two vectors (columns 2c, 2c + 1)
    VecInfo w[2];
    float sv[2];
    int in0 = 0x7fffffff, in1 = 0;      // keys that some vector sees
    int all0 = 0, all1 = 0x7fffffff;    // keys that every vector sees
    bool one_row = true;
#pragma unroll
    for (int v = 0; v < NV; ++v)
      if (v < u.nv) {
        const int lo = vi[v].lo, hi = vi[v].hi;
        if (hi > lo) {
          in0 = min(in0, lo);
          in1 = max(in1, hi);
        }
        all0 = max(all0, lo);
        all1 = min(all1, hi);
      }
    one_row = u.v0 + u.nv <= a.n_rep;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      w[h] = vi[2 * c + h];
      sv[h] = a.scale / (HL ? qmul[2 * c + h] : 1.f);
      if (!(a.cap > 0.f)) sv[h] *= kLog2e;
      w[h].slope *= kLog2e;
    }
    const float icap = a.cap > 0.f ? 1.f / a.cap : 0.f, cap2 = a.cap * kLog2e;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, ot[KS][4];
#pragma unroll
    for (int i = 0; i < KS; ++i) ot[i][0] = ot[i][1] = ot[i][2] = ot[i][3] = 0.f;
    for (int k = u.k0 + 16 * warp; k < u.k1; k += 16 * kRowWarps) {
      issue(used + NST);
      const int s = used % NST;
      if (alive) alive = mbar_wait(&bar[s], (used / NST) & 1, a.err, DEV_TIMEOUT_FULL);
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
      const bool full = k >= all0 && k + 16 <= all1;  // the same in every lane
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
          auto half_mask = [&](int key) { return key >= in0 && key < in1 ? 0xffffu : 0u; };
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
          mma_16816(ot[i], af, h0, h1);
          if (HL) mma_16816(ot[i], af, l0, l1);
        }
      } else {
        // rows that see different keys of this page: in fp32, each vector over its own keys
        pt[warp][g][2 * c] = p[0];
        pt[warp][g][2 * c + 1] = p[1];
        pt[warp][g + 8][2 * c] = p[2];
        pt[warp][g + 8][2 * c + 1] = p[3];
        __syncwarp();
        for (int t = 0; t < 16; ++t) {
          const float p0 = pt[warp][t][2 * c], p1 = pt[warp][t][2 * c + 1];
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
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) l[h] += __shfl_xor_sync(0xffffffffu, l[h], o);
    // the warps' results in pairs (2 and 3 into 0 and 1), then those two
    auto deposit = [&](float (*b)[HD + 2]) {
#pragma unroll
      for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) b[2 * c + (e & 1)][i * 16 + g + (e >> 1) * 8] = ot[i][e];
      if (g == 0)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          b[2 * c + h][HD] = m[h];
          b[2 * c + h][HD + 1] = l[h];
        }
    };
    if (warp >= 2) deposit(mrg[warp - 2]);
    __syncthreads();
    if (warp < 2) {
      const float(*b)[HD + 2] = mrg[warp];
      float f1[2], f2[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float m2 = b[2 * c + h][HD], M = fmaxf(m[h], m2);
        f1[h] = M == -INFINITY ? 1.f : ex2(m[h] - M);
        f2[h] = M == -INFINITY ? 1.f : ex2(m2 - M);
        l[h] = l[h] * f1[h] + b[2 * c + h][HD + 1] * f2[h];
        m[h] = M;
      }
#pragma unroll
      for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          ot[i][e] = ot[i][e] * f1[e & 1] + b[2 * c + (e & 1)][i * 16 + g + (e >> 1) * 8] * f2[e & 1];
      __syncwarp();
      deposit(mrg[warp]);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < u.nv * HD; i += kRowWarps * 32) {
      const int v = i / HD, d = i % HD;
      const float M = fmaxf(mrg[0][v][HD], mrg[1][v][HD]);
      float L = 0.f, O = 0.f;
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const float f = M == -INFINITY ? 1.f : ex2(mrg[q][v][HD] - M);
        L += mrg[q][v][HD + 1] * f;
        O += mrg[q][v][d] * f;
      }
      if (u.slot >= 0) {
        a.part_o[(size_t)(u.slot + v) * HD + d] = O;
        if (d == 0) a.part_ml[u.slot + v] = make_float2(M, L);
      } else {
        const float r = L == 0.f ? 0.f : O / L;
        const size_t at = (size_t)(u.row0 + (u.v0 + v) / a.n_rep) * a.ldo + (size_t)vi[v].head * HD + d;
        if (HL) reinterpret_cast<float*>(a.out)[at] = r;
        else reinterpret_cast<__half*>(a.out)[at] = __float2half_rn(r);
      }
    }
    if (u.slot >= 0) {
      if (HL) join_last<HD, float>(a, u);
      else join_last<HD, __half>(a, u);
    }
  }
}

// Joins the parts of the tile items.
template <int HD, class TO>
__global__ void __launch_bounds__(256) rows_join_kernel(const __grid_constant__ RowAttnArgs a) {
  const JoinItem it = a.joins[a.n_small_joins + blockIdx.x];
  const int v = blockIdx.y * (256 / (HD / 4)) + threadIdx.x / (HD / 4);
  if (v < it.nv) join_vec<HD, TO>(a, it, v, threadIdx.x % (HD / 4) * 4);
}

}  // namespace

template <int HD, int HL>
static cudaError_t launch_mma(const RowAttnArgs& a, cudaStream_t s) {
  int dev = 0;
  cudaGetDevice(&dev);
  if (cudaError_t e = ensure_smem_attr(rows_mma_kernel<HD, HL>, MmaCfg<HD>::SMEM, dev)) return e;
  rows_mma_kernel<HD, HL><<<a.n_cta, kRowWarps * 32, MmaCfg<HD>::SMEM, s>>>(a);
  return cudaGetLastError();
}

template <int HD, int NV>
static cudaError_t launch_f32(const RowAttnArgs& a, cudaStream_t s) {
  int dev = 0;
  cudaGetDevice(&dev);
  constexpr int smem = F32Cfg<HD>::SMEM;
  if (a.q16) {
    if (cudaError_t e = ensure_smem_attr(rows_f32_kernel<HD, NV, __half>, smem, dev)) return e;
    rows_f32_kernel<HD, NV, __half><<<a.n_cta, kRowWarps * 32, smem, s>>>(a);
  } else {
    if (cudaError_t e = ensure_smem_attr(rows_f32_kernel<HD, NV, float>, smem, dev)) return e;
    rows_f32_kernel<HD, NV, float><<<a.n_cta, kRowWarps * 32, smem, s>>>(a);
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
  if (a.n_cta < 1) return cudaSuccess;
  if (a.kv.f16) {
    if (a.kv.hd == 128) return a.q16 ? launch_mma<128, 0>(a, s) : launch_mma<128, 1>(a, s);
    return a.q16 ? launch_mma<64, 0>(a, s) : launch_mma<64, 1>(a, s);
  }
  return a.kv.hd == 128 ? launch_f32_vecs<128>(a, s) : launch_f32_vecs<64>(a, s);
}

cudaError_t rows_join_launch(const RowAttnArgs& a, cudaStream_t s) {
  const int n = a.n_joins - a.n_small_joins;
  if (n < 1) return cudaSuccess;
  const dim3 g(n, kTileVecs * a.kv.hd / 4 / 256);
  if (a.kv.hd == 128) {
    if (a.q16) rows_join_kernel<128, __half><<<g, 256, 0, s>>>(a);
    else rows_join_kernel<128, float><<<g, 256, 0, s>>>(a);
  } else {
    if (a.q16) rows_join_kernel<64, __half><<<g, 256, 0, s>>>(a);
    else rows_join_kernel<64, float><<<g, 256, 0, s>>>(a);
  }
  return cudaGetLastError();
}

}  // namespace rb
