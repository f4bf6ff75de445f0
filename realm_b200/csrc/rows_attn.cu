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

// Scalar kernel: any cache type; K and V read straight from the pages.
template <int HD, class T>
__global__ void __launch_bounds__(kRowWarps * 32) rows_scalar_kernel(const __grid_constant__ RowAttnArgs a) {
  constexpr int NV = kSmallVecs, DPL = HD / 32;
  __shared__ __align__(16) float qs[NV][HD];
  __shared__ VecInfo vi[NV];
  __shared__ float pb[kRowWarps][NV][16];
  __shared__ float mo[kRowWarps][NV][HD];
  __shared__ float mm[kRowWarps][NV], ml[kRowWarps][NV];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, j = lane & 15, hh = lane >> 4;
  const T* pool = reinterpret_cast<const T*>(a.kv.pool);
  for (int ui = a.cta[blockIdx.x]; ui < a.cta[blockIdx.x + 1]; ++ui) {
    const AttnUnit u = a.units[ui];
    __syncthreads();
    for (int i = threadIdx.x; i < NV * HD; i += blockDim.x) {
      const int v = i / HD, d = i % HD;
      float x = 0.f;
      if (v < u.nv) {
        const int row = u.row0 + (u.v0 + v) / a.n_rep, head = u.kvh * a.n_rep + (u.v0 + v) % a.n_rep;
        const size_t at = (size_t)row * a.ldq + (size_t)head * HD + d;
        x = a.q16 ? ld_f32<__half>(a.q, at) : ld_f32<float>(a.q, at);
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
      const int page = a.kv.ptab[(size_t)u.tenant * a.kv.ptab_stride + (k >> 4)];
      const T* kb = pool + ((((size_t)page * a.kv.n_layers + a.layer) * 2) * a.kv.n_kv + u.kvh) * 16 * HD;
      const T* vb = kb + (size_t)a.kv.n_kv * 16 * HD;
      float dot[NV];
#pragma unroll
      for (int v = 0; v < NV; ++v) dot[v] = 0.f;
      for (int d = hh * (HD / 2); d < (hh + 1) * (HD / 2); d += 4) {
        float kf[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) kf[e] = ld_f32<T>(kb, j * HD + d + e);
#pragma unroll
        for (int v = 0; v < NV; ++v) {
          const float4 q = *reinterpret_cast<const float4*>(&qs[v][d]);
          dot[v] = fmaf(q.x, kf[0], fmaf(q.y, kf[1], fmaf(q.z, kf[2], fmaf(q.w, kf[3], dot[v]))));
        }
      }
      const int key = k + j;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        float x = (dot[v] + __shfl_xor_sync(0xffffffffu, dot[v], 16)) * a.scale;
        if (a.cap > 0.f) x = a.cap * tanhf(x / a.cap);
        x = (x - vi[v].slope * fabsf((float)(vi[v].pos - key))) * kLog2e;
        const bool in = key >= vi[v].lo && key < vi[v].hi;
        float mx = in ? x : -INFINITY;
#pragma unroll
        for (int s = 8; s > 0; s >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, s));
        const float mn = fmaxf(m[v], mx);
        const float alpha = mn == -INFINITY ? 1.f : exp2f(m[v] - mn);
        const float p = in ? exp2f(x - (mn == -INFINITY ? 0.f : mn)) : 0.f;
        float sum = p;
#pragma unroll
        for (int s = 8; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
        l[v] = l[v] * alpha + sum;
        m[v] = mn;
        if (hh == 0) pb[warp][v][j] = p;
#pragma unroll
        for (int d = 0; d < DPL; ++d) o[v][d] *= alpha;
      }
      __syncwarp();
      const int nk = min(16, u.k1 - k);
      for (int t = 0; t < nk; ++t) {
        float vf[DPL];
#pragma unroll
        for (int d = 0; d < DPL; ++d) vf[d] = ld_f32<T>(vb, t * HD + lane * DPL + d);
#pragma unroll
        for (int v = 0; v < NV; ++v) {
          const float p = pb[warp][v][t];
          // a masked key adds nothing, whatever its value holds
#pragma unroll
          for (int d = 0; d < DPL; ++d) o[v][d] = p == 0.f ? o[v][d] : fmaf(p, vf[d], o[v][d]);
        }
      }
      __syncwarp();
    }
#pragma unroll
    for (int v = 0; v < NV; ++v) {
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
      float M = -INFINITY;
#pragma unroll
      for (int w = 0; w < kRowWarps; ++w) M = fmaxf(M, mm[w][v]);
      float L = 0.f, O = 0.f;
      if (M != -INFINITY)
#pragma unroll
        for (int w = 0; w < kRowWarps; ++w) {
          const float f = exp2f(mm[w][v] - M);
          L += ml[w][v] * f;
          O += mo[w][v][d] * f;
        }
      else
#pragma unroll
        for (int w = 0; w < kRowWarps; ++w) L += ml[w][v];  // a score that is not a number leaves M unset
      if (u.slot >= 0) {
        a.part_o[(size_t)(u.slot + v) * HD + d] = O;
        if (d == 0) a.part_ml[u.slot + v] = make_float2(M, L);
      } else {
        const float r = L == 0.f ? 0.f : M == -INFINITY ? L : O / L;
        const int row = u.row0 + (u.v0 + v) / a.n_rep;
        const size_t at = (size_t)row * a.ldo + (size_t)vi[v].head * HD + d;
        if (a.q16) reinterpret_cast<__half*>(a.out)[at] = __float2half_rn(r);
        else reinterpret_cast<float*>(a.out)[at] = r;
      }
    }
  }
}

// Joins the parts of an item: one CTA per (item, vector), parts in order.
template <int HD>
__global__ void __launch_bounds__(HD) rows_join_kernel(const __grid_constant__ RowAttnArgs a) {
  const JoinItem it = a.joins[blockIdx.x];
  const int d = threadIdx.x;
  for (int v = blockIdx.y; v < it.nv; v += gridDim.y) {
    float M = -INFINITY;
    for (int p = 0; p < it.n_parts; ++p) M = fmaxf(M, a.part_ml[it.slot0 + p * it.nv + v].x);
    float L = 0.f, O = 0.f;
    for (int p = 0; p < it.n_parts; ++p) {
      const int s = it.slot0 + p * it.nv + v;
      const float2 ml = a.part_ml[s];
      const float f = M == -INFINITY ? 1.f : exp2f(ml.x - M);
      L += ml.y * f;
      O += a.part_o[(size_t)s * HD + d] * f;
    }
    const float r = L == 0.f ? 0.f : M == -INFINITY ? L : O / L;
    const int row = it.row0 + (it.v0 + v) / a.n_rep, head = it.kvh * a.n_rep + (it.v0 + v) % a.n_rep;
    const size_t at = (size_t)row * a.ldo + (size_t)head * HD + d;
    if (a.q16) reinterpret_cast<__half*>(a.out)[at] = __float2half_rn(r);
    else reinterpret_cast<float*>(a.out)[at] = r;
  }
}

}  // namespace

cudaError_t rows_small_launch(const RowAttnArgs& a, cudaStream_t s) {
  if (a.n_cta < 1) return cudaSuccess;
  const dim3 g(a.n_cta), b(kRowWarps * 32);
  if (a.kv.f16) {
    if (a.kv.hd == 128) rows_scalar_kernel<128, __half><<<g, b, 0, s>>>(a);
    else rows_scalar_kernel<64, __half><<<g, b, 0, s>>>(a);
  } else {
    if (a.kv.hd == 128) rows_scalar_kernel<128, float><<<g, b, 0, s>>>(a);
    else rows_scalar_kernel<64, float><<<g, b, 0, s>>>(a);
  }
  return cudaGetLastError();
}

cudaError_t rows_join_launch(const RowAttnArgs& a, cudaStream_t s) {
  if (a.n_joins < 1) return cudaSuccess;
  const dim3 g(a.n_joins, kSmallVecs);
  if (a.kv.hd == 128) rows_join_kernel<128><<<g, 128, 0, s>>>(a);
  else rows_join_kernel<64><<<g, 64, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace rb
