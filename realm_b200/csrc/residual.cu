// What lies between a block's last projection and the next block's first one:
//   z = y w1 / sqrt(mean y^2 + eps), h = x + scale * gate * z, out = h w2 / sqrt(mean h^2 + eps)
// in one pass: a row stays in registers from its reads to its writes, and the two sums of
// squares are all that its threads exchange. fp32 throughout, each output rounded once.
//
// A group of T threads has a row, each thread up to NC chunks of 8 consecutive
// elements, T chunks apart: 16 or 32 bytes a load, coalesced. Rows off 16 bytes (odd
// widths) take single elements T apart instead: as many bytes in flight, all lines still
// used whole.
//
// Bound by memory: 8192 x 4096, fp16 on an fp32 stream with a shared gate 75 us (403 MB, 5.4 TB/s, 83 % of a copy's
// rate); with one chunk of 512 threads 79 us, four of 128 80 us, one with registers cut for a third CTA 82. One row of 4096
// is the call: 9 us, of which the kernel about 3.
#include <algorithm>

#include "common.cuh"
#include "residual.cuh"

namespace rb {

namespace {

constexpr int kE = 8;  // elements of a chunk

template <class T>
__device__ __forceinline__ void load8(const T* p, float (&v)[kE]) {
  if constexpr (sizeof(T) == 2) {
    const uint4 q = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(u32_as_h2(w[i]));
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  } else {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  }
}
template <class T>
__device__ __forceinline__ void store8(T* p, const float (&v)[kE]) {
  if constexpr (sizeof(T) == 2) {
    uint4 q;
    q.x = h2_as_u32(__floats2half2_rn(v[0], v[1]));
    q.y = h2_as_u32(__floats2half2_rn(v[2], v[3]));
    q.z = h2_as_u32(__floats2half2_rn(v[4], v[5]));
    q.w = h2_as_u32(__floats2half2_rn(v[6], v[7]));
    *reinterpret_cast<uint4*>(p) = q;
  } else {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
  }
}

// A thread's elements of a row: f(index of element e of chunk c) where it is below dim.
template <class T, int NC, bool VEC>
struct Row {
  int dim, t, threads;
  __device__ __forceinline__ int at(int c, int e) const {
    return VEC ? (c * threads + t) * kE + e : (c * kE + e) * threads + t;
  }
  template <class U>
  __device__ __forceinline__ void load(const U* p, int c, float (&v)[kE]) const {
    if constexpr (VEC) {
      if (at(c, 0) < dim) {
        load8(p + at(c, 0), v);
        return;
      }
#pragma unroll
      for (int e = 0; e < kE; ++e) v[e] = 0.f;
    } else {
#pragma unroll
      for (int e = 0; e < kE; ++e) v[e] = at(c, e) < dim ? (float)p[at(c, e)] : 0.f;
    }
  }
  template <class U>
  __device__ __forceinline__ void store(U* p, int c, const float (&v)[kE]) const {
    if constexpr (VEC) {
      if (at(c, 0) < dim) store8(p + at(c, 0), v);
    } else {
#pragma unroll
      for (int e = 0; e < kE; ++e)
        if (at(c, e) < dim) p[at(c, e)] = (U)v[e];
    }
  }
};

// sum over the row's threads; with more than a warp of them through `red`
__device__ __forceinline__ float row_sum(float v, float* red, int threads) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (threads == 32) return v;
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  const int n = threads >> 5;
  v = (int)(threadIdx.x & 31) < n ? red[threadIdx.x & 31] : 0.f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <class TY, class TX, int NC, bool VEC, int MAXT>
__global__ void __launch_bounds__(MAXT) residual_kernel(const __grid_constant__ ResidualArgs a) {
  __shared__ float red[2][32];
  pdl_launch_dependents();
  pdl_wait();
  const int row = blockIdx.x * blockDim.y + threadIdx.y;
  if (row >= a.n_rows) return;  // whole warps; a block with several rows has no barrier
  const Row<TY, NC, VEC> r{a.dim, (int)threadIdx.x, (int)blockDim.x};
  const TY* yp = reinterpret_cast<const TY*>(a.y) + (int64_t)row * a.ldy;
  const TX* xp = reinterpret_cast<const TX*>(a.x) + (int64_t)row * a.ldx;
  // the widest rows read x after the first sum: their threads have 64 registers
  constexpr bool LATE = MAXT == 1024;
  float z[NC][kE], h[LATE ? 1 : NC][kE];
#pragma unroll
  for (int c = 0; c < NC; ++c) r.load(yp, c, z[c]);
  if (!LATE) {
#pragma unroll
    for (int c = 0; c < NC; ++c) r.load(xp, c, h[LATE ? 0 : c]);
  }
  float f = 1.f;
  if (a.post) {
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < kE; ++e) s = fmaf(z[c][e], z[c][e], s);
    f = 1.f / sqrtf(row_sum(s, red[0], r.threads) / (float)a.dim + a.eps);
  }
  float s = 0.f;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    float w[kE];
    if (a.post) {
      r.load(a.post, c, w);
#pragma unroll
      for (int e = 0; e < kE; ++e) z[c][e] = z[c][e] * f * w[e];
    }
    if (a.gate) {
      r.load(reinterpret_cast<const TY*>(a.gate) + (int64_t)row * a.ldg, c, w);
#pragma unroll
      for (int e = 0; e < kE; ++e) z[c][e] *= w[e];
    }
    float(&x)[kE] = h[LATE ? 0 : c];
    if (LATE) r.load(xp, c, x);
#pragma unroll
    for (int e = 0; e < kE; ++e) {
      z[c][e] = fmaf(a.scale, z[c][e], x[e]);  // h from here on
      // places past the row hold 0 unless the scale or f is not finite
      if (VEC ? r.at(c, 0) < a.dim : r.at(c, e) < a.dim) s = fmaf(z[c][e], z[c][e], s);
    }
    r.store(reinterpret_cast<TX*>(a.x_out) + (int64_t)row * a.ldxo, c, z[c]);
  }
  if (!a.out) return;
  f = 1.f / sqrtf(row_sum(s, red[1], r.threads) / (float)a.dim + a.eps);
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    float w[kE];
    r.load(a.pre, c, w);
#pragma unroll
    for (int e = 0; e < kE; ++e) w[e] *= z[c][e] * f;
    r.store(reinterpret_cast<TY*>(a.out) + (int64_t)row * a.ldo, c, w);
  }
}

template <class TY, class TX, int NC, bool VEC, int MAXT>
cudaError_t launch(const ResidualArgs& a, int threads, int rows, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((a.n_rows + rows - 1) / rows));
  cfg.blockDim = dim3((unsigned)threads, (unsigned)rows);
  cfg.stream = s;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, residual_kernel<TY, TX, NC, VEC, MAXT>, a);
}

template <class TY, class TX, bool VEC>
cudaError_t launch_chunks(const ResidualArgs& a, cudaStream_t s) {
  const int chunks = (a.dim + kE - 1) / kE;
  const int nc = chunks <= 256 ? 1 : chunks <= 1024 ? 2 : 4, most = chunks <= 2048 ? 512 : 1024;
  const int threads = std::min(most, ((chunks + nc - 1) / nc + 31) / 32 * 32);
  const int rows = threads == 32 ? 4 : 1;
  if (nc == 1) return launch<TY, TX, 1, VEC, 512>(a, threads, rows, s);
  if (nc == 2) return launch<TY, TX, 2, VEC, 512>(a, threads, rows, s);
  if (most == 512) return launch<TY, TX, 4, VEC, 512>(a, threads, rows, s);
  return launch<TY, TX, 4, VEC, 1024>(a, threads, rows, s);
}

template <class TY, class TX>
cudaError_t launch_type(const ResidualArgs& a, cudaStream_t s) {
  auto on16 = [&](const void* p, int64_t ld, int esz) {
    return !p || ((uintptr_t)p % 16 == 0 && (a.n_rows == 1 || ld * esz % 16 == 0));
  };
  const int ey = sizeof(TY), ex = sizeof(TX);
  const bool vec = a.dim % kE == 0 && on16(a.y, a.ldy, ey) && on16(a.gate, a.ldg, ey) && on16(a.out, a.ldo, ey) &&
                   on16(a.x, a.ldx, ex) && on16(a.x_out, a.ldxo, ex) && on16(a.post, 0, 4) && on16(a.pre, 0, 4);
  return vec ? launch_chunks<TY, TX, true>(a, s) : launch_chunks<TY, TX, false>(a, s);
}

}  // namespace

cudaError_t residual_launch(const ResidualArgs& a, cudaStream_t s) {
  if (a.y16) return a.x16 ? launch_type<__half, __half>(a, s) : launch_type<__half, float>(a, s);
  return a.x16 ? launch_type<float, __half>(a, s) : launch_type<float, float>(a, s);
}

}  // namespace rb
