// Rows of a step into the paged cache: per-head norms of queries and keys, the
// position rotation and the append in one pass over q, k and v.
//
//   norm:     y_i = x_i w_i / sqrt(mean_j x_j^2 + eps)        (each head by itself)
//   rotation: (y_a, y_b) <- (y_a c - y_b s, y_b c + y_a s)    (pairs a, b of the first
//             `rotary` elements; c, s of the row's position from the table)
//
// in fp32, rounded once into q_out and the cache. Bound by memory: every element
// is read once and written once.
#include "common.cuh"
#include "rows.cuh"

namespace rb {

namespace {

template <class T, int E>
__device__ __forceinline__ void load_vec(const T* p, float* x) {
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int i = 0; i < E; ++i) x[i] = __half2float(p[i]);
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i) x[i] = p[i];
  }
}
template <class T, int E>
__device__ __forceinline__ void store_vec(T* p, const float* x) {
#pragma unroll
  for (int i = 0; i < E; ++i) {
    if constexpr (sizeof(T) == 2) p[i] = __float2half_rn(x[i]);
    else p[i] = x[i];
  }
}

// One warp per (row, head vector): heads 0 .. n_heads - 1 are q's, then k's, then v's.
template <int HD, class TI, class TC>
__global__ void __launch_bounds__(256) rows_append_kernel(const __grid_constant__ RowAppendArgs a) {
  constexpr int E = HD / 32;
  const int lane = threadIdx.x & 31, n_q = a.q ? a.n_heads : 0, n_kv = a.kv.n_kv, per = n_q + 2 * n_kv;
  const long long w = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  if (w >= (long long)a.n_rows * per) return;
  const int row = (int)(w / per), h = (int)(w % per), d = lane * E;
  const RowInfo r = a.rows[row];
  float x[E];
  const float* norm = nullptr;
  bool turn = false;
  if (h < n_q) {
    load_vec<TI, E>(reinterpret_cast<const TI*>(a.q) + (size_t)row * a.ldq + (size_t)h * HD + d, x);
    norm = a.q_norm;
    turn = true;
  } else if (h < n_q + n_kv) {
    load_vec<TI, E>(reinterpret_cast<const TI*>(a.k) + (size_t)row * a.ldk + (size_t)(h - n_q) * HD + d, x);
    norm = a.k_norm;
    turn = true;
  } else {
    load_vec<TI, E>(reinterpret_cast<const TI*>(a.v) + (size_t)row * a.ldv + (size_t)(h - n_q - n_kv) * HD + d, x);
  }
  if (norm) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float inv = rsqrtf(ss * (1.f / HD) + a.eps);
#pragma unroll
    for (int i = 0; i < E; ++i) x[i] *= inv * norm[d + i];
  }
  if (turn && a.rotary) {
    const float* cs = a.rope + (size_t)r.pos * a.rotary;
    const int half = a.rotary / 2;
    if (a.adjacent) {
      if (d < a.rotary)
#pragma unroll
        for (int i = 0; i < E; i += 2) {
          const float c = cs[(d + i) / 2], s = cs[half + (d + i) / 2];
          const float y0 = x[i] * c - x[i + 1] * s, y1 = x[i + 1] * c + x[i] * s;
          x[i] = y0;
          x[i + 1] = y1;
        }
    } else {
      // rotary is a multiple of 8, so the partner of a lane's elements lies in one other lane
      const bool low = d < half;
      const int partner = low ? lane + half / E : lane - half / E;
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const float y = __shfl_sync(0xffffffffu, x[i], partner & 31);
        if (d < a.rotary) {
          const int at = low ? d + i : d + i - half;
          const float c = cs[at], s = cs[half + at];
          x[i] = low ? x[i] * c - y * s : x[i] * c + y * s;
        }
      }
    }
  }
  if (h < n_q) {
    store_vec<TI, E>(reinterpret_cast<TI*>(a.q_out) + (size_t)row * a.ldo + (size_t)h * HD + d, x);
  } else {
    const int which = h >= n_q + n_kv, kvh = h - n_q - which * n_kv;
    const int page = a.kv.ptab[(size_t)r.tenant * a.kv.ptab_stride + (r.pos >> 4)];
    const size_t at = ((((size_t)page * a.kv.n_layers + a.layer) * 2 + which) * n_kv + kvh) * 16 + (r.pos & 15);
    store_vec<TC, E>(reinterpret_cast<TC*>(a.kv.pool) + at * HD + d, x);
  }
}

template <int HD>
cudaError_t launch_hd(const RowAppendArgs& a, cudaStream_t s) {
  const long long warps = (long long)a.n_rows * ((a.q ? a.n_heads : 0) + 2 * a.kv.n_kv);
  const unsigned g = (unsigned)((warps + 7) / 8);
  if (a.in16) {
    if (a.kv.f16) rows_append_kernel<HD, __half, __half><<<g, 256, 0, s>>>(a);
    else rows_append_kernel<HD, __half, float><<<g, 256, 0, s>>>(a);
  } else {
    if (a.kv.f16) rows_append_kernel<HD, float, __half><<<g, 256, 0, s>>>(a);
    else rows_append_kernel<HD, float, float><<<g, 256, 0, s>>>(a);
  }
  return cudaGetLastError();
}

}  // namespace

cudaError_t rows_append_launch(const RowAppendArgs& a, int num_sms, cudaStream_t s) {
  (void)num_sms;
  return a.kv.hd == 128 ? launch_hd<128>(a, s) : launch_hd<64>(a, s);
}

}  // namespace rb
