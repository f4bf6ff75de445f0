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

// N floats at a place aligned to them (8 or 16 bytes)
template <int N>
__device__ __forceinline__ void load_f32(const float* p, float* x) {
  if constexpr (N == 2) {
    *reinterpret_cast<float2*>(x) = __ldg(reinterpret_cast<const float2*>(p));
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) *reinterpret_cast<float4*>(x + i) = __ldg(reinterpret_cast<const float4*>(p + i));
  }
}
// E elements at a place aligned to them
template <class T, int E>
__device__ __forceinline__ void store_vec16(T* p, const float* x) {
  if constexpr (sizeof(T) == 2) {
    uint32_t h[E / 2];
#pragma unroll
    for (int i = 0; i < E / 2; ++i) h[i] = h2_as_u32(__floats2half2_rn(x[2 * i], x[2 * i + 1]));
    if constexpr (E == 8) *reinterpret_cast<uint4*>(p) = make_uint4(h[0], h[1], h[2], h[3]);
    else *reinterpret_cast<uint2*>(p) = make_uint2(h[0], h[1]);
  } else {
#pragma unroll
    for (int i = 0; i < E; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
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

// The same with 16-byte accesses: a head vector takes LPH lanes of E elements, a
// warp HPW of them at a time and U such groups in flight. Needs the tables and every
// row of q, k, v and q_out on 16 bytes, and rotation pairs that lie E-aligned in one lane each (or
// adjacent ones).
template <int HD, class TI, class TC, int U>
__global__ void __launch_bounds__(256) rows_append_vec_kernel(const __grid_constant__ RowAppendArgs a, int groups) {
  constexpr int E = 16 / sizeof(TI), LPH = HD / E, HPW = 32 / LPH;
  const int lane = threadIdx.x & 31, sub = lane / LPH, d = (lane % LPH) * E;
  const int n_q = a.q ? a.n_heads : 0, n_kv = a.kv.n_kv, per = n_q + 2 * n_kv;
  const long long w = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  const int row = (int)(w / groups), h0 = (int)(w % groups) * (HPW * U) + sub;
  if (row >= a.n_rows) return;
  const RowInfo r = a.rows[row];
  uint4 raw[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int h = h0 + i * HPW;
    const TI* p = nullptr;
    if (h < n_q) p = reinterpret_cast<const TI*>(a.q) + (size_t)row * a.ldq + (size_t)h * HD;
    else if (h < n_q + n_kv) p = reinterpret_cast<const TI*>(a.k) + (size_t)row * a.ldk + (size_t)(h - n_q) * HD;
    else if (h < per) p = reinterpret_cast<const TI*>(a.v) + (size_t)row * a.ldv + (size_t)(h - n_q - n_kv) * HD;
    raw[i] = p ? *reinterpret_cast<const uint4*>(p + d) : make_uint4(0, 0, 0, 0);
  }
  const int page = a.kv.ptab[(size_t)r.tenant * a.kv.ptab_stride + (r.pos >> 4)];
  // the lane's cosines and sines: E of each (half split) or E / 2 (adjacent pairs)
  const bool turned = d < a.rotary;
  const int half = a.rotary / 2;
  const bool low = d < half;
  float cs[E], sn[E];
  if (turned) {
    const float* t = a.rope + (size_t)r.pos * a.rotary;
    if (a.adjacent) {
      float c2[E / 2], s2[E / 2];
      load_f32<E / 2>(t + d / 2, c2);
      load_f32<E / 2>(t + half + d / 2, s2);
#pragma unroll
      for (int i = 0; i < E; ++i) {
        cs[i] = c2[i / 2];
        sn[i] = s2[i / 2];
      }
    } else {
      const int at = low ? d : d - half;
      load_f32<E>(t + at, cs);
      load_f32<E>(t + half + at, sn);
    }
  }
  // the lane with the other halves of this lane's pairs, in the same head
  const int partner = low ? lane + half / E : lane - half / E;
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int h = h0 + i * HPW;
    float x[E];
    load_vec<TI, E>(reinterpret_cast<const TI*>(&raw[i]), x);
    const float* norm = h < n_q ? a.q_norm : h < n_q + n_kv ? a.k_norm : nullptr;
    if (a.q_norm || a.k_norm) {
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) ss = fmaf(x[e], x[e], ss);
#pragma unroll
      for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      if (norm) {
        const float inv = rsqrtf(ss * (1.f / HD) + a.eps);
        float wn[E];
        load_f32<E>(norm + d, wn);
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] *= inv * wn[e];
      }
    }
    if (a.rotary) {
      const bool turn = turned && h < n_q + n_kv;
      if (a.adjacent) {
        if (turn)
#pragma unroll
          for (int e = 0; e < E; e += 2) {
            const float y0 = x[e] * cs[e] - x[e + 1] * sn[e], y1 = x[e + 1] * cs[e] + x[e] * sn[e];
            x[e] = y0;
            x[e + 1] = y1;
          }
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float y = __shfl_sync(0xffffffffu, x[e], partner & 31);
          if (turn) x[e] = low ? x[e] * cs[e] - y * sn[e] : x[e] * cs[e] + y * sn[e];
        }
      }
    }
    if (h >= per) continue;
    if (h < n_q) {
      store_vec16<TI, E>(reinterpret_cast<TI*>(a.q_out) + (size_t)row * a.ldo + (size_t)h * HD + d, x);
    } else {
      const int which = h >= n_q + n_kv, kvh = h - n_q - which * n_kv;
      const size_t at = ((((size_t)page * a.kv.n_layers + a.layer) * 2 + which) * n_kv + kvh) * 16 + (r.pos & 15);
      store_vec16<TC, E>(reinterpret_cast<TC*>(a.kv.pool) + at * HD + d, x);
    }
  }
}

template <int HD, class TI, class TC>
cudaError_t launch_types(const RowAppendArgs& a, int num_sms, cudaStream_t s) {
  constexpr int E = 16 / sizeof(TI), HPW = 32 / (HD / E);
  const long long per = (a.q ? a.n_heads : 0) + 2 * a.kv.n_kv;
  auto bad = [&](const void* p, int64_t ld) { return p && ((reinterpret_cast<uintptr_t>(p) | (size_t)ld * sizeof(TI)) & 15); };
  const uintptr_t tables = reinterpret_cast<uintptr_t>(a.rope) | reinterpret_cast<uintptr_t>(a.q_norm) |
                           reinterpret_cast<uintptr_t>(a.k_norm);
  const bool vec = !(tables & 15) && !bad(a.q, a.ldq) && !bad(a.k, a.ldk) && !bad(a.v, a.ldv) && !bad(a.q_out, a.ldo) &&
                   (a.adjacent || a.rotary / 2 % E == 0);
  if (!vec) {
    const long long warps = a.n_rows * per;
    rows_append_kernel<HD, TI, TC><<<(unsigned)((warps + 7) / 8), 256, 0, s>>>(a);
    return cudaGetLastError();
  }
  // one group a warp while that leaves no SM with more than a few warps, else four
  const long long one = (per + HPW - 1) / HPW;
  if (a.n_rows * one <= 32ll * num_sms) {
    rows_append_vec_kernel<HD, TI, TC, 1><<<(unsigned)((a.n_rows * one + 7) / 8), 256, 0, s>>>(a, (int)one);
  } else {
    const long long four = (per + 4 * HPW - 1) / (4 * HPW);
    rows_append_vec_kernel<HD, TI, TC, 4><<<(unsigned)((a.n_rows * four + 7) / 8), 256, 0, s>>>(a, (int)four);
  }
  return cudaGetLastError();
}

template <int HD>
cudaError_t launch_hd(const RowAppendArgs& a, int num_sms, cudaStream_t s) {
  if (a.in16) return a.kv.f16 ? launch_types<HD, __half, __half>(a, num_sms, s) : launch_types<HD, __half, float>(a, num_sms, s);
  return a.kv.f16 ? launch_types<HD, float, __half>(a, num_sms, s) : launch_types<HD, float, float>(a, num_sms, s);
}

}  // namespace

cudaError_t rows_append_launch(const RowAppendArgs& a, int num_sms, cudaStream_t s) {
  return a.kv.hd == 128 ? launch_hd<128>(a, num_sms, s) : launch_hd<64>(a, num_sms, s);
}

}  // namespace rb
