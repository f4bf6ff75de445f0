// Rows of a step into the paged cache: per-head norms of queries and keys, the
// position rotation and the append in one pass over q, k and v.
//
//   norm:     y_i = x_i w_i / sqrt(mean_j x_j^2 + eps)        (each head by itself)
//   rotation: (y_a, y_b) <- (y_a c - y_b s, y_b c + y_a s)    (pairs a, b of the first
//             `rotary` elements; c, s of the row's position from the table)
//
// in fp32, rounded once into q_out and the cache. Bound by memory: every element
// is read once and written once.
#include <type_traits>

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

// The same with wide accesses. A lane has two chunks of four elements, the two that the
// rotation pairs with one another where it does (so nothing is exchanged for it), and a
// head takes HD / 8 lanes; a warp takes 32 / (HD / 8) heads at a time and U such groups
// in flight. Needs chunks and tables aligned to their size.
// 8188 rows of 32 + 8 + 8 heads of 128 (fp16, 205 MB): 40 us, 5.1 TB/s; with 8 elements in
// a row a lane and the partners' fetched by shuffles 56 us, with 2-byte accesses 97 us.
template <class T>
__device__ __forceinline__ void load4(const T* p, float* x) {
  if constexpr (sizeof(T) == 2) {
    const uint2 r = *reinterpret_cast<const uint2*>(p);
    const float2 a = __half22float2(u32_as_h2(r.x)), b = __half22float2(u32_as_h2(r.y));
    x[0] = a.x;
    x[1] = a.y;
    x[2] = b.x;
    x[3] = b.y;
  } else {
    *reinterpret_cast<float4*>(x) = *reinterpret_cast<const float4*>(p);
  }
}
template <class T>
__device__ __forceinline__ void store4(T* p, const float* x) {
  if constexpr (sizeof(T) == 2)
    *reinterpret_cast<uint2*>(p) =
        make_uint2(h2_as_u32(__floats2half2_rn(x[0], x[1])), h2_as_u32(__floats2half2_rn(x[2], x[3])));
  else
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
}

template <class TD, int U, int HPW>
__device__ __forceinline__ void store_heads(TD* dst, int stride, int h0, int n, int d0, int d1, float (&x)[U][8]) {
#pragma unroll
  for (int i = 0; i < U; ++i)
    if (h0 + i * HPW < n) {
      store4(dst + i * HPW * stride + d0, x[i]);
      store4(dst + i * HPW * stride + d1, x[i] + 4);
    }
}

// A warp's heads are all of q, of k or of v (gq, gk groups, and then v's).
template <int HD, class TI, class TC, int U>
__global__ void __launch_bounds__(256) rows_append_vec_kernel(const __grid_constant__ RowAppendArgs a, int groups, int gq,
                                                              int gk) {
  constexpr int LPH = HD / 8, HPW = 32 / LPH;
  const int lane = threadIdx.x & 31, l = lane % LPH;
  const unsigned w = (blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  const int row = (int)(w / (unsigned)groups), g = (int)(w % (unsigned)groups);
  if (row >= a.n_rows) return;
  const int kind = g < gq ? 0 : g < gq + gk ? 1 : 2;
  const int n = kind == 0 ? a.n_heads : a.kv.n_kv;
  const int h0 = (kind == 0 ? g : kind == 1 ? g - gq : g - gq - gk) * (HPW * U) + lane / LPH;
  // the first `pairs` lanes have the rotated chunks l and l + pairs, the others what follows
  const int pairs = a.rotary / 8;
  const bool turned = l < pairs;
  const int d0 = turned ? 4 * l : 8 * l, d1 = turned ? 4 * (l + pairs) : 8 * l + 4;
  const RowInfo r = a.rows[row];
  float x[U][8];
  {
    const TI* src = reinterpret_cast<const TI*>(kind == 0 ? a.q : kind == 1 ? a.k : a.v) +
                    (size_t)row * (kind == 0 ? a.ldq : kind == 1 ? a.ldk : a.ldv) + h0 * HD;
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (h0 + i * HPW < n) {
        load4(src + i * HPW * HD + d0, x[i]);
        load4(src + i * HPW * HD + d1, x[i] + 4);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[i][e] = 0.f;
      }
  }
  const float* norm = kind == 0 ? a.q_norm : kind == 1 ? a.k_norm : nullptr;
  const int page = kind ? a.kv.ptab[(size_t)r.tenant * a.kv.ptab_stride + (r.pos >> 4)] : 0;
  if (kind < 2) {
    float cs[4], sn[4];
    if (turned) {
      const float* t = a.rope + (size_t)r.pos * a.rotary;
      if (a.adjacent) {  // chunk c has pairs 2 c and 2 c + 1: those of chunk l, then of chunk l + pairs
        *reinterpret_cast<float2*>(cs) = *reinterpret_cast<const float2*>(t + d0 / 2);
        *reinterpret_cast<float2*>(cs + 2) = *reinterpret_cast<const float2*>(t + d1 / 2);
        *reinterpret_cast<float2*>(sn) = *reinterpret_cast<const float2*>(t + a.rotary / 2 + d0 / 2);
        *reinterpret_cast<float2*>(sn + 2) = *reinterpret_cast<const float2*>(t + a.rotary / 2 + d1 / 2);
      } else {
        *reinterpret_cast<float4*>(cs) = *reinterpret_cast<const float4*>(t + d0);
        *reinterpret_cast<float4*>(sn) = *reinterpret_cast<const float4*>(t + a.rotary / 2 + d0);
      }
    }
    if (norm) {
      const float4 w0 = *reinterpret_cast<const float4*>(norm + d0), w1 = *reinterpret_cast<const float4*>(norm + d1);
      const float wn[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
      for (int i = 0; i < U; ++i) {
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(x[i][e], x[i][e], ss);
#pragma unroll
        for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float inv = rsqrtf(ss * (1.f / HD) + a.eps);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[i][e] *= inv * wn[e];
      }
    }
    if (turned) {
      if (a.adjacent) {
#pragma unroll
        for (int i = 0; i < U; ++i)
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            const float u = x[i][e] * cs[e / 2] - x[i][e + 1] * sn[e / 2], v = x[i][e + 1] * cs[e / 2] + x[i][e] * sn[e / 2];
            x[i][e] = u;
            x[i][e + 1] = v;
          }
      } else {
#pragma unroll
        for (int i = 0; i < U; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float u = x[i][e] * cs[e] - x[i][e + 4] * sn[e], v = x[i][e + 4] * cs[e] + x[i][e] * sn[e];
            x[i][e] = u;
            x[i][e + 4] = v;
          }
      }
    }
  }
  if (kind == 0) {
    store_heads<TI, U, HPW>(reinterpret_cast<TI*>(a.q_out) + (size_t)row * a.ldo + h0 * HD, HD, h0, n, d0, d1, x);
  } else {
    const size_t at = ((((size_t)page * a.kv.n_layers + a.layer) * 2 + (kind - 1)) * n + h0) * 16 + (r.pos & 15);
    store_heads<TC, U, HPW>(reinterpret_cast<TC*>(a.kv.pool) + at * HD, 16 * HD, h0, n, d0, d1, x);
  }
}

template <int HD, class TI, class TC>
cudaError_t launch_types(const RowAppendArgs& a, int num_sms, cudaStream_t s) {
  constexpr int HPW = 32 / (HD / 8), CHUNK = 4 * sizeof(TI);
  const long long per = (a.q ? a.n_heads : 0) + 2 * a.kv.n_kv;
  auto bad = [&](const void* p, int64_t ld) {
    return p && ((reinterpret_cast<uintptr_t>(p) | (size_t)ld * sizeof(TI)) & (CHUNK - 1));
  };
  const uintptr_t tables = reinterpret_cast<uintptr_t>(a.rope) | reinterpret_cast<uintptr_t>(a.q_norm) |
                           reinterpret_cast<uintptr_t>(a.k_norm);
  // without the alignment: 2048 rows take 31.7 us against 19.2
  if ((tables & 15) || bad(a.q, a.ldq) || bad(a.k, a.ldk) || bad(a.v, a.ldv) || bad(a.q_out, a.ldo)) {
    const long long warps = a.n_rows * per;
    rows_append_kernel<HD, TI, TC><<<(unsigned)((warps + 7) / 8), 256, 0, s>>>(a);
    return cudaGetLastError();
  }
  auto run = [&](auto u) {
    constexpr int U = decltype(u)::value, S = HPW * U;
    const int gq = a.q ? (a.n_heads + S - 1) / S : 0, gk = (a.kv.n_kv + S - 1) / S, groups = gq + 2 * gk;
    rows_append_vec_kernel<HD, TI, TC, U>
        <<<(unsigned)(((long long)a.n_rows * groups + 7) / 8), 256, 0, s>>>(a, groups, gq, gk);
  };
  // One group of heads a warp while that leaves no SM with more than 32 warps, else four. Rows of
  // 32 + 8 + 8 heads of 128, one against four, us: 128 rows 7.3/8.3, 192 rows 8.4/9.0, 256 rows
  // 10.0/9.0, 1024 rows 15.4/12.3, 2048 rows 22.8/19.2; two were slower than four at 8188 rows.
  if (a.n_rows * ((per + HPW - 1) / HPW) <= 32ll * num_sms) run(std::integral_constant<int, 1>());
  else run(std::integral_constant<int, 4>());
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
