// Low-rank adapters beside a shared projection: out_r = y_r + scale_a up_a (down_a x_r) for
// the row's adapter a. Here single tokens of many tenants; tiles of many rows are in
// adapters_tile.cu.
//
// A cluster of CTAs has up to R rows that share an adapter. Its CTAs split k for
// v = down x and then n for up v; in between each sends its part of v to all of them
// (distributed shared memory), which add the parts in CTA order. So there is one launch, nothing
// is kept in memory between the two products, and no result depends on an order of atomics.
// fp32 throughout, the weights' fp16 values are exact in it.
//
// The rows of an adapter find one another in the kernel: cluster i of a block of kBlock
// rows takes the block's i-th item, an item being the next R rows of one slot, counted from the
// block's first row; clusters past the last item have nothing to do. A lone row takes a quarter of the work of four.
//
// Bound by latency: the slots, an adapter's rank, x and down, the exchange, up, one after the other; up and
// y are on their way to L2 from the start. Nothing in L2, about 3 us of launch within: one row of rank 16 (k = n =
// 4096, 0.3 MB) 9.5 us, rank 64 11.5, rank 128 16; 64 rows of 64 adapters of rank 64 (67 MB) 29 us, 2.3 TB/s; 48
// rows of 31 adapters of rank 8 to 64, n = 11008 (32 MB), 25.8 us. With up read four blocks of two columns at a time
// instead of one by one 64 rows went from 35 to 29 us.
#include <cooperative_groups.h>

#include <algorithm>

#include "adapters.cuh"
#include "common.cuh"

namespace cg = cooperative_groups;

namespace rb {

namespace {

constexpr int kT = 256, kWarps = kT / 32;
constexpr int kBlock = 64;        // rows among which an item's rows are found
constexpr int kGroup = 8;         // ranks a warp works on at a time: a line of weights
constexpr int kTileK = 1536;      // elements of x in shared memory at a time
constexpr int kMaxCluster = 16;  // where the GPU has it (adapters_max_cluster)
static_assert(kWarps * kGroup <= kAdapterMaxRank && kTileK % 8 == 0, "");

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <class T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

__device__ __forceinline__ void unpack8(uint4 q, float (&f)[8]) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = __half22float2(u32_as_h2(w[i]));
    f[2 * i] = v.x;
    f[2 * i + 1] = v.y;
  }
}

// The slot of a row, or -1 where it has no adapter.
__device__ __forceinline__ int slot_of(const AdapterArgs& a, int row) {
  const int s = a.slots[row];
  return s >= 0 && s < a.w.n_slots && a.w.meta[s].rank > 0 ? s : -1;
}

template <int R>
struct ItemShared {
  __align__(16) float xs[R][kTileK];
  float part[kAdapterMaxRank * R];             // [k part][rank][row]
  __align__(16) float v[kAdapterMaxRank * R];  // [rank][row]
};

// Up to R rows of one slot, by a cluster.
template <class T, int R, int RS>
__device__ __forceinline__ void run_item(const AdapterArgs& a, ItemShared<RS>& sh, float* parts, int slot, const int (&rows)[R], int nr) {
  auto& xs = sh.xs;
  float *part = sh.part, *v = sh.v;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), c = (int)cluster.block_rank();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const T* x = reinterpret_cast<const T*>(a.x);
  const T* y = reinterpret_cast<const T*>(a.y);
  T* out = reinterpret_cast<T*>(a.out);
  // this CTA's columns of out
  const int n0 = (int)((int64_t)a.w.n * c / C), n1 = (int)((int64_t)a.w.n * (c + 1) / C);
  cluster.barrier_arrive();
  const AdapterMeta meta = a.w.meta[slot];
  const int rank = meta.rank;
  const int groups = (rank + kGroup - 1) / kGroup, r16 = (rank + 15) / 16 * 16;
  // warps are split over groups of ranks, and with few of those over k
  const int ks = groups >= kWarps ? 1 : kWarps / groups, kpart = ks == 1 ? 0 : warp / groups;
  const int chunks = a.w.kp / 8, c0 = (int)((int64_t)chunks * c / C), c1 = (int)((int64_t)chunks * (c + 1) / C);
  const uint16_t* down = a.w.down + (int64_t)slot * a.w.rp * a.w.kp;
  const uint16_t* up = a.w.up + (int64_t)slot * a.w.rp * a.w.n;
  // what comes after v on its way to L2: a line of 128 bytes a thread
  for (int i = tid, per = (n1 - n0 + 7) / 8; i < per * ((rank + 7) / 8); i += kT)
    asm volatile("prefetch.global.L2 [%0];" ::"l"(up + ((int64_t)(i / per) * a.w.n + n0 + i % per * 8) * 8));
#pragma unroll
  for (int r = 0; r < R; ++r)
    for (int j = n0 + tid * 32; r < nr && j < n1; j += kT * 32)
      asm volatile("prefetch.global.L2 [%0];" ::"l"(y + rows[r] * a.ldy + j));
  const int stride = a.w.rp * R;       // between the CTAs' parts
  const int nv = groups * kGroup * R;  // of a k part; ks > 1: at most kWarps groups in all
  for (int i = tid; i < ks * nv; i += kT) part[i] = 0.f;
  for (int t0 = c0; t0 < c1; t0 += kTileK / 8) {
    const int t1 = min(c1, t0 + kTileK / 8), len = (t1 - t0) * 8, k0 = t0 * 8;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r)
      for (int j = tid; j < len; j += kT) xs[r][j] = r < nr && k0 + j < a.w.k ? to_f(x[rows[r] * a.ldx + k0 + j]) : 0.f;
    __syncthreads();
    if (kpart < ks) {
      const int b0 = (t1 - t0) * kpart / ks, b1 = (t1 - t0) * (kpart + 1) / ks;
      for (int g = ks == 1 ? warp : warp % groups; g < groups; g += ks == 1 ? kWarps : groups) {
        float acc[R];
#pragma unroll
        for (int r = 0; r < R; ++r) acc[r] = 0.f;
        // a lane has rank g * 8 + lane % 8 of every fourth block of 8 elements
        const uint4* w = reinterpret_cast<const uint4*>(down) + (int64_t)t0 * r16 + g * kGroup + (lane & 7);
#pragma unroll 4
        for (int b = b0 + (lane >> 3); b < b1; b += 4) {
          float f[8];
          unpack8(__ldg(w + (int64_t)b * r16), f);
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const float4 lo = *reinterpret_cast<const float4*>(&xs[r][b * 8]),
                         hi = *reinterpret_cast<const float4*>(&xs[r][b * 8 + 4]);
            const float xv[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[r] = fmaf(f[e], xv[e], acc[r]);
          }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
          acc[r] += __shfl_xor_sync(0xffffffffu, acc[r], 8);
          acc[r] += __shfl_xor_sync(0xffffffffu, acc[r], 16);
          if (lane < 8) part[kpart * nv + (g * kGroup + lane) * R + r] += acc[r];
        }
      }
    }
  }
  __syncthreads();
  cluster.barrier_wait();  // every CTA of the cluster runs before its shared memory is written
  for (int i = tid; i < nv; i += kT) {
    float s = 0.f;
    for (int p = 0; p < ks; ++p) s += part[p * nv + i];
    for (int d = 0; d < C; ++d) *cluster.map_shared_rank(parts + c * stride + i, d) = s;
  }
  cluster.sync();
  for (int i = tid; i < (rank + 7) / 8 * 8 * R; i += kT) {
    float s = 0.f;
    if (i < nv)
      for (int d = 0; d < C; ++d) s += parts[d * stride + i];
    v[i] = s * meta.scale * meta.f1 * meta.f2;
  }
  __syncthreads();
  const int blocks8 = (rank + 7) / 8;
  for (int j0 = n0 + tid; j0 < n1; j0 += 2 * kT) {  // two columns at a time, up to four blocks of each on their way
    float acc[2][R];
#pragma unroll
    for (int c2 = 0; c2 < 2; ++c2)
#pragma unroll
      for (int r = 0; r < R; ++r)
        acc[c2][r] = 0.f;
#pragma unroll 1
    for (int h0 = 0; h0 < blocks8; h0 += 4) {
      uint4 q[2][4];
#pragma unroll
      for (int h = 0; h < 4; ++h)
#pragma unroll
        for (int c2 = 0; c2 < 2; ++c2) {
          q[c2][h] = make_uint4(0, 0, 0, 0);
          if (h0 + h < blocks8 && j0 + c2 * kT < n1)
            q[c2][h] = __ldg(reinterpret_cast<const uint4*>(up + ((int64_t)(h0 + h) * a.w.n + j0 + c2 * kT) * 8));
        }
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        if (h0 + h >= blocks8) continue;
#pragma unroll
        for (int c2 = 0; c2 < 2; ++c2) {
          float f[8];
          unpack8(q[c2][h], f);
#pragma unroll
          for (int e = 0; e < 8; ++e)
#pragma unroll
            for (int r = 0; r < R; ++r) acc[c2][r] = fmaf(f[e], v[((h0 + h) * 8 + e) * R + r], acc[c2][r]);
        }
      }
    }
    // y last: no product is rounded at y's size (and read here, it takes no registers before: 48 rows 25.7 us, else 27)
    float yv[2][R];
#pragma unroll
    for (int c2 = 0; c2 < 2; ++c2)
#pragma unroll
      for (int r = 0; r < R; ++r) yv[c2][r] = r < nr && j0 + c2 * kT < n1 ? to_f(y[rows[r] * a.ldy + j0 + c2 * kT]) : 0.f;
#pragma unroll
    for (int c2 = 0; c2 < 2; ++c2)
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (r < nr && j0 + c2 * kT < n1) out[rows[r] * a.ldo + j0 + c2 * kT] = from_f<T>(yv[c2][r] + acc[c2][r]);
  }
}

template <class T, int R>
__global__ void __launch_bounds__(kT, 4) adapters_kernel(const __grid_constant__ AdapterArgs a) {
  __shared__ ItemShared<R> sh;
  extern __shared__ float parts[];  // [CTA of the cluster][rank][row] of v
  __shared__ int s_slot[kBlock], s_rows[R], s_n;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), c = (int)cluster.block_rank();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_launch_dependents();
  pdl_wait();
  const int id = blockIdx.x / C;
  int slot, rows[R], nr = 1;
  if (R == 1) {
    rows[0] = id;
    slot = slot_of(a, id);
  } else {
    const int b0 = id / kBlock * kBlock, nb = min(kBlock, a.n_rows - b0);
    if (tid < nb) s_slot[tid] = slot_of(a, b0 + tid);
    if (tid == 0) s_n = 0;
    __syncthreads();
    if (warp == 0) {
      // rows b0 + lane and b0 + 32 + lane: which of its slot's rows is it; a row without an adapter is one by itself
      int lead[2], nth[2];
      unsigned before = 0;
      int first = -1;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = h * 32 + lane, s = r < nb ? s_slot[r] : -2;
        const unsigned same = __match_any_sync(0xffffffffu, s);
        int rank = __popc(same & ((1u << lane) - 1));
        if (h == 1)
          for (int j = 0; j < 32; ++j) rank += s_slot[j] == s;
        nth[h] = rank;
        lead[h] = r < nb && (s < 0 || rank % R == 0);
        const unsigned leads = __ballot_sync(0xffffffffu, lead[h]);
        const int item = (int)before + __popc(leads & ((1u << lane) - 1));
        if (lead[h] && item == id - b0) first = r;
        before += __popc(leads);
      }
      const unsigned who = __ballot_sync(0xffffffffu, first >= 0);
      if (who) {
        const int src = __ffs(who) - 1;
        first = __shfl_sync(0xffffffffu, first, src);
        const int s = s_slot[first], n0 = __shfl_sync(0xffffffffu, first < 32 ? nth[0] : nth[1], src);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = h * 32 + lane;
          const bool in = r < nb && (s < 0 ? r == first : s_slot[r] == s && nth[h] >= n0 && nth[h] < n0 + R);
          if (in) {
            s_rows[s < 0 ? 0 : nth[h] - n0] = b0 + r;
            atomicAdd(&s_n, 1);
          }
        }
      }
    }
    __syncthreads();
    nr = s_n;
    if (nr == 0) return;  // the whole cluster: no item is left for it
    slot = s_slot[s_rows[0] - b0];
#pragma unroll
    for (int r = 0; r < R; ++r) rows[r] = s_rows[min(r, nr - 1)];
  }
  if (slot < 0) {
    if (a.out != a.y)
      for (int j = (int)((int64_t)a.w.n * c / C) + tid; j < (int)((int64_t)a.w.n * (c + 1) / C); j += kT) reinterpret_cast<T*>(a.out)[rows[0] * a.ldo + j] = reinterpret_cast<const T*>(a.y)[rows[0] * a.ldy + j];
    return;  // the whole cluster
  }
  if (R > 1 && nr == 1) {
    const int one[1] = {rows[0]};
    run_item<T, 1, R>(a, sh, parts, slot, one, 1);
  } else {
    run_item<T, R, R>(a, sh, parts, slot, rows, nr);
  }
}

template <class T, int R>
cudaError_t launch(const AdapterArgs& a, int cluster, cudaStream_t s) {
  const int smem = cluster * a.w.rp * R * 4;
  int dev = 0;
  cudaGetDevice(&dev);
  if (cudaError_t e = ensure_smem_attr(adapters_kernel<T, R>, kMaxCluster * kAdapterMaxRank * R * 4, dev)) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)a.n_rows * cluster);
  cfg.blockDim = dim3(kT);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)cluster;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, adapters_kernel<T, R>, a);
}

// The largest finite elements of fp32 factors, as bits (which order like the values), into a.most[0] and [1].
__global__ void adapters_most_kernel(const __grid_constant__ AdapterSetArgs a) {
  const int64_t at = (int64_t)blockIdx.x * blockDim.x + threadIdx.x, step = (int64_t)gridDim.x * blockDim.x;
#pragma unroll
  for (int f = 0; f < 2; ++f) {
    const uint32_t* p = reinterpret_cast<const uint32_t*>(f ? a.src_up : a.src_down);
    uint32_t most = 0;
    for (int64_t i = at; i < (int64_t)a.rank * (f ? a.n : a.k); i += step) {
      const uint32_t x = p[i] & 0x7fffffffu;
      if (x < 0x7f800000u) most = max(most, x);
    }
    most = __reduce_max_sync(0xffffffffu, most);
    if ((threadIdx.x & 31) == 0) atomicMax(a.most + f, most);
  }
}

// The power of two that brings a factor's largest element to [2^14, 2^15): 2^126 at most, behind which the
// smallest numbers of fp32 are still multiples of fp16's.
__device__ __forceinline__ int lift_of(uint32_t most) {
  return most ? min(14 - ilogbf(__uint_as_float(most)), 126) : 0;
}

template <class S>
__global__ void adapters_set_kernel(const __grid_constant__ AdapterSetArgs a) {
  const S *sd = reinterpret_cast<const S*>(a.src_down), *su = reinterpret_cast<const S*>(a.src_up);
  const int r16 = (a.rank + 15) / 16 * 16;
  const int lift_d = a.most ? lift_of(a.most[0]) : 0, lift_u = a.most ? lift_of(a.most[1]) : 0;
  const int64_t nd = (int64_t)r16 * a.kp, nu = (int64_t)r16 * a.n;
  const int64_t at = (int64_t)blockIdx.x * blockDim.x + threadIdx.x, step = (int64_t)gridDim.x * blockDim.x;
  for (int64_t i = at; i < nd; i += step) {
    const int64_t v = i / 8;  // [k / 8][r16][8]
    const int r = (int)(v % r16), j = (int)(v / r16) * 8 + (int)(i % 8);
    a.down[i] = r < a.rank && j < a.k ? __half_as_ushort(from_f<__half>(scalbnf(to_f(sd[(int64_t)r * a.k + j]), lift_d))) : 0;
  }
  for (int64_t i = at; i < nu; i += step) {  // [rank / 8][n][8]
    const int64_t v = i / 8;
    const int r = (int)(v / a.n) * 8 + (int)(i % 8), j = (int)(v % a.n);
    a.up[i] = r < a.rank ? __half_as_ushort(from_f<__half>(scalbnf(to_f(su[(int64_t)j * a.rank + r]), lift_u))) : 0;
  }
  if (at == 0) {
    const int e = -lift_d - lift_u;  // in -252 .. 226
    *a.meta = AdapterMeta{a.rank, a.scale, scalbnf(1.f, e / 2), scalbnf(1.f, e - e / 2)};
  }
}

__global__ void adapters_clear_kernel(AdapterMeta* meta) { *meta = AdapterMeta{0, 0.f, 1.f, 1.f}; }

}  // namespace

cudaError_t adapters_set_launch(const AdapterSetArgs& a, cudaStream_t s) {
  const int64_t most = (int64_t)(a.rank + 15) / 16 * 16 * std::max(a.kp, a.n);
  const int blocks = (int)std::min<int64_t>(1184, (most + 255) / 256);
  if (a.most) {
    if (cudaError_t e = cudaMemsetAsync(a.most, 0, 8, s)) return e;
    adapters_most_kernel<<<blocks, 256, 0, s>>>(a);
  }
  if (a.in16) adapters_set_kernel<__half><<<blocks, 256, 0, s>>>(a);
  else adapters_set_kernel<float><<<blocks, 256, 0, s>>>(a);
  return cudaGetLastError();
}

int adapters_max_cluster() {
  // more than eight CTAs are not portable: asked for by the kernels that may have them, and had where so many SMs lie
  // together, which a part of a GPU may not have
  auto fits = [](auto kernel) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) return false;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(kMaxCluster);
    cfg.blockDim = dim3(kT);
    cfg.dynamicSmemBytes = kMaxCluster * kAdapterMaxRank * 4;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = kMaxCluster;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    int n = 0;
    return cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) == cudaSuccess && n > 0;
  };
  const bool all = fits(adapters_kernel<float, 1>) && fits(adapters_kernel<__half, 1>);
  cudaGetLastError();
  return all ? kMaxCluster : 8;
}

cudaError_t adapters_clear_launch(AdapterMeta* meta, cudaStream_t s) {
  adapters_clear_kernel<<<1, 1, 0, s>>>(meta);
  return cudaGetLastError();
}

cudaError_t adapters_launch(const AdapterArgs& a, int num_sms, cudaStream_t s) {
  // One launch for rows of any slots, whose number is not known here. Rows of one adapter, k = n = 4096, fp32, rank 64: 256
  // rows 33 us here and 51 in tiles, 384 47 and 53, 512 54 and 55, 1024 100 and 57; every row another's: 256 rows 82 and
  // 612, 1024 258 and 593. So up to 384 rows here, and up to 1024 where there are slots for rows mostly apart. It is the
  // set's slots that count, not those that its rows have, which are not known here: 1024 rows of one adapter take 52 us
  // with a set of 8 slots and 98 with one of 256.
  if (a.n_rows > 1024 || (a.n_rows > 384 && a.n_rows > 4 * a.w.n_slots)) return adapters_tile_launch(a, num_sms, s);
  // Sixteen CTAs a row where there are few: one row 11.5 us and 15.6 with eight (rank 64, k = n = 4096), 17.6 and 28 at k =
  // 11008; 64 rows of 64 adapters 39 and 29. (Nothing in L2, as above; the times include about 3 us of launch.)
  const int cluster = a.n_rows <= 16 ? a.max_cluster : 8;
  if (a.n_rows <= 16) return a.x16 ? launch<__half, 1>(a, cluster, s) : launch<float, 1>(a, cluster, s);
  return a.x16 ? launch<__half, 4>(a, cluster, s) : launch<float, 4>(a, cluster, s);
}

}  // namespace rb
