// Low-rank adapters of many tenants beside one projection (adapters.cu, adapters_tile.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace rb {

constexpr int kAdapterMaxRank = 128;
constexpr int kAdapterMaxSlots = 4096;
constexpr int kAdapterMaxDim = 1 << 20;  // of k and n

struct __align__(16) AdapterMeta {  // one load
  int32_t rank;  // 0: the slot is empty
  float scale;
  float f1, f2;  // down and up are held behind powers of two: their products are f1 f2 of what is held, two powers of one side of 1
};

// Adapters of one projection [n][k], in slots of equal size:
//   down  [n_slots][kp / 8][r16][8] fp16 (as much of rp * kp as the rank needs)
//   up    [n_slots][rp / 8][n][8] fp16
// with zeros past the rank and past k. Factors given in fp32 are multiplied by a power of two that
// brings their largest element to [2^14, 2^15), so that none is infinite and small ones keep their 11 bits
// (AdapterMeta); those given in fp16 lie as they are. r16, rp: the rank and max_rank rounded up to a multiple of 16;
// kp: k to one of 64. Blocks of 8 rows x 16 bytes, as tensor-core operands lie, so that
// they are copied as they are; eight elements a load for a thread.
struct AdapterView {
  const uint16_t *down = nullptr, *up = nullptr;
  const AdapterMeta* meta = nullptr;
  int32_t n = 0, k = 0, kp = 0, rp = 0, n_slots = 0;
};

struct AdapterArgs {
  AdapterView w;
  const void *x = nullptr, *y = nullptr;
  void* out = nullptr;
  int64_t ldx = 0, ldy = 0, ldo = 0;
  int32_t x16 = 0;  // x, y and out are fp16, else fp32
  int32_t n_rows = 0;
  const int32_t* slots = nullptr;
  uint32_t* err = nullptr;
  int32_t max_cluster = 8;  // adapters_max_cluster()
};

struct AdapterSetArgs {
  uint16_t *down = nullptr, *up = nullptr;  // of the slot
  AdapterMeta* meta = nullptr;              // of the slot
  uint32_t* most = nullptr;                 // of the slot, fp32 factors: the largest element of down, of up
  int32_t n = 0, k = 0, kp = 0, rp = 0, rank = 0, in16 = 0;
  float scale = 0.f;
  const void *src_down = nullptr, *src_up = nullptr;  // [rank][k], [n][rank]
};

// CTAs that a cluster may have on the current device: 16, or 8 where so many do not fit. Not while a stream is captured.
int adapters_max_cluster();
cudaError_t adapters_set_launch(const AdapterSetArgs& a, cudaStream_t s);
cudaError_t adapters_clear_launch(AdapterMeta* meta, cudaStream_t s);
cudaError_t adapters_launch(const AdapterArgs& a, int num_sms, cudaStream_t s);
// many rows: tiles on the tensor cores
cudaError_t adapters_tile_launch(const AdapterArgs& a, int num_sms, cudaStream_t s);

}  // namespace rb
