// Rows of a step around the paged cache: the plan's work lists (rows_plan.cpp),
// the append with per-head norms and rotation (rows_append.cu) and masked
// attention (rows_attn.cu, rows_tile.cu).
#pragma once
#include <stdint.h>

#include <vector>

namespace rb {

constexpr int kRowPage = 16;      // tokens per cache page
constexpr int kSmallVecs = 8;     // query vectors per item of the small kernels
constexpr int kTileVecs = 256;    // query vectors per item of the tile kernel (two tiles of 128)
constexpr int kTileKeys = 128;    // keys per block of the tile kernel
constexpr int kTileBlocks = 256;  // blocks of a unit of the tile kernel, at most
constexpr int kMaxRep = 64;       // query heads per kv head
constexpr int kRowWarps = 4;      // warps a CTA of the small kernels, two CTAs an SM

// One row as the kernels see it: the keys [lo, hi) of its tenant (hi <= lo: none).
struct RowInfo {
  int32_t pos, lo, hi, tenant;
};

// A piece of one item. An item is up to kSmallVecs (kTileVecs) query vectors of
// one kv head over consecutive rows of one tenant: vector i is head
// kvh * n_rep + (v0 + i) % n_rep of row row0 + (v0 + i) / n_rep. A unit covers the
// item's keys [k0, k1) (k0 a multiple of the page size). slot < 0: the unit is the
// whole item and writes the output; else its vectors' partial results go to
// slot .. slot + nv.
struct AttnUnit {
  int32_t row0, v0, nv, kvh, tenant, k0, k1, slot;
  int32_t all0, all1;        // keys that every row of the item sees [all0, all1)
  int32_t in0, in1;          // and that some row sees [in0, in1)
};

// An item cut into n_parts units: part p of vector i lies at slot0 + p * nv + i.
struct JoinItem {
  int32_t row0, v0, nv, kvh, slot0, n_parts;
};

// What the rows of a tile unit see: keys that every row of tile t sees [all0, all1),
// and that some row of the unit sees [in0, in1).
struct TileSpan {
  int32_t all0[2], all1[2], in0, in1;
};

// Work lists of one plan. Warp w of the small kernels runs the units
// [small_warp[w], small_warp[w + 1]), CTA b of the tile kernel unit b.
struct RowWork {
  std::vector<AttnUnit> small, tile;
  std::vector<TileSpan> spans;       // of the tile units
  std::vector<int32_t> small_warp;
  std::vector<JoinItem> joins;       // items that were cut
  int32_t join_nv = 0;               // vectors of the largest of them
  int64_t n_slots = 0;      // partial result vectors (a plan is refused where they pass 32 bits)
  int32_t max_nv = 0;       // vectors of the largest small item
};

// rows: the plan's rows in call order; use_tile: whether long runs go to the tile
// kernel (fp16 caches). Pure host code.
void rows_partition(const std::vector<RowInfo>& rows, int n_heads, int n_kv, int num_sms, bool use_tile, RowWork& out);

}  // namespace rb

#ifdef __CUDACC__
#include "attention.cuh"

namespace rb {

struct RowAttnArgs {
  CUtensorMap tmap;  // fp16 caches (kv_tensor_map)
  const void* q = nullptr;
  void* out = nullptr;
  int64_t ldq = 0, ldo = 0;  // elements between rows
  int32_t q16 = 0;           // 1: q and out are fp16, 0: fp32
  int32_t layer = 0, n_heads = 0, n_rep = 1;
  float scale = 1.f, cap = 0.f;
  const float* slopes = nullptr;  // [n_heads] or null
  KvView kv;
  const RowInfo* rows = nullptr;
  const AttnUnit* units = nullptr;
  const int32_t* warps = nullptr;  // small kernels: [n_warps + 1]
  int32_t n_warps = 0, n_units = 0, max_nv = 0;  // max_nv: vectors of the largest small item
  const TileSpan* spans = nullptr;  // tile kernel
  const JoinItem* joins = nullptr;
  int32_t n_joins = 0, join_nv = 0;  // join_nv: vectors of the largest cut item
  float* part_o = nullptr;   // [n_slots][hd]
  float2* part_ml = nullptr; // [n_slots] (maximum in base-2 units, sum)
  // tile kernel: places for kTileVecs vectors of up to 128 elements ([elements in fours][128 vectors] of
  // each of their tiles), one for each CTA that runs at a time, and which are taken
  float* hold = nullptr;
  int32_t* hold_busy = nullptr;
  int32_t n_hold = 0;
  uint32_t* err = nullptr;
};

struct RowAppendArgs {
  const void *q = nullptr, *k = nullptr, *v = nullptr;  // q may be null
  void* q_out = nullptr;
  int64_t ldq = 0, ldk = 0, ldv = 0, ldo = 0;
  int32_t in16 = 0;
  int32_t n_rows = 0, n_heads = 0, layer = 0;
  const float *q_norm = nullptr, *k_norm = nullptr;
  float eps = 0.f;
  const float* rope = nullptr;  // [rope_len][rotary]: cosines, then sines
  int32_t rotary = 0, adjacent = 0;
  const RowInfo* rows = nullptr;
  KvView kv;
};

cudaError_t rows_append_launch(const RowAppendArgs& a, int num_sms, cudaStream_t s);
// the small kernel over a.units / a.warps
cudaError_t rows_small_launch(const RowAttnArgs& a, cudaStream_t s);
// the tile kernel over a.units (one CTA each)
cudaError_t rows_tile_launch(const RowAttnArgs& a, cudaStream_t s);
// joins the items that were cut, after both
cudaError_t rows_join_launch(const RowAttnArgs& a, cudaStream_t s);

}  // namespace rb
#endif
