// Work lists of a row plan: which keys each CTA of the attention kernels reads
// for which query vectors. Host code without CUDA; the kernels trust these lists.
#include "rows.cuh"

#include <algorithm>

namespace rb {

namespace {

struct Item {
  int row0, v0, nv, tenant, k0, k1;
};

// Cuts the rows [r0, r1) (one tenant) into items of at most `vecs` query vectors
// and takes the union of their rows' keys, its start rounded down to `align`.
void cut_run(const std::vector<RowInfo>& rows, int r0, int r1, int n_rep, int vecs, int align, std::vector<Item>& out) {
  const long long total = (long long)(r1 - r0) * n_rep;
  for (long long v = 0; v < total; v += vecs) {
    const int nv = (int)std::min<long long>(vecs, total - v);
    Item it{r0 + (int)(v / n_rep), (int)(v % n_rep), nv, rows[r0].tenant, 0, 0};
    int lo = 0, hi = 0;
    bool any = false;
    for (int r = it.row0; r <= r0 + (int)((v + nv - 1) / n_rep); ++r)
      if (rows[r].hi > rows[r].lo) {
        lo = any ? std::min(lo, rows[r].lo) : rows[r].lo;
        hi = any ? std::max(hi, rows[r].hi) : rows[r].hi;
        any = true;
      }
    if (any) {
      it.k0 = lo / align * align;
      it.k1 = hi;
    }
    out.push_back(it);
  }
}

int blocks_of(const Item& it, int width) { return (it.k1 - it.k0 + width - 1) / width; }

}  // namespace

void rows_partition(const std::vector<RowInfo>& rows, int n_heads, int n_kv, int num_sms, bool use_tile, RowWork& out) {
  out = RowWork();
  const int n_rep = n_heads / n_kv, n = (int)rows.size();
  std::vector<Item> small, tile;
  for (int r = 0; r < n;) {
    int e = r + 1;
    while (e < n && rows[e].tenant == rows[r].tenant) ++e;
    if (use_tile && (long long)(e - r) * n_rep >= 64)
      cut_run(rows, r, e, n_rep, kTileVecs, kRowPage, tile);
    else
      cut_run(rows, r, e, n_rep, kSmallVecs, kRowPage, small);
    r = e;
  }

  // small items: the pages of all (item, kv head) pairs form one sequence; every
  // CTA takes an equal contiguous share of it, at least four pages (one a warp)
  long long pages = 0;
  for (const Item& it : small) pages += (long long)n_kv * blocks_of(it, kRowPage);
  const long long most = 2ll * num_sms;
  const long long G = std::max<long long>(1, std::min(most, (pages + 3) / 4));
  if (!small.empty()) {
    out.small_cta.assign(1, 0);
    long long at = 0, cta = 0;  // pages handed out so far, CTA being filled
    auto cta_end = [&](long long c) { return pages * (c + 1) / G; };
    for (const Item& it : small) {
      out.max_nv = std::max(out.max_nv, it.nv);
      for (int h = 0; h < n_kv; ++h) {
        const int np = blocks_of(it, kRowPage);
        const size_t first = out.small.size();
        int p = 0;
        do {
          while (cta + 1 < G && at >= cta_end(cta)) {
            out.small_cta.push_back((int)out.small.size());
            ++cta;
          }
          const int take = (int)std::min<long long>(np - p, cta + 1 < G ? cta_end(cta) - at : np - p);
          AttnUnit u{it.row0, it.v0, it.nv, h, it.tenant, it.k0 + p * kRowPage,
                     std::min(it.k1, it.k0 + (p + take) * kRowPage), -1, -1};
          out.small.push_back(u);
          p += take;
          at += take;
        } while (p < np);
        const int parts = (int)(out.small.size() - first);
        if (parts > 1) {
          out.joins.push_back({it.row0, it.v0, it.nv, h, out.n_slots, parts});
          for (size_t i = first; i < out.small.size(); ++i) {
            out.small[i].join = (int)out.joins.size() - 1;
            out.small[i].slot = out.n_slots;
            out.n_slots += it.nv;
          }
        }
      }
    }
    while ((long long)out.small_cta.size() <= G) out.small_cta.push_back((int)out.small.size());
  }
  out.n_small_joins = (int)out.joins.size();

  // tile items: one CTA per unit, the longest first. Their keys are cut only where
  // the items are fewer than the SMs, and not below four blocks: a unit's start and
  // end cost about as much as those. (Cutting the longest of 256 uneven items as well,
  // for the balance at the end, took 257 us and 19 us of joining instead of 237 us.)
  if (!tile.empty()) {
    long long blocks = 0;
    for (const Item& it : tile) blocks += (long long)n_kv * std::max(1, blocks_of(it, kTileKeys));
    const long long seg = std::max<long long>(4, (blocks + num_sms - 1) / num_sms);
    const bool cut = (long long)tile.size() * n_kv < num_sms;
    for (const Item& it : tile) {
      const int nb = blocks_of(it, kTileKeys);
      const int parts = cut && nb > seg ? (int)((nb + seg - 1) / seg) : 1;
      for (int h = 0; h < n_kv; ++h) {
        if (parts > 1) {
          out.joins.push_back({it.row0, it.v0, it.nv, h, out.n_slots, parts});
        }
        for (int p = 0; p < parts; ++p) {
          const int b0 = (int)((long long)nb * p / parts), b1 = (int)((long long)nb * (p + 1) / parts);
          AttnUnit u{it.row0, it.v0, it.nv, h, it.tenant, it.k0 + b0 * kTileKeys,
                     std::min(it.k1, it.k0 + b1 * kTileKeys), -1, -1};
          if (parts > 1) {
            u.slot = out.n_slots;
            out.n_slots += it.nv;
          }
          out.tile.push_back(u);
        }
      }
    }
    std::stable_sort(out.tile.begin(), out.tile.end(),
                     [](const AttnUnit& a, const AttnUnit& b) { return a.k1 - a.k0 > b.k1 - b.k0; });
    for (const AttnUnit& u : out.tile) {
      TileSpan s{{0, 0}, {0x7fffffff, 0x7fffffff}, 0, 0};
      bool any = false;
      for (int t = 0; t < 2; ++t) {
        const int v0 = u.v0 + t * (kTileVecs / 2), v1 = u.v0 + std::min(u.nv, (t + 1) * (kTileVecs / 2));
        if (v0 >= v1) continue;
        for (int r = u.row0 + v0 / n_rep; r <= u.row0 + (v1 - 1) / n_rep; ++r) {
          s.all0[t] = std::max(s.all0[t], rows[r].lo);
          s.all1[t] = std::min(s.all1[t], rows[r].hi);
          if (rows[r].hi > rows[r].lo) {
            s.in0 = any ? std::min(s.in0, rows[r].lo) : rows[r].lo;
            s.in1 = std::max(s.in1, rows[r].hi);
            any = true;
          }
        }
      }
      out.spans.push_back(s);
    }
  }
}

}  // namespace rb
