// Work lists of a row plan: which keys each CTA of the attention kernels reads
// for which query vectors. Host code without CUDA; the kernels trust these lists.
#include "rows.cuh"

#include <algorithm>

namespace rb {

namespace {

struct Item {
  int row0, v0, nv, tenant, k0, k1, all0, all1, in0, in1;
};

// Cuts the rows [r0, r1) (one tenant) into items of at most `vecs` query vectors
// and takes the union of their rows' keys, its start rounded down to `align`.
void cut_run(const std::vector<RowInfo>& rows, int r0, int r1, int n_rep, int vecs, int align, std::vector<Item>& out) {
  const long long total = (long long)(r1 - r0) * n_rep;
  for (long long v = 0; v < total; v += vecs) {
    const int nv = (int)std::min<long long>(vecs, total - v);
    Item it{r0 + (int)(v / n_rep), (int)(v % n_rep), nv, rows[r0].tenant, 0, 0, 0, 0x7fffffff, 0, 0};
    bool any = false;
    for (int r = it.row0; r <= r0 + (int)((v + nv - 1) / n_rep); ++r) {
      it.all0 = std::max(it.all0, rows[r].lo);
      it.all1 = std::min(it.all1, rows[r].hi);
      if (rows[r].hi <= rows[r].lo) continue;
      it.in0 = any ? std::min(it.in0, rows[r].lo) : rows[r].lo;
      it.in1 = std::max(it.in1, rows[r].hi);
      any = true;
    }
    if (any) {
      it.k0 = it.in0 / align * align;
      it.k1 = it.in1;
    }
    out.push_back(it);
  }
}

int blocks_of(const Item& it, int width) { return (it.k1 - it.k0 + width - 1) / width; }

// The unit of blocks [b0, b1) of an item, of `width` keys each.
AttnUnit unit_of(const Item& it, int kvh, int b0, int b1, int width) {
  return {it.row0, it.v0, it.nv, kvh, it.tenant, it.k0 + b0 * width, std::min(it.k1, it.k0 + b1 * width), -1,
          it.all0, it.all1, it.in0, it.in1};
}

}  // namespace

void rows_partition(const std::vector<RowInfo>& rows, int n_heads, int n_kv, int num_sms, bool use_tile, RowWork& out) {
  out = RowWork();
  const int n_rep = n_heads / n_kv, n = (int)rows.size();
  std::vector<Item> small, tile;
  // Runs of at least 24 query vectors a kv head take the tile kernel. Tiles against small
  // items, us, for runs of 16, 24, 32 and 64 vectors, 64 tenants x 1024 tokens, 8 kv heads:
  // fp16 rows at head size 128 92/103, 92/161, 94/196, 94/335; at 64 72/71, 74/99, 74/122,
  // 74/220; fp32 rows at 128 162/101, 164/167, 164/206, 166/339; at 64 106/73, 107/101,
  // 109/126, 109/226. (16 tenants x 2048, fp32 rows at 128: 89/67, 91/71, 93/93, 97/159.)
  for (int r = 0; r < n;) {
    int e = r + 1;
    while (e < n && rows[e].tenant == rows[r].tenant) ++e;
    if (use_tile && (long long)(e - r) * n_rep >= 24)
      cut_run(rows, r, e, n_rep, kTileVecs, kRowPage, tile);
    else
      cut_run(rows, r, e, n_rep, kSmallVecs, kRowPage, small);
    r = e;
  }

  // Small items: every warp works for itself. The warps go in groups of n_kv, one for
  // each kv head, and every group takes an equal contiguous share of all items' pages:
  // the heads of a page lie next to one another in memory and are read at the same
  // time. With few pages a group, a share does not cross into another item, since
  // starting on a second one takes a warp as long as several pages.
  if (!small.empty()) {
    long long pages = 0, longest = 0;
    for (const Item& it : small) {
      pages += blocks_of(it, kRowPage);
      longest = std::max<long long>(longest, blocks_of(it, kRowPage));
      out.max_nv = std::max(out.max_nv, it.nv);
    }
    const long long most = std::max(1ll, 2ll * kRowWarps * num_sms / n_kv);  // groups
    long long share = (pages + most - 1) / most;
    // (fp32 rows, apart against equal shares, us: 1 x 513 13.3/15.3, 1 x 4096 21.5/27.6, 16 x 512
    // 19.5/21.5, 8 x 2048 27.6/29.6, 16 x 1024 33.8/29.7, 32 x 1000 50.2/43.1)
    const bool apart = share <= 8;
    if (apart) {
      // A page takes a warp about 0.8 us, sixteen parts their join about 1 us: for one
      // tenant of 513 tokens 3 pages a warp and one round of joining (10.3 us in all)
      // against 4 pages (12.3 us); of 4096 tokens 4 and four (16.4) against 2 and eight (20.5).
      long long best = 0, at = share;
      for (long long s = std::max(2ll, share); s <= 8; ++s) {
        const long long parts = (longest + s - 1) / s, cost = 8 * s + (parts > 1 ? 10 * ((parts + 15) / 16) : 0);
        if (!best || cost < best) best = cost, at = s;
      }
      share = at;
    }
    struct Piece {
      int item, p0, p1, slot, parts;
    };
    std::vector<std::vector<Piece>> groups;
    long long at = 0, g = 0;  // pages handed out so far, group whose share they are in
    for (int i = 0; i < (int)small.size(); ++i) {
      const Item& it = small[i];
      const int np = blocks_of(it, kRowPage);
      std::vector<std::pair<long long, int>> cuts;  // group and end of each piece
      if (apart) {
        const int n = std::max(1, (int)((np + share - 1) / share));
        for (int q = 1; q <= n; ++q) cuts.push_back({(long long)groups.size() + q - 1, (int)((long long)np * q / n)});
      } else {
        int p = 0;
        do {
          while (g + 1 < most && pages * (g + 1) / most <= at + p) ++g;
          p = g + 1 < most ? (int)std::min<long long>(np, pages * (g + 1) / most - at) : np;
          cuts.push_back({g, p});
        } while (p < np);
      }
      const int parts = (int)cuts.size();
      const int slot = (int)out.n_slots;
      if (parts > 1)
        for (int h = 0; h < n_kv; ++h) {
          out.joins.push_back({it.row0, it.v0, it.nv, h, (int)out.n_slots, parts});
          out.n_slots += parts * it.nv;
        }
      for (int q = 0; q < parts; ++q) {
        if ((long long)groups.size() <= cuts[q].first) groups.resize(cuts[q].first + 1);
        groups[cuts[q].first].push_back({i, q ? cuts[q - 1].second : 0, cuts[q].second, parts > 1 ? slot + q * it.nv : -1, parts});
      }
      at += np;
    }
    out.small_warp.push_back(0);
    for (const auto& group : groups) {
      if (group.empty()) continue;
      for (int h = 0; h < n_kv; ++h) {
        for (const Piece& pc : group) {
          const Item& it = small[pc.item];
          AttnUnit u = unit_of(it, h, pc.p0, pc.p1, kRowPage);
          if (pc.slot >= 0) u.slot = pc.slot + h * pc.parts * it.nv;
          out.small.push_back(u);
        }
        out.small_warp.push_back((int)out.small.size());
      }
    }
  }
  // tile items: one CTA per unit, the longest first. Their keys are cut only where
  // the items are fewer than the SMs, and not below four blocks: a unit's start and
  // end cost about as much as those. (Cutting the longest of 256 uneven items as well,
  // for the balance at the end, took 257 us and 19 us of joining instead of 237 us.)
  // No unit has more than kTileBlocks: what the tensor core cuts off its running sums adds
  // up, 5e-8 of the output a product of 16 keys, to 1e-4 there, which fp16 rows have room for.
  if (!tile.empty()) {
    long long blocks = 0;
    for (const Item& it : tile) blocks += (long long)n_kv * std::max(1, blocks_of(it, kTileKeys));
    const long long seg = std::max<long long>(4, (blocks + num_sms - 1) / num_sms);
    const bool cut = (long long)tile.size() * n_kv < num_sms;
    for (const Item& it : tile) {
      const int nb = blocks_of(it, kTileKeys);
      const int fit = (nb + kTileBlocks - 1) / kTileBlocks;
      const int parts = std::max({1, fit, cut && nb > seg ? (int)((nb + seg - 1) / seg) : 1});
      for (int h = 0; h < n_kv; ++h) {
        if (parts > 1) {
          out.joins.push_back({it.row0, it.v0, it.nv, h, (int)out.n_slots, parts});
        }
        for (int p = 0; p < parts; ++p) {
          const int b0 = (int)((long long)nb * p / parts), b1 = (int)((long long)nb * (p + 1) / parts);
          AttnUnit u = unit_of(it, h, b0, b1, kTileKeys);
          if (parts > 1) {
            u.slot = (int)out.n_slots;
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
  for (const JoinItem& j : out.joins) out.join_nv = std::max(out.join_nv, j.nv);
}

}  // namespace rb
