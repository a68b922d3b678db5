// How the two attention kernels divide their work, as integer arithmetic that
// the device and the host compile alike: the kernels (attn_packed.cuh,
// attn_paged.cuh) call it lane by lane, a test on the CPU walks whole batches.
#pragma once

#if defined(__CUDACC__)
#define QIB_SPLIT __host__ __device__ __forceinline__
#else
#define QIB_SPLIT inline
#endif

namespace qib {

QIB_SPLIT int split_min(int a, int b) { return a < b ? a : b; }
QIB_SPLIT int split_max(int a, int b) { return a > b ? a : b; }

// ---------------------------------------------------------------------------
// packed sequences
// ---------------------------------------------------------------------------

struct PackedShape {
  int heads;
  int pair_heads;  // 1: an item is two heads x 128 tokens, 0: one head x 256 tokens
  int causal;
};

// First rows and lengths of a sequence (zeros behind the last one).
struct PackedSpan {
  int q0, lq, k0, lk;
};

// One work item, or the part of one that falls to a CTA, as the scheduling
// warp puts it into shared memory.
struct PackedItem {
  int q0, lq;          // first query row and length of the sequence
  int k0, lk;          // first key row of the part; keys of the sequence from there on
  int m[2], head[2];   // first token (inside the sequence) and head of the two tiles
  int n[2];            // 128-key steps of the two tiles (0: nothing visible, or no rows)
  int diag;            // last visible key of token i is i + diag (counted from k0), at most lk - 1
  int part;            // -1: whole; else the CTA's workspace place that takes the partial result
  int last;            // 1: there is no item, the CTA is done
};

// Which item a partial result belongs to; two places per CTA: 0 for an item
// that an earlier CTA begins, 1 for one that the CTA begins and a later one goes on with.
struct PackedRecord {
  int used, ends;           // there is a partial result; it is the item's last
  int row[2], rows[2], head[2];
  int k0, end[2], limit[2];  // the item's first key row; keys in its steps; last visible key of the first row
};

// Query blocks of a sequence, and items of a block.
QIB_SPLIT int packed_blocks(const PackedShape& p, const PackedSpan& s) {
  const int shift = p.pair_heads ? 7 : 8;
  return (s.lq + (1 << shift) - 1) >> shift;
}
QIB_SPLIT int packed_head_items(const PackedShape& p) { return p.pair_heads ? p.heads / 2 : p.heads; }

// 128-key steps of tile t of query block `level`.
QIB_SPLIT int packed_tile_steps(const PackedShape& p, const PackedSpan& s, int level, int t) {
  const int m = p.pair_heads ? level * 128 : level * 256 + 128 * t;
  const int rows = split_min(128, s.lq - m);
  const int visible = p.causal ? split_min(s.lk, m + rows + s.lk - s.lq) : s.lk;
  return rows > 0 && visible > 0 ? (visible + 127) / 128 : 0;
}
QIB_SPLIT int packed_steps(const PackedShape& p, const PackedSpan& s, int level) {
  return split_max(packed_tile_steps(p, s, level, 0), packed_tile_steps(p, s, level, 1));
}

// Steps [lo, hi) of an item (counted from its first key); whole where that is all of it.
QIB_SPLIT PackedItem packed_item(const PackedShape& p, const PackedSpan& s, int level, int head_item, int lo, int hi,
                                 int part) {
  PackedItem it;
  it.q0 = s.q0, it.lq = s.lq;
  it.k0 = s.k0 + lo * 128, it.lk = s.lk - lo * 128;
  for (int t = 0; t < 2; ++t) {
    it.head[t] = p.pair_heads ? 2 * head_item + t : head_item;
    it.m[t] = p.pair_heads ? level * 128 : level * 256 + 128 * t;
    it.n[t] = split_max(0, split_min(packed_tile_steps(p, s, level, t), hi) - lo);
  }
  it.diag = p.causal ? it.lk - it.lq : 0x3fffffff - s.lq;
  it.part = part;
  it.last = 0;
  return it;
}

// What an item costs beside its steps, in steps (measured: 4 us for an item of
// one step, 1.8 us for every further one).
constexpr int kPackedItemCost = 2;

// Cost of an item of n steps (without steps only zeros are written), and of one
// head item of every block of a sequence; `longest` follows the longest item.
QIB_SPLIT int packed_cost(int n) { return n > 0 ? n + kPackedItemCost : 0; }
QIB_SPLIT long long packed_seq_cost(const PackedShape& p, const PackedSpan& s, int& longest) {
  const int nb = packed_blocks(p, s);
  long long sum = 0;
  for (int level = 0; level < nb; ++level) {
    const int n = packed_steps(p, s, level);
    sum += packed_cost(n);
    longest = split_max(longest, n + kPackedItemCost);
  }
  return sum;
}

// An even split pays where the longest-first order leaves SMs idle for longer
// than writing and joining the partial results takes (about 12 us, 7 steps).
// What that order leaves idle: at most one item per CTA, the longest; equal
// items, what the last round lacks; falling lengths, about half the length of
// the last round's items.
QIB_SPLIT bool packed_even_split(long long cost, long long items, int longest, int G, int causal) {
  const long long even = cost / G;
  long long order;
  if (items <= G) order = longest;
  else if (!causal) order = (items + G - 1) / G * longest;
  else order = even + static_cast<long long>(longest) * G / (2 * items);
  return order - even > 7;
}

// The even split: the costs of all items end to end (sequences in order, blocks
// in order, heads; an item's fixed cost, then its steps from the last to the
// first), cut into equal ranges long enough for three steps, so that the parts
// of an item are those of consecutive CTAs.  Range c is [begin(c), begin(c + 1)).
QIB_SPLIT long long packed_cuts(long long total, int G) {
  const long long most = total / (kPackedItemCost + 3);
  return most < 1 ? 1 : (most < G ? most : G);
}
QIB_SPLIT long long packed_cut_begin(long long total, long long cuts, long long c) {
  return total * (c < cuts ? c : cuts) / cuts;
}
// Of an item of n steps whose cost begins at u, what the range [lo, hi) holds:
// steps [n - to, n - from), nothing where from >= to; the part's place.
struct PackedCut {
  int from, to, part;
};
QIB_SPLIT PackedCut packed_cut_item(long long u, int n, long long lo, long long hi) {
  const long long a = lo - u - kPackedItemCost, b = hi - u - kPackedItemCost;
  PackedCut c;
  c.from = static_cast<int>(a < 0 ? 0 : (a < n ? a : n));
  c.to = static_cast<int>(b < 0 ? 0 : (b < n ? b : n));
  c.part = c.from == 0 && c.to == n ? -1 : (c.from == 0 ? 1 : 0);
  return c;
}
// The record of a part that ends `to` steps from the item's end.
QIB_SPLIT PackedRecord packed_record(const PackedShape& p, const PackedSpan& s, int level, int n, int to,
                                     const PackedItem& it) {
  PackedRecord r;
  r.used = 1;
  r.ends = to == n;
  for (int t = 0; t < 2; ++t) {
    r.row[t] = it.q0 + it.m[t];
    r.rows[t] = split_max(0, split_min(128, it.lq - it.m[t]));
    r.head[t] = it.head[t];
    r.end[t] = split_min(s.lk, 128 * packed_tile_steps(p, s, level, t));
    r.limit[t] = it.m[t] + it.diag + 128 * (n - to);
  }
  r.k0 = s.k0;
  return r;
}

// ---------------------------------------------------------------------------
// paged cache
// ---------------------------------------------------------------------------

// Units of 2^shift tokens.
QIB_SPLIT int paged_unit_count(int len, int shift) {
  return static_cast<int>((static_cast<long long>(len) + (1 << shift) - 1) >> shift);
}
// Ranges that T units are cut into: none of them is empty, so the partial
// results of an item are those of consecutive CTAs.
QIB_SPLIT long long paged_ranges(long long T, int ctas) { return T < ctas ? T : ctas; }
QIB_SPLIT long long paged_range_begin(long long c, long long T, long long G) { return T * c / G; }
// CTA whose range holds unit u.
QIB_SPLIT int paged_owner(long long u, long long T, long long G) { return static_cast<int>(((u + 1) * G - 1) / T); }

}  // namespace qib
