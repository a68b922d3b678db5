"""The two attention kernels' work splits on CPU: the integer arithmetic of
``qi_b200/csrc/attn_split.h``, which the kernels compile too, walked over whole
batches the way the kernels' warps walk it (a loop in place of the lanes)."""

import ctypes
import random
import subprocess

import pytest

from qi_b200 import build

SHIM = r"""
#include "attn_split.h"
#include <cstddef>
using namespace qib;

// What a CTA is handed: sequence, query block, head item, its item, and of a cut one the record.
struct Row { int cta, seq, level, head_item; PackedItem it; PackedRecord rec; };

static PackedSpan span_of(const int* lq, const int* lk, int b) {
  PackedSpan s = {0, lq[b], 0, lk[b]};
  for (int i = 0; i < b; ++i) s.q0 += lq[i], s.k0 += lk[i];
  return s;
}

extern "C" long long seq_cost(int pair_heads, int causal, int lq, int lk, int* longest) {
  return packed_seq_cost(PackedShape{2, pair_heads, causal}, PackedSpan{0, lq, 0, lk}, *longest);
}

// Whether the batch is cut evenly, and with `rows` the items of every CTA under the even split.
extern "C" long long even_split(int n_seq, const int* lq, const int* lk, int heads, int pair_heads, int causal, int G,
                                int* even, Row* rows, long long most) {
  const PackedShape p = {heads, pair_heads, causal};
  const int head_items = packed_head_items(p);
  long long total = 0, blocks = 0, count = 0;
  int longest = 0;
  for (int b = 0; b < n_seq; ++b) {
    total += packed_seq_cost(p, span_of(lq, lk, b), longest);
    blocks += packed_blocks(p, span_of(lq, lk, b));
  }
  total *= head_items;
  *even = packed_even_split(total, blocks * head_items, longest, G, causal);
  const long long cuts = packed_cuts(total, G);
  for (int me = 0; me < G; ++me) {
    const long long lo = packed_cut_begin(total, cuts, me), hi = packed_cut_begin(total, cuts, me + 1);
    long long at = 0;
    int idle = 0;
    for (int b = 0; b < n_seq; ++b) {
      const PackedSpan s = span_of(lq, lk, b);
      for (int level = 0; level < packed_blocks(p, s); ++level) {
        const int n = packed_steps(p, s, level);
        if (n == 0) {  // zeros to write: the CTAs take turns at them
          for (int h = (me + idle) % G; h < head_items; h += G)
            if (count < most) rows[count++] = {me, b, level, h, packed_item(p, s, level, h, 0, 0, -1), {}};
          ++idle;
          continue;
        }
        for (int h = 0; h < head_items; ++h, at += packed_cost(n)) {
          const PackedCut c = packed_cut_item(at, n, lo, hi);
          if (c.from >= c.to) continue;
          Row r = {me, b, level, h, packed_item(p, s, level, h, n - c.to, n - c.from, c.part), {}};
          if (c.part >= 0) r.rec = packed_record(p, s, level, n, c.to, r.it);
          if (count < most) rows[count++] = r;
        }
      }
    }
    if (at != total) return -1;
  }
  return count;
}

extern "C" int tile_steps(int heads, int pair_heads, int causal, int lq, int lk, int level, int t) {
  return packed_tile_steps(PackedShape{heads, pair_heads, causal}, PackedSpan{0, lq, 0, lk}, level, t);
}
extern "C" int unit_count(int len, int shift) { return paged_unit_count(len, shift); }
extern "C" long long range_begin(int c, long long T, int ctas) { return paged_range_begin(c, T, paged_ranges(T, ctas)); }
extern "C" int owner(long long u, long long T, int ctas) { return paged_owner(u, T, paged_ranges(T, ctas)); }
"""

I, LL = ctypes.c_int, ctypes.c_longlong


class Item(ctypes.Structure):
    _fields_ = [("q0", I), ("lq", I), ("k0", I), ("lk", I), ("m", I * 2), ("head", I * 2), ("n", I * 2), ("diag", I),
                ("part", I), ("last", I)]


class Record(ctypes.Structure):
    _fields_ = [("used", I), ("ends", I), ("row", I * 2), ("rows", I * 2), ("head", I * 2), ("k0", I), ("end", I * 2),
                ("limit", I * 2)]


class Row(ctypes.Structure):
    _fields_ = [("cta", I), ("seq", I), ("level", I), ("head_item", I), ("it", Item), ("rec", Record)]


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("split")
    (d / "shim.cpp").write_text(SHIM)
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-I", str(build.CSRC),
                    str(d / "shim.cpp"), "-o", str(d / "shim.so")], check=True)
    so = ctypes.CDLL(str(d / "shim.so"))
    so.seq_cost.restype = so.even_split.restype = so.range_begin.restype = LL
    return so


def batch(rng):
    """Lengths, heads and CTAs; about half of the batches are such as the kernel would cut."""
    n = rng.choice((1, 1, 2, 3, 5, 12, 40))
    most = rng.choice((40, 300, 1500, 6000))
    lq = [rng.choice((0, 1, 128, 129, 256, rng.randint(1, most))) for _ in range(n)]
    lk = [max(0, a + rng.choice((0, 0, rng.randint(-a, 2 * most)))) for a in lq]
    pair = rng.randint(0, 1)
    return lq, lk, rng.choice((1, 2, 3, 5)) * (2 if pair else 1), pair, rng.randint(0, 1), rng.choice((1, 2, 7, 148))


def items_of(lib, lq, lk, heads, pair, causal, G):
    even, arr = I(0), lambda v: (I * max(1, len(v)))(*v)
    most = 400_000
    rows = (Row * most)()
    count = lib.even_split(len(lq), arr(lq), arr(lk), heads, pair, causal, G, ctypes.byref(even), rows, LL(most))
    assert 0 <= count < most
    return bool(even.value), rows[:count]


@pytest.mark.parametrize("seed", range(60))
def test_even_split_of_packed_items(lib, seed):
    """Every step of every item falls to one CTA, blocks without keys to one CTA as well; the parts of a cut item are
    those of consecutive CTAs, the first in its place 1 and the rest in place 0, no place is used twice, and the last
    part alone is marked as the end; a part's mask and record are the whole item's."""
    rng = random.Random(seed)
    lq, lk, heads, pair, causal, G = batch(rng)
    _, rows = items_of(lib, lq, lk, heads, pair, causal, G)
    block = 128 if pair else 256
    want = {(b, level, h) for b in range(len(lq)) for level in range(-(-lq[b] // block))
            for h in range(heads // 2 if pair else heads)}
    parts, places = {}, set()
    for r in rows:
        parts.setdefault((r.seq, r.level, r.head_item), []).append(r)
    assert set(parts) == want
    for (b, level, h), rs in parts.items():
        steps = [lib.tile_steps(heads, pair, causal, lq[b], lk[b], level, t) for t in (0, 1)]
        for t in (0, 1):  # as from the definition: keys that the tile's last row sees
            m = level * 128 if pair else level * 256 + 128 * t
            last = min(lq[b], m + 128) - 1
            seen = 0 if last < m else (max(0, min(lk[b], last + lk[b] - lq[b] + 1)) if causal else lk[b])
            assert steps[t] == -(-seen // 128)
        ctas = [r.cta for r in rs]
        assert ctas == list(range(ctas[0], ctas[0] + len(rs)))
        covered = [0, 0]
        for i, r in enumerate(rs):
            it = r.it
            first = (it.k0 - sum(lk[:b])) // 128  # first step of the part
            assert it.k0 - sum(lk[:b]) == 128 * first and it.lk == lk[b] - 128 * first
            for t in (0, 1):
                assert first + it.n[t] <= steps[t] or it.n[t] == 0
                covered[t] += it.n[t]
                if causal:  # the last visible key of a token is the same, counted from the sequence's first
                    assert it.diag + 128 * first == lk[b] - lq[b]
                else:  # every key: beyond lk for all tokens of a sequence, inside 32 bits
                    assert it.lk - 1 <= it.diag and it.diag + lq[b] < 1 << 31
            assert it.part == (-1 if len(rs) == 1 else (1 if i == 0 else 0))
            if it.part < 0:
                continue
            assert (r.cta, it.part) not in places
            places.add((r.cta, it.part))
            assert r.rec.used == 1 and r.rec.ends == (i == len(rs) - 1) and r.rec.k0 == sum(lk[:b])
            for t in (0, 1):
                assert r.rec.row[t] == sum(lq[:b]) + it.m[t] and r.rec.head[t] == it.head[t]
                assert r.rec.rows[t] == max(0, min(128, lq[b] - it.m[t]))
                assert r.rec.end[t] == min(lk[b], 128 * steps[t])
                if causal:
                    assert r.rec.limit[t] == it.m[t] + lk[b] - lq[b]
        assert covered == steps  # parts go from the last step to the first without a gap:
        firsts = [(r.it.k0 - sum(lk[:b])) // 128 for r in rs]
        assert firsts == sorted(firsts, reverse=True) and firsts[-1] == 0
        for a, b2 in zip(rs, rs[1:]):
            top = (b2.it.k0 - a.it.k0) // -128
            assert max(b2.it.n) == top  # the later part ends where the earlier one begins


@pytest.mark.parametrize("lq,lk,heads,pair,causal,even", [
    ([129], [9000], 2, 0, 1, True),            # few items over many keys
    ([512, 512, 300, 1000], [4608, 8192, 300, 2777], 16, 1, 1, True),
    ([16384], [16384], 24, 0, 1, False),       # many items, longest first is even enough
    ([1, 17, 600, 128], [1, 17, 600, 128], 32, 1, 1, False),
])
def test_when_packed_items_are_cut(lib, lq, lk, heads, pair, causal, even):
    assert items_of(lib, lq, lk, heads, pair, causal, 148)[0] == even


def test_cost_of_long_sequences_passes_32_bits(lib):
    """2,368 query blocks (16 for each of 148 SMs) over 2^29 keys."""
    longest = I(0)
    lq, lk = 2368 * 128, 1 << 29
    want = sum(-(-(128 * (level + 1) + lk - lq) // 128) + 2 for level in range(2368))
    assert lib.seq_cost(1, 1, lq, lk, ctypes.byref(longest)) == want > 1 << 32
    assert longest.value == (1 << 22) + 2


@pytest.mark.parametrize("seed", range(20))
def test_ranges_of_paged_units(lib, seed):
    """The ranges are those of consecutive units, none empty, and the owner of a unit is the CTA whose range holds it;
    units are counted up to the longest lengths."""
    rng = random.Random(seed)
    ctas = rng.choice((1, 3, 148))
    T = rng.choice((1, 2, ctas, rng.randint(1, 3000), rng.randint(1, 1 << 44)))
    G = min(T, ctas)
    begin = [lib.range_begin(c, LL(T), ctas) for c in range(G + 1)]
    assert begin[0] == 0 and begin[G] == T and all(a < b for a, b in zip(begin, begin[1:]))
    for c in range(G):
        for u in {begin[c], begin[c + 1] - 1, rng.randint(begin[c], begin[c + 1] - 1)}:
            assert lib.owner(LL(u), LL(T), ctas) == c
    for length in (0, 1, 15, 16, 17, 0x7fff0000, rng.randint(0, 0x7fff0000)):
        for shift in (4, 5, 6):
            assert lib.unit_count(length, shift) == -(-length // (1 << shift))
