// Host side of newton_schulz.hip: how the products are scaled and shared out.
#pragma once

#include <algorithm>
#include <array>
#include <cmath>
#include <cstdint>
#include <limits>
#include <stdexcept>
#include <vector>

#include "newton_schulz.h"

namespace lo {

constexpr int64_t kNsSide = 1 << 20;
// Blocks that run at once at two on each CU, as 128 x 128 tiles run. 64 x 64
// tiles beyond them run three a CU (ns_product_kernel's MANY); what a single
// matrix leaves over is counted in these rounds all the same.
constexpr int64_t kNsSlots = 512;

inline int64_t ns_up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

// The coefficients (a, b, c of each step) with the scales that keep every
// stored value below 2^15: with singular values in [0, s] before a step, X's
// entries stay below s, A's below s^2, C's below max |a + b q + c q^2| over
// q in [0, s^2] and the next X's below max t |a + b t^2 + c t^4| over [0, s].
// Singular values may go to 2^20 and, between steps, down to 2^-20, A's and C's
// entries to the squares of that: with coefficients of fp32 all factors of the
// products (at most sa^2 = 2^110) stay within fp32's range.
// ops.functional._ns_bounds refuses the same ones.
inline std::vector<NsStep> ns_steps(const std::vector<double>& coeffs) {
  if (coeffs.empty() || coeffs.size() % 3)
    throw std::invalid_argument(
        "coefficients come in threes, for one step at least");
  // the power of two for values up to a bound, which is 0 or from 1 / most on
  auto scale = [](double bound, double most) {
    if (!(bound < most))
      throw std::invalid_argument(
          "these coefficients let the singular values grow past 2^20, or a "
          "step's polynomial past 2^40");
    int e;
    std::frexp(std::max(bound * 1.001, 1 / most), &e);  // bound < 2^e
    return (float)std::ldexp(1.0, 15 - e);
  };
  constexpr double kX = 1l << 20, kA = 1l << 40;
  std::vector<NsStep> st(coeffs.size() / 3);
  double s = 1.001;
  float sx = scale(s, kX);
  for (size_t i = 0; i < st.size(); ++i) {
    const double a = coeffs[3 * i], b = coeffs[3 * i + 1], c = coeffs[3 * i + 2];
    const double end = s * s;
    if (s != 0 && s < 1 / kX)
      throw std::invalid_argument(
          "these coefficients let the singular values fall below 2^-20 before "
          "a step");
    for (double v : {a, b, c})
      if (!(std::abs(v) <= (double)std::numeric_limits<float>::max()))
        throw std::invalid_argument("coefficients must be finite in fp32");
    double most_c = 0, most_x = 0;
    auto try_at = [&](double q) {
      if (!(q >= 0 && q <= end)) return;
      const double v = std::abs(a + b * q + c * q * q);
      most_c = std::max(most_c, v);
      most_x = std::max(most_x, std::sqrt(q) * v);
    };
    try_at(0);
    try_at(end);
    if (c != 0) {  // where either one's derivative in q is zero
      try_at(-b / (2 * c));
      const double d = 9 * b * b - 20 * a * c;
      if (d >= 0) {
        try_at((-3 * b + std::sqrt(d)) / (10 * c));
        try_at((-3 * b - std::sqrt(d)) / (10 * c));
      }
    } else if (b != 0) {
      try_at(-a / (3 * b));
    }
    if (most_c != 0 && most_c < 1 / kA)
      throw std::invalid_argument(
          "these coefficients make a step's polynomial fall below 2^-40");
    st[i] = {(float)a, (float)b, (float)c, sx, scale(end, kA),
             scale(most_c, kA), scale(most_x, kX)};
    sx = st[i].sn;
    s = most_x * 1.001;
  }
  return st;
}

// what a plan's matrices need together
struct NsNeeds {
  int64_t halfs = 0, chunks = 0, splits = 0, parts = 0, slots = 0;
  int64_t kinds[NS_KINDS] = {};
};

inline int64_t ns_tiles(const NsMat& m, int kind) {
  const int64_t tm = m.mp / m.kind[kind].tile, tn = m.np / m.kind[kind].tile;
  return kind == NS_APPLY ? tm * tn : tm * (tm + 1) / 2;
}

inline int64_t ns_depth(const NsMat& m, int kind) {
  return (kind == NS_GRAM ? m.np : m.mp) / 32;
}

// Tile l of a product, in bands of eight tile rows, down a band's columns
// first: 64 tiles in turn read 8 + 8 panels. APPLY covers tm x tn tiles, the
// symmetric ones the lower triangle of tm x tm.
__host__ __device__ inline void ns_tile_at(int kind, int l, int tm, int tn,
                                           int& ti, int& tj) {
  int band = 0, left = 0;  // the band, and the columns left of its triangle
  if (kind == NS_APPLY) {
    if (tm > 8) band = l / (8 * tn);
    l -= band * 8 * tn;
    left = tn;
  } else if (tm > 8) {
    // band b starts at tile 32 b (b - 1) + 36 b
    band = (int)sqrtf((float)l * (1.f / 32.f));
    while (32 * band * (band - 1) + 36 * band > l) --band;
    while (32 * band * (band + 1) + 36 * (band + 1) <= l) ++band;
    l -= 32 * band * (band - 1) + 36 * band;
    left = 8 * band;
  }
  const int h = tm - 8 * band < 8 ? tm - 8 * band : 8;
  if (l < h * left) {
    tj = l / h;
    ti = 8 * band + l - tj * h;
    return;
  }
  l -= h * left;
  const int r = (l >= 1) + (l >= 3) + (l >= 6) + (l >= 10) + (l >= 15) +
                (l >= 21) + (l >= 28);
  ti = 8 * band + r;
  tj = 8 * band + l - r * (r + 1) / 2;
}

inline int64_t ns_blocks(const NsMat& m, int kind) {
  const NsTiles& k = m.kind[kind];
  return k.whole + (ns_tiles(m, kind) - k.whole) * k.splits;
}

// Whether one block's registers hold each matrix (see ns_small_kernel), given
// the largest of their short and of their long sides. In one block / by the
// products' launches, us: 16 x 16 17 / 56, 64 x 256 32 / 78, 64 x 800 66 / 81,
// 64 x 1024 74 / 75, 32 x 2048 60 / 73, 300 of 64 x 512 105 / 204
inline bool ns_fit_block(int shortest, int longest) {
  return shortest <= 32 ? longest <= 2048 : shortest <= 64 && longest <= 1024;
}

// What a tile size costs, in microseconds, to rank the choices by, fitted to
// launches of single products with 3 to 1300 tiles and 8 to 128 steps (but for
// 64's shared step, see below): a
// launch with its first loads and its end; a step of 32 values of the sum (8,
// 16 or 32 KiB of operands) in a block alone on its CU; a step and a block's
// own start and end where several blocks share one; handing over the parts of
// a split sum, for each part that the last block adds and for each part on the
// chip. So 256 x 3136 took 232 us with every sum split, 150 us with only deep
// ones split on 64 x 64 tiles, and 115 us with A and C on 32 x 32; 512 x 512
// 148 us on 64 x 64 tiles and 95 us on 32 x 32.
// A step of 64 x 64 tiles that share a CU is 0.22 us at two blocks a CU; three
// take the 0.19 here, set by whole calls and used for all such launches:
// ResNet-50's group takes 979 us with A and C on 64 x 64 tiles, 1033 us with A
// on 128 x 128; 2048 x 2048 653 us with A and C on 64 x 64, 748 us on
// 128 x 128; with 0.16, 12 x 768 x 768 went from 477 to 512 us.
struct NsCost {
  int tile;
  double launch, alone, step, block, join, add, part;
};
constexpr NsCost kNsCosts[] = {{32, 3.4, 0.10, 0.10, 0.35, 1.0, 0.3, 0.004},
                               {64, 4.1, 0.21, 0.19, 1.0, 1.0, 0.5, 0.006},
                               {128, 5.0, 1.0, 0.62, 2.0, 4.0, 1.2, 0.02}};
constexpr int64_t kNsCus = 256;

// the cost of one product over the matrices (copies of each), every sum cut
// into parts of at most `most` steps; fills in how
inline double ns_share(std::vector<NsMat>& mats, int64_t copies, int kind,
                       const NsCost& want, int64_t most) {
  double longest = 0, sum = 0, join = 0, parts = 0;
  int64_t blocks = 0;
  for (NsMat& m : mats) {
    const bool fits = m.mp % want.tile == 0 && m.np % want.tile == 0;
    const NsCost& c = fits ? want : kNsCosts[1];
    NsTiles& k = m.kind[kind];
    k.tile = c.tile;
    const int64_t tiles = ns_tiles(m, kind), depth = ns_depth(m, kind);
    const int64_t s = std::min((depth + most - 1) / most, depth / 2);
    k.splits = (int)s;
    k.whole = s > 1 ? 0 : (int)tiles;
    const double steps = (double)depth / s;
    longest = std::max(longest, steps * c.alone);
    blocks += tiles * copies * s;
    sum += (double)(tiles * copies * s) * (steps * c.step + c.block);
    if (s > 1) {
      join = std::max(join, c.join + c.add * s);
      parts += c.part * (double)(tiles * copies * s);
    }
  }
  // a CU's share: whole blocks of the average length while those are few and
  // alike (of different ones the short fill the gaps; and what is left over of
  // a single matrix's large tiles is split, see ns_plan)
  const bool even = blocks > 8 * kNsCus || mats.size() > 1 ||
                    (want.tile == 128 && copies == 1);
  const double share =
      blocks <= kNsCus ? 0
                       : (even ? (double)blocks : (double)ns_up(blocks, kNsCus)) /
                             kNsCus * (sum / blocks);
  return want.launch + std::max(longest, share) + join + parts;
}

// Shapes, and for each product the tiles and their sharing, of `copies` of
// each of the matrices: the cheapest tile size and cut of the sums for all.
inline std::vector<NsMat> ns_plan(
    const std::vector<std::pair<int64_t, int64_t>>& sides, int64_t copies) {
  int64_t big = 0;
  for (auto [rows, cols] : sides)
    big += ns_up(rows, 128) / 128 * (ns_up(cols, 128) / 128) * copies;
  std::vector<NsMat> mats;
  for (auto [rows, cols] : sides) {
    NsMat m{};
    m.rows = (int)rows;
    m.cols = (int)cols;
    // whole tiles of 128 only where there will be many of them
    const int64_t pad = big >= 256 && std::min(rows, cols) > 64 ? 128 : 64;
    m.mp = (int)ns_up(std::min(rows, cols), pad);
    m.np = (int)ns_up(std::max(rows, cols), pad);
    m.chunks = (int)(ns_up(rows * cols, kNsChunk) / kNsChunk);
    mats.push_back(m);
  }
  for (int kind = 0; kind < NS_KINDS; ++kind) {
    const NsCost* tile = &kNsCosts[1];
    int64_t cut = kNsSide;
    double best = 1e300;
    for (const NsCost& c : kNsCosts) {
      if (c.tile == 128 && big < 256) continue;
      for (int64_t most : {kNsSide, 96l, 64l, 48l, 32l, 24l, 16l, 12l, 8l}) {
        const double cost = ns_share(mats, copies, kind, c, most);
        if (cost < best) best = cost, tile = &c, cut = most;
      }
    }
    ns_share(mats, copies, kind, *tile, cut);
    // a single matrix's tiles beyond full rounds of the chip, if those are few
    NsTiles& k = mats[0].kind[kind];
    const int64_t tiles = ns_tiles(mats[0], kind), rest = tiles % kNsSlots;
    if (mats.size() * copies == 1 && k.splits == 1 && tiles > kNsSlots &&
        tiles < 4 * kNsSlots && rest) {
      const int64_t depth = ns_depth(mats[0], kind);
      const int64_t s = std::min(
          {kNsSlots / rest, (int64_t)std::sqrt((double)depth), depth / 16});
      if (s > 1) k.whole = (int)(tiles - rest), k.splits = (int)s;
    }
  }
  return mats;
}

// the size of a product's tiles, 0 where matrices differ
inline int ns_tile(const std::vector<NsMat>& mats, int kind) {
  int tile = mats[0].kind[kind].tile;
  for (const NsMat& m : mats)
    if (m.kind[kind].tile != tile) tile = 0;
  return tile;
}

// gives the matrices their places, one after the other, and adds them up (the
// products of a step run one after the other and share parts and slots)
inline void ns_place(std::vector<NsMat>& mats, NsNeeds& sum) {
  int64_t part[NS_KINDS] = {}, slot[NS_KINDS] = {};
  for (NsMat& m : mats) {
    m.ws = sum.halfs;
    m.sum = (int)sum.chunks;
    sum.halfs += 4l * m.mp * m.np + 4l * m.mp * m.mp;
    sum.chunks += m.chunks;
    sum.splits += (int64_t)(m.mp / 64) * (m.np / 64);
    for (int k = 0; k < NS_KINDS; ++k) {
      const int64_t cut = ns_tiles(m, k) - m.kind[k].whole;
      part[k] += cut * m.kind[k].splits * m.kind[k].tile * m.kind[k].tile;
      slot[k] += cut;
      sum.kinds[k] += ns_blocks(m, k);
      sum.parts = std::max(sum.parts, part[k]);
      sum.slots = std::max(sum.slots, slot[k]);
    }
  }
  const int64_t most = INT32_MAX;
  if (sum.chunks > most || sum.splits > most || sum.kinds[NS_APPLY] > most ||
      sum.kinds[NS_GRAM] > most)
    throw std::invalid_argument("too many elements for one plan");
}

// Neighbouring blocks that share a die: ResNet-50's matrices take 1042 us with
// 16, 1057 with 32, 1075 with 64, and 1114 with neighbours on all dies.
constexpr size_t kNsPiece = 16;

// The blocks of one product over placed matrices, longest sums first, so that
// none of those starts last. Blocks go to the dies in turn, so a piece of a
// matrix, some neighbouring tiles of one part of the sum, is listed eight
// places apart and meets its operands in one die's cache.
inline std::vector<NsTask> ns_tasks(const std::vector<NsMat>& mats, int kind) {
  std::vector<int> order(mats.size());
  for (size_t i = 0; i < mats.size(); ++i) order[i] = (int)i;
  auto work = [&](int i) {
    const NsMat& m = mats[i];
    const NsTiles& k = m.kind[kind];
    return ns_depth(m, kind) * k.tile * k.tile / k.splits;
  };
  std::stable_sort(order.begin(), order.end(),
                   [&](int a, int b) { return work(a) > work(b); });
  std::array<std::vector<NsTask>, 8> dies;
  std::array<int64_t, 8> load{};
  int64_t part = 0, slot = 0, count = 0;
  for (int i : order) {
    const NsMat& m = mats[i];
    const auto [tile, whole, splits] = m.kind[kind];
    const int tiles = (int)ns_tiles(m, kind), depth = (int)ns_depth(m, kind);
    std::vector<NsTask> mine;
    for (int slice = 0; slice < splits; ++slice)
      for (int l = slice ? whole : 0; l < tiles; ++l) {
        NsTask t{};
        t.ws = m.ws;
        t.mat = i;
        t.tile = tile;
        t.mp = m.mp;
        t.np = m.np;
        ns_tile_at(kind, l, m.mp / tile, m.np / tile, t.ti, t.tj);
        t.splits = l < whole ? 1 : splits;
        t.slice = slice;
        t.k1 = depth;
        if (l >= whole) {
          t.part = part + (int64_t)(l - whole) * splits * tile * tile;
          t.slot = (int)(slot + l - whole);
          t.k0 = depth / 2 * slice / splits * 2;
          t.k1 = depth / 2 * (slice + 1) / splits * 2;
        }
        mine.push_back(t);
      }
    part += (int64_t)(tiles - whole) * splits * tile * tile;
    slot += tiles - whole;
    const size_t piece = std::max<size_t>(kNsPiece, (mine.size() + 7) / 8);
    for (size_t at = 0; at < mine.size(); at += piece) {
      const size_t end = std::min(mine.size(), at + piece);
      const size_t die = std::min_element(load.begin(), load.end()) - load.begin();
      for (size_t j = at; j < end; ++j) {
        dies[die].push_back(mine[j]);
        load[die] += (int64_t)(mine[j].k1 - mine[j].k0) * tile * tile;
      }
    }
    count += (int64_t)mine.size();
  }
  std::vector<NsTask> tasks;
  std::array<size_t, 8> next{};
  while ((int64_t)tasks.size() < count) {
    size_t die = tasks.size() % 8;
    if (next[die] == dies[die].size())  // the longest queue helps out
      for (size_t d = 0; d < 8; ++d)
        if (dies[d].size() - next[d] > dies[die].size() - next[die]) die = d;
    tasks.push_back(dies[die][next[die]++]);
  }
  return tasks;
}

}  // namespace lo
