// Attention of many query rows over the paged 8-bit cache: the plan on the host, and the call (kernels: paged_wide.hpp).
#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstring>
#include <functional>
#include <utility>
#include <vector>

#include "paged_wide.hpp"
#include "pages_describe.hpp"

namespace kvq {
namespace {

constexpr int64_t kSlots = 512, kMostRep = 128;

struct PlanItem {
  int32_t w[kItemWords];
};
struct PlanMerge {
  int32_t w[kMergeWords];
};
struct PlanWords {
  std::vector<PlanItem> items;
  std::vector<PlanMerge> merges;
  int64_t parts = 0, most_parts = 0;          // of a row that is joined
  int waves = 4;                              // of a workgroup: 32 rows of a tile each
};

// A tile of rows over the units [u0, u1) of a slot
struct Tile {
  int64_t row0, toks, slot, u0, u1, vis0, step, len, buf;
  int64_t front;                              // its front's first tile, or -1
  int64_t front_row0;                         // first packed row of that one
  bool joins, is_front;
  int64_t part, cut;
};

// What a call costs, in units of 64 tokens of a tile of 128 rows (2.2 us with two workgroups to a CU): the start of a tile; the
// joins' launch; a tile's sums out and in, which the places share (128 KB at 5 TB/s: 26 ns of all of them)
constexpr int64_t kStartUnits = 2, kMergeUnits = 2, kPartsPerUnit = 80, kPartUnits = 9, kLeastUnits = 3, kAloneUnits = 3;
// Rows a KV head of neighbours over shared pages that the decode's kernels take, in multiples of those of one sequence
constexpr int64_t kFewShared = 4;

int64_t units_before(int64_t tokens, int64_t len, int64_t page) {   // units of a slot that hold its first `tokens` tokens
  const int64_t full = len / page * page, u_full = (full + kUnit - 1) / kUnit;
  return tokens <= full ? (tokens + kUnit - 1) / kUnit : u_full + (tokens - full + kUnit - 1) / kUnit;
}

// Sequences of the call: rows that see all of one slot, behind one another, are one
struct Seq {
  int64_t slot, row0, count, len;
  bool wide;                                  // or few rows, for the decode's kernels
};

// Neighbours some[i .. j) that share whole pages in front which all their rows see
struct Group {
  size_t i, j;
  int64_t pages, tokens;                      // shared pages, rows' tokens
};

std::vector<Group> group(const std::vector<Seq>& some, const int32_t* table, int64_t max_blocks, int64_t page, bool causal) {
  auto whole = [&](const Seq& s) { return (causal ? s.len - s.count : s.len) / page; };
  std::vector<Group> out;
  for (size_t i = 0; i < some.size();) {
    Group g{i, i + 1, 0, some[i].count};
    for (; g.j < some.size(); ++g.j) {
      const int64_t a = whole(some[i]), b = whole(some[g.j]), most = a < b ? a : b;
      const int64_t c = shared(table, max_blocks, some[i].slot, some[g.j].slot, g.j > i + 1 && g.pages < most ? g.pages : most);
      if (c * page < kUnit || 2 * c < g.pages) break;
      g.pages = c;
      g.tokens += some[g.j].count;
    }
    out.push_back(g);
    i = g.j;
  }
  return out;
}

std::vector<Tile> tiles_for(const std::vector<Seq>& some, const std::vector<Group>& groups, const uint8_t* open, int64_t page, int64_t per_tile,
                            bool causal) {
  auto tiles_of = [&](int64_t count) { return (count + per_tile - 1) / per_tile; };
  std::vector<Tile> tiles;
  for (const Group& g : groups) {
    int64_t apart = 0, tokens = 0;
    for (size_t b = g.i; b < g.j; ++b) {
      tokens += some[b].wide ? some[b].count : 0;
      apart += some[b].wide ? tiles_of(some[b].count) : 0;
    }
    if (!tokens) continue;                    // all of a group are wide, or none
    int64_t front = g.j > g.i + 1 ? g.pages * page / kUnit : 0;
    // with a front its tiles, and joins for all of them, instead of the front's units in every sequence's tiles
    if (front && (apart - tiles_of(tokens)) * front <= kPartUnits * (apart + tiles_of(tokens))) front = 0;
    const int64_t first = static_cast<int64_t>(tiles.size()), row0 = some[g.i].row0;
    if (front)
      for (int64_t t = 0; t < tokens; t += per_tile)
        tiles.push_back({row0 + t, tokens - t < per_tile ? tokens - t : per_tile, some[g.i].slot, 0, front, front * kUnit, 0,
                         front * kUnit, 0, -1, 0, true, true, 0, 0});
    for (size_t b = g.i; b < g.j; ++b) {
      const Seq& s = some[b];
      for (int64_t t = 0; t < s.count; t += per_tile) {
        const int64_t toks = s.count - t < per_tile ? s.count - t : per_tile;
        const int64_t vis0 = causal ? s.len - s.count + t + 1 : s.len, seen = causal ? vis0 + toks - 1 : s.len;
        tiles.push_back({s.row0 + t, toks, s.slot, front, units_before(seen, s.len, page), vis0, causal ? 1 : 0, s.len, open[s.slot] & 1,
                         front ? first : -1, row0, front > 0, false, 0, 0});
      }
    }
  }
  return tiles;
}

// How the tiles are cut along the tokens: into even parts of `most` units at most, or, with the tiles' work in a row, where a place's
// share of it ends
struct Cut {
  int64_t most, share, end;                   // end: when the call is done
};
// f(first unit, end) of each part of a tile, `before` units of work behind the first; returns their number
template <class F>
int64_t parts_of(const Tile& t, const Cut& c, int64_t before, F&& f) {
  const int64_t units = t.u1 - t.u0;
  int64_t count = 0;
  if (c.share == 0) {
    count = std::max<int64_t>((units + c.most - 1) / c.most, 1);
    for (int64_t i = 0; i < count; ++i) f(units * i / count, units * (i + 1) / count);
    return count;
  }
  before += kStartUnits;
  int64_t from = 0;
  for (int64_t at = (before / c.share + 1) * c.share - before; at < units; at += c.share) {
    if (at - from < kLeastUnits || units - at < kLeastUnits) continue;
    f(from, at);
    from = at;
    ++count;
  }
  f(from, units);
  return count + 1;
}

// The way with which a call is done the earliest: the places take the longest workgroup first, each the next when it is done.  Tiles
// that are many to a place stay whole.
Cut best_cut(const std::vector<Tile>& tiles, int64_t places, int64_t H) {
  int64_t longest = 1, all = 0, work = 0;
  for (const Tile& t : tiles) {
    longest = std::max(longest, t.u1 - t.u0);
    work += t.u1 - t.u0 + kStartUnits;
    all += t.u1 - t.u0 + kStartUnits + (t.joins ? kPartUnits : 0);
  }
  const int64_t many = 4 * places;
  if (static_cast<int64_t>(tiles.size()) > many) return {longest, 0, all / places};
  Cut best{longest, 0, INT64_MAX};
  std::vector<int64_t> costs, ends(places);
  auto look = [&](Cut c) {
    costs.clear();
    int64_t parts = 0, before = 0;
    for (const Tile& t : tiles) {
      const size_t at = costs.size();
      // the kernel rounds units up to an odd number
      const int64_t count = parts_of(t, c, before, [&](int64_t a, int64_t b) { costs.push_back(((b - a) | 1) + kStartUnits); });
      before += t.u1 - t.u0 + kStartUnits;
      if (!t.joins && count == 1) continue;
      parts += count;
      for (size_t i = at; i < costs.size(); ++i) ++costs[i];
    }
    if (static_cast<int64_t>(costs.size()) > many) return false;
    std::sort(costs.begin(), costs.end(), std::greater<int64_t>());
    std::fill(ends.begin(), ends.end(), 0);
    for (int64_t x : costs) {
      std::pop_heap(ends.begin(), ends.end(), std::greater<int64_t>());
      ends.back() += x;
      std::push_heap(ends.begin(), ends.end(), std::greater<int64_t>());
    }
    c.end = *std::max_element(ends.begin(), ends.end()) + (parts ? kMergeUnits + parts * H / kPartsPerUnit : 0);
    if (c.end < best.end) best = c;
    return true;
  };
  for (int64_t k : {1, 2, 3, 4, 5, 6, 8, 10, 12, 16, 20, 24, 32, 48, 64, 96, 128}) {
    const int64_t most = (longest + k - 1) / k | 1;
    if (!look({most, 0, 0}) || most <= kLeastUnits) break;
  }
  for (int64_t k : {1, 2}) look({longest, std::max((work + k * places - 1) / (k * places), kLeastUnits), 0});
  return best;
}

// Eight wavefronts to a workgroup, one of them to a CU, widen a code for twice the rows: a unit of their 256 rows takes 0.92 of the
// time of two of 128 (32 questions of 301 to 700 tokens behind 16384, 8 KV heads of 128: 4082 -> 3748 us; four of 1613 to 2146 behind
// 10323, 4 KV heads: 691 -> 640).  But a workgroup that has a CU to itself is no faster, tiles that are not full cost twice as much, and
// nothing runs beside the start of its next one: only where the chip is full of tiles, with kAloneUnits for each start behind the first
// (six texts of three readers of 52 to 280 tokens: 31 us with 256 rows, 27 with 128).
void plan_wide(const std::vector<Seq>& some, const std::vector<Group>& groups, const uint8_t* open, int64_t page, int64_t rep, int64_t H,
               int64_t D, bool causal, PlanWords& out) {
  out.waves = 4;
  int64_t per_tile = 128 / rep;               // tokens of a tile of rows
  std::vector<Tile> tiles = tiles_for(some, groups, open, page, per_tile, causal);
  Cut cut = best_cut(tiles, std::max<int64_t>(kSlots / H, 1), H);
  if (D == 128 && static_cast<int64_t>(tiles.size()) * H >= kSlots) {
    std::vector<Tile> wider = tiles_for(some, groups, open, page, 256 / rep, causal);
    const int64_t places = std::max<int64_t>(kSlots / 2 / H, 1);
    const Cut other = best_cut(wider, places, 2 * H);
    const int64_t starts = (static_cast<int64_t>(wider.size()) + places - 1) / places;       // of a place
    if ((other.end + kAloneUnits * (starts - 1)) * 92 < cut.end * 100) {
      tiles.swap(wider);
      cut = other;
      per_tile = 256 / rep;
      out.waves = 8;
    }
  }
  int64_t before = 0;
  for (Tile& t : tiles) {
    std::vector<std::pair<int64_t, int64_t>> parts;
    t.cut = parts_of(t, cut, before, [&](int64_t a, int64_t b) { parts.push_back({a, b}); });
    before += t.u1 - t.u0 + kStartUnits;
    t.joins = t.joins || t.cut > 1;
    if (t.joins && t.u1 == t.u0) t.cut = 0;   // all of it is in the front
    t.part = out.parts;
    if (t.joins) out.parts += t.cut;
    for (int64_t c = 0; c < (t.joins ? t.cut : 1); ++c) {
      const int64_t w[kItemWords] = {t.row0, t.toks, t.slot, t.u0 + parts[c].first, t.u0 + parts[c].second, t.vis0, t.step, t.len, t.buf,
                                     t.joins ? t.part + c : -1, 0, 0};
      PlanItem it;
      for (int k = 0; k < kItemWords; ++k) it.w[k] = static_cast<int32_t>(w[k]);
      out.items.push_back(it);
    }
  }
  for (const Tile& t : tiles) {
    if (!t.joins || t.is_front) continue;
    for (int64_t a = 0; a < t.toks;) {
      int64_t toks = t.toks - a, w[kMergeWords] = {t.row0 + a, 0, t.part, t.cut, a, 0, 0, 0};
      if (t.front >= 0) {
        const int64_t at = t.row0 + a - t.front_row0, in = at % per_tile;
        const Tile& f = tiles[t.front + at / per_tile];
        toks = std::min(toks, per_tile - in);
        w[5] = f.part;
        w[6] = f.cut;
        w[7] = in;
      }
      w[1] = toks;
      out.most_parts = std::max(out.most_parts, std::max(w[3], w[6]));
      PlanMerge m;
      for (int k = 0; k < kMergeWords; ++k) m.w[k] = static_cast<int32_t>(w[k]);
      out.merges.push_back(m);
      a += toks;
    }
  }
  // the longest first: the last workgroups to end are short ones
  std::sort(out.items.begin(), out.items.end(), [](const PlanItem& x, const PlanItem& y) {
    const int32_t a = x.w[4] - x.w[3], b = y.w[4] - y.w[3];
    return a != b ? a > b : x.w[0] != y.w[0] ? x.w[0] < y.w[0] : x.w[3] < y.w[3];
  });
}

}  // namespace
}  // namespace kvq

using namespace kvq;

extern "C" int kvq_paged_plan(const int64_t* lens, const int32_t* table, const uint8_t* open, int64_t slots, int64_t max_blocks, int64_t page,
                              const int64_t* seq, const int64_t* counts, int64_t n, int64_t rep, int64_t H, int64_t D, int causal,
                              int64_t few_rows, int64_t few_work, int64_t split_cap, int64_t few_cap, int64_t few_units, int32_t* words, int64_t words_cap,
                              int64_t* info) {
  KVQ_REQUIRE(lens && table && open && info && n >= 0 && (n == 0 || (seq && counts)), "kvq_paged_plan: null pointer");
  KVQ_REQUIRE(rep >= 1 && rep <= kMostRep && H >= 1 && (D == 64 || D == 128) && (page == 32 || page == 64 || page == 128), "kvq_paged_plan: bad sizes");
  int64_t rows = 0;
  for (int64_t i = 0; i < n; ++i) {
    KVQ_REQUIRE(seq[i] >= 0 && seq[i] < slots, "kvq_paged_plan: no slot %lld (of %lld)", static_cast<long long>(seq[i]), static_cast<long long>(slots));
    KVQ_REQUIRE(counts[i] >= 0 && counts[i] < INT64_C(1) << 31, "kvq_paged_plan: counts must not be negative, and below 2^31");
    KVQ_REQUIRE(!causal || counts[i] <= lens[seq[i]], "kvq_paged_plan: slot %lld holds %lld tokens, %lld query rows are to be its last ones",
                static_cast<long long>(seq[i]), static_cast<long long>(lens[seq[i]]), static_cast<long long>(counts[i]));
    rows += counts[i];
    KVQ_REQUIRE(rows < INT64_C(1) << 31, "kvq_paged_plan: too many rows");
  }
  try {
    std::vector<Seq> some;
    int64_t row = 0;
    for (int64_t i = 0; i < n; ++i) {
      if (counts[i] > 0) {
        if (!causal && !some.empty() && some.back().slot == seq[i]) some.back().count += counts[i];
        else some.push_back({seq[i], row, counts[i], lens[seq[i]], true});
      }
      row += counts[i];
    }
    const std::vector<Group> groups = group(some, table, max_blocks, page, causal != 0);
    int64_t few = 0, wide = 0, few_units_all = 0;
    for (const Group& g : groups) {
      bool many = g.tokens * rep > (g.j > g.i + 1 ? kFewShared : 1) * few_rows;
      for (size_t b = g.i; b < g.j; ++b) many = many || some[b].count * rep > few_rows;
      for (size_t b = g.i; b < g.j; ++b) {
        some[b].wide = many;
        ++(many ? wide : few);
        few_units_all += many ? 0 : units_of(some[b].len, page) * H;
      }
    }
    // beside others that are many the launches of a few rows have to save that much
    if (wide && few && few_units_all < few_work) {
      for (Seq& s : some) s.wide = true;
      wide += few;
      few = 0;
    }
    PlanWords p;
    if (wide) plan_wide(some, groups, open, page, rep, H, D, causal != 0, p);
    KVQ_REQUIRE(p.parts < INT64_C(1) << 31, "kvq_paged_plan: too many parts");
    const int64_t m = static_cast<int64_t>(some.size());
    std::vector<int32_t> desc(few ? kStepHead + kStepSeq * (m + 1) + kStepRun * (2 * m + 1) : 0);
    if (few)
      describe([&](int64_t i) {
        const Seq& s = some[i];
        const int64_t count = s.wide ? 0 : s.count;
        // a slot without tokens has a unit all the same, whose rows come out as zeros
        return StepRows{s.slot, s.count, count, causal ? s.len - s.count : s.len, std::max<int64_t>(s.len, 1), 1};
      }, open, table, max_blocks, page, m, std::max(split_cap, m), few_cap, few_units, INT64_C(1) << 31, INT64_C(1) << 31, desc.data());
    const int64_t found[12] = {static_cast<int64_t>(p.items.size()), static_cast<int64_t>(p.merges.size()), p.parts, p.waves,
                               static_cast<int64_t>(desc.size()), few ? m : 0, few ? desc[2] : 0, few ? desc[6] : 0, few ? desc[7] : 0,
                               few ? desc[10] : 0, few ? desc[8] > m : 0, p.most_parts};
    memcpy(info, found, sizeof(found));
    KVQ_REQUIRE(!few || found[8] >= 0, "kvq_paged_plan: too many rows");
    if (!words || words_cap < kItemWords * info[0] + kMergeWords * info[1] + info[4]) return KVQ_OK;
    if (info[0]) memcpy(words, p.items.data(), sizeof(PlanItem) * p.items.size());
    if (info[1]) memcpy(words + kItemWords * info[0], p.merges.data(), sizeof(PlanMerge) * p.merges.size());
    if (few) memcpy(words + kItemWords * info[0] + kMergeWords * info[1], desc.data(), sizeof(int32_t) * desc.size());
  } catch (...) {
    KVQ_REQUIRE(false, "kvq_paged_plan: out of host memory");
  }
  return KVQ_OK;
}

extern "C" int64_t kvq_paged_attention_workspace(int64_t parts, int64_t waves, int64_t H, int64_t D) {
  return parts < 0 || H < 1 || (D != 64 && D != 128) || (waves != 4 && (waves != 8 || D != 128)) ? -1 : parts * H * 32 * waves * (D + 2);
}

extern "C" int kvq_paged_attention(const void* q, int64_t q_st, int64_t q_sh, int dtype, int64_t Hq, int64_t H, int64_t D, float scaling,
                                   const int32_t* words, int64_t items, int64_t merges, int64_t parts, int64_t most_parts, int64_t waves, const int32_t* table,
                                   int64_t max_blocks, int64_t P, int code, const uint8_t* kc, const uint8_t* vc, const float* sc,
                                   const void* ko, const void* vo, void* out, float* workspace, int64_t workspace_floats, void* stream) {
  KVQ_REQUIRE(D == 64 || D == 128, "kvq_paged_attention: head_dim must be 64 or 128 (got %lld)", static_cast<long long>(D));
  KVQ_REQUIRE(P == 32 || P == 64 || P == 128, "kvq_paged_attention: pages hold 32, 64 or 128 tokens");
  KVQ_REQUIRE(dtype == KVQ_F16 || dtype == KVQ_BF16, "kvq_paged_attention: queries must be fp16 or bf16");
  KVQ_REQUIRE(code == kCodeInt8 || code == kCodeE4M3, "kvq_paged_attention: unknown code %d", code);
  KVQ_REQUIRE(H > 0 && Hq > 0 && Hq % H == 0 && Hq / H <= kMostRep && items >= 0 && merges >= 0 && parts >= 0, "kvq_paged_attention: bad sizes");
  if (items == 0) return KVQ_OK;
  KVQ_REQUIRE(q && words && table && kc && vc && sc && ko && vo && out && (workspace || !parts), "kvq_paged_attention: null pointer");
  KVQ_REQUIRE((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(workspace)) % 16 == 0 &&
                  (q_st | q_sh) % 8 == 0,
              "kvq_paged_attention: rows and strides must be multiples of 16 bytes");
  const int64_t need = kvq_paged_attention_workspace(parts, waves, H, D);
  KVQ_REQUIRE(need >= 0, "kvq_paged_attention: workgroups of 4 wavefronts, or of 8 with head_dim 128 (got %lld)", static_cast<long long>(waves));
  KVQ_REQUIRE(workspace_floats >= need, "kvq_paged_attention: workspace of %lld floats, %lld needed",
              static_cast<long long>(workspace_floats), static_cast<long long>(need));
  // a launch counts its threads in 32 bits
  const int64_t rows = 32 * waves, join_threads = most_parts >= kSpread ? rows * 256 : rows * (D / 4);
  KVQ_REQUIRE(items <= ((INT64_C(1) << 32) - 1) / (2 * rows) / H && merges <= ((INT64_C(1) << 32) - 1) / join_threads / H && items * H < INT64_C(1) << 24,
              "kvq_paged_attention: too many rows");
  // a scaling of nothing would make a NaN of a hidden score's -inf: the smallest one, which makes zeros of the others
  const float scale = std::fabs(scaling) * 1.44269504088896341f;
  const WideArgs a{static_cast<const uint16_t*>(q), q_st, q_sh, words, table, max_blocks, static_cast<int>(H), static_cast<int>(Hq / H),
                   scale < FLT_MIN ? FLT_MIN : scale, std::signbit(scaling) ? 0x80008000u : 0u, kc, vc, sc,
                   static_cast<const uint16_t*>(ko), static_cast<const uint16_t*>(vo), static_cast<uint16_t*>(out), workspace};
  (D == 64 ? launch_wide_64 : launch_wide_128)(a, static_cast<int>(P), code, dtype == KVQ_BF16, static_cast<int>(waves), items, merges, most_parts, static_cast<hipStream_t>(stream));
  KVQ_LAUNCH_CHECK("kvq_paged_attention");
  return KVQ_OK;
}
