// A step's description (pages.hpp) from the accounts, on the host: its sequences, runs and split items.
#pragma once
#include <algorithm>
#include <cstdint>
#include <cstring>

#include "pages.hpp"

namespace kvq {
namespace {

// Rows of one sequence: `rows` of them behind those of the one before it, of which `count` (all or none) are described.  They are
// the tokens from `before` on, or see all of these; `seen` tokens of the slot are visible to the last one.  held: 1 where the slot
// holds the rows' tokens already, -1 where they are to come.
struct StepRows {
  int64_t slot, rows, count, before, seen;
  int held;
};

// Units of a sequence: those of its full blocks, and those of its open one
int64_t units_of(int64_t len, int64_t page) {
  const int64_t full = len / page * page;
  return (full + kUnit - 1) / kUnit + (len - full + kUnit - 1) / kUnit;
}

// Pages in front that slots a and b share, of the first `most`
int64_t shared(const int32_t* table, int64_t max_blocks, int64_t a, int64_t b, int64_t most) {
  int64_t i = 0;
  while (i < most && table[a * max_blocks + i] == table[b * max_blocks + i]) ++i;
  return i;
}

// A front is worth a run of its own from this many units on: one for each wavefront of a workgroup.
constexpr int64_t kFront = 4;
constexpr int64_t kUneven = 16;

// Fills the description of n sequences, rows_of(i) each, from the open buffers and the table; pages are written by the caller.  split_cap bounds
// the split items (those of a front weighted by the workgroups that its rows take at four query heads per KV head: the real
// number is not known here, with one or eight of them the weight is four times too large or half).
// With few_cap, the workgroups that have a CU each: of no more than few_units units there are few_cap items, unless that
// makes the longest one more than twice an even share, or there are more sequences and long ones among them; and up to twice split_cap where the longest item is kUneven units
// and 1.5 times an even share at least, and all sequences start at once (8 KV heads of 128: 64 sequences of 100 to 4000
// tokens 61 -> 54 us, but 64 of 3000 to 4000 94 -> 98, and 256 of 16 to 3000 with 16 rows each 187 -> 209).  More sequences
// than places are one item each, however long: 64 of 1000 tokens beside one of 32768 wait for its 513 units, 16 with 63.
// most_run, most_tokens: where the step has to fit a launch that was captured; fronts that do not are left out.
template <class Of>
void describe(Of&& rows_of, const uint8_t* open, const int32_t* table, int64_t max_blocks, int64_t page, int64_t n, int64_t split_cap,
              int64_t few_cap, int64_t few_units, int64_t most_run, int64_t most_tokens, int32_t* desc) {
  int64_t row = 0, item = 0, longest = 0, most_count = 0;
  bool even = true;
  for (int64_t i = 0; i < n; ++i) {
    int32_t* e = desc + kStepHead + kStepSeq * i;
    const StepRows r = rows_of(i);
    const int64_t s = r.slot, pos0 = r.before, count = r.count, end = pos0 + count;
    const int src = open[s] & 1, dst = r.held < 0 && pos0 % page && end / page > pos0 / page && end % page ? src ^ 1 : src;
    e[0] = static_cast<int32_t>(s);
    e[1] = static_cast<int32_t>(pos0);
    e[2] = static_cast<int32_t>(count);
    e[3] = static_cast<int32_t>(row);
    e[4] = static_cast<int32_t>(item);
    e[6] = src | dst << 1;
    row += r.rows;
    longest = r.rows > longest ? r.rows : longest;
    most_count = count > most_count ? count : most_count;
    item += count ? (end - 1) / page - pos0 / page + 1 : 0;
    even = even && item == i + 1;
  }
  int32_t* last = desc + kStepHead + kStepSeq * n;
  memset(last, 0, sizeof(int32_t) * kStepSeq);
  last[3] = static_cast<int32_t>(row);
  last[4] = static_cast<int32_t>(item);
  int32_t* runs = desc + kStepHead + kStepSeq * (n + 1);
  for (int fronts = 1; fronts >= 0; --fronts) {
    int64_t nr = 0, widest = most_count;
    auto add = [&](int64_t slot, int64_t row0, int64_t tokens, int64_t u0, int64_t u1, int64_t b) {
      int32_t* r = runs + kStepRun * nr++;
      r[0] = static_cast<int32_t>(slot);
      r[1] = static_cast<int32_t>(row0);
      r[2] = static_cast<int32_t>(tokens);
      r[3] = static_cast<int32_t>(u0);
      r[4] = static_cast<int32_t>(tokens ? u1 : u0);
      r[7] = static_cast<int32_t>(b);
      const int32_t* e = desc + kStepHead + kStepSeq * (b < 0 ? 0 : b);
      r[8] = b < 0 ? 0 : e[1];
      r[9] = b < 0 ? 0 : e[6] >> 1;
      r[10] = b < 0 ? 0 : e[7];
    };
    for (int64_t i = 0; i < n;) {
      const StepRows first = rows_of(i);
      int64_t j = i + 1, common = 0, tokens = first.count;
      for (; fronts && first.count && j < n && rows_of(j).count; ++j) {
        const int64_t a = first.before / page, b = rows_of(j).before / page, most = a < b ? a : b;
        const int64_t c = shared(table, max_blocks, first.slot, rows_of(j).slot, j > i + 1 && common < most ? common : most);
        if (c * page < kFront * kUnit || 2 * c < common) break;
        common = c;
        tokens += rows_of(j).count;
      }
      const int64_t front = j > i + 1 ? common * page / kUnit : 0;
      if (front) add(first.slot, desc[kStepHead + kStepSeq * i + 3], tokens, 0, front, -1);
      widest = front && tokens > widest ? tokens : widest;
      const int64_t of = front ? nr : 0;      // 1 + its index
      for (int64_t b = i; b < j; ++b) {
        int32_t* e = desc + kStepHead + kStepSeq * b;
        e[5] = static_cast<int32_t>(nr);
        e[7] = static_cast<int32_t>(of);
        const StepRows r = rows_of(b);
        add(r.slot, e[3], r.count, front, units_of(r.seen, page), b);
      }
      i = j;
    }
    int64_t most = 4;                         // a wavefront takes a unit at least
    for (int64_t i = 0; i < nr; ++i) most = runs[kStepRun * i + 4] - runs[kStepRun * i + 3] > most ? runs[kStepRun * i + 4] - runs[kStepRun * i + 3] : most;
    auto splits = [&](int64_t i, int64_t per) { return (runs[kStepRun * i + 4] - runs[kStepRun * i + 3] + per - 1) / per; };
    auto weighted = [&](int64_t per) {
      int64_t w = 0;
      for (int64_t i = 0; i < nr; ++i) w += splits(i, per) * (runs[kStepRun * i + 7] < 0 ? (runs[kStepRun * i + 2] + 3) / 4 : 1);
      return w;
    };
    auto units = [&](int64_t cap) {           // of an item, so that there are at most `cap` items
      int64_t lo = 4, hi = most;
      while (lo < hi) {
        const int64_t mid = (lo + hi) / 2;
        if (weighted(mid) <= cap) hi = mid;
        else lo = mid + 1;
      }
      return lo;
    };
    int64_t lo = units(split_cap), cap = split_cap;
    const int64_t all = weighted(1), active = [&] { int64_t c = 0; for (int64_t i = 0; i < n; ++i) c += rows_of(i).count > 0; return c; }();
    auto even_share = [&](int64_t items) { const int64_t x = (all + items - 1) / items; return x > 4 ? x : 4; };
    const int64_t few = few_cap > 0 && few_cap < split_cap && all <= few_units ? units(few_cap) : 0;
    if (few && few <= 2 * even_share(few_cap) && (few < kUneven || weighted(few) <= few_cap)) {
      lo = few;
    } else if (lo >= kUneven && active <= 2 * few_cap && 2 * lo > 3 * even_share(split_cap)) {
      cap = 2 * split_cap;
      lo = units(cap);
    }
    int64_t split = 0, base = 0;
    bool ones = true, joins = nr > n;
    for (int64_t i = 0; i < nr; ++i) {
      int32_t* r = runs + kStepRun * i;
      r[5] = static_cast<int32_t>(split);
      r[6] = static_cast<int32_t>(base);
      r[11] = static_cast<int32_t>(splits(i, lo));
      split += splits(i, lo);
      base += splits(i, lo) * r[2];
      ones = ones && splits(i, lo) == 1;
      joins = joins || splits(i, lo) > 1;
    }
    if (fronts && nr > n && (weighted(lo) > cap || widest > most_run || base > most_tokens)) continue;
    int32_t* r = runs + kStepRun * nr;
    memset(r, 0, sizeof(int32_t) * kStepRun);
    r[5] = static_cast<int32_t>(split);
    r[6] = static_cast<int32_t>(base);
    desc[0] = static_cast<int32_t>(n);
    desc[1] = static_cast<int32_t>(item);
    desc[2] = static_cast<int32_t>(split);
    desc[3] = static_cast<int32_t>(lo);
    desc[4] = even;
    desc[5] = static_cast<int32_t>(longest);
    desc[6] = static_cast<int32_t>(widest);
    desc[7] = base < INT64_C(1) << 31 ? static_cast<int32_t>(base) : -1;
    desc[8] = static_cast<int32_t>(nr);
    desc[9] = static_cast<int32_t>(kStepHead + kStepSeq * (n + 1) + kStepRun * (nr + 1));
    desc[10] = joins;
    desc[11] = ones;
    last[5] = static_cast<int32_t>(nr);
    return;
  }
}

}  // namespace
}  // namespace kvq
